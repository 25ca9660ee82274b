// Shared by the training kernels (train_norm.hip, train_embed.hip,
// train_loss.hip, train_adamw.hip): vectors of a runtime storage type as fp32,
// and sums and maxima over a wavefront or a workgroup.
#pragma once

#include <type_traits>

#include "skv_common.h"

namespace skv {
namespace train {

typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));

// Two values rounded to nearest even, in one instruction.
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2_t){lo, hi}, bf16x2_t));
}

// N consecutive elements of a row as they are stored (T float, or uint16_t for bf16),
// N elements a power of two of words. load, stream and store take aligned vectors,
// load_any and store_any those at any element (gfx950 reads and writes them as they are).
// load_row and stream_row read elements j .. j + N of a row of d, zeros past its end, j a
// multiple of N below d. Where rows are no multiple of N elements (kOdd), a vector that
// would leave its row is the row's last N elements instead, and settle(), called before the
// values are used, shifts it to its place: no load waits for another. Rows below N
// elements (kTiny) are read one by one. stream and store_stream carry the nt bit: what is
// read or written once does not push other lines out of the caches.
enum RowKind { kEven, kOdd, kTiny };
inline RowKind row_kind(int d, int N) { return d % N == 0 ? kEven : d > N ? kOdd : kTiny; }

template <typename T, int N>
struct Vec {
  static constexpr bool kF32 = sizeof(T) == 4;
  static constexpr int NW = N * (int)sizeof(T) / 4;  // words
  typedef uint32_t raw_t __attribute__((ext_vector_type(NW), aligned(NW < 4 ? NW * 4 : 16)));
  typedef uint32_t any_t __attribute__((ext_vector_type(NW), aligned(sizeof(T))));
  uint32_t w[NW];

  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < NW; ++i) w[i] = 0u;
  }
  template <typename R>
  __device__ __forceinline__ void set(R r) {
#pragma unroll
    for (int i = 0; i < NW; ++i) w[i] = r[i];
  }
  __device__ __forceinline__ void load(const T* p) { set(*reinterpret_cast<const raw_t*>(p)); }
  __device__ __forceinline__ void load_any(const T* p) { set(*reinterpret_cast<const any_t*>(p)); }
  __device__ __forceinline__ void stream(const T* p) {
    set(__builtin_nontemporal_load(reinterpret_cast<const raw_t*>(p)));
  }
  template <int KIND>
  __device__ __forceinline__ void load_row(const T* row, int j, int d) {
    if constexpr (KIND == kEven) load(row + j);
    else if constexpr (KIND == kOdd) load_any(row + min(j, d - N));
    else load_part(row + j, d - j);
  }
  template <int KIND>
  __device__ __forceinline__ void stream_row(const T* row, int j, int d) {
    if constexpr (KIND == kEven) stream(row + j);
    else if constexpr (KIND == kOdd)
      set(__builtin_nontemporal_load(reinterpret_cast<const any_t*>(row + min(j, d - N))));
    else load_part(row + j, d - j);
  }
  template <int KIND>
  __device__ __forceinline__ void settle(int j, int d) {
    if constexpr (KIND == kOdd) {
      if (j > d - N) shift(j - (d - N));
    }
  }
  // element i becomes element i + by, zeros past the last
  __device__ __forceinline__ void shift(int by) {
    if constexpr (!kF32) {
      if (by & 1) {
#pragma unroll
        for (int i = 0; i < NW; ++i) w[i] = (w[i] >> 16) | (i + 1 < NW ? w[i + 1] << 16 : 0u);
      }
      by >>= 1;
    }
#pragma unroll
    for (int s = 1; s < NW; s <<= 1) {
      if (by & s) {
#pragma unroll
        for (int i = 0; i < NW; ++i) w[i] = i + s < NW ? w[i + s] : 0u;
      }
    }
  }
  __device__ __forceinline__ void load_part(const T* p, int left) {
    T x[N];
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = i < left ? p[i] : T(0);
#pragma unroll
    for (int i = 0; i < NW; ++i) {
      if constexpr (kF32) w[i] = __float_as_uint(x[i]);
      else w[i] = (uint32_t)x[2 * i] | ((uint32_t)x[2 * i + 1] << 16);
    }
  }
  __device__ __forceinline__ float get(int i) const {
    if constexpr (kF32) return __uint_as_float(w[i]);
    else return (i & 1) ? bf16w_hi(w[i >> 1]) : bf16w_lo(w[i >> 1]);
  }
  // What get() returned before is not kept in registers for later calls: the packed
  // words of bf16 are half as many.
  __device__ __forceinline__ void keep() {
    if constexpr (!kF32) {
#pragma unroll
      for (int i = 0; i < NW; ++i) asm volatile("" : "+v"(w[i]));
    }
  }
  // The load of the words has ended.
  __device__ __forceinline__ void arrive() {
#pragma unroll
    for (int i = 0; i < NW; ++i) asm volatile("" ::"v"(w[i]));
  }
  template <typename R>
  static __device__ __forceinline__ R words(const float (&x)[N]) {
    R r;
#pragma unroll
    for (int i = 0; i < NW; ++i) {
      if constexpr (kF32) r[i] = __float_as_uint(x[i]);
      else r[i] = pack_bf16(x[2 * i], x[2 * i + 1]);
    }
    return r;
  }
  static __device__ __forceinline__ void store(T* p, const float (&x)[N]) {
    *reinterpret_cast<raw_t*>(p) = words<raw_t>(x);
  }
  static __device__ __forceinline__ void store_any(T* p, const float (&x)[N]) {
    *reinterpret_cast<any_t*>(p) = words<any_t>(x);
  }
  static __device__ __forceinline__ void store_stream(T* p, const float (&x)[N]) {
    __builtin_nontemporal_store(words<raw_t>(x), reinterpret_cast<raw_t*>(p));
  }
  template <int KIND>
  static __device__ __forceinline__ void store_row(T* row, int j, int d, const float (&x)[N]) {
    if constexpr (KIND == kEven) store(row + j, x);
    else if (j + N <= d) store_any(row + j, x);
    else store_part(row + j, x, d - j);
  }
  template <int KIND>
  static __device__ __forceinline__ void store_stream_row(T* row, int j, int d,
                                                          const float (&x)[N]) {
    if constexpr (KIND == kEven) store_stream(row + j, x);
    else if (j + N <= d)
      __builtin_nontemporal_store(words<any_t>(x), reinterpret_cast<any_t*>(row + j));
    else store_part(row + j, x, d - j);
  }
  static __device__ __forceinline__ void store_part(T* p, const float (&x)[N], int left) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (i < left) {
        if constexpr (kF32) p[i] = x[i];
        else p[i] = f32_to_bf16(x[i]);
      }
    }
  }
};

// Every lane gets the sum (maximum) over the wavefront, the same bits in all.
__device__ __forceinline__ float xor16_sum(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false,
                                                  false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float xor16_max(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false,
                                                  false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float wave_sum(float x) { return xor32_sum(xor16_sum(row16_sum(x))); }
__device__ __forceinline__ float wave_max(float x) { return xor32_max(xor16_max(row16_max(x))); }

// Whether a launch can have so many workgroups: fewer than 2^32 lanes.
inline bool launchable(size_t groups, int lanes) { return groups * lanes < (size_t)1 << 32; }

constexpr int kMaxRows = 1 << 30;  // rows that a kernel's 32-bit loops pass over

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// An operand's memory (p NULL: there is none). may_be: the number of an output that
// may be the same buffer, or -1.
struct Span {
  const void* p;
  size_t bytes;
  const char* name;
  int may_be = -1;
};

// An error if an output overlaps another output or an input that it may not be.
template <int NO, int NI>
int apart(const char* fn, const Span (&out)[NO], const Span (&in)[NI]) {
  const auto over = [](const Span& a, const Span& b) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a.p), y = reinterpret_cast<uintptr_t>(b.p);
    return x && y && x < y + b.bytes && y < x + a.bytes;
  };
  for (int i = 0; i < NO; ++i) {
    for (int j = i + 1; j < NO; ++j)
      SKV_REQUIRE(!over(out[i], out[j]), SKV_E_INVALID, "%s: %s overlaps %s", fn, out[i].name,
                  out[j].name);
    for (int j = 0; j < NI; ++j)
      SKV_REQUIRE(!over(out[i], in[j]) || (in[j].may_be == i && in[j].p == out[i].p), SKV_E_INVALID,
                  "%s: %s overlaps %s", fn, out[i].name, in[j].name);
  }
  return SKV_OK;
}

}  // namespace train
}  // namespace skv
