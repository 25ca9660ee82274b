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

// N consecutive elements of a row as they are stored; the pointer is a multiple
// of N elements' bytes.
template <typename T, int N>
struct Vec;

template <int N>
struct Vec<float, N> {
  typedef float raw_t __attribute__((ext_vector_type(N == 1 ? 2 : N), aligned(N < 4 ? 8 : 16)));
  float v[N];
  __device__ __forceinline__ void load(const float* p) {
    if constexpr (N == 1) {
      v[0] = *p;
    } else {
      const raw_t r = *reinterpret_cast<const raw_t*>(p);
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = r[i];
    }
  }
  // what is read once (nt bit): it does not push other lines out of the caches
  __device__ __forceinline__ void stream(const float* p) {
    if constexpr (N == 1) {
      v[0] = __builtin_nontemporal_load(p);
    } else {
      const raw_t r = __builtin_nontemporal_load(reinterpret_cast<const raw_t*>(p));
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = r[i];
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = 0.f;
  }
  __device__ __forceinline__ float get(int i) const { return v[i]; }
  __device__ __forceinline__ void keep() {}
  static __device__ __forceinline__ void store(float* p, const float (&x)[N]) {
    if constexpr (N == 1) {
      *p = x[0];
    } else {
      raw_t r;
#pragma unroll
      for (int i = 0; i < N; ++i) r[i] = x[i];
      *reinterpret_cast<raw_t*>(p) = r;
    }
  }
  static __device__ __forceinline__ void store_stream(float* p, const float (&x)[N]) {
    if constexpr (N == 1) {
      __builtin_nontemporal_store(x[0], p);
    } else {
      raw_t r;
#pragma unroll
      for (int i = 0; i < N; ++i) r[i] = x[i];
      __builtin_nontemporal_store(r, reinterpret_cast<raw_t*>(p));
    }
  }
};

// Two values rounded to nearest even, in one instruction.
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2_t){lo, hi}, bf16x2_t));
}

template <int N>
struct Vec<uint16_t, N> {  // N even
  static constexpr int NW = N / 2;
  typedef uint32_t raw_t __attribute__((ext_vector_type(NW == 1 ? 2 : NW), aligned(NW < 4 ? 8 : 16)));
  uint32_t w[NW];
  __device__ __forceinline__ void load(const uint16_t* p) {
    if constexpr (NW == 1) {
      w[0] = *reinterpret_cast<const uint32_t*>(p);
    } else {
      const raw_t r = *reinterpret_cast<const raw_t*>(p);
#pragma unroll
      for (int i = 0; i < NW; ++i) w[i] = r[i];
    }
  }
  __device__ __forceinline__ void stream(const uint16_t* p) {
    if constexpr (NW == 1) {
      w[0] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(p));
    } else {
      const raw_t r = __builtin_nontemporal_load(reinterpret_cast<const raw_t*>(p));
#pragma unroll
      for (int i = 0; i < NW; ++i) w[i] = r[i];
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < NW; ++i) w[i] = 0u;
  }
  __device__ __forceinline__ float get(int i) const {
    return (i & 1) ? bf16w_hi(w[i >> 1]) : bf16w_lo(w[i >> 1]);
  }
  // What get() returned before is not kept in registers for later calls: the packed
  // words are half as many.
  __device__ __forceinline__ void keep() {
#pragma unroll
    for (int i = 0; i < NW; ++i) asm volatile("" : "+v"(w[i]));
  }
  static __device__ __forceinline__ void store(uint16_t* p, const float (&x)[N]) {
    if constexpr (NW == 1) {
      *reinterpret_cast<uint32_t*>(p) = pack_bf16(x[0], x[1]);
    } else {
      raw_t r;
#pragma unroll
      for (int i = 0; i < NW; ++i) r[i] = pack_bf16(x[2 * i], x[2 * i + 1]);
      *reinterpret_cast<raw_t*>(p) = r;
    }
  }
  static __device__ __forceinline__ void store_stream(uint16_t* p, const float (&x)[N]) {
    if constexpr (NW == 1) {
      __builtin_nontemporal_store(pack_bf16(x[0], x[1]), reinterpret_cast<uint32_t*>(p));
    } else {
      raw_t r;
#pragma unroll
      for (int i = 0; i < NW; ++i) r[i] = pack_bf16(x[2 * i], x[2 * i + 1]);
      __builtin_nontemporal_store(r, reinterpret_cast<raw_t*>(p));
    }
  }
};

template <>
struct Vec<uint16_t, 1> {
  uint16_t h;
  __device__ __forceinline__ void load(const uint16_t* p) { h = *p; }
  __device__ __forceinline__ void stream(const uint16_t* p) { h = __builtin_nontemporal_load(p); }
  __device__ __forceinline__ void zero() { h = 0; }
  __device__ __forceinline__ float get(int) const { return bf16_to_f32(h); }
  __device__ __forceinline__ void keep() {}
  static __device__ __forceinline__ void store(uint16_t* p, const float (&x)[1]) {
    *p = f32_to_bf16(x[0]);
  }
  static __device__ __forceinline__ void store_stream(uint16_t* p, const float (&x)[1]) {
    __builtin_nontemporal_store(f32_to_bf16(x[0]), p);
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
