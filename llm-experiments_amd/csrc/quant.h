// The block-scaled cache formats (SKV_MXFP4, SKV_MXFP8) on gfx950, shared by
// their append and read kernels (quant_cache.hip), the decode attention
// (quant_decode.hip) and the prefill (prefill_attn.hip).
//
// 32 consecutive elements of a head's row share one scale 2^e, stored as the
// byte e + 127; an element is an E2M1 (4 bits, two to a byte, the even one in
// the low half) or E4M3 (8 bits) number c and stands for c 2^e.
//
// Writing: e is the smallest integer with max|x| <= T 2^e, T = 7 (E2M1) or 464
// (E4M3) being the largest element plus half the step below it: the smallest
// scale at which no value saturates by more than half a step, as every other
// value rounds. c = x 2^-e (exact: a power of two), clamped to the largest
// element, rounded to nearest even by the conversion instruction; so the
// stored bytes are defined bit by bit. e is at least -100 (smaller groups
// round towards zero there) and at most 125 or 119, where the largest element
// still is a finite fp32. A group that holds a NaN or an infinity takes the
// scale byte 255 and zero codes: it reads back as NaN.
//
// Reading: the conversion instructions take the scale as an fp32 operand, and
// byte << 23 is that operand for every byte: 2^e, and for 255 an exponent they
// answer with NaN (checked on MI355X for every code of both formats). c 2^e
// has at most 4 significant bits and an exponent of a normal bf16, so bf16
// holds it exactly.
#pragma once

#include "skv_common.h"

namespace skv {
namespace quant {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr int kGroup = 32;  // elements that share a scale
constexpr int kMaxD = 256;  // largest head dim
constexpr int kMaxCap = 1 << 30;  // most tokens of a sequence, so that sums with a tile stay ints

// A quantised cache of one layer. Rows are head-major: row (b, h, t) of a
// contiguous cache is (b * Hkv + h) * T_cap + t, of a paged one
// (page * Hkv + h) * page_size + t % page_size with page = bt[b * max_blocks +
// t / page_size]; a row has D * bits / 8 code bytes and D / 32 scale bytes.
// (A head's rows lie end to end because a 4-bit row is 64 bytes at head dim
// 128, half a cache line: token-major rows would make the workgroups of two
// heads fetch the same lines.)
struct Cache {
  uint8_t* k;
  uint8_t* ks;
  uint8_t* v;
  uint8_t* vs;
  const int32_t* bt;  // NULL: contiguous
  int max_blocks, bs_shift;
  int Hkv, D;
  int T_cap;
  int cap;  // tokens a sequence can hold: T_cap, or max_blocks << bs_shift
};

template <bool PAGED>
__device__ __forceinline__ size_t row_of(const Cache& c, int b, int h, int t) {
  if constexpr (PAGED) {
    const int blk = c.bt[(size_t)b * c.max_blocks + (t >> c.bs_shift)];
    return (((size_t)blk * c.Hkv + h) << c.bs_shift) + (t & ((1 << c.bs_shift) - 1));
  } else {
    return ((size_t)b * c.Hkv + h) * c.T_cap + t;
  }
}

__device__ __forceinline__ float scale_f32(uint32_t byte) { return __uint_as_float(byte << 23); }

// BITS = 4 or 8. Eight elements are NW words.
template <int BITS>
struct Fmt {
  static constexpr int NW = BITS / 4;
  static constexpr uint32_t kTopMant = BITS == 4 ? 0x600000u : 0x680000u;  // T = (1 + .) 2^kTopExp
  static constexpr int kTopExp = BITS == 4 ? 2 : 8;
  static constexpr int kMaxE = BITS == 4 ? 125 : 119;
  static constexpr float kMax = BITS == 4 ? 6.f : 448.f;
};
constexpr int kMinE = -100;

// The scale byte of a group whose largest magnitude is amax (NaN bits or
// infinity: 255).
template <int BITS>
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax_bits) {
  if (amax_bits >= 0x7f800000u) return 255u;
  // amax = m 2^x, m in [1, 2): e = x - kTopExp, one more where m exceeds T's
  // mantissa (the addition carries into the exponent exactly then)
  const int x = (int)((amax_bits + (0x7fffffu - Fmt<BITS>::kTopMant)) >> 23) - 127;
  const int e = x - Fmt<BITS>::kTopExp;
  return (uint32_t)(min(max(e, kMinE), Fmt<BITS>::kMaxE) + 127);
}

// Eight values to NW words of codes under the scale byte (255: zeros).
template <int BITS>
__device__ __forceinline__ void encode8(const float (&x)[8], uint32_t byte,
                                        uint32_t (&w)[Fmt<BITS>::NW]) {
  const float inv = __uint_as_float((254u - min(byte, 254u)) << 23);  // 2^-e
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i)
    y[i] = fminf(fmaxf(x[i] * inv, -Fmt<BITS>::kMax), Fmt<BITS>::kMax);
  if constexpr (BITS == 4) {
    uint32_t r = 0;
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, y[0], y[1], 1.f, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, y[2], y[3], 1.f, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, y[4], y[5], 1.f, 2);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, y[6], y[7], 1.f, 3);
    w[0] = byte == 255u ? 0u : r;
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      int r = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * i], y[4 * i + 1], 0, false);
      r = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * i + 2], y[4 * i + 3], r, true);
      w[i] = byte == 255u ? 0u : (uint32_t)r;
    }
  }
}

// Eight codes to bf16 (exact).
template <int BITS>
__device__ __forceinline__ bf16x8 decode8_bf16(const uint32_t* w, float s) {
  bf16x2 a, b, c, d;
  if constexpr (BITS == 4) {
    a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[0], s, 0);
    b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[0], s, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[0], s, 2);
    d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[0], s, 3);
  } else {
    a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[0], s, false);
    b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[0], s, true);
    c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[1], s, false);
    d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[1], s, true);
  }
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Eight elements of a runtime-dtype row quantised by this lane, four
// neighbouring lanes (an aligned quad, all active) holding a group: the codes
// in w, the group's scale byte returned. NaN orders above infinity as bits, so
// the integer maximum of the magnitudes finds both.
template <int BITS>
__device__ __forceinline__ uint32_t quantise8(const float (&x)[8], uint32_t (&w)[Fmt<BITS>::NW]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(x[i]) & 0x7fffffffu);
  m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, DPP_QUAD_XOR1, 0xF, 0xF, false));
  m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, DPP_QUAD_XOR2, 0xF, 0xF, false));
  const uint32_t byte = scale_byte<BITS>(m);
  encode8<BITS>(x, byte, w);
  return byte;
}

// Row `row`'s octet o (elements 8 o .. 8 o + 7) and, from its quad's first
// lane, the group's scale byte.
template <int BITS>
__device__ __forceinline__ void store8(uint8_t* codes, uint8_t* scales, size_t row, int D, int o,
                                       const uint32_t (&w)[Fmt<BITS>::NW], uint32_t byte) {
  uint8_t* p = codes + row * (size_t)(D * BITS / 8) + o * BITS;
  if constexpr (BITS == 4) *reinterpret_cast<uint32_t*>(p) = w[0];
  else *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
  if ((o & 3) == 0) scales[row * (size_t)(D / kGroup) + (o >> 2)] = (uint8_t)byte;
}

// Inclusive prefix sum over the wavefront (DPP row shifts and broadcasts).
__device__ __forceinline__ int wave_scan(int x) {
#define SKV_SCAN(CTRL, ROWS) x += __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xF, true)
  SKV_SCAN(0x111, 0xF);
  SKV_SCAN(0x112, 0xF);
  SKV_SCAN(0x114, 0xF);
  SKV_SCAN(0x118, 0xF);
  SKV_SCAN(0x142, 0xA);  // lane 15 of each row to the next row (rows 1, 3)
  SKV_SCAN(0x143, 0xC);  // lane 31 to rows 2, 3
#undef SKV_SCAN
  return x;
}

// Small host integers, one a sequence, as a kernel argument: no copy to the
// device, which would be a launch of its own (or hold the host until it landed).
constexpr int kInts = 256;
struct Ints {
  int32_t v[kInts];
};

}  // namespace quant

// ---- host ----

// skv_q_append_chunk's kernel with the counts on the device (n_new), on the host
// (n_host; copied to n_copy on the way unless that is NULL) or neither; the
// fills, which it does not advance, copied to start unless that is NULL.
int quant_append_chunk(const quant::Cache& c, int fmt, const void* k_new, const void* v_new,
                       const int32_t* lens, const int32_t* n_new, const int32_t* n_host,
                       int32_t* n_copy, int32_t* start, int B, int C, int in_dt, hipStream_t s,
                       const char* fn);

// Whether fmt is a block-scaled format.
inline bool is_quant(int fmt) { return fmt == SKV_MXFP4 || fmt == SKV_MXFP8; }

// Checks the arguments every block-scaled entry point shares and fills c.
int quant_cache_args(quant::Cache* c, void* k, void* k_scale, void* v, void* v_scale,
                     const int32_t* block_table, int max_blocks, int block_size, int B, int H_kv,
                     int D, int T_cap, int fmt, const char* fn);

}  // namespace skv
