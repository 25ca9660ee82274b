// One AdamW step of every tensor of a model in one launch.
//
//   m' = b1 m + (1 - b1) g,  v' = b2 v + (1 - b2) g^2
//   p' = p (1 - lr wd) - lr / (1 - b1^t) m' / (sqrt(v' / (1 - b2^t)) + eps)
//
// Bound by HBM: 28 bytes an element with fp32 gradients and moments. The tensors
// are cut into chunks of 4096 elements, a table on the device names each chunk's
// tensor, and one workgroup of 512 lanes a CU walks over the chunks, the next
// chunk's place read ahead. More workgroups are slower, in HBM (203 million elements,
// bf16 gradients and copies: 1101 us = 5.15 TB/s with 256 x 512 lanes, 1129 with 512 x
// 512, 1170 with 1024 x 256; a copy runs at 4.71 TB/s read and write) and for their
// arrivals below (3.2 million elements: 16.5, 18.8 and 22.7 us).
// Vectors lie at any element: 33.5 million elements in tensors that begin 4 bytes behind a
// 16-byte granule take 215 us, 208 at its begin, and 256 element by element.
//
// The step count t is in device memory, so that a captured step counts on when
// it is replayed: every workgroup reads t before it does anything, and the last
// one to finish (an arrival counter that it sets back to zero) writes t + 1.
//
// 8-bit moments. Blocks of 128 consecutive elements of a tensor share a scale
// 2^k in a byte, k + 127; k is the exponent of the block's largest magnitude,
// clamped to [-90, 126]. A block with a NaN or an infinity takes the byte 255 and
// zero codes, and reads back as NaN.
//   m: sign and E4M3, y = m 2^(7 - k): the largest lies in [128, 256) of 448
//   v: no sign, 5 exponent and 3 mantissa bits, y = v 2^-k: the largest in [1, 2),
//      the smallest step 2^-32. A v above zero never takes the code 0: m / eps would
//      be a step of any size
// With b2 = 0.999 a v that moves by a thousandth stays where it is if it is
// rounded to the nearest of steps of a sixteenth, for ever; so both moments are
// rounded up or down at random, in proportion. The random bits are a hash of
// (seed, t, place in the state): the same state and gradients give the same bits.
// All of it is exact but for b1 m + (1 - b1) g and its like, whose products and
// sum are rounded one by one.
#include <math.h>

#include "train_common.h"

namespace skv {
namespace {

using namespace train;

constexpr int kThreads = 512;
constexpr int kChunk = kThreads * 8;  // elements of a workgroup and turn
constexpr int kBlock = 128;   // elements that share a scale: 16 lanes of 8

struct Tensor {  // skv_adamw_tensor
  float* p;
  const void* g;
  uint16_t* copy;
  int64_t n;   // elements
  int64_t at;  // its first element's place in the state, a multiple of kBlock
  int64_t decay;
};

struct Step {
  int n_chunks;
  void* m;
  void* v;
  uint8_t* m_scale;
  uint8_t* v_scale;
  int32_t* count;  // t, then the arrivals
  double log_b1, log_b2;  // log(beta1), log(beta2)
  float b1, omb1, b2, omb2;  // beta1, 1 - beta1, ..., each rounded from 64 bits
  float lr, weight_decay, eps, grad_scale;
  const float* lr_dev;          // in place of lr, or NULL
  const float* grad_scale_dev;  // in place of grad_scale, or NULL
  uint32_t seed;
};

constexpr uint32_t kMul1 = 0x9E3779B9u, kMul2 = 0x6A09E667u, kMul3 = 0xBB67AE85u;

__device__ __forceinline__ uint32_t hash_key(uint32_t seed, uint32_t t) {
  uint32_t w = seed * kMul1 + t * kMul2;
  w = (w ^ (w >> 15)) * kMul3;
  return w ^ (w >> 16);
}
__device__ __forceinline__ uint32_t hash_mix(uint32_t u) {  // u = place * kMul1 + key
  u = (u ^ (u >> 15)) * kMul2;
  return u ^ (u >> 16);
}

// The block's exponent k + 127 of the bits of its largest magnitude, 255 if it is
// not finite.
__device__ __forceinline__ uint32_t block_byte(uint32_t amax_bits) {
  const int k = (int)(amax_bits >> 23);
  return k >= 255 ? 255u : (uint32_t)min(max(k, 127 - 90), 127 + 126);
}

__device__ __forceinline__ uint32_t row16_umax(uint32_t x) {
  const auto step = [&](auto ctrl) {
    const uint32_t y = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, ctrl.value, 0xF, 0xF, false);
    x = x > y ? x : y;
  };
  step(std::integral_constant<int, DPP_QUAD_XOR1>{});
  step(std::integral_constant<int, DPP_QUAD_XOR2>{});
  step(std::integral_constant<int, DPP_ROW_HALF_MIRROR>{});
  step(std::integral_constant<int, DPP_ROW_MIRROR>{});
  return x;
}

__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// A magnitude y to a code with 3 mantissa bits, up or down by 16 random bits. LOW:
// the exponent of the smallest normal number. Below it the sum with 2^LOW holds y
// as a fixed-point number in steps of the subnormals'.
template <int LOW>
__device__ __forceinline__ uint32_t round_code(float y, uint32_t r16) {
  constexpr float kLow = LOW == -6 ? 0x1p-6f : 0x1p-29f;
  constexpr uint32_t kFirst = (uint32_t)(LOW + 127) << 3;  // the code of 2^LOW is 8
  const bool small = y < kLow;
  const uint32_t b = __float_as_uint(small ? y + kLow : y) + (r16 << 4) + 8u;
  return (b >> 20) - (small ? kFirst : kFirst - 8);
}

__device__ __forceinline__ uint32_t code_m(float m, float enc, uint32_t r16) {
  const float y = m * enc;
  const uint32_t c = round_code<-6>(fabsf(y), r16);
  return min(c, 126u) | (__float_as_uint(y) >> 31 << 7);
}
__device__ __forceinline__ uint32_t code_v(float v, float enc, uint32_t r16) {
  const uint32_t c = min(round_code<-29>(v * enc, r16), 255u);
  return v > 0.f ? max(c, 1u) : c;
}
// Codes back: their bits are an fp32's exponent and mantissa, but for its bias.
__device__ __forceinline__ float value_m(uint32_t c, float dec) {
  const float y = __uint_as_float((c & 127u) << 20) * 0x1p120f;
  return __uint_as_float(__float_as_uint(y) | (c >> 7 << 31)) * dec;
}
__device__ __forceinline__ float value_v(uint32_t c, float dec) {
  return __uint_as_float(c << 20) * 0x1p97f * dec;
}
__device__ __forceinline__ float dec_m(uint32_t byte) {
  return byte == 255u ? NAN : pow2((int)byte - 127 - 7);
}
__device__ __forceinline__ float dec_v(uint32_t byte) {
  return byte == 255u ? NAN : pow2((int)byte - 127);
}

constexpr float kLowV = 0x1p-126f;  // the least normal number

struct Coef {
  float b1, omb1, b2, omb2, step, root, eps, keep, gs;
};

// products and sums rounded one by one: moments are the same bits in every build
// of the formula
__device__ __forceinline__ void moments(float& m, float& v, float g, const Coef& c) {
#pragma clang fp contract(off)
  const float m1 = c.b1 * m, m2 = c.omb1 * g;
  m = m1 + m2;
  const float g2 = g * g;
  const float v1 = c.b2 * v, v2 = c.omb2 * g2;
  v = v1 + v2;
}

// p (1 - lr wd) - step m / (sqrt(v) root + eps): square root and quotient on the
// hardware's units, 1 ulp each. LOW: some v may be subnormal, which that root takes
// for 0; v is taken 2^64 up, exactly, and its root 2^32 down.
template <bool LOW>
__device__ __forceinline__ float stepped(float p, float m, float v, const Coef& c, float keep) {
  const bool low = LOW && v < kLowV;
  const float root = low ? __builtin_amdgcn_sqrtf(v * 0x1p64f) * 0x1p-32f : __builtin_amdgcn_sqrtf(v);
  return p * keep - c.step * m * __builtin_amdgcn_rcpf(fmaf(root, c.root, c.eps));
}

// E elements of a tensor from i0 on, zeros past its end.
template <int E>
__device__ __forceinline__ void load_f32(float (&x)[E], const float* p, bool vec, int left) {
  if (vec) {
    Vec<float, E> v;
    v.load_any(p);
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = v.get(e);
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = e < left ? p[e] : 0.f;
  }
}
template <int E>
__device__ __forceinline__ void load_f32(float (&x)[E], const uint16_t* p, bool vec, int left) {
  if (vec) {
    Vec<uint16_t, E> v;
    v.load_any(p);
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = v.get(e);
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = e < left ? bf16_to_f32(p[e]) : 0.f;
  }
}
template <int E>
__device__ __forceinline__ void store_f32(float* p, const float (&x)[E], bool vec, int left) {
  if (vec) {
    Vec<float, E>::store_any(p, x);
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (e < left) p[e] = x[e];
  }
}
template <int E>
__device__ __forceinline__ void store_bf16(uint16_t* p, const float (&x)[E], bool vec, int left) {
  if (vec) {
    Vec<uint16_t, E>::store_any(p, x);
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (e < left) p[e] = f32_to_bf16(x[e]);
  }
}

// One chunk of a tensor. BITS of a moment; TG: how gradients are stored. A lane has E
// consecutive elements at a time: 4 of them where the moments are fp32, so that every
// load of a wavefront is 1 KB in a row, and 8 where they are bytes. FULL: the chunk
// lies inside the tensor. All loads come before any store: the compiler cannot tell the
// tensors apart.
template <typename TG, int BITS, bool FULL>
__device__ __forceinline__ void step_chunk(const Step& a, const Tensor& x, int chunk, const Coef& c,
                                           uint32_t key) {
  constexpr int E = BITS == 32 ? 4 : 8, kParts = 8 / E;
  const float keep = x.decay ? c.keep : 1.f;
  // a tensor's place in the state is filled up to whole blocks
  const int64_t blocks_end = (x.n + kBlock - 1) / kBlock * kBlock;
  float p[kParts][E], g[kParts][E], m[kParts][E], v[kParts][E];
  const auto first = [&](int part) {
    return (int64_t)chunk * kChunk + part * kThreads * E + threadIdx.x * E;
  };
  const auto left_of = [&](int part) {
    return FULL ? E : (int)min((int64_t)E, max((int64_t)0, x.n - first(part)));
  };
#pragma unroll
  for (int part = 0; part < kParts; ++part) {
    const int64_t i0 = first(part);
    const size_t at = (size_t)(x.at + i0);  // in the state
    const int left = left_of(part);
    const bool whole = FULL || left == E, here = FULL || i0 < blocks_end;
    load_f32<E>(p[part], x.p + i0, whole, left);
    load_f32<E>(g[part], (const TG*)x.g + i0, whole, left);
    if constexpr (BITS == 32) {
      load_f32<E>(m[part], (const float*)a.m + at, here, 0);
      load_f32<E>(v[part], (const float*)a.v + at, here, 0);
    } else {
      uint2 wm = make_uint2(0, 0), wv = make_uint2(0, 0);
      uint32_t bm = 0, bv = 0;
      if (here) {
        wm = *reinterpret_cast<const uint2*>((const uint8_t*)a.m + at);
        wv = *reinterpret_cast<const uint2*>((const uint8_t*)a.v + at);
        bm = a.m_scale[at / kBlock];
        bv = a.v_scale[at / kBlock];
      }
      const float dm = dec_m(bm), dv = dec_v(bv);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        m[part][e] = value_m(((e < 4 ? wm.x : wm.y) >> (8 * (e & 3))) & 255u, dm);
        v[part][e] = value_v(((e < 4 ? wv.x : wv.y) >> (8 * (e & 3))) & 255u, dv);
      }
    }
  }
#pragma unroll
  for (int part = 0; part < kParts; ++part) {
    const int64_t i0 = first(part);
    const size_t at = (size_t)(x.at + i0);
    const int left = left_of(part);
    const bool whole = FULL || left == E, here = FULL || i0 < blocks_end;
#pragma unroll
    for (int e = 0; e < E; ++e) moments(m[part][e], v[part][e], g[part][e] * c.gs, c);
    // a branch for all of a lane's elements: chosen element by element, 3.1 million of them
    // with 8-bit moments take 14.6 us, 14.2 so
    float least = v[part][0];
#pragma unroll
    for (int e = 1; e < E; ++e) least = fminf(least, v[part][e]);
    const auto step = [&](auto LOW) {
#pragma unroll
      for (int e = 0; e < E; ++e)
        p[part][e] = stepped<LOW.value>(p[part][e], m[part][e], v[part][e], c, keep);
    };
    if (least < kLowV) step(std::true_type{});
    else step(std::false_type{});
    store_f32<E>(x.p + i0, p[part], whole, left);
    if (x.copy) store_bf16<E>(x.copy + i0, p[part], whole, left);
    if constexpr (BITS == 32) {
      store_f32<E>((float*)a.m + at, m[part], whole, left);
      store_f32<E>((float*)a.v + at, v[part], whole, left);
    } else {
      uint32_t am = 0, av = 0;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        if (e >= left) m[part][e] = v[part][e] = 0.f;  // a block read back as NaN has them too
        am = max(am, __float_as_uint(m[part][e]) & 0x7fffffffu);
        av = max(av, __float_as_uint(v[part][e]));
      }
      am = row16_umax(am);
      av = row16_umax(av);
      const uint32_t bm = block_byte(am), bv = block_byte(av);
      const float em = pow2(127 + 7 - (int)min(bm, 253u)), ev = pow2(127 - (int)min(bv, 253u));
      uint32_t u = (uint32_t)at * kMul1 + key;
      uint32_t wm[2] = {0, 0}, wv[2] = {0, 0};
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const uint32_t h = hash_mix(u);
        u += kMul1;
        wm[e / 4] |= code_m(m[part][e], em, h & 0xffffu) << (8 * (e & 3));
        wv[e / 4] |= code_v(v[part][e], ev, h >> 16) << (8 * (e & 3));
      }
      if (here) {
        *reinterpret_cast<uint2*>((uint8_t*)a.m + at) =
            bm == 255u ? make_uint2(0, 0) : make_uint2(wm[0], wm[1]);
        *reinterpret_cast<uint2*>((uint8_t*)a.v + at) =
            bv == 255u ? make_uint2(0, 0) : make_uint2(wv[0], wv[1]);
        if ((threadIdx.x & 15) == 0) {
          a.m_scale[at / kBlock] = (uint8_t)bm;
          a.v_scale[at / kBlock] = (uint8_t)bv;
        }
      }
    }
  }
}

// tensors, chunks: (tensor, its chunk). The next chunk's tensor is known before this
// chunk's data are waited for.
template <typename TG, int BITS>
__global__ __launch_bounds__(kThreads) void k_adamw(Step a, const Tensor* __restrict__ tensors,
                                                    const int2* __restrict__ chunks) {
  int ch = blockIdx.x;
  int2 which = chunks[ch];
  Tensor x = tensors[which.x];
  const int t = a.count[0] + 1;
  Coef c;
  c.b1 = a.b1;
  c.omb1 = a.omb1;
  c.b2 = a.b2;
  c.omb2 = a.omb2;
  c.eps = a.eps;
  {
    const float lr = a.lr_dev ? *a.lr_dev : a.lr;
    c.step = lr / -expm1f((float)(t * a.log_b1));
    c.root = 1.f / sqrtf(-expm1f((float)(t * a.log_b2)));
    c.keep = fmaf(-lr, a.weight_decay, 1.f);
    c.gs = a.grad_scale_dev ? *a.grad_scale_dev : a.grad_scale;
  }
  const uint32_t key = hash_key(a.seed, (uint32_t)t);
  for (;;) {
    const int after = ch + gridDim.x;
    const int2 next = chunks[min(after, a.n_chunks - 1)];
    const Tensor next_x = tensors[next.x];
    if ((int64_t)(which.y + 1) * kChunk <= x.n)
      step_chunk<TG, BITS, true>(a, x, which.y, c, key);
    else
      step_chunk<TG, BITS, false>(a, x, which.y, c, key);
    if (after >= a.n_chunks) break;
    ch = after;
    which = next;
    x = next_x;
  }
  __syncthreads();  // every lane has read the count
  if (threadIdx.x == 0 && atomicAdd(a.count + 1, 1) == (int)gridDim.x - 1) {
    a.count[0] = t;
    a.count[1] = 0;
  }
}

// 8-bit moments as values: 8 a lane.
template <typename T>
__global__ __launch_bounds__(256) void k_adamw_read(T* __restrict__ m_out, T* __restrict__ v_out,
                                                    const uint8_t* __restrict__ m,
                                                    const uint8_t* __restrict__ v,
                                                    const uint8_t* __restrict__ m_scale,
                                                    const uint8_t* __restrict__ v_scale, size_t n) {
  const size_t at = ((size_t)blockIdx.x * 256 + threadIdx.x) * 8;
  if (at >= n) return;
  const uint2 wm = *reinterpret_cast<const uint2*>(m + at);
  const uint2 wv = *reinterpret_cast<const uint2*>(v + at);
  const float dm = dec_m(m_scale[at / kBlock]), dv = dec_v(v_scale[at / kBlock]);
  float xm[8], xv[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    xm[e] = value_m(((e < 4 ? wm.x : wm.y) >> (8 * (e & 3))) & 255u, dm);
    xv[e] = value_v(((e < 4 ? wv.x : wv.y) >> (8 * (e & 3))) & 255u, dv);
  }
  Vec<T, 8>::store(m_out + at, xm);
  Vec<T, 8>::store(v_out + at, xv);
}

static_assert(sizeof(Tensor) == sizeof(skv_adamw_tensor), "skv_adamw_tensor");

}  // namespace
}  // namespace skv

using namespace skv;

extern "C" int skv_adamw(const skv_adamw_tensor* tensors, const int32_t* chunks, int n_chunks,
                         void* m, void* v, uint8_t* m_scale, uint8_t* v_scale, int32_t* count,
                         int bits, int grad_dt, double lr, const float* lr_dev, double beta1,
                         double beta2, double eps, double weight_decay, double grad_scale,
                         const float* grad_scale_dev, uint32_t seed, skv_stream_t stream) {
  SKV_REQUIRE(tensors && chunks && m && v && count, SKV_E_INVALID,
              "skv_adamw: null pointer argument");
  SKV_REQUIRE(bits == 32 || bits == 8, SKV_E_INVALID, "skv_adamw: bits must be 32 or 8, got %d",
              bits);
  SKV_REQUIRE(bits == 32 || (m_scale && v_scale), SKV_E_INVALID,
              "skv_adamw: null pointer argument");
  SKV_REQUIRE(n_chunks > 0, SKV_E_INVALID, "skv_adamw: n_chunks must be > 0");
  SKV_REQUIRE(n_chunks <= kMaxRows, SKV_E_UNSUPPORTED, "skv_adamw: n_chunks=%d > 2^30", n_chunks);
  SKV_REQUIRE(grad_dt == SKV_F32 || grad_dt == SKV_BF16, SKV_E_INVALID, "skv_adamw: bad dtype");
  SKV_REQUIRE(beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1, SKV_E_INVALID,
              "skv_adamw: beta1 and beta2 must lie in [0, 1)");
  // a subnormal one would be taken for 0: 0 / eps a NaN
  SKV_REQUIRE(eps == 0 || eps >= 0x1p-126, SKV_E_INVALID,
              "skv_adamw: eps must be 0 or at least 2^-126");
  SKV_REQUIRE(aligned16(m) && aligned16(v), SKV_E_INVALID,
              "skv_adamw: the state must be 16-byte aligned");
  Step a;
  a.n_chunks = n_chunks;
  a.m = m;
  a.v = v;
  a.m_scale = m_scale;
  a.v_scale = v_scale;
  a.count = count;
  a.log_b1 = log(beta1);
  a.log_b2 = log(beta2);
  a.b1 = (float)beta1;
  a.omb1 = (float)(1.0 - beta1);
  a.b2 = (float)beta2;
  a.omb2 = (float)(1.0 - beta2);
  a.lr = (float)lr;
  a.weight_decay = (float)weight_decay;
  a.eps = (float)eps;
  a.grad_scale = (float)grad_scale;
  a.lr_dev = lr_dev;
  a.grad_scale_dev = grad_scale_dev;
  a.seed = seed;
  const Tensor* x = (const Tensor*)tensors;
  const int2* ch = (const int2*)chunks;
  const dim3 grid(n_chunks < 256 ? n_chunks : 256);
  hipStream_t s = (hipStream_t)stream;
  if (bits == 32) {
    if (grad_dt == SKV_BF16) k_adamw<uint16_t, 32><<<grid, kThreads, 0, s>>>(a, x, ch);
    else k_adamw<float, 32><<<grid, kThreads, 0, s>>>(a, x, ch);
  } else {
    if (grad_dt == SKV_BF16) k_adamw<uint16_t, 8><<<grid, kThreads, 0, s>>>(a, x, ch);
    else k_adamw<float, 8><<<grid, kThreads, 0, s>>>(a, x, ch);
  }
  return check_launch("skv_adamw");
}

extern "C" int skv_adamw_read(void* m_out, void* v_out, const uint8_t* m, const uint8_t* v,
                              const uint8_t* m_scale, const uint8_t* v_scale, long long n,
                              int out_dt, skv_stream_t stream) {
  SKV_REQUIRE(m_out && v_out && m && v && m_scale && v_scale, SKV_E_INVALID,
              "skv_adamw_read: null pointer argument");
  SKV_REQUIRE(n > 0 && n % kBlock == 0, SKV_E_INVALID,
              "skv_adamw_read: n must be a positive multiple of %d", kBlock);
  const size_t groups = ((size_t)n / 8 + 255) / 256;
  SKV_REQUIRE(launchable(groups, 256), SKV_E_UNSUPPORTED,
              "skv_adamw_read: n=%lld is too large for a launch", n);
  SKV_REQUIRE(out_dt == SKV_F32 || out_dt == SKV_BF16, SKV_E_INVALID, "skv_adamw_read: bad dtype");
  SKV_REQUIRE(aligned16(m_out) && aligned16(v_out) && aligned16(m) && aligned16(v), SKV_E_INVALID,
              "skv_adamw_read: pointers must be 16-byte aligned");
  const size_t out = (size_t)n * (out_dt == SKV_BF16 ? 2 : 4);
  if (int rc = apart("skv_adamw_read", {{m_out, out, "m"}, {v_out, out, "v"}},
                     {{m, (size_t)n, "the state's m"}, {v, (size_t)n, "the state's v"},
                      {m_scale, (size_t)n / kBlock, "the state's m_scale"},
                      {v_scale, (size_t)n / kBlock, "the state's v_scale"}}))
    return rc;
  const unsigned grid = (unsigned)groups;
  hipStream_t s = (hipStream_t)stream;
  if (out_dt == SKV_BF16)
    k_adamw_read<<<grid, 256, 0, s>>>((uint16_t*)m_out, (uint16_t*)v_out, m, v, m_scale, v_scale,
                                      (size_t)n);
  else
    k_adamw_read<<<grid, 256, 0, s>>>((float*)m_out, (float*)v_out, m, v, m_scale, v_scale,
                                      (size_t)n);
  return check_launch("skv_adamw_read");
}
