// Writing and reading the block-scaled cache formats: one token a sequence, a
// chunk, and rows back as fp32 or bf16 (quant.h has the formats).
//
// The reference appends unquantised rows only (kv_cache_update,
// simple-llm/src/gpu/gpu_kv_cache.py:113-186); these are its append for the
// block-scaled storage.
//
// All three are bound by memory: a lane moves eight elements (16 bytes of
// bf16, 32 of fp32, against 4 or 8 of codes and a quarter of a scale byte),
// and the group's maximum is two DPP steps over the quad of lanes that holds
// it. No LDS, no second pass over the input.
#include "quant.h"

namespace skv {
namespace {

using namespace quant;

// One workgroup a sequence, all of its heads: the fill is read by this
// workgroup alone, which then advances it.
template <int BITS, bool PAGED>
__global__ __launch_bounds__(256) void k_q_append_one(Cache c, const void* __restrict__ kn,
                                                      const void* __restrict__ vn, int in_dt,
                                                      int32_t* __restrict__ lens) {
  const int b = blockIdx.x;
  const int pos = lens[b];
  if (pos < 0 || pos >= c.cap) return;  // full (or corrupt): nothing is written
  const int opr = c.D / 8;
  const int n = c.Hkv * opr;
  for (int i = threadIdx.x; i < 2 * n; i += 256) {  // K, then V; quads never straddle the two
    const bool isv = i >= n;
    const int u = isv ? i - n : i, h = u / opr, o = u - h * opr;
    float x[8];
    load8_f32(isv ? vn : kn, (size_t)b * c.Hkv * c.D + (size_t)u * 8, in_dt, x);
    uint32_t w[Fmt<BITS>::NW];
    const uint32_t byte = quantise8<BITS>(x, w);
    const size_t row = row_of<PAGED>(c, b, h, pos);
    store8<BITS>(isv ? c.v : c.k, isv ? c.vs : c.ks, row, c.D, o, w, byte);
  }
  __syncthreads();  // every lane has read lens[b] before it moves
  if (threadIdx.x == 0) lens[b] = pos + 1;
}

// Tokens of one head a workgroup moves: 256 / (D / 8), so its stores are one
// run of the head's rows (1 KB of 4-bit codes at head dim 128) and its loads
// whole rows of the token-major input.
__host__ __device__ __forceinline__ int tokens_per_wg(int D) { return 256 / (D / 8); }

// Chunk append, grid (token tiles, H_kv, B). Row i < n_new[b] goes to position
// lens[b] + i; lens is read only.
template <int BITS, bool PAGED>
__global__ __launch_bounds__(256) void k_q_append_chunk(Cache c, const void* __restrict__ kn,
                                                        const void* __restrict__ vn, int in_dt,
                                                        const int32_t* __restrict__ lens,
                                                        const int32_t* __restrict__ n_new, int C) {
  const int b = blockIdx.z, h = blockIdx.y;
  const int opr = c.D / 8, tpw = tokens_per_wg(c.D);
  const int r = threadIdx.x / opr, o = threadIdx.x - r * opr;
  const int i = blockIdx.x * tpw + r;
  const int n = n_new ? min(n_new[b], C) : C;
  const int p0 = lens[b];
  if (r >= tpw || i >= n || p0 < 0 || i >= c.cap - p0) return;  // whole quads: opr % 4 == 0
  const size_t src = (((size_t)b * C + i) * c.Hkv + h) * c.D + o * 8;
  float xk[8], xv[8];
  load8_f32(kn, src, in_dt, xk);
  load8_f32(vn, src, in_dt, xv);
  const size_t row = row_of<PAGED>(c, b, h, p0 + i);
  uint32_t w[Fmt<BITS>::NW];
  uint32_t byte = quantise8<BITS>(xk, w);
  store8<BITS>(c.k, c.ks, row, c.D, o, w, byte);
  byte = quantise8<BITS>(xv, w);
  store8<BITS>(c.v, c.vs, row, c.D, o, w, byte);
}

// Eight elements out: 16 bytes of bf16 or 32 of fp32.
template <int BITS>
__device__ __forceinline__ void put8(void* out, size_t i, int out_dt, const uint32_t* w, float s,
                                     bool here) {
  if (out_dt == SKV_BF16) {
    const bf16x8 x = decode8_bf16<BITS>(w, s);
    const uint4 y = __builtin_bit_cast(uint4, x);
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(out) + i) =
        here ? y : make_uint4(0, 0, 0, 0);
  } else {
    float x[8];
    decode8_f32<BITS>(w, s, x);
#pragma unroll
    for (int e = 0; e < 8; e += 4)
      *reinterpret_cast<float4*>(static_cast<float*>(out) + i + e) =
          here ? make_float4(x[e], x[e + 1], x[e + 2], x[e + 3]) : make_float4(0, 0, 0, 0);
  }
}

// First positions of a read, as a kernel argument: no copy to the device, which
// would be a launch of its own (or hold the host until it landed).
constexpr int kStarts = 256;
struct Starts {
  int32_t v[kStarts];
};

// Rows back, grid (token tiles, H_kv, sequences b0 ..): row i is position
// start.v[b - b0] + i, or zeros outside [0, fill).
template <int BITS, bool PAGED>
__global__ __launch_bounds__(256) void k_q_read(Cache c, void* __restrict__ ko,
                                                void* __restrict__ vo, int out_dt,
                                                const int32_t* __restrict__ lens, Starts start,
                                                int b0, int C) {
  const int b = b0 + blockIdx.z, h = blockIdx.y;
  const int opr = c.D / 8, tpw = tokens_per_wg(c.D);
  const int r = threadIdx.x / opr, o = threadIdx.x - r * opr;
  const int i = blockIdx.x * tpw + r;
  if (r >= tpw || i >= C) return;
  const long long pos = (long long)start.v[blockIdx.z] + i;
  const bool here = pos >= 0 && pos < min(max(lens[b], 0), c.cap);
  uint32_t wk[Fmt<BITS>::NW] = {}, wv[Fmt<BITS>::NW] = {};
  uint32_t sk = 0, sv = 0;
  if (here) {
    const size_t row = row_of<PAGED>(c, b, h, (int)pos);
    const size_t at = row * (size_t)(c.D * BITS / 8) + o * BITS;
    const size_t sat = row * (size_t)(c.D / kGroup) + (o >> 2);
#pragma unroll
    for (int j = 0; j < Fmt<BITS>::NW; ++j) {
      wk[j] = reinterpret_cast<const uint32_t*>(c.k + at)[j];
      wv[j] = reinterpret_cast<const uint32_t*>(c.v + at)[j];
    }
    sk = c.ks[sat];
    sv = c.vs[sat];
  }
  const size_t dst = (((size_t)b * C + i) * c.Hkv + h) * c.D + o * 8;
  put8<BITS>(ko, dst, out_dt, wk, scale_f32(sk), here);
  put8<BITS>(vo, dst, out_dt, wv, scale_f32(sv), here);
}

bool dt_ok(int dt) { return dt == SKV_F32 || dt == SKV_BF16; }

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace

int quant_cache_args(quant::Cache* c, void* k, void* k_scale, void* v, void* v_scale,
                     const int32_t* block_table, int max_blocks, int block_size, int B, int H_kv,
                     int D, int T_cap, int fmt, const char* fn) {
  SKV_REQUIRE(k && k_scale && v && v_scale, SKV_E_INVALID, "%s: null cache pointer", fn);
  SKV_REQUIRE(is_quant(fmt), SKV_E_INVALID, "%s: fmt %d is not a block-scaled format", fn, fmt);
  SKV_REQUIRE(B > 0 && H_kv > 0 && D > 0, SKV_E_INVALID,
              "%s: dims must be > 0 (B=%d H_kv=%d D=%d)", fn, B, H_kv, D);
  SKV_REQUIRE(D % quant::kGroup == 0 && D <= quant::kMaxD, SKV_E_UNSUPPORTED,
              "%s: head_dim %d (block-scaled caches take multiples of 32 up to 256)", fn, D);
  SKV_REQUIRE(B <= 65535 && H_kv <= 65535, SKV_E_UNSUPPORTED,
              "%s: B=%d, H_kv=%d exceed the grid limit", fn, B, H_kv);
  SKV_REQUIRE(aligned16(k) && aligned16(v), SKV_E_INVALID,
              "%s: the caches must be 16-byte aligned", fn);
  c->k = static_cast<uint8_t*>(k);
  c->ks = static_cast<uint8_t*>(k_scale);
  c->v = static_cast<uint8_t*>(v);
  c->vs = static_cast<uint8_t*>(v_scale);
  c->bt = block_table;
  c->Hkv = H_kv;
  c->D = D;
  c->T_cap = T_cap;
  c->max_blocks = c->bs_shift = 0;
  if (block_table) {
    SKV_REQUIRE(block_size > 0 && (block_size & (block_size - 1)) == 0, SKV_E_INVALID,
                "%s: block_size=%d not a power of two", fn, block_size);
    c->bs_shift = __builtin_ctz((unsigned)block_size);
    SKV_REQUIRE(max_blocks > 0 && ((long)max_blocks << c->bs_shift) < (1L << 31), SKV_E_INVALID,
                "%s: max_blocks=%d out of range", fn, max_blocks);
    c->max_blocks = max_blocks;
    c->cap = max_blocks << c->bs_shift;
  } else {
    SKV_REQUIRE(T_cap > 0, SKV_E_INVALID, "%s: T_cap must be > 0", fn);
    c->cap = T_cap;
  }
  return SKV_OK;
}

}  // namespace skv

using namespace skv;

// The kernel of (fmt, paged).
#define SKV_Q_CASES(KERNEL, ...)                                                        \
  do {                                                                                  \
    if (fmt == SKV_MXFP4 && c.bt) hipLaunchKernelGGL((KERNEL<4, true>), __VA_ARGS__);   \
    else if (fmt == SKV_MXFP4) hipLaunchKernelGGL((KERNEL<4, false>), __VA_ARGS__);     \
    else if (c.bt) hipLaunchKernelGGL((KERNEL<8, true>), __VA_ARGS__);                  \
    else hipLaunchKernelGGL((KERNEL<8, false>), __VA_ARGS__);                           \
  } while (0)

extern "C" int skv_q_append(void* k, void* k_scale, void* v, void* v_scale, const void* k_new,
                            const void* v_new, int32_t* lens, const int32_t* block_table,
                            int max_blocks, int block_size, int B, int H_kv, int D, int T_cap,
                            int fmt, int in_dt, skv_stream_t stream) {
  const char* fn = "skv_q_append";
  quant::Cache c;
  int rc = quant_cache_args(&c, k, k_scale, v, v_scale, block_table, max_blocks, block_size, B,
                            H_kv, D, T_cap, fmt, fn);
  if (rc) return rc;
  SKV_REQUIRE(k_new && v_new && lens, SKV_E_INVALID, "%s: null pointer argument", fn);
  SKV_REQUIRE(dt_ok(in_dt), SKV_E_INVALID, "%s: bad dtype", fn);
  SKV_REQUIRE(aligned16(k_new) && aligned16(v_new), SKV_E_INVALID,
              "%s: k_new and v_new must be 16-byte aligned", fn);
  SKV_REQUIRE((long)H_kv * D < (1L << 30), SKV_E_UNSUPPORTED, "%s: rows too wide", fn);
  SKV_Q_CASES(k_q_append_one, dim3(B), dim3(256), 0, (hipStream_t)stream, c, k_new, v_new, in_dt,
              lens);
  return check_launch(fn);
}

extern "C" int skv_q_append_chunk(void* k, void* k_scale, void* v, void* v_scale,
                                  const void* k_new, const void* v_new, const int32_t* lens,
                                  const int32_t* n_new, const int32_t* block_table,
                                  int max_blocks, int block_size, int B, int C, int H_kv, int D,
                                  int T_cap, int fmt, int in_dt, skv_stream_t stream) {
  const char* fn = "skv_q_append_chunk";
  quant::Cache c;
  int rc = quant_cache_args(&c, k, k_scale, v, v_scale, block_table, max_blocks, block_size, B,
                            H_kv, D, T_cap, fmt, fn);
  if (rc) return rc;
  SKV_REQUIRE(k_new && v_new && lens && C > 0, SKV_E_INVALID, "%s: bad arguments", fn);
  SKV_REQUIRE(dt_ok(in_dt), SKV_E_INVALID, "%s: bad dtype", fn);
  SKV_REQUIRE(aligned16(k_new) && aligned16(v_new), SKV_E_INVALID,
              "%s: k_new and v_new must be 16-byte aligned", fn);
  const int tpw = tokens_per_wg(D);
  SKV_Q_CASES(k_q_append_chunk, dim3((unsigned)(((long)C + tpw - 1) / tpw), H_kv, B), dim3(256), 0,
              (hipStream_t)stream, c, k_new, v_new, in_dt, lens, n_new, C);
  return check_launch(fn);
}

extern "C" int skv_q_read(void* k_out, void* v_out, const void* k, const void* k_scale,
                          const void* v, const void* v_scale, const int32_t* lens,
                          const int32_t* start, int n_start, const int32_t* block_table,
                          int max_blocks, int block_size, int B, int C, int H_kv, int D,
                          int T_cap, int fmt, int out_dt, skv_stream_t stream) {
  const char* fn = "skv_q_read";
  quant::Cache c;
  int rc = quant_cache_args(&c, const_cast<void*>(k), const_cast<void*>(k_scale),
                            const_cast<void*>(v), const_cast<void*>(v_scale), block_table,
                            max_blocks, block_size, B, H_kv, D, T_cap, fmt, fn);
  if (rc) return rc;
  SKV_REQUIRE(k_out && v_out && lens && start && C > 0 && (n_start == 1 || n_start == B),
              SKV_E_INVALID, "%s: bad arguments", fn);
  SKV_REQUIRE(dt_ok(out_dt), SKV_E_INVALID, "%s: bad dtype", fn);
  SKV_REQUIRE(aligned16(k_out) && aligned16(v_out), SKV_E_INVALID,
              "%s: k_out and v_out must be 16-byte aligned", fn);
  const int tpw = tokens_per_wg(D);
  for (int b0 = 0; b0 < B; b0 += kStarts) {
    const int nb = B - b0 < kStarts ? B - b0 : kStarts;
    Starts st;
    for (int i = 0; i < nb; ++i) st.v[i] = start[n_start == 1 ? 0 : b0 + i];
    SKV_Q_CASES(k_q_read, dim3((unsigned)(((long)C + tpw - 1) / tpw), H_kv, nb), dim3(256), 0,
                (hipStream_t)stream, c, k_out, v_out, out_dt, lens, st, b0, C);
  }
  return check_launch(fn);
}
