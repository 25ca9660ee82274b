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
// it. No LDS, no second pass over the input. 4 x 16 x 128, 2048 tokens of bf16
// into 4 bits: 22 us (85 MB, 3.9 TB/s; a copy reads and writes at 5.0), back to
// bf16 16; 8192 tokens back 54 to 60 us a call (340 MB, 5.7 to 6.3 TB/s), from 8
// bits 67 (6.1), to fp32 100 (6.1) and 101 (6.7); one token of 64 sequences 3.1.
#include <cstring>

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

// Tokens of one head in a run, 256 / (D / 8): its code rows are one stretch of
// the cache (1 KB of 4 bits at head dim 128), its other side that many rows of
// the token-major tensor.
__host__ __device__ __forceinline__ int tokens_per_wg(int D) { return 256 / (D / 8); }

// Runs of tokens_per_wg tokens a workgroup takes: four where that still leaves
// every CU eight workgroups, for loads in flight; one in smaller calls. (Runs
// of four neighbouring heads, side by side in the token-major tensor, were no
// faster: 4 x 8192 x 16 x 128 back to bf16 60 us against 57.)
constexpr int kRuns = 4;

// Chunk append, grid (token tiles, H_kv, sequences b0 ..). Row i < n goes to
// position lens[b] + i, n being n_new[b], or without n_new the host's count
// (HOST), or C; lens is read only. The first workgroup of a sequence stores the
// host's count in n_copy[b] and the fill in start[b] (unless NULL) for the
// kernels behind this one. The input is loaded before
// the fill is known (its place depends on neither): one round trip to memory,
// not two (4 x 2048 x 16 x 128 bf16 into 4 bits: 18.8 us with the fill first
// and one run).
struct NoInts {};
template <int BITS, bool PAGED, int RUNS, typename HOST>
__global__ __launch_bounds__(256) void k_q_append_chunk(Cache c, const void* __restrict__ kn,
                                                        const void* __restrict__ vn, int in_dt,
                                                        const int32_t* __restrict__ lens,
                                                        const int32_t* __restrict__ n_new,
                                                        HOST n_host, int32_t* __restrict__ n_copy,
                                                        int32_t* __restrict__ start, int b0,
                                                        int C) {
  constexpr bool kHost = sizeof(HOST) == sizeof(Ints);
  const int b = b0 + blockIdx.z, h = blockIdx.y;
  const int opr = c.D / 8, tpw = tokens_per_wg(c.D);
  const int r = threadIdx.x / opr, o = threadIdx.x - r * opr;
  if (r >= tpw) return;  // whole quads: opr % 4 == 0
  const int i0 = blockIdx.x * (tpw * RUNS) + r;
  float xk[RUNS][8], xv[RUNS][8];
#pragma unroll
  for (int u = 0; u < RUNS; ++u) {
    const int i = min(i0 + u * tpw, C - 1);
    const size_t src = (((size_t)b * C + i) * c.Hkv + h) * c.D + o * 8;
    load8_f32(kn, src, in_dt, xk[u]);
    load8_f32(vn, src, in_dt, xv[u]);
  }
  const bool first = blockIdx.x == 0 && h == 0 && threadIdx.x == 0;
  int n = C;
  if constexpr (kHost) {
    n = n_host.v[blockIdx.z];
    if (n_copy != nullptr && first) n_copy[b] = n;
  } else if (n_new) {
    n = min(n_new[b], C);
  }
  const int p0 = lens[b];
  if (start != nullptr && first) start[b] = p0;
#pragma unroll
  for (int u = 0; u < RUNS; ++u) {
    const int i = i0 + u * tpw;
    if (i >= n || p0 < 0 || i >= c.cap - p0) return;  // later runs are further on
    const size_t row = row_of<PAGED>(c, b, h, p0 + i);
    uint32_t w[Fmt<BITS>::NW];
    uint32_t byte = quantise8<BITS>(xk[u], w);
    store8<BITS>(c.k, c.ks, row, c.D, o, w, byte);
    byte = quantise8<BITS>(xv[u], w);
    store8<BITS>(c.v, c.vs, row, c.D, o, w, byte);
  }
}

// A lane's elements of a row on their way out: eight as 16 bytes of bf16, four
// as 16 of fp32, so that a wavefront stores one stretch (two 16-byte stores a
// lane, 32 bytes apart, took 84 us for 4 x 4096 x 16 x 128; 160 non-temporal).
template <int BITS, int OUT>
struct Piece {
  static constexpr int N = OUT == SKV_BF16 ? 8 : 4;
  static constexpr int BYTES = N * BITS / 8;  // 2, 4 or 8
  uint32_t w[BYTES > 4 ? 2 : 1];
  uint32_t scale;
  __device__ __forceinline__ void load(const uint8_t* p, const uint8_t* s) {
    if constexpr (BYTES == 8) {
      const uint2 x = *reinterpret_cast<const uint2*>(p);
      w[0] = x.x;
      w[1] = x.y;
    } else if constexpr (BYTES == 4) {
      w[0] = *reinterpret_cast<const uint32_t*>(p);
    } else {
      w[0] = *reinterpret_cast<const uint16_t*>(p);
    }
    scale = *s;
  }
  __device__ __forceinline__ void zero() {
    w[0] = scale = 0;
    if constexpr (BYTES == 8) w[1] = 0;
  }
  __device__ __forceinline__ u32x4_t value() const {
    const float s = scale_f32(scale);
    if constexpr (OUT == SKV_BF16) {
      return __builtin_bit_cast(u32x4_t, decode8_bf16<BITS>(w, s));
    } else {
      const f32x2 a = BITS == 4 ? __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[0], s, 0)
                                : __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w[0], s, false);
      const f32x2 b = BITS == 4 ? __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[0], s, 1)
                                : __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w[0], s, true);
      return u32x4_t{__float_as_uint(a[0]), __float_as_uint(a[1]), __float_as_uint(b[0]),
                     __float_as_uint(b[1])};
    }
  }
};

// lens[b] advanced by the host's counts, as skv_advance.
__global__ __launch_bounds__(kInts) void k_q_advance(int32_t* __restrict__ lens, Ints n, int b0,
                                                     int nb, int cap) {
  const int i = threadIdx.x;
  if (i < nb) lens[b0 + i] = min(lens[b0 + i] + n.v[i], cap);
}

// Rows back, grid (token tiles, H_kv, sequences b0 ..): row i is position
// start.v[b - b0] + i, or zeros outside [0, fill).
template <int BITS, bool PAGED, int RUNS, int OUT>
__global__ __launch_bounds__(256) void k_q_read(Cache c, void* __restrict__ ko,
                                                void* __restrict__ vo,
                                                const int32_t* __restrict__ lens, Ints start,
                                                int b0, int C) {
  using P = Piece<BITS, OUT>;
  const int b = b0 + blockIdx.z, h = blockIdx.y;
  const int lpr = c.D / P::N, tpw = 256 / lpr;  // lanes a row, rows a run
  const int r = threadIdx.x / lpr, o = threadIdx.x - r * lpr;
  if (r >= tpw) return;
  const int i0 = blockIdx.x * (tpw * RUNS) + r;
  const int fill = min(max(lens[b], 0), c.cap);
  P k[RUNS], v[RUNS];
#pragma unroll
  for (int u = 0; u < RUNS; ++u) {
    const long long pos = (long long)start.v[blockIdx.z] + i0 + u * tpw;
    // Rows of a contiguous cache are loaded before the fill is known; a page
    // past the fill may be no page.
    k[u].zero();
    v[u].zero();
    if (pos >= 0 && pos < (PAGED ? fill : c.cap)) {
      const size_t row = row_of<PAGED>(c, b, h, (int)pos);
      const size_t at = row * (size_t)(c.D * BITS / 8) + o * P::BYTES;
      const size_t sat = row * (size_t)(c.D / kGroup) + o * P::N / kGroup;
      k[u].load(c.k + at, c.ks + sat);
      v[u].load(c.v + at, c.vs + sat);
    }
  }
#pragma unroll
  for (int u = 0; u < RUNS; ++u) {
    const int i = i0 + u * tpw;
    if (i >= C) return;
    const long long pos = (long long)start.v[blockIdx.z] + i;
    const bool here = pos >= 0 && pos < fill;
    const size_t dst = ((((size_t)b * C + i) * c.Hkv + h) * c.D + o * P::N) * (16 / P::N);
    const u32x4_t z = u32x4_t{0, 0, 0, 0};
    __builtin_nontemporal_store(here ? k[u].value() : z,
                                reinterpret_cast<u32x4_t*>(static_cast<uint8_t*>(ko) + dst));
    __builtin_nontemporal_store(here ? v[u].value() : z,
                                reinterpret_cast<u32x4_t*>(static_cast<uint8_t*>(vo) + dst));
  }
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
  SKV_REQUIRE(c->cap <= quant::kMaxCap, SKV_E_UNSUPPORTED,
              "%s: a sequence of %d tokens (block-scaled caches take up to 2^30)", fn, c->cap);
  return SKV_OK;
}

}  // namespace skv

using namespace skv;

// The kernel of (fmt, paged), more template arguments after these.
#define SKV_Q_CASES(LAUNCH)                                    \
  do {                                                         \
    if (fmt == SKV_MXFP4 && c.bt) LAUNCH(4, true);             \
    else if (fmt == SKV_MXFP4) LAUNCH(4, false);               \
    else if (c.bt) LAUNCH(8, true);                            \
    else LAUNCH(8, false);                                     \
  } while (0)

// Whether a call over C tokens of B * H_kv heads fills the card with kRuns runs
// a workgroup (8 workgroups per CU).
static bool long_call(int B, int H_kv, int C, int D) {
  return (long)B * H_kv * (C / (tokens_per_wg(D) * kRuns)) >= 8 * 256;
}

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
#define SKV_LAUNCH(BITS, PAGED)                                                              \
  hipLaunchKernelGGL((k_q_append_one<BITS, PAGED>), dim3(B), dim3(256), 0, (hipStream_t)stream, \
                     c, k_new, v_new, in_dt, lens)
  SKV_Q_CASES(SKV_LAUNCH);
#undef SKV_LAUNCH
  return check_launch(fn);
}

int skv::quant_append_chunk(const quant::Cache& c, int fmt, const void* k_new, const void* v_new,
                            const int32_t* lens, const int32_t* n_new, const int32_t* n_host,
                            int32_t* n_copy, int32_t* start, int B, int C, int in_dt,
                            hipStream_t s, const char* fn) {
  const bool runs = long_call(B, c.Hkv, C, c.D);
  const int tpw = tokens_per_wg(c.D) * (runs ? kRuns : 1);
  for (int b0 = 0; b0 < B; b0 += n_host ? kInts : B) {
    const int nb = n_host && B - b0 > kInts ? kInts : B - b0;
    const dim3 grid((unsigned)(((long)C + tpw - 1) / tpw), c.Hkv, nb);
    Ints cnt;
    if (n_host) memcpy(cnt.v, n_host + b0, (size_t)nb * sizeof(int32_t));
#define SKV_CHUNK(BITS, PAGED, RUNS, COUNTS)                                                   \
  hipLaunchKernelGGL((k_q_append_chunk<BITS, PAGED, RUNS, decltype(COUNTS)>), grid, dim3(256), 0, \
                     s, c, k_new, v_new, in_dt, lens, n_new, COUNTS, n_copy, start, b0, C)
#define SKV_LAUNCH(BITS, PAGED)                                  \
  do {                                                           \
    if (n_host) {                                                \
      if (runs) SKV_CHUNK(BITS, PAGED, kRuns, cnt);              \
      else SKV_CHUNK(BITS, PAGED, 1, cnt);                       \
    } else {                                                     \
      if (runs) SKV_CHUNK(BITS, PAGED, kRuns, NoInts{});         \
      else SKV_CHUNK(BITS, PAGED, 1, NoInts{});                  \
    }                                                            \
  } while (0)
    SKV_Q_CASES(SKV_LAUNCH);
#undef SKV_LAUNCH
#undef SKV_CHUNK
  }
  return check_launch(fn);
}

extern "C" int skv_q_append_chunk(void* k, void* k_scale, void* v, void* v_scale,
                                  const void* k_new, const void* v_new, int32_t* lens,
                                  const int32_t* n_new, const int32_t* n_host, int advance,
                                  const int32_t* block_table, int max_blocks, int block_size,
                                  int B, int C, int H_kv, int D, int T_cap, int fmt, int in_dt,
                                  skv_stream_t stream) {
  const char* fn = "skv_q_append_chunk";
  quant::Cache c;
  int rc = quant_cache_args(&c, k, k_scale, v, v_scale, block_table, max_blocks, block_size, B,
                            H_kv, D, T_cap, fmt, fn);
  if (rc) return rc;
  SKV_REQUIRE(k_new && v_new && lens && C > 0, SKV_E_INVALID, "%s: bad arguments", fn);
  SKV_REQUIRE(dt_ok(in_dt), SKV_E_INVALID, "%s: bad dtype", fn);
  SKV_REQUIRE(aligned16(k_new) && aligned16(v_new), SKV_E_INVALID,
              "%s: k_new and v_new must be 16-byte aligned", fn);
  SKV_REQUIRE(!n_new || !n_host, SKV_E_INVALID, "%s: counts on the device or the host", fn);
  for (int b = 0; n_host && b < B; ++b)
    SKV_REQUIRE(n_host[b] >= 0 && n_host[b] <= C, SKV_E_INVALID, "%s: n_host[%d]=%d outside [0, %d]",
                fn, b, n_host[b], C);
  hipStream_t s = (hipStream_t)stream;
  rc = quant_append_chunk(c, fmt, k_new, v_new, lens, n_new, n_host, nullptr, nullptr, B, C, in_dt, s,
                          fn);
  if (rc || !advance) return rc;
  if (!n_host) return skv_advance(lens, n_new, C, B, c.cap, stream);
  for (int b0 = 0; b0 < B; b0 += kInts) {
    const int nb = B - b0 < kInts ? B - b0 : kInts;
    Ints cnt;
    memcpy(cnt.v, n_host + b0, (size_t)nb * sizeof(int32_t));
    hipLaunchKernelGGL(k_q_advance, dim3(1), dim3(kInts), 0, s, lens, cnt, b0, nb, c.cap);
  }
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
  const bool runs = long_call(B, H_kv, C, D);
  const int tpw = 256 / (D / (out_dt == SKV_BF16 ? 8 : 4)) * (runs ? kRuns : 1);
  for (int b0 = 0; b0 < B; b0 += kInts) {
    const int nb = B - b0 < kInts ? B - b0 : kInts;
    Ints st;
    for (int i = 0; i < nb; ++i) st.v[i] = start[n_start == 1 ? 0 : b0 + i];
    const dim3 grid((unsigned)(((long)C + tpw - 1) / tpw), H_kv, nb);
#define SKV_READ(BITS, PAGED, RUNS, OUT)                                                      \
  hipLaunchKernelGGL((k_q_read<BITS, PAGED, RUNS, OUT>), grid, dim3(256), 0, (hipStream_t)stream, \
                     c, k_out, v_out, lens, st, b0, C)
#define SKV_LAUNCH(BITS, PAGED)                                       \
  do {                                                                \
    if (out_dt == SKV_BF16) {                                         \
      if (runs) SKV_READ(BITS, PAGED, kRuns, SKV_BF16);               \
      else SKV_READ(BITS, PAGED, 1, SKV_BF16);                        \
    } else {                                                          \
      if (runs) SKV_READ(BITS, PAGED, kRuns, SKV_F32);                \
      else SKV_READ(BITS, PAGED, 1, SKV_F32);                         \
    }                                                                 \
  } while (0)
    SKV_Q_CASES(SKV_LAUNCH);
#undef SKV_LAUNCH
#undef SKV_READ
  }
  return check_launch(fn);
}
