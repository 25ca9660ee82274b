// Cached single-query attention over a block-scaled cache (quant.h): split-K
// flash decoding with both products on the matrix cores.
//
//   o[b, h] = softmax(scale * q[b, h] . K[b, 0:len, h / G]^T) . V[b, 0:len, h / G]
//
// attention_with_kv_cache of the reference
// (simple-llm/src/gpu/gpu_kv_cache.py:194-289) over the 4- and 8-bit storage.
//
// Work split: workgroup (chunk, b, kv head) of four wavefronts takes `chunk`
// consecutive tokens of one kv head for its G query heads (1 to 16), each
// wavefront every fourth 32-token tile; the head-major cache makes a tile one
// run of bytes (2 KB of 4-bit codes at head dim 128). The wavefronts merge
// through LDS, and the chunks in a second launch, which also advances the
// fills of a fused append; one chunk a row writes the output itself.
//
// A tile:
//  * S = K q^T (v_mfma_f32_16x16x32_bf16). Lane (r, kb) of a 16-token half
//    loads the codes of token r, elements [kb DP/4, (kb + 1) DP/4): the
//    contraction may take the elements in any order as long as q does too, so
//    the eight-element pieces go to the matrix core as they lie, and a lane's
//    piece has one scale. Converted to bf16 with the scale they are exact.
//    Column c of the product is query head c.
//  * Online softmax in fp32, each lane holding 8 of the 32 scores of its
//    column. The running max moves lazily: only when a score passes it by 8
//    (log2 units), which is also the only time the four lanes of a column
//    exchange anything; until then p <= 256 and the sums stay consistent.
//  * O^T += V^T P: V goes through LDS as bf16 (converted where the lane still
//    holds one group with one scale; after a transposition of the codes the
//    eight tokens of a lane would have eight), row-major with XOR-swizzled
//    16-byte chunks, and comes back transposed (ds_read_b64_tr_b16). The
//    probabilities are already in the operand's token order.
// Precision: K and V enter exactly. fp32 q is three bf16 parts (all of its
// bits) and p three (2^-24 of p); bf16 q is one part and, the output being
// bf16, p two (2^-17).
// Tokens past the chunk reread its last row and get weight 0: no memory past
// the fill is touched, none of it meets a zero weight.
// No atomics: results are bitwise reproducible, and a paged cache gives the
// bits of the same rows in a contiguous one.
#include "quant.h"

namespace skv {
namespace {

using namespace quant;

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short i16x4 __attribute__((ext_vector_type(4)));

constexpr int kWaves = 4;
constexpr int kTile = 32;     // tokens per wavefront tile
constexpr float kLazy = 8.f;  // the running max moves when a score passes it by more (log2 units)
constexpr int kMaxG = 16;     // query heads per kv head

struct QDecodeArgs {
  Cache c;
  void* out;
  const void* q;
  const int32_t* lens;
  int B, Hq, G;
  float qscale;  // softmax scale * log2(e)
  int q_dt, out_dt;
  int chunk, n_chunks;
  float* ws_o;   // [B * Hq][n_chunks][D]
  float* ws_ml;  // [B * Hq][n_chunks][2]
  const void* new_k;  // fused append, or NULL
  const void* new_v;
  int in_dt;
};

__device__ __forceinline__ bool appends(const QDecodeArgs& a, int len) {
  return a.new_k != nullptr && len >= 0 && len < a.c.cap;
}

// W words from p (aligned to min(4 W, 16) bytes), read once: non-temporal.
template <int W>
__device__ __forceinline__ void load_words(const uint8_t* p, uint32_t* w) {
  if constexpr (W >= 4) {
#pragma unroll
    for (int i = 0; i < W / 4; ++i) {
      const u32x4_t x = stream_load16(p + 16 * i);
      w[4 * i] = x.x; w[4 * i + 1] = x.y; w[4 * i + 2] = x.z; w[4 * i + 3] = x.w;
    }
  } else if constexpr (W == 2) {
    const u32x2_t x = stream_load8(p);
    w[0] = x.x; w[1] = x.y;
  } else {
    w[0] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(p));
  }
}

// ds_read_b64_tr_b16: within each 16-lane group, lane i receives as its slot j
// the element i%4 of the four 16-bit values addressed by lane 4j + i/4.
__device__ __forceinline__ i16x4 lds_read_tr16(const uint16_t* p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4*)(p));
}

// The swizzle of a bf16 V row in LDS: 16-byte chunk ch of token t lies at
// chunk ch ^ key(t), so that the transposed reads (4 adjacent chunks of 4
// consecutive rows per 32 lanes) hit distinct banks.
template <int DP>
__device__ __forceinline__ int v_at(int t, int ch) {
  int key;
  if constexpr (DP >= 128) key = 4 * (t & 3) + ((t >> 2) & 3);
  else if constexpr (DP == 64) key = 4 * ((t >> 1) & 1) + ((t >> 2) & 3);
  else key = (t >> 2) & 3;
  return t * DP + ((ch ^ key) * 8);
}

// LDS written by some lanes of a wavefront is read by others: LDS operations
// of a wavefront complete in order, so only the compiler must keep theirs.
__device__ __forceinline__ void wave_lds_order() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// DP: head dim padded to a power of two (elements past D: q is zero, rows of
// O^T are not stored). NQ parts of q, NP of p.
template <int DP, int BITS, bool PAGED, int NQ, int NP>
__global__ __launch_bounds__(kWaves * 64) void k_q_decode(QDecodeArgs a) {
  constexpr int NW = Fmt<BITS>::NW;
  constexpr int KE = DP / 4;                     // elements of a K row per lane
  constexpr int KO = KE / 8;                     // ... in pieces of 8: MFMAs per half tile
  constexpr int KS = KE > kGroup ? KE / kGroup : 1;  // scales per lane and half tile
  constexpr int VL = DP / kGroup;                // lanes (groups) of a V row
  constexpr int VR = VL == 1 ? kTile : 64 / VL;  // V rows a pass moves (head dim 32: half the lanes)
  constexpr int VP = kTile / VR;                 // passes
  constexpr int DB = DP / 16;
  __shared__ __attribute__((aligned(16))) uint16_t sv[kWaves][kTile * DP];
  __shared__ float sml[kWaves][kMaxG][2];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n_rows = a.B * a.c.Hkv;
  const int ci = blockIdx.x / n_rows, bh = blockIdx.x - ci * n_rows;
  const int b = bh / a.c.Hkv, hk = bh - b * a.c.Hkv;
  const int D = a.c.D, G = a.G;
  const int fill = a.lens[b];
  const bool app = appends(a, fill);
  const int len = min(max(fill, 0), a.c.cap) + (app ? 1 : 0);
  const int start = ci * a.chunk;
  const int end = min(len, start + a.chunk);
  const size_t head0 = (size_t)b * a.Hq + hk * G;  // first query head's output row

  if (start >= end) {
    // Nothing to attend: chunk 0 of an empty sequence stands for a zero
    // output (m = 0, l = 1, o = 0); others have no weight (l = 0, o unread).
    const bool zero = ci == 0;
    for (int i = tid; i < G * D; i += kWaves * 64) {
      const int g = i / D, d = i - g * D;
      if (a.n_chunks == 1) store_elem(a.out, (head0 + g) * D + d, a.out_dt, 0.f);
      else if (zero) a.ws_o[(head0 + g) * a.n_chunks * D + d] = 0.f;
    }
    if (a.n_chunks > 1 && tid < G)
      *reinterpret_cast<float2*>(a.ws_ml + ((head0 + tid) * a.n_chunks + ci) * 2) =
          zero ? make_float2(0.f, 1.f) : make_float2(-INFINITY, 0.f);
    return;
  }

  // A fused append: the chunk that holds the new token writes its row first
  // (one wavefront: 2 D / 8 <= 64 lanes), and the workgroup reads it back from
  // the cache as any other.
  const bool outgrown = ci == a.n_chunks - 1 && len > end;  // the plan does not cover the fill
  if (app && (end == len || outgrown)) {
    const int opr = D / 8;
    if (tid < 2 * opr) {
      const bool isv = tid >= opr;
      const int o = isv ? tid - opr : tid;
      float x[8];
      load8_f32(isv ? a.new_v : a.new_k, ((size_t)b * a.c.Hkv + hk) * D + o * 8, a.in_dt, x);
      uint32_t w[NW];
      const uint32_t byte = quantise8<BITS>(x, w);
      store8<BITS>(isv ? a.c.v : a.c.k, isv ? a.c.vs : a.c.ks, row_of<PAGED>(a.c, b, hk, len - 1),
                   D, o, w, byte);
    }
    __builtin_amdgcn_s_waitcnt(0);  // the stores have completed
    __syncthreads();
  }

  const int cl = lane & 15, kb = lane >> 4;  // MFMA row/column, k block

  // ---- queries, operand B: column cl is head cl, elements kb KE + 8 i ----
  bf16x8 qf[NQ][KO];
#pragma unroll
  for (int i = 0; i < KO; ++i) {
    const int e = kb * KE + 8 * i;
    const bool used = cl < G && e < D;
    float x[8];
    load8_f32(a.q, (head0 + (cl < G ? cl : 0)) * D + (e < D ? e : 0), a.q_dt, x);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float r = used ? x[j] : 0.f;
#pragma unroll
      for (int p = 0; p < NQ; ++p) {
        const __bf16 h = (__bf16)r;
        qf[p][i][j] = h;
        r -= (float)h;
      }
    }
  }

  const int cb = D * BITS / 8, sb = D / kGroup;  // code and scale bytes of a row
  // this lane's place in a K row: code offset of each scale's run, scale index
  int ko[KS], ks[KS];
#pragma unroll
  for (int i = 0; i < KS; ++i) {
    const int e = kb * KE + i * kGroup;
    ko[i] = e < D ? e * BITS / 8 : 0;
    ks[i] = e < D ? e / kGroup : 0;
  }
  // ... and in a V row
  const int vg = VL == 1 ? 0 : lane % VL, vr = VL == 1 ? (lane & (kTile - 1)) : lane / VL;
  const int vgl = vg < sb ? vg : 0;

  constexpr int KWS = KO * NW / KS;  // words under one scale
  uint32_t kw[2][KO * NW], kscale[2][KS], vw[VP][4 * NW], vscale[VP];
  auto load_tile = [&](int t0) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const size_t row = row_of<PAGED>(a.c, b, hk, min(t0 + 16 * u + cl, end - 1));
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        load_words<KWS>(a.c.k + row * cb + ko[i], &kw[u][i * KWS]);
        kscale[u][i] = a.c.ks[row * sb + ks[i]];
      }
    }
#pragma unroll
    for (int p = 0; p < VP; ++p) {
      const size_t row = row_of<PAGED>(a.c, b, hk, min(t0 + p * VR + vr, end - 1));
      load_words<4 * NW>(a.c.v + row * cb + vgl * (kGroup * BITS / 8), vw[p]);
      vscale[p] = a.c.vs[row * sb + vgl];
    }
  };

  f32x4 o[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) o[db] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m_run = -INFINITY, l_run = 0.f;
  uint16_t* svw = sv[wave];

  int t0 = start + wave * kTile;
  if (t0 < end) load_tile(t0);
  for (; t0 < end; t0 += kWaves * kTile) {
    // ---- scores of the two halves ----
    f32x4 sc[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      sc[u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < KO; ++i) {
        const bf16x8 kf = decode8_bf16<BITS>(&kw[u][i * NW], scale_f32(kscale[u][i * KS / KO]));
#pragma unroll
        for (int p = 0; p < NQ; ++p)
          sc[u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[p][i], sc[u], 0, 0, 0);
      }
    }
    // ---- V to LDS as bf16 ----
#pragma unroll
    for (int p = 0; p < VP; ++p)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bf16x8 x = decode8_bf16<BITS>(&vw[p][i * NW], scale_f32(vscale[p]));
        *reinterpret_cast<bf16x8*>(svw + v_at<DP>(p * VR + vr, vg * 4 + i)) = x;
      }
    // the next tile's codes, in flight over the rest of this one
    const bool mask = t0 + kTile > end;
    if (t0 + kWaves * kTile < end) load_tile(t0 + kWaves * kTile);

    // ---- softmax: lane (cl, kb) has tokens t0 + 16 u + 4 kb + j ----
    float s[8];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float x = sc[u][j] * a.qscale;
        s[4 * u + j] = mask && t0 + 16 * u + 4 * kb + j >= end ? -INFINITY : x;
      }
    float mt = s[0];
#pragma unroll
    for (int j = 1; j < 8; ++j) mt = fmaxf(mt, s[j]);
    if (__ballot(mt > m_run + kLazy) != 0ull) {  // uniform
      mt = fmaxf(mt, __shfl_xor(mt, 16));
      mt = xor32_max(mt);
      const float mn = fmaxf(m_run, mt);
      const float al = mn == m_run ? 1.f : fast_exp2(m_run - mn);  // 0 on the first tile
      m_run = mn;
      l_run *= al;
#pragma unroll
      for (int db = 0; db < DB; ++db) o[db] *= al;
    }
    const float m_use = m_run == -INFINITY ? 0.f : m_run;  // every score so far is -inf
    bf16x8 pf[NP];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float r = fast_exp2(s[j] - m_use);
      l_run += r;
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        const __bf16 h = (__bf16)r;
        pf[p][j] = h;
        r -= (float)h;
      }
    }
    // ---- O^T += V^T P: slots 0-3 are tokens 4 kb + j, 4-7 are 16 + 4 kb + j ----
    wave_lds_order();
#pragma unroll
    for (int db = 0; db < DB; ++db) {
      const int ch = 2 * db + ((cl & 3) >> 1), in = 4 * (cl & 1);
      const i16x4 lo = lds_read_tr16(svw + v_at<DP>(4 * kb + (cl >> 2), ch) + in);
      const i16x4 hi = lds_read_tr16(svw + v_at<DP>(16 + 4 * kb + (cl >> 2), ch) + in);
      const bf16x8 va =
          __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
      for (int p = 0; p < NP; ++p)
        o[db] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va, pf[p], o[db], 0, 0, 0);
    }
    wave_lds_order();
  }

  // ---- the wavefronts' parts merge through the V tiles' space ----
  float lt = l_run + __shfl_xor(l_run, 16);
  lt = xor32_sum(lt);
  __syncthreads();
  float* mo = reinterpret_cast<float*>(&sv[0][0]);  // [kWaves][G][DP]
  static_assert(sizeof(sv) >= (size_t)kWaves * kMaxG * DP * sizeof(float), "merge space");
  if (cl < G) {
#pragma unroll
    for (int db = 0; db < DB; ++db)
      *reinterpret_cast<f32x4*>(mo + (wave * G + cl) * DP + 16 * db + 4 * kb) = o[db];
    if (kb == 0) {
      sml[wave][cl][0] = m_run;
      sml[wave][cl][1] = lt;
    }
  }
  __syncthreads();
  const int vpr = D / 4;
  for (int i = tid; i < G * vpr; i += kWaves * 64) {
    const int g = i / vpr, d = (i - g * vpr) * 4;
    float M = sml[0][g][0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) M = fmaxf(M, sml[w][g][0]);
    float L = 0.f;
    f32x4 O = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float mw = sml[w][g][0];
      const float wt = mw == -INFINITY ? 0.f : fast_exp2(mw - M);
      L = fmaf(wt, sml[w][g][1], L);
      O += wt * *reinterpret_cast<const f32x4*>(mo + (w * G + g) * DP + d);
    }
    if (outgrown) L = __builtin_nanf("");
    if (a.n_chunks == 1) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        store_elem(a.out, (head0 + g) * D + d + e, a.out_dt, O[e] / L);
    } else {
      const size_t slot = (head0 + g) * a.n_chunks + ci;
      *reinterpret_cast<f32x4*>(a.ws_o + slot * D + d) = O;
      if (d == 0) *reinterpret_cast<float2*>(a.ws_ml + slot * 2) = make_float2(M, L);
    }
  }
}

// Merge of the chunks' partials, grid (H_q, B): DP / 4 lanes of four elements
// by 1024 / DP streams of chunks, then the streams through LDS. adv (fused
// append): the fills, each advanced by its sequence's first workgroup; nothing
// else here reads them (a chunk without tokens left m = -inf, l = 0).
template <int DP>
__global__ __launch_bounds__(256) void k_q_merge(QDecodeArgs a, int32_t* adv) {
  constexpr int LN = DP / 4, NS = 256 / LN;
  __shared__ __attribute__((aligned(16))) float so[NS][DP];
  __shared__ float sml[NS][2];
  const int h = blockIdx.x, b = blockIdx.y;
  const int D = a.c.D;
  const int li = threadIdx.x % LN, st = threadIdx.x / LN;
  if (adv != nullptr && h == 0 && threadIdx.x == 0) {
    const int fill = adv[b];
    if (appends(a, fill)) adv[b] = fill + 1;
  }
  const size_t row = (size_t)b * a.Hq + h;
  const float* ml = a.ws_ml + row * a.n_chunks * 2;
  const float* po = a.ws_o + row * a.n_chunks * D;
  const bool here = li * 4 < D;
  float M = -INFINITY, L = 0.f;
  f32x4 O = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int s = st; s < a.n_chunks; s += NS) {
    const float2 x = *reinterpret_cast<const float2*>(ml + 2 * s);
    if (x.x == -INFINITY && x.y == 0.f) continue;  // no weight (and perhaps no o)
    const f32x4 v = here ? *reinterpret_cast<const f32x4*>(po + (size_t)s * D + li * 4)
                         : f32x4{0.f, 0.f, 0.f, 0.f};
    const float mn = fmaxf(M, x.x);
    const float ref = mn == -INFINITY ? 0.f : mn;
    const float wa = fast_exp2(M - ref), wb = fast_exp2(x.x - ref);
    L = fmaf(wb, x.y, wa * L);
    O = O * wa + v * wb;
    M = mn;
  }
  *reinterpret_cast<f32x4*>(&so[st][li * 4]) = O;
  if (li == 0) {
    sml[st][0] = M;
    sml[st][1] = L;
  }
  __syncthreads();
  for (int d = threadIdx.x; d < D; d += 256) {
    float MM = -INFINITY;
#pragma unroll
    for (int s = 0; s < NS; ++s) MM = fmaxf(MM, sml[s][0]);
    float LL = 0.f, OO = 0.f;
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      const float ms = sml[s][0];
      const float w = ms == -INFINITY ? 0.f : fast_exp2(ms - MM);
      LL = fmaf(w, sml[s][1], LL);
      OO = fmaf(w, so[s][d], OO);
    }
    store_elem(a.out, row * D + d, a.out_dt, OO / LL);
  }
}

bool dt_ok(int dt) { return dt == SKV_F32 || dt == SKV_BF16; }

int padded(int D) { return D <= 32 ? 32 : D <= 64 ? 64 : D <= 128 ? 128 : 256; }

constexpr int kCUs = 256;
constexpr int kStep = kWaves * kTile;  // tokens a workgroup takes at a time

template <int DP, int BITS, bool PAGED>
void launch_decode(const QDecodeArgs& a, unsigned blocks, bool exact32, hipStream_t s) {
  if (exact32)
    hipLaunchKernelGGL((k_q_decode<DP, BITS, PAGED, 3, 3>), dim3(blocks), dim3(kWaves * 64), 0, s,
                       a);
  else
    hipLaunchKernelGGL((k_q_decode<DP, BITS, PAGED, 1, 2>), dim3(blocks), dim3(kWaves * 64), 0, s,
                       a);
}

}  // namespace
}  // namespace skv

using namespace skv;

extern "C" int skv_q_decode_plan(int B, int H_kv, int max_len, long long total_len,
                                 int chunk_hint, int* chunk_tokens, int* n_chunks) {
  const char* fn = "skv_q_decode_plan";
  SKV_REQUIRE(chunk_tokens && n_chunks, SKV_E_INVALID, "%s: null output", fn);
  SKV_REQUIRE(B > 0 && H_kv > 0 && max_len > 0, SKV_E_INVALID,
              "%s: dims must be > 0 (B=%d H_kv=%d max_len=%d)", fn, B, H_kv, max_len);
  if (total_len <= 0 || total_len > (long long)B * max_len) total_len = (long long)B * max_len;
  long long chunk = chunk_hint;
  if (chunk <= 0) chunk = total_len * H_kv / (4 * kCUs);
  chunk = (chunk + kStep - 1) / kStep * kStep;
  if (chunk < kStep) chunk = kStep;
  const long long most = ((long long)max_len + kStep - 1) / kStep * kStep;
  if (chunk > most) chunk = most;
  *chunk_tokens = (int)chunk;
  *n_chunks = (int)((max_len + chunk - 1) / chunk);
  return SKV_OK;
}

extern "C" size_t skv_q_decode_workspace_bytes(int B, int H_q, int D, int n_chunks) {
  if (B <= 0 || H_q <= 0 || D <= 0 || n_chunks <= 0) return 0;
  return (size_t)B * H_q * n_chunks * (size_t)(D + 2) * sizeof(float);
}

extern "C" int skv_q_decode_attn(void* out, const void* q, void* k, void* k_scale, void* v,
                                 void* v_scale, const void* new_k, const void* new_v,
                                 int32_t* lens, const int32_t* block_table, int max_blocks,
                                 int block_size, int B, int H_q, int H_kv, int D, int T_cap,
                                 float scale, int chunk_tokens, int n_chunks, void* ws,
                                 size_t ws_bytes, int fmt, int in_dt, int q_dt, int out_dt,
                                 skv_stream_t stream) {
  const char* fn = "skv_q_decode_attn";
  QDecodeArgs a;
  int rc = quant_cache_args(&a.c, k, k_scale, v, v_scale, block_table, max_blocks, block_size, B,
                            H_kv, D, T_cap, fmt, fn);
  if (rc) return rc;
  SKV_REQUIRE(out && q && lens, SKV_E_INVALID, "%s: null pointer argument", fn);
  SKV_REQUIRE(!new_k == !new_v, SKV_E_INVALID, "%s: new_k and new_v come together", fn);
  SKV_REQUIRE(dt_ok(q_dt) && dt_ok(out_dt) && (!new_k || dt_ok(in_dt)), SKV_E_INVALID,
              "%s: bad dtype", fn);
  SKV_REQUIRE((((uintptr_t)out | (uintptr_t)q | (uintptr_t)ws | (uintptr_t)new_k |
                (uintptr_t)new_v) & 15) == 0,
              SKV_E_INVALID, "%s: out, q, ws, new_k and new_v must be 16-byte aligned", fn);
  SKV_REQUIRE(H_q > 0 && H_q % H_kv == 0, SKV_E_INVALID, "%s: H_q=%d not a multiple of H_kv=%d",
              fn, H_q, H_kv);
  SKV_REQUIRE(H_q / H_kv <= kMaxG, SKV_E_UNSUPPORTED,
              "%s: %d query heads per kv head (block-scaled caches take up to %d)", fn, H_q / H_kv,
              kMaxG);
  SKV_REQUIRE(chunk_tokens > 0 && chunk_tokens % kStep == 0 && n_chunks >= 1, SKV_E_INVALID,
              "%s: chunk_tokens=%d must be a positive multiple of %d, n_chunks=%d positive", fn,
              chunk_tokens, kStep, n_chunks);
  const long long blocks = (long long)B * H_kv * n_chunks;
  SKV_REQUIRE(blocks < (1LL << 31) && (long long)chunk_tokens * n_chunks < (1LL << 31),
              SKV_E_UNSUPPORTED, "%s: grid too large", fn);
  const bool parts = n_chunks > 1;
  SKV_REQUIRE(!parts || (ws && ws_bytes >= skv_q_decode_workspace_bytes(B, H_q, D, n_chunks)),
              SKV_E_WORKSPACE, "%s: workspace %zu bytes < %zu required", fn, ws_bytes,
              skv_q_decode_workspace_bytes(B, H_q, D, n_chunks));
  a.out = out;
  a.q = q;
  a.lens = lens;
  a.B = B;
  a.Hq = H_q;
  a.G = H_q / H_kv;
  a.qscale = scale * LOG2E;
  a.q_dt = q_dt;
  a.out_dt = out_dt;
  a.chunk = chunk_tokens;
  a.n_chunks = n_chunks;
  a.ws_o = static_cast<float*>(ws);
  a.ws_ml = parts ? a.ws_o + (size_t)B * H_q * n_chunks * D : nullptr;
  a.new_k = new_k;
  a.new_v = new_v;
  a.in_dt = in_dt;
  const bool exact32 = q_dt == SKV_F32 || out_dt == SKV_F32;
  const int DP = padded(D), bits = fmt == SKV_MXFP4 ? 4 : 8;
  hipStream_t s = (hipStream_t)stream;
#define SKV_QD(DD, BB)                                                                          \
  if (DP == DD && bits == BB) {                                                                 \
    if (a.c.bt) launch_decode<DD, BB, true>(a, (unsigned)blocks, exact32, s);                    \
    else launch_decode<DD, BB, false>(a, (unsigned)blocks, exact32, s);                          \
  }
  SKV_QD(32, 4) SKV_QD(64, 4) SKV_QD(128, 4) SKV_QD(256, 4)
  SKV_QD(32, 8) SKV_QD(64, 8) SKV_QD(128, 8) SKV_QD(256, 8)
#undef SKV_QD
  rc = check_launch(fn);
  if (rc) return rc;
  if (parts) {
    int32_t* adv = new_k ? lens : nullptr;
    const dim3 grid(H_q, B);
    if (DP == 32) hipLaunchKernelGGL((k_q_merge<32>), grid, dim3(256), 0, s, a, adv);
    else if (DP == 64) hipLaunchKernelGGL((k_q_merge<64>), grid, dim3(256), 0, s, a, adv);
    else if (DP == 128) hipLaunchKernelGGL((k_q_merge<128>), grid, dim3(256), 0, s, a, adv);
    else hipLaunchKernelGGL((k_q_merge<256>), grid, dim3(256), 0, s, a, adv);
    return check_launch(fn);
  }
  if (!new_k) return SKV_OK;
  return skv_advance(lens, nullptr, 1, B, a.c.cap, stream);
}
