// Cached single-query attention over a block-scaled cache (quant.h): split-K
// flash decoding with both products on the matrix cores.
//
//   o[b, h] = softmax(scale * q[b, h] . K[b, 0:len, h / G]^T) . V[b, 0:len, h / G]
//
// attention_with_kv_cache of the reference
// (simple-llm/src/gpu/gpu_kv_cache.py:194-289) over the 4- and 8-bit storage.
//
// Work split: a workgroup of four wavefronts takes `chunk` consecutive tokens
// of one kv head of one sequence for its G query heads (1 to 16), each
// wavefront every fourth 32-token tile; the head-major cache makes a tile one
// run of bytes (2 KB of 4-bit codes at head dim 128). The wavefronts merge
// through LDS, and the chunks in a second launch, which also advances the
// fills of a fused append; one chunk a row writes the output itself.
//
// Bound by HBM: 4 x 16 x 128 of 32000 4-bit tokens (279 MB of codes and scales)
// take 49 us in the first launch (5.7 TB/s; its loads alone as long) and 4.6 in
// the merge, 50 to 53 us a call; 64 ragged paged sequences of 8 x 4 x 128 (144,900
// tokens) 38 us (159 MB, 4-bit) and 68 us (308 MB, 8-bit). Calls of different
// size fit 7.6 TB/s and 12 us of start and end. With 32000 tokens of 4 sequences,
// us a call, bf16 | fp32 in and out (4 x Hkv x G x D; 0.28 GB of 4-bit, 0.54 of
// 8-bit rows each):
//   4-bit  16 x 1 x 128 50 | 53,  x 4 51 | 54,  x 5 52 | 63,  x 16 58 | 70
//   8-bit  16 x 1 x 128 89 | 89,  x 16 94 | 97
//   4-bit   8 x 1 x 256 53 | 55,  x 8 57 | 78
//   8-bit   8 x 1 x 256 94 | 98,  x 8 97 | 105,  x 16 102 | 118
//
// A tile:
//  * S = K q^T (v_mfma_f32_16x16x32_bf16). Lane (r, kb) of a 16-token half
//    loads every fourth 16-byte piece of token r's codes, the kb-th first: the
//    contraction may take the elements in any order as long as q does too, so
//    eight elements at a time go to the matrix core as they lie, and a piece
//    has one scale. Converted to bf16 with the scale they are exact.
//  * Online softmax in fp32, each lane holding 8 of the 32 scores of its
//    column. The running max moves lazily: only when a score passes it by 8
//    (log2 units), which is also the only time the four lanes of a column
//    exchange anything; until then p <= 256 and the sums stay consistent.
//  * O^T += V^T P: V goes through LDS as bf16 (converted where the lane still
//    holds one group with one scale; after a transposition of the codes the
//    eight tokens of a lane would have eight), row-major with XOR-swizzled
//    16-byte chunks, and comes back transposed (ds_read_b64_tr_b16). The
//    probabilities are already in the operand's token order.
//    (The scaled f8f6f4 product takes 4- and 8-bit codes unconverted, against q
//    as two E4M3 parts: 1 to 2 % faster, but its sums carry fewer bits, and
//    outputs moved by about 2^-15 where these move by 2^-19: not taken.)
// Precision: K and V enter exactly. With fp32 in or out, q and p are three bf16
// parts (all bits of q, 2^-24 of p; what lies below 2^-133 is lost); with bf16
// in and out q is one part and p two (2^-17). The parts use the matrix core's columns that few heads leave
// idle: column c is head c % HC, slot c / HC, HC = 16, 8 or (three parts
// only) 4 being the smallest that holds G, and slot s takes part s (as the
// plain grouped-query kernel's duplicated columns do); parts beyond the slots
// are products of their own. Up to four heads cost the same at either
// precision. A head's scores are summed over the slots by rotations of the
// 16-lane row whose additions are symmetric, so every slot has the same bits
// and splits the same p.
// Tokens past the chunk reread its last row and get weight 0: no memory past
// the fill is touched, none of it meets a zero weight.
// No atomics: results are bitwise reproducible, and a paged cache gives the
// bits of the same rows in a contiguous one.
#include <cmath>

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
  // scores are qscale * ((qsign * q) . k), in log2 units: qscale = |softmax
  // scale| * log2(e), qsign its sign (0 for a scale of 0, with qscale 1)
  float qscale, qsign;
  int q_dt, out_dt;
  int chunk, n_chunks;  // tokens a workgroup takes; chunks the workspace has room for
  int n_wg;             // workgroups of a kv head
  float* ws_o;   // [B * Hq][n_chunks][D]
  float* ws_ml;  // [B * Hq][n_chunks][4]: m, l, and in chunk 0 the number of chunks (int), 0
  const void* new_k;  // fused append, or NULL
  const void* new_v;
  int in_dt;
};

__device__ __forceinline__ bool appends(const QDecodeArgs& a, int len) {
  return a.new_k != nullptr && len >= 0 && len < a.c.cap;
}

// W <= 4 words from p (aligned to 4 W bytes), read once: non-temporal (4 x 16 x
// 128 of 32000 tokens, 4-bit, 59 -> 53 us). One instruction takes all that a
// lane reads of its 64-byte stretch: as two of 16 bytes at a stride of 32 the
// 8-bit rows were fetched twice (64 ragged sequences 66 -> 82 us).
template <int W>
__device__ __forceinline__ void load_words(const uint8_t* p, uint32_t* w) {
  if constexpr (W == 4) {
    const u32x4_t x = stream_load16(p);
    w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w;
  } else if constexpr (W == 2) {
    const u32x2_t x = stream_load8(p);
    w[0] = x.x; w[1] = x.y;
  } else {
    static_assert(W == 1, "1, 2 or 4 words");
    w[0] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(p));
  }
}

// ds_read_b64_tr_b16: within each 16-lane group, lane i receives as its slot j
// the element i%4 of the four 16-bit values addressed by lane 4j + i/4.
__device__ __forceinline__ i16x4 lds_read_tr16(const uint16_t* p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4*)(p));
}

// The swizzle of a bf16 V row in LDS (element offset of 16-byte chunk ch of
// token t). Two patterns must each hit distinct banks of the 256-byte sweep: eight
// lanes' stores take every second (8-bit) or fourth chunk of their rows, a
// transposed read two adjacent chunks of 8 consecutive rows. (With a key that spread four
// adjacent chunks of four rows instead, LDS was busy 76 % of the time over
// 4 x 16 x 128 of 32000 tokens, two thirds of it conflicts.)
template <int DP>
__device__ __forceinline__ int v_at(int t, int ch) {
  int key;
  if constexpr (DP == 256) key = 2 * (t & 7) ^ 2 * (ch >> 4);
  else if constexpr (DP == 128) key = 2 * (t & 7);
  else if constexpr (DP == 64) key = 2 * ((t >> 1) & 3);
  else key = 2 * ((t >> 2) & 1);
  return t * DP + ((ch ^ key) * 8);
}

// LDS written by some lanes of a wavefront is read by others: LDS operations
// of a wavefront complete in order, so only the compiler must keep theirs.
__device__ __forceinline__ void wave_lds_order() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Where the rows of a tile lie. The address of a load is a base that is the
// same for the whole wavefront (of a run of rows that lie end to end) plus a
// 32-bit lane offset: with 64-bit rows per lane a quarter of the loop's
// instructions computed addresses.
enum Pages {
  kContig = 0,      // no pages
  kPages16 = 1,     // pages of at least 16 tokens: a half tile lies in one
  kPagesSmall = 2,  // smaller ones: every lane looks its row up
};

// What is left of x after its first bf16 part (exact).
__device__ __forceinline__ float rest(float x) { return x - (float)(__bf16)x; }

// What this lane's slot takes of x: the part after the `slot` first ones
// (after the conversion to bf16). f[i] is 1 where slot > i, else 0. Three parts
// are all of an fp32 value, so a fourth slot takes 0.
template <int SL>
__device__ __forceinline__ float slot_part(float x, const float (&f)[3]) {
#pragma unroll
  for (int i = 0; i < SL - 1; ++i) x = fmaf(-f[i], (float)(__bf16)x, x);
  return x;
}

// x + the same head's values of the other slots, the same bits in each (SL
// slots of 16 / SL columns; rotations within the 16-lane row).
template <int CTRL>
__device__ __forceinline__ float ror(float x) {  // every lane has a source: part of the add
  return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), CTRL, 0xF, 0xF, true));
}
template <int SL>
__device__ __forceinline__ float slot_sum(float x) {
  if constexpr (SL >= 2) x += ror<0x128>(x);  // row_ror:8
  if constexpr (SL >= 4) x += ror<0x124>(x);  // row_ror:4
  return x;
}

// Four consecutive outputs.
__device__ __forceinline__ void store4_out(void* out, size_t i, int dt, f32x4 x) {
  if (dt == SKV_BF16) {
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(out) + i) =
        make_uint2((uint32_t)f32_to_bf16(x[0]) | ((uint32_t)f32_to_bf16(x[1]) << 16),
                   (uint32_t)f32_to_bf16(x[2]) | ((uint32_t)f32_to_bf16(x[3]) << 16));
  } else {
    *reinterpret_cast<f32x4*>(static_cast<float*>(out) + i) = x;
  }
}

// The row of a fused append at position t: threads [0, 2 D / 8) of the
// workgroup, all of them of its first wavefront.
template <int BITS, bool PAGED>
__device__ __forceinline__ void append_row(const QDecodeArgs& a, int b, int hk, int t, int tid) {
  const int opr = a.c.D / 8;
  if (tid >= 2 * opr) return;
  const bool isv = tid >= opr;
  const int o = isv ? tid - opr : tid;
  float x[8];
  load8_f32(isv ? a.new_v : a.new_k, ((size_t)b * a.c.Hkv + hk) * a.c.D + o * 8, a.in_dt, x);
  uint32_t w[Fmt<BITS>::NW];
  const uint32_t byte = quantise8<BITS>(x, w);
  store8<BITS>(isv ? a.c.v : a.c.k, isv ? a.c.vs : a.c.ks, row_of<PAGED>(a.c, b, hk, t), a.c.D, o,
               w, byte);
}

// Which sequence and chunk workgroup w of a kv head has, and what it needs to
// know of the sequence.
struct Piece {
  int b, ci, len;
  int n;     // chunks of the sequence
  bool app;  // a fused append adds its token (len counts it)
  bool cut;  // the grid does not hold all of its chunks
};

__device__ __forceinline__ int row_len(const QDecodeArgs& a, int fill, bool* app) {
  *app = appends(a, fill);
  return min(max(fill, 0), a.c.cap) + (*app ? 1 : 0);
}

// Chunks of a row: at least one (which stores an empty sequence's zeros), at
// most what the workspace holds.
__device__ __forceinline__ int n_pieces(const QDecodeArgs& a, int len) {
  return min(max((len + a.chunk - 1) / a.chunk, 1), a.n_chunks);
}

// Batches of up to this many sequences run only the workgroups that have
// tokens: each finds its place by a prefix sum over the sequences' chunk
// counts. (With one for every chunk of the longest row, those of shorter rows
// wait for a workgroup's LDS only to leave: 64 ragged sequences of 8 kv heads,
// 146,000 tokens in 8 chunks of the longest, 45 us against 33 for equal ones.
// In larger batches the chunks of the longest row are few: ragged, 8 kv heads x
// 4 x 128, 192 and 256 sequences with the scan 3.4 and 3.8 TB/s, 257, 288 and 320
// without it 4.4, 3.7 and 4.4.)
constexpr int kMaxScan = 256;

// Uniform over the wavefront. b = a.B: no sequence.
__device__ __forceinline__ Piece find_piece(const QDecodeArgs& a, int w, int lane) {
  Piece p;
  if (a.n_chunks == 1 || a.B > kMaxScan) {  // chunks slowest
    p.ci = a.n_chunks == 1 ? 0 : w / a.B;
    p.b = w - p.ci * a.B;
    p.len = row_len(a, a.lens[p.b], &p.app);
    p.n = n_pieces(a, p.len);
    p.cut = false;
    return p;
  }
  p.b = a.B;
  p.ci = 0;
  p.len = 0;
  p.n = 0;
  p.app = p.cut = false;
  int base = 0;
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    const int b = b0 + lane;
    bool app;
    const int len = row_len(a, a.lens[min(b, a.B - 1)], &app);
    const int n = b < a.B ? n_pieces(a, len) : 0;
    const int incl = base + wave_scan(n);
    const int total = __builtin_amdgcn_readlane(incl, 63);
    if (w < total) {
      const int at = __popcll(__ballot(incl <= w));  // the first lane whose chunks pass w
      p.b = b0 + at;
      p.ci = w - __builtin_amdgcn_readlane(incl - n, at);
      p.len = __builtin_amdgcn_readlane(len, at);
      p.n = __builtin_amdgcn_readlane(n, at);
      p.app = __builtin_amdgcn_readlane((int)app, at) != 0;
      p.cut = __builtin_amdgcn_readlane(incl, at) > a.n_wg;
      return p;
    }
    base = total;
  }
  return p;
}

// The last workgroup of a kv head also takes the sequences behind its own, which
// exist only where the fills outgrew the plan: NaN rows (chunk 0 alone, l =
// NaN), a fused append's token stored all the same.
template <int BITS, bool PAGED>
__device__ __forceinline__ void left_over(const QDecodeArgs& a, int hk, const Piece& pc, int tid) {
  // a sequence's first chunk is its own workgroup: those after pc.b have none
  for (int b = pc.b + 1; b < a.B; ++b) {
    bool app;
    const int len = row_len(a, a.lens[b], &app);
    if (app) append_row<BITS, PAGED>(a, b, hk, len - 1, tid);
    if (tid < a.G)
      *reinterpret_cast<float4*>(
          a.ws_ml + ((size_t)b * a.Hq + hk * a.G + tid) * a.n_chunks * 4) =
          make_float4(0.f, __builtin_nanf(""), __int_as_float(1), 0.f);
  }
}

// Wavefronts per SIMD the registers are kept for, and so workgroups per CU: as
// many as fit without spilling. At head dim 128 four instead of three are worth
// 59 -> 52 us on 4 x 16 x 128 of 32000 4-bit tokens; 8-bit ones need three
// (100 -> 92 us; at four a few registers spill in the loop).
constexpr int min_waves(int DP, int BITS, int SL, bool F32) {
  if (DP <= 64) return 4;
  if (DP == 128) return F32 && SL < 4 ? 2 : BITS == 4 ? 4 : 3;
  return F32 && (SL < 4 || BITS == 8) ? 1 : 2;
}

// Slots of 16 / slots columns for G heads.
constexpr int slots_for(int G, bool F32) { return G > 8 ? 1 : F32 && G <= 4 ? 4 : 2; }

// DP: head dim padded to a power of two (elements past D: q is zero, rows of
// O^T are not stored). SL slots of HC = 16 / SL heads; F32: fp32 products.
template <int DP, int BITS, int PG, int SL, bool F32>
__global__ __launch_bounds__(kWaves * 64, min_waves(DP, BITS, SL, F32)) void k_q_decode(
    QDecodeArgs a) {
  constexpr int NW = Fmt<BITS>::NW;
  constexpr int E16 = 128 / BITS;                // elements in 16 bytes (one scale)
  constexpr int KE = DP / 4;                     // elements of a K row per lane
  constexpr int KO = KE / 8;                     // ... by eight: MFMAs per half tile
  constexpr int PE = KE < E16 ? KE : E16;        // elements of a lane's piece of a K row
  constexpr int KP = KE / PE;                    // pieces
  constexpr int VL = DP / E16;                   // lanes of a V row
  constexpr int VR = VL == 1 ? kTile : 64 / VL;  // V rows a pass moves (one lane a row: half idle)
  constexpr int VP = kTile / VR;                 // passes
  constexpr int DB = DP / 16;
  constexpr int HC = 16 / SL;
  constexpr int QS = F32 ? (3 + SL - 1) / SL : 1;          // operand sets of q ...
  constexpr int PS = ((F32 ? 3 : 2) + SL - 1) / SL;        // ... and of p
  __shared__ __attribute__((aligned(16))) uint16_t sv[kWaves][kTile * DP];
  __shared__ float sml[kWaves][kMaxG][2];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hk = blockIdx.x;
  const Piece pc = find_piece(a, blockIdx.y, lane);
  const int D = a.c.D, G = a.G;
  if (a.B <= kMaxScan && a.n_chunks > 1 && (int)blockIdx.y == a.n_wg - 1)
    left_over<BITS, PG != kContig>(a, hk, pc, tid);
  const int b = pc.b, ci = pc.ci, len = pc.len;
  if (b >= a.B || ci >= pc.n) return;
  const bool app = pc.app;
  const int start = ci * a.chunk;
  const int end = min(len, start + a.chunk);
  const size_t head0 = (size_t)b * a.Hq + hk * G;  // first query head's output row
  // the plan does not cover the fill: NaN
  const bool outgrown = (ci == a.n_chunks - 1 && len > end) || (ci == 0 && pc.cut);

  if (len == 0) {
    // nothing to attend: a zero output (as a part: m = 0, l = 1, o = 0)
    for (int i = tid; i < G * D; i += kWaves * 64) {
      const int g = i / D, d = i - g * D;
      if (a.n_chunks == 1) store_elem(a.out, (head0 + g) * D + d, a.out_dt, 0.f);
      else a.ws_o[(head0 + g) * a.n_chunks * D + d] = 0.f;
    }
    if (a.n_chunks > 1 && tid < G)
      *reinterpret_cast<float4*>(a.ws_ml + (head0 + tid) * a.n_chunks * 4) =
          make_float4(0.f, 1.f, __int_as_float(1), 0.f);
    return;
  }

  // A fused append: the chunk that holds the new token writes its row first
  // and the workgroup reads it back from the cache as any other.
  if (app && (end == len || outgrown)) {
    append_row<BITS, PG != kContig>(a, b, hk, len - 1, tid);
    __builtin_amdgcn_s_waitcnt(0);  // the stores have completed
    __syncthreads();
  }

  const int cl = lane & 15, kb = lane >> 4;  // MFMA row/column, k block

  const int cb = D * BITS / 8, sb = D / kGroup;  // code and scale bytes of a row
  // this lane's places in a K row: code offset and scale index of each piece
  // (past the head dim: the first group's, which meet a zero query)
  auto k_el = [&](int i) { return (4 * i + kb) * PE; };
  int ko[KP], ks[KP];
#pragma unroll
  for (int i = 0; i < KP; ++i) {
    ko[i] = k_el(i) < D ? k_el(i) * BITS / 8 : 0;
    ks[i] = k_el(i) < D ? k_el(i) / kGroup : 0;
  }
  // ... and in a V row
  const int vg = VL == 1 ? 0 : lane % VL, vr = VL == 1 ? (lane & (kTile - 1)) : lane / VL;
  const int vo = vg * E16 < D ? vg * 16 : 0, vs = vg * E16 < D ? vg * E16 / kGroup : 0;

  constexpr int PW = PE * BITS / 32;  // words of a K piece
  uint32_t kw[2][KP * PW], kscale[2][KP], vw[VP][4], vscale[VP];
  // Pages of this wavefront's next 32 tiles, lane 2 i + u holding half u of the
  // i-th (kPages16): one load in 32 tiles instead of a scalar one in each, whose
  // wait is for all LDS operations too.
  int pages = 0, tile = 0;
  // First row of each half of the tile at t0 and its last one that may be read
  // (relative); a half wholly past the end rereads the first.
  size_t r0[2] = {0, 0};
  int lim[2] = {0, 0};
  auto place = [&](int t0) {
    if constexpr (PG == kPages16) {
      if (tile % 32 == 0) {
        const int T = t0 + (lane >> 1) * (kWaves * kTile) + (lane & 1) * 16;
        pages = a.c.bt[(size_t)b * a.c.max_blocks + (min(T, end - 1) >> a.c.bs_shift)];
      }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int T = t0 + 16 * u < end ? t0 + 16 * u : t0;
      lim[u] = min(15, end - 1 - T);
      if constexpr (PG == kPages16)
        r0[u] = (((size_t)__builtin_amdgcn_readlane(pages, 2 * (tile & 31) + (T != t0 ? u : 0)) *
                      a.c.Hkv + hk) << a.c.bs_shift) + (T & ((1 << a.c.bs_shift) - 1));
      else
        r0[u] = ((size_t)b * a.c.Hkv + hk) * a.c.T_cap + T;
    }
    ++tile;
  };
  auto load_k = [&](int t0) {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      size_t base = r0[u];
      uint32_t r = min(cl, lim[u]);
      if constexpr (PG == kPagesSmall) {
        base = row_of<true>(a.c, b, hk, min(t0 + 16 * u + cl, end - 1));
        r = 0;
      }
#pragma unroll
      for (int i = 0; i < KP; ++i) {
        load_words<PW>(a.c.k + base * cb + (r * (uint32_t)cb + ko[i]), &kw[u][i * PW]);
        kscale[u][i] = (a.c.ks + base * sb)[r * (uint32_t)sb + ks[i]];
      }
    }
  };
  auto load_v = [&](int t0) {
#pragma unroll
    for (int p = 0; p < VP; ++p) {
      size_t base;
      uint32_t r;
      if constexpr (PG == kPagesSmall) {
        base = row_of<true>(a.c, b, hk, min(t0 + p * VR + vr, end - 1));
        r = 0;
      } else if constexpr (VR <= 16) {  // a pass lies in one half
        const int u = p * VR / 16;
        base = r0[u];
        r = min(p * VR % 16 + vr, lim[u]);
      } else if constexpr (PG == kContig) {  // the tile's rows lie end to end
        base = r0[0];
        r = min(vr, min(kTile - 1, end - 1 - t0));
      } else {
        base = vr < 16 ? r0[0] : r0[1];
        r = min(vr & 15, vr < 16 ? lim[0] : lim[1]);
      }
      load_words<4>(a.c.v + base * cb + (r * (uint32_t)cb + vo), vw[p]);
      vscale[p] = (a.c.vs + base * sb)[r * (uint32_t)sb + vs];
    }
  };

  // the first tile's codes, in flight while the queries are converted
  int t0 = start + wave * kTile;
  if (t0 < end) {
    place(t0);
    load_k(t0);
    load_v(t0);
  }

  // ---- queries, operand B: column cl is head cl % HC, in the
  // order of a lane's pieces ----
  const int head = cl % HC, slot = cl / HC;
  const float sf[3] = {slot > 0 ? 1.f : 0.f, slot > 1 ? 1.f : 0.f, slot > 2 ? 1.f : 0.f};
  bf16x8 qf[QS][KO];
  float xq[KO][8];
#pragma unroll
  for (int i = 0; i < KO; ++i) {
    const int e = k_el(i / (PE / 8)) + i % (PE / 8) * 8;
    load8_f32(a.q, (head0 + (head < G ? head : 0)) * D + (e < D ? e : 0), a.q_dt, xq[i]);
  }
  // Parts below bf16's smallest number (2^-133) are lost: a query whose elements
  // all are below 2^-64 enters 2^40 times as large.
  float qsign = a.qsign, qscale = a.qscale;
  if constexpr (F32) {
    float big = 0.f;
#pragma unroll
    for (int i = 0; i < KO; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) big = fmaxf(big, fabsf(xq[i][j]));
    big = xor32_max(fmaxf(big, __shfl_xor(big, 16)));
    if (big < 0x1p-64f) {
      qsign *= 0x1p40f;
      qscale *= 0x1p-40f;
    }
  }
#pragma unroll
  for (int i = 0; i < KO; ++i) {
    const int e = k_el(i / (PE / 8)) + i % (PE / 8) * 8;
    const bool used = head < G && e < D;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float r = used ? xq[i][j] * qsign : 0.f;
#pragma unroll
      for (int t = 0; t < QS; ++t) {
        // bf16: every slot takes q itself and has the whole score
        qf[t][i][j] = (__bf16)(F32 ? slot_part<SL>(r, sf) : r);
#pragma unroll
        for (int k = 0; k < SL; ++k) r = rest(r);
      }
    }
  }

  f32x4 o[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) o[db] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m_run = -INFINITY, l_run = 0.f;
  uint16_t* svw = sv[wave];

  for (; t0 < end; t0 += kWaves * kTile) {
    // ---- scores of the two halves ----
    f32x4 sc[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      sc[u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < KO; ++i) {
        const bf16x8 kf = decode8_bf16<BITS>(&kw[u][i * NW], scale_f32(kscale[u][i * KP / KO]));
#pragma unroll
        for (int t = 0; t < QS; ++t)
          sc[u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[t][i], sc[u], 0, 0, 0);
      }
      if constexpr (F32)
#pragma unroll
        for (int j = 0; j < 4; ++j) sc[u][j] = slot_sum<SL>(sc[u][j]);
    }
    // The next tile's codes are on their way as soon as this one's have left
    // the registers: K's now, V's after they went to LDS as bf16.
    const int tn = t0 + kWaves * kTile;
    if (tn < end) {
      place(tn);
      load_k(tn);
    }
#pragma unroll
    for (int p = 0; p < VP; ++p)
#pragma unroll
      for (int i = 0; i < E16 / 8; ++i) {
        const bf16x8 x = decode8_bf16<BITS>(&vw[p][i * NW], scale_f32(vscale[p]));
        *reinterpret_cast<bf16x8*>(svw + v_at<DP>(p * VR + vr, vg * (E16 / 8) + i)) = x;
      }
    if (tn < end) load_v(tn);

    // ---- softmax: lane (cl, kb) has tokens t0 + 16 u + 4 kb + j ----
    if (t0 + kTile > end) {  // uniform
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (t0 + 16 * u + 4 * kb + j >= end) sc[u][j] = -INFINITY;
    }
    float mt = sc[0][0];
#pragma unroll
    for (int j = 1; j < 8; ++j) mt = fmaxf(mt, sc[j >> 2][j & 3]);
    mt *= qscale;
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
    bf16x8 pf[PS];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float r = fast_exp2(fmaf(sc[j >> 2][j & 3], qscale, -m_use));
      l_run += r;
#pragma unroll
      for (int t = 0; t < PS; ++t) {
        pf[t][j] = (__bf16)slot_part<SL>(r, sf);
        if (t + 1 < PS)
#pragma unroll
          for (int k = 0; k < SL; ++k) r = rest(r);
      }
    }
    // ---- O^T += V^T P: elements 0-3 are tokens 4 kb + j, 4-7 are 16 + 4 kb + j ----
    wave_lds_order();
#pragma unroll
    for (int db = 0; db < DB; ++db) {
      const int ch = 2 * db + ((cl & 3) >> 1), in = 4 * (cl & 1);
      const i16x4 lo = lds_read_tr16(svw + v_at<DP>(4 * kb + (cl >> 2), ch) + in);
      const i16x4 hi = lds_read_tr16(svw + v_at<DP>(16 + 4 * kb + (cl >> 2), ch) + in);
      const bf16x8 va =
          __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
      for (int t = 0; t < PS; ++t)
        o[db] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va, pf[t], o[db], 0, 0, 0);
    }
    wave_lds_order();
  }

  // ---- the wavefronts' parts merge through the V tiles' space ----
  float lt = l_run + __shfl_xor(l_run, 16);
  lt = xor32_sum(lt);
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int j = 0; j < 4; ++j) o[db][j] = slot_sum<SL>(o[db][j]);
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
  constexpr int LN = DP / 4;  // four elements a thread
  const int d = tid % LN * 4;
  for (int g = tid / LN; g < G; g += kWaves * 64 / LN) {
    if (d >= D) break;
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
      store4_out(a.out, (head0 + g) * D + d, a.out_dt, O * (1.f / L));
    } else {
      const size_t at = (head0 + g) * a.n_chunks + ci;
      *reinterpret_cast<f32x4*>(a.ws_o + at * D + d) = O;
      if (d == 0)
        *reinterpret_cast<float4*>(a.ws_ml + at * 4) =
            make_float4(M, L, __int_as_float(pc.n), 0.f);
    }
  }
}

// Merge of the chunks' partials, grid (H_q, B): DP / 4 lanes of four elements
// by 1024 / DP streams of chunks, then the streams through LDS. adv (fused
// append): the fills, each advanced by its sequence's first workgroup; nothing
// else here reads them (chunk 0 has the number of chunks). The first four (m, l)
// and o of a stream are loaded together, before it is known whether the row has
// those chunks: one round trip to memory.
template <int DP>
__global__ __launch_bounds__(256) void k_q_merge(QDecodeArgs a, int32_t* adv) {
  constexpr int LN = DP / 4, NS = 256 / LN, U = 4;
  __shared__ __attribute__((aligned(16))) float so[NS][DP];
  __shared__ float sml[NS][2];
  const int h = blockIdx.x, b = blockIdx.y;
  const int D = a.c.D;
  const int li = threadIdx.x % LN, st = threadIdx.x / LN;
  const size_t row = (size_t)b * a.Hq + h;
  const float* ml = a.ws_ml + row * a.n_chunks * 4;
  const float* po = a.ws_o + row * a.n_chunks * D + (li * 4 < D ? li * 4 : 0);
  int n = __float_as_int(ml[2]);
  float M = -INFINITY, L = 0.f;
  f32x4 O = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int s0 = st; s0 < a.n_chunks; s0 += U * NS) {
    float2 x[U];
    f32x4 v[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int s = min(s0 + k * NS, a.n_chunks - 1);
      x[k] = *reinterpret_cast<const float2*>(ml + 4 * s);
      v[k] = *reinterpret_cast<const f32x4*>(po + (size_t)s * D);
    }
    float mn = M;
#pragma unroll
    for (int k = 0; k < U; ++k)
      if (s0 + k * NS < n) mn = fmaxf(mn, x[k].x);
    const float ref = mn == -INFINITY ? 0.f : mn;
    const float wa = fast_exp2(M - ref);
    L *= wa;
    O *= wa;
#pragma unroll
    for (int k = 0; k < U; ++k)
      if (s0 + k * NS < n) {
        const float w = fast_exp2(x[k].x - ref);
        L = fmaf(w, x[k].y, L);
        O += w * v[k];
      }
    M = mn;
    if (s0 + U * NS >= n) break;
  }
  if (adv != nullptr && h == 0 && threadIdx.x == 0) {
    const int fill = adv[b];
    if (appends(a, fill)) adv[b] = fill + 1;
  }
  *reinterpret_cast<f32x4*>(&so[st][li * 4]) = O;
  if (li == 0) {
    sml[st][0] = M;
    sml[st][1] = L;
  }
  __syncthreads();
  if (threadIdx.x * 4 >= D) return;
  const int d = threadIdx.x * 4;
  float MM = -INFINITY;
#pragma unroll
  for (int s = 0; s < NS; ++s) MM = fmaxf(MM, sml[s][0]);
  float LL = 0.f;
  f32x4 OO = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    const float ms = sml[s][0];
    const float w = ms == -INFINITY ? 0.f : fast_exp2(ms - MM);
    LL = fmaf(w, sml[s][1], LL);
    OO += w * *reinterpret_cast<const f32x4*>(&so[s][d]);
  }
  store4_out(a.out, row * D + d, a.out_dt, OO * (1.f / LL));
}

bool dt_ok(int dt) { return dt == SKV_F32 || dt == SKV_BF16; }

int padded(int D) { return D <= 32 ? 32 : D <= 64 ? 64 : D <= 128 ? 128 : 256; }

constexpr int kCUs = 256;
constexpr int kStep = kWaves * kTile;  // tokens a workgroup takes at a time

template <int DP, int BITS, int PG>
void launch_decode(const QDecodeArgs& a, bool f32, hipStream_t s) {
  const dim3 grid(a.c.Hkv, a.n_wg), block(kWaves * 64);
#define SKV_QS(SL, F) hipLaunchKernelGGL((k_q_decode<DP, BITS, PG, SL, F>), grid, block, 0, s, a)
  const int sl = slots_for(a.G, f32);
  if (f32 && sl == 4) SKV_QS(4, true);
  else if (f32 && sl == 2) SKV_QS(2, true);
  else if (f32) SKV_QS(1, true);
  else if (sl == 2) SKV_QS(2, false);
  else SKV_QS(1, false);
#undef SKV_QS
}

}  // namespace
}  // namespace skv

using namespace skv;

// The chunk: one round of workgroups, all resident (slots below). Equal rows
// take a whole number of chunks each, and one where the round holds two or
// fewer. That is the better choice past 512 rows only, us in one | two chunks
// (8 kv heads x 128, 4-bit, in bf16):
//   400 rows of 2288 tokens 31 | 29, of 8000 94 | 80, of 32000 354 | 278
//   512                     32 | 31,         99 | 95,          373 | 330
//   640                     37 | 45,        114 | 136,         435 | 484
// Rows that differ, by a token already, take the second rule, whose chunk comes
// out a little shorter than such rows: 640 of 32000, one of 31999, 650 us.
// Ragged ones leave half a chunk a row, which the round has to hold too (64
// sequences x 8 heads, 146,000 tokens: 49 us without that, 44 with). A chunk of
// 1024 tokens or more is no multiple of 512: workgroups that start whole multiples
// of 32 KB apart meet in the same memory channels (4 x 16 x 128 of 32000 4-bit
// tokens in a cache of 131072 positions, chunks of 2048 and 2176: 59.2 and 52.1
// us, in one of 32001 both 53.8; 1 x 8 x 4 x 128 of 131000, 1024 and 1152: 37.7
// and 35.4; 64 ragged x 8 x 4 x 128, 1536 and 1664: 39.8 and 38.8. Multiples of
// 256 gain nothing by a step more).
extern "C" int skv_q_decode_plan(int B, int H_q, int H_kv, int D, int fmt, int q_dt, int out_dt,
                                 int max_len, long long total_len, int covering, int chunk_hint,
                                 int* chunk_tokens, int* n_chunks, int* n_wg) {
  const char* fn = "skv_q_decode_plan";
  SKV_REQUIRE(chunk_tokens && n_chunks && n_wg, SKV_E_INVALID, "%s: null output", fn);
  SKV_REQUIRE(B > 0 && B <= 65535 && H_kv > 0 && H_q > 0 && H_q % H_kv == 0 && D > 0 &&
                  max_len > 0,
              SKV_E_INVALID, "%s: bad dims (B=%d H_q=%d H_kv=%d D=%d max_len=%d)", fn, B, H_q,
              H_kv, D, max_len);
  if (total_len <= 0 || total_len > (long long)B * max_len) total_len = (long long)B * max_len;
  const bool f32 = q_dt == SKV_F32 || out_dt == SKV_F32;
  const long long slots =
      (long long)kCUs * min_waves(padded(D), fmt == SKV_MXFP4 ? 4 : 8,
                                  slots_for(H_q / H_kv, f32), f32);
  const long long rows = (long long)B * H_kv;
  long long chunk = chunk_hint;
  if (chunk <= 0 && total_len == (long long)B * max_len) {
    const long long n = slots / rows;
    chunk = n <= 2 ? max_len : (max_len + n - 1) / n;
  } else if (chunk <= 0) {
    const long long whole = rows < slots ? slots - rows / 2 : slots / 2;
    chunk = total_len * H_kv / whole;
  }
  const long long most = ((long long)max_len + kStep - 1) / kStep * kStep;
  const long long n_most = 65535 / B;  // chunks a row that the grid holds
  const long long least = (max_len + n_most - 1) / n_most;
  if (chunk < least) chunk = least;
  chunk = (chunk + kStep - 1) / kStep * kStep;
  if (chunk_hint <= 0 && chunk >= 1024 && chunk % 512 == 0) chunk += kStep;
  if (chunk < kStep) chunk = kStep;
  if (chunk > most) chunk = most;
  if (chunk > quant::kMaxCap) chunk = quant::kMaxCap;
  const long long n = (max_len + chunk - 1) / chunk;
  // sum of ceil(len / chunk) <= total / chunk + B
  const long long some = total_len / chunk + B;
  *chunk_tokens = (int)chunk;
  *n_chunks = (int)n;
  *n_wg = (int)(covering || B > kMaxScan || some > B * n ? B * n : some);
  return SKV_OK;
}

extern "C" size_t skv_q_decode_workspace_bytes(int B, int H_q, int D, int n_chunks) {
  if (B <= 0 || H_q <= 0 || D <= 0 || n_chunks <= 0) return 0;
  return (size_t)B * H_q * n_chunks * (size_t)(D + 4) * sizeof(float);
}

extern "C" int skv_q_decode_attn(void* out, const void* q, void* k, void* k_scale, void* v,
                                 void* v_scale, const void* new_k, const void* new_v,
                                 int32_t* lens, const int32_t* block_table, int max_blocks,
                                 int block_size, int B, int H_q, int H_kv, int D, int T_cap,
                                 float scale, int chunk_tokens, int n_chunks, int n_wg, void* ws,
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
  SKV_REQUIRE(std::isfinite(scale), SKV_E_INVALID, "%s: scale must be finite", fn);
  SKV_REQUIRE(H_q / H_kv <= kMaxG, SKV_E_UNSUPPORTED,
              "%s: %d query heads per kv head (block-scaled caches take up to %d)", fn, H_q / H_kv,
              kMaxG);
  SKV_REQUIRE(chunk_tokens > 0 && chunk_tokens % kStep == 0 && n_chunks >= 1, SKV_E_INVALID,
              "%s: chunk_tokens=%d must be a positive multiple of %d, n_chunks=%d positive", fn,
              chunk_tokens, kStep, n_chunks);
  SKV_REQUIRE(chunk_tokens <= quant::kMaxCap && (long long)chunk_tokens * n_chunks < (1LL << 31) &&
                  (long long)B * H_q * n_chunks < (1LL << 31),
              SKV_E_UNSUPPORTED, "%s: plan too large", fn);
  // every chunk of every sequence, unless a batch small enough to be scanned
  // needs fewer workgroups
  const long long all = (long long)B * n_chunks;
  SKV_REQUIRE(n_wg == all || (B <= kMaxScan && n_wg >= B && n_wg < all), SKV_E_INVALID,
              "%s: n_wg=%d for %d sequences of %d chunks", fn, n_wg, B, n_chunks);
  SKV_REQUIRE(n_wg <= 65535, SKV_E_UNSUPPORTED, "%s: grid too large (%d workgroups a head)", fn,
              n_wg);
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
  a.qscale = scale == 0.f ? 1.f : fabsf(scale) * LOG2E;
  a.qsign = scale == 0.f ? 0.f : copysignf(1.f, scale);
  a.q_dt = q_dt;
  a.out_dt = out_dt;
  a.chunk = chunk_tokens;
  a.n_chunks = n_chunks;
  a.n_wg = n_wg;
  a.ws_o = static_cast<float*>(ws);
  a.ws_ml = parts ? a.ws_o + (size_t)B * H_q * n_chunks * D : nullptr;
  a.new_k = new_k;
  a.new_v = new_v;
  a.in_dt = in_dt;
  const bool f32 = q_dt == SKV_F32 || out_dt == SKV_F32;
  const int DP = padded(D), bits = fmt == SKV_MXFP4 ? 4 : 8;
  hipStream_t s = (hipStream_t)stream;
#define SKV_QD(DD, BB)                                                                          \
  if (DP == DD && bits == BB) {                                                                 \
    if (!a.c.bt) launch_decode<DD, BB, kContig>(a, f32, s);                                     \
    else if (a.c.bs_shift >= 4) launch_decode<DD, BB, kPages16>(a, f32, s);                     \
    else launch_decode<DD, BB, kPagesSmall>(a, f32, s);                                         \
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
