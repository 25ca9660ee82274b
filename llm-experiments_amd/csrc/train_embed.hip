// The embedding lookup of a training step, and the gradient of its table.
//
//   out[i]  = scale table[id[i]] + pos[i mod n]
//   grad[v] = (what was there, or 0) + scale sum over id[i] = v of dout[i]
//
// An id outside [0, V) is padding: it adds no table row and no gradient.
//
// The gradient sorts the tokens by id (stably), so that a table row's tokens lie
// together and its sum runs in token order: no atomics on floats, the same bits
// every time. Three kernels:
//
//   sort  a workgroup has a bucket of consecutive ids. It counts their tokens
//         and the tokens of all smaller ids (where its part of the order begins)
//         in a scan over all ids, and places the tokens. Beside these workgroups
//         others set the table to zero, which is most of what this operator
//         writes and would otherwise wait for the order.
//   sum   a wavefront has 64 columns' vectors and a range of kRange sorted tokens,
//         whatever their ids: the work is even however unevenly the ids occur. A
//         row whose tokens all lie in the range is written; one that crosses a
//         range's border leaves its part.
//   join  adds the parts of each such row, in order.
//
// 16384 zipf tokens, table 50304 x 768 fp32 (154 MB written, 50 read): sort 29 us, most of
// it the zeros (6.5 without them), sum 14, join 5; 46 us in all. One bucket per CU and not
// two: 52.5 against 57 us. Zeros with the nt bit: 51 -> 47. The sort of 65536 tokens: 14
// to 19 us, 28 to 36 with every run read twice and its batches' places found unasked.
#include "train_common.h"

namespace skv {
namespace {

using namespace train;

constexpr int kMaxD = 1 << 22;
constexpr int kBucket = 256;  // ids of a bucket, at most
constexpr int kWaves = 16;    // wavefronts of a sorting workgroup
constexpr int kBatches = 8;   // batches of 64 tokens a sorting wavefront reads at a time
constexpr int kList = 1280;   // the tokens that it can list
constexpr int kRange = 16;    // sorted tokens of a summing wavefront
constexpr int kJoinWaves = 8;
constexpr int kZeroGroups = 128;  // workgroups that zero the table

// ---------------------------------------------------------------------------
// lookup
// ---------------------------------------------------------------------------

// A token has LPT lanes, a wavefront or, where that leaves a lane two vectors or fewer, a
// quarter of one (65536 tokens: 64 columns of fp32 11.2 -> 5.7 us, 256 of bf16 14.3 -> 9.0;
// 256 of fp32 would be 15.2 -> 16.1); VEC columns a lane and step.
template <typename TT, typename TO, int VEC, int LPT, int KIND>
__global__ __launch_bounds__(256) void k_embed_rows(TO* __restrict__ out,
                                                    const int32_t* __restrict__ ids,
                                                    const TT* __restrict__ table,
                                                    const float* __restrict__ pos, int T, int V,
                                                    int d, int n_pos, float scale) {
  const int i = blockIdx.x * (256 / LPT) + threadIdx.x / LPT, lane = threadIdx.x % LPT;
  if (i >= T) return;
  const int id = ids[i];
  const bool real = (unsigned)id < (unsigned)V;
  const TT* row = table + (size_t)(real ? id : 0) * d;
  const float* pr = pos ? pos + (size_t)(i % n_pos) * d : nullptr;
  TO* o = out + (size_t)i * d;
#pragma unroll 4
  for (int j = lane * VEC; j < d; j += LPT * VEC) {
    Vec<TT, VEC> t;
    Vec<float, VEC> p;
    t.zero();
    p.zero();
    if (real) t.template load_row<KIND>(row, j, d);
    if (pr) p.template load_row<KIND>(pr, j, d);
    t.template settle<KIND>(j, d);
    p.template settle<KIND>(j, d);
    float r[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) r[e] = t.get(e) * scale + p.get(e);
    Vec<TO, VEC>::template store_stream_row<KIND>(o, j, d, r);
  }
}

// ---------------------------------------------------------------------------
// gradient: the tokens sorted by id
// ---------------------------------------------------------------------------

struct Sorted {
  int32_t* pos;    // [T] tokens in order of their ids
  int32_t* id;     // [T] their ids
  int32_t* begin;  // [V + 1] where an id's tokens begin
  int2* goes_on;   // [ranges] of a row that begins in a range and goes on: its id and the
                   // number of ranges it lies in; or (-1, 0)
};

// what the wavefront's other lanes wrote to LDS is read behind this
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

__device__ __forceinline__ int wave_isum(int x) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) x += __shfl_xor(x, o);
  return x;
}

// width: ids of a bucket. Each wavefront has a run of consecutive tokens; an id's tokens
// are placed by wavefront, then by token. The bucket's own tokens go to a list in LDS, in
// order: it is short but for a bucket of frequent ids (of 16384 zipf tokens a bucket of 197
// ids has 64 on average, the largest some 700, 50 to 100 in a wavefront), and what finds an
// id's rank among 64 tokens costs 0.3 us. Where the list does not hold them, the run is read again.
__global__ __launch_bounds__(kWaves * 64, 8) void k_embed_sort(Sorted s,
                                                               const int32_t* __restrict__ ids,
                                                               int T, int V, int width, int buckets,
                                                               float* __restrict__ grad,
                                                               size_t n_zero) {
  if ((int)blockIdx.x >= buckets) {
    const size_t step = (size_t)(gridDim.x - buckets) * kWaves * 64 * 4;
    const size_t i0 = (size_t)(blockIdx.x - buckets) * kWaves * 64 + threadIdx.x;
    for (size_t i = i0 * 4; i + 4 <= n_zero; i += step)
      __builtin_nontemporal_store(f32x4_t{0.f, 0.f, 0.f, 0.f}, reinterpret_cast<f32x4_t*>(grad + i));
    if (i0 < n_zero % 4) grad[n_zero - 1 - i0] = 0.f;
    return;
  }
  constexpr int kRead = kBatches * 64;
  __shared__ int cnt[kWaves][kBucket];
  __shared__ int tot[kBucket];   // tokens of an id
  __shared__ int base[kBucket];  // where they begin in the bucket
  __shared__ int less[kWaves];
  __shared__ uint16_t list_t[kWaves][kList];  // the bucket's tokens in the run
  __shared__ uint8_t list_l[kWaves][kList];   // and their ids' places in the bucket
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int lo = blockIdx.x * width, n_ids = min(width, V - lo);
  const int per = ((T + kWaves * 64 - 1) / (kWaves * 64)) * 64;
  const int t0 = min(w * per, T), t1 = min(t0 + per, T);
  int upto = 0, n = 0;  // tokens of ids below lo + n_ids; tokens in the list
  const auto load = [&](int (&id)[kBatches], int t) {
    if (t + kRead <= t1) {
#pragma unroll
      for (int i = 0; i < kBatches; ++i) id[i] = (ids + t)[lane + i * 64];
    } else {
#pragma unroll
      for (int i = 0; i < kBatches; ++i) {
        const int k = t + i * 64 + lane, x = ids[min(k, t1 - 1)];
        id[i] = k < t1 ? x : -1;
      }
    }
  };
  // the bucket's tokens of those read to the list; `at` is the place of the first of them
  const auto enlist = [&](const int (&id)[kBatches], int at) {
#pragma unroll
    for (int i = 0; i < kBatches; ++i) {
      const unsigned l = (unsigned)id[i] - lo;
      const bool in = l < (unsigned)n_ids;
      upto += __popcll(__ballot((unsigned)id[i] < (unsigned)(lo + n_ids)));
      const uint64_t mask = __ballot(in);
      if (mask) {  // most batches have none
        if (in) {
          const int to = n + __popcll(mask & ((1ull << lane) - 1));
          list_t[w][to] = (uint16_t)(at + i * 64 + lane);
          list_l[w][to] = (uint8_t)l;
        }
        n += __popcll(mask);
      }
    }
  };
  const auto count = [&]() {
    wave_sync();
    for (int i = lane; i < n; i += 64) atomicAdd(&cnt[w][list_l[w][i]], 1);
  };
  for (int j = lane; j < kBucket; j += 64) cnt[w][j] = 0;  // the wavefront's own
  bool listed = per <= 1 << 16;
  if (t0 < t1) {
    int id[kBatches], next[kBatches];
    load(next, t0);
    for (int t = t0; t < t1; t += kRead) {
#pragma unroll
      for (int i = 0; i < kBatches; ++i) id[i] = next[i];
      if (t + kRead < t1) load(next, t + kRead);
      if (n > kList - kRead) {
        count();
        wave_sync();
        listed = false;
        n = 0;
      }
      enlist(id, t - t0);
    }
    count();
  }
  if (lane == 0) less[w] = upto;
  __syncthreads();
  if (threadIdx.x < kBucket) {
    int sum = 0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
      const int c = cnt[i][threadIdx.x];
      cnt[i][threadIdx.x] = sum;  // tokens of this id in earlier wavefronts' runs
      sum += c;
    }
    tot[threadIdx.x] = sum;
  }
  __syncthreads();
  if (w == 0) {  // exclusive sums over the bucket's ids, four a lane
    int c[4], sum = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      c[i] = sum;
      sum += tot[lane * 4 + i];
    }
    int incl = sum;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int up = __shfl_up(incl, o);
      if (lane >= o) incl += up;
    }
    // where the bucket begins: the tokens of ids up to its last, without its own
    const int first = wave_isum(lane < kWaves ? less[lane] : 0) - __shfl(incl, 63);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int b = first + incl - sum + c[i];
      base[lane * 4 + i] = b;
      if (lane * 4 + i < n_ids) s.begin[lo + lane * 4 + i] = b;
    }
    if ((int)blockIdx.x == buckets - 1 && lane == 63) s.begin[V] = first + incl;
  }
  __syncthreads();
  const auto place = [&](int t) {  // t: the token that the list counts from
    wave_sync();
    for (int i = 0; i < n; i += 64) {
      const bool in = i + lane < n;
      const int l = in ? list_l[w][i + lane] : 0;
      uint64_t same = __ballot(in);
#pragma unroll
      for (int b = 0; b < 8; ++b) {  // lanes whose id is this lane's
        const uint64_t has = __ballot(in && ((l >> b) & 1));
        same &= (l >> b) & 1 ? has : ~has;
      }
      if (in) {
        const int to = base[l] + cnt[w][l] + __popcll(same & ((1ull << lane) - 1));
        s.pos[to] = t + list_t[w][i + lane];
        s.id[to] = lo + l;
      }
      wave_sync();
      if (in && (same >> lane) == 1) cnt[w][l] += __popcll(same);  // the last of them
      wave_sync();
    }
  };
  if (listed) {
    place(t0);
  } else {
    for (int t = t0; t < t1; t += kRead) {
      int id[kBatches];
      load(id, t);
      n = 0;
      enlist(id, 0);
      place(t);
    }
  }
}

// part: [ranges][2][dp]: of a row that began in an earlier range, and of one that
// goes on in the next.
template <typename TY, int KIND, bool ACC>
__global__ __launch_bounds__(256) void k_embed_sum(float* __restrict__ grad,
                                                   float* __restrict__ part,
                                                   const TY* __restrict__ dy, Sorted s, int T, int V,
                                                   int d, int dp, float scale, int tiles,
                                                   int ranges) {
  constexpr int VEC = 4;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int unit = blockIdx.x * 4 + w;
  const int r = unit / tiles, tile = unit - r * tiles, c = tile * 64 * VEC + lane * VEC;
  if (r >= ranges) return;
  const int k0 = r * kRange;
  const bool here = c < d;
  // lane i: token i of the range, lane kRange the first of the next one; read before the
  // number of sorted tokens is known (what lies behind them is not used)
  int my_pos = 0, my_id = -1;
  if (lane < kRange && k0 + lane < T) my_pos = s.pos[k0 + lane];
  if (lane <= kRange && k0 + lane < T) my_id = s.id[k0 + lane];
  const int before = k0 > 0 ? s.id[k0 - 1] : -1;
  const int n = s.begin[V], cnt = min(kRange, n - k0);
  if (cnt <= 0) {
    if (lane == 0 && tile == 0) s.goes_on[r] = make_int2(-1, 0);
    return;
  }
  if (k0 + lane >= n) my_id = -1;
  // where an id's tokens end, the last token of the range included
  const int next_id = __shfl_down(my_id, 1);  // by all lanes, before any branch
  const uint64_t ends = __ballot(lane < cnt && (lane == cnt - 1 || my_id != next_id));
  const int first_end = __builtin_ctzll(ends);
  const bool opened = before == __builtin_amdgcn_readlane(my_id, 0);
  const bool goes_on = __builtin_amdgcn_readlane(my_id, cnt) ==
                       __builtin_amdgcn_readlane(my_id, cnt - 1);
  // the row that begins here and goes on, and where its tokens end: used behind the sums
  const bool begins = goes_on && !(opened && first_end == cnt - 1);
  const int on = begins ? __builtin_amdgcn_readlane(my_id, cnt - 1) : -1;
  const int on_end = s.begin[on + 1];
  float acc[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) acc[e] = 0.f;
  // Every load before any store, and waited for together: the compiler cannot count past the
  // stores, whose branches are taken or not, and would wait for each of them.
  constexpr int U = 8;
  const int col = here ? c : 0;
  for (int k = 0; k < cnt; k += U) {
    Vec<TY, VEC> v[U];
    Vec<float, VEC> was[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = min(k + u, cnt - 1);
      v[u].template load_row<KIND>(dy + (size_t)__builtin_amdgcn_readlane(my_pos, i) * d, col, d);
      if constexpr (ACC) {
        was[u].zero();
        if ((ends >> i) & 1)
          was[u].template load_row<KIND>(grad + (size_t)__builtin_amdgcn_readlane(my_id, i) * d, col,
                                        d);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      v[u].arrive();
      if constexpr (ACC) was[u].arrive();
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = k + u;
      if (i < cnt) {
        v[u].template settle<KIND>(c, d);
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[e] += v[u].get(e);
        if ((ends >> i) & 1) {
          const bool head = i == first_end && opened, tail = i == cnt - 1 && goes_on;
          if (here) {
            if (head || tail) {
              Vec<float, VEC>::store(part + ((size_t)r * 2 + !head) * dp + c, acc);
            } else {
              float o[VEC];
              if constexpr (ACC) was[u].template settle<KIND>(c, d);
#pragma unroll
              for (int e = 0; e < VEC; ++e) o[e] = (ACC ? was[u].get(e) : 0.f) + acc[e] * scale;
              Vec<float, VEC>::template store_row<KIND>(
                  grad + (size_t)__builtin_amdgcn_readlane(my_id, i) * d, c, d, o);
            }
          }
#pragma unroll
          for (int e = 0; e < VEC; ++e) acc[e] = 0.f;
        }
      }
    }
  }
  if (lane == 0 && tile == 0)
    s.goes_on[r] = make_int2(on, begins ? (on_end - 1) / kRange - r + 1 : 0);
}

// grad's row `id`, columns from c on, is (what was there +) scale * sum
template <int VEC, int KIND, bool ACC>
__device__ __forceinline__ void put_row(float* __restrict__ grad, int id, int c, int d, float scale,
                                        Vec<float, VEC> was, const float (&sum)[VEC]) {
  was.template settle<KIND>(c, d);
  float o[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) o[e] = ACC ? was.get(e) + sum[e] * scale : sum[e] * scale;
  Vec<float, VEC>::template store_row<KIND>(grad + (size_t)id * d, c, d, o);
}

// A workgroup has kJoinWaves ranges and a column tile: a wavefront the row that begins
// in its range and goes on, where that is a row of few ranges (most are: about every
// other range ends inside a row); then, together, those of many, each wavefront a run
// of consecutive ranges and the wavefronts' sums in order.
template <int KIND, bool ACC>
__global__ __launch_bounds__(kJoinWaves * 64) void k_embed_join(float* __restrict__ grad,
                                                                const float* __restrict__ part,
                                                                const int2* __restrict__ goes_on,
                                                                int ranges, int d, int dp,
                                                                float scale) {
  constexpr int VEC = 4, kFew = 8;
  __shared__ __align__(16) float sh[kJoinWaves][64 * VEC];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, r0 = blockIdx.x * kJoinWaves;
  const int c = blockIdx.y * 64 * VEC + lane * VEC;
  int2 mine = make_int2(-1, 0);
  if (lane < kJoinWaves && r0 + lane < ranges) mine = goes_on[r0 + lane];
  uint64_t rows = __ballot(mine.y > kFew);  // the same in every wavefront
  Vec<float, VEC> was;
  was.zero();
  float acc[VEC];
  {
    const int id = __builtin_amdgcn_readlane(mine.x, w), n = __builtin_amdgcn_readlane(mine.y, w);
    if (id >= 0 && n <= kFew && c < d) {
      const float* p = part + (size_t)(r0 + w) * 2 * dp + c;
      Vec<float, VEC> v[kFew];
      if (ACC) was.template load_row<KIND>(grad + (size_t)id * d, c, d);
#pragma unroll
      for (int j = 0; j < kFew; ++j) {
        v[j].zero();
        if (j < n) v[j].load(p + ((size_t)j * 2 + (j == 0)) * dp);
      }
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        acc[e] = 0.f;
#pragma unroll
        for (int j = 0; j < kFew; ++j) acc[e] += v[j].get(e);
      }
      put_row<VEC, KIND, ACC>(grad, id, c, d, scale, was, acc);
    }
  }
  while (rows) {
    const int i = __builtin_ctzll(rows), r = r0 + i;
    rows &= rows - 1;
    const int id = __builtin_amdgcn_readlane(mine.x, i), n = __builtin_amdgcn_readlane(mine.y, i);
    const int per = (n + kJoinWaves - 1) / kJoinWaves;
    if (ACC && w == 0 && c < d) was.template load_row<KIND>(grad + (size_t)id * d, c, d);
#pragma unroll
    for (int e = 0; e < VEC; ++e) acc[e] = 0.f;
    if (c < d) {
#pragma unroll 8
      for (int j = w * per; j < min((w + 1) * per, n); ++j) {
        Vec<float, VEC> v;
        v.load(part + ((size_t)(r + j) * 2 + (j == 0)) * dp + c);
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[e] += v.get(e);
      }
    }
    __syncthreads();  // the sums of the row before have been read
    Vec<float, VEC>::store(&sh[w][lane * VEC], acc);
    __syncthreads();
    if (w == 0 && c < d) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        acc[e] = 0.f;
#pragma unroll
        for (int q = 0; q < kJoinWaves; ++q) acc[e] += sh[q][lane * VEC + e];
      }
      put_row<VEC, KIND, ACC>(grad, id, c, d, scale, was, acc);
    }
  }
}

int ranges_of(int T) { return (T - 1) / kRange + 1; }
size_t padded(int d) { return ((size_t)d + 3) / 4 * 4; }
size_t ints_of(int T, int V) {
  return ((size_t)2 * ranges_of(T) + 2 * (size_t)T + V + 1 + 3) / 4 * 4;
}

}  // namespace
}  // namespace skv

using namespace skv;

extern "C" int skv_embedding_fwd(void* out, const int32_t* ids, const void* table,
                                 const float* pos_table, int T, int V, int d, int n_pos,
                                 float scale, int table_dt, int out_dt, skv_stream_t stream) {
  SKV_REQUIRE(out && ids && table, SKV_E_INVALID, "skv_embedding_fwd: null pointer argument");
  SKV_REQUIRE(T > 0 && V > 0 && d > 0, SKV_E_INVALID, "skv_embedding_fwd: dims must be > 0");
  SKV_REQUIRE(d <= kMaxD && launchable(((size_t)T + 3) / 4, 256), SKV_E_UNSUPPORTED,
              "skv_embedding_fwd: T=%d, d=%d: up to 2^26 tokens and 2^22 columns", T, d);
  SKV_REQUIRE(!pos_table || n_pos > 0, SKV_E_INVALID, "skv_embedding_fwd: n_pos must be > 0");
  SKV_REQUIRE((table_dt == SKV_F32 || table_dt == SKV_BF16) &&
                  (out_dt == SKV_F32 || out_dt == SKV_BF16),
              SKV_E_INVALID, "skv_embedding_fwd: bad dtype");
  SKV_REQUIRE(aligned16(out) && aligned16(table) && aligned16(pos_table), SKV_E_INVALID,
              "skv_embedding_fwd: pointers must be 16-byte aligned");
  if (int rc = apart("skv_embedding_fwd",
                     {{out, (size_t)T * d * (out_dt == SKV_BF16 ? 2 : 4), "output"}},
                     {{table, (size_t)V * d * (table_dt == SKV_BF16 ? 2 : 4), "table"},
                      {ids, (size_t)T * 4, "tokens"},
                      {pos_table, (size_t)n_pos * d * 4, "pos_table"}}))
    return rc;
  const auto run = [&](auto* o, auto* t) {
    using TO = std::remove_pointer_t<decltype(o)>;
    using TT = std::remove_const_t<std::remove_pointer_t<decltype(t)>>;
    constexpr int VEC = sizeof(TT) == 2 && sizeof(TO) == 2 ? 8 : 4;
    const auto rows = [&](auto LPT, auto KIND) {
      constexpr unsigned tokens = 256 / LPT.value;
      k_embed_rows<TT, TO, VEC, LPT.value, KIND.value>
          <<<((unsigned)T + tokens - 1) / tokens, 256, 0, (hipStream_t)stream>>>(
              o, ids, t, pos_table, T, V, d, n_pos, scale);
    };
    using std::integral_constant;
    const RowKind kind = row_kind(d, VEC);
    const auto with_kind = [&](auto LPT) {
      if (kind == kEven) rows(LPT, integral_constant<int, kEven>{});
      else rows(LPT, integral_constant<int, kOdd>{});
    };
    if (kind == kTiny) rows(integral_constant<int, 16>{}, integral_constant<int, kTiny>{});
    else if (d <= 32 * VEC) with_kind(integral_constant<int, 16>{});
    else with_kind(integral_constant<int, 64>{});
  };
  if (table_dt == SKV_BF16) {
    if (out_dt == SKV_BF16) run((uint16_t*)out, (const uint16_t*)table);
    else run((float*)out, (const uint16_t*)table);
  } else {
    if (out_dt == SKV_BF16) run((uint16_t*)out, (const float*)table);
    else run((float*)out, (const float*)table);
  }
  return check_launch("skv_embedding_fwd");
}

extern "C" size_t skv_embedding_bwd_workspace_bytes(int T, int V, int d) {
  if (T <= 0 || V <= 0 || d <= 0) return 0;
  return ints_of(T, V) * sizeof(int32_t) + (size_t)ranges_of(T) * 2 * padded(d) * sizeof(float);
}

extern "C" int skv_embedding_bwd(float* grad, const void* dout, const int32_t* ids, int T, int V,
                                 int d, float scale, int accumulate, void* ws, size_t ws_bytes,
                                 int dt, skv_stream_t stream) {
  SKV_REQUIRE(grad && dout && ids && ws, SKV_E_INVALID, "skv_embedding_bwd: null pointer argument");
  SKV_REQUIRE(T > 0 && V > 0 && d > 0, SKV_E_INVALID, "skv_embedding_bwd: dims must be > 0");
  SKV_REQUIRE(dt == SKV_F32 || dt == SKV_BF16, SKV_E_INVALID, "skv_embedding_bwd: bad dtype");
  const int width = V <= 256 * kBucket ? (V + 255) / 256 : kBucket;  // one bucket to a CU
  const int buckets = (V - 1) / width + 1, tiles = (d - 1) / 256 + 1;
  const size_t units = (size_t)ranges_of(T) * tiles;
  SKV_REQUIRE(d <= kMaxD && T <= kMaxRows && launchable((size_t)buckets + kZeroGroups, 1024) &&
                  launchable((units + 3) / 4, 256) &&
                  launchable((units + kJoinWaves - 1) / kJoinWaves, kJoinWaves * 64),
              SKV_E_UNSUPPORTED,
              "skv_embedding_bwd: T=%d, V=%d, d=%d are too many for a launch (up to 2^22 columns, "
              "2^29 table rows, nearly 2^30 tokens a 256 columns)", T, V, d);
  SKV_REQUIRE(aligned16(grad) && aligned16(dout) && aligned16(ws), SKV_E_INVALID,
              "skv_embedding_bwd: pointers must be 16-byte aligned");
  SKV_REQUIRE(ws_bytes >= skv_embedding_bwd_workspace_bytes(T, V, d), SKV_E_WORKSPACE,
              "skv_embedding_bwd: workspace of %zu bytes, %zu needed", ws_bytes,
              skv_embedding_bwd_workspace_bytes(T, V, d));
  if (int rc = apart("skv_embedding_bwd",
                     {{grad, (size_t)V * d * 4, "grad_table"}, {ws, ws_bytes, "the workspace"}},
                     {{dout, (size_t)T * d * (dt == SKV_BF16 ? 2 : 4), "grad_output"},
                      {ids, (size_t)T * 4, "tokens"}}))
    return rc;
  hipStream_t st = (hipStream_t)stream;
  Sorted s;
  const int ranges = ranges_of(T), dp = padded(d);
  s.goes_on = (int2*)ws;
  s.pos = (int32_t*)(s.goes_on + ranges);
  s.id = s.pos + T;
  s.begin = s.id + T;
  float* part = (float*)((int32_t*)ws + ints_of(T, V));
  const size_t n_zero = accumulate ? 0 : (size_t)V * d;
  const int sort_grid = buckets + (n_zero ? kZeroGroups : 0);
  k_embed_sort<<<sort_grid, kWaves * 64, 0, st>>>(s, ids, T, V, width, buckets, grad, n_zero);
  if (int rc = check_launch("skv_embedding_bwd")) return rc;
  const unsigned grid = (unsigned)((units + 3) / 4);
  const dim3 join((ranges + kJoinWaves - 1) / kJoinWaves, tiles);
  const auto run = [&](auto* y, auto KIND, auto ACC) {
    using TY = std::remove_const_t<std::remove_pointer_t<decltype(y)>>;
    k_embed_sum<TY, KIND.value, ACC.value><<<grid, 256, 0, st>>>(grad, part, y, s, T, V, d, dp, scale,
                                                                tiles, ranges);
    k_embed_join<KIND.value, ACC.value><<<join, kJoinWaves * 64, 0, st>>>(grad, part, s.goes_on,
                                                                         ranges, d, dp, scale);
  };
  const auto with = [&](auto* y) {
    const auto kind = [&](auto KIND) {
      if (accumulate) run(y, KIND, std::true_type{});
      else run(y, KIND, std::false_type{});
    };
    const RowKind k = row_kind(d, 4);
    if (k == kEven) kind(std::integral_constant<int, kEven>{});
    else if (k == kOdd) kind(std::integral_constant<int, kOdd>{});
    else kind(std::integral_constant<int, kTiny>{});
  };
  if (dt == SKV_BF16) with((const uint16_t*)dout);
  else with((const float*)dout);
  return check_launch("skv_embedding_bwd");
}
