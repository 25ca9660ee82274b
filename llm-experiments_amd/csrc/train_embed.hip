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
//         in one scan over the ids, and places the tokens in a second; the ids
//         come from L2 after the first workgroup's read. It also writes the zero
//         rows of ids without tokens, which are most of a large table and most of
//         what this operator writes, while the scans wait on loads.
//   sum   a wavefront has 64 columns' vectors and a range of kRange sorted tokens,
//         whatever their ids: the work is even however unevenly the ids occur. A
//         row whose tokens all lie in the range is written; one that crosses a
//         range's border leaves its part.
//   join  adds the parts of each such row, in order.
#include "train_common.h"

namespace skv {
namespace {

using namespace train;

constexpr int kBucket = 256;  // ids of a bucket, at most
constexpr int kWaves = 16;    // wavefronts of a sorting workgroup
constexpr int kRange = 32;    // sorted tokens of a summing wavefront
constexpr int kJoinWaves = 8;

// ---------------------------------------------------------------------------
// lookup
// ---------------------------------------------------------------------------

// A workgroup's four wavefronts have a token each; VEC columns a lane and step.
template <typename TT, typename TO, int VEC>
__global__ __launch_bounds__(256) void k_embed_rows(TO* __restrict__ out,
                                                    const int32_t* __restrict__ ids,
                                                    const TT* __restrict__ table,
                                                    const float* __restrict__ pos, int T, int V,
                                                    int d, int n_pos, float scale) {
  const int i = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (i >= T) return;
  const int id = ids[i];
  const bool real = (unsigned)id < (unsigned)V;
  const TT* row = table + (size_t)(real ? id : 0) * d;
  const float* pr = pos ? pos + (size_t)(i % n_pos) * d : nullptr;
  TO* o = out + (size_t)i * d;
#pragma unroll 4
  for (int j = lane * VEC; j < d; j += 64 * VEC) {
    Vec<TT, VEC> t;
    Vec<float, VEC> p;
    t.zero();
    p.zero();
    if (real) t.load(row + j);
    if (pr) p.load(pr + j);
    float r[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) r[e] = t.get(e) * scale + p.get(e);
    Vec<TO, VEC>::store(o + j, r);
  }
}

// ---------------------------------------------------------------------------
// gradient: the tokens sorted by id
// ---------------------------------------------------------------------------

struct Sorted {
  int32_t* pos;    // [T] tokens in order of their ids
  int32_t* id;     // [T] their ids
  int32_t* begin;  // [V + 1] where an id's tokens begin
};

__device__ __forceinline__ int wave_isum(int x) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) x += __shfl_xor(x, o);
  return x;
}

// width: ids of a bucket. Each wavefront has a run of consecutive tokens in both
// scans; an id's tokens are placed by wavefront, then by token.
__global__ __launch_bounds__(kWaves * 64) void k_embed_sort(Sorted s,
                                                            const int32_t* __restrict__ ids,
                                                            float* __restrict__ grad, int T, int V,
                                                            int d, int width, int fill_zero) {
  __shared__ int cnt[kWaves][kBucket];
  __shared__ int tot[kBucket];   // tokens of an id
  __shared__ int base[kBucket];  // where they begin in the bucket
  __shared__ int less[kWaves];
  const int w = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int lo = blockIdx.x * width, n_ids = min(width, V - lo);
  for (int j = threadIdx.x; j < kWaves * kBucket; j += kWaves * 64) cnt[j / kBucket][j % kBucket] = 0;
  __syncthreads();
  const int per = ((T + kWaves * 64 - 1) / (kWaves * 64)) * 64;
  const int t0 = min(w * per, T), t1 = min(t0 + per, T);
  int below = 0;
#pragma unroll 8
  for (int t = t0 + lane; t < t1; t += 64) {
    const int id = ids[t], l = id - lo;
    below += id >= 0 && l < 0;
    if ((unsigned)l < (unsigned)n_ids) atomicAdd(&cnt[w][l], 1);
  }
  below = wave_isum(below);
  if (lane == 0) less[w] = below;
  __syncthreads();
  if (threadIdx.x < kBucket) {
    int sum = 0;
    for (int i = 0; i < kWaves; ++i) {
      const int c = cnt[i][threadIdx.x];
      cnt[i][threadIdx.x] = sum;  // tokens of this id in earlier wavefronts' runs
      sum += c;
    }
    tot[threadIdx.x] = sum;
  }
  __syncthreads();
  int first = 0;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) first += less[i];
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
#pragma unroll
    for (int i = 0; i < 4; ++i) base[lane * 4 + i] = first + incl - sum + c[i];
    if (blockIdx.x == gridDim.x - 1 && lane == 63) s.begin[V] = first + incl;
  }
  __syncthreads();
  for (int j = threadIdx.x; j < n_ids; j += kWaves * 64) s.begin[lo + j] = base[j];
  for (int j = threadIdx.x; j < kWaves * kBucket; j += kWaves * 64)
    cnt[j / kBucket][j % kBucket] += base[j % kBucket];
  __syncthreads();
  for (int t = t0; t < t1; t += 64) {
    const int id = t + lane < t1 ? ids[t + lane] : -1, l = id - lo;
    const bool in = id >= 0 && (unsigned)l < (unsigned)n_ids;
    uint64_t same = __ballot(in);
    if (!same) continue;
#pragma unroll
    for (int b = 0; b < 8; ++b) {  // lanes whose id is this lane's
      const uint64_t has = __ballot(in && ((l >> b) & 1));
      same &= (l >> b) & 1 ? has : ~has;
    }
    if (in) {
      const int at = cnt[w][l] + __popcll(same & ((1ull << lane) - 1));
      s.pos[at] = t + lane;
      s.id[at] = id;
    }
    __builtin_amdgcn_wave_barrier();
    if (in && (same >> lane) == 1) cnt[w][l] += __popcll(same);  // the last of them
    __builtin_amdgcn_wave_barrier();
  }
  if (fill_zero) {
    for (int j = w; j < n_ids; j += kWaves) {
      if (tot[j]) continue;
      float* g = grad + (size_t)(lo + j) * d;
      if (d % 4 == 0) {
        for (int c = lane * 4; c < d; c += 256)
          *reinterpret_cast<f32x4_t*>(g + c) = f32x4_t{0.f, 0.f, 0.f, 0.f};
      } else {
        for (int c = lane; c < d; c += 64) g[c] = 0.f;
      }
    }
  }
}

// part: [ranges][2][dp]: of a row that began in an earlier range, and of one that
// goes on in the next.
template <typename T, int VEC, bool ACC>
__global__ __launch_bounds__(256) void k_embed_sum(float* __restrict__ grad,
                                                   float* __restrict__ part,
                                                   const T* __restrict__ dy, Sorted s, int V, int d,
                                                   int dp, float scale, int tiles) {
  const int lane = threadIdx.x & 63;
  const int unit = blockIdx.x * 4 + (threadIdx.x >> 6);
  const int r = unit / tiles, c = (unit - r * tiles) * 64 * VEC + lane * VEC;
  const int n = s.begin[V], k0 = r * kRange, cnt = min(kRange, n - k0);
  if (cnt <= 0) return;
  const bool here = c < d;
  // lane i: token i of the range, lane kRange the first of the next one
  int my_pos = 0, my_id = -1;
  if (lane < cnt) my_pos = s.pos[k0 + lane];
  if (lane <= cnt && k0 + lane < n) my_id = s.id[k0 + lane];
  const int before = k0 > 0 ? s.id[k0 - 1] : -1;
  // where an id's tokens end, the last token of the range included
  const int next_id = __shfl_down(my_id, 1);  // by all lanes, before any branch
  const uint64_t ends = __ballot(lane < cnt && (lane == cnt - 1 || my_id != next_id));
  const int first_end = __builtin_ctzll(ends);
  const bool opened = before == __builtin_amdgcn_readlane(my_id, 0);
  const bool goes_on = __builtin_amdgcn_readlane(my_id, cnt) ==
                       __builtin_amdgcn_readlane(my_id, cnt - 1);
  float acc[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) acc[e] = 0.f;
  constexpr int U = 8;
  for (int k = 0; k < cnt; k += U) {
    Vec<T, VEC> v[U];
    Vec<float, VEC> was[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = min(k + u, cnt - 1);
      const int p = __builtin_amdgcn_readlane(my_pos, i);
      v[u].zero();
      was[u].zero();
      if (here && k + u < cnt) {
        v[u].load(dy + (size_t)p * d + c);
        if (ACC && ((ends >> i) & 1))
          was[u].load(grad + (size_t)__builtin_amdgcn_readlane(my_id, i) * d + c);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = k + u;
      if (i < cnt) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[e] += v[u].get(e);
        if ((ends >> i) & 1) {
          const bool head = i == first_end && opened, tail = i == cnt - 1 && goes_on;
          if (here) {
            if (head || tail) {
              Vec<float, VEC>::store(part + ((size_t)r * 2 + !head) * dp + c, acc);
            } else {
              float o[VEC];
#pragma unroll
              for (int e = 0; e < VEC; ++e) o[e] = was[u].get(e) + acc[e] * scale;
              Vec<float, VEC>::store(
                  grad + (size_t)__builtin_amdgcn_readlane(my_id, i) * d + c, o);
            }
          }
#pragma unroll
          for (int e = 0; e < VEC; ++e) acc[e] = 0.f;
        }
      }
    }
  }
}

// One workgroup a range and column tile; those whose last row goes on in the
// next range, and began in this one, add up its parts: each wavefront a run of
// consecutive ranges, then the wavefronts' sums in order.
template <int VEC>
__global__ __launch_bounds__(kJoinWaves * 64) void k_embed_join(float* __restrict__ grad,
                                                                const float* __restrict__ part,
                                                                Sorted s, int V, int d, int dp,
                                                                float scale, int accumulate) {
  __shared__ float sh[kJoinWaves][64 * VEC];
  const int r = blockIdx.x, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int k1 = (r + 1) * kRange;
  if (k1 >= s.begin[V]) return;
  const int id = s.id[k1 - 1];
  if (s.id[k1] != id) return;
  const int b = s.begin[id], e1 = s.begin[id + 1];
  if (b < k1 - kRange) return;  // an earlier range's
  const int last = (e1 - 1) / kRange, n = last - r + 1;  // ranges of this row
  const int per = (n + kJoinWaves - 1) / kJoinWaves;
  const int c = blockIdx.y * 64 * VEC + lane * VEC;
  float acc[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) acc[e] = 0.f;
  if (c < d) {
#pragma unroll 8
    for (int i = w * per; i < min((w + 1) * per, n); ++i) {
      Vec<float, VEC> v;
      v.load(part + ((size_t)(r + i) * 2 + (i == 0)) * dp + c);
#pragma unroll
      for (int e = 0; e < VEC; ++e) acc[e] += v.get(e);
    }
  }
  Vec<float, VEC>::store(&sh[w][lane * VEC], acc);
  __syncthreads();
  if (w == 0 && c < d) {
    float* g = grad + (size_t)id * d + c;
    Vec<float, VEC> was;
    was.zero();
    if (accumulate) was.load(g);
    float o[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      float t = 0.f;
#pragma unroll
      for (int i = 0; i < kJoinWaves; ++i) t += sh[i][lane * VEC + e];
      o[e] = was.get(e) + t * scale;
    }
    Vec<float, VEC>::store(g, o);
  }
}

int ranges_of(int T) { return (T + kRange - 1) / kRange; }
int padded(int d) { return (d + 3) / 4 * 4; }
size_t ints_of(int T, int V) { return ((size_t)2 * T + V + 1 + 3) / 4 * 4; }

}  // namespace
}  // namespace skv

using namespace skv;

extern "C" int skv_embedding_fwd(void* out, const int32_t* ids, const void* table,
                                 const float* pos_table, int T, int V, int d, int n_pos,
                                 float scale, int table_dt, int out_dt, skv_stream_t stream) {
  SKV_REQUIRE(out && ids && table, SKV_E_INVALID, "skv_embedding_fwd: null pointer argument");
  SKV_REQUIRE(T > 0 && V > 0 && d > 0, SKV_E_INVALID, "skv_embedding_fwd: dims must be > 0");
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
  const dim3 grid((T + 3) / 4);
  const auto run = [&](auto* o, auto* t) {
    using TO = std::remove_pointer_t<decltype(o)>;
    using TT = std::remove_const_t<std::remove_pointer_t<decltype(t)>>;
    const auto rows = [&](auto VEC) {
      k_embed_rows<TT, TO, VEC.value><<<grid, 256, 0, (hipStream_t)stream>>>(
          o, ids, t, pos_table, T, V, d, n_pos, scale);
    };
    if (table_dt == SKV_BF16 && out_dt == SKV_BF16 && d % 8 == 0)
      rows(std::integral_constant<int, 8>{});
    else if (d % 4 == 0) rows(std::integral_constant<int, 4>{});
    else if (d % 2 == 0) rows(std::integral_constant<int, 2>{});
    else rows(std::integral_constant<int, 1>{});
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
  SKV_REQUIRE(T <= 1 << 30 && V <= 1 << 30, SKV_E_UNSUPPORTED,
              "skv_embedding_bwd: up to 2^30 tokens and table rows");
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
  s.pos = (int32_t*)ws;
  s.id = s.pos + T;
  s.begin = s.id + T;
  float* part = (float*)((int32_t*)ws + ints_of(T, V));
  const int dp = padded(d);
  // about two buckets to a CU, so that the zero rows are written by all of them
  int width = (V + 511) / 512;
  width = width < 16 ? 16 : width > kBucket ? kBucket : width;
  k_embed_sort<<<(V + width - 1) / width, kWaves * 64, 0, st>>>(s, ids, grad, T, V, d, width,
                                                                !accumulate);
  if (int rc = check_launch("skv_embedding_bwd")) return rc;
  const int ranges = ranges_of(T);
  const auto run = [&](auto* y, auto VEC) {
    using TY = std::remove_const_t<std::remove_pointer_t<decltype(y)>>;
    const int tiles = (d + 64 * VEC.value - 1) / (64 * VEC.value);
    const size_t units = (size_t)ranges * tiles;
    const unsigned grid = (unsigned)((units + 3) / 4);
    if (accumulate)
      k_embed_sum<TY, VEC.value, true><<<grid, 256, 0, st>>>(grad, part, y, s, V, d, dp, scale,
                                                             tiles);
    else
      k_embed_sum<TY, VEC.value, false><<<grid, 256, 0, st>>>(grad, part, y, s, V, d, dp, scale,
                                                              tiles);
    if (ranges > 1)
      k_embed_join<VEC.value><<<dim3(ranges - 1, tiles), kJoinWaves * 64, 0, st>>>(
          grad, part, s, V, d, dp, scale, accumulate);
  };
  const auto with = [&](auto* y) {
    if (d % 4 == 0) run(y, std::integral_constant<int, 4>{});
    else if (d % 2 == 0) run(y, std::integral_constant<int, 2>{});
    else run(y, std::integral_constant<int, 1>{});
  };
  if (dt == SKV_BF16) with((const uint16_t*)dout);
  else with((const float*)dout);
  return check_launch("skv_embedding_bwd");
}
