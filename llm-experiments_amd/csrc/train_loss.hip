// Cross-entropy over a vocabulary and its gradient.
//
//   row[m] = logsumexp(x[m]) - x[m][t], loss = mean of the rows that count
//   dx[m]  = (softmax(x[m]) - onehot(t)) grad_scale / rows that count
//
// A row counts if its target t lies in [0, V); the others get a loss and a
// gradient of 0, and their logits are not read. Bound by HBM: a row is read once
// into the registers of its workgroup, which takes the maximum, the sum of
// exponentials and then writes the gradient from them (each exponential is
// computed twice, which is cheaper than the registers to keep it in). Rows of more
// than 16384 vectors (131072 logits in bf16, 65536 in fp32) are read a second time.
//
// Rows of any length start anywhere: a lane's vectors are the aligned ones inside the
// row, and the up to 63 + 7 elements before and after them are one element each of the
// first lanes.
#include "train_common.h"

namespace skv {
namespace {

using namespace train;

template <typename T>
constexpr int kVec = 16 / (int)sizeof(T);

// ws: the count of rows, then the rows' losses
struct LossArgs {
  const void* x;
  void* dx;
  const int32_t* targets;
  float* row;  // [M]
  const float* inv;  // grad_scale / rows that count, or NULL: every wavefront counts them
  float grad_scale;
  int M, V;
};

// Where the wavefronts count the rows themselves: one launch less (255 x 257 fp32: two
// launches of 2 us instead of three), and at most 4 MB more from L2.
constexpr int kCountRows = 1024;

// A gradient that the 256 MB of the last-level cache do not hold goes past the caches, and
// so do its logits (PAST: the nt bit): 8192 x 50304 bf16, 290 us without, 265 with; and with
// the three products around the loss, 4096 x 50304: 1201 and 1166 us. One that fits is
// there for the products that read it: 16384 x 5000 with them, 455 us kept and 474 past.
constexpr size_t kCached = 256u << 20;

__device__ __forceinline__ float row_scale(const LossArgs& a) {
  if (a.inv) return *a.inv;
  int n = 0;
#pragma unroll 4
  for (int i = threadIdx.x & 63; i < a.M; i += 64) n += (unsigned)a.targets[i] < (unsigned)a.V;
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) n += __shfl_xor(n, o);
  return a.grad_scale / (float)max(n, 1);
}

// e^(x - from). The difference comes first: with finite logits of any size it is 0 at x =
// from and overflows to -inf only. (The product with log2(e) first, one operation less,
// leaves up to 2^-25 of itself where it is rounded, which 2^x cannot take from 3e9 on, and
// gains nothing: 8192 x 50304 bf16 267.3 us, 267.8 so.)
__device__ __forceinline__ float exp_from(float x, float from) {
  return fast_exp2((x - from) * LOG2E);
}

// A maximum and the sum of e^(x - ref) of what a wavefront has seen. ref is top, or 0
// where top is -inf (nothing seen, or only NaN).
struct Stats {
  float top, sum;
};
__device__ __forceinline__ float ref_of(float top) { return top == -INFINITY ? 0.f : top; }

// The statistics of the workgroup's NW wavefronts: one barrier, and then a lane has
// those of wavefront lane % NW (so a row of 16 lanes has each 16 / NW times).
template <int NW>
__device__ __forceinline__ Stats group_stats(Stats s, float2* sh) {
  if constexpr (NW > 1) {
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = make_float2(s.top, s.sum);
    __syncthreads();
    const float2 o = sh[threadIdx.x % NW];
    s.top = row16_max(o.x);
    // a NaN sum stays one under a factor of 0
    const float f = o.x == -INFINITY ? 0.f : exp_from(o.x, s.top);
    s.sum = row16_sum(o.y * f) * (NW / 16.f);
  }
  return s;
}

// WIDE: on several wavefronts, whose vectors then begin on a cache line, so that no line is
// in two wavefronts' loads and stores: 8192 x 50257 bf16, 295 us from a 16-byte granule, 278
// from a line. Lines are counted from the first row, not from address 0: which elements are
// summed together, and so the result's bits, depend on sizes alone. (Where the logits
// themselves begin inside a line, the vectors do too.)
template <typename T, bool WIDE>
struct Row {
  static constexpr int kLine = WIDE ? 128 : 16;  // bytes
  static constexpr int kHead = WIDE ? 64 : 8;    // lanes for the elements before the vectors
  const T* x;   // the row
  int head;     // elements before its first vector
  int n_vec;    // whole vectors from there
  int tail_at;  // the first element behind them
  __device__ __forceinline__ Row(const T* base, int m, int V) {
    x = base + (size_t)m * V;
    const size_t from = WIDE ? (size_t)m * V * sizeof(T) : reinterpret_cast<uintptr_t>(x);
    const int off = (int)((from & (kLine - 1)) / sizeof(T));
    head = min(off ? kLine / (int)sizeof(T) - off : 0, V);
    n_vec = (V - head) / kVec<T>;
    tail_at = head + n_vec * kVec<T>;
  }
  // vector j of a row that begins at p (its own or the gradient's): the offset in bytes
  // fits 32 bits, so that a lane keeps one register for its address
  __device__ __forceinline__ const T* vec(const T* p, unsigned j) const {
    return reinterpret_cast<const T*>(reinterpret_cast<const char*>(p + head) + j * 16u);
  }
  __device__ __forceinline__ T* vec(T* p, unsigned j) const {
    return reinterpret_cast<T*>(reinterpret_cast<char*>(p + head) + j * 16u);
  }
  // the single element of thread t, or -1
  __device__ __forceinline__ int edge(int t, int V) const {
    if (t < head) return t;
    t -= kHead;
    return t >= 0 && t < V - tail_at ? tail_at + t : -1;
  }
};

__device__ __forceinline__ float as_f32(float x) { return x; }
__device__ __forceinline__ float as_f32(uint16_t x) { return bf16_to_f32(x); }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(uint16_t* p, float v) { *p = f32_to_bf16(v); }

// The vectors of a lane that every lane has: all but the last three of NV (a row of NV or
// NV - 1 vectors a lane has at most 9 fewer than its length allows).
constexpr int sure(int NV) { return NV > 3 ? NV - 3 : 0; }

// A row on NW wavefronts, NV vectors a lane, sure(NV) of them without a test for the
// row's end; with NW = 1 a workgroup has four.
template <typename T, int NW, int NV, bool GRAD, bool PAST>
__global__ __launch_bounds__(NW == 1 ? 256 : NW * 64) void k_loss_rows(LossArgs a) {
  __shared__ float2 sh[NW];
  constexpr int N = kVec<T>;
  const int t = NW == 1 ? threadIdx.x & 63 : threadIdx.x;
  const int m = NW == 1 ? blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)
                        : blockIdx.x;
  if (m >= a.M) return;
  const Row<T, (NW > 1)> row((const T*)a.x, m, a.V);
  T* dx = (T*)a.dx + (size_t)m * a.V;
  const int target = a.targets[m], at = row.edge(t, a.V);
  if ((unsigned)target >= (unsigned)a.V) {
    if (t == 0) a.row[m] = 0.f;
    if constexpr (GRAD) {
      const float z[N] = {};
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const unsigned j = i * NW * 64 + t;
        if (i < sure(NV) || j < (unsigned)row.n_vec) Vec<T, N>::store(row.vec(dx, j), z);
      }
      if (at >= 0) put(dx + at, 0.f);
    }
    return;
  }
  Vec<T, N> v[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const unsigned j = i * NW * 64 + t;
    if (i < sure(NV) || j < (unsigned)row.n_vec) {
      if constexpr (PAST) v[i].stream(row.vec(row.x, j));
      else v[i].load(row.vec(row.x, j));
    }
  }
  const float edge = at >= 0 ? as_f32(row.x[at]) : 0.f;
  const float picked = as_f32(row.x[target]);
  const float inv = GRAD ? row_scale(a) : 0.f;
  float top = at >= 0 ? edge : -INFINITY;
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (i < sure(NV) || i * NW * 64 + t < row.n_vec) {
#pragma unroll
      for (int e = 0; e < N; ++e) top = fmaxf(top, v[i].get(e));
    }
  top = wave_max(top);
  const float ref = ref_of(top);
  float sum = at >= 0 ? exp_from(edge, ref) : 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    v[i].keep();
    if (i < sure(NV) || i * NW * 64 + t < row.n_vec) {
#pragma unroll
      for (int e = 0; e < N; ++e) sum += exp_from(v[i].get(e), ref);
    }
  }
  const Stats s = group_stats<NW>({top, wave_sum(sum)}, sh);
  if (t == 0) a.row[m] = (s.top - picked) + logf(s.sum);  // NaN where all is -inf
  if constexpr (GRAD) {
    const float k = inv / s.sum;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      unsigned j = i * NW * 64 + t;
      asm volatile("" : "+v"(j));  // formed here, not kept since the loads
      v[i].keep();
      if (i < sure(NV) || j < (unsigned)row.n_vec) {
        const unsigned first = row.head + j * N;
        float o[N];
#pragma unroll
        for (int e = 0; e < N; ++e) o[e] = exp_from(v[i].get(e), s.top) * k;
        if ((unsigned)target - first < (unsigned)N) {
#pragma unroll
          for (int e = 0; e < N; ++e) o[e] -= first + e == (unsigned)target ? inv : 0.f;
        }
        if constexpr (PAST) Vec<T, N>::store_stream(row.vec(dx, j), o);
        else Vec<T, N>::store(row.vec(dx, j), o);
      }
    }
    if (at >= 0) put(dx + at, exp_from(edge, s.top) * k - (at == target ? inv : 0.f));
  }
}

// Any length: the row is read for its statistics and again for its gradient.
template <typename T, bool GRAD, bool PAST>
__global__ __launch_bounds__(1024) void k_loss_long(LossArgs a) {
  __shared__ float2 sh[16];
  constexpr int N = kVec<T>;
  const int t = threadIdx.x, m = blockIdx.x;
  const Row<T, true> row((const T*)a.x, m, a.V);
  T* dx = (T*)a.dx + (size_t)m * a.V;
  const int target = a.targets[m], at = row.edge(t, a.V);
  const bool counts = (unsigned)target < (unsigned)a.V;
  const float inv = GRAD && counts ? row_scale(a) : 0.f;
  const float edge = at >= 0 ? as_f32(row.x[at]) : 0.f;
  float whole = 0.f, k = 0.f;  // the row's maximum, the gradient's factor
  if (counts) {
    const float picked = as_f32(row.x[target]);
    // a lane's sum is taken on to a larger maximum where its vectors have one
    float top = at >= 0 ? edge : -INFINITY, ref = ref_of(top);
    float sum = at >= 0 ? exp_from(edge, ref) : 0.f;
#pragma unroll 4
    for (unsigned j = t; j < (unsigned)row.n_vec; j += 1024) {
      Vec<T, N> v;
      v.load(row.vec(row.x, j));
      float most = top;
#pragma unroll
      for (int e = 0; e < N; ++e) most = fmaxf(most, v.get(e));
      if (most > top) {
        sum *= top == -INFINITY ? 1.f : exp_from(top, most);
        top = ref = most;
      }
#pragma unroll
      for (int e = 0; e < N; ++e) sum += exp_from(v.get(e), ref);
    }
    const float wtop = wave_max(top);
    sum *= top == -INFINITY ? 1.f : exp_from(top, wtop);
    const Stats s = group_stats<16>({wtop, wave_sum(sum)}, sh);
    whole = s.top;
    if (t == 0) a.row[m] = (s.top - picked) + logf(s.sum);
    k = inv / s.sum;
  } else if (t == 0) {
    a.row[m] = 0.f;
  }
  if constexpr (GRAD) {
#pragma unroll 4
    for (unsigned j = t; j < (unsigned)row.n_vec; j += 1024) {
      const unsigned first = row.head + j * N;
      Vec<T, N> v;
      float o[N];
      v.load(row.vec(row.x, j));
#pragma unroll
      for (int e = 0; e < N; ++e)
        o[e] = counts ? exp_from(v.get(e), whole) * k - (first + e == (unsigned)target ? inv : 0.f) : 0.f;
      if constexpr (PAST) Vec<T, N>::store_stream(row.vec(dx, j), o);
      else Vec<T, N>::store(row.vec(dx, j), o);
    }
    if (at >= 0)
      put(dx + at, counts ? exp_from(edge, whole) * k - (at == target ? inv : 0.f) : 0.f);
  }
}

// out[0] = grad_scale / rows that count
__global__ __launch_bounds__(1024) void k_loss_count(float* __restrict__ out,
                                                     const int32_t* __restrict__ targets, int M,
                                                     int V, float grad_scale) {
  __shared__ int sh[16];
  int n = 0;
#pragma unroll 8
  for (int i = threadIdx.x; i < M; i += 1024) n += (unsigned)targets[i] < (unsigned)V;
  for (int o = 32; o >= 1; o >>= 1) n += __shfl_xor(n, o);
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = n;
  __syncthreads();
  if (threadIdx.x == 0) {
    n = 0;
    for (int i = 0; i < 16; ++i) n += sh[i];
    out[0] = grad_scale / (float)max(n, 1);
  }
}

// loss = mean of the rows' losses over those that count
__global__ __launch_bounds__(1024) void k_loss_mean(float* __restrict__ loss,
                                                    const float* __restrict__ row,
                                                    const int32_t* __restrict__ targets, int M,
                                                    int V) {
  __shared__ double sh[16];
  __shared__ int cnt[16];
  int n = 0;
  double s = 0.0;
#pragma unroll 8
  for (int i = threadIdx.x; i < M; i += 1024) {
    n += (unsigned)targets[i] < (unsigned)V;
    s += (double)row[i];
  }
  for (int o = 32; o >= 1; o >>= 1) {
    n += __shfl_xor(n, o);
    s += __shfl_xor(s, o);
  }
  if ((threadIdx.x & 63) == 0) {
    sh[threadIdx.x >> 6] = s;
    cnt[threadIdx.x >> 6] = n;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    n = 0;
    s = 0.0;
    for (int i = 0; i < 16; ++i) {
      n += cnt[i];
      s += sh[i];
    }
    loss[0] = (float)(s / (double)max(n, 1));
  }
}

// Wavefronts of a row by its vectors: one up to 4 vectors a lane (no barrier), then 4 and 8
// up to 8 and 16 up to 16, so that a CU's registers hold many rows in different phases
// (50304 bf16 logits x 8192: 16 wavefronts of 7 vectors 290 us, 8 of 13 295, before PAST).
int waves_of(int n) { return n <= 256 ? 1 : n <= 2048 ? 4 : n <= 4096 ? 8 : 16; }

template <typename T, bool GRAD, bool PAST>
void launch_rows(const LossArgs& a, hipStream_t s) {
  const int n = (a.V + kVec<T> - 1) / kVec<T>;
  const auto rows = [&](auto NW, auto NV) {
    constexpr int nw = NW.value;
    k_loss_rows<T, nw, NV.value, GRAD, PAST>
        <<<nw == 1 ? (a.M + 3) / 4 : a.M, nw == 1 ? 256 : nw * 64, 0, s>>>(a);
  };
  const auto with = [&](auto NW) {  // even numbers of vectors: 5 to 8 a lane, or 16
    const int nv = (n + NW.value * 64 - 1) / (NW.value * 64);
    if constexpr (NW.value == 16) {
      if (nv > 14) return rows(NW, std::integral_constant<int, 16>{});
      if (nv > 12) return rows(NW, std::integral_constant<int, 14>{});
      if (nv > 10) return rows(NW, std::integral_constant<int, 12>{});
      if (nv > 8) return rows(NW, std::integral_constant<int, 10>{});
    }
    if (nv > 6) rows(NW, std::integral_constant<int, 8>{});
    else rows(NW, std::integral_constant<int, 6>{});
  };
  using std::integral_constant;
  const int nw = waves_of(n);
  if (n <= 64) rows(integral_constant<int, 1>{}, integral_constant<int, 1>{});
  else if (n <= 128) rows(integral_constant<int, 1>{}, integral_constant<int, 2>{});
  else if (nw == 1) rows(integral_constant<int, 1>{}, integral_constant<int, 4>{});
  else if (n <= 512) rows(integral_constant<int, 4>{}, integral_constant<int, 2>{});
  else if (n <= 1024) rows(integral_constant<int, 4>{}, integral_constant<int, 4>{});
  else if (nw == 4) with(integral_constant<int, 4>{});
  else if (nw == 8) with(integral_constant<int, 8>{});
  else if (n <= 16384) with(integral_constant<int, 16>{});
  else k_loss_long<T, GRAD, PAST><<<a.M, 1024, 0, s>>>(a);
}

}  // namespace
}  // namespace skv

using namespace skv;

extern "C" size_t skv_cross_entropy_workspace_bytes(int M) {
  return M <= 0 ? 0 : 16 + (size_t)M * sizeof(float);
}

extern "C" int skv_cross_entropy(float* loss, float* row_loss, void* dx, const void* x,
                                 const int32_t* targets, int M, int V, float grad_scale, void* ws,
                                 size_t ws_bytes, int dt, skv_stream_t stream) {
  SKV_REQUIRE(loss && x && targets && ws, SKV_E_INVALID, "skv_cross_entropy: null pointer argument");
  SKV_REQUIRE(M > 0 && V > 0, SKV_E_INVALID, "skv_cross_entropy: dims must be > 0");
  SKV_REQUIRE(dt == SKV_F32 || dt == SKV_BF16, SKV_E_INVALID, "skv_cross_entropy: bad dtype");
  SKV_REQUIRE(V <= 1 << 28, SKV_E_UNSUPPORTED, "skv_cross_entropy: V=%d > 2^28", V);
  const int n_vec = (V - 1) / (dt == SKV_BF16 ? 8 : 4) + 1, waves = waves_of(n_vec);
  SKV_REQUIRE(waves == 1 ? launchable(((size_t)M + 3) / 4, 256) : launchable(M, waves * 64),
              SKV_E_UNSUPPORTED, "skv_cross_entropy: %d rows of %d are too many for a launch", M, V);
  SKV_REQUIRE(aligned16(dx) && aligned16(x) && aligned16(ws), SKV_E_INVALID,
              "skv_cross_entropy: pointers must be 16-byte aligned");
  SKV_REQUIRE(ws_bytes >= skv_cross_entropy_workspace_bytes(M), SKV_E_WORKSPACE,
              "skv_cross_entropy: workspace of %zu bytes, %zu needed", ws_bytes,
              skv_cross_entropy_workspace_bytes(M));
  const size_t n = (size_t)M * V * (dt == SKV_BF16 ? 2 : 4), row = (size_t)M * 4;
  if (int rc = apart("skv_cross_entropy",
                     {{dx, n, "grad_logits"}, {loss, 4, "loss"}, {row_loss, row, "row_losses"},
                      {ws, ws_bytes, "the workspace"}},
                     {{x, n, "logits", 0}, {targets, row, "targets"}}))
    return rc;
  hipStream_t s = (hipStream_t)stream;
  float* inv = (float*)ws;
  LossArgs a = {x, dx, targets, row_loss ? row_loss : inv + 4, M > kCountRows ? inv : nullptr,
                grad_scale, M, V};
  if (dx && a.inv) k_loss_count<<<1, 1024, 0, s>>>(inv, targets, M, V, grad_scale);
  const auto with = [&](auto* x) {
    using T = std::remove_pointer_t<decltype(x)>;
    if (!dx) launch_rows<T, false, false>(a, s);
    else if (n <= kCached) launch_rows<T, true, false>(a, s);
    else launch_rows<T, true, true>(a, s);
  };
  if (dt == SKV_BF16) with((uint16_t*)dx);
  else with((float*)dx);
  k_loss_mean<<<1, 1024, 0, s>>>(loss, a.row, targets, M, V);
  return check_launch("skv_cross_entropy");
}
