// Cross-entropy over a vocabulary and its gradient.
//
//   row[m] = logsumexp(x[m]) - x[m][t], loss = mean of the rows that count
//   dx[m]  = (softmax(x[m]) - onehot(t)) grad_scale / rows that count
//
// A row counts if its target t lies in [0, V); the others get a loss and a
// gradient of 0, and their logits are not read. Bound by HBM: a row is read once
// into the registers of its workgroup, which takes the maximum, the sum of
// exponentials and then writes the gradient from them (each exponential is
// computed twice, which is cheaper than the registers to keep it in). Rows
// longer than 65536 logits are read a second time.
//
// Rows of any length start anywhere in a 16-byte granule: a lane's vectors are
// the aligned ones inside the row, and the up to 7 + 7 elements before and after
// them are one element each of the first lanes.
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
  const float* inv;  // grad_scale / rows that count
  int M, V;
};

// Over the workgroup's NW wavefronts; sh [NW].
template <int NW>
__device__ __forceinline__ float group_max(float x, float* sh) {
  x = wave_max(x);
  if constexpr (NW > 1) {
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = x;
    __syncthreads();
    x = sh[0];
#pragma unroll
    for (int i = 1; i < NW; ++i) x = fmaxf(x, sh[i]);
  }
  return x;
}
template <int NW>
__device__ __forceinline__ float group_sum(float x, float* sh) {
  x = wave_sum(x);
  if constexpr (NW > 1) {
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = x;
    __syncthreads();
    x = 0.f;
#pragma unroll
    for (int i = 0; i < NW; ++i) x += sh[i];
  }
  return x;
}

// 2^(x log2(e) - top2), the difference rounded once
__device__ __forceinline__ float exp_from(float x, float top2) {
  return fast_exp2(fmaf(x, LOG2E, -top2));
}

// top + log of the sum of exp(x - top) - picked, from the sum over exp_from: top2
// is top log2(e) rounded, and what the rounding left is taken out again.
__device__ __forceinline__ float loss_of(float top, float top2, float sum, float picked) {
  return (top - picked) + (logf(sum) - fmaf(top, LOG2E, -top2) * LN2);
}

template <typename T>
struct Row {
  const T* x;   // the row
  int head;     // elements before its first aligned vector
  int n_vec;    // aligned vectors
  int tail_at;  // the first element behind them
  __device__ __forceinline__ Row(const T* base, int m, int V) {
    x = base + (size_t)m * V;
    const int off = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
    head = min(off ? kVec<T> - off : 0, V);
    n_vec = (V - head) / kVec<T>;
    tail_at = head + n_vec * kVec<T>;
  }
  // the single element of thread t, or -1
  __device__ __forceinline__ int edge(int t, int V) const {
    if (t < head) return t;
    t -= 8;
    return t >= 0 && t < V - tail_at ? tail_at + t : -1;
  }
};

__device__ __forceinline__ float as_f32(float x) { return x; }
__device__ __forceinline__ float as_f32(uint16_t x) { return bf16_to_f32(x); }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(uint16_t* p, float v) { *p = f32_to_bf16(v); }

// A row on NW wavefronts, NV vectors a lane; with NW = 1 a workgroup has four.
template <typename T, int NW, int NV, bool GRAD>
__global__ __launch_bounds__(NW == 1 ? 256 : NW * 64) void k_loss_rows(LossArgs a) {
  __shared__ float sh[2][NW];
  constexpr int N = kVec<T>;
  const int t = NW == 1 ? threadIdx.x & 63 : threadIdx.x;
  const int m = NW == 1 ? blockIdx.x * 4 + (threadIdx.x >> 6) : blockIdx.x;
  if (m >= a.M) return;
  const Row<T> row((const T*)a.x, m, a.V);
  T* dx = (T*)a.dx + (size_t)m * a.V;
  const int target = a.targets[m], at = row.edge(t, a.V);
  if ((unsigned)target >= (unsigned)a.V) {
    if (t == 0) a.row[m] = 0.f;
    if constexpr (GRAD) {
      const float z[N] = {};
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int j = i * NW * 64 + t;
        if (j < row.n_vec) Vec<T, N>::store(dx + row.head + j * N, z);
      }
      if (at >= 0) put(dx + at, 0.f);
    }
    return;
  }
  Vec<T, N> v[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int j = i * NW * 64 + t;
    if (j < row.n_vec) v[i].load(row.x + row.head + j * N);
  }
  const float edge = at >= 0 ? as_f32(row.x[at]) : 0.f;
  const float picked = as_f32(row.x[target]);
  const float inv = GRAD ? *a.inv : 0.f;
  float top = at >= 0 ? edge : -INFINITY;
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (i * NW * 64 + t < row.n_vec) {
#pragma unroll
      for (int e = 0; e < N; ++e) top = fmaxf(top, v[i].get(e));
    }
  top = group_max<NW>(top, sh[0]);
  const float top2 = top * LOG2E;
  float sum = at >= 0 ? exp_from(edge, top2) : 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (i * NW * 64 + t < row.n_vec) {
#pragma unroll
      for (int e = 0; e < N; ++e) sum += exp_from(v[i].get(e), top2);
    }
  sum = group_sum<NW>(sum, sh[1]);
  if (t == 0) a.row[m] = loss_of(top, top2, sum, picked);
  if constexpr (GRAD) {
    const float k = inv / sum;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int j = i * NW * 64 + t;
      if (j < row.n_vec) {
        const int first = row.head + j * N;
        float o[N];
#pragma unroll
        for (int e = 0; e < N; ++e)
          o[e] = exp_from(v[i].get(e), top2) * k - (first + e == target ? inv : 0.f);
        Vec<T, N>::store(dx + first, o);
      }
    }
    if (at >= 0) put(dx + at, exp_from(edge, top2) * k - (at == target ? inv : 0.f));
  }
}

// Any length: the row is read for its statistics and again for its gradient.
template <typename T, bool GRAD>
__global__ __launch_bounds__(1024) void k_loss_long(LossArgs a) {
  __shared__ float sh[2][16];
  constexpr int N = kVec<T>;
  const int t = threadIdx.x, m = blockIdx.x;
  const Row<T> row((const T*)a.x, m, a.V);
  T* dx = (T*)a.dx + (size_t)m * a.V;
  const int target = a.targets[m], at = row.edge(t, a.V);
  const bool counts = (unsigned)target < (unsigned)a.V;
  const float inv = GRAD && counts ? *a.inv : 0.f;
  const float edge = at >= 0 ? as_f32(row.x[at]) : 0.f;
  float top2 = 0.f, k = 0.f;
  if (counts) {
    const float picked = as_f32(row.x[target]);
    float top = at >= 0 ? edge : -INFINITY;
#pragma unroll 4
    for (int j = t; j < row.n_vec; j += 1024) {
      Vec<T, N> v;
      v.load(row.x + row.head + j * N);
#pragma unroll
      for (int e = 0; e < N; ++e) top = fmaxf(top, v.get(e));
    }
    top = group_max<16>(top, sh[0]);
    top2 = top * LOG2E;
    float sum = at >= 0 ? exp_from(edge, top2) : 0.f;
#pragma unroll 4
    for (int j = t; j < row.n_vec; j += 1024) {
      Vec<T, N> v;
      v.load(row.x + row.head + j * N);
#pragma unroll
      for (int e = 0; e < N; ++e) sum += exp_from(v.get(e), top2);
    }
    sum = group_sum<16>(sum, sh[1]);
    if (t == 0) a.row[m] = loss_of(top, top2, sum, picked);
    k = inv / sum;
  } else if (t == 0) {
    a.row[m] = 0.f;
  }
  if constexpr (GRAD) {
#pragma unroll 4
    for (int j = t; j < row.n_vec; j += 1024) {
      const int first = row.head + j * N;
      Vec<T, N> v;
      float o[N];
      v.load(row.x + first);
#pragma unroll
      for (int e = 0; e < N; ++e)
        o[e] = counts ? exp_from(v.get(e), top2) * k - (first + e == target ? inv : 0.f) : 0.f;
      Vec<T, N>::store(dx + first, o);
    }
    if (at >= 0)
      put(dx + at, counts ? exp_from(edge, top2) * k - (at == target ? inv : 0.f) : 0.f);
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

// By the row's aligned vectors: one wavefront up to 4 vectors a lane (no
// barrier), 4 wavefronts up to 8, 8 wavefronts up to 16; fp32 rows past that, and
// up to 65536 logits, on 16.
template <typename T, bool GRAD>
void launch_rows(const LossArgs& a, hipStream_t s) {
  const int n = (a.V + kVec<T> - 1) / kVec<T>;
  const auto rows = [&](auto NW, auto NV) {
    constexpr int nw = NW.value;
    k_loss_rows<T, nw, NV.value, GRAD>
        <<<nw == 1 ? (a.M + 3) / 4 : a.M, nw == 1 ? 256 : nw * 64, 0, s>>>(a);
  };
  using std::integral_constant;
  if (n <= 64) rows(integral_constant<int, 1>{}, integral_constant<int, 1>{});
  else if (n <= 256) rows(integral_constant<int, 1>{}, integral_constant<int, 4>{});
  else if (n <= 1024) rows(integral_constant<int, 4>{}, integral_constant<int, 4>{});
  else if (n <= 2048) rows(integral_constant<int, 4>{}, integral_constant<int, 8>{});
  else if (n <= 4096) rows(integral_constant<int, 8>{}, integral_constant<int, 8>{});
  else if (n <= 8192) rows(integral_constant<int, 8>{}, integral_constant<int, 16>{});
  else if (n <= 16384) rows(integral_constant<int, 16>{}, integral_constant<int, 16>{});
  else k_loss_long<T, GRAD><<<a.M, 1024, 0, s>>>(a);
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
  SKV_REQUIRE(aligned16(dx) && aligned16(x) && aligned16(ws), SKV_E_INVALID,
              "skv_cross_entropy: pointers must be 16-byte aligned");
  SKV_REQUIRE(ws_bytes >= skv_cross_entropy_workspace_bytes(M), SKV_E_WORKSPACE,
              "skv_cross_entropy: workspace of %zu bytes, %zu needed", ws_bytes,
              skv_cross_entropy_workspace_bytes(M));
  hipStream_t s = (hipStream_t)stream;
  float* inv = (float*)ws;
  LossArgs a = {x, dx, targets, row_loss ? row_loss : inv + 4, inv, M, V};
  if (dx) k_loss_count<<<1, 1024, 0, s>>>(inv, targets, M, V, grad_scale);
  if (dt == SKV_BF16) {
    if (dx) launch_rows<uint16_t, true>(a, s);
    else launch_rows<uint16_t, false>(a, s);
  } else {
    if (dx) launch_rows<float, true>(a, s);
    else launch_rows<float, false>(a, s);
  }
  k_loss_mean<<<1, 1024, 0, s>>>(loss, a.row, targets, M, V);
  return check_launch("skv_cross_entropy");
}
