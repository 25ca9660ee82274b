// LayerNorm for training: the forward with its row statistics, and the
// gradients of its input, weight and bias.
//
//   y  = (x - mean) rstd gamma + beta,   rstd = 1 / sqrt(var + eps)
//   dx = rstd (g - mean(g) - xh mean(g xh)) [+ residual],
//        g = dy gamma, xh = (x - mean) rstd
//   dgamma = sum over rows of dy xh, dbeta = sum over rows of dy
//
// Both directions are bound by HBM: a row is read once into registers, its sums go over
// the row's lanes, and the result is written. A row is on 16, 32 or 64 lanes of a wavefront
// up to 1024 columns or, of many rows, 1280 in fp32 and 2048 in bf16 (no LDS, no barrier), on
// 4 wavefronts up to 4096 (8192 in a bf16 forward), and on 16 up to 16384.
// 16384 x 1024 bf16 forward: 11.6 us = 5.8 TB/s (its output with the nt bit; 13.0
// without). 16384 x 768 fp32 backward with a residual: 36.3 us = 5.5 TB/s (rows read with
// the nt bit; 43.5 without), 4 of them for the weight gradients' second pass. Rows that
// end inside a vector, 8192 x 1001: 8.7 us forward bf16 and 23.4 backward fp32, where
// 1024 columns take 7.3 and 22.2.
#include "train_common.h"

namespace skv {
namespace {

using namespace train;

constexpr int kMaxD = 16384;
constexpr int kLaneCols = 16;  // columns of a row that a lane has

constexpr int bwd_threads(int WPR) { return WPR == 16 ? 1024 : 512; }

// A row's place in a workgroup of THREADS lanes: LPR lanes of a wavefront (16, 32 or 64)
// with WPR = 1, or WPR whole wavefronts.
template <int LPR, int WPR, int THREADS>
struct Place {
  static constexpr int kLanes = LPR * WPR;
  static constexpr int kRows = THREADS / kLanes;  // rows at a time
  static __device__ __forceinline__ int row() { return threadIdx.x / kLanes; }
  static __device__ __forceinline__ int lane() { return threadIdx.x % kLanes; }
};

// Sums over a row's lanes: sh [2][wavefronts][2] (two calls in a row do not share a
// slot, so one barrier a call is enough).
template <int LPR, int WPR, int THREADS>
__device__ __forceinline__ void row_sums(float& a, float& b, float* sh, int& turn) {
  a = row16_sum(a);
  b = row16_sum(b);
  if constexpr (LPR >= 32) {
    a = xor16_sum(a);
    b = xor16_sum(b);
  }
  if constexpr (LPR == 64) {
    a = xor32_sum(a);
    b = xor32_sum(b);
  }
  if constexpr (WPR > 1) {
    float* s = sh + turn * 2 * (THREADS / 64);
    turn ^= 1;
    const int w = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) {
      s[2 * w] = a;
      s[2 * w + 1] = b;
    }
    __syncthreads();
    s += w / WPR * WPR * 2;
    a = b = 0.f;
#pragma unroll
    for (int i = 0; i < WPR; ++i) {
      a += s[2 * i];
      b += s[2 * i + 1];
    }
  }
}

template <typename T, int NCH, int LPR, int WPR, int KIND>
__global__ __launch_bounds__(WPR == 16 ? 1024 : 256) void k_ln_fwd(
    T* y, float* __restrict__ mean_out, float* __restrict__ rstd_out, const T* x,
    const float* __restrict__ gamma, const float* __restrict__ beta, int M, int d, float eps) {
  constexpr int kThreads = WPR == 16 ? 1024 : 256, VEC = 16 / sizeof(T);
  using P = Place<LPR, WPR, kThreads>;
  __shared__ float sh[4 * WPR];
  const int m = blockIdx.x * P::kRows + P::row();
  if (m >= M) return;  // only where there are several rows, and then no barrier below
  const int c0 = P::lane() * VEC;
  constexpr int kStep = P::kLanes * VEC;
  const T* xr = x + (size_t)m * d;
  Vec<T, VEC> v[NCH];
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    v[i].zero();
    const int j = c0 + i * kStep;
    if (j < d) v[i].template load_row<KIND>(xr, j, d);
  }
#pragma unroll
  for (int i = 0; i < NCH; ++i) v[i].template settle<KIND>(c0 + i * kStep, d);
  float s = 0.f, q = 0.f;
#pragma unroll
  for (int i = 0; i < NCH; ++i)
#pragma unroll
    for (int e = 0; e < VEC; ++e) s += v[i].get(e);
  int turn = 0;
  row_sums<LPR, WPR, kThreads>(s, q, sh, turn);
  const float fd = (float)d;
  const float mean = s / fd;
  // deviations from the rounded mean, and their own mean c: what the rounding
  // of a mean far from zero leaves
  s = q = 0.f;
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    if (c0 + i * kStep < d) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float t = v[i].get(e) - mean;
        if (KIND == kEven || c0 + i * kStep + e < d) {
          s += t;
          q += t * t;
        }
      }
    }
  }
  row_sums<LPR, WPR, kThreads>(s, q, sh, turn);
  const float c = s / fd;
  const float var = q / fd - c * c;
  const float rstd = 1.f / sqrtf((var < 0.f ? 0.f : var) + eps);  // a NaN stays one
  if (P::lane() == 0) {
    if (mean_out) mean_out[m] = c == c ? mean + c : mean;  // an infinite mean has no deviations
    if (rstd_out) rstd_out[m] = rstd;
  }
  T* yr = y + (size_t)m * d;
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const int j = c0 + i * kStep;
    if (j < d) {
      Vec<float, VEC> g, b;
      g.template load_row<KIND>(gamma, j, d);
      b.template load_row<KIND>(beta, j, d);
      g.template settle<KIND>(j, d);
      b.template settle<KIND>(j, d);
      float o[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        o[e] = ((v[i].get(e) - mean) - c) * rstd * g.get(e) + b.get(e);
      Vec<T, VEC>::template store_stream_row<KIND>(yr, j, d, o);
    }
  }
}

// A workgroup's rows, kRows at a time: a lane holds the same columns of every row, so
// the sums of dgamma and dbeta stay in its registers until the end, and then go over
// the row places in LDS, in their order. part: the workgroup's sums, [grid][2][dp].
// (Reading the next row while one is worked on gained nothing: 8 wavefronts a CU hide it.)
template <typename T, int NCH, int LPR, int WPR, int KIND, bool RES>
__global__ __launch_bounds__(bwd_threads(WPR)) void k_ln_bwd(
    T* dx, float* __restrict__ part, const T* dy, const T* x, const float* __restrict__ gamma,
    const float* __restrict__ mean, const float* __restrict__ rstd, const T* residual, int M, int d,
    int dp) {
  constexpr int kThreads = bwd_threads(WPR), VEC = 16 / sizeof(T);
  using P = Place<LPR, WPR, kThreads>;
  __shared__ float sh[4 * (kThreads / 64)];
  const int c0 = P::lane() * VEC;
  constexpr int kStep = P::kLanes * VEC;
  const float inv_d = 1.f / (float)d;
  float ga[NCH][VEC], sg[NCH][VEC], sb[NCH][VEC];
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    Vec<float, VEC> g;
    g.zero();
    const int j = c0 + i * kStep;
    if (j < d) g.template load_row<KIND>(gamma, j, d);
    g.template settle<KIND>(j, d);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      ga[i][e] = g.get(e);
      sg[i][e] = sb[i][e] = 0.f;
    }
  }
  int turn = 0;
  for (int m0 = blockIdx.x * P::kRows; m0 < M; m0 += gridDim.x * P::kRows) {
    const int m = m0 + P::row();
    const bool here = m < M;  // a place without a row: zeros, and nothing is stored
    const size_t at = (size_t)m * d;
    Vec<T, VEC> vx[NCH], vy[NCH], vr[NCH];
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      vx[i].zero();
      vy[i].zero();
      const int j = c0 + i * kStep;
      if (here && j < d) {
        vx[i].template stream_row<KIND>(x + at, j, d);
        vy[i].template stream_row<KIND>(dy + at, j, d);
        if constexpr (RES) vr[i].template stream_row<KIND>(residual + at, j, d);
      }
    }
    const float mu = here ? mean[m] : 0.f, rs = here ? rstd[m] : 0.f;
    float a = 0.f, b = 0.f;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      vx[i].template settle<KIND>(c0 + i * kStep, d);
      vy[i].template settle<KIND>(c0 + i * kStep, d);
      if (c0 + i * kStep < d) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float xh = (vx[i].get(e) - mu) * rs, t = vy[i].get(e);
          const float g = t * ga[i][e];
          a += g;
          // past the row's end, in its last vectors, g is 0 but xh may be infinite
          if (KIND == kEven || i < NCH - 1 || c0 + i * kStep + e < d) b += g * xh;
          sg[i][e] += t * xh;
          sb[i][e] += t;
        }
      }
    }
    row_sums<LPR, WPR, kThreads>(a, b, sh, turn);
    a *= inv_d;
    b *= inv_d;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const int j = c0 + i * kStep;
      if (here && j < d) {
        if constexpr (RES) vr[i].template settle<KIND>(j, d);
        float r[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float xh = (vx[i].get(e) - mu) * rs;
          r[e] = rs * (vy[i].get(e) * ga[i][e] - a - xh * b);
          if constexpr (RES) r[e] += vr[i].get(e);
        }
        Vec<T, VEC>::template store_row<KIND>(dx + at, j, d, r);
      }
    }
  }
  float* out = part + (size_t)blockIdx.x * 2 * dp;
  constexpr int kSlots = kThreads / 64 / WPR;  // sums that come together
  if constexpr (kSlots > 1) {
    __shared__ float acc[kSlots][2][P::kLanes * VEC * NCH];
    const int slot = (threadIdx.x >> 6) / WPR;
    if constexpr (LPR < 64) {  // a wavefront's places first
#pragma unroll
      for (int i = 0; i < NCH; ++i)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          if constexpr (LPR == 16) {
            sg[i][e] = xor16_sum(sg[i][e]);
            sb[i][e] = xor16_sum(sb[i][e]);
          }
          sg[i][e] = xor32_sum(sg[i][e]);
          sb[i][e] = xor32_sum(sb[i][e]);
        }
    }
    if ((threadIdx.x & 63) < LPR) {
#pragma unroll
      for (int i = 0; i < NCH; ++i)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          acc[slot][0][c0 + i * kStep + e] = sg[i][e];
          acc[slot][1][c0 + i * kStep + e] = sb[i][e];
        }
    }
    __syncthreads();
    for (int j = threadIdx.x; j < d; j += kThreads) {
      float g = 0.f, b = 0.f;
#pragma unroll
      for (int q = 0; q < kSlots; ++q) {
        g += acc[q][0][j];
        b += acc[q][1][j];
      }
      out[j] = g;
      out[dp + j] = b;
    }
  } else {
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const int j = c0 + i * kStep;
      if (j < d) {
        Vec<float, VEC>::template store_row<KIND>(out, j, d, sg[i]);
        Vec<float, VEC>::template store_row<KIND>(out + dp, j, d, sb[i]);
      }
    }
  }
}

// dgamma and dbeta: the columns' sums over the P workgroups' parts, in a fixed
// order. A workgroup has 64 columns: 16 lanes of 4 by 64 groups of rows, four to a
// wavefront; a group's parts, 4 at most, are in flight at once.
__global__ __launch_bounds__(1024) void k_ln_wgrad(float* __restrict__ dgamma,
                                                   float* __restrict__ dbeta,
                                                   const float* __restrict__ part, int P, int d,
                                                   int dp, int accumulate) {
  __shared__ float sh[16][64];
  const int c = threadIdx.x & 15, r = threadIdx.x >> 4;
  const int j = blockIdx.x * 64 + c * 4;  // of 2 dp columns
  f32x4_t s = {0.f, 0.f, 0.f, 0.f};
  if (j < 2 * dp) {
#pragma unroll 4
    for (int p = r; p < P; p += 64)
      s += *reinterpret_cast<const f32x4_t*>(part + (size_t)p * 2 * dp + j);
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) s[e] = xor32_sum(xor16_sum(s[e]));
  if ((threadIdx.x & 63) < 16) *reinterpret_cast<f32x4_t*>(&sh[threadIdx.x >> 6][c * 4]) = s;
  __syncthreads();
  const int at = blockIdx.x * 64 + threadIdx.x;
  if (threadIdx.x < 64 && at < 2 * dp) {
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < 16; ++w) t += sh[w][threadIdx.x];
    const int col = at < dp ? at : at - dp;
    float* out = (at < dp ? dgamma : dbeta) + col;
    if (col < d) *out = accumulate ? *out + t : t;
  }
}

// Lanes of a row in one wavefront: 16, 32 or 64. Few, so that narrow rows leave few lanes
// idle: up to kLaneCols columns a lane (32768 x 257 bf16 backward: 28.5 us with 64 lanes,
// 23.0 with 32). More, down to half as many columns, where there are too few rows for a
// backward workgroup on every CU (2048 x 390: 7.1 us with 64, 7.9 with 32).
int lanes_of(int M, int d) {
  const auto fits = [&](int lanes) {
    return d <= lanes * (M >= 256 * (512 / lanes) ? kLaneCols : kLaneCols / 2);
  };
  return fits(16) ? 16 : fits(32) ? 32 : 64;
}
// Wavefronts of a row: 1, 4 or 16, by kLaneCols columns a lane. Where the rows are enough for
// eight wavefronts a CU all the same, a lane has more of them: on one wavefront 32 columns of
// bf16 and 20 of fp32 (backward, 65536 rows: 1500 of bf16 198 us on four and 121 on one, 2048
// of bf16 175 and 132, 1025 of fp32 195 and 141, but 1536 of fp32 224 and 243; forward: 114 and
// 87, 116 and 102, 139 and 109, 152 and 156), and in the forward 32 of bf16 on four (16384 x
// 5000: 102 us on sixteen, 72; the backward gains nothing).
int waves_of(int M, int d, int dt, bool forward) {
  const bool wide = dt == SKV_BF16;
  if (d <= (M < 2048 ? 64 * kLaneCols : wide ? 128 * kLaneCols : 80 * kLaneCols)) return 1;
  return d <= (forward && wide && M >= 512 ? 512 : 256) * kLaneCols ? 4 : 16;
}
// Rows of a workgroup of `threads` lanes.
int rows_of(int M, int d, int waves, int threads) { return threads / (lanes_of(M, d) * waves); }

// f(vectors of VEC elements a lane, exactly, lanes and wavefronts of a row, the rows' kind) as
// compile-time constants. MANY: the most vectors a lane of rows on four wavefronts.
template <int VEC, int MANY, typename F>
void dispatch(int M, int d, int wpr, F f) {
  using std::integral_constant;
  const int lpr = lanes_of(M, d);
  const int n = (d + lpr * wpr * VEC - 1) / (lpr * wpr * VEC);
  const RowKind kind = row_kind(d, VEC);
  const integral_constant<int, 1> one;
  const auto with_kind = [&](auto N, auto L, auto W) {
    if (kind == kEven) f(N, L, W, integral_constant<int, kEven>{});
    else f(N, L, W, integral_constant<int, kOdd>{});
  };
  // run(the row's vectors a lane), MOST (2 or 4) or fewer. On 32 lanes and more a row has over
  // kLaneCols / 4 columns a lane: two vectors of fp32 at least.
  const auto few = [&](auto LANES, auto MOST, auto run) {
    if constexpr (LANES.value == 16 || VEC > kLaneCols / 4) {
      if (n <= 1) return run(one);
    }
    if constexpr (MOST.value > 2) {
      if (n <= 2) return run(integral_constant<int, 2>{});
      if (n <= 3) return run(integral_constant<int, 3>{});
    }
    run(MOST);
  };
  const integral_constant<int, kLaneCols / VEC> most;
  if (kind == kTiny) return f(one, integral_constant<int, 16>{}, one, integral_constant<int, kTiny>{});
  if (lpr == 16) {
    const integral_constant<int, 16> L;
    few(L, most, [&](auto N) { with_kind(N, L, one); });
  } else if (lpr == 32) {
    const integral_constant<int, 32> L;
    few(L, most, [&](auto N) { with_kind(N, L, one); });
  } else if (wpr == 1) {
    const integral_constant<int, 64> L;
    if constexpr (VEC == 4) {
      if (n > 4) return with_kind(integral_constant<int, 5>{}, L, one);
    }
    few(L, integral_constant<int, 4>{}, [&](auto N) { with_kind(N, L, one); });
  } else if (wpr == 4) {
    const integral_constant<int, 64> L;
    few(L, integral_constant<int, MANY>{},
        [&](auto N) { with_kind(N, L, integral_constant<int, 4>{}); });
  } else {
    const integral_constant<int, 64> L;
    few(L, most, [&](auto N) { with_kind(N, L, integral_constant<int, 16>{}); });
  }
}

// Workgroups of the backward: one to a CU (each leaves a part of the weight gradients,
// to be read again), no more than there are rows for.
int bwd_groups(int M, int d, int dt) {
  const int waves = waves_of(M, d, dt, false), rows = rows_of(M, d, waves, bwd_threads(waves));
  const int need = (M + rows - 1) / rows;
  return need < 256 ? need : 256;
}

int padded(int d) { return (d + 3) / 4 * 4; }

int check(const char* fn, int M, int d, int dt) {
  SKV_REQUIRE(M > 0 && d > 0, SKV_E_INVALID, "%s: dims must be > 0", fn);
  SKV_REQUIRE(dt == SKV_F32 || dt == SKV_BF16, SKV_E_INVALID, "%s: bad dtype", fn);
  SKV_REQUIRE(d <= kMaxD, SKV_E_UNSUPPORTED, "%s: d=%d > %d", fn, d, kMaxD);
  SKV_REQUIRE(M <= kMaxRows, SKV_E_UNSUPPORTED, "%s: M=%d > 2^30", fn, M);
  return SKV_OK;
}

}  // namespace
}  // namespace skv

using namespace skv;

extern "C" int skv_layernorm_fwd(void* y, float* mean, float* rstd, const void* x,
                                 const float* gamma, const float* beta, int M, int d, float eps,
                                 int dt, skv_stream_t stream) {
  SKV_REQUIRE(y && x && gamma && beta, SKV_E_INVALID, "skv_layernorm_fwd: null pointer argument");
  if (int rc = check("skv_layernorm_fwd", M, d, dt)) return rc;
  const int waves = waves_of(M, d, dt, true), threads = waves == 16 ? 1024 : 256;
  const int rows = rows_of(M, d, waves, threads);
  const unsigned grid = (M + rows - 1) / rows;
  SKV_REQUIRE(launchable(grid, threads), SKV_E_UNSUPPORTED,
              "skv_layernorm_fwd: %d rows of %d are too many for a launch", M, d);
  SKV_REQUIRE(aligned16(y) && aligned16(x) && aligned16(gamma) && aligned16(beta), SKV_E_INVALID,
              "skv_layernorm_fwd: pointers must be 16-byte aligned");
  const size_t act = (size_t)M * d * (dt == SKV_BF16 ? 2 : 4), row = (size_t)M * 4;
  if (int rc = apart("skv_layernorm_fwd",
                     {{y, act, "output"}, {mean, row, "mean"}, {rstd, row, "rstd"}},
                     {{x, act, "input", 0}, {gamma, (size_t)d * 4, "gamma"},
                      {beta, (size_t)d * 4, "beta"}}))
    return rc;
  const auto run = [&](auto* yt) {
    using T = std::remove_pointer_t<decltype(yt)>;
    dispatch<16 / sizeof(T), 4>(M, d, waves, [&](auto N, auto L, auto W, auto KIND) {
      k_ln_fwd<T, N.value, L.value, W.value, KIND.value>
          <<<grid, threads, 0, (hipStream_t)stream>>>(
              yt, mean, rstd, (const T*)x, gamma, beta, M, d, eps);
    });
  };
  if (dt == SKV_BF16) run((uint16_t*)y);
  else run((float*)y);
  return check_launch("skv_layernorm_fwd");
}

extern "C" size_t skv_layernorm_bwd_workspace_bytes(int M, int d) {
  if (M <= 0 || M > kMaxRows || d <= 0 || d > kMaxD) return 0;
  // 256 for both types where their wavefronts differ, from 2048 rows on
  return (size_t)bwd_groups(M, d, SKV_F32) * 2 * padded(d) * sizeof(float);
}

extern "C" int skv_layernorm_bwd(void* dx, float* dgamma, float* dbeta, const void* dy,
                                 const void* x, const float* gamma, const float* mean,
                                 const float* rstd, const void* residual, int M, int d,
                                 int accumulate, void* ws, size_t ws_bytes, int dt,
                                 skv_stream_t stream) {
  SKV_REQUIRE(dx && dgamma && dbeta && dy && x && gamma && mean && rstd && ws, SKV_E_INVALID,
              "skv_layernorm_bwd: null pointer argument");
  if (int rc = check("skv_layernorm_bwd", M, d, dt)) return rc;
  SKV_REQUIRE(aligned16(dx) && aligned16(dy) && aligned16(x) && aligned16(gamma) &&
                  aligned16(residual) && aligned16(ws),
              SKV_E_INVALID, "skv_layernorm_bwd: pointers must be 16-byte aligned");
  SKV_REQUIRE(ws_bytes >= skv_layernorm_bwd_workspace_bytes(M, d), SKV_E_WORKSPACE,
              "skv_layernorm_bwd: workspace of %zu bytes, %zu needed", ws_bytes,
              skv_layernorm_bwd_workspace_bytes(M, d));
  const size_t act = (size_t)M * d * (dt == SKV_BF16 ? 2 : 4), row = (size_t)M * 4,
               col = (size_t)d * 4;
  if (int rc = apart("skv_layernorm_bwd",
                     {{dx, act, "grad_input"}, {dgamma, col, "grad_gamma"},
                      {dbeta, col, "grad_beta"}, {ws, ws_bytes, "the workspace"}},
                     {{dy, act, "grad_output", 0}, {x, act, "input", 0},
                      {residual, act, "residual", 0}, {gamma, col, "gamma"}, {mean, row, "mean"},
                      {rstd, row, "rstd"}}))
    return rc;
  const int P = bwd_groups(M, d, dt), dp = padded(d);
  float* part = (float*)ws;
  const auto run = [&](auto* xt) {
    using T = std::remove_pointer_t<decltype(xt)>;
    constexpr int vec = 16 / sizeof(T);
    dispatch<vec, kLaneCols / vec>(M, d, waves_of(M, d, dt, false), [&](auto N, auto L, auto W,
                                                                       auto KIND) {
      constexpr int threads = bwd_threads(W.value);
      const auto go = [&](auto RES) {
        k_ln_bwd<T, N.value, L.value, W.value, KIND.value, RES.value>
            <<<P, threads, 0, (hipStream_t)stream>>>(xt, part, (const T*)dy, (const T*)x, gamma, mean,
                                                     rstd, (const T*)residual, M, d, dp);
      };
      if (residual) go(std::true_type{});
      else go(std::false_type{});
    });
  };
  if (dt == SKV_BF16) run((uint16_t*)dx);
  else run((float*)dx);
  if (int rc = check_launch("skv_layernorm_bwd")) return rc;
  k_ln_wgrad<<<(2 * dp + 63) / 64, 1024, 0, (hipStream_t)stream>>>(dgamma, dbeta, part, P, d, dp,
                                                                   accumulate);
  return check_launch("skv_layernorm_bwd");
}
