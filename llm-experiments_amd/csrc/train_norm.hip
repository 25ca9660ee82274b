// LayerNorm for training: the forward with its row statistics, and the
// gradients of its input, weight and bias.
//
//   y  = (x - mean) rstd gamma + beta,   rstd = 1 / sqrt(var + eps)
//   dx = rstd (g - mean(g) - xh mean(g xh)) [+ residual],
//        g = dy gamma, xh = (x - mean) rstd
//   dgamma = sum over rows of dy xh, dbeta = sum over rows of dy
//
// Both directions are bound by HBM: a row is read once into registers, its sums
// go over the row's wavefronts, and the result is written. A row is on one
// wavefront up to 1024 columns (no LDS, no barrier), on 4 up to 4096 and on 16 up
// to 16384. 16384 x 1024 bf16 forward: 11.6 us = 5.8 TB/s (its output with the nt bit;
// 13.0 without). 16384 x 768 fp32 backward with a residual: 37.9 us = 5.3 TB/s (rows
// read with the nt bit; 43.5 without), 4 of them for the weight gradients' second pass.
#include "train_common.h"

namespace skv {
namespace {

using namespace train;

constexpr int kMaxD = 16384;
constexpr int kLaneCols = 16;  // columns of a row a lane holds

// Sums of a row over its WPR wavefronts: sh [2][WPR][2] (two calls in a row do
// not share a slot, so one barrier a call is enough).
template <int WPR>
__device__ __forceinline__ void row_sums(float& a, float& b, float* sh, int& turn) {
  a = wave_sum(a);
  b = wave_sum(b);
  if constexpr (WPR > 1) {
    float* s = sh + turn * 2 * WPR;
    turn ^= 1;
    const int w = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) {
      s[2 * w] = a;
      s[2 * w + 1] = b;
    }
    __syncthreads();
    a = b = 0.f;
#pragma unroll
    for (int i = 0; i < WPR; ++i) {
      a += s[2 * i];
      b += s[2 * i + 1];
    }
  }
}

template <typename T, int VEC, int NCH, int WPR>
__global__ __launch_bounds__(WPR == 16 ? 1024 : 256) void k_ln_fwd(
    T* y, float* __restrict__ mean_out, float* __restrict__ rstd_out, const T* x,
    const float* __restrict__ gamma, const float* __restrict__ beta, int M, int d, float eps) {
  __shared__ float sh[4 * WPR];
  constexpr int kRows = WPR == 1 ? 4 : 1;  // rows of a workgroup
  const int w = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int m = blockIdx.x * kRows + (WPR == 1 ? w : 0);
  if (m >= M) return;  // WPR = 1: no barrier below
  const int c0 = ((WPR == 1 ? 0 : w) * 64 + lane) * VEC;
  constexpr int kStep = WPR * 64 * VEC;
  const T* xr = x + (size_t)m * d;
  Vec<T, VEC> v[NCH];
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    v[i].zero();
    if (c0 + i * kStep < d) v[i].load(xr + c0 + i * kStep);
  }
  float s = 0.f, q = 0.f;
#pragma unroll
  for (int i = 0; i < NCH; ++i)
#pragma unroll
    for (int e = 0; e < VEC; ++e) s += v[i].get(e);
  int turn = 0;
  row_sums<WPR>(s, q, sh, turn);
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
        s += t;
        q += t * t;
      }
    }
  }
  row_sums<WPR>(s, q, sh, turn);
  const float c = s / fd;
  const float rstd = 1.f / sqrtf(fmaxf(q / fd - c * c, 0.f) + eps);
  if (lane == 0 && (WPR == 1 || w == 0)) {
    if (mean_out) mean_out[m] = mean + c;
    if (rstd_out) rstd_out[m] = rstd;
  }
  T* yr = y + (size_t)m * d;
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    const int j = c0 + i * kStep;
    if (j < d) {
      Vec<float, VEC> g, b;
      g.load(gamma + j);
      b.load(beta + j);
      float o[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        o[e] = ((v[i].get(e) - mean) - c) * rstd * g.get(e) + b.get(e);
      Vec<T, VEC>::store_stream(yr + j, o);
    }
  }
}

// Rows m0, m0 + stride, ... of a workgroup (of each of its wavefronts where a
// row is one wavefront's); a lane holds the same columns of every row, so the
// sums of dgamma and dbeta stay in its registers until the end. part: the
// workgroup's sums, [grid][2][dp].
template <typename T, int VEC, int NCH, int WPR, bool RES>
__global__ __launch_bounds__(WPR == 16 ? 1024 : 256) void k_ln_bwd(
    T* dx, float* __restrict__ part, const T* dy, const T* x, const float* __restrict__ gamma,
    const float* __restrict__ mean, const float* __restrict__ rstd, const T* residual, int M, int d,
    int dp) {
  __shared__ float sh[4 * WPR];
  const int w = threadIdx.x >> 6, lane = threadIdx.x & 63;
  constexpr int kRows = WPR == 1 ? 4 : 1;
  const int c0 = ((WPR == 1 ? 0 : w) * 64 + lane) * VEC;
  constexpr int kStep = WPR * 64 * VEC;
  const float inv_d = 1.f / (float)d;
  float ga[NCH][VEC], sg[NCH][VEC], sb[NCH][VEC];
#pragma unroll
  for (int i = 0; i < NCH; ++i) {
    Vec<float, VEC> g;
    g.zero();
    if (c0 + i * kStep < d) g.load(gamma + c0 + i * kStep);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      ga[i][e] = g.get(e);
      sg[i][e] = sb[i][e] = 0.f;
    }
  }
  int turn = 0;
  for (int m = blockIdx.x * kRows + (WPR == 1 ? w : 0); m < M; m += gridDim.x * kRows) {
    const T* xr = x + (size_t)m * d;
    const T* yr = dy + (size_t)m * d;
    Vec<T, VEC> vx[NCH], vy[NCH], vr[NCH];
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      vx[i].zero();
      vy[i].zero();
      const int j = c0 + i * kStep;
      if (j < d) {
        vx[i].stream(xr + j);
        vy[i].stream(yr + j);
        if constexpr (RES) vr[i].stream(residual + (size_t)m * d + j);
      }
    }
    const float mu = mean[m], rs = rstd[m];
    float a = 0.f, b = 0.f;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      if (c0 + i * kStep < d) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float xh = (vx[i].get(e) - mu) * rs, t = vy[i].get(e);
          const float g = t * ga[i][e];
          a += g;
          b += g * xh;
          sg[i][e] += t * xh;
          sb[i][e] += t;
        }
      }
    }
    row_sums<WPR>(a, b, sh, turn);
    a *= inv_d;
    b *= inv_d;
    T* o = dx + (size_t)m * d;
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const int j = c0 + i * kStep;
      if (j < d) {
        float r[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float xh = (vx[i].get(e) - mu) * rs;
          r[e] = rs * (vy[i].get(e) * ga[i][e] - a - xh * b);
          if constexpr (RES) r[e] += vr[i].get(e);
        }
        Vec<T, VEC>::store(o + j, r);
      }
    }
  }
  float* out = part + (size_t)blockIdx.x * 2 * dp;
  if constexpr (WPR == 1) {  // the four wavefronts' sums, in their order
    __shared__ float acc[2][64 * VEC * NCH];
    for (int t = 0; t < 4; ++t) {
      if (w == t) {
#pragma unroll
        for (int i = 0; i < NCH; ++i)
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            const int j = c0 + i * kStep + e;
            acc[0][j] = t ? acc[0][j] + sg[i][e] : sg[i][e];
            acc[1][j] = t ? acc[1][j] + sb[i][e] : sb[i][e];
          }
      }
      __syncthreads();
    }
    for (int j = threadIdx.x; j < d; j += 256) {
      out[j] = acc[0][j];
      out[dp + j] = acc[1][j];
    }
  } else {
#pragma unroll
    for (int i = 0; i < NCH; ++i) {
      const int j = c0 + i * kStep;
      if (j < d) {
        Vec<float, VEC>::store(out + j, sg[i]);
        Vec<float, VEC>::store(out + dp + j, sb[i]);
      }
    }
  }
}

// dgamma and dbeta: the columns' sums over the P workgroups' parts, in a fixed
// order. A workgroup has 64 columns: 16 lanes of 4 by 64 groups of rows, four to a
// wavefront; up to 512 parts each group's loads are in flight at once.
__global__ __launch_bounds__(1024) void k_ln_wgrad(float* __restrict__ dgamma,
                                                   float* __restrict__ dbeta,
                                                   const float* __restrict__ part, int P, int d,
                                                   int dp, int accumulate) {
  __shared__ float sh[16][64];
  const int c = threadIdx.x & 15, r = threadIdx.x >> 4;
  const int j = blockIdx.x * 64 + c * 4;  // of 2 dp columns
  f32x4_t s = {0.f, 0.f, 0.f, 0.f};
  if (j < 2 * dp) {
#pragma unroll 8
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

// Vector widths: 16 bytes of a row where every row is aligned to them, else
// pairs, else single elements.
int vec_of(int d, int dt) {
  const int full = dt == SKV_BF16 ? 8 : 4;
  if (d % full == 0) return full;
  return d % 2 == 0 ? 2 : 1;
}

int waves_of(int d) { return d <= 64 * kLaneCols ? 1 : d <= 256 * kLaneCols ? 4 : 16; }

// f(vector width, vectors a lane, wavefronts a row) as compile-time constants
template <int FULL, typename F>
void dispatch(int d, int vec, F f) {
  const int wpr = waves_of(d);
  auto with_vec = [&](auto V) {
    constexpr int v = decltype(V)::value;
    const int n = (d + 64 * wpr * v - 1) / (64 * wpr * v);  // vectors a lane
    auto with_n = [&](auto N) {
      if (wpr == 1) f(V, N, std::integral_constant<int, 1>{});
      else if (wpr == 4) f(V, N, std::integral_constant<int, 4>{});
      else f(V, N, std::integral_constant<int, 16>{});
    };
    if constexpr (kLaneCols / v >= 1)
      if (n <= 1) return with_n(std::integral_constant<int, 1>{});
    if constexpr (kLaneCols / v >= 4)
      if (n <= 2) return with_n(std::integral_constant<int, 2>{});
    if constexpr (kLaneCols / v >= 4 && v >= 4)
      if (n <= 3) return with_n(std::integral_constant<int, 3>{});
    if constexpr (kLaneCols / v >= 8)
      if (n <= 4) return with_n(std::integral_constant<int, 4>{});
    if constexpr (kLaneCols / v >= 16)
      if (n <= 8) return with_n(std::integral_constant<int, 8>{});
    with_n(std::integral_constant<int, kLaneCols / v>{});
  };
  if (vec == FULL) with_vec(std::integral_constant<int, FULL>{});
  else if (vec == 2) with_vec(std::integral_constant<int, 2>{});
  else with_vec(std::integral_constant<int, 1>{});
}

// Workgroups of the backward: two to a CU, no more than there are rows for.
int bwd_groups(int M, int d) {
  const int rows = waves_of(d) == 1 ? 4 : 1;
  const int need = (M + rows - 1) / rows;
  return need < 512 ? need : 512;
}

int padded(int d) { return (d + 3) / 4 * 4; }

int check(const char* fn, int M, int d, int dt) {
  SKV_REQUIRE(M > 0 && d > 0, SKV_E_INVALID, "%s: dims must be > 0", fn);
  SKV_REQUIRE(dt == SKV_F32 || dt == SKV_BF16, SKV_E_INVALID, "%s: bad dtype", fn);
  SKV_REQUIRE(d <= kMaxD, SKV_E_UNSUPPORTED, "%s: d=%d > %d", fn, d, kMaxD);
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
  SKV_REQUIRE(aligned16(y) && aligned16(x) && aligned16(gamma) && aligned16(beta), SKV_E_INVALID,
              "skv_layernorm_fwd: pointers must be 16-byte aligned");
  const size_t act = (size_t)M * d * (dt == SKV_BF16 ? 2 : 4), row = (size_t)M * 4;
  if (int rc = apart("skv_layernorm_fwd",
                     {{y, act, "output"}, {mean, row, "mean"}, {rstd, row, "rstd"}},
                     {{x, act, "input", 0}, {gamma, (size_t)d * 4, "gamma"},
                      {beta, (size_t)d * 4, "beta"}}))
    return rc;
  const int rows = waves_of(d) == 1 ? 4 : 1;
  const dim3 grid((M + rows - 1) / rows);
  auto run = [&](auto* yt, auto FULL) {
    using T = std::remove_pointer_t<decltype(yt)>;
    dispatch<decltype(FULL)::value>(d, vec_of(d, dt), [&](auto V, auto N, auto W) {
      k_ln_fwd<T, V.value, N.value, W.value>
          <<<grid, W.value == 16 ? 1024 : 256, 0, (hipStream_t)stream>>>(
              yt, mean, rstd, (const T*)x, gamma, beta, M, d, eps);
    });
  };
  if (dt == SKV_BF16) run((uint16_t*)y, std::integral_constant<int, 8>{});
  else run((float*)y, std::integral_constant<int, 4>{});
  return check_launch("skv_layernorm_fwd");
}

extern "C" size_t skv_layernorm_bwd_workspace_bytes(int M, int d) {
  if (M <= 0 || d <= 0 || d > kMaxD) return 0;
  return (size_t)bwd_groups(M, d) * 2 * padded(d) * sizeof(float);
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
  const int P = bwd_groups(M, d), dp = padded(d);
  float* part = (float*)ws;
  auto run = [&](auto* xt, auto FULL) {
    using T = std::remove_pointer_t<decltype(xt)>;
    dispatch<decltype(FULL)::value>(d, vec_of(d, dt), [&](auto V, auto N, auto W) {
      const int threads = W.value == 16 ? 1024 : 256;
      if (residual)
        k_ln_bwd<T, V.value, N.value, W.value, true><<<P, threads, 0, (hipStream_t)stream>>>(
            xt, part, (const T*)dy, (const T*)x, gamma, mean, rstd, (const T*)residual, M, d, dp);
      else
        k_ln_bwd<T, V.value, N.value, W.value, false><<<P, threads, 0, (hipStream_t)stream>>>(
            xt, part, (const T*)dy, (const T*)x, gamma, mean, rstd, (const T*)nullptr, M, d, dp);
    });
  };
  if (dt == SKV_BF16) run((uint16_t*)dx, std::integral_constant<int, 8>{});
  else run((float*)dx, std::integral_constant<int, 4>{});
  if (int rc = check_launch("skv_layernorm_bwd")) return rc;
  k_ln_wgrad<<<(2 * dp + 63) / 64, 1024, 0, (hipStream_t)stream>>>(dgamma, dbeta, part, P, d, dp,
                                                                   accumulate);
  return check_launch("skv_layernorm_bwd");
}
