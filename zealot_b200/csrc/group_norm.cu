// group_norm.cu -- group norm over channels-last rows with an activation, and
// its gradient.
//
// x [N, L, C], groups of w = C / G neighbouring channels; per (n, g), over
// L x w elements: mu, var, xh = (x - mu) / sqrt(var + eps); then
// y = act(gamma xh + beta).  Gradient, with dz = dy act'(z):
//   dbeta = sum dz, dgamma = sum dz xh,
//   dx = rstd (gamma dz - mean(gamma dz) - xh mean(gamma dz xh)).
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "seq_common.cuh"

namespace zrl {
namespace {

constexpr int kThreads = 256;

struct NormArgs {
  const void *x, *dy;
  const float *gamma, *beta;
  void *y, *dx;
  float *mean, *rstd;
  int64_t N, L, sxn, sxl, syn, syl, sdn, sdl;  // strides of x, y / dy, dx
  int32_t C, G, w, act;
  float eps;
};

// act(z) and act'(z)
__device__ __forceinline__ float act_value(float z, int act) {
  if (act == ZRL_ACT_ELU) return z > 0.0f ? z : expm1f(z);
  if (act == ZRL_ACT_SILU) return z / (1.0f + expf(-z));
  if (act == ZRL_ACT_GELU) return 0.5f * z * (1.0f + erff(z * 0.70710678f));
  return z;
}
__device__ __forceinline__ float act_slope(float z, int act) {
  if (act == ZRL_ACT_ELU) return z > 0.0f ? 1.0f : expf(z);
  if (act == ZRL_ACT_SILU) {
    const float s = 1.0f / (1.0f + expf(-z));
    return s * (1.0f + z * (1.0f - s));
  }
  if (act == ZRL_ACT_GELU)
    return 0.5f * (1.0f + erff(z * 0.70710678f)) + z * 0.39894228f * expf(-0.5f * z * z);
  return 1.0f;
}

// Sum over the block, the same in every thread; buf holds one float per warp.
__device__ __forceinline__ float block_sum(float v, float *buf) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.0f;
  for (int i = 0; i < kThreads / 32; ++i) v += buf[i];
  return v;
}

// One block per (n, g).
template <typename T>
__global__ void __launch_bounds__(kThreads) norm_kernel(const NormArgs a) {
  __shared__ float buf[kThreads / 32];
  const int64_t n_el = a.L * a.w;
  const float inv = n_el ? 1.0f / (float)n_el : 0.0f;
  for (int64_t ng = blockIdx.x; ng < a.N * a.G; ng += gridDim.x) {
    const int64_t n = ng / a.G;
    const int c0 = (int)(ng - n * a.G) * a.w;
    const T *x = static_cast<const T *>(a.x) + n * a.sxn + c0;
    T *y = static_cast<T *>(a.y) + n * a.syn + c0;
    float s = 0.0f;
    for (int64_t e = threadIdx.x; e < n_el; e += kThreads)
      s += to_f32(x[(e / a.w) * a.sxl + e % a.w]);
    const float mu = block_sum(s, buf) * inv;
    s = 0.0f;
    for (int64_t e = threadIdx.x; e < n_el; e += kThreads) {
      const float d = to_f32(x[(e / a.w) * a.sxl + e % a.w]) - mu;
      s += d * d;
    }
    const float rstd = rsqrtf(block_sum(s, buf) * inv + a.eps);
    for (int64_t e = threadIdx.x; e < n_el; e += kThreads) {
      const int64_t l = e / a.w;
      const int c = (int)(e - l * a.w);
      const float xh = (to_f32(x[l * a.sxl + c]) - mu) * rstd;
      const float z = xh * (a.gamma ? a.gamma[c0 + c] : 1.0f) + (a.beta ? a.beta[c0 + c] : 0.0f);
      y[l * a.syl + c] = from_f32<T>(act_value(z, a.act));
    }
    if (threadIdx.x == 0) {
      if (a.mean) a.mean[ng] = mu;
      if (a.rstd) a.rstd[ng] = rstd;
    }
  }
}

// One block per (n, g): the two means, then dx.
template <typename T>
__global__ void __launch_bounds__(kThreads) norm_dx_kernel(const NormArgs a) {
  __shared__ float buf[kThreads / 32];
  const int64_t n_el = a.L * a.w;
  const float inv = n_el ? 1.0f / (float)n_el : 0.0f;
  for (int64_t ng = blockIdx.x; ng < a.N * a.G; ng += gridDim.x) {
    const int64_t n = ng / a.G;
    const int c0 = (int)(ng - n * a.G) * a.w;
    const T *x = static_cast<const T *>(a.x) + n * a.sxn + c0;
    const T *dy = static_cast<const T *>(a.dy) + n * a.syn + c0;
    T *dx = static_cast<T *>(a.dx) + n * a.sdn + c0;
    const float mu = a.mean[ng], rstd = a.rstd[ng];
    float s1 = 0.0f, s2 = 0.0f;
    for (int64_t e = threadIdx.x; e < n_el; e += kThreads) {
      const int64_t l = e / a.w;
      const int c = (int)(e - l * a.w);
      const float ga = a.gamma ? a.gamma[c0 + c] : 1.0f;
      const float xh = (to_f32(x[l * a.sxl + c]) - mu) * rstd;
      const float z = xh * ga + (a.beta ? a.beta[c0 + c] : 0.0f);
      const float d = to_f32(dy[l * a.syl + c]) * act_slope(z, a.act) * ga;
      s1 += d;
      s2 += d * xh;
    }
    s1 = block_sum(s1, buf) * inv;
    s2 = block_sum(s2, buf) * inv;
    for (int64_t e = threadIdx.x; e < n_el; e += kThreads) {
      const int64_t l = e / a.w;
      const int c = (int)(e - l * a.w);
      const float ga = a.gamma ? a.gamma[c0 + c] : 1.0f;
      const float xh = (to_f32(x[l * a.sxl + c]) - mu) * rstd;
      const float z = xh * ga + (a.beta ? a.beta[c0 + c] : 0.0f);
      const float d = to_f32(dy[l * a.syl + c]) * act_slope(z, a.act) * ga;
      dx[l * a.sdl + c] = from_f32<T>(rstd * (d - s1 - xh * s2));
    }
  }
}

// Channel sums of dz xh and dz: a block takes 32 channels and one slice of the
// rows and writes part[slice][2][C].
template <typename T>
__global__ void __launch_bounds__(kThreads) norm_param_kernel(const NormArgs a, float *part) {
  __shared__ float sg[kThreads / 32][32], sb[kThreads / 32][32];
  const int lane = threadIdx.x & 31, wy = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  const int64_t rows = a.N * a.L;
  const int64_t per = (rows + gridDim.y - 1) / gridDim.y;
  const int64_t r0 = per * blockIdx.y, r1 = min(rows, r0 + per);
  float dg = 0.0f, db = 0.0f;
  if (c < a.C) {
    const float ga = a.gamma ? a.gamma[c] : 1.0f, be = a.beta ? a.beta[c] : 0.0f;
    for (int64_t r = r0 + wy; r < r1; r += kThreads / 32) {
      const int64_t n = r / a.L, l = r - n * a.L, ng = n * a.G + c / a.w;
      const float xh =
          (to_f32(static_cast<const T *>(a.x)[n * a.sxn + l * a.sxl + c]) - a.mean[ng]) *
          a.rstd[ng];
      const float dz = to_f32(static_cast<const T *>(a.dy)[n * a.syn + l * a.syl + c]) *
                       act_slope(xh * ga + be, a.act);
      dg += dz * xh;
      db += dz;
    }
  }
  sg[wy][lane] = dg;
  sb[wy][lane] = db;
  __syncthreads();
  if (wy == 0 && c < a.C) {
    for (int i = 1; i < kThreads / 32; ++i) {
      dg += sg[i][lane];
      db += sb[i][lane];
    }
    float *p = part + (int64_t)blockIdx.y * 2 * a.C;
    p[c] = dg;
    p[a.C + c] = db;
  }
}

// Folds the slices in order.
__global__ void norm_fold_kernel(const float *part, int slices, int C, float *dgamma,
                                 float *dbeta) {
  const int c = blockIdx.x * blockDim.x + threadIdx.x;
  if (c >= C) return;
  float dg = 0.0f, db = 0.0f;
  for (int i = 0; i < slices; ++i) {
    dg += part[(int64_t)i * 2 * C + c];
    db += part[(int64_t)i * 2 * C + C + c];
  }
  if (dgamma) dgamma[c] = dg;
  if (dbeta) dbeta[c] = db;
}

int param_slices(int64_t rows) {
  return (int)std::max<int64_t>(1, std::min<int64_t>(128, (rows + 63) / 64));
}

zrl_status check_norm(const char *what, int64_t N, int64_t L, int64_t C, int32_t groups,
                      int32_t dtype, int32_t act) {
  if (N < 0 || L < 0 || C < 0 || C > (int64_t)1 << 30)
    return seq_fail(ZRL_INVALID_ARG, "%s: N, L >= 0 and 0 <= C <= 2^30", what);
  if (groups < 1 || C % groups)
    return seq_fail(ZRL_INVALID_ARG, "%s: %lld channels in %d groups", what, (long long)C, groups);
  if (!dtype_ok(dtype)) return seq_fail(ZRL_INVALID_ARG, "%s: unknown dtype %d", what, dtype);
  if (act < ZRL_ACT_NONE || act > ZRL_ACT_GELU)
    return seq_fail(ZRL_INVALID_ARG, "%s: unknown activation %d", what, act);
  return ZRL_OK;
}

}  // namespace
}  // namespace zrl

using namespace zrl;

extern "C" int64_t zrl_group_norm_workspace(int64_t N, int64_t L, int64_t C, int32_t groups,
                                            int32_t grad) {
  if (N <= 0 || L <= 0 || C <= 0 || groups < 1) return 0;
  return grad ? (int64_t)param_slices(N * L) * 2 * C * (int64_t)sizeof(float) : 0;
}

extern "C" zrl_status zrl_group_norm(const void *x, const float *gamma, const float *beta,
                                     int64_t N, int64_t L, int64_t C, int32_t groups,
                                     int32_t dtype, int32_t act, float eps,
                                     const int64_t *strides, void *y, float *mean, float *rstd,
                                     void *workspace, int64_t workspace_bytes, void *stream) {
  const zrl_status s = check_norm("group_norm", N, L, C, groups, dtype, act);
  if (s != ZRL_OK) return s;
  if (!(eps >= 0.0f) || isinf(eps)) return seq_fail(ZRL_INVALID_ARG, "group_norm: eps");
  if (N == 0 || C == 0) return ZRL_OK;
  if (L && (!x || !y)) return seq_fail(ZRL_INVALID_ARG, "group_norm: x or y is NULL");
  const int es = dtype_size(dtype);
  if (!aligned(x, es) || !aligned(y, es) || !aligned(gamma, 4) || !aligned(beta, 4) ||
      !aligned(mean, 4) || !aligned(rstd, 4))
    return seq_fail(ZRL_INVALID_ARG, "group_norm: a pointer is not aligned to its element");
  if (workspace_bytes < zrl_group_norm_workspace(N, L, C, groups, 0))
    return seq_fail(ZRL_INVALID_ARG, "group_norm: workspace too small");
  (void)workspace;
  NormArgs a{};
  a.x = x;
  a.y = y;
  a.gamma = gamma;
  a.beta = beta;
  a.mean = mean;
  a.rstd = rstd;
  a.N = N;
  a.L = L;
  a.C = (int32_t)C;
  a.G = groups;
  a.w = (int32_t)(C / groups);
  a.act = act;
  a.eps = eps;
  a.sxn = strides ? strides[0] : L * C;
  a.sxl = strides ? strides[1] : C;
  a.syn = strides ? strides[2] : L * C;
  a.syl = strides ? strides[3] : C;
  const int64_t blocks = std::min<int64_t>(N * groups, (int64_t)1 << 30);
  with_dtype(dtype, [&](auto t) {
    norm_kernel<decltype(t)>
        <<<(unsigned)blocks, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(a);
  });
  return seq_launched("group_norm");
}

extern "C" zrl_status zrl_group_norm_grad(const void *x, const void *dy, const float *gamma,
                                          const float *beta, const float *mean,
                                          const float *rstd, int64_t N, int64_t L, int64_t C,
                                          int32_t groups, int32_t dtype, int32_t act,
                                          const int64_t *strides, void *dx, float *dgamma,
                                          float *dbeta, void *workspace,
                                          int64_t workspace_bytes, void *stream) {
  const zrl_status s = check_norm("group_norm_grad", N, L, C, groups, dtype, act);
  if (s != ZRL_OK) return s;
  if (C == 0) return ZRL_OK;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (!aligned(dgamma, 4) || !aligned(dbeta, 4))
    return seq_fail(ZRL_INVALID_ARG, "group_norm_grad: a pointer is not aligned to its element");
  const unsigned cb = (unsigned)((C + 255) / 256);
  if (N == 0 || L == 0) {  // no rows: the sums are zero
    norm_fold_kernel<<<cb, 256, 0, st>>>(nullptr, 0, (int)C, dgamma, dbeta);
    return seq_launched("group_norm_grad");
  }
  if (!x || !dy || !dx || !mean || !rstd)
    return seq_fail(ZRL_INVALID_ARG, "group_norm_grad: x, dy, dx, mean or rstd is NULL");
  const int es = dtype_size(dtype);
  if (!aligned(x, es) || !aligned(dy, es) || !aligned(dx, es) || !aligned(gamma, 4) ||
      !aligned(beta, 4) || !aligned(mean, 4) || !aligned(rstd, 4) || !aligned(workspace, 16))
    return seq_fail(ZRL_INVALID_ARG, "group_norm_grad: a pointer is not aligned to its element");
  if (!workspace || workspace_bytes < zrl_group_norm_workspace(N, L, C, groups, 1))
    return seq_fail(ZRL_INVALID_ARG, "group_norm_grad: workspace too small");
  NormArgs a{};
  a.x = x;
  a.dy = dy;
  a.dx = dx;
  a.gamma = gamma;
  a.beta = beta;
  a.mean = const_cast<float *>(mean);
  a.rstd = const_cast<float *>(rstd);
  a.N = N;
  a.L = L;
  a.C = (int32_t)C;
  a.G = groups;
  a.w = (int32_t)(C / groups);
  a.act = act;
  a.sxn = strides ? strides[0] : L * C;
  a.sxl = strides ? strides[1] : C;
  a.syn = strides ? strides[2] : L * C;
  a.syl = strides ? strides[3] : C;
  a.sdn = strides ? strides[4] : L * C;
  a.sdl = strides ? strides[5] : C;
  const int64_t blocks = std::min<int64_t>(N * groups, (int64_t)1 << 30);
  const int slices = param_slices(N * L);
  float *part = static_cast<float *>(workspace);
  with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    norm_dx_kernel<T><<<(unsigned)blocks, kThreads, 0, st>>>(a);
    norm_param_kernel<T>
        <<<dim3((unsigned)((C + 31) / 32), (unsigned)slices), kThreads, 0, st>>>(a, part);
  });
  norm_fold_kernel<<<cb, 256, 0, st>>>(part, slices, (int)C, dgamma, dbeta);
  return seq_launched("group_norm_grad");
}
