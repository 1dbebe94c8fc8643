// group_norm.cuh -- what the forms of group norm share: arguments, activations,
// parameters.
#pragma once

#include "seq_common.cuh"

namespace zrl {
namespace {

constexpr int kThreads = 256;
constexpr int kSms = 148;

struct NormArgs {
  const void *x, *dy;
  const float *gamma, *beta;
  void *y, *dx;
  float *mean, *rstd, *part;
  float2 *means;
  int64_t N, L, sxn, sxl, syn, syl, sdn, sdl;  // strides of x, y / dy, dx
  int32_t C, G, w, act;
  float eps;
  bool wide;  // gamma and beta start on 16 bytes
  // rows: lanes per group, groups of a block, rows of a block
  int32_t p, gb, rb;
  // samples: channels of a block at most, parts of a wide group, stretches of
  // positions, positions of one
  int32_t cols, parts, stretches;
  int64_t stretch;
};

// 1 / (1 + exp(-z))
template <int V>
__device__ __forceinline__ Vec<V> sigmoid(const Vec<V> &z) {
  Vec<V> t = mul(z, -kLog2e);
#pragma unroll
  for (int i = 0; i < V; ++i) t[i] = ex2(t[i]);
  t = add(t, 1.0f);
#pragma unroll
  for (int i = 0; i < V; ++i) t[i] = rcp(t[i]);
  return t;
}

// Phi(z), the normal distribution's, and e = exp(-z^2 / 2).  The tail beyond |z| is
// e R(|z|), R(x) = erfc(x / sqrt 2) exp(x^2 / 2) / 2, a smooth function that falls
// like 1 / x: t P(t) with t = 1 / (1 + 0.3 x), P of degree 7 fitted to it on [0, 14],
// where e ends, within 1.1e-7 relative (6.5e-7 with all roundings).  So a small Phi
// keeps its digits, but for those that z^2 loses in the exponent.
template <int V>
__device__ __forceinline__ Vec<V> normal_cdf(const Vec<V> &z, Vec<V> &e) {
  Vec<V> t;
  e = mul(mul(z, z), -0.5f * kLog2e);
#pragma unroll
  for (int i = 0; i < V; ++i) e[i] = ex2(e[i]), t[i] = fabsf(z[i]);
  t = fma(t, 0.3f, 1.0f);
#pragma unroll
  for (int i = 0; i < V; ++i) t[i] = rcp(t[i]);
  Vec<V> p = fma(t, 0.035649579f, -0.157097667f);
  p = fma(p, t, 0.206167474f);
  p = fma(p, t, -0.0535032786f);
  p = fma(p, t, 0.128457516f);
  p = fma(p, t, 0.0999490991f);
  p = fma(p, t, 0.120747402f);
  p = fma(p, t, 0.119629785f);
  p = mul(mul(p, t), e);
  const Vec<V> q = fma(p, -1.0f, 1.0f);
#pragma unroll
  for (int i = 0; i < V; ++i) p[i] = z[i] < 0.0f ? p[i] : q[i];
  return p;
}

// ELU of z, with the digits of a small z: from -1/2 on e^z - 1 is z + z^2 p(z), p
// fitted to (e^z - 1 - z) / z^2 there (9e-8 of e^z - 1, 1.5e-7 with its roundings);
// below, where the difference loses at most a bit and a half, the exponential less 1.
// Above 0 the square is 0.
template <int V>
__device__ __forceinline__ Vec<V> elu(const Vec<V> &z) {
  Vec<V> t = mul(z, kLog2e), n;
#pragma unroll
  for (int i = 0; i < V; ++i) t[i] = ex2(t[i]), n[i] = fminf(z[i], 0.0f);
  t = add(t, -1.0f);
  Vec<V> p = fma(n, 0.00680760853f, 0.0410424843f);
  p = fma(p, n, 0.1665636f);
  p = fma(p, n, 0.499994636f);
  p = fma(mul(n, n), p, z);
#pragma unroll
  for (int i = 0; i < V; ++i) t[i] = z[i] > -0.5f ? p[i] : t[i];
  return t;
}

// z becomes act(z), for U vectors at a time so that the branch is taken once for
// them.
template <int U, int V>
__device__ __forceinline__ void act_values(Vec<V> (&z)[U], int act) {
  if (act == ZRL_ACT_ELU) {
#pragma unroll
    for (int u = 0; u < U; ++u) z[u] = elu(z[u]);
  } else if (act == ZRL_ACT_SILU) {
#pragma unroll
    for (int u = 0; u < U; ++u) z[u] = mul(z[u], sigmoid(z[u]));
  } else if (act == ZRL_ACT_GELU) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      Vec<V> e;
      z[u] = mul(z[u], normal_cdf(z[u], e));
    }
  }
}
// z becomes act'(z).
template <int U, int V>
__device__ __forceinline__ void act_slopes(Vec<V> (&z)[U], int act) {
  if (act == ZRL_ACT_ELU) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const Vec<V> t = mul(z[u], kLog2e);
#pragma unroll
      for (int i = 0; i < V; ++i) z[u][i] = z[u][i] > 0.0f ? 1.0f : ex2(t[i]);
    }
  } else if (act == ZRL_ACT_SILU) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const Vec<V> t = sigmoid(z[u]);
      z[u] = fma(mul(z[u], t), fma(t, -1.0f, 1.0f), t);
    }
  } else if (act == ZRL_ACT_GELU) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      Vec<V> e;
      const Vec<V> p = normal_cdf(z[u], e);
      z[u] = fma(mul(z[u], 0.39894228f), e, p);
    }
  } else {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < V; ++i) z[u][i] = z[u][i] == z[u][i] ? 1.0f : z[u][i];
  }
}

// gamma or beta of V channels from p + at, or c where p is NULL; one access of
// 16 bytes for four where wide says that they are aligned.
template <int V>
__device__ __forceinline__ Vec<V> params(const float *p, int64_t at, float c, bool wide) {
  Vec<V> r = all<V>(c);
  if (!p) return r;
  if constexpr (V % 4 == 0) {
    if (wide) {
#pragma unroll
      for (int i = 0; i < V; i += 4) {
        const float4 f = *reinterpret_cast<const float4 *>(p + at + i);
        r[i] = f.x, r[i + 1] = f.y, r[i + 2] = f.z, r[i + 3] = f.w;
      }
      return r;
    }
  }
#pragma unroll
  for (int i = 0; i < V; ++i) r[i] = p[at + i];
  return r;
}

// Each v summed over the p (a power of two) neighbouring lanes of a group.
template <int U>
__device__ __forceinline__ void lanes_sum(float (&v)[U], int p) {
#pragma unroll
  for (int o = 16; o; o >>= 1)
    if (p > o) {
#pragma unroll
      for (int u = 0; u < U; ++u) v[u] += __shfl_xor_sync(0xffffffffu, v[u], o);
    }
}

extern __shared__ __align__(16) unsigned char norm_smem[];

}  // namespace
}  // namespace zrl
