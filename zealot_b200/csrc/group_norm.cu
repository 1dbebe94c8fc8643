// group_norm.cu -- group norm over channels-last rows with an activation, and
// its gradient.
//
// x [N, L, C], groups of w = C / G neighbouring channels; per (n, g), over
// L x w elements: mu, var, xh = (x - mu) / sqrt(var + eps); then
// y = act(gamma xh + beta).  Gradient, with dz = dy act'(z):
//   dbeta = sum dz, dgamma = sum dz xh,
//   dx = rstd (gamma dz - mean(gamma dz) - xh mean(gamma dz xh)).
//
// Two forms.  L = 1 and a group that fits the registers of a few lanes: one
// pass, a group's lanes next to one another in a warp (norm_rows_kernel,
// norm_rows_grad_kernel).  Else two passes over a sample, the second from L2
// where the samples of one launch fit there: sums per stretch of positions,
// then the outputs.
#include <math.h>

#include <algorithm>
#include <initializer_list>
#include <type_traits>

#include "column_sum.cuh"
#include "seq_common.cuh"

namespace zrl {
namespace {

constexpr int kThreads = 256;
constexpr int kSms = 148;
constexpr int64_t kBatchBytes = 48 << 20;

struct NormArgs {
  const void *x, *dy;
  const float *gamma, *beta;
  void *y, *dx;
  float *mean, *rstd, *part;
  int64_t N, L, sxn, sxl, syn, syl, sdn, sdl;  // strides of x, y / dy, dx
  int32_t C, G, w, act;
  float eps;
  // rows: lanes per group, groups of a block, rows of a block
  int32_t p, gb, rb;
  // samples: channels of a block at most, parts of a wide group, stretches of
  // positions, positions of one
  int32_t cols, parts, stretches;
  int64_t stretch;
};

__device__ __forceinline__ float ex2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float rcp(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
constexpr float kLog2e = 1.44269504f;

// act(z).  ELU's and SiLU's exponentials are absolute to 1e-7 of 1, as z itself
// is of max(1, |z|).
template <int V>
__device__ __forceinline__ void act_values(float *z, int act) {
  if (act == ZRL_ACT_ELU) {
#pragma unroll
    for (int i = 0; i < V; ++i) z[i] = z[i] > 0.0f ? z[i] : ex2(z[i] * kLog2e) - 1.0f;
  } else if (act == ZRL_ACT_SILU) {
#pragma unroll
    for (int i = 0; i < V; ++i) z[i] = z[i] * rcp(1.0f + ex2(z[i] * -kLog2e));
  } else if (act == ZRL_ACT_GELU) {
#pragma unroll
    for (int i = 0; i < V; ++i) z[i] = 0.5f * z[i] * (1.0f + erff(z[i] * 0.70710678f));
  }
}
// z becomes act'(z).
template <int V>
__device__ __forceinline__ void act_slopes(float *z, int act) {
  if (act == ZRL_ACT_ELU) {
#pragma unroll
    for (int i = 0; i < V; ++i) z[i] = z[i] > 0.0f ? 1.0f : ex2(z[i] * kLog2e);
  } else if (act == ZRL_ACT_SILU) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float s = rcp(1.0f + ex2(z[i] * -kLog2e));
      z[i] = fmaf(z[i] * s, 1.0f - s, s);
    }
  } else if (act == ZRL_ACT_GELU) {
#pragma unroll
    for (int i = 0; i < V; ++i)
      z[i] = 0.5f * (1.0f + erff(z[i] * 0.70710678f)) +
             z[i] * 0.39894228f * ex2(z[i] * z[i] * (-0.5f * kLog2e));
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) z[i] = z[i] == z[i] ? 1.0f : z[i];
  }
}

// Sum over the p (a power of two) neighbouring lanes of a group.
__device__ __forceinline__ float lanes_sum(float v, int p) {
  for (int o = p >> 1; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// A thread of the row form: E vectors of VEC channels of one group, the same
// ones in every row it meets, so its gammas and betas stay in registers.
template <typename T, int VEC, int E>
struct RowLanes {
  int r, g, first, step, w;  // row within the block, group, first channel in the group
  bool on;
  float ga[E][VEC], be[E][VEC];
  __device__ __forceinline__ explicit RowLanes(const NormArgs &a) {
    const int per_row = a.gb * a.p, tid = threadIdx.x;
    r = tid / per_row;
    const int rem = tid - r * per_row;
    g = blockIdx.y * a.gb + rem / a.p;
    first = (rem % a.p) * VEC;
    step = a.p * VEC;
    w = a.w;
    on = r < a.rb && g < a.G;
#pragma unroll
    for (int e = 0; e < E; ++e)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        ga[e][i] = has(e) && a.gamma ? a.gamma[channel(e) + i] : 1.0f;
        be[e][i] = has(e) && a.beta ? a.beta[channel(e) + i] : 0.0f;
      }
  }
  __device__ __forceinline__ bool has(int e) const { return on && first + e * step < w; }
  __device__ __forceinline__ int channel(int e) const { return g * w + first + e * step; }
};

// Mean and 1 / sd of U groups held in registers, centred sums.
template <typename T, int VEC, int E, int U>
__device__ __forceinline__ void row_stats(const RowLanes<T, VEC, E> &k, const float (*x)[E][VEC],
                                          int p, float inv, float eps, float *mu, float *rstd) {
#pragma unroll
  for (int u = 0; u < U; ++u) {
    float s = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (k.has(e))
#pragma unroll
        for (int i = 0; i < VEC; ++i) s += x[u][e][i];
    mu[u] = s;
  }
#pragma unroll
  for (int u = 0; u < U; ++u) mu[u] = lanes_sum(mu[u], p) * inv;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    float s = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (k.has(e))
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float d = x[u][e][i] - mu[u];
          s = fmaf(d, d, s);
        }
    rstd[u] = s;
  }
#pragma unroll
  for (int u = 0; u < U; ++u) rstd[u] = rsqrtf(lanes_sum(rstd[u], p) * inv + eps);
}

template <typename T, int VEC, int E>
__global__ void __launch_bounds__(kThreads) norm_rows_kernel(const __grid_constant__ NormArgs a) {
  constexpr int U = E == 1 ? 2 : 1;
  const RowLanes<T, VEC, E> k(a);
  const float inv = 1.0f / (float)a.w;
  for (int64_t n0 = (int64_t)blockIdx.x * a.rb * U; n0 < a.N; n0 += (int64_t)gridDim.x * a.rb * U) {
    float x[U][E][VEC], mu[U], rstd[U];
    Raw<T, VEC> raw[U][E];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t n = n0 + u * a.rb + k.r;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        raw[u][e] = Raw<T, VEC>{};
        if (n < a.N && k.has(e))
          raw[u][e] = *reinterpret_cast<const Raw<T, VEC> *>(static_cast<const T *>(a.x) +
                                                             n * a.sxn + k.channel(e));
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < E; ++e) unpack<T, VEC>(raw[u][e], x[u][e]);
    row_stats<T, VEC, E, U>(k, x, a.p, inv, a.eps, mu, rstd);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t n = n0 + u * a.rb + k.r;
      if (n >= a.N || !k.on) continue;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        if (!k.has(e)) continue;
        float z[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i)
          z[i] = fmaf((x[u][e][i] - mu[u]) * rstd[u], k.ga[e][i], k.be[e][i]);
        act_values<VEC>(z, a.act);
        store_vec<T, VEC>(static_cast<T *>(a.y) + n * a.syn + k.channel(e), z);
      }
      if (k.first == 0) {
        if (a.mean) a.mean[n * a.G + k.g] = mu[u];
        if (a.rstd) a.rstd[n * a.G + k.g] = rstd[u];
      }
    }
  }
}

// dx, and part[block][2][C]: the block's sums for dgamma and dbeta, kept in
// registers over all its rows.
template <typename T, int VEC, int E>
__global__ void __launch_bounds__(kThreads)
    norm_rows_grad_kernel(const __grid_constant__ NormArgs a) {
  __shared__ float buf[kThreads];
  const RowLanes<T, VEC, E> k(a);
  const float inv = 1.0f / (float)a.w;
  float dg[E][VEC] = {}, db[E][VEC] = {};
  for (int64_t n0 = (int64_t)blockIdx.x * a.rb; n0 < a.N; n0 += (int64_t)gridDim.x * a.rb) {
    const int64_t n = n0 + k.r;
    const bool on = n < a.N && k.on;
    float x[E][VEC], d[E][VEC];
    Raw<T, VEC> rx[E], rd[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      rx[e] = rd[e] = Raw<T, VEC>{};
      if (on && k.has(e)) {
        rx[e] = *reinterpret_cast<const Raw<T, VEC> *>(static_cast<const T *>(a.x) + n * a.sxn +
                                                       k.channel(e));
        rd[e] = *reinterpret_cast<const Raw<T, VEC> *>(static_cast<const T *>(a.dy) + n * a.syn +
                                                       k.channel(e));
      }
    }
    const float mu = on ? a.mean[n * a.G + k.g] : 0.0f, rstd = on ? a.rstd[n * a.G + k.g] : 0.0f;
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      unpack<T, VEC>(rx[e], x[e]);
      unpack<T, VEC>(rd[e], d[e]);
      if (!on || !k.has(e)) continue;
      float z[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        x[e][i] = (x[e][i] - mu) * rstd;
        z[i] = fmaf(x[e][i], k.ga[e][i], k.be[e][i]);
      }
      act_slopes<VEC>(z, a.act);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float dz = d[e][i] * z[i];
        db[e][i] += dz;
        dg[e][i] = fmaf(dz, x[e][i], dg[e][i]);
        d[e][i] = dz * k.ga[e][i];
        s1 += d[e][i];
        s2 = fmaf(d[e][i], x[e][i], s2);
      }
    }
    s1 = lanes_sum(s1, a.p) * inv;
    s2 = lanes_sum(s2, a.p) * inv;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (!on || !k.has(e)) continue;
#pragma unroll
      for (int i = 0; i < VEC; ++i) d[e][i] = rstd * (d[e][i] - fmaf(x[e][i], s2, s1));
      store_vec<T, VEC>(static_cast<T *>(a.dx) + n * a.sdn + k.channel(e), d[e]);
    }
  }
  // the rows of the block, in order
  const int per_row = a.gb * a.p;
#pragma unroll
  for (int e = 0; e < E; ++e)
#pragma unroll
    for (int i = 0; i < VEC; ++i)
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        __syncthreads();
        buf[threadIdx.x] = which ? db[e][i] : dg[e][i];
        __syncthreads();
        if (k.r == 0 && k.has(e)) {
          float s = 0.0f;
          for (int r = 0; r < a.rb; ++r) s += buf[r * per_row + threadIdx.x];
          a.part[((int64_t)blockIdx.x * 2 + which) * a.C + k.channel(e) + i] = s;
        }
      }
}

// ---------------------------------------------------------------- samples

// A block of the sample form: cols channels (whole groups, or a part of one
// wide group) by a stretch of positions of sample blockIdx.y; a thread has VEC
// channels of one group and every rows-th position.
template <int VEC>
struct Patch {
  int c0, width, lanes, rows, col, row, g0, groups, part, local;
  int64_t n, l0, l1;
  bool on;
  __device__ __forceinline__ explicit Patch(const NormArgs &a) {
    n = blockIdx.y;
    if (a.parts == 1) {
      const int per = a.cols / a.w;
      g0 = blockIdx.z * per;
      groups = min(per, a.G - g0);
      part = 0;
      c0 = g0 * a.w;
      width = groups * a.w;
    } else {
      g0 = blockIdx.z / a.parts;
      part = blockIdx.z - g0 * a.parts;
      groups = 1;
      c0 = g0 * a.w + part * a.cols;
      width = min(a.cols, a.w - part * a.cols);
    }
    lanes = width / VEC;
    rows = kThreads / lanes;
    row = threadIdx.x / lanes;
    col = threadIdx.x - row * lanes;
    on = row < rows;
    local = a.parts == 1 ? col * VEC / a.w : 0;  // group within the block
    l0 = blockIdx.x * a.stretch;
    l1 = min(a.L, l0 + a.stretch);
  }
  __device__ __forceinline__ int channel() const { return c0 + col * VEC; }
};

// For every group of the block the sum of v over its threads, in a fixed order:
// buf gets the threads' values, then a warp sums a lane column over the rows,
// then a thread the columns of its group.  out[group] in shared memory.
template <int VEC>
__device__ __forceinline__ void patch_sum(const NormArgs &a, const Patch<VEC> &k, float v,
                                          float *buf, float *cols, float *out) {
  __syncthreads();
  if (k.on) buf[threadIdx.x] = v;
  __syncthreads();
  const int lane = threadIdx.x & 31;
  for (int c = threadIdx.x >> 5; c < k.lanes; c += kThreads / 32) {
    float s = 0.0f;
    for (int r = lane; r < k.rows; r += 32) s += buf[r * k.lanes + c];
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) cols[c] = s;
  }
  __syncthreads();
  const int per = k.lanes / k.groups;
  for (int g = threadIdx.x; g < k.groups; g += kThreads) {
    float s = 0.0f;
    for (int c = 0; c < per; ++c) s += cols[g * per + c];
    out[g] = s;
  }
  __syncthreads();
}

// Sums over the pieces of a group (stretches x parts) by the warp, lanes in
// order: f(piece) summed.
template <typename F>
__device__ __forceinline__ float pieces_sum(int pieces, F f) {
  float s = 0.0f;
  for (int i = threadIdx.x & 31; i < pieces; i += 32) s += f(i);
#pragma unroll
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return s;
}

// First pass: part[n][group][piece] = (mean, sum of squares about it) of the
// block's piece.  A thread takes four positions at a time, centres them, and
// merges (count, mean, squares) with what it has.
template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads) norm_stats_kernel(const __grid_constant__ NormArgs a) {
  __shared__ float buf[kThreads], cols[kThreads], sums[kThreads];
  const Patch<VEC> k(a);
  constexpr int U = 4;
  float cnt = 0.0f, mean = 0.0f, m2 = 0.0f;
  if (k.on) {
    const T *x = static_cast<const T *>(a.x) + k.n * a.sxn + k.channel();
    int64_t l = k.l0 + k.row;
    auto merge = [&](float nb, float mb, float sb) {
      const float d = mb - mean, total = cnt + nb, share = nb * rcp(total);
      mean = fmaf(d, share, mean);
      m2 += fmaf(d * d * cnt, share, sb);
      cnt = total;
    };
    for (; l + (int64_t)(U - 1) * k.rows < k.l1; l += (int64_t)U * k.rows) {
      Raw<T, VEC> raw[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        raw[u] = *reinterpret_cast<const Raw<T, VEC> *>(x + (l + (int64_t)u * k.rows) * a.sxl);
      float v[U][VEC], s = 0.0f, q = 0.0f;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        unpack<T, VEC>(raw[u], v[u]);
#pragma unroll
        for (int i = 0; i < VEC; ++i) s += v[u][i];
      }
      s *= 1.0f / (U * VEC);
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float d = v[u][i] - s;
          q = fmaf(d, d, q);
        }
      merge((float)(U * VEC), s, q);
    }
    for (; l < k.l1; l += k.rows) {
      float v[VEC], s = 0.0f, q = 0.0f;
      load_vec<T, VEC>(x + l * a.sxl, v);
#pragma unroll
      for (int i = 0; i < VEC; ++i) s += v[i];
      s *= 1.0f / VEC;
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float d = v[i] - s;
        q = fmaf(d, d, q);
      }
      merge((float)VEC, s, q);
    }
  }
  const float n_piece =
      (float)(k.l1 - k.l0) * (float)(a.parts == 1 ? a.w : k.width);
  patch_sum(a, k, cnt * mean, buf, cols, sums);
  const float mu = sums[k.local] / n_piece;
  float mine = 0.0f;
  const int pieces = a.stretches * a.parts, piece = blockIdx.x * a.parts + k.part;
  if ((int)threadIdx.x < k.groups) mine = sums[threadIdx.x] / n_piece;
  const float d = mean - mu;
  patch_sum(a, k, fmaf(cnt * d, d, m2), buf, cols, sums);
  for (int g = threadIdx.x; g < k.groups; g += kThreads) {
    float *p = a.part + 2 * ((k.n * a.G + k.g0 + g) * pieces + piece);
    p[0] = mine;
    p[1] = sums[g];
  }
}

// Second pass: the pieces' means and squares give the group's, then y.
template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads) norm_apply_kernel(const __grid_constant__ NormArgs a) {
  __shared__ float smu[kThreads], srs[kThreads];
  const Patch<VEC> k(a);
  const int pieces = a.stretches * a.parts;
  for (int g = threadIdx.x >> 5; g < k.groups; g += kThreads / 32) {
    const int64_t ng = k.n * a.G + k.g0 + g;
    const float *p = a.part + 2 * ng * pieces;
    auto count = [&](int i) {
      const int64_t l0 = (int64_t)(i / a.parts) * a.stretch;
      const int c0 = (i % a.parts) * a.cols;
      return (float)(min(a.L, l0 + a.stretch) - l0) *
             (float)(a.parts == 1 ? a.w : min(a.cols, a.w - c0));
    };
    const float inv = 1.0f / ((float)a.L * (float)a.w);
    const float mu = pieces_sum(pieces, [&](int i) { return count(i) * p[2 * i]; }) * inv;
    const float var = pieces_sum(pieces, [&](int i) {
                        const float d = p[2 * i] - mu;
                        return fmaf(count(i) * d, d, p[2 * i + 1]);
                      }) * inv;
    if ((threadIdx.x & 31) == 0) {
      smu[g] = mu;
      srs[g] = rsqrtf(var + a.eps);
      if (blockIdx.x == 0 && k.part == 0) {
        if (a.mean) a.mean[ng] = mu;
        if (a.rstd) a.rstd[ng] = srs[g];
      }
    }
  }
  __syncthreads();
  if (!k.on) return;
  const float mu = smu[k.local], rstd = srs[k.local];
  float ga[VEC], be[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    ga[i] = a.gamma ? a.gamma[k.channel() + i] : 1.0f;
    be[i] = a.beta ? a.beta[k.channel() + i] : 0.0f;
  }
  const T *x = static_cast<const T *>(a.x) + k.n * a.sxn + k.channel();
  T *y = static_cast<T *>(a.y) + k.n * a.syn + k.channel();
  constexpr int U = 4;
  for (int64_t l = k.l0 + k.row; l < k.l1; l += (int64_t)U * k.rows) {
    Raw<T, VEC> raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t at = l + (int64_t)u * k.rows;
      if (at < k.l1) raw[u] = *reinterpret_cast<const Raw<T, VEC> *>(x + at * a.sxl);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t at = l + (int64_t)u * k.rows;
      if (at >= k.l1) break;
      float z[VEC];
      unpack<T, VEC>(raw[u], z);
#pragma unroll
      for (int i = 0; i < VEC; ++i) z[i] = fmaf((z[i] - mu) * rstd, ga[i], be[i]);
      act_values<VEC>(z, a.act);
      store_vec<T, VEC>(y + at * a.syl, z);
    }
  }
}

// Gradient, first pass: part[n][stretch][2][C], the sums of dz xh and dz of each
// channel over the block's positions.  They give dgamma and dbeta, and, with
// gamma over a group's channels, the two means of dx.
template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads)
    norm_grad_sums_kernel(const __grid_constant__ NormArgs a) {
  __shared__ float buf[kThreads];
  const Patch<VEC> k(a);
  float dg[VEC] = {}, db[VEC] = {};
  if (k.on) {
    const int64_t ng = k.n * a.G + k.g0 + k.local;
    const float mu = a.mean[ng], rstd = a.rstd[ng];
    float ga[VEC], be[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      ga[i] = a.gamma ? a.gamma[k.channel() + i] : 1.0f;
      be[i] = a.beta ? a.beta[k.channel() + i] : 0.0f;
    }
    const T *x = static_cast<const T *>(a.x) + k.n * a.sxn + k.channel();
    const T *dy = static_cast<const T *>(a.dy) + k.n * a.syn + k.channel();
    constexpr int U = 2;
    for (int64_t l = k.l0 + k.row; l < k.l1; l += (int64_t)U * k.rows) {
      Raw<T, VEC> rx[U], rd[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t at = l + (int64_t)u * k.rows;
        if (at < k.l1) {
          rx[u] = *reinterpret_cast<const Raw<T, VEC> *>(x + at * a.sxl);
          rd[u] = *reinterpret_cast<const Raw<T, VEC> *>(dy + at * a.syl);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (l + (int64_t)u * k.rows >= k.l1) break;
        float xh[VEC], d[VEC], z[VEC];
        unpack<T, VEC>(rx[u], xh);
        unpack<T, VEC>(rd[u], d);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          xh[i] = (xh[i] - mu) * rstd;
          z[i] = fmaf(xh[i], ga[i], be[i]);
        }
        act_slopes<VEC>(z, a.act);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float dz = d[i] * z[i];
          db[i] += dz;
          dg[i] = fmaf(dz, xh[i], dg[i]);
        }
      }
    }
  }
  float *p = a.part + (k.n * a.stretches + blockIdx.x) * 2 * a.C;
#pragma unroll
  for (int i = 0; i < VEC; ++i)
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      __syncthreads();
      if (k.on) buf[threadIdx.x] = which ? db[i] : dg[i];
      __syncthreads();
      if ((int)threadIdx.x < k.lanes) {
        float s = 0.0f;
        for (int r = 0; r < k.rows; ++r) s += buf[r * k.lanes + threadIdx.x];
        p[which * (int64_t)a.C + k.c0 + threadIdx.x * VEC + i] = s;
      }
    }
}

// Gradient, second pass: dx.
template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads)
    norm_grad_apply_kernel(const __grid_constant__ NormArgs a) {
  __shared__ float s1[kThreads], s2[kThreads];
  const Patch<VEC> k(a);
  const float inv = 1.0f / ((float)a.L * (float)a.w);
  for (int g = threadIdx.x >> 5; g < k.groups; g += kThreads / 32) {
    const int c0 = (k.g0 + g) * a.w;
    const float *p = a.part + k.n * a.stretches * 2 * a.C;
    const int items = a.stretches * a.w;
    const float m2 = pieces_sum(items, [&](int i) {
                       const int c = c0 + i % a.w;
                       return (a.gamma ? a.gamma[c] : 1.0f) * p[(int64_t)(i / a.w) * 2 * a.C + c];
                     }) * inv;
    const float m1 = pieces_sum(items, [&](int i) {
                       const int c = c0 + i % a.w;
                       return (a.gamma ? a.gamma[c] : 1.0f) *
                              p[((int64_t)(i / a.w) * 2 + 1) * a.C + c];
                     }) * inv;
    if ((threadIdx.x & 31) == 0) s1[g] = m1, s2[g] = m2;
  }
  __syncthreads();
  if (!k.on) return;
  const int64_t ng = k.n * a.G + k.g0 + k.local;
  const float mu = a.mean[ng], rstd = a.rstd[ng], m1 = s1[k.local], m2 = s2[k.local];
  float ga[VEC], be[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    ga[i] = a.gamma ? a.gamma[k.channel() + i] : 1.0f;
    be[i] = a.beta ? a.beta[k.channel() + i] : 0.0f;
  }
  const T *x = static_cast<const T *>(a.x) + k.n * a.sxn + k.channel();
  const T *dy = static_cast<const T *>(a.dy) + k.n * a.syn + k.channel();
  T *dx = static_cast<T *>(a.dx) + k.n * a.sdn + k.channel();
  constexpr int U = 2;
  for (int64_t l = k.l0 + k.row; l < k.l1; l += (int64_t)U * k.rows) {
    Raw<T, VEC> rx[U], rd[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t at = l + (int64_t)u * k.rows;
      if (at < k.l1) {
        rx[u] = *reinterpret_cast<const Raw<T, VEC> *>(x + at * a.sxl);
        rd[u] = *reinterpret_cast<const Raw<T, VEC> *>(dy + at * a.syl);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t at = l + (int64_t)u * k.rows;
      if (at >= k.l1) break;
      float xh[VEC], d[VEC], z[VEC];
      unpack<T, VEC>(rx[u], xh);
      unpack<T, VEC>(rd[u], d);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        xh[i] = (xh[i] - mu) * rstd;
        z[i] = fmaf(xh[i], ga[i], be[i]);
      }
      act_slopes<VEC>(z, a.act);
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        d[i] = rstd * (d[i] * z[i] * ga[i] - fmaf(xh[i], m2, m1));
      store_vec<T, VEC>(dx + at * a.sdl, d);
    }
  }
}

// No positions: the statistics of nothing, and parameter gradients of zero.
__global__ void norm_empty_kernel(float *mean, float *rstd, int64_t count, float eps) {
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= count) return;
  if (mean) mean[i] = 0.0f;
  if (rstd) rstd[i] = rsqrtf(eps);
}

// Columns of part: dgamma's C, then dbeta's.
struct ParamOut {
  float *dgamma, *dbeta;
  int64_t C;
  __device__ __forceinline__ void operator()(int64_t c, float sum) const {
    if (c < C) {
      if (dgamma) dgamma[c] = sum;
    } else if (dbeta) {
      dbeta[c - C] = sum;
    }
  }
};

// How a call is laid out.  VEC: the largest of 16 bytes, 4 bytes and one element
// that divides the group's width and that pointers and strides are aligned to.
// The row form takes a group on p lanes with E vectors each.  For vectors E = 1
// while 32 lanes are enough; single channels go by eight lanes first, which
// costs six shuffles for four channels instead of ten for one.
struct NormPlan {
  bool rows;
  int vec, E, p, gb, rb, blocks, across;  // row form
  int cols, parts, stretches, depth;      // sample form (depth: blocks over channels)
  int64_t stretch;
  int64_t batch;  // samples of one pair of launches
};

int vector_of(int es, int64_t w, bool aligned16, bool aligned4) {
  const int big = 16 / es, small = 4 / es;
  if (aligned16 && w % big == 0) return big;
  if (es == 2 && aligned4 && w % small == 0) return small;
  return 1;
}

NormPlan plan_norm(int64_t N, int64_t L, int64_t C, int32_t G, int vec, int es, bool grad) {
  NormPlan p{};
  p.vec = vec;
  const int64_t w = C / G, nv = w / vec;
  if (L == 1 && nv <= (vec == 1 ? 128 : 64)) {
    int64_t e = vec == 1 ? std::min<int64_t>(4, (nv + 7) / 8) : (nv + 31) / 32;
    p.E = e <= 1 ? 1 : e <= 2 ? 2 : 4;
    const int64_t need = (nv + p.E - 1) / p.E;
    p.p = 1;
    while (p.p < need) p.p *= 2;
    if (p.p <= 32) {
      p.rows = true;
      p.gb = (int)std::min<int64_t>(G, kThreads / p.p);
      p.rb = kThreads / (p.gb * p.p);
      p.across = (G + p.gb - 1) / p.gb;
      const int64_t blocks = (N + p.rb - 1) / p.rb;
      // the gradient's blocks each leave a row of sums, so they stay resident
      p.blocks = (int)std::max<int64_t>(
          1, std::min<int64_t>(blocks, (grad ? kSms * 4 : kSms * 8) / p.across));
      return p;
    }
  }
  const int64_t most = (int64_t)kThreads * vec;
  if (w <= most) {
    p.parts = 1;
    p.cols = (int)(std::min<int64_t>(most / w, G) * w);
    p.depth = (int)((G + p.cols / w - 1) / (p.cols / w));
  } else {
    p.parts = (int)((w + most - 1) / most);
    p.cols = (int)most;
    p.depth = G * p.parts;
  }
  // samples that stay in L2 between the two passes
  const int64_t bytes = std::max<int64_t>(1, L * C * es * (grad ? 2 : 1));
  p.batch = std::max<int64_t>(1, std::min<int64_t>({N, (int64_t)65535, kBatchBytes / bytes}));
  // stretches: enough blocks, and at least a few positions a thread
  const int64_t rows = std::max<int64_t>(1, kThreads / (p.cols / vec));
  const int64_t want = std::max<int64_t>(1, kSms * 8 / (p.batch * p.depth));
  const int64_t fit = std::max<int64_t>(1, L / (rows * 4));
  p.stretches = (int)std::max<int64_t>(1, std::min<int64_t>({want, fit, (int64_t)256}));
  p.stretch = (L + p.stretches - 1) / p.stretches;
  p.stretches = (int)((L + p.stretch - 1) / p.stretch);
  return p;
}

int64_t workspace_floats(const NormPlan &p, int64_t N, int64_t C, int32_t G, bool grad) {
  if (p.rows) return grad ? (int64_t)p.blocks * 2 * C : 0;
  if (grad) return N * p.stretches * 2 * C;
  return N * G * p.stretches * p.parts * 2;
}

template <typename F>
void with_vec(int32_t dtype, int vec, F &&f) {
  with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    if (vec * sizeof(T) == 16) f(t, std::integral_constant<int, 16 / (int)sizeof(T)>{});
    else if (vec == 1) f(t, std::integral_constant<int, 1>{});
    else if constexpr (sizeof(T) == 2) f(t, std::integral_constant<int, 2>{});
  });
}
template <int VEC, typename F>
void with_e(int E, F &&f) {
  if (E == 1) f(std::integral_constant<int, 1>{});
  else if (E == 2) f(std::integral_constant<int, 2>{});
  else if constexpr (VEC == 1) f(std::integral_constant<int, 4>{});
}

void use_plan(NormArgs &a, const NormPlan &p, void *workspace) {
  a.p = p.p;
  a.gb = p.gb;
  a.rb = p.rb;
  a.cols = p.cols;
  a.parts = p.parts;
  a.stretches = p.stretches;
  a.stretch = p.stretch;
  a.part = static_cast<float *>(workspace);
}

zrl_status check_norm(const char *what, int64_t N, int64_t L, int64_t C, int32_t groups,
                      int32_t dtype, int32_t act) {
  if (N < 0 || L < 0 || C < 0 || C > (int64_t)1 << 23)
    return seq_fail(ZRL_INVALID_ARG, "%s: N, L >= 0 and 0 <= C <= 2^23", what);
  if (groups < 1 || C % groups)
    return seq_fail(ZRL_INVALID_ARG, "%s: %lld channels in %d groups", what, (long long)C, groups);
  if (!dtype_ok(dtype)) return seq_fail(ZRL_INVALID_ARG, "%s: unknown dtype %d", what, dtype);
  if (act < ZRL_ACT_NONE || act > ZRL_ACT_GELU)
    return seq_fail(ZRL_INVALID_ARG, "%s: unknown activation %d", what, act);
  return ZRL_OK;
}

// The vector that the call's pointers and strides allow.
int vector_for(const NormArgs &a, int es, std::initializer_list<const void *> ptrs) {
  bool ok16 = true, ok4 = true;
  for (const void *p : ptrs) {
    ok16 = ok16 && aligned(p, 16);
    ok4 = ok4 && aligned(p, 4);
  }
  for (int64_t s : {a.sxn, a.sxl, a.syn, a.syl, a.sdn, a.sdl}) {
    ok16 = ok16 && s * es % 16 == 0;
    ok4 = ok4 && s * es % 4 == 0;
  }
  return vector_of(es, a.w, ok16, ok4);
}

// The arguments of the samples from n0 on.
NormArgs samples_from(NormArgs a, int64_t n0, int es) {
  auto move = [&](auto &p, int64_t elements) {
    if (p) p = (std::remove_reference_t<decltype(p)>)((char *)p + elements * es);
  };
  move(a.x, n0 * a.sxn);
  move(a.y, n0 * a.syn);
  move(a.dy, n0 * a.syn);
  move(a.dx, n0 * a.sdn);
  if (a.mean) a.mean += n0 * a.G;
  if (a.rstd) a.rstd += n0 * a.G;
  // sums per sample: the gradient's per stretch and channel, else per piece
  a.part += n0 * (a.dx ? (int64_t)a.stretches * 2 * a.C
                       : (int64_t)a.G * a.stretches * a.parts * 2);
  return a;
}

}  // namespace
}  // namespace zrl

using namespace zrl;

// The largest workspace any alignment of the tensors may ask for.
extern "C" int64_t zrl_group_norm_workspace(int64_t N, int64_t L, int64_t C, int32_t groups,
                                            int32_t grad) {
  if (N <= 0 || L <= 0 || C <= 0 || groups < 1 || C % groups) return 0;
  int64_t most = 0;
  for (int es = 2; es <= 4; es += 2)
    for (int vec : {16 / es, 4 / es, 1})
      if (C / groups % vec == 0)
        most = std::max(most, workspace_floats(plan_norm(N, L, C, groups, vec, es, grad != 0), N,
                                               C, groups, grad != 0));
  return most * (int64_t)sizeof(float);
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
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (L == 0) {
    norm_empty_kernel<<<(unsigned)((N * groups + 255) / 256), 256, 0, st>>>(mean, rstd,
                                                                            N * groups, eps);
    return seq_launched("group_norm");
  }
  const int vec = vector_for(a, es, {x, y});
  const NormPlan p = plan_norm(N, L, C, groups, vec, es, false);
  if (workspace_bytes < zrl_group_norm_workspace(N, L, C, groups, 0) || !aligned(workspace, 16) ||
      (!workspace && workspace_floats(p, N, C, groups, false)))
    return seq_fail(ZRL_INVALID_ARG, "group_norm: workspace too small or not aligned");
  use_plan(a, p, workspace);
  with_vec(dtype, vec, [&](auto t, auto v) {
    using T = decltype(t);
    constexpr int VEC = decltype(v)::value;
    if (p.rows) {
      with_e<VEC>(p.E, [&](auto e) {
        norm_rows_kernel<T, VEC, decltype(e)::value>
            <<<dim3((unsigned)p.blocks, (unsigned)p.across), kThreads, 0, st>>>(a);
      });
      return;
    }
    for (int64_t n0 = 0; n0 < N; n0 += p.batch) {
      const NormArgs b = samples_from(a, n0, es);
      const dim3 grid((unsigned)p.stretches, (unsigned)std::min(p.batch, N - n0),
                      (unsigned)p.depth);
      norm_stats_kernel<T, VEC><<<grid, kThreads, 0, st>>>(b);
      norm_apply_kernel<T, VEC><<<grid, kThreads, 0, st>>>(b);
    }
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
  if (N == 0 || L == 0) {  // no rows: the sums are zero
    launch_column_sum(nullptr, 0, 2 * C, ParamOut{dgamma, dbeta, C}, st);
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
  const int vec = vector_for(a, es, {x, dy, dx});
  const NormPlan p = plan_norm(N, L, C, groups, vec, es, true);
  use_plan(a, p, workspace);
  with_vec(dtype, vec, [&](auto t, auto v) {
    using T = decltype(t);
    constexpr int VEC = decltype(v)::value;
    if (p.rows) {
      with_e<VEC>(p.E, [&](auto e) {
        norm_rows_grad_kernel<T, VEC, decltype(e)::value>
            <<<dim3((unsigned)p.blocks, (unsigned)p.across), kThreads, 0, st>>>(a);
      });
      return;
    }
    for (int64_t n0 = 0; n0 < N; n0 += p.batch) {
      const NormArgs b = samples_from(a, n0, es);
      const dim3 grid((unsigned)p.stretches, (unsigned)std::min(p.batch, N - n0),
                      (unsigned)p.depth);
      norm_grad_sums_kernel<T, VEC><<<grid, kThreads, 0, st>>>(b);
      norm_grad_apply_kernel<T, VEC><<<grid, kThreads, 0, st>>>(b);
    }
  });
  const int64_t sums = p.rows ? p.blocks : N * p.stretches;
  launch_column_sum(a.part, sums, 2 * C, ParamOut{dgamma, dbeta, C}, st);
  return seq_launched("group_norm_grad");
}
