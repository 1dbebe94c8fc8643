// group_norm_samples.cuh -- group norm of samples with several positions.
//
// A thread has VEC neighbouring channels and every rows-th position of a
// stretch, and keeps sums per channel, so that vectors need not end where groups
// do; a block then sums the channels of its groups.  Where a block's columns of
// a whole sample fit its shared memory, that is one pass (norm_block_kernel,
// norm_block_grad_kernel); else two, the second from L2 where the samples of one
// pair of launches fit there.
#pragma once

#include "group_norm.cuh"

namespace zrl {
namespace {

// Channels a thread has at most, and blocks an SM holds, which bounds their
// registers: eight channels at two blocks are as fast within a tenth (64 x 5046 x
// 64 f16 forward 28 and 28 us, 16 x 6360 x 256 bf16 GELU with gradient 124 and 126),
// two channels at six blocks slower (36 and 156).
constexpr int kMaxChannels = 4;
constexpr int sample_blocks(bool grad) { return grad ? 3 : 4; }

// A block's channels (whole groups, or a part of one wide group) and positions.
template <int VEC>
struct Patch {
  int c0, width, lanes, rows, col, row, g0, groups, part, per;  // per: channels of a group here
  int64_t n, l0, l1;
  bool on;
  __device__ __forceinline__ explicit Patch(const NormArgs &a) {
    n = blockIdx.y;
    if (a.parts == 1) {
      const int most = a.cols / a.w;
      g0 = blockIdx.z * most;
      groups = min(most, a.G - g0);
      part = 0;
      c0 = g0 * a.w;
      width = groups * a.w;
      per = a.w;
    } else {
      g0 = blockIdx.z / a.parts;
      part = blockIdx.z - g0 * a.parts;
      groups = 1;
      c0 = g0 * a.w + part * a.cols;
      width = min(a.cols, a.w - part * a.cols);
      per = width;
    }
    lanes = width / VEC;
    rows = kThreads / lanes;
    row = threadIdx.x / lanes;
    col = threadIdx.x - row * lanes;
    on = row < rows;
    l0 = blockIdx.x * a.stretch;
    l1 = min(a.L, l0 + a.stretch);
  }
  __device__ __forceinline__ int channel() const { return on ? c0 + col * VEC : 0; }
  // f(channel group) for each of the thread's channels, from shared memory
  __device__ __forceinline__ Vec<VEC> of_groups(const float *f) const {
    Vec<VEC> r;
    int g = on ? col * VEC / per : 0, left = on ? (g + 1) * per - col * VEC : VEC;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      if (left == 0) ++g, left = per;
      r[i] = f[g];
      --left;
    }
    return r;
  }
};

// out[group] = the sum of v over the group's channels and the block's threads, in
// a fixed order; buf holds a value per thread and channel.
template <int VEC>
__device__ __forceinline__ void group_sums(const Patch<VEC> &k, const Vec<VEC> &v, float *buf,
                                           float *out) {
  __syncthreads();
  if (k.on)
#pragma unroll
    for (int i = 0; i < VEC; ++i) buf[k.row * k.width + k.col * VEC + i] = v[i];
  __syncthreads();
  const int count = k.per * k.rows;
  if (count <= 8) {  // many narrow groups: a thread each
    for (int g = threadIdx.x; g < k.groups; g += kThreads) {
      float s = 0.0f;
      for (int r = 0; r < k.rows; ++r)
        for (int c = 0; c < k.per; ++c) s += buf[r * k.width + g * k.per + c];
      out[g] = s;
    }
  } else {
    const int lane = threadIdx.x & 31;
    for (int g = threadIdx.x >> 5; g < k.groups; g += kThreads / 32) {
      float s = 0.0f;
      for (int i = lane; i < count; i += 32) {
        const int r = i / k.per;
        s += buf[r * k.width + g * k.per + (i - r * k.per)];
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      if (lane == 0) out[g] = s;
    }
  }
  __syncthreads();
}

// out[channel] = the sum of v over the block's rows of threads, in order.
template <int VEC>
__device__ __forceinline__ void channel_sums(const Patch<VEC> &k, const Vec<VEC> &v, float *buf,
                                             float *out) {
  __syncthreads();
  if (k.on)
#pragma unroll
    for (int i = 0; i < VEC; ++i) buf[k.row * k.width + k.col * VEC + i] = v[i];
  __syncthreads();
  for (int c = threadIdx.x; c < k.width; c += kThreads) {
    float s = 0.0f;
    for (int r = 0; r < k.rows; ++r) s += buf[r * k.width + c];
    out[c] = s;
  }
}

// f(group, sum1, sum2) with the sums of x(piece), y(piece) over the pieces of each
// group of the block: by warps, lanes in order, or by threads where there are few
// pieces.
template <int VEC, typename X, typename F>
__device__ __forceinline__ void pieces_sums(const Patch<VEC> &k, int pieces, X x, F f) {
  if (pieces <= 4) {
    for (int g = threadIdx.x; g < k.groups; g += kThreads) {
      float s = 0.0f;
      for (int i = 0; i < pieces; ++i) s += x(g, i);
      f(g, s);
    }
  } else {
    const int lane = threadIdx.x & 31;
    for (int g = threadIdx.x >> 5; g < k.groups; g += kThreads / 32) {
      float s = 0.0f;
      for (int i = lane; i < pieces; i += 32) s += x(g, i);
#pragma unroll
      for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      if (lane == 0) f(g, s);
    }
  }
}

// (count, mean, squares about the mean) per channel of what a thread has seen; a
// batch of positions is centred, then merged.
template <int VEC>
struct Spread {
  float cnt = 0.0f;
  Vec<VEC> mean = all<VEC>(0.0f), m2 = mean;
  template <int U>
  __device__ __forceinline__ void take(Vec<VEC> (&v)[U]) {
    Vec<VEC> s = v[0], q = all<VEC>(0.0f);
#pragma unroll
    for (int u = 1; u < U; ++u) s = add(s, v[u]);
    s = mul(s, 1.0f / U);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      v[u] = add(v[u], mul(s, -1.0f));
      q = fma(v[u], v[u], q);
    }
    const float total = cnt + U, share = U * rcp(total);
    const Vec<VEC> d = add(s, mul(mean, -1.0f));
    mean = fma(d, share, mean);
    m2 = add(m2, fma(mul(d, d), cnt * share, q));
    cnt = total;
  }
  // the values of a turn of each_position
  template <typename T, int U, typename R>
  __device__ __forceinline__ void take_turn(const Raw<T, VEC> (&raw)[U][1], int count, R reload) {
    Vec<VEC> v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = values<T, VEC>(raw[u][0]);
    reload();
    if (count == U) {
      take(v);
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (u >= count) break;
        Vec<VEC> one[1] = {v[u]};
        take(one);
      }
    }
  }
};

// A thread's places in one tensor: its channels at its first position, and the
// bytes from one of its positions to the next.
template <typename T>
struct Run {
  T *p;
  int64_t step;
  template <int VEC>
  __device__ __forceinline__ Run(const void *base, const Patch<VEC> &k, int64_t sn, int64_t sl)
      : p(const_cast<T *>(static_cast<const T *>(base)) + k.n * sn + (k.l0 + k.row) * sl +
          k.channel()),
        step(k.rows * sl * (int64_t)sizeof(T)) {}
  __device__ __forceinline__ void next() { p = (T *)((char *)p + step); }
};

// f(raw, count, reload) over the thread's positions, U at a time (count of them in
// the last turn); f calls reload() when it is done with raw, so that the next
// ones' loads are in flight while it works.
template <int U, typename T, int VEC, int TENSORS, typename F>
__device__ __forceinline__ void each_position(const Patch<VEC> &k, Run<T> (&x)[TENSORS], F f) {
  Raw<T, VEC> raw[U][TENSORS];
  int left = k.on ? (int)((k.l1 - k.l0 - k.row + k.rows - 1) / k.rows) : 0;
  auto load = [&](int n) {
    if (n >= U) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < TENSORS; ++i) {
          raw[u][i] = *reinterpret_cast<const Raw<T, VEC> *>(x[i].p);
          x[i].next();
        }
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (u < n)
#pragma unroll
          for (int i = 0; i < TENSORS; ++i) {
            raw[u][i] = *reinterpret_cast<const Raw<T, VEC> *>(x[i].p);
            x[i].next();
          }
    }
  };
  load(left);
  for (; left > 0; left -= U) f(raw, min(left, U), [&]() { load(left - U); });
}

template <typename T, int VEC>
using Sums = float[kThreads * VEC];  // a value per thread and channel, or per group

// mu[group], m2[group]: mean and squares about it of the block's n_piece elements
// of each group.
template <int VEC>
__device__ __forceinline__ void block_spread(const Patch<VEC> &k, const Spread<VEC> &t,
                                             float n_piece, float *buf, float *mu, float *m2) {
  group_sums(k, mul(t.mean, t.cnt), buf, mu);
  for (int g = threadIdx.x; g < k.groups; g += kThreads) mu[g] /= n_piece;
  __syncthreads();
  const Vec<VEC> d = add(t.mean, mul(k.of_groups(mu), -1.0f));
  group_sums(k, fma(mul(d, d), t.cnt, t.m2), buf, m2);
}

// First pass: part[n][group][piece] = (mean, squares about it) of the block's
// piece.  64 x 5046 x 64 f16 14 us (2.9 TB/s): a block lives for 15 turns, its ramp and
// its sums are a third of that.
template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads, sample_blocks(false))
    norm_stats_kernel(const __grid_constant__ NormArgs a) {
  __shared__ Sums<T, VEC> buf, mu, m2;
  const Patch<VEC> k(a);
  Spread<VEC> t;
  Run<T> x[1] = {Run<T>(a.x, k, a.sxn, a.sxl)};
  each_position<4, T, VEC, 1>(k, x, [&](Raw<T, VEC>(&raw)[4][1], int count, auto reload) {
    t.template take_turn<T, 4>(raw, count, reload);
  });
  let_next_start();
  block_spread(k, t, (float)(k.l1 - k.l0) * (float)k.per, buf, mu, m2);
  const int pieces = a.stretches * a.parts, piece = blockIdx.x * a.parts + k.part;
  float2 *p = reinterpret_cast<float2 *>(a.part);
  for (int g = threadIdx.x; g < k.groups; g += kThreads)
    p[(k.n * a.G + k.g0 + g) * pieces + piece] = make_float2(mu[g], m2[g]);
}

// y = act((x - mu) gamma rstd + beta) of a position
template <int VEC>
struct Scale {
  Vec<VEC> mu, gr, be;
  __device__ __forceinline__ Scale(const NormArgs &a, const Patch<VEC> &k, const float *mean,
                                   const float *rstd) {
    mu = mul(k.of_groups(mean), -1.0f);
    gr = mul(params<VEC>(a.gamma, k.channel(), 1.0f, a.wide), k.of_groups(rstd));
    be = params<VEC>(a.beta, k.channel(), 0.0f, a.wide);
  }
  template <typename T>
  __device__ __forceinline__ void write(const Vec<VEC> &x, int act, T *y) const {
    Vec<VEC> z = fma(add(x, mu), gr, be);
    act_values<VEC>(z, act);
    store_vec<T, VEC>(y, z.v);
  }
};

// Second pass: the pieces' means and squares give the group's, then y.  64 x 5046 x
// 64 f16 ELU 14 us, 16 x 6360 x 256 bf16 GELU 31 us (26 issue slots a value).
template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads, sample_blocks(false))
    norm_apply_kernel(const __grid_constant__ NormArgs a) {
  __shared__ Sums<T, VEC> mean, rstd;
  const Patch<VEC> k(a);
  const int pieces = a.stretches * a.parts;
  const float2 *p = reinterpret_cast<const float2 *>(a.part) + (k.n * a.G + k.g0) * pieces;
  const float inv = 1.0f / ((float)a.L * (float)a.w);
  auto count = [&](int i) {
    const int64_t l0 = (int64_t)(i / a.parts) * a.stretch;
    const int c0 = (i % a.parts) * a.cols;
    return (float)(min(a.L, l0 + a.stretch) - l0) *
           (float)(a.parts == 1 ? a.w : min(a.cols, a.w - c0));
  };
  wait_for_previous();
  pieces_sums(k, pieces, [&](int g, int i) { return count(i) * p[g * pieces + i].x; },
              [&](int g, float s) { mean[g] = s * inv; });
  __syncthreads();
  pieces_sums(k, pieces,
              [&](int g, int i) {
                const float2 f = p[g * pieces + i];
                const float d = f.x - mean[g];
                return fmaf(count(i) * d, d, f.y);
              },
              [&](int g, float s) {
                rstd[g] = rsqrtf(fmaf(s, inv, a.eps));
                if (blockIdx.x == 0 && k.part == 0) {
                  if (a.mean) a.mean[k.n * a.G + k.g0 + g] = mean[g];
                  if (a.rstd) a.rstd[k.n * a.G + k.g0 + g] = rstd[g];
                }
              });
  __syncthreads();
  if (!k.on) return;
  const Scale<VEC> scale(a, k, mean, rstd);
  Run<T> x[1] = {Run<T>(a.x, k, a.sxn, a.sxl)}, y(a.y, k, a.syn, a.syl);
  each_position<4, T, VEC, 1>(k, x, [&](Raw<T, VEC>(&raw)[4][1], int count, auto reload) {
    Vec<VEC> v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) v[u] = values<T, VEC>(raw[u][0]);
    reload();
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (u >= count) break;
      scale.write(v[u], a.act, y.p);
      y.next();
    }
  });
}

// xh = (x - mu) rstd and dz = dy act'(gamma xh + beta) of a position
template <int VEC>
struct Slope {
  Vec<VEC> mu, rs, ga, be;
  __device__ __forceinline__ Slope(const NormArgs &a, const Patch<VEC> &k) {
    int g = k.on ? k.col * VEC / k.per : 0, left = k.on ? (g + 1) * k.per - k.col * VEC : VEC;
    const int64_t ng = k.n * a.G + k.g0;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      if (left == 0) ++g, left = k.per;
      mu[i] = -a.mean[ng + g];
      rs[i] = a.rstd[ng + g];
      --left;
    }
    ga = params<VEC>(a.gamma, k.channel(), 1.0f, a.wide);
    be = params<VEC>(a.beta, k.channel(), 0.0f, a.wide);
  }
  __device__ __forceinline__ Vec<VEC> dz(const Vec<VEC> &x, const Vec<VEC> &dy, int act,
                                         Vec<VEC> &xh) const {
    xh = mul(add(x, mu), rs);
    Vec<VEC> z = fma(xh, ga, be);
    act_slopes<VEC>(z, act);
    return mul(dy, z);
  }
};

// part[n][stretch][2][C]: the sums of dz xh and dz of each channel over the
// block's positions, for dgamma and dbeta; s1, s2[group]: the sums of gamma dz and
// gamma dz xh.
template <int VEC>
__device__ __forceinline__ void grad_sums(const NormArgs &a, const Patch<VEC> &k,
                                          const Vec<VEC> &dg, const Vec<VEC> &db,
                                          const Vec<VEC> &ga, float *buf, float *s1, float *s2) {
  float *p = a.part + (k.n * a.stretches + blockIdx.x) * 2 * a.C + k.c0;
  channel_sums(k, dg, buf, p);
  channel_sums(k, db, buf, p + a.C);
  group_sums(k, mul(db, ga), buf, s1);
  group_sums(k, mul(dg, ga), buf, s2);
}

// Gradient, first pass: grad_sums, the groups' into means[n][group][piece].  16 x
// 6360 x 256 bf16 GELU 35 us (3.0 TB/s); 26 issue slots a value.
template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads, sample_blocks(true))
    norm_grad_sums_kernel(const __grid_constant__ NormArgs a) {
  __shared__ Sums<T, VEC> buf, s1, s2;
  const Patch<VEC> k(a);
  Vec<VEC> dg = all<VEC>(0.0f), db = dg;
  const Slope<VEC> slope(a, k);
  Run<T> xs[2] = {Run<T>(a.x, k, a.sxn, a.sxl), Run<T>(a.dy, k, a.syn, a.syl)};
  each_position<2, T, VEC, 2>(k, xs, [&](Raw<T, VEC>(&raw)[2][2], int count, auto reload) {
    Vec<VEC> x[2], d[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) x[u] = values<T, VEC>(raw[u][0]), d[u] = values<T, VEC>(raw[u][1]);
    reload();
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if (u >= count) break;
      Vec<VEC> xh;
      const Vec<VEC> dz = slope.dz(x[u], d[u], a.act, xh);
      db = add(db, dz);
      dg = fma(dz, xh, dg);
    }
  });
  let_next_start();
  grad_sums(a, k, dg, db, slope.ga, buf, s1, s2);
  const int pieces = a.stretches * a.parts, piece = blockIdx.x * a.parts + k.part;
  for (int g = threadIdx.x; g < k.groups; g += kThreads)
    a.means[(k.n * a.G + k.g0 + g) * pieces + piece] = make_float2(s1[g], s2[g]);
}

// dx = rstd (gamma dz - m1 - xh m2) of a position; m1 and m2 come times rstd
template <int VEC, typename T>
__device__ __forceinline__ void write_dx(const Slope<VEC> &slope, const Vec<VEC> &m1,
                                         const Vec<VEC> &m2, const Vec<VEC> &x,
                                         const Vec<VEC> &dy, int act, T *dx) {
  Vec<VEC> xh;
  const Vec<VEC> dz = slope.dz(x, dy, act, xh);
  const Vec<VEC> o = fma(mul(dz, slope.ga), slope.rs, mul(fma(xh, m2, m1), -1.0f));
  store_vec<T, VEC>(dx, o.v);
}

// Gradient, second pass: dx.  As the first 39 us.
template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads, sample_blocks(true))
    norm_grad_apply_kernel(const __grid_constant__ NormArgs a) {
  __shared__ Sums<T, VEC> s1, s2;
  const Patch<VEC> k(a);
  const int pieces = a.stretches * a.parts;
  const float2 *p = a.means + (k.n * a.G + k.g0) * pieces;
  wait_for_previous();
  pieces_sums(k, pieces, [&](int g, int i) { return p[g * pieces + i].x; },
              [&](int g, float s) { s1[g] = s; });
  pieces_sums(k, pieces, [&](int g, int i) { return p[g * pieces + i].y; },
              [&](int g, float s) { s2[g] = s; });
  __syncthreads();
  if (!k.on) return;
  const Slope<VEC> slope(a, k);
  const float inv = 1.0f / ((float)a.L * (float)a.w);
  const Vec<VEC> m1 = mul(mul(k.of_groups(s1), inv), slope.rs);
  const Vec<VEC> m2 = mul(mul(k.of_groups(s2), inv), slope.rs);
  Run<T> xs[2] = {Run<T>(a.x, k, a.sxn, a.sxl), Run<T>(a.dy, k, a.syn, a.syl)};
  Run<T> dx(a.dx, k, a.sdn, a.sdl);
  each_position<2, T, VEC, 2>(k, xs, [&](Raw<T, VEC>(&raw)[2][2], int count, auto reload) {
    Vec<VEC> x[2], d[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) x[u] = values<T, VEC>(raw[u][0]), d[u] = values<T, VEC>(raw[u][1]);
    reload();
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if (u >= count) break;
      write_dx(slope, m1, m2, x[u], d[u], a.act, dx.p);
      dx.next();
    }
  });
  let_next_start();
}

// ------------------------------------------------ samples held by a block

// The block keeps what it read in shared memory; a thread reads back only its
// own.  200 x 300 x 96 bf16 11 us (2.1 TB/s), latency of one turn of the blocks.
// Clusters of up to 16 blocks that held larger samples together and exchanged sums
// took 34 us for 64 x 5046 x 64 f16, where two passes take 28.
template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads, sample_blocks(false))
    norm_block_kernel(const __grid_constant__ NormArgs a) {
  __shared__ Sums<T, VEC> buf, mu, m2;
  const Patch<VEC> k(a);
  Raw<T, VEC> *kept = reinterpret_cast<Raw<T, VEC> *>(norm_smem) + threadIdx.x;
  Spread<VEC> t;
  Run<T> x[1] = {Run<T>(a.x, k, a.sxn, a.sxl)};
  int slot = 0;
  each_position<4, T, VEC, 1>(k, x, [&](Raw<T, VEC>(&raw)[4][1], int count, auto reload) {
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (u < count) kept[slot++ * kThreads] = raw[u][0];
    t.template take_turn<T, 4>(raw, count, reload);
  });
  const float n_el = (float)a.L * (float)a.w;
  block_spread(k, t, n_el, buf, mu, m2);
  for (int g = threadIdx.x; g < k.groups; g += kThreads) {
    const float rstd = rsqrtf(m2[g] / n_el + a.eps);
    m2[g] = rstd;
    if (a.mean) a.mean[k.n * a.G + k.g0 + g] = mu[g];
    if (a.rstd) a.rstd[k.n * a.G + k.g0 + g] = rstd;
  }
  __syncthreads();
  if (!k.on) return;
  const Scale<VEC> scale(a, k, mu, m2);
  Run<T> y(a.y, k, a.syn, a.syl);
  for (int i = 0; i < slot; ++i, y.next())
    scale.write(values<T, VEC>(kept[i * kThreads]), a.act, y.p);
}

template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads, sample_blocks(true))
    norm_block_grad_kernel(const __grid_constant__ NormArgs a) {
  __shared__ Sums<T, VEC> buf, s1, s2;
  const Patch<VEC> k(a);
  Raw<T, VEC> *kept = reinterpret_cast<Raw<T, VEC> *>(norm_smem) + threadIdx.x;
  Vec<VEC> dg = all<VEC>(0.0f), db = dg;
  const Slope<VEC> slope(a, k);
  Run<T> xs[2] = {Run<T>(a.x, k, a.sxn, a.sxl), Run<T>(a.dy, k, a.syn, a.syl)};
  int slot = 0;
  each_position<2, T, VEC, 2>(k, xs, [&](Raw<T, VEC>(&raw)[2][2], int count, auto reload) {
    Vec<VEC> x[2], d[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      x[u] = values<T, VEC>(raw[u][0]), d[u] = values<T, VEC>(raw[u][1]);
      if (u < count) {
        kept[2 * slot * kThreads] = raw[u][0];
        kept[(2 * slot++ + 1) * kThreads] = raw[u][1];
      }
    }
    reload();
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if (u >= count) break;
      Vec<VEC> xh;
      const Vec<VEC> dz = slope.dz(x[u], d[u], a.act, xh);
      db = add(db, dz);
      dg = fma(dz, xh, dg);
    }
  });
  let_next_start();
  grad_sums(a, k, dg, db, slope.ga, buf, s1, s2);
  if (!k.on) return;
  const float inv = 1.0f / ((float)a.L * (float)a.w);
  const Vec<VEC> m1 = mul(mul(k.of_groups(s1), inv), slope.rs);
  const Vec<VEC> m2 = mul(mul(k.of_groups(s2), inv), slope.rs);
  Run<T> dx(a.dx, k, a.sdn, a.sdl);
  for (int i = 0; i < slot; ++i, dx.next())
    write_dx(slope, m1, m2, values<T, VEC>(kept[2 * i * kThreads]),
             values<T, VEC>(kept[(2 * i + 1) * kThreads]), a.act, dx.p);
}

}  // namespace
}  // namespace zrl
