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
// 64 f16 forward 28 and 28 us, 16 x 6360 x 256 bf16 GELU with gradient 124 and 126,
// before the blocks' sums were taken by teams), two channels at six blocks slower
// (36 and 156).
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

// f(i, lane, t, lead) for each i < n (groups, channels): t (a power of two)
// neighbouring lanes of a warp, lane 0 to t - 1; lead for one of them.  Lanes with no
// i of their own come along for the shuffles, with a lane beyond any loop.  As
// many lanes as let all be taken at once: with a warp a group, one after the
// other, and the first loads after them, the second pass of 16 x 6360 x 256 took
// 34 us instead of 27.
template <typename F>
__device__ __forceinline__ void each_team(int n, F f) {
  int shift = 5;
  while (shift && (n << shift) > kThreads) --shift;
  const int t = 1 << shift, lane = threadIdx.x & (t - 1);
  for (int first = 0; first < n; first += kThreads >> shift) {
    const int i = first + ((int)threadIdx.x >> shift);
    f(min(i, n - 1), i < n ? lane : 1 << 30, t, i < n && lane == 0);
  }
}
__device__ __forceinline__ float team_sum(float v, int t) {
  for (int o = t >> 1; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <int VEC>
using Pairs = float2[kThreads * VEC];  // a pair per thread and channel

// buf[row][channel] = (a, b) of the block's rows of threads.
template <int VEC>
__device__ __forceinline__ void leave_pairs(const Patch<VEC> &k, const Vec<VEC> &a,
                                            const Vec<VEC> &b, float2 *buf) {
  if (k.on)
#pragma unroll
    for (int i = 0; i < VEC; ++i) buf[k.row * k.width + k.col * VEC + i] = make_float2(a[i], b[i]);
  __syncthreads();
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

struct Nothing {
  __device__ __forceinline__ void operator()() const {}
};
// f(raw, count, reload) over the thread's positions, U at a time (count of them in
// the last turn; after them the first one's x again, whose (x - mean) rstd is as
// finite as the data, and zeros for dy); f calls reload() when it is done with raw, so that the next
// ones' loads are in flight while it works.  meanwhile() runs once, by all
// threads, when the first loads are on their way.
template <int U, typename T, int VEC, int TENSORS, typename M, typename F>
__device__ __forceinline__ void each_position(const Patch<VEC> &k, Run<T> (&x)[TENSORS],
                                              M meanwhile, F f) {
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
#pragma unroll
        for (int i = 0; i < TENSORS; ++i) {
          raw[u][i] = i == 0 && u > 0 ? raw[0][0] : Raw<T, VEC>{};
          if (u < n) {
            raw[u][i] = *reinterpret_cast<const Raw<T, VEC> *>(x[i].p);
            x[i].next();
          }
        }
    }
  };
  load(left);
  meanwhile();
  for (; left > 0; left -= U) f(raw, min(left, U), [&]() { load(left - U); });
}

// done(group, mean, squares about it) of the block's elements of each group:
// channel by channel over the rows of threads, then over the group's channels.
template <int VEC, typename F>
__device__ __forceinline__ void block_spread(const Patch<VEC> &k, const Spread<VEC> &t,
                                             float2 *buf, F done) {
  const int positions = (int)(k.l1 - k.l0);
  leave_pairs(k, t.mean, t.m2, buf);
  const int turns = positions / k.rows, more = positions - turns * k.rows;
  auto count = [&](int r) { return (float)(turns + (r < more)); };
  each_team(k.width, [&](int c, int lane, int team, bool lead) {
    float mean = 0.0f, m2 = 0.0f;
#pragma unroll 4
    for (int r = lane; r < k.rows; r += team) mean = fmaf(count(r), buf[r * k.width + c].x, mean);
    mean = team_sum(mean, team) / positions;
#pragma unroll 4
    for (int r = lane; r < k.rows; r += team) {
      const float2 f = buf[r * k.width + c];
      m2 += fmaf(count(r) * (f.x - mean), f.x - mean, f.y);
    }
    m2 = team_sum(m2, team);
    if (lead) buf[c] = make_float2(mean, m2);  // only this team reads the column
  });
  __syncthreads();
  each_team(k.groups, [&](int g, int lane, int team, bool lead) {
    const float2 *f = buf + g * k.per;
    float mean = 0.0f, m2 = 0.0f;
    for (int c = lane; c < k.per; c += team) mean += f[c].x;
    mean = team_sum(mean, team) / k.per;
    for (int c = lane; c < k.per; c += team)
      m2 += fmaf(positions * (f[c].x - mean), f[c].x - mean, f[c].y);
    m2 = team_sum(m2, team);
    if (lead) done(g, mean, m2);
  });
}

// Positions of a turn of the first pass: six take 13.3 us at 64 x 5046 x 64 f16, four
// 14.1; fp32's spill.
template <typename T> constexpr int kTurn = sizeof(T) == 2 ? 6 : 4;

// First pass: part[n][group][piece] = (mean, squares about it) of the block's
// piece.  64 x 5046 x 64 f16 13 us (3.1 TB/s), 16 x 6360 x 256 bf16 16 us: a block lives
// for ten turns, its ramp and its sums are a quarter of that.
template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads, sample_blocks(false))
    norm_stats_kernel(const __grid_constant__ NormArgs a) {
  __shared__ Pairs<VEC> buf;
  const Patch<VEC> k(a);
  Spread<VEC> t;
  Run<T> x[1] = {Run<T>(a.x, k, a.sxn, a.sxl)};
  each_position<kTurn<T>, T, VEC, 1>(k, x, Nothing{}, [&](Raw<T, VEC>(&raw)[kTurn<T>][1], int count, auto reload) {
    t.template take_turn<T, kTurn<T>>(raw, count, reload);
  });
  let_next_start();
  const int pieces = a.stretches * a.parts, piece = blockIdx.x * a.parts + k.part;
  float2 *p = reinterpret_cast<float2 *>(a.part) + (k.n * a.G + k.g0) * pieces + piece;
  block_spread(k, t, buf, [&](int g, float mean, float m2) {
    p[g * pieces] = make_float2(mean, m2);
  });
}

// y = act((x - mu) gamma rstd + beta) of a position
template <int VEC>
struct Scale {
  Vec<VEC> mu, gr, be;
  Scale() = default;
  __device__ __forceinline__ Scale(const NormArgs &a, const Patch<VEC> &k, const float *mean,
                                   const float *rstd) {
    mu = mul(k.of_groups(mean), -1.0f);
    gr = mul(params<VEC>(a.gamma, k.channel(), 1.0f, a.wide), k.of_groups(rstd));
    be = params<VEC>(a.beta, k.channel(), 0.0f, a.wide);
  }
  // writes the first count of U positions
  template <typename T, int U>
  __device__ __forceinline__ void write(Vec<VEC> (&x)[U], int count, int act, Run<T> &y) const {
#pragma unroll
    for (int u = 0; u < U; ++u) x[u] = fma(add(x[u], mu), gr, be);
    act_values(x, act);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (u < count) store_vec<T, VEC>(y.p, x[u].v);
      y.next();
    }
  }
};

// Second pass: the pieces' means and squares give the group's, then y.  64 x 5046 x
// 64 f16 ELU 19 us, 16 x 6360 x 256 bf16 GELU 28 us, at 67 and 62 % of the issue
// slots: its warps mostly wait for their turn at them, and the rest is the start and
// the end of the blocks.
template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads, sample_blocks(false))
    norm_apply_kernel(const __grid_constant__ NormArgs a) {
  __shared__ float mean[kThreads * VEC], rstd[kThreads * VEC];
  const Patch<VEC> k(a);
  Scale<VEC> scale;
  auto join = [&]() {
    const int pieces = a.stretches * a.parts;
    const float2 *p = reinterpret_cast<const float2 *>(a.part) + (k.n * a.G + k.g0) * pieces;
    const float inv = 1.0f / ((float)a.L * (float)a.w);
    auto count = [&](int i) {
      if (a.parts == 1) return (float)min(a.L - i * a.stretch, a.stretch) * (float)a.w;
      const int64_t l0 = (int64_t)(i / a.parts) * a.stretch;
      const int c0 = (i % a.parts) * a.cols;
      return (float)min(a.L - l0, a.stretch) * (float)min(a.cols, a.w - c0);
    };
    wait_for_previous();
    each_team(k.groups, [&](int g, int lane, int team, bool lead) {
      const float2 *f = p + (int64_t)g * pieces;
      float mu = 0.0f, m2 = 0.0f;
#pragma unroll 4
      for (int i = lane; i < pieces; i += team) mu = fmaf(count(i), f[i].x, mu);
      mu = team_sum(mu, team) * inv;
#pragma unroll 4
      for (int i = lane; i < pieces; i += team)
        m2 += fmaf(count(i) * (f[i].x - mu), f[i].x - mu, f[i].y);
      m2 = team_sum(m2, team);
      if (lead) {
        const float rs = rsqrtf(fmaf(m2, inv, a.eps));
        mean[g] = mu;
        rstd[g] = rs;
        if (blockIdx.x == 0 && k.part == 0) {
          if (a.mean) a.mean[k.n * a.G + k.g0 + g] = mu;
          if (a.rstd) a.rstd[k.n * a.G + k.g0 + g] = rs;
        }
      }
    });
    __syncthreads();
    scale = Scale<VEC>(a, k, mean, rstd);
  };
  Run<T> x[1] = {Run<T>(a.x, k, a.sxn, a.sxl)}, y(a.y, k, a.syn, a.syl);
  each_position<4, T, VEC, 1>(k, x, join, [&](Raw<T, VEC>(&raw)[4][1], int count, auto reload) {
    Vec<VEC> v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) v[u] = values<T, VEC>(raw[u][0]);
    reload();
    scale.write(v, count, a.act, y);
  });
}

// xh = (x - mu) rstd and dz = dy act'(gamma xh + beta) of U positions
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
  // x becomes xh, dy dz
  template <int U>
  __device__ __forceinline__ void dz(Vec<VEC> (&x)[U], Vec<VEC> (&dy)[U], int act) const {
    Vec<VEC> z[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      x[u] = mul(add(x[u], mu), rs);
      z[u] = fma(x[u], ga, be);
    }
    act_slopes(z, act);
#pragma unroll
    for (int u = 0; u < U; ++u) dy[u] = mul(dy[u], z[u]);
  }
};

// part[n][stretch][2][C]: the sums of dz xh and dz of each channel over the
// block's positions, for dgamma and dbeta; done(group, s1, s2): the sums of gamma dz
// and gamma dz xh.
template <int VEC, typename F>
__device__ __forceinline__ void grad_sums(const NormArgs &a, const Patch<VEC> &k,
                                          const Vec<VEC> &dg, const Vec<VEC> &db, float2 *buf,
                                          F done) {
  float *p = a.part + (k.n * a.stretches + blockIdx.x) * 2 * a.C + k.c0;
  leave_pairs(k, dg, db, buf);
  each_team(k.width, [&](int c, int lane, int team, bool lead) {
    const float ga = a.gamma ? a.gamma[k.c0 + c] : 1.0f;
    float2 s = make_float2(0.0f, 0.0f);
#pragma unroll 4
    for (int r = lane; r < k.rows; r += team) {
      const float2 f = buf[r * k.width + c];
      s.x += f.x, s.y += f.y;
    }
    s.x = team_sum(s.x, team);
    s.y = team_sum(s.y, team);
    if (lead) {
      p[c] = s.x;
      p[a.C + c] = s.y;
      buf[c] = make_float2(s.y * ga, s.x * ga);  // only this team reads the column
    }
  });
  __syncthreads();
  each_team(k.groups, [&](int g, int lane, int team, bool lead) {
    float s1 = 0.0f, s2 = 0.0f;
    for (int c = lane; c < k.per; c += team) s1 += buf[g * k.per + c].x, s2 += buf[g * k.per + c].y;
    s1 = team_sum(s1, team);
    s2 = team_sum(s2, team);
    if (lead) done(g, s1, s2);
  });
}

// Gradient, first pass: grad_sums, the groups' into means[n][group][piece].  16 x
// 6360 x 256 bf16 GELU 35 us (3.0 TB/s), 56 % of the issue slots at 29 % of the warps
// (31 without the block's sums, and no more without the GELU, where it took 33); four
// positions a turn take as long.
template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads, sample_blocks(true))
    norm_grad_sums_kernel(const __grid_constant__ NormArgs a) {
  __shared__ Pairs<VEC> buf;
  const Patch<VEC> k(a);
  Vec<VEC> dg = all<VEC>(0.0f), db = dg;
  const Slope<VEC> slope(a, k);
  Run<T> xs[2] = {Run<T>(a.x, k, a.sxn, a.sxl), Run<T>(a.dy, k, a.syn, a.syl)};
  each_position<2, T, VEC, 2>(k, xs, Nothing{}, [&](Raw<T, VEC>(&raw)[2][2], int count, auto reload) {
    Vec<VEC> x[2], d[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) x[u] = values<T, VEC>(raw[u][0]), d[u] = values<T, VEC>(raw[u][1]);
    reload();
    slope.dz(x, d, a.act);  // positions after the last have zeros for dy: they add nothing
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      db = add(db, d[u]);
      dg = fma(d[u], x[u], dg);
    }
  });
  let_next_start();
  const int pieces = a.stretches * a.parts, piece = blockIdx.x * a.parts + k.part;
  float2 *p = a.means + (k.n * a.G + k.g0) * pieces + piece;
  grad_sums(a, k, dg, db, buf, [&](int g, float s1, float s2) {
    p[g * pieces] = make_float2(s1, s2);
  });
}

// dx = rstd (gamma dz - m1 - xh m2) of a position; m1 and m2 come times rstd
template <int VEC, typename T>
__device__ __forceinline__ void write_dx(const Slope<VEC> &slope, const Vec<VEC> &m1,
                                         const Vec<VEC> &m2, const Vec<VEC> &x,
                                         const Vec<VEC> &dy, int act, Run<T> &dx) {
  Vec<VEC> xh[1] = {x}, dz[1] = {dy};
  slope.dz(xh, dz, act);
  const Vec<VEC> o = fma(mul(dz[0], slope.ga), slope.rs, mul(fma(xh[0], m2, m1), -1.0f));
  store_vec<T, VEC>(dx.p, o.v);
  dx.next();
}

// Gradient, second pass: dx.  As the first 41 us, 58 % of the issue slots.
template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads, sample_blocks(true))
    norm_grad_apply_kernel(const __grid_constant__ NormArgs a) {
  __shared__ float s1[kThreads * VEC], s2[kThreads * VEC];
  const Patch<VEC> k(a);
  const Slope<VEC> slope(a, k);
  Vec<VEC> m1, m2;
  auto join = [&]() {
    const int pieces = a.stretches * a.parts;
    const float2 *p = a.means + (k.n * a.G + k.g0) * pieces;
    wait_for_previous();
    each_team(k.groups, [&](int g, int lane, int team, bool lead) {
      float2 s = make_float2(0.0f, 0.0f);
#pragma unroll 4
      for (int i = lane; i < pieces; i += team) {
        const float2 f = p[(int64_t)g * pieces + i];
        s.x += f.x, s.y += f.y;
      }
      s.x = team_sum(s.x, team);
      s.y = team_sum(s.y, team);
      if (lead) s1[g] = s.x, s2[g] = s.y;
    });
    __syncthreads();
    const float inv = 1.0f / ((float)a.L * (float)a.w);
    m1 = mul(mul(k.of_groups(s1), inv), slope.rs);
    m2 = mul(mul(k.of_groups(s2), inv), slope.rs);
  };
  Run<T> xs[2] = {Run<T>(a.x, k, a.sxn, a.sxl), Run<T>(a.dy, k, a.syn, a.syl)};
  Run<T> dx(a.dx, k, a.sdn, a.sdl);
  each_position<2, T, VEC, 2>(k, xs, join, [&](Raw<T, VEC>(&raw)[2][2], int count, auto reload) {
    Vec<VEC> x[2], d[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) x[u] = values<T, VEC>(raw[u][0]), d[u] = values<T, VEC>(raw[u][1]);
    reload();
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if (u >= count) break;
      write_dx(slope, m1, m2, x[u], d[u], a.act, dx);
    }
  });
  let_next_start();
}

// ------------------------------------------------ samples held by a block

// The block keeps what it read in shared memory; a thread reads back only its
// own.  200 x 300 x 96 bf16 ELU 12.5 us (1.8 TB/s), latency of one turn of the blocks.
// Clusters of up to 16 blocks that held larger samples together and exchanged sums
// took 34 us for 64 x 5046 x 64 f16, where two passes take 28.
template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads, sample_blocks(false))
    norm_block_kernel(const __grid_constant__ NormArgs a) {
  __shared__ Pairs<VEC> buf;
  __shared__ float mu[kThreads * VEC], rstd[kThreads * VEC];
  const Patch<VEC> k(a);
  Raw<T, VEC> *kept = reinterpret_cast<Raw<T, VEC> *>(norm_smem) + threadIdx.x;
  Spread<VEC> t;
  Run<T> x[1] = {Run<T>(a.x, k, a.sxn, a.sxl)};
  int slot = 0;
  each_position<4, T, VEC, 1>(k, x, Nothing{}, [&](Raw<T, VEC>(&raw)[4][1], int count, auto reload) {
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (u < count) kept[slot++ * kThreads] = raw[u][0];
    t.template take_turn<T, 4>(raw, count, reload);
  });
  const float inv = 1.0f / ((float)a.L * (float)a.w);
  block_spread(k, t, buf, [&](int g, float mean, float m2) {
    const float rs = rsqrtf(fmaf(m2, inv, a.eps));
    mu[g] = mean;
    rstd[g] = rs;
    if (a.mean) a.mean[k.n * a.G + k.g0 + g] = mean;
    if (a.rstd) a.rstd[k.n * a.G + k.g0 + g] = rs;
  });
  __syncthreads();
  if (!k.on) return;
  const Scale<VEC> scale(a, k, mu, rstd);
  Run<T> y(a.y, k, a.syn, a.syl);
  for (int i = 0; i < slot; i += 2) {
    Vec<VEC> v[2] = {values<T, VEC>(kept[i * kThreads]),
                     values<T, VEC>(kept[(i + 1 < slot ? i + 1 : i) * kThreads])};
    scale.write(v, slot - i, a.act, y);
  }
}

template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads, sample_blocks(true))
    norm_block_grad_kernel(const __grid_constant__ NormArgs a) {
  __shared__ Pairs<VEC> buf;
  __shared__ float s1[kThreads * VEC], s2[kThreads * VEC];
  const Patch<VEC> k(a);
  Raw<T, VEC> *kept = reinterpret_cast<Raw<T, VEC> *>(norm_smem) + threadIdx.x;
  Vec<VEC> dg = all<VEC>(0.0f), db = dg;
  const Slope<VEC> slope(a, k);
  Run<T> xs[2] = {Run<T>(a.x, k, a.sxn, a.sxl), Run<T>(a.dy, k, a.syn, a.syl)};
  int slot = 0;
  each_position<2, T, VEC, 2>(k, xs, Nothing{}, [&](Raw<T, VEC>(&raw)[2][2], int count, auto reload) {
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
    slope.dz(x, d, a.act);  // positions after the last have zeros for dy: they add nothing
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      db = add(db, d[u]);
      dg = fma(d[u], x[u], dg);
    }
  });
  let_next_start();
  grad_sums(a, k, dg, db, buf, [&](int g, float p, float q) { s1[g] = p, s2[g] = q; });
  __syncthreads();
  if (!k.on) return;
  const float inv = 1.0f / ((float)a.L * (float)a.w);
  const Vec<VEC> m1 = mul(mul(k.of_groups(s1), inv), slope.rs);
  const Vec<VEC> m2 = mul(mul(k.of_groups(s2), inv), slope.rs);
  Run<T> dx(a.dx, k, a.sdn, a.sdl);
  for (int i = 0; i < slot; ++i)
    write_dx(slope, m1, m2, values<T, VEC>(kept[2 * i * kThreads]),
             values<T, VEC>(kept[(2 * i + 1) * kThreads]), a.act, dx);
}

}  // namespace
}  // namespace zrl
