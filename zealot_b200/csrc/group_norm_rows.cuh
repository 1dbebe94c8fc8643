// group_norm_rows.cuh -- group norm of rows by themselves (L = 1): one pass, a
// group's channels in the registers of a few lanes next to one another in a
// warp, the next rows' loads in flight.
#pragma once

#include "group_norm.cuh"

namespace zrl {
namespace {

// Resident blocks, which bounds the registers; one number for all forms.  Three spill
// where a lane has four single channels: 98304 x 250 f32 forward 62 -> 109 us.  (Not
// measured for the forms of one vector a lane, which have room.  At two, the gradient
// with two vectors of eight channels spills: 276 bytes a thread stored, 148 loaded.)
constexpr int kLaneBlocks = 2;

template <int VEC, int V>
__device__ __forceinline__ Vec<VEC> slice(const Vec<V> &x, int e) {
  Vec<VEC> r;
#pragma unroll
  for (int i = 0; i < VEC; ++i) r[i] = x[e * VEC + i];
  return r;
}

// A thread of the row form: E vectors of VEC channels of one group, the same
// ones in every row it meets, so its gammas and betas stay in registers.
template <typename T, int VEC, int E>
struct RowLanes {
  int r, g;  // row within the block, group
  bool on, lead, has[E];
  int64_t at[E];  // first channel of each vector
  Vec<E * VEC> ga, be;
  __device__ __forceinline__ explicit RowLanes(const NormArgs &a) {
    const int per_row = a.gb * a.p, tid = threadIdx.x;
    r = tid / per_row;
    const int rem = tid - r * per_row, lane = rem & (a.p - 1);
    g = blockIdx.y * a.gb + rem / a.p;
    on = r < a.rb && g < a.G;
    lead = on && lane == 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int c = (lane + e * a.p) * VEC;
      has[e] = on && c < a.w;
      at[e] = has[e] ? (int64_t)g * a.w + c : 0;  // a place that can be read
      const Vec<VEC> p = has[e] ? params<VEC>(a.gamma, at[e], 1.0f, a.wide) : all<VEC>(0.0f);
      const Vec<VEC> q = has[e] ? params<VEC>(a.beta, at[e], 0.0f, a.wide) : all<VEC>(0.0f);
#pragma unroll
      for (int i = 0; i < VEC; ++i) ga[e * VEC + i] = p[i], be[e * VEC + i] = q[i];
    }
  }
  // the lane's channels, vector after vector
  __device__ __forceinline__ Vec<E * VEC> row(const Raw<T, VEC> (&raw)[E]) const {
    Vec<E * VEC> r;
#pragma unroll
    for (int e = 0; e < E; ++e) unpack<T, VEC>(raw[e], r.v + e * VEC);
    return r;
  }
  __device__ __forceinline__ void write(T *p, const Vec<E * VEC> &x) const {
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (has[e]) store_vec<T, VEC>(p + at[e], x.v + e * VEC);
  }
};

// U rows rb apart at a time; the next ones' loads are in flight.  A lane's vectors
// are taken as one, so that single channels go through the packed instructions
// too.  24576 x 512 bf16 in groups of 32 ELU 14 us (3.7 TB/s), 98304 x 250 f32 in groups
// of 25 SiLU 53 us (3.7 TB/s; vector by vector 62, rows staged as flat tiles in shared
// memory 70), at 63 and 66 % of the issue slots: sixteen warps an SM, the most that its
// registers allow, do not cover the latency of one product after the other and of
// the sums' shuffles.
template <typename T, int VEC, int E>
__global__ void __launch_bounds__(kThreads, kLaneBlocks)
    norm_rows_kernel(const __grid_constant__ NormArgs a) {
  constexpr int V = E * VEC, U = V > 8 ? 1 : V == 8 ? 2 : 4;
  const RowLanes<T, VEC, E> k(a);
  const float inv = 1.0f / (float)a.w;
  const int64_t pace = (int64_t)gridDim.x * a.rb * U;
  int64_t n = (int64_t)blockIdx.x * a.rb * U + k.r;  // this thread's first row
  // rows follow by adding strides; a vector's offset is added at each access
  const T *x0 = static_cast<const T *>(a.x) + n * a.sxn;
  T *y0 = static_cast<T *>(a.y) + n * a.syn;
  const int64_t xu = a.rb * a.sxn, yu = a.rb * a.syn;
  Raw<T, VEC> raw[U][E];
  auto load = [&](int64_t first) {
    const T *xr = x0;
#pragma unroll
    for (int u = 0; u < U; ++u, xr += xu)
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (first + u * a.rb < a.N && k.has[e])
          raw[u][e] = *reinterpret_cast<const Raw<T, VEC> *>(xr + k.at[e]);
    x0 += pace * a.sxn;
  };
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int e = 0; e < E; ++e) raw[u][e] = Raw<T, VEC>{};
  load(n);
  // the same number of turns for every thread of the block: n - k.r is shared
  for (; n - k.r < a.N; n += pace) {
    Vec<V> x[U];
    float mu[U], rstd[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      x[u] = k.row(raw[u]);
      mu[u] = sum(x[u]);  // zero where a lane has no channels
    }
    load(n + pace);
    lanes_sum(mu, a.p);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      mu[u] *= inv;
      Vec<V> m;
#pragma unroll
      for (int i = 0; i < V; ++i) m[i] = k.has[i / VEC] ? -mu[u] : 0.0f;
      x[u] = add(x[u], m);
      rstd[u] = sum(mul(x[u], x[u]));
    }
    lanes_sum(rstd, a.p);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      rstd[u] = rsqrtf(fmaf(rstd[u], inv, a.eps));
      x[u] = fma(x[u], mul(k.ga, rstd[u]), k.be);
    }
    act_values(x, a.act);
    T *yr = y0;
#pragma unroll
    for (int u = 0; u < U; ++u, yr += yu) {
      const int64_t row = n + u * a.rb;
      if (row >= a.N) break;
      k.write(yr, x[u]);
      if (k.lead && a.mean) a.mean[row * a.G + k.g] = mu[u];
      if (k.lead && a.rstd) a.rstd[row * a.G + k.g] = rstd[u];
    }
    y0 += pace * a.syn;
  }
}

// dx, and part[block][2][C]: the block's sums for dgamma and dbeta, kept in
// registers over all its rows.  98304 x 250 f32 in groups of 25 SiLU 102 us (2.9
// TB/s; 119 with a lane's vectors taken as one), 58 % of the issue slots: single
// elements a load, which are waited for.
template <typename T, int VEC, int E>
__global__ void __launch_bounds__(kThreads, kLaneBlocks)
    norm_rows_grad_kernel(const __grid_constant__ NormArgs a) {
  constexpr int U = E * VEC >= 8 ? 1 : 2;
  __shared__ float buf[kThreads];
  const RowLanes<T, VEC, E> k(a);
  const float inv = 1.0f / (float)a.w;
  Vec<VEC> dg[E], db[E];
#pragma unroll
  for (int e = 0; e < E; ++e) dg[e] = db[e] = all<VEC>(0.0f);
  const int64_t pace = (int64_t)gridDim.x * a.rb * U;
  int64_t n = (int64_t)blockIdx.x * a.rb * U + k.r;
  // rows follow by adding strides; a vector's offset is added at each access
  const T *x0 = static_cast<const T *>(a.x) + n * a.sxn;
  const T *d0 = static_cast<const T *>(a.dy) + n * a.syn;
  T *o0 = static_cast<T *>(a.dx) + n * a.sdn;
  const int64_t xu = a.rb * a.sxn, du = a.rb * a.syn, ou = a.rb * a.sdn;
  Raw<T, VEC> rx[U][E], rd[U][E];
  float mu[U], rstd[U];
  auto load = [&](int64_t first) {
    const T *xr = x0, *dr = d0;
#pragma unroll
    for (int u = 0; u < U; ++u, xr += xu, dr += du) {
      const int64_t row = first + u * a.rb;
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (row < a.N && k.has[e]) {
          rx[u][e] = *reinterpret_cast<const Raw<T, VEC> *>(xr + k.at[e]);
          rd[u][e] = *reinterpret_cast<const Raw<T, VEC> *>(dr + k.at[e]);
        }
      if (row < a.N && k.on) {
        mu[u] = a.mean[row * a.G + k.g];
        rstd[u] = a.rstd[row * a.G + k.g];
      } else {  // adds nothing to any sum
#pragma unroll
        for (int e = 0; e < E; ++e) rx[u][e] = rd[u][e] = Raw<T, VEC>{};
        mu[u] = 0.0f, rstd[u] = 0.0f;
      }
    }
    x0 += pace * a.sxn;
    d0 += pace * a.syn;
  };
#pragma unroll
  for (int u = 0; u < U; ++u) {
    mu[u] = rstd[u] = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) rx[u][e] = rd[u][e] = Raw<T, VEC>{};
  }
  load(n);
  for (; n - k.r < a.N; n += pace) {
    Vec<VEC> x[U][E], d[U][E];
    float s1[U], s2[U], rs[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      rs[u] = rstd[u];
      Vec<VEC> t1 = all<VEC>(0.0f), t2 = all<VEC>(0.0f);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const Vec<VEC> ga = slice<VEC>(k.ga, e);
        // no mean where a lane has no channels: (0 - mean) rstd may be infinite
        x[u][e] = mul(add(values<T, VEC>(rx[u][e]), k.has[e] ? -mu[u] : 0.0f), rs[u]);
        Vec<VEC> z[1] = {fma(x[u][e], ga, slice<VEC>(k.be, e))};
        act_slopes(z, a.act);
        // zero where a lane has no channels: dy is zero there
        const Vec<VEC> dz = mul(values<T, VEC>(rd[u][e]), z[0]);
        db[e] = add(db[e], dz);
        dg[e] = fma(dz, x[u][e], dg[e]);
        d[u][e] = mul(dz, ga);
        t1 = add(t1, d[u][e]);
        t2 = fma(d[u][e], x[u][e], t2);
      }
      s1[u] = sum(t1), s2[u] = sum(t2);
    }
    load(n + pace);
    lanes_sum(s1, a.p);
    lanes_sum(s2, a.p);
    T *orow = o0;
#pragma unroll
    for (int u = 0; u < U; ++u, orow += ou) {
      if (n + u * a.rb >= a.N) break;
      const float m1 = s1[u] * inv, m2 = s2[u] * inv;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const Vec<VEC> o = mul(add(d[u][e], fma(x[u][e], -m2, -m1)), rs[u]);
        if (k.has[e]) store_vec<T, VEC>(orow + k.at[e], o.v);
      }
    }
    o0 += pace * a.sdn;
  }
  let_next_start();
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
        if (k.r == 0 && k.has[e]) {
          float s = 0.0f;
          for (int r = 0; r < a.rb; ++r) s += buf[r * per_row + threadIdx.x];
          a.part[((int64_t)blockIdx.x * 2 + which) * a.C + k.at[e] + i] = s;
        }
      }
}

}  // namespace
}  // namespace zrl
