// group_norm_rows.cuh -- group norm of rows by themselves (L = 1).
//
// Two forms, both one pass over the data with the next rows' loads in flight.
// Lanes: a group's channels are whole vectors, held in registers by a few lanes
// next to one another in a warp.  Tiles: any other width; a tile of rows goes
// through shared memory, in and out as a flat run of 16-byte vectors.
#pragma once

#include "group_norm.cuh"

namespace zrl {
namespace {

#ifndef RB
#define RB 2
#endif
#ifndef TB
#define TB 6
#endif
#ifndef TGB
#define TGB 4
#endif
constexpr int kLaneBlocks = RB;  // resident blocks of the lanes form

// A thread of the row form: E vectors of VEC channels of one group, the same
// ones in every row it meets, so its gammas and betas stay in registers.
template <typename T, int VEC, int E>
struct RowLanes {
  int r, g;  // row within the block, group
  bool on, lead, has[E];
  int64_t at[E];  // first channel of each vector
  Vec<VEC> ga[E], be[E];
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
      ga[e] = has[e] ? params<VEC>(a.gamma, at[e], 1.0f, a.wide) : all<VEC>(0.0f);
      be[e] = has[e] ? params<VEC>(a.beta, at[e], 0.0f, a.wide) : all<VEC>(0.0f);
    }
  }
};

// p + stride as one multiply-add (one is 1, which the compiler cannot know).
template <typename P>
__device__ __forceinline__ void advance(P *&p, int32_t stride, int32_t one) {
  asm("mad.wide.s32 %0, %1, %2, %0;" : "+l"(p) : "r"(stride), "r"(one));
}

// A thread's places in one tensor: a running pointer per vector, U steps of rb
// rows a turn.
template <typename T, int E>
struct RowPlaces {
  T *p[E];
  int32_t step;  // bytes from a row to the one rb below
  int64_t jump;  // bytes from the end of a turn to the next
  __device__ __forceinline__ RowPlaces(const void *base, int64_t stride, const int64_t *at,
                                       int64_t first, const NormArgs &a, int U) {
#pragma unroll
    for (int e = 0; e < E; ++e)
      p[e] = const_cast<T *>(static_cast<const T *>(base)) + first * stride + at[e];
    step = (int32_t)(a.rb * stride * (int64_t)sizeof(T));
    jump = (int64_t)(gridDim.x - 1) * U * step;
  }
  __device__ __forceinline__ void next_row(int32_t one) {
#pragma unroll
    for (int e = 0; e < E; ++e) advance(p[e], step, one);
  }
  __device__ __forceinline__ void next_turn() {
#pragma unroll
    for (int e = 0; e < E; ++e) p[e] = (T *)((char *)p[e] + jump);
  }
};

// U rows rb apart at a time; the next ones' loads are in flight.
template <typename T, int VEC, int E>
__global__ void __launch_bounds__(kThreads, kLaneBlocks)
    norm_rows_kernel(const __grid_constant__ NormArgs a) {
  constexpr int U = E * VEC >= 8 ? 2 : 4;
  const RowLanes<T, VEC, E> k(a);
  const float inv = 1.0f / (float)a.w;
  const int64_t pace = (int64_t)gridDim.x * a.rb * U;
  int64_t n = (int64_t)blockIdx.x * a.rb * U + k.r;  // this thread's first row
  RowPlaces<T, E> xs(a.x, a.sxn, k.at, n, a, U), ys(a.y, a.syn, k.at, n, a, U);
  Raw<T, VEC> raw[U][E];
  auto load = [&](int64_t first) {
    const bool whole = first + (U - 1) * a.rb < a.N;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (whole || first + u * a.rb < a.N) {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (k.has[e]) raw[u][e] = *reinterpret_cast<const Raw<T, VEC> *>(xs.p[e]);
      }
      xs.next_row(a.one);
    }
    xs.next_turn();
  };
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int e = 0; e < E; ++e) raw[u][e] = Raw<T, VEC>{};
  load(n);
  // the same number of turns for every thread of the block: n - k.r is shared
  for (; n - k.r < a.N; n += pace) {
    Vec<VEC> x[U][E];
    float mu[U], rstd[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int e = 0; e < E; ++e) x[u][e] = values<T, VEC>(raw[u][e]);
      Vec<VEC> s = x[u][0];  // zero where a lane has no channels
#pragma unroll
      for (int e = 1; e < E; ++e) s = add(s, x[u][e]);
      mu[u] = sum(s);
    }
    load(n + pace);
    lanes_sum(mu, a.p);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      mu[u] *= inv;
      Vec<VEC> q = all<VEC>(0.0f);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        x[u][e] = add(x[u][e], k.has[e] ? -mu[u] : 0.0f);
        q = fma(x[u][e], x[u][e], q);
      }
      rstd[u] = sum(q);
    }
    lanes_sum(rstd, a.p);
    const bool whole = n + (U - 1) * a.rb < a.N;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float r = rsqrtf(fmaf(rstd[u], inv, a.eps));
      if (whole || n + u * a.rb < a.N) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
          Vec<VEC> z = fma(x[u][e], mul(k.ga[e], r), k.be[e]);
          act_values<VEC>(z, a.act);
          if (k.has[e]) store_vec<T, VEC>(ys.p[e], z.v);
        }
        if (k.lead && a.mean) a.mean[(n + u * a.rb) * a.G + k.g] = mu[u];
        if (k.lead && a.rstd) a.rstd[(n + u * a.rb) * a.G + k.g] = r;
      }
      ys.next_row(a.one);
    }
    ys.next_turn();
  }
}

// dx, and part[block][2][C]: the block's sums for dgamma and dbeta, kept in
// registers over all its rows.
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
  RowPlaces<T, E> xs(a.x, a.sxn, k.at, n, a, U), ds(a.dy, a.syn, k.at, n, a, U),
      os(a.dx, a.sdn, k.at, n, a, U);
  Raw<T, VEC> rx[U][E], rd[U][E];
  float mu[U], rstd[U];
  auto load = [&](int64_t first) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t row = first + u * a.rb;
      if (row < a.N) {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (k.has[e]) {
            rx[u][e] = *reinterpret_cast<const Raw<T, VEC> *>(xs.p[e]);
            rd[u][e] = *reinterpret_cast<const Raw<T, VEC> *>(ds.p[e]);
          }
        if (k.on) {
          mu[u] = a.mean[row * a.G + k.g];
          rstd[u] = a.rstd[row * a.G + k.g];
        }
      } else {  // adds nothing to any sum
#pragma unroll
        for (int e = 0; e < E; ++e) rx[u][e] = rd[u][e] = Raw<T, VEC>{};
        mu[u] = 0.0f, rstd[u] = 0.0f;
      }
      xs.next_row(a.one);
      ds.next_row(a.one);
    }
    xs.next_turn();
    ds.next_turn();
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
        x[u][e] = mul(add(values<T, VEC>(rx[u][e]), -mu[u]), rs[u]);
        Vec<VEC> z = fma(x[u][e], k.ga[e], k.be[e]);
        act_slopes<VEC>(z, a.act);
        // zero where a lane has no channels: dy is zero there
        const Vec<VEC> dz = mul(values<T, VEC>(rd[u][e]), z);
        db[e] = add(db[e], dz);
        dg[e] = fma(dz, x[u][e], dg[e]);
        d[u][e] = mul(dz, k.ga[e]);
        t1 = add(t1, d[u][e]);
        t2 = fma(d[u][e], x[u][e], t2);
      }
      s1[u] = sum(t1), s2[u] = sum(t2);
    }
    load(n + pace);
    lanes_sum(s1, a.p);
    lanes_sum(s2, a.p);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (n + u * a.rb < a.N) {
        const float m1 = s1[u] * inv, m2 = s2[u] * inv;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const Vec<VEC> o = mul(add(d[u][e], fma(x[u][e], -m2, -m1)), rs[u]);
          if (k.has[e]) store_vec<T, VEC>(os.p[e], o.v);
        }
      }
      os.next_row(a.one);
    }
    os.next_turn();
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
        if (k.r == 0 && k.has[e]) {
          float s = 0.0f;
          for (int r = 0; r < a.rb; ++r) s += buf[r * per_row + threadIdx.x];
          a.part[((int64_t)blockIdx.x * 2 + which) * a.C + k.at[e] + i] = s;
        }
      }
}

// ---------------------------------------------------------------- tiles

constexpr int kTileVecs = 4;  // 16-byte vectors of a tile a thread and tensor
template <typename T>
constexpr int tile_elements() { return kTileVecs * kThreads * (16 / (int)sizeof(T)); }

// A tile of rb rows of a dense [N, C] tensor as whole 16-byte vectors: from the
// vector that its first element lies in to the one of its last.  The vectors at
// the two ends may hold elements of the neighbours, which are read and not used,
// and are written element by element.
template <typename T>
struct TileSpan {
  static constexpr int VEC = 16 / (int)sizeof(T);
  int64_t begin, start, end;  // elements; start: begin rounded down to a vector
  int rows;
  __device__ __forceinline__ TileSpan(const NormArgs &a, int64_t tile) {
    rows = (int)min((int64_t)a.rb, a.N - tile * a.rb);
    begin = tile * a.rb * a.C;
    start = begin / VEC * VEC;
    end = begin + (int64_t)rows * a.C;
  }
  __device__ __forceinline__ int64_t at(int v) const {
    return start + (int64_t)(v * kThreads + threadIdx.x) * VEC;
  }
  __device__ __forceinline__ void load(const void *p, int64_t total,
                                       Raw<T, VEC> (&raw)[kTileVecs]) const {
    const T *x = static_cast<const T *>(p);
#pragma unroll
    for (int v = 0; v < kTileVecs; ++v) {
      const int64_t f = at(v);
      if (f + VEC <= total && f < end) {
        raw[v] = *reinterpret_cast<const Raw<T, VEC> *>(x + f);
      } else if (f < end) {
        T e[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) e[i] = f + i < total ? x[f + i] : T{};
        memcpy(&raw[v], e, sizeof(raw[v]));
      }
    }
  }
  __device__ __forceinline__ void put(const Raw<T, VEC> (&raw)[kTileVecs], float *s) const {
#pragma unroll
    for (int v = 0; v < kTileVecs; ++v) {
      if (at(v) >= end) break;
      float e[VEC];
      unpack<T, VEC>(raw[v], e);
      float4 *to = reinterpret_cast<float4 *>(s + (v * kThreads + threadIdx.x) * VEC);
#pragma unroll
      for (int i = 0; i < VEC; i += 4) to[i / 4] = make_float4(e[i], e[i + 1], e[i + 2], e[i + 3]);
    }
  }
  __device__ __forceinline__ void store(void *p, const float *s) const {
    T *y = static_cast<T *>(p);
#pragma unroll
    for (int v = 0; v < kTileVecs; ++v) {
      const int64_t f = at(v);
      if (f >= end) break;
      float e[VEC];
      const float4 *from = reinterpret_cast<const float4 *>(s + (v * kThreads + threadIdx.x) * VEC);
#pragma unroll
      for (int i = 0; i < VEC; i += 4) {
        const float4 q = from[i / 4];
        e[i] = q.x, e[i + 1] = q.y, e[i + 2] = q.z, e[i + 3] = q.w;
      }
      if (f >= begin && f + VEC <= end) {
        store_vec<T, VEC>(y + f, e);
      } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i)
          if (f + i >= begin && f + i < end) y[f + i] = from_f32<T>(e[i]);
      }
    }
  }
};

// Group r, g of the tile for each p lanes; f(row, group, lane, on) is called by
// whole warps.
template <typename F>
__device__ __forceinline__ void each_group(const NormArgs &a, int rows, F f) {
  const int count = rows * a.G, at_once = kThreads / a.p, lane = threadIdx.x & (a.p - 1);
  for (int t0 = 0; t0 < count; t0 += at_once) {
    const int t = t0 + threadIdx.x / a.p, r = t / a.G;
    f(r, t - r * a.G, lane, t < count);
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads, TB)
    norm_tile_kernel(const __grid_constant__ NormArgs a) {
  constexpr int VEC = 16 / (int)sizeof(T);
  float *s = reinterpret_cast<float *>(norm_smem);
  float *ga = s + tile_elements<T>(), *be = ga + a.C;
  for (int c = threadIdx.x; c < a.C; c += kThreads) {
    ga[c] = a.gamma ? a.gamma[c] : 1.0f;
    be[c] = a.beta ? a.beta[c] : 0.0f;
  }
  const int64_t tiles = (a.N + a.rb - 1) / a.rb, total = a.N * a.C;
  const float inv = 1.0f / (float)a.w;
  Raw<T, VEC> raw[kTileVecs] = {};
  int64_t tile = blockIdx.x;
  if (tile < tiles) TileSpan<T>(a, tile).load(a.x, total, raw);
  for (; tile < tiles; tile += gridDim.x) {
    const TileSpan<T> span(a, tile);
    span.put(raw, s);
    __syncthreads();
    if (tile + gridDim.x < tiles) TileSpan<T>(a, tile + gridDim.x).load(a.x, total, raw);
    float *own = s + (span.begin - span.start);
    each_group(a, span.rows, [&](int r, int g, int lane, bool on) {
      float *x = own + r * a.C + g * a.w;
      const int w = on ? a.w : 0;
      float mu[1] = {0.0f}, q[1] = {0.0f};
#pragma unroll 4
      for (int j = lane; j < w; j += a.p) mu[0] += x[j];
      lanes_sum(mu, a.p);
      mu[0] *= inv;
#pragma unroll 4
      for (int j = lane; j < w; j += a.p) {
        const float d = x[j] - mu[0];
        q[0] = fmaf(d, d, q[0]);
      }
      lanes_sum(q, a.p);
      const float rstd = rsqrtf(fmaf(q[0], inv, a.eps));
      const float *gg = ga + g * a.w, *bb = be + g * a.w;
#pragma unroll 4
      for (int j = lane; j < w; j += a.p) {
        Vec<1> z;
        z[0] = fmaf((x[j] - mu[0]) * rstd, gg[j], bb[j]);
        act_values<1>(z, a.act);
        x[j] = z[0];
      }
      if (on && lane == 0) {
        const int64_t ng = (tile * a.rb + r) * a.G + g;
        if (a.mean) a.mean[ng] = mu[0];
        if (a.rstd) a.rstd[ng] = rstd;
      }
    });
    __syncthreads();
    span.store(a.y, s);
    __syncthreads();
  }
}

// dx, and part[block][2][C] as norm_rows_grad_kernel.  In shared memory x becomes
// xh, then dx; dy becomes dz.
template <typename T>
__global__ void __launch_bounds__(kThreads, TGB)
    norm_tile_grad_kernel(const __grid_constant__ NormArgs a) {
  constexpr int VEC = 16 / (int)sizeof(T);
  float *s = reinterpret_cast<float *>(norm_smem), *d = s + tile_elements<T>();
  float *ga = d + tile_elements<T>(), *be = ga + a.C, *dg = be + a.C, *db = dg + a.C;
  float *m1 = db + a.C, *m2 = m1 + a.rb * a.G;  // of each group of the tile, by rstd
  for (int c = threadIdx.x; c < a.C; c += kThreads) {
    ga[c] = a.gamma ? a.gamma[c] : 1.0f;
    be[c] = a.beta ? a.beta[c] : 0.0f;
    dg[c] = db[c] = 0.0f;
  }
  const int64_t tiles = (a.N + a.rb - 1) / a.rb, total = a.N * a.C;
  const float inv = 1.0f / (float)a.w;
  Raw<T, VEC> rx[kTileVecs] = {}, rd[kTileVecs] = {};
  int64_t tile = blockIdx.x;
  if (tile < tiles) {
    TileSpan<T>(a, tile).load(a.x, total, rx);
    TileSpan<T>(a, tile).load(a.dy, total, rd);
  }
  for (; tile < tiles; tile += gridDim.x) {
    const TileSpan<T> span(a, tile);
    span.put(rx, s);
    span.put(rd, d);
    __syncthreads();
    if (tile + gridDim.x < tiles) {
      const TileSpan<T> next(a, tile + gridDim.x);
      next.load(a.x, total, rx);
      next.load(a.dy, total, rd);
    }
    const int skip = (int)(span.begin - span.start);
    each_group(a, span.rows, [&](int r, int g, int lane, bool on) {
      float *x = s + skip + r * a.C + g * a.w, *dz = d + skip + r * a.C + g * a.w;
      const float *gg = ga + g * a.w, *bb = be + g * a.w;
      const int w = on ? a.w : 0;
      const int64_t ng = (tile * a.rb + r) * a.G + g;
      const float mu = on ? a.mean[ng] : 0.0f, rstd = on ? a.rstd[ng] : 0.0f;
      float t1[1] = {0.0f}, t2[1] = {0.0f};
#pragma unroll 4
      for (int j = lane; j < w; j += a.p) {
        const float xh = (x[j] - mu) * rstd;
        Vec<1> z;
        z[0] = fmaf(xh, gg[j], bb[j]);
        act_slopes<1>(z, a.act);
        const float e = dz[j] * z[0], f = e * gg[j];
        x[j] = xh;
        dz[j] = e;
        t1[0] += f;
        t2[0] = fmaf(f, xh, t2[0]);
      }
      lanes_sum(t1, a.p);
      lanes_sum(t2, a.p);
      if (on && lane == 0) {
        m1[r * a.G + g] = t1[0] * inv * rstd;
        m2[r * a.G + g] = t2[0] * inv * rstd;
      }
    });
    __syncthreads();
    for (int c = threadIdx.x; c < a.C; c += kThreads) {
      float sg = dg[c], sb = db[c];
#pragma unroll 4
      for (int r = 0; r < span.rows; ++r) {
        const float e = d[skip + r * a.C + c];
        sg = fmaf(e, s[skip + r * a.C + c], sg);
        sb += e;
      }
      dg[c] = sg;
      db[c] = sb;
    }
    __syncthreads();
    each_group(a, span.rows, [&](int r, int g, int lane, bool on) {
      if (!on) return;
      float *x = s + skip + r * a.C + g * a.w;
      const float *dz = d + skip + r * a.C + g * a.w, *gg = ga + g * a.w;
      const float rstd = a.rstd[(tile * a.rb + r) * a.G + g];
      const float n1 = m1[r * a.G + g], n2 = m2[r * a.G + g];
#pragma unroll 4
      for (int j = lane; j < a.w; j += a.p)
        x[j] = fmaf(dz[j] * gg[j], rstd, -fmaf(x[j], n2, n1));
    });
    __syncthreads();
    span.store(a.dx, s);
    __syncthreads();
  }
  for (int c = threadIdx.x; c < a.C; c += kThreads) {
    a.part[((int64_t)blockIdx.x * 2) * a.C + c] = dg[c];
    a.part[((int64_t)blockIdx.x * 2 + 1) * a.C + c] = db[c];
  }
}

}  // namespace
}  // namespace zrl
