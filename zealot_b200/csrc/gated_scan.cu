// gated_scan.cu -- a gated linear recurrence over time, and its gradient.
//
// Per channel, with rate = c softplus(lam), s_r = sigmoid(rec),
// s_i = sigmoid(inp):
//   a_t = exp(-rate s_r), or 0 where an episode begins (resets_t != 0)
//   m_t = sqrt(1 - a_t^2),  h_t = a_t h_{t-1} + m_t s_i x_t
// Gradient, with g_t = dh_t + a_{t+1} g_{t+1} (dh_last joins dh_{T-1}):
//   dx = g m s_i,  dinp = g m x s_i (1 - s_i),  dh0 = a_0 g_0
//   q = g (h_{t-1} a - s_i x a^2 / m)            (the slope along log a)
//   drec = -rate s_r (1 - s_r) q,  dlam = -c sigmoid(lam) sum s_r q
#include <math.h>

#include <algorithm>
#include <initializer_list>
#include <type_traits>

#include "seq_common.cuh"

namespace zrl {
namespace {

constexpr int kSteps = 8;       // steps one warp takes from a tile
constexpr int kWarps = 8;       // warps of a block at most
constexpr int kMaxCluster = 16;
// A tile of a long row: kWarps x kSteps steps.  The forward call keeps the
// state at every kChunk-th step, where the gradient's tiles start from.
constexpr int kChunk = kSteps * kWarps;
constexpr float kLog2e = 1.44269504f;
constexpr float kSeriesMax = 0.35f;
constexpr float kTinySquare = 7.5231638e-37f;  // 2^-120

struct ScanArgs {
  const void *x, *rec, *inp, *dh;
  const float *lam, *h0, *dh_last;
  const uint8_t *resets;
  void *h, *dx, *drec, *dinp;
  float *h_last, *carry, *dh0, *part;
  int64_t B, T, D, K;   // K: chunk starts after the first
  int64_t units, tiles; // units of V channels; tiles of one row
  int64_t xb, xt, rb, rt, ib, it, zb, zt, hb, ht, gb, gt, dxb, dxt, drb, drt, dib, dit;
  float c;
};

__device__ __forceinline__ float softplus(float v) {
  return fmaxf(v, 0.0f) + log1pf(expf(-fabsf(v)));
}
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
__device__ __forceinline__ float rsq(float v) {
  float r;
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
// NaN stays NaN, unlike fminf and fmaxf
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// One element's gates.  With u = rate sigmoid(rec), e = 1 - a = 1 - exp(-u)
// comes from its series up to u = 0.35 (seven terms, 2e-8 relative): a = 1 - e
// is then within half a unit of exp(-u) at every step, so the roundings of a
// long memory do not add up in one direction, and 1 - a^2 = e (2 - e) keeps its
// digits where a is near 1.  Above (only SLOW looks), a comes from ex2.
// m sigmoid(inp) = s / sqrt(s q^2) with s = 1 - a^2, q = 1 + exp(-inp): one
// reciprocal square root for the square root and the quotient.  exp(-inp) is
// held to 2^60, exp(-rec) to 2^126 and s to at least 2^-120, so nothing
// overflows or divides by zero.
struct Gate {
  float sr, e, s, q, ms;  // sigmoid(rec), 1 - a, 1 - a^2, 1 + exp(-inp), m sigmoid(inp)
  float w;                // 1 / (sqrt(s) q)
};
template <bool SLOW>
__device__ __forceinline__ Gate gate(float rec, float inp, float rate, bool reset) {
  Gate g;
  g.sr = rcp(1.0f + ex2(min_nan(rec * -kLog2e, 126.0f)));
  g.q = 1.0f + ex2(min_nan(inp * -kLog2e, 60.0f));
  const float u = rate * g.sr;
  float p = fmaf(u, 1.0f / 5040.0f, -1.0f / 720.0f);
  p = fmaf(u, p, 1.0f / 120.0f);
  p = fmaf(u, p, -1.0f / 24.0f);
  p = fmaf(u, p, 1.0f / 6.0f);
  p = fmaf(u, p, -0.5f);
  p = fmaf(u, p, 1.0f);
  g.e = u * p;
  if (SLOW) {
    if (u > kSeriesMax) g.e = 1.0f - ex2(u * -kLog2e);
    if (reset) g.e = 1.0f;  // a = 0, m = 1
  }
  g.s = max_nan(fmaf(-g.e, g.e, 2.0f * g.e), kTinySquare);
  g.w = rsq(g.s * g.q * g.q);
  g.ms = g.s * g.w;
  return g;
}

// A stretch of steps maps the state before it to h -> P h + H.  P is -0 where
// an episode begins inside: then nothing of h is used, infinity and NaN
// included.
__device__ __forceinline__ float through(float P, float H, float h) {
  return __float_as_int(P) < 0 ? H : fmaf(P, h, H);
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;"
               ::: "memory");
}
// Stores a pair at the same shared-memory place of another block of the cluster.
__device__ __forceinline__ void store_pair_at(float2 *p, uint32_t rank, float2 v) {
  uint32_t a = (uint32_t)__cvta_generic_to_shared(p), r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
  asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(r), "f"(v.x), "f"(v.y)
               : "memory");
}

// The reset marks of steps t .. t + n - 1 of the lane's row, bit s for step s.
// A warp whose lanes share a row reads each mark once.
__device__ __forceinline__ uint32_t reset_bits(const ScanArgs &a, int64_t b, int64_t t, int n,
                                               bool one_row) {
  if (!a.resets) return 0;
  const uint8_t *z = a.resets + b * a.zb + t * a.zt;
  uint32_t bits = 0;
  if (one_row) {
    const int lane = threadIdx.x;
    const bool on = lane < n && z[lane * a.zt];
    bits = __ballot_sync(0xffffffffu, on);
  } else {
    for (int s = 0; s < n; ++s) bits |= (z[s * a.zt] ? 1u : 0u) << s;
  }
  return bits;
}

// Which channels a lane has: V of them from d in row b.
template <int V>
struct Place {
  int64_t b, d;
  bool live, one_row;
  __device__ __forceinline__ Place(const ScanArgs &a, int64_t q) {
    live = q < a.units;
    if (!live) q = a.units - 1;  // reads what the last lane reads, writes nothing
    const int64_t per = a.D / V;
    if (a.units >> 31) {
      b = q / per;
    } else {
      b = (uint32_t)q / (uint32_t)per;
    }
    d = (q - b * per) * V;
    one_row = __all_sync(0xffffffffu, b == __shfl_sync(0xffffffffu, b, 0));
  }
};

// Blocks of 32 lanes x W warps along time x Z groups of lanes.  A tile is W
// times S steps: every warp folds its S steps from a zero state in registers,
// the warps (and, through distributed shared memory, the blocks of a cluster,
// which take neighbouring tiles) exchange (P, H), and every warp runs its
// steps again from its true state and stores them.  One pass over the data.
template <typename T, int V, int S>
__global__ void __launch_bounds__(256) scan_kernel(const __grid_constant__ ScanArgs a) {
  __shared__ float2 agg[2][kWarps][32 * V];
  __shared__ float2 cagg[2][kMaxCluster][32 * V];
  const int lane = threadIdx.x, wt = threadIdx.y, W = blockDim.y;
  const int slot = threadIdx.z * W;
  const uint32_t ranks = cluster_size(), rank = cluster_rank();
  const Place<V> at(a, ((int64_t)(blockIdx.x / ranks) * blockDim.z + threadIdx.z) * 32 + lane);
  float rate[V], carry[V];
  bool big = false;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    rate[v] = a.c * softplus(a.lam[at.d + v]);
    big |= rate[v] > kSeriesMax;
    carry[v] = a.h0 ? a.h0[at.b * a.D + at.d + v] : 0.0f;
  }
  big = __any_sync(0xffffffffu, big);
  const T *xp = static_cast<const T *>(a.x) + at.b * a.xb + at.d;
  const T *rp = static_cast<const T *>(a.rec) + at.b * a.rb + at.d;
  const T *ip = static_cast<const T *>(a.inp) + at.b * a.ib + at.d;
  T *hp = static_cast<T *>(a.h) + at.b * a.hb + at.d;
  if (ranks > 1) cluster_barrier();  // every block of the cluster runs

  int par = 0;
  for (int64_t k0 = 0; k0 < a.tiles; k0 += ranks, par ^= 1) {
    const int64_t k = k0 + rank, t0 = (k * W + wt) * S;
    const int n = (int)max((int64_t)0, min((int64_t)S, a.T - t0));
    Raw<T, V> rr[S], ri[S], rx[S];
#pragma unroll
    for (int s = 0; s < S; ++s) {
      if (s < n) {
        rr[s] = *reinterpret_cast<const Raw<T, V> *>(rp + (t0 + s) * a.rt);
        ri[s] = *reinterpret_cast<const Raw<T, V> *>(ip + (t0 + s) * a.it);
        rx[s] = *reinterpret_cast<const Raw<T, V> *>(xp + (t0 + s) * a.xt);
      } else {
        rr[s] = ri[s] = rx[s] = Raw<T, V>{};
      }
    }
    const uint32_t z = n ? reset_bits(a, at.b, t0, n, at.one_row) : 0;
    const bool slow = big || n < S || __any_sync(0xffffffffu, z != 0);
    float A[S][V], Bv[S][V], P[V], H[V];
    auto fold = [&](auto tag) {
      constexpr bool SLOW = decltype(tag)::value;
#pragma unroll
      for (int v = 0; v < V; ++v) P[v] = 1.0f, H[v] = 0.0f;
#pragma unroll
      for (int s = 0; s < S; ++s) {
        float r[V], i[V], x[V];
        unpack<T, V>(rr[s], r);
        unpack<T, V>(ri[s], i);
        unpack<T, V>(rx[s], x);
        const bool reset = SLOW && (z >> s & 1);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const Gate g = gate<SLOW>(r[v], i[v], rate[v], reset);
          A[s][v] = 1.0f - g.e;
          Bv[s][v] = g.ms * x[v];
          if (SLOW && s >= n) A[s][v] = 1.0f, Bv[s][v] = 0.0f;
          H[v] = reset ? Bv[s][v] : fmaf(A[s][v], H[v], Bv[s][v]);
          P[v] = reset ? -0.0f : P[v] * A[s][v];
        }
      }
    };
    if (slow) fold(std::true_type{});
    else fold(std::false_type{});

#pragma unroll
    for (int v = 0; v < V; ++v) agg[par][slot + wt][v * 32 + lane] = make_float2(P[v], H[v]);
    __syncthreads();
    float in[V];
    if (ranks > 1) {
      // this block's (P, H) to every block, then the blocks before this one
      float cp[V], ch[V];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float2 f = agg[par][slot][v * 32 + lane];
        cp[v] = f.x, ch[v] = f.y;
        for (int w = 1; w < W; ++w) {
          f = agg[par][slot + w][v * 32 + lane];
          ch[v] = through(f.x, f.y, ch[v]);
          cp[v] = __float_as_int(f.x) < 0 ? f.x : f.x * cp[v];
        }
      }
      for (uint32_t r = wt; r < ranks; r += W)
#pragma unroll
        for (int v = 0; v < V; ++v)
          store_pair_at(&cagg[par][rank][v * 32 + lane], r, make_float2(cp[v], ch[v]));
      cluster_barrier();
#pragma unroll
      for (int v = 0; v < V; ++v) {
        for (uint32_t r = 0; r < ranks; ++r) {
          if (r == rank) in[v] = carry[v];
          const float2 f = cagg[par][r][v * 32 + lane];
          carry[v] = through(f.x, f.y, carry[v]);
        }
      }
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v) in[v] = carry[v];
    }
    if (a.carry && wt == 0 && k > 0 && n > 0 && at.live) {
      float *c = a.carry + (at.b * a.K + k - 1) * a.D + at.d;
#pragma unroll
      for (int v = 0; v < V; ++v) c[v] = in[v];
    }
    float h[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      h[v] = in[v];
      for (int w = 0; w < W; ++w) {
        const float2 f = agg[par][slot + w][v * 32 + lane];
        if (w == wt) h[v] = in[v];
        in[v] = through(f.x, f.y, in[v]);
      }
      if (ranks == 1) carry[v] = in[v];
    }
#pragma unroll
    for (int s = 0; s < S; ++s) {
#pragma unroll
      for (int v = 0; v < V; ++v)
        h[v] = slow && (z >> s & 1) ? Bv[s][v] : fmaf(A[s][v], h[v], Bv[s][v]);
      if (s < n && at.live) store_vec<T, V>(hp + (t0 + s) * a.ht, h);
    }
  }
  if (a.h_last && wt == 0 && rank == 0 && at.live) {
#pragma unroll
    for (int v = 0; v < V; ++v) a.h_last[at.b * a.D + at.d + v] = carry[v];
  }
}

// The gradient, tile by tile from the end (the blocks of a cluster take
// neighbouring tiles, the last first).  A tile's states start from the forward
// call's carry; the gradient's own recurrence runs backwards with the same P:
// gamma_t = a_t g_t, g_t = dh_t + gamma_{t+1}.
template <typename T, int V, int S>
__global__ void __launch_bounds__(256) scan_grad_kernel(const __grid_constant__ ScanArgs a) {
  __shared__ float2 agg[2][kWarps][32 * V];  // (P, H)
  __shared__ float back[2][kWarps][32 * V];  // gamma of a stretch from zero
  __shared__ float2 cagg[2][kMaxCluster][32 * V];
  const int lane = threadIdx.x, wt = threadIdx.y, W = blockDim.y;
  const int slot = threadIdx.z * W;
  const uint32_t ranks = cluster_size(), rank = cluster_rank();
  const Place<V> at(a, ((int64_t)(blockIdx.x / ranks) * blockDim.z + threadIdx.z) * 32 + lane);
  float rate[V], gam[V], dl[V];
  bool big = false;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    rate[v] = a.c * softplus(a.lam[at.d + v]);
    big |= rate[v] > kSeriesMax;
    gam[v] = a.dh_last ? a.dh_last[at.b * a.D + at.d + v] : 0.0f;
    dl[v] = 0.0f;
  }
  big = __any_sync(0xffffffffu, big);
  const T *xp = static_cast<const T *>(a.x) + at.b * a.xb + at.d;
  const T *rp = static_cast<const T *>(a.rec) + at.b * a.rb + at.d;
  const T *ip = static_cast<const T *>(a.inp) + at.b * a.ib + at.d;
  const T *gp = static_cast<const T *>(a.dh) + at.b * a.gb + at.d;
  T *dxp = static_cast<T *>(a.dx) + at.b * a.dxb + at.d;
  T *drp = static_cast<T *>(a.drec) + at.b * a.drb + at.d;
  T *dip = static_cast<T *>(a.dinp) + at.b * a.dib + at.d;
  if (ranks > 1) cluster_barrier();

  int par = 0;
  for (int64_t k0 = a.tiles - 1; k0 >= 0; k0 -= ranks, par ^= 1) {
    const int64_t k = k0 - rank, t0 = (k * W + wt) * S;
    const int n = k < 0 ? 0 : (int)max((int64_t)0, min((int64_t)S, a.T - t0));
    Raw<T, V> rr[S], ri[S], rx[S], rg[S];
#pragma unroll
    for (int s = 0; s < S; ++s) {
      if (s < n) {
        rr[s] = *reinterpret_cast<const Raw<T, V> *>(rp + (t0 + s) * a.rt);
        ri[s] = *reinterpret_cast<const Raw<T, V> *>(ip + (t0 + s) * a.it);
        rx[s] = *reinterpret_cast<const Raw<T, V> *>(xp + (t0 + s) * a.xt);
        rg[s] = *reinterpret_cast<const Raw<T, V> *>(gp + (t0 + s) * a.gt);
      } else {
        rr[s] = ri[s] = rx[s] = rg[s] = Raw<T, V>{};
      }
    }
    float h[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      h[v] = 0.0f;
      if (k > 0) h[v] = a.carry[(at.b * a.K + k - 1) * a.D + at.d + v];
      else if (k == 0 && a.h0) h[v] = a.h0[at.b * a.D + at.d + v];
    }
    const uint32_t z = n ? reset_bits(a, at.b, t0, n, at.one_row) : 0;
    const bool slow = big || n < S || __any_sync(0xffffffffu, z != 0);
    float E[S][V], SR[S][V], MS[S][V], SI[S][V], P[V], H[V], G[V];
    auto fold = [&](auto tag) {
      constexpr bool SLOW = decltype(tag)::value;
#pragma unroll
      for (int v = 0; v < V; ++v) P[v] = 1.0f, H[v] = 0.0f, G[v] = 0.0f;
#pragma unroll
      for (int s = 0; s < S; ++s) {
        float r[V], i[V], x[V];
        unpack<T, V>(rr[s], r);
        unpack<T, V>(ri[s], i);
        unpack<T, V>(rx[s], x);
        const bool reset = SLOW && (z >> s & 1);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const Gate g = gate<SLOW>(r[v], i[v], rate[v], reset);
          E[s][v] = g.e;
          SR[s][v] = g.sr;
          MS[s][v] = g.ms;
          // sigmoid(inp) = q w^2 s
          SI[s][v] = g.q * g.w * g.ms;
          if (SLOW && s >= n) E[s][v] = 0.0f, MS[s][v] = 0.0f;
          const float A = 1.0f - E[s][v], b = MS[s][v] * x[v];
          H[v] = reset ? b : fmaf(A, H[v], b);
          P[v] = reset ? -0.0f : P[v] * A;
        }
      }
#pragma unroll
      for (int s = S - 1; s >= 0; --s) {
        float g[V];
        unpack<T, V>(rg[s], g);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float A = 1.0f - E[s][v];
          G[v] = SLOW && (z >> s & 1) ? 0.0f : A * (G[v] + g[v]);
        }
      }
    };
    if (slow) fold(std::true_type{});
    else fold(std::false_type{});

#pragma unroll
    for (int v = 0; v < V; ++v) {
      agg[par][slot + wt][v * 32 + lane] = make_float2(P[v], H[v]);
      back[par][slot + wt][v * 32 + lane] = G[v];
    }
    __syncthreads();
    if (ranks > 1) {
      float cp[V], cg[V];
#pragma unroll
      for (int v = 0; v < V; ++v) {
        cp[v] = agg[par][slot + W - 1][v * 32 + lane].x;
        cg[v] = back[par][slot + W - 1][v * 32 + lane];
        for (int w = W - 2; w >= 0; --w) {
          const float p = agg[par][slot + w][v * 32 + lane].x;
          cg[v] = through(p, back[par][slot + w][v * 32 + lane], cg[v]);
          cp[v] = __float_as_int(p) < 0 ? p : p * cp[v];
        }
      }
      for (uint32_t r = wt; r < ranks; r += W)
#pragma unroll
        for (int v = 0; v < V; ++v)
          store_pair_at(&cagg[par][rank][v * 32 + lane], r, make_float2(cp[v], cg[v]));
      cluster_barrier();
    }
    float g[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      // the state before this warp's steps
      for (int w = 0; w < wt; ++w) {
        const float2 f = agg[par][slot + w][v * 32 + lane];
        h[v] = through(f.x, f.y, h[v]);
      }
      // gamma after this warp's steps
      float in = gam[v];
      if (ranks > 1) {
        for (uint32_t r = 0; r < ranks; ++r) {
          if (r == rank) in = gam[v];
          const float2 f = cagg[par][r][v * 32 + lane];
          gam[v] = through(f.x, f.y, gam[v]);
        }
      }
      g[v] = in;
      for (int w = W - 1; w >= 0; --w) {
        if (w == wt) g[v] = in;
        in = through(agg[par][slot + w][v * 32 + lane].x, back[par][slot + w][v * 32 + lane], in);
      }
      if (ranks == 1) gam[v] = in;
    }
    float before[S][V];
#pragma unroll
    for (int s = 0; s < S; ++s) {
      float x[V];
      unpack<T, V>(rx[s], x);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const float b = MS[s][v] * x[v];
        const bool reset = slow && (z >> s & 1);
        before[s][v] = reset ? 0.0f : h[v];
        h[v] = reset ? b : fmaf(1.0f - E[s][v], h[v], b);
      }
    }
#pragma unroll
    for (int s = S - 1; s >= 0; --s) {
      float x[V], d[V], ox[V], orec[V], oinp[V];
      unpack<T, V>(rx[s], x);
      unpack<T, V>(rg[s], d);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const bool reset = slow && (z >> s & 1);
        const float e = E[s][v], A = 1.0f - e;
        const float sq = max_nan(fmaf(-e, e, 2.0f * e), kTinySquare);
        const float gt = d[v] + g[v];
        const float gm = gt * MS[s][v];
        // g (h a - sigmoid(inp) x a^2 / m), and a^2 / m = (m / s) a^2
        const float q = reset ? 0.0f
                              : A * (gt * before[s][v] - gm * x[v] * A * rcp(sq));
        ox[v] = gm;
        oinp[v] = gm * x[v] * (1.0f - SI[s][v]);
        const float sq_r = SR[s][v] * q;
        orec[v] = -rate[v] * (1.0f - SR[s][v]) * sq_r;
        if (s < n) dl[v] += sq_r;
        g[v] = reset ? 0.0f : A * gt;
      }
      if (s < n && at.live) {
        store_vec<T, V>(dxp + (t0 + s) * a.dxt, ox);
        store_vec<T, V>(drp + (t0 + s) * a.drt, orec);
        store_vec<T, V>(dip + (t0 + s) * a.dit, oinp);
      }
    }
  }
  // the block's sum for dlam
  __syncthreads();
#pragma unroll
  for (int v = 0; v < V; ++v) back[0][slot + wt][v * 32 + lane] = dl[v];
  __syncthreads();
  if (wt == 0 && at.live) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      for (int w = 1; w < W; ++w) dl[v] += back[0][slot + w][v * 32 + lane];
      a.part[((int64_t)rank * a.B + at.b) * a.D + at.d + v] = dl[v];
      if (a.dh0 && rank == 0) a.dh0[at.b * a.D + at.d + v] = gam[v];
    }
  }
}

// dlam = -c sigmoid(lam) * (column sums of part [rows, D]): a cluster takes 32
// columns, its blocks every ranks-th stretch of rows; all sums in a fixed order.
__global__ void __launch_bounds__(1024) scan_dlam_kernel(const float *part, const float *lam,
                                                         int64_t rows, int64_t D, float c,
                                                         float *dlam) {
  __shared__ float buf[32][33];
  __shared__ float2 whole[kMaxCluster][32];
  const uint32_t ranks = cluster_size(), rank = cluster_rank();
  const int lane = threadIdx.x & 31, wy = threadIdx.x >> 5;
  const int64_t d = (int64_t)(blockIdx.x / ranks) * 32 + lane;
  if (ranks > 1) cluster_barrier();
  float s = 0.0f;
  if (d < D) {
#pragma unroll 4
    for (int64_t r = (int64_t)rank * 32 + wy; r < rows; r += (int64_t)ranks * 32)
      s += part[r * D + d];
  }
  buf[wy][lane] = s;
  __syncthreads();
  if (wy == 0) {
    s = 0.0f;
#pragma unroll
    for (int i = 0; i < 32; ++i) s += buf[i][lane];
    if (ranks > 1) store_pair_at(&whole[rank][lane], 0, make_float2(s, 0.0f));
  }
  if (ranks > 1) {
    cluster_barrier();
    if (wy == 0) {
      s = 0.0f;
      for (uint32_t r = 0; r < ranks; ++r) s += whole[r][lane].x;
    }
  }
  if (wy == 0 && rank == 0 && d < D) dlam[d] = -c * s / (1.0f + expf(-lam[d]));
}

// How a call is laid out.  T <= 64: ceil(T / 8) warps cover the whole row, and
// a block has as many groups of lanes as fit.  Longer rows: 64-step tiles, and
// where there are too few rows and channels for the SMs, clusters of up to 16
// blocks that share a row's tiles.
struct ScanPlan {
  int V, S, W, Z, ranks;
  int64_t units, tiles, blocks;
};

ScanPlan plan_scan(int64_t B, int64_t T, int64_t D, int V) {
  ScanPlan p{};
  p.V = V;
  p.S = T <= 1 ? 1 : kSteps;
  p.W = (int)std::min<int64_t>(kWarps, std::max<int64_t>(1, (T + p.S - 1) / p.S));
  p.Z = kWarps / p.W;
  p.units = B * (D / V);
  p.tiles = (T + p.W * p.S - 1) / (p.W * p.S);
  const int64_t groups = (p.units + 31) / 32;
  p.Z = (int)std::max<int64_t>(1, std::min<int64_t>(p.Z, groups));
  const int64_t base = (groups + p.Z - 1) / p.Z;
  p.ranks = 1;
  if (p.Z == 1)
    while (p.ranks < kMaxCluster && base * p.ranks < 2 * 148 && p.tiles >= 2 * p.ranks)
      p.ranks *= 2;
  p.blocks = base * p.ranks;
  return p;
}

template <typename K, typename... A>
cudaError_t launch_cluster(K kernel, unsigned blocks, dim3 threads, int ranks, cudaStream_t st,
                           A... args) {
  if (ranks > 8) {
    const cudaError_t e =
        cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = threads;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)ranks;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

int64_t chunk_starts(int64_t T) { return T > 0 ? (T - 1) / kChunk : 0; }

// Whether pairs of channels can be read and written as one access.
bool pairs_fit(std::initializer_list<const void *> ptrs, const int64_t *strides, int n, int64_t D,
               int es) {
  if (D % 2) return false;
  for (const void *p : ptrs)
    if (!aligned(p, 2 * es)) return false;
  for (int i = 0; i < n; ++i)
    if (strides[i] % 2) return false;
  return true;
}

template <typename F>
void with_plan(int32_t dtype, const ScanPlan &p, F &&f) {
  using std::integral_constant;
  with_dtype(dtype, [&](auto t) {
    if (p.V == 2 && p.S == 1) f(t, integral_constant<int, 2>{}, integral_constant<int, 1>{});
    else if (p.V == 2) f(t, integral_constant<int, 2>{}, integral_constant<int, kSteps>{});
    else if (p.S == 1) f(t, integral_constant<int, 1>{}, integral_constant<int, 1>{});
    else f(t, integral_constant<int, 1>{}, integral_constant<int, kSteps>{});
  });
}

zrl_status scan_launched(const char *what, cudaError_t e) {
  if (e == cudaSuccess) return seq_launched(what);
  (void)cudaGetLastError();  // reported here
  return seq_fail(ZRL_CUDA_ERROR, "%s: %s", what, cudaGetErrorString(e));
}

zrl_status check_scan(const char *what, int64_t B, int64_t T, int64_t D, int32_t dtype, float c) {
  if (B < 0 || T < 0 || D < 0) return seq_fail(ZRL_INVALID_ARG, "%s: a negative size", what);
  if (!dtype_ok(dtype)) return seq_fail(ZRL_INVALID_ARG, "%s: unknown dtype %d", what, dtype);
  if (!(c > 0.0f) || isinf(c)) return seq_fail(ZRL_INVALID_ARG, "%s: c > 0, finite", what);
  return ZRL_OK;
}

void scan_inputs(ScanArgs &a, const void *x, const void *rec, const void *inp, const float *lam,
                 const float *h0, const uint8_t *resets, int64_t B, int64_t T, int64_t D, float c,
                 const int64_t *strides) {
  a.x = x;
  a.rec = rec;
  a.inp = inp;
  a.lam = lam;
  a.h0 = h0;
  a.resets = resets;
  a.B = B;
  a.T = T;
  a.D = D;
  a.K = chunk_starts(T);
  a.c = c;
  a.xb = strides ? strides[0] : T * D;
  a.xt = strides ? strides[1] : D;
  a.rb = strides ? strides[2] : T * D;
  a.rt = strides ? strides[3] : D;
  a.ib = strides ? strides[4] : T * D;
  a.it = strides ? strides[5] : D;
  a.zb = strides ? strides[6] : T;
  a.zt = strides ? strides[7] : 1;
}

}  // namespace
}  // namespace zrl

using namespace zrl;

extern "C" int64_t zrl_gated_scan_carry(int64_t B, int64_t T, int64_t D) {
  return B > 0 && D > 0 ? B * chunk_starts(T) * D : 0;
}

extern "C" zrl_status zrl_gated_scan(const void *x, const void *rec, const void *inp,
                                     const float *lam, const float *h0, const uint8_t *resets,
                                     int64_t B, int64_t T, int64_t D, int32_t dtype, float c,
                                     const int64_t *strides, void *h, float *h_last,
                                     float *carry, void *stream) {
  const zrl_status s = check_scan("gated_scan", B, T, D, dtype, c);
  if (s != ZRL_OK) return s;
  if (B == 0 || D == 0) return ZRL_OK;
  if (!lam || (T && (!x || !rec || !inp || !h)))
    return seq_fail(ZRL_INVALID_ARG, "gated_scan: x, rec, inp, lam or h is NULL");
  const int es = dtype_size(dtype);
  if (!aligned(x, es) || !aligned(rec, es) || !aligned(inp, es) || !aligned(h, es) ||
      !aligned(lam, 4) || !aligned(h0, 4) || !aligned(h_last, 4) || !aligned(carry, 4))
    return seq_fail(ZRL_INVALID_ARG, "gated_scan: a pointer is not aligned to its element");
  ScanArgs a{};
  scan_inputs(a, x, rec, inp, lam, h0, resets, B, T, D, c, strides);
  a.h = h;
  a.hb = strides ? strides[8] : T * D;
  a.ht = strides ? strides[9] : D;
  a.h_last = h_last;
  a.carry = a.K ? carry : nullptr;
  const int64_t str[] = {a.xb, a.xt, a.rb, a.rt, a.ib, a.it, a.hb, a.ht};
  const ScanPlan p = plan_scan(B, T, D, pairs_fit({x, rec, inp, h}, str, 8, D, es) ? 2 : 1);
  if (p.blocks > 0x7fffffff) return seq_fail(ZRL_NOT_SUPPORTED, "gated_scan: B * D too large");
  a.units = p.units;
  a.tiles = p.tiles;
  cudaError_t e = cudaSuccess;
  with_plan(dtype, p, [&](auto t, auto v, auto s) {
    e = launch_cluster(scan_kernel<decltype(t), decltype(v)::value, decltype(s)::value>,
                       (unsigned)p.blocks, dim3(32, p.W, p.Z), p.ranks,
                       static_cast<cudaStream_t>(stream), a);
  });
  return scan_launched("gated_scan", e);
}

extern "C" int64_t zrl_gated_scan_grad_workspace(int64_t B, int64_t T, int64_t D) {
  if (B <= 0 || D <= 0) return 0;
  // dlam's sums, one per row, channel and block of a cluster
  const int ranks = std::max(plan_scan(B, T, D, 1).ranks, plan_scan(B, T, D, 2).ranks);
  return B * D * ranks * (int64_t)sizeof(float);
}

extern "C" zrl_status zrl_gated_scan_grad(
    const void *x, const void *rec, const void *inp, const float *lam, const float *h0,
    const uint8_t *resets, const float *carry, const void *dh, const float *dh_last, int64_t B,
    int64_t T, int64_t D, int32_t dtype, float c, const int64_t *strides, void *dx, void *drec,
    void *dinp, float *dlam, float *dh0, void *workspace, int64_t workspace_bytes,
    void *stream) {
  const zrl_status s = check_scan("gated_scan_grad", B, T, D, dtype, c);
  if (s != ZRL_OK) return s;
  if (D == 0) return ZRL_OK;
  if (!lam || !dlam || (B && T && (!x || !rec || !inp || !dh || !dx || !drec || !dinp)))
    return seq_fail(ZRL_INVALID_ARG, "gated_scan_grad: a required pointer is NULL");
  if (B && chunk_starts(T) && !carry)
    return seq_fail(ZRL_INVALID_ARG,
                    "gated_scan_grad: more than %d steps need the forward call's carry", kChunk);
  const int es = dtype_size(dtype);
  if (!aligned(x, es) || !aligned(rec, es) || !aligned(inp, es) || !aligned(dh, es) ||
      !aligned(dx, es) || !aligned(drec, es) || !aligned(dinp, es) || !aligned(lam, 4) ||
      !aligned(h0, 4) || !aligned(carry, 4) || !aligned(dh_last, 4) || !aligned(dlam, 4) ||
      !aligned(dh0, 4) || !aligned(workspace, 16))
    return seq_fail(ZRL_INVALID_ARG, "gated_scan_grad: a pointer is not aligned to its element");
  if (workspace_bytes < zrl_gated_scan_grad_workspace(B, T, D) || (B && !workspace))
    return seq_fail(ZRL_INVALID_ARG, "gated_scan_grad: workspace too small");
  ScanArgs a{};
  scan_inputs(a, x, rec, inp, lam, h0, resets, B, T, D, c, strides);
  a.carry = const_cast<float *>(carry);
  a.dh = dh;
  a.dh_last = dh_last;
  a.dx = dx;
  a.drec = drec;
  a.dinp = dinp;
  a.dh0 = dh0;
  a.part = static_cast<float *>(workspace);
  a.gb = strides ? strides[8] : T * D;
  a.gt = strides ? strides[9] : D;
  a.dxb = strides ? strides[10] : T * D;
  a.dxt = strides ? strides[11] : D;
  a.drb = strides ? strides[12] : T * D;
  a.drt = strides ? strides[13] : D;
  a.dib = strides ? strides[14] : T * D;
  a.dit = strides ? strides[15] : D;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int64_t str[] = {a.xb,  a.xt,  a.rb,  a.rt,  a.ib,  a.it,  a.gb,
                         a.gt,  a.dxb, a.dxt, a.drb, a.drt, a.dib, a.dit};
  const ScanPlan p =
      plan_scan(B, T, D, pairs_fit({x, rec, inp, dh, dx, drec, dinp}, str, 14, D, es) ? 2 : 1);
  if (p.blocks > 0x7fffffff)
    return seq_fail(ZRL_NOT_SUPPORTED, "gated_scan_grad: B * D too large");
  a.units = p.units;
  a.tiles = p.tiles;
  cudaError_t e = cudaSuccess;
  if (B)
    with_plan(dtype, p, [&](auto t, auto v, auto s) {
      e = launch_cluster(scan_grad_kernel<decltype(t), decltype(v)::value, decltype(s)::value>,
                         (unsigned)p.blocks, dim3(32, p.W, p.Z), p.ranks, st, a);
    });
  if (e == cudaSuccess) {
    const int64_t rows = B * p.ranks;
    const int ranks = rows >= 1024 ? 8 : 1;
    e = launch_cluster(scan_dlam_kernel, (unsigned)((D + 31) / 32 * ranks), dim3(1024), ranks, st,
                       (const float *)a.part, lam, rows, D, c, dlam);
  }
  return scan_launched("gated_scan_grad", e);
}
