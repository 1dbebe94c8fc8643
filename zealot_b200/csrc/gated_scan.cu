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
#include <type_traits>

#include "seq_common.cuh"

#ifndef ROWS_GROUPS
#define ROWS_GROUPS 148 * 16
#endif
namespace zrl {
namespace {

constexpr int kSteps = 8;       // steps of a stretch
constexpr int kWarps = 8;       // warps of a block at most
constexpr int kMaxCluster = 16;
// The forward call keeps the state before every stretch after the first; the
// gradient recomputes the states inside a stretch from there.
constexpr int kChunk = kSteps;
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
  int64_t xb, rb, ib, zb, zt, hb, gb, dxb, drb, dib;  // strides, elements
  int32_t xt, rt, it, ht, gt, dxt, drt, dit;          // strides along time, bytes
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
// long memory do not add up in one direction, and s = 1 - a^2 = e (2 - e)
// keeps its digits where a is near 1.  Above (only SLOW looks), a comes from
// ex2.  exp(-rec) is held to 2^126 and s to at least 2^-120, so nothing
// overflows or divides by zero.
struct Decay {
  float sr, e;  // sigmoid(rec), 1 - a
};
template <bool SLOW>
__device__ __forceinline__ Decay decay(float rec, float rate, bool reset) {
  Decay g;
  g.sr = rcp(1.0f + ex2(min_nan(rec * -kLog2e, 126.0f)));
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
  return g;
}
// m sigmoid(inp) = s w with w = 1 / sqrt(s q^2), q = 1 + exp(-inp): one
// reciprocal square root for the square root and the quotient.  exp(-inp) is
// held to 2^60.
struct Feed {
  float ms, w, q;
};
__device__ __forceinline__ Feed feed(float inp, float e) {
  Feed f;
  f.q = 1.0f + ex2(min_nan(inp * -kLog2e, 60.0f));
  const float s = max_nan(fmaf(-e, e, 2.0f * e), kTinySquare);
  f.w = rsq(s * f.q * f.q);
  f.ms = s * f.w;
  return f;
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

// Element (row b, step t, channel d) of a [B, T, D] tensor; the steps of a stretch
// follow by adding the stride.
template <typename T>
__device__ __forceinline__ const char *at_step(const void *p, int64_t b, int64_t sb, int64_t t,
                                               int32_t st, int64_t d) {
  return static_cast<const char *>(p) + (b * sb + d) * (int64_t)sizeof(T) + t * st;
}
template <typename T, int V>
__device__ __forceinline__ Raw<T, V> load_step(const char *p) {
  return *reinterpret_cast<const Raw<T, V> *>(p);
}
template <typename T, int V>
__device__ __forceinline__ void store_step(const char *p, const float *v) {
  *reinterpret_cast<Raw<T, V> *>(const_cast<char *>(p)) = pack<T, V>(v);
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
#pragma unroll 1
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

template <int V>
__device__ __forceinline__ bool load_rates(const ScanArgs &a, const Place<V> &at, float *rate) {
  bool big = false;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    rate[v] = a.c * softplus(a.lam[at.d + v]);
    big |= rate[v] > kSeriesMax;
  }
  return __any_sync(0xffffffffu, big);
}

// Rows in one piece: a thread takes its V channels through all steps, with the
// loads of the S steps ahead in flight.
template <typename T, int V, int S>
__global__ void __launch_bounds__(256) scan_rows_kernel(const __grid_constant__ ScanArgs a) {
  const Place<V> at(a, ((int64_t)blockIdx.x * blockDim.z + threadIdx.z) * 32 + threadIdx.x);
  Raw<T, V> rr[S], ri[S], rx[S];
  const char *rp = at_step<T>(a.rec, at.b, a.rb, 0, a.rt, at.d);
  const char *ip = at_step<T>(a.inp, at.b, a.ib, 0, a.it, at.d);
  const char *xp = at_step<T>(a.x, at.b, a.xb, 0, a.xt, at.d);
#pragma unroll
  for (int s = 0; s < S; ++s) {
    rr[s] = ri[s] = rx[s] = Raw<T, V>{};
    if (s < a.T) {
      rr[s] = load_step<T, V>(rp);
      ri[s] = load_step<T, V>(ip);
      rx[s] = load_step<T, V>(xp);
    }
    rp += a.rt, ip += a.it, xp += a.xt;
  }
  float h[V], rate[V];
#pragma unroll
  for (int v = 0; v < V; ++v) h[v] = a.h0 ? a.h0[at.b * a.D + at.d + v] : 0.0f;
  const bool big = load_rates<V>(a, at, rate);
  const char *hp = at_step<T>(a.h, at.b, a.hb, 0, a.ht, at.d);
  for (int64_t t0 = 0; t0 < a.T; t0 += S) {
    const int n = (int)min((int64_t)S, a.T - t0);
    const int ahead = (int)max((int64_t)0, min((int64_t)S, a.T - t0 - S));
    const uint32_t z = reset_bits(a, at.b, t0, n, at.one_row);
    if (a.carry && t0 && at.live) {
#pragma unroll
      for (int v = 0; v < V; ++v)
        a.carry[(at.b * a.K + t0 / kChunk - 1) * a.D + at.d + v] = h[v];
    }
    auto run = [&](auto tag) {
      constexpr bool SLOW = decltype(tag)::value;
#pragma unroll
      for (int s = 0; s < S; ++s) {
        if (SLOW && s >= n) break;
        float r[V], i[V], x[V];
        unpack<T, V>(rr[s], r);
        unpack<T, V>(ri[s], i);
        unpack<T, V>(rx[s], x);
        if (s < ahead) {
          rr[s] = load_step<T, V>(rp);
          ri[s] = load_step<T, V>(ip);
          rx[s] = load_step<T, V>(xp);
          rp += a.rt, ip += a.it, xp += a.xt;
        }
        const bool reset = SLOW && (z >> s & 1);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float e = decay<SLOW>(r[v], rate[v], reset).e;
          const float b = feed(i[v], e).ms * x[v];
          h[v] = reset ? b : fmaf(1.0f - e, h[v], b);
        }
        if (at.live) store_step<T, V>(hp, h);
        hp += a.ht;
      }
    };
    if (big || n < S || __any_sync(0xffffffffu, z != 0)) run(std::true_type{});
    else run(std::false_type{});
  }
  if (a.h_last && at.live) {
#pragma unroll
    for (int v = 0; v < V; ++v) a.h_last[at.b * a.D + at.d + v] = h[v];
  }
}

// Too few rows and channels for that: blocks of 32 lanes x W warps along time
// x Z groups of lanes.  A tile is W stretches of S steps: every warp folds its
// stretch from a zero state in registers to (P, H); the fold threads (one per
// channel) run through the warps' pairs and give each warp the state before
// its stretch; every warp then runs its steps again from there and stores
// them.  In a cluster the blocks take neighbouring tiles and exchange their
// pairs through distributed shared memory.  One pass over the data; the next
// tile's loads are in flight during the exchange.
template <typename T, int V, int S>
__global__ void __launch_bounds__(256, 2) scan_tile_kernel(const __grid_constant__ ScanArgs a) {
  __shared__ float2 agg[kWarps][32 * V];
  __shared__ float pre[kWarps][32 * V];
  __shared__ float2 cagg[2][kMaxCluster][32 * V];
  const int lane = threadIdx.x, wt = threadIdx.y, W = blockDim.y;
  const int slot = threadIdx.z * W;
  const uint32_t ranks = cluster_size(), rank = cluster_rank();
  const Place<V> at(a, ((int64_t)(blockIdx.x / ranks) * blockDim.z + threadIdx.z) * 32 + lane);
  Raw<T, V> rr[S], ri[S], rx[S];
  auto load = [&](int64_t t0, int n) {
    const char *r0 = at_step<T>(a.rec, at.b, a.rb, t0, a.rt, at.d);
    const char *i0 = at_step<T>(a.inp, at.b, a.ib, t0, a.it, at.d);
    const char *x0 = at_step<T>(a.x, at.b, a.xb, t0, a.xt, at.d);
#pragma unroll
    for (int s = 0; s < S; ++s) {
      if (s < n) {
        rr[s] = load_step<T, V>(r0);
        ri[s] = load_step<T, V>(i0);
        rx[s] = load_step<T, V>(x0);
        r0 += a.rt, i0 += a.it, x0 += a.xt;
      }
    }
  };
  auto steps = [&](int64_t t0) {
    return (int)max((int64_t)0, min((int64_t)S, a.T - t0));
  };
#pragma unroll
  for (int s = 0; s < S; ++s) rr[s] = ri[s] = rx[s] = Raw<T, V>{};
  int64_t t0 = ((int64_t)rank * W + wt) * S;
  int n = steps(t0);
  load(t0, n);
  uint32_t z = reset_bits(a, at.b, t0, n, at.one_row);
  float rate[V], carry[V];
#pragma unroll
  for (int v = 0; v < V; ++v) carry[v] = a.h0 ? a.h0[at.b * a.D + at.d + v] : 0.0f;
  const bool big = load_rates<V>(a, at, rate);
  if (ranks > 1) cluster_barrier();  // every block of the cluster runs

  int par = 0;
  for (int64_t k0 = 0; k0 < a.tiles; k0 += ranks, par ^= 1) {
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
          const float e = decay<SLOW>(r[v], rate[v], reset).e;
          A[s][v] = 1.0f - e;
          Bv[s][v] = feed(i[v], e).ms * x[v];
          if (SLOW && s >= n) A[s][v] = 1.0f, Bv[s][v] = 0.0f;
          H[v] = reset ? Bv[s][v] : fmaf(A[s][v], H[v], Bv[s][v]);
          P[v] = reset ? -0.0f : P[v] * A[s][v];
        }
      }
    };
    const bool slow = big || n < S || __any_sync(0xffffffffu, z != 0);
    if (slow) fold(std::true_type{});
    else fold(std::false_type{});
    const int64_t t_now = t0;
    const int n_now = n;
    const uint32_t z_now = z;
    t0 += (int64_t)ranks * W * S;
    n = steps(t0);
    load(t0, n);
    z = reset_bits(a, at.b, t0, n, at.one_row);

#pragma unroll
    for (int v = 0; v < V; ++v) agg[slot + wt][v * 32 + lane] = make_float2(P[v], H[v]);
    __syncthreads();
    if (ranks > 1) {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        if (v % W != wt) continue;
        // this block's (P, H), to every block
        const int c = v * 32 + lane;
        float2 f = agg[slot][c];
        for (int w = 1; w < W; ++w) {
          const float2 g = agg[slot + w][c];
          f.y = through(g.x, g.y, f.y);
          f.x = __float_as_int(g.x) < 0 ? g.x : g.x * f.x;
        }
        for (uint32_t r = 0; r < ranks; ++r) store_pair_at(&cagg[par][rank][c], r, f);
      }
      cluster_barrier();
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
      if (v % W != wt) continue;
      const int c = v * 32 + lane;
      float h = carry[v];
      if (ranks > 1) {
        for (uint32_t r = 0; r < ranks; ++r) {
          if (r == rank) h = carry[v];
          const float2 f = cagg[par][r][c];
          carry[v] = through(f.x, f.y, carry[v]);
        }
      }
      for (int w = 0; w < W; ++w) {
        pre[slot + w][c] = h;
        const float2 f = agg[slot + w][c];
        h = through(f.x, f.y, h);
      }
      if (ranks == 1) carry[v] = h;
    }
    __syncthreads();
    float h[V];
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = pre[slot + wt][v * 32 + lane];
    if (a.carry && t_now && n_now && at.live) {
#pragma unroll
      for (int v = 0; v < V; ++v)
        a.carry[(at.b * a.K + t_now / kChunk - 1) * a.D + at.d + v] = h[v];
    }
    const char *h0 = at_step<T>(a.h, at.b, a.hb, t_now, a.ht, at.d);
    if (slow) {
#pragma unroll
      for (int s = 0; s < S; ++s) {
#pragma unroll
        for (int v = 0; v < V; ++v)
          h[v] = z_now >> s & 1 ? Bv[s][v] : fmaf(A[s][v], h[v], Bv[s][v]);
        if (s < n_now && at.live) store_step<T, V>(h0, h);
        h0 += a.ht;
      }
    } else {
#pragma unroll
      for (int s = 0; s < S; ++s) {
#pragma unroll
        for (int v = 0; v < V; ++v) h[v] = fmaf(A[s][v], h[v], Bv[s][v]);
        if (at.live) store_step<T, V>(h0, h);
        h0 += a.ht;
      }
    }
  }
  if (a.h_last && rank == 0 && at.live) {
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (v % W == wt) a.h_last[at.b * a.D + at.d + v] = carry[v];
  }
}

// The gradient, stretch by stretch from the end.  Backwards through a stretch,
// g_t = dh_t + gamma_{t+1}, gamma_t = a_t g_t, from the decays alone; then
// forwards, with the states running on from the kept one and every output made
// as its step comes by.  So every gate is computed once and only a, sigmoid(rec)
// and g of a stretch are held.
//
// Rows in one piece (TILED false): a thread takes its channels through all
// stretches.  Else the warps of a block take the stretches of a tile, and the
// blocks of a cluster neighbouring tiles, the last first; the pairs (P, gamma
// from zero) are exchanged as in scan_tile_kernel.
template <typename T, int V, int S, bool TILED>
__global__ void __launch_bounds__(256, 2)
    scan_grad_kernel(const __grid_constant__ ScanArgs a) {
  __shared__ float2 agg[TILED ? kWarps : 1][32 * V];  // (P, gamma of a stretch from zero)
  __shared__ float pre[TILED ? kWarps : 1][32 * V];   // gamma after a warp's stretch
  __shared__ float2 cagg[2][TILED ? kMaxCluster : 1][32 * V];
  const int lane = threadIdx.x, wt = TILED ? threadIdx.y : 0, W = TILED ? blockDim.y : 1;
  const int slot = TILED ? threadIdx.z * W : 0;
  const uint32_t ranks = TILED ? cluster_size() : 1, rank = TILED ? cluster_rank() : 0;
  const Place<V> at(a, ((int64_t)(blockIdx.x / ranks) * blockDim.z + threadIdx.z) * 32 + lane);
  Raw<T, V> rr[S], ri[S], rx[S], rg[S];
  float h[V];
  auto steps = [&](int64_t t0) {
    return t0 < 0 ? 0 : (int)max((int64_t)0, min((int64_t)S, a.T - t0));
  };
  auto load_back = [&](int64_t t0, int n) {
    const char *r0 = at_step<T>(a.rec, at.b, a.rb, t0, a.rt, at.d);
    const char *g0 = at_step<T>(a.dh, at.b, a.gb, t0, a.gt, at.d);
#pragma unroll
    for (int s = 0; s < S; ++s) {
      if (s < n) {
        rr[s] = load_step<T, V>(r0);
        rg[s] = load_step<T, V>(g0);
        r0 += a.rt, g0 += a.gt;
      }
    }
  };
  auto load_fwd = [&](int64_t t0, int n) {
    const char *i0 = at_step<T>(a.inp, at.b, a.ib, t0, a.it, at.d);
    const char *x0 = at_step<T>(a.x, at.b, a.xb, t0, a.xt, at.d);
#pragma unroll
    for (int s = 0; s < S; ++s) {
      if (s < n) {
        ri[s] = load_step<T, V>(i0);
        rx[s] = load_step<T, V>(x0);
        i0 += a.it, x0 += a.xt;
      }
    }
    if (n) {
#pragma unroll
      for (int v = 0; v < V; ++v) {
        h[v] = 0.0f;
        if (t0 > 0) h[v] = a.carry[(at.b * a.K + t0 / kChunk - 1) * a.D + at.d + v];
        else if (a.h0) h[v] = a.h0[at.b * a.D + at.d + v];
      }
    }
  };
#pragma unroll
  for (int s = 0; s < S; ++s) rr[s] = ri[s] = rx[s] = rg[s] = Raw<T, V>{};
#pragma unroll
  for (int v = 0; v < V; ++v) h[v] = 0.0f;
  int64_t t0 = ((a.tiles - 1 - rank) * W + wt) * S;
  int n = steps(t0);
  load_back(t0, n);
  load_fwd(t0, n);
  uint32_t z = reset_bits(a, at.b, t0, n, at.one_row);
  float rate[V], gam[V], dl[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    gam[v] = a.dh_last ? a.dh_last[at.b * a.D + at.d + v] : 0.0f;
    dl[v] = 0.0f;
  }
  const bool big = load_rates<V>(a, at, rate);
  if (TILED && ranks > 1) cluster_barrier();

  int par = 0;
  for (int64_t k0 = a.tiles - 1; k0 >= 0; k0 -= ranks, par ^= 1) {
    const bool slow = big || n < S || __any_sync(0xffffffffu, z != 0);
    const int64_t t_now = t0;
    const int n_now = n;
    const uint32_t z_now = z;
    float E[S][V], SR[S][V], g[S][V];
    float P[V], in[V];
    auto back = [&](auto tag) {
      constexpr bool SLOW = decltype(tag)::value;
#pragma unroll
      for (int v = 0; v < V; ++v) P[v] = 1.0f, in[v] = 0.0f;
#pragma unroll
      for (int s = S - 1; s >= 0; --s) {
        float r[V];
        unpack<T, V>(rr[s], r);
        unpack<T, V>(rg[s], g[s]);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const bool reset = SLOW && (z_now >> s & 1);
          const Decay q = decay<SLOW>(r[v], rate[v], reset);
          E[s][v] = q.e;
          SR[s][v] = q.sr;
          if (SLOW && s >= n_now) E[s][v] = 0.0f, g[s][v] = 0.0f;
          if (TILED) {
            const float A = 1.0f - E[s][v];
            P[v] = reset ? -0.0f : P[v] * A;
            in[v] = reset ? 0.0f : A * (in[v] + g[s][v]);
          }
        }
      }
    };
    if (slow) back(std::true_type{});
    else back(std::false_type{});
    t0 -= (int64_t)ranks * W * S;
    n = steps(t0);
    load_back(t0, n);

    if (TILED) {
#pragma unroll
      for (int v = 0; v < V; ++v)
        agg[slot + wt][v * 32 + lane] =
            make_float2(slow && z_now ? -0.0f : P[v], in[v]);
      __syncthreads();
      if (ranks > 1) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
          if (v % W != wt) continue;
          const int c = v * 32 + lane;
          float2 f = agg[slot + W - 1][c];
          for (int w = W - 2; w >= 0; --w) {
            const float2 q = agg[slot + w][c];
            f.y = through(q.x, q.y, f.y);
            f.x = __float_as_int(q.x) < 0 ? q.x : q.x * f.x;
          }
          for (uint32_t r = 0; r < ranks; ++r) store_pair_at(&cagg[par][rank][c], r, f);
        }
        cluster_barrier();
      }
#pragma unroll
      for (int v = 0; v < V; ++v) {
        if (v % W != wt) continue;
        const int c = v * 32 + lane;
        float y = gam[v];
        if (ranks > 1) {
          for (uint32_t r = 0; r < ranks; ++r) {
            if (r == rank) y = gam[v];
            const float2 f = cagg[par][r][c];
            gam[v] = through(f.x, f.y, gam[v]);
          }
        }
        for (int w = W - 1; w >= 0; --w) {
          pre[slot + w][c] = y;
          const float2 f = agg[slot + w][c];
          y = through(f.x, f.y, y);
        }
        if (ranks == 1) gam[v] = y;
      }
      __syncthreads();
#pragma unroll
      for (int v = 0; v < V; ++v) in[v] = pre[slot + wt][v * 32 + lane];
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v) in[v] = gam[v];
    }

    const char *dx0 = at_step<T>(a.dx, at.b, a.dxb, t_now, a.dxt, at.d);
    const char *dr0 = at_step<T>(a.drec, at.b, a.drb, t_now, a.drt, at.d);
    const char *di0 = at_step<T>(a.dinp, at.b, a.dib, t_now, a.dit, at.d);
    auto finish = [&](auto tag) {
      constexpr bool SLOW = decltype(tag)::value;
#pragma unroll
      for (int s = S - 1; s >= 0; --s) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
          g[s][v] += in[v];
          in[v] = SLOW && (z_now >> s & 1) ? 0.0f : (1.0f - E[s][v]) * g[s][v];
        }
      }
      if (!TILED) {
#pragma unroll
        for (int v = 0; v < V; ++v) gam[v] = in[v];
      }
#pragma unroll
      for (int s = 0; s < S; ++s) {
        if (SLOW && s >= n_now) break;
        float i[V], x[V], ox[V], orec[V], oinp[V];
        unpack<T, V>(ri[s], i);
        unpack<T, V>(rx[s], x);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const bool reset = SLOW && (z_now >> s & 1);
          const float A = 1.0f - E[s][v];
          const Feed f = feed(i[v], E[s][v]);
          const float b = f.ms * x[v];
          ox[v] = g[s][v] * f.ms;
          const float gx = ox[v] * x[v];
          // 1 - sigmoid(inp) = (q - 1) / q and 1 / q = m s_i / m = ms w q
          const float wq = f.w * f.q;
          oinp[v] = gx * (1.0f - f.ms * wq);
          // g (h a - s_i x a^2 / m) = a (g h - g m s_i x a / s), 1 / s = (w q)^2
          const float q =
              reset ? 0.0f : A * fmaf(g[s][v], h[v], -(gx * A) * (wq * wq));
          const float sq = SR[s][v] * q;
          orec[v] = rate[v] * (SR[s][v] - 1.0f) * sq;
          dl[v] += sq;
          h[v] = reset ? b : fmaf(A, h[v], b);
        }
        if (at.live) {
          store_step<T, V>(dx0, ox);
          store_step<T, V>(dr0, orec);
          store_step<T, V>(di0, oinp);
        }
        dx0 += a.dxt, dr0 += a.drt, di0 += a.dit;
      }
    };
    if (slow) finish(std::true_type{});
    else finish(std::false_type{});
    load_fwd(t0, n);
    z = reset_bits(a, at.b, t0, n, at.one_row);
  }
  // the block's sum for dlam
  if (TILED) {
    __syncthreads();
#pragma unroll
    for (int v = 0; v < V; ++v) pre[slot + wt][v * 32 + lane] = dl[v];
    __syncthreads();
  }
  if (at.live) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      if (v % W != wt) continue;
      float s = dl[v];
      if (TILED) {
        const int c = v * 32 + lane;
        s = pre[slot][c];
        for (int w = 1; w < W; ++w) s += pre[slot + w][c];
      }
      a.part[((int64_t)rank * a.B + at.b) * a.D + at.d + v] = s;
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

// How a call is laid out.  Rows in one piece where their channels fill the
// SMs (or there is one stretch); else tiles: ceil(T / 8) warps cover a row of up
// to 64 steps, and a block has as many groups of lanes as fit; longer rows go
// by 64-step tiles, and where there are too few rows and channels for the SMs,
// clusters of up to 16 blocks share a row's tiles.
struct ScanPlan {
  bool rows;
  int V, S, W, Z, ranks;
  int64_t units, tiles, blocks;
};

ScanPlan plan_scan(int64_t B, int64_t T, int64_t D, int V) {
  ScanPlan p{};
  p.V = V;
  p.S = T <= 1 ? 1 : kSteps;
  p.units = B * (D / V);
  const int64_t groups = (p.units + 31) / 32;
  p.ranks = 1;
  p.rows = T <= kSteps || groups >= ROWS_GROUPS;
  if (p.rows) {
    p.W = 1;
    p.tiles = (T + p.S - 1) / p.S;
    p.Z = kWarps;
    p.blocks = (groups + p.Z - 1) / p.Z;
    return p;
  }
  p.W = (int)std::min<int64_t>(kWarps, (T + kSteps - 1) / kSteps);
  p.Z = (int)std::max<int64_t>(1, std::min<int64_t>(kWarps / p.W, groups));
  p.tiles = (T + p.W * kSteps - 1) / (p.W * kSteps);
  const int64_t base = (groups + p.Z - 1) / p.Z;
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

// A [B, T, D] tensor of a call: where its strides stand in the caller's array
// and in the kernel's arguments.
struct ScanTensor {
  const void *p;
  int at;
  int64_t *batch;
  int32_t *time;
};

// Fills in the strides; *pairs says whether pairs of channels can be read and
// written as one access.  False: a time stride does not fit 32 bits of bytes.
bool place_tensors(ScanTensor *ts, int n, const int64_t *strides, int64_t T, int64_t D, int es,
                   bool *pairs) {
  *pairs = D % 2 == 0;
  for (int i = 0; i < n; ++i) {
    const int64_t sb = strides ? strides[ts[i].at] : T * D;
    int64_t st = strides ? strides[ts[i].at + 1] : D;
    if (T <= 1) st = 0;  // one step: its stride is not used
    if (st > INT32_MAX / es || st < -(INT32_MAX / es)) return false;
    *ts[i].batch = sb;
    *ts[i].time = (int32_t)(st * es);
    if (sb % 2 || st % 2 || !aligned(ts[i].p, 2 * es)) *pairs = false;
  }
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
  a.h_last = h_last;
  a.carry = a.K ? carry : nullptr;
  ScanTensor ts[] = {{x, 0, &a.xb, &a.xt}, {rec, 2, &a.rb, &a.rt}, {inp, 4, &a.ib, &a.it},
                     {h, 8, &a.hb, &a.ht}};
  bool pairs = false;
  if (!place_tensors(ts, 4, strides, T, D, es, &pairs))
    return seq_fail(ZRL_NOT_SUPPORTED, "gated_scan: a time stride of 2 GiB or more");
  const ScanPlan p = plan_scan(B, T, D, pairs ? 2 : 1);
  if (p.blocks > 0x7fffffff) return seq_fail(ZRL_NOT_SUPPORTED, "gated_scan: B * D too large");
  a.units = p.units;
  a.tiles = p.tiles;
  cudaError_t e = cudaSuccess;
  with_plan(dtype, p, [&](auto t, auto v, auto s) {
    using E = decltype(t);
    constexpr int V = decltype(v)::value, S = decltype(s)::value;
    const dim3 threads(32, p.W, p.Z);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (p.rows) {
      scan_rows_kernel<E, V, S><<<(unsigned)p.blocks, threads, 0, st>>>(a);
      e = cudaGetLastError();
    } else if constexpr (S == kSteps) {
      e = launch_cluster(scan_tile_kernel<E, V, S>, (unsigned)p.blocks, threads, p.ranks, st, a);
    }
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
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  ScanTensor ts[] = {{x, 0, &a.xb, &a.xt},     {rec, 2, &a.rb, &a.rt},    {inp, 4, &a.ib, &a.it},
                     {dh, 8, &a.gb, &a.gt},    {dx, 10, &a.dxb, &a.dxt},  {drec, 12, &a.drb, &a.drt},
                     {dinp, 14, &a.dib, &a.dit}};
  bool pairs = false;
  if (!place_tensors(ts, 7, strides, T, D, es, &pairs))
    return seq_fail(ZRL_NOT_SUPPORTED, "gated_scan_grad: a time stride of 2 GiB or more");
  const ScanPlan p = plan_scan(B, T, D, pairs ? 2 : 1);
  if (p.blocks > 0x7fffffff)
    return seq_fail(ZRL_NOT_SUPPORTED, "gated_scan_grad: B * D too large");
  a.units = p.units;
  a.tiles = p.tiles;
  cudaError_t e = cudaSuccess;
  if (B)
    with_plan(dtype, p, [&](auto t, auto v, auto s) {
      using E = decltype(t);
      constexpr int V = decltype(v)::value, S = decltype(s)::value;
      const dim3 threads(32, p.W, p.Z);
      if (p.rows) {
        scan_grad_kernel<E, V, S, false><<<(unsigned)p.blocks, threads, 0, st>>>(a);
        e = cudaGetLastError();
      } else if constexpr (S == kSteps) {
        e = launch_cluster(scan_grad_kernel<E, V, S, true>, (unsigned)p.blocks, threads, p.ranks,
                           st, a);
      }
    });
  if (e == cudaSuccess) {
    const int64_t rows = B * p.ranks;
    const int ranks = rows >= 1024 ? 8 : 1;
    e = launch_cluster(scan_dlam_kernel, (unsigned)((D + 31) / 32 * ranks), dim3(1024), ranks, st,
                       (const float *)a.part, lam, rows, D, c, dlam);
  }
  return scan_launched("gated_scan_grad", e);
}
