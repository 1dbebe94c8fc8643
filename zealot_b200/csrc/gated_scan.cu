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

#include "column_sum.cuh"
#include "seq_common.cuh"

namespace zrl {
namespace {

constexpr int kSteps = 8;       // steps of a stretch
constexpr int kWarps = 8;       // warps of a block at most
constexpr int kMinSlab = 16;    // steps of a slab at least
// The forward call keeps the state before every stretch after the first; the
// gradient recomputes the states inside a stretch from there.
constexpr int kChunk = kSteps;
constexpr int kRun = 256;       // steps whose terms of dlam are summed one after the other
constexpr float kSeriesMax = 0.35f;
constexpr float kSmallest = 1.17549435e-38f;  // 2^-126

// Blocks of 256 threads an SM holds, which bounds their registers.  Measured
// (device us, 2 / 3 / 4 blocks): forward 1024 x 24 x 512 bf16 36 / 34 / 32, 4096 x
// 24 x 128 f32 42 / 48 / 55; gradient of the former 50 / 118 / -.  The fastest of
// them spill as well, less than they gain: bf16 pairs store / load 124 / 208 bytes a
// thread in scan_kernel, 140 / 144 in the first pass, 56 / 84 in the gradient.
template <typename T> constexpr int resident() { return sizeof(T) == 2 ? 4 : 2; }
// (f32's gradient takes one channel a lane: pairs spill, 78 against 106 us.)
constexpr int kGradResident = 2;

struct ScanArgs {
  const void *x, *rec, *inp, *dh;
  const float *lam, *h0, *dh_last;
  const uint8_t *resets;
  void *h, *dx, *drec, *dinp;
  float *h_last, *carry, *dh0, *part;
  float2 *fold;         // [slab blocks][B D], then [slabs][B D]
  int64_t B, T, D, K;   // K: stretches after the first
  int64_t units;        // units of V channels
  int64_t slab_steps;   // steps of a slab, a multiple of kSteps (one slab: T or more)
  int32_t slabs;
  int64_t xb, rb, ib, zb, zt, hb, gb, dxb, drb, dib;  // strides, elements
  int32_t xt, rt, it, ht, gt, dxt, drt, dit;          // strides along time, bytes
  float c;
  int32_t one;  // 1
};

// softplus(v) = max(v, 0) + log(1 + y), y = exp(-|v|), with
// log(1 + y) = 2 artanh(z), z = y / (2 + y) <= 1/3: its series to z^15 is within
// 2e-9 relative and keeps the digits of a small y.  7e-7 relative with ex2's
// and the quotient's roundings; the decays' logarithms scale with it.
__device__ __forceinline__ float softplus(float v) {
  const float y = ex2(-fabsf(v) * kLog2e);
  const float z = y * rcp(2.0f + y), z2 = z * z;
  float p = fmaf(z2, 1.0f / 15.0f, 1.0f / 13.0f);
  p = fmaf(z2, p, 1.0f / 11.0f);
  p = fmaf(z2, p, 1.0f / 9.0f);
  p = fmaf(z2, p, 1.0f / 7.0f);
  p = fmaf(z2, p, 1.0f / 5.0f);
  p = fmaf(z2, p, 1.0f / 3.0f);
  p = fmaf(z2, p, 1.0f);
  return (v > 0.0f ? v : v != v ? v : 0.0f) + 2.0f * z * p;
}

// What the steps of a stretch need looked at: nothing; marks and the stretch's
// end; those and rates beyond the series' range.
enum Way { kPlain, kMarks, kFar };
template <Way W> using Is = std::integral_constant<Way, W>;
// Whether scan_kernel has a path of its own for kMarks.  Device us with / without:
// 1024 x 24 x 512 bf16 32 / 35 (fewer spills), 4096 x 24 x 128 f32 44 / 42.  The fold
// and the gradient are faster without: 8 x 8191 x 480 bf16 62 / 61 and 128 / 125.
template <typename T> constexpr bool kMarksApart = sizeof(T) == 2;

// The gates of one step.  With u = rate sigmoid(rec), e = 1 - a = 1 - exp(-u)
// comes from its series up to u = 0.35 (seven terms, 2e-8 relative): a = 1 - e
// is then within half a unit of exp(-u) at every step, so the roundings of a
// long memory do not add up in one direction, and s = 1 - a^2 = e (2 - e)
// keeps its digits where a is near 1.  Above (only kFar looks), a comes from
// ex2, so that a small a keeps its digits too, and e = 1 - a from it.  exp(-rec)
// may be infinite: sigmoid(rec) and e are then 0.
template <int V>
struct Decay {
  Vec<V> sr, e, a;  // sigmoid(rec), 1 - a, a
};
template <Way WAY, int V>
__device__ __forceinline__ Decay<V> decay(const Vec<V> &rec, const Vec<V> &rate, bool reset) {
  Decay<V> g;
  Vec<V> t = mul(rec, -kLog2e);
#pragma unroll
  for (int v = 0; v < V; ++v) t[v] = ex2(t[v]);
  t = add(t, 1.0f);
#pragma unroll
  for (int v = 0; v < V; ++v) g.sr[v] = rcp(t[v]);
  const Vec<V> u = mul(rate, g.sr);
  Vec<V> p = fma(u, 1.0f / 5040.0f, -1.0f / 720.0f);
  p = fma(u, p, 1.0f / 120.0f);
  p = fma(u, p, -1.0f / 24.0f);
  p = fma(u, p, 1.0f / 6.0f);
  p = fma(u, p, -0.5f);
  p = fma(u, p, 1.0f);
  g.e = mul(u, p);
  if (WAY == kMarks && reset) g.e = all<V>(1.0f);
  g.a = fma(g.e, -1.0f, 1.0f);
  if (WAY == kFar) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      if (u[v] > kSeriesMax) {
        g.a[v] = ex2(u[v] * -kLog2e);
        g.e[v] = 1.0f - g.a[v];
      }
      if (reset) g.a[v] = 0.0f, g.e[v] = 1.0f;  // m = 1
    }
  }
  return g;
}
// a and e in one register a channel, without loss: e up to 1/2, where 1 - e is a
// to the last bit, else -a (an a of 0 as e = 1).
template <Way WAY, int V>
__device__ __forceinline__ Vec<V> hold(const Decay<V> &g) {
  Vec<V> k = g.e;
  if (WAY == kFar) {
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (g.e[v] > 0.5f && g.a[v] > 0.0f) k[v] = -g.a[v];
  }
  return k;
}
template <Way WAY, int V>
__device__ __forceinline__ void held(const Vec<V> &k, Vec<V> &e, Vec<V> &a) {
  e = k;
  a = fma(k, -1.0f, 1.0f);
  if (WAY == kFar) {
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (k[v] < 0.0f) a[v] = -k[v], e[v] = 1.0f + k[v];
  }
}
// s = 1 - a^2 and sigmoid(inp), each to a few units in its last place however nearly
// shut its gate: a reciprocal and a root of their own.  (One reciprocal square root of
// s (1 + exp(-inp))^2 for both overflows from inp = -45 down, and needs s held above 0.)
// exp(-inp) may be infinite: sigmoid(inp) is then 0.
template <int V>
__device__ __forceinline__ Vec<V> square(const Vec<V> &e, const Vec<V> &a) {
  return mul(e, add(a, 1.0f));
}
template <int V>
__device__ __forceinline__ Vec<V> gate(const Vec<V> &inp) {
  Vec<V> t = mul(inp, -kLog2e);
#pragma unroll
  for (int v = 0; v < V; ++v) t[v] = ex2(t[v]);
  t = add(t, 1.0f);
#pragma unroll
  for (int v = 0; v < V; ++v) t[v] = rcp(t[v]);
  return t;
}
// m sigmoid(inp)
template <int V>
__device__ __forceinline__ Vec<V> feed(const Vec<V> &inp, const Vec<V> &e, const Vec<V> &a) {
  Vec<V> m = square(e, a);
#pragma unroll
  for (int v = 0; v < V; ++v) m[v] = root(m[v]);
  return mul(m, gate(inp));
}

// A stretch of steps maps the state before it to h -> P h + H.  P is -0 where
// an episode begins inside: then nothing of h is used, infinity and NaN
// included.
__device__ __forceinline__ float through(float P, float H, float h) {
  return __float_as_int(P) < 0 ? H : fmaf(P, h, H);
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
__device__ __forceinline__ void store_step(const char *p, const Vec<V> &x) {
  *reinterpret_cast<Raw<T, V> *>(const_cast<char *>(p)) = pack<T, V>(x.v);
}

// p + stride as one multiply-add (one is 1, which the compiler cannot know).
__device__ __forceinline__ void advance(const char *&p, int32_t stride, int32_t one) {
  asm("mad.wide.s32 %0, %1, %2, %0;" : "+l"(p) : "r"(stride), "r"(one));
}

// The reset marks of steps t .. t + n - 1 of the lane's row, to be turned into
// bits (bit s for step s) where they are needed, so that their latency is not
// waited for.  A warp whose lanes share a row reads each mark once.
__device__ __forceinline__ uint32_t load_marks(const ScanArgs &a, int64_t b, int64_t t, int n,
                                               bool one_row) {
  if (!a.resets) return 0;
  const uint8_t *z = a.resets + b * a.zb + t * a.zt;
  if (one_row) return (int)threadIdx.x < n ? z[threadIdx.x * a.zt] : 0;
  uint32_t bits = 0;
#pragma unroll 1
  for (int s = 0; s < n; ++s) bits |= (z[s * a.zt] ? 1u : 0u) << s;
  return bits;
}
__device__ __forceinline__ uint32_t mark_bits(const ScanArgs &a, uint32_t marks, bool one_row) {
  if (!a.resets) return 0;
  return one_row ? __ballot_sync(0xffffffffu, marks != 0) : marks;
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
__device__ __forceinline__ bool load_rates(const ScanArgs &a, const Place<V> &at, Vec<V> &rate) {
  bool big = false;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    rate[v] = a.c * softplus(a.lam[at.d + v]);
    big |= rate[v] > kSeriesMax;
  }
  return __any_sync(0xffffffffu, big);
}

// Blocks of 32 lanes x 8 warps.  One slab: the warps take neighbouring groups of
// lanes.  Several: they take neighbouring slabs of one group.
struct Slab {
  int64_t group, begin, end;
  int32_t index;
  __device__ __forceinline__ explicit Slab(const ScanArgs &a) {
    if (a.slabs == 1) {
      group = (int64_t)blockIdx.x * kWarps + threadIdx.y;
      index = 0;
    } else {
      group = blockIdx.x;
      index = blockIdx.y * kWarps + threadIdx.y;
    }
    begin = index * a.slab_steps;
    end = min(a.T, begin + a.slab_steps);
  }
};

// What a slab does to the state before it (BACK: to the gradient after it), as a
// pair (P, H): every warp folds its slab, then the block writes, per warp, the
// pair of the block's slabs before (after) it, and the pair of them all.
// Bound by memory where elements have four bytes: 1 x 65536 x 512 f32 72 us (5.6
// TB/s).  Where they have two no unit is full: 8 x 8191 x 480 bf16 65 us (2.9 TB/s),
// backwards 43 us, the special functions at 66 and 43 % of their rate, 55 and 59 %
// of the issue slots, and warps that mostly wait for their loads.
template <typename T, int V, bool BACK>
__global__ void __launch_bounds__(256, resident<T>()) scan_fold_kernel(const __grid_constant__ ScanArgs a) {
  constexpr int S = kSteps;
  __shared__ float2 agg[kWarps][32 * V];
  const int lane = threadIdx.x, wt = threadIdx.y;
  const Slab slab(a);
  const Place<V> at(a, slab.group * 32 + lane);
  const int64_t steps = max((int64_t)0, slab.end - slab.begin);
  // in the order of the recurrence: forward from begin, or back from end - 1
  const int dir = BACK ? -1 : 1;
  const int64_t first = BACK ? slab.end - 1 : slab.begin;
  const char *rp = at_step<T>(a.rec, at.b, a.rb, first, a.rt, at.d);
  const char *ip = BACK ? at_step<T>(a.dh, at.b, a.gb, first, a.gt, at.d)
                        : at_step<T>(a.inp, at.b, a.ib, first, a.it, at.d);
  const char *xp = at_step<T>(a.x, at.b, a.xb, first, a.xt, at.d);
  const int32_t rt = dir * a.rt, it = BACK ? -a.gt : a.it, xt = a.xt;
  Raw<T, V> rr[S], ri[S], rx[S];
#pragma unroll
  for (int s = 0; s < S; ++s) {
    rr[s] = ri[s] = rx[s] = Raw<T, V>{};
    if (s < steps) {
      rr[s] = load_step<T, V>(rp);
      ri[s] = load_step<T, V>(ip);
      if (!BACK) rx[s] = load_step<T, V>(xp);
    }
    advance(rp, rt, a.one);
    advance(ip, it, a.one);
    if (!BACK) advance(xp, xt, a.one);
  }
  Vec<V> rate;
  const bool big = load_rates<V>(a, at, rate);
  Vec<V> P = all<V>(1.0f), H = all<V>(0.0f);
  // marks of the n steps that follow done steps, bit s for the lowest step
  auto marks_of = [&](int64_t done, int n) {
    return load_marks(a, at.b, BACK ? slab.end - done - n : slab.begin + done, n, at.one_row);
  };
  uint32_t marks = marks_of(0, (int)min((int64_t)S, steps));
  for (int64_t t = 0; t < steps; t += S) {
    const int n = (int)min((int64_t)S, steps - t);
    const int ahead = (int)max((int64_t)0, min((int64_t)S, steps - t - S));
    const uint32_t z = mark_bits(a, marks, at.one_row);
    marks = marks_of(t + S, ahead);
    auto run = [&](auto way, auto more) {
      constexpr Way WAY = decltype(way)::value;
      constexpr bool SLOW = WAY != kPlain, MORE = decltype(more)::value;
#pragma unroll
      for (int s = 0; s < S; ++s) {
        if (SLOW && s >= n) break;
        const Vec<V> r = values<T, V>(rr[s]), i = values<T, V>(ri[s]), x = values<T, V>(rx[s]);
        if (MORE || (SLOW && s < ahead)) {
          rr[s] = load_step<T, V>(rp);
          ri[s] = load_step<T, V>(ip);
          if (!BACK) rx[s] = load_step<T, V>(xp);
          advance(rp, rt, a.one);
          advance(ip, it, a.one);
          if (!BACK) advance(xp, xt, a.one);
        }
        const bool reset = SLOW && (z >> (BACK ? n - 1 - s : s) & 1);
        const Decay<V> g = decay<WAY>(r, rate, reset);
        if (BACK) {
          H = mul(g.a, add(H, i));
          if (reset) H = all<V>(0.0f);
        } else {
          const Vec<V> b = mul(feed(i, g.e, g.a), x);
          if (reset) H = b;
          else H = fma(g.a, H, b);
        }
        if (reset) P = all<V>(-0.0f);
        else P = mul(P, g.a);
      }
    };
    if (big || n < S || (ahead != 0 && ahead != S) || __any_sync(0xffffffffu, z != 0))
      run(Is<kFar>{}, std::false_type{});
    else if (ahead)
      run(Is<kPlain>{}, std::true_type{});
    else
      run(Is<kPlain>{}, std::false_type{});
  }
  let_next_start();
#pragma unroll
  for (int v = 0; v < V; ++v) agg[wt][v * 32 + lane] = make_float2(P[v], H[v]);
  __syncthreads();
  if (!at.live) return;
  float2 *whole = a.fold + (int64_t)blockIdx.y * a.B * a.D;
  float2 *own = a.fold + ((int64_t)gridDim.y + slab.index) * a.B * a.D;
  const int64_t c = at.b * a.D + at.d;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    float2 f = make_float2(1.0f, 0.0f);
    for (int i = 0; i < kWarps; ++i) {
      const int w = BACK ? kWarps - 1 - i : i;
      if (w == wt) own[c + v] = f;
      const float2 g = agg[w][v * 32 + lane];
      f.y = through(g.x, g.y, f.y);
      f.x = __float_as_int(g.x) < 0 ? g.x : g.x * f.x;
    }
    if (wt == 0) whole[c + v] = f;
  }
}

// The state before a slab (BACK: the gradient after it) from first, the state
// before the row (the gradient after it): through the blocks of slabs, then
// the slabs of its own block.
template <bool BACK, int V>
__device__ __forceinline__ void enter_slab(const ScanArgs &a, const Slab &slab, const Place<V> &at,
                                           Vec<V> &h) {
  if (a.slabs == 1) return;
  wait_for_previous();
  const int64_t c = at.b * a.D + at.d, row = a.B * a.D;
  const int blocks = gridDim.y, mine = blockIdx.y;
#pragma unroll 8
  for (int i = 0; i < (BACK ? blocks - 1 - mine : mine); ++i) {
    const float2 *f = a.fold + (BACK ? blocks - 1 - i : i) * row + c;
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = through(f[v].x, f[v].y, h[v]);
  }
  const float2 *f = a.fold + (blocks + slab.index) * row + c;
#pragma unroll
  for (int v = 0; v < V; ++v) h[v] = through(f[v].x, f[v].y, h[v]);
}

// A thread takes its V channels through the steps of its slab, with the loads
// of the eight steps ahead in flight: each step's gates are independent work, only
// one multiply-add a step is in sequence, and nothing is exchanged.  Measured:
// 4096 x 24 x 128 f32 42 us (4.8 TB/s), 1024 x 24 x 512 bf16 32 us (3.3 TB/s), 1 x
// 65536 x 512 f32 86 us (6.3 TB/s).  The last is bound by memory; the others wait for
// loads, with what 16 (f32) and 32 warps an SM can keep in flight: in bf16 57 % of the
// issue slots and of the special functions' rate, five of them a step and channel.
// Blocks that split the steps of a tile among warps and met in shared memory took 59,
// 55 and 278 us.
template <typename T, int V>
__global__ void __launch_bounds__(256, resident<T>()) scan_kernel(const __grid_constant__ ScanArgs a) {
  constexpr int S = kSteps;
  const Slab slab(a);
  const Place<V> at(a, slab.group * 32 + threadIdx.x);
  if (!__any_sync(0xffffffffu, at.live)) return;
  const char *rp = at_step<T>(a.rec, at.b, a.rb, slab.begin, a.rt, at.d);
  const char *ip = at_step<T>(a.inp, at.b, a.ib, slab.begin, a.it, at.d);
  const char *xp = at_step<T>(a.x, at.b, a.xb, slab.begin, a.xt, at.d);
  Raw<T, V> rr[S], ri[S], rx[S];
#pragma unroll
  for (int s = 0; s < S; ++s) {
    rr[s] = ri[s] = rx[s] = Raw<T, V>{};
    if (slab.begin + s < slab.end) {
      rr[s] = load_step<T, V>(rp);
      ri[s] = load_step<T, V>(ip);
      rx[s] = load_step<T, V>(xp);
    }
    advance(rp, a.rt, a.one);
    advance(ip, a.it, a.one);
    advance(xp, a.xt, a.one);
  }
  auto count = [&](int64_t t) {
    return (int)max((int64_t)0, min((int64_t)S, slab.end - t));
  };
  uint32_t marks = load_marks(a, at.b, slab.begin, count(slab.begin), at.one_row);
  Vec<V> h, rate;
#pragma unroll
  for (int v = 0; v < V; ++v) h[v] = a.h0 ? a.h0[at.b * a.D + at.d + v] : 0.0f;
  enter_slab<false>(a, slab, at, h);
  const bool big = load_rates<V>(a, at, rate);
  const char *hp = at_step<T>(a.h, at.b, a.hb, slab.begin, a.ht, at.d);
  for (int64_t t0 = slab.begin; t0 < slab.end; t0 += S) {
    const int n = count(t0), ahead = count(t0 + S);
    const uint32_t z = mark_bits(a, marks, at.one_row);
    marks = load_marks(a, at.b, t0 + S, ahead, at.one_row);
    if (a.carry && t0) {
#pragma unroll
      for (int v = 0; v < V; ++v)
        a.carry[(at.b * a.K + t0 / kChunk - 1) * a.D + at.d + v] = h[v];
    }
    // A lane beyond the last channel repeats the last one's steps and stores.
    auto run = [&](auto way, auto more) {
      constexpr Way WAY = decltype(way)::value;
      constexpr bool SLOW = WAY != kPlain, MORE = decltype(more)::value;
#pragma unroll
      for (int s = 0; s < S; ++s) {
        if (SLOW && s >= n) break;
        const Vec<V> r = values<T, V>(rr[s]), i = values<T, V>(ri[s]), x = values<T, V>(rx[s]);
        if (MORE || (SLOW && s < ahead)) {
          rr[s] = load_step<T, V>(rp);
          ri[s] = load_step<T, V>(ip);
          rx[s] = load_step<T, V>(xp);
          advance(rp, a.rt, a.one);
          advance(ip, a.it, a.one);
          advance(xp, a.xt, a.one);
        }
        const bool reset = SLOW && (z >> s & 1);
        const Decay<V> g = decay<WAY>(r, rate, reset);
        const Vec<V> b = mul(feed(i, g.e, g.a), x);
        if (reset) h = b;
        else h = fma(g.a, h, b);
        store_step<T, V>(hp, h);
        advance(hp, a.ht, a.one);
      }
    };
    const bool marked = n < S || (ahead != 0 && ahead != S) || __any_sync(0xffffffffu, z != 0);
    if (kMarksApart<T> ? big : big || marked)
      run(Is<kFar>{}, std::false_type{});
    else if (kMarksApart<T> && marked)
      run(Is<kMarksApart<T> ? kMarks : kFar>{}, std::false_type{});
    else if (ahead)
      run(Is<kPlain>{}, std::true_type{});
    else
      run(Is<kPlain>{}, std::false_type{});
  }
  if (a.h_last && slab.index == a.slabs - 1) {
#pragma unroll
    for (int v = 0; v < V; ++v) a.h_last[at.b * a.D + at.d + v] = h[v];
  }
}

// The gradient, stretch by stretch from a slab's end.  Backwards through a
// stretch, g_t = dh_t + gamma_{t+1}, gamma_t = a_t g_t, from the decays alone;
// then forwards, with the states running on from the kept one and every output
// made as its step comes by.  So every gate is computed once and only the decay,
// sigmoid(rec) and g of a stretch are held.  1024 x 24 x 512 bf16 50 us (3.6 TB/s), 8 x
// 8191 x 480 bf16 126 us (3.6 TB/s), at 56 and 52 % of the issue slots: with the sixteen
// warps an SM that its registers allow, of which 3.5 a scheduler run, it waits for
// loads and for its own chains of products in about equal parts.
template <typename T, int V>
__global__ void __launch_bounds__(256, kGradResident)
    scan_grad_kernel(const __grid_constant__ ScanArgs a) {
  constexpr int S = kSteps;
  const Slab slab(a);
  const Place<V> at(a, slab.group * 32 + threadIdx.x);
  if (!__any_sync(0xffffffffu, at.live)) return;
  Raw<T, V> rr[S], ri[S], rx[S], rg[S];
  Vec<V> h = all<V>(0.0f);
  auto count = [&](int64_t t) {
    return t < slab.begin ? 0 : (int)max((int64_t)0, min((int64_t)S, slab.end - t));
  };
  auto load_back = [&](int64_t t0, int n) {
    const char *r0 = at_step<T>(a.rec, at.b, a.rb, t0, a.rt, at.d);
    const char *g0 = at_step<T>(a.dh, at.b, a.gb, t0, a.gt, at.d);
#pragma unroll
    for (int s = 0; s < S; ++s) {
      if (s < n) {
        rr[s] = load_step<T, V>(r0);
        rg[s] = load_step<T, V>(g0);
        advance(r0, a.rt, a.one);
        advance(g0, a.gt, a.one);
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
        advance(i0, a.it, a.one);
        advance(x0, a.xt, a.one);
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
  int64_t t0 = slab.begin + (slab.end - slab.begin - 1) / S * S;
  int n = count(t0);
  load_back(t0, n);
  load_fwd(t0, n);
  uint32_t marks = load_marks(a, at.b, t0, n, at.one_row);
  Vec<V> rate, gam, dl = all<V>(0.0f), runs = dl;  // dlam's sum of this run, of the runs
#pragma unroll
  for (int v = 0; v < V; ++v)
    gam[v] = a.dh_last ? a.dh_last[at.b * a.D + at.d + v] : 0.0f;
  enter_slab<true>(a, slab, at, gam);
  const bool big = load_rates<V>(a, at, rate);

  while (n > 0) {
    const uint32_t z = mark_bits(a, marks, at.one_row);
    const bool slow = big || n < S || __any_sync(0xffffffffu, z != 0);
    const int64_t t_now = t0;
    const int n_now = n;
    t0 -= S;
    n = count(t0);
    marks = load_marks(a, at.b, t0, n, at.one_row);
    Vec<V> kept[S], SR[S], g[S];
    auto back = [&](auto tag) {
      constexpr Way WAY = decltype(tag)::value;
      constexpr bool SLOW = WAY != kPlain;
#pragma unroll
      for (int s = S - 1; s >= 0; --s) {
        const bool reset = SLOW && (z >> s & 1);
        const Decay<V> q = decay<WAY>(values<T, V>(rr[s]), rate, reset);
        kept[s] = hold<WAY>(q), SR[s] = q.sr;
        g[s] = add(gam, values<T, V>(rg[s]));
        if (!SLOW || s < n_now) {
          gam = mul(q.a, g[s]);
          if (reset) gam = all<V>(0.0f);
        }
      }
    };
    if (slow) back(Is<kFar>{});
    else back(Is<kPlain>{});
    load_back(t0, n);

    const char *dx0 = at_step<T>(a.dx, at.b, a.dxb, t_now, a.dxt, at.d);
    const char *dr0 = at_step<T>(a.drec, at.b, a.drb, t_now, a.drt, at.d);
    const char *di0 = at_step<T>(a.dinp, at.b, a.dib, t_now, a.dit, at.d);
    auto finish = [&](auto tag) {
      constexpr Way WAY = decltype(tag)::value;
      constexpr bool SLOW = WAY != kPlain;
#pragma unroll
      for (int s = 0; s < S; ++s) {
        if (SLOW && s >= n_now) break;
        const Vec<V> i = values<T, V>(ri[s]), x = values<T, V>(rx[s]);
        const bool reset = SLOW && (z >> s & 1);
        Vec<V> e, A;
        held<WAY>(kept[s], e, A);
        // 1 / m, kept finite where m is 0, so that nothing comes of it there
        const Vec<V> sq_m = square(e, A), si = gate(i);
        Vec<V> inv_m;
#pragma unroll
        for (int v = 0; v < V; ++v) inv_m[v] = rsq(fmaxf(sq_m[v], kSmallest));
        const Vec<V> ms = mul(mul(sq_m, inv_m), si);
        const Vec<V> dx = mul(g[s], ms), gx = mul(dx, x);
        const Vec<V> dinp = fma(mul(gx, si), -1.0f, gx);
        // q = g (h a - s_i x a^2 / m) = a (g h - g m s_i x a / m^2)
        Vec<V> q = mul(mul(gx, A), mul(inv_m, inv_m));
        q = mul(A, fma(q, -1.0f, mul(g[s], h)));
        if (reset) q = all<V>(0.0f);
        const Vec<V> sq = mul(SR[s], q);
        const Vec<V> drec = mul(mul(rate, add(SR[s], -1.0f)), sq);
        dl = add(dl, sq);
        const Vec<V> b = mul(ms, x);
        if (reset) h = b;
        else h = fma(A, h, b);
        store_step<T, V>(dx0, dx);
        store_step<T, V>(dr0, drec);
        store_step<T, V>(di0, dinp);
        advance(dx0, a.dxt, a.one);
        advance(dr0, a.drt, a.one);
        advance(di0, a.dit, a.one);
      }
    };
    if (slow) finish(Is<kFar>{});
    else finish(Is<kPlain>{});
    load_fwd(t0, n);
    if (t_now % kRun == 0) runs = add(runs, dl), dl = all<V>(0.0f);
  }
  runs = add(runs, dl);
  let_next_start();
  if (at.live && slab.index < a.slabs) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      a.part[((int64_t)slab.index * a.B + at.b) * a.D + at.d + v] = runs[v];
      if (a.dh0 && slab.index == 0) a.dh0[at.b * a.D + at.d + v] = gam[v];
    }
  }
}

// One step for many rows (a rollout's): a thread keeps its V channels' rates and
// takes every gridDim.y-th block of rows, four at a time.  4096 x 512 bf16 7.6 us
// (4.5 TB/s); with the rates made per row, as in scan_kernel, 13 us.
template <typename T, int V>
__global__ void __launch_bounds__(256) scan_step_kernel(const __grid_constant__ ScanArgs a,
                                                        int cols) {
  const int64_t unit = (int64_t)blockIdx.x * cols + threadIdx.x % cols, per = a.D / V;
  const int64_t d = unit * V;
  const int rows = 256 / cols;
  if (unit >= per || (int)threadIdx.x >= rows * cols) return;
  Vec<V> rate;
  bool big = false;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    rate[v] = a.c * softplus(a.lam[d + v]);
    big |= rate[v] > kSeriesMax;
  }
  constexpr int R = 4;
  const int64_t pace = (int64_t)gridDim.y * rows;
  for (int64_t b0 = (int64_t)blockIdx.y * rows + threadIdx.x / cols; b0 < a.B; b0 += R * pace) {
    Raw<T, V> rr[R], ri[R], rx[R];
    Vec<V> h[R];
    uint8_t z[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int64_t b = b0 + i * pace;
      if (b < a.B) {
        rr[i] = load_step<T, V>(at_step<T>(a.rec, b, a.rb, 0, 0, d));
        ri[i] = load_step<T, V>(at_step<T>(a.inp, b, a.ib, 0, 0, d));
        rx[i] = load_step<T, V>(at_step<T>(a.x, b, a.xb, 0, 0, d));
        z[i] = a.resets ? a.resets[b * a.zb] : 0;
#pragma unroll
        for (int v = 0; v < V; ++v) h[i][v] = a.h0 ? a.h0[b * a.D + d + v] : 0.0f;
      }
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int64_t b = b0 + i * pace;
      if (b >= a.B) break;
      const Vec<V> r = values<T, V>(rr[i]);
      const Decay<V> g = big || z[i] ? decay<kFar>(r, rate, z[i] != 0) : decay<kPlain>(r, rate, false);
      const Vec<V> f =
          mul(feed(values<T, V>(ri[i]), g.e, g.a), values<T, V>(rx[i]));
      const Vec<V> y = z[i] ? f : fma(g.a, h[i], f);
      store_step<T, V>(at_step<T>(a.h, b, a.hb, 0, 0, d), y);
      if (a.h_last) {
#pragma unroll
        for (int v = 0; v < V; ++v) a.h_last[b * a.D + d + v] = y[v];
      }
    }
  }
}

// dlam from the column sums
struct DlamOut {
  const float *lam;
  float *dlam;
  float c;
  __device__ __forceinline__ void operator()(int64_t d, float sum) const {
    dlam[d] = -c * sum / (1.0f + expf(-lam[d]));
  }
};

// How a call is laid out.  A thread takes a row's channels through all steps
// where rows and channels fill the SMs (kFull groups of lanes) or the row is
// short; else the row is cut into slabs, whose effect on the state is folded in
// a first pass: as many blocks of eight slabs as fill one to three waves of the
// resident blocks best.  Measured (device us): 1 x 65536 x 512 f32 fold + scan in 1
// / 1.5 / 3 waves 152 / 171 / 169; 200 x 400 x 480 bf16 with gradient (1,500 groups) in
// one piece 315, in slabs 369; 16 x 100 x 200 f16 (50 groups) 65 and 38.
constexpr int kSms = 148;
constexpr int64_t kFull = kSms * 8;
struct ScanPlan {
  int V, slabs, slab_blocks;
  int64_t units, slab_steps, blocks;
};

ScanPlan plan_scan(int64_t B, int64_t T, int64_t D, int V, int resident) {
  ScanPlan p{};
  p.V = V;
  p.units = B * (D / V);
  const int64_t groups = std::max<int64_t>(1, (p.units + 31) / 32);
  p.slabs = p.slab_blocks = 1;
  p.slab_steps = T;
  p.blocks = (groups + kWarps - 1) / kWarps;
  if (groups < kFull && T >= 4 * kMinSlab) {
    int64_t best = 1;
    double filled = 0.0;
    for (int waves = 1; waves <= 3; ++waves) {
      const int64_t room = (int64_t)waves * kSms * resident;
      const double f = (double)(room / groups * groups) / room;
      if (f > filled + 0.05) filled = f, best = room / groups;
    }
    const int64_t want = std::min<int64_t>(std::max<int64_t>(1, best) * kWarps, T / kMinSlab);
    p.slab_steps = ((T + want - 1) / want + kSteps - 1) / kSteps * kSteps;
    p.slabs = (int)((T + p.slab_steps - 1) / p.slab_steps);
    p.slab_blocks = (p.slabs + kWarps - 1) / kWarps;
    p.blocks = groups;
  }
  return p;
}
int fwd_resident(int es) { return es == 2 ? resident<__half>() : resident<float>(); }

// Pairs of the first pass: per block of slabs and per slab (whole blocks).
int64_t fold_pairs(const ScanPlan &p, int64_t B, int64_t D) {
  return p.slabs > 1 ? (int64_t)p.slab_blocks * (1 + kWarps) * B * D : 0;
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
  with_dtype(dtype, [&](auto t) {
    if (p.V == 2) f(t, std::integral_constant<int, 2>{});
    else f(t, std::integral_constant<int, 1>{});
  });
}

void use_plan(ScanArgs &a, const ScanPlan &p, void *workspace) {
  a.units = p.units;
  a.slabs = p.slabs;
  a.slab_steps = p.slab_steps;
  a.fold = static_cast<float2 *>(workspace);
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
  a.one = 1;
  a.zb = strides ? strides[6] : T;
  a.zt = strides ? strides[7] : 1;
}

}  // namespace
}  // namespace zrl

using namespace zrl;

extern "C" int64_t zrl_gated_scan_carry(int64_t B, int64_t T, int64_t D) {
  return B > 0 && D > 0 ? B * chunk_starts(T) * D : 0;
}

// Enough for every element type and for one or two channels a lane.
extern "C" int64_t zrl_gated_scan_workspace(int64_t B, int64_t T, int64_t D) {
  if (B <= 0 || D <= 0) return 0;
  int64_t pairs = 0;
  for (int V = 1; V <= 2; ++V)
    for (int es = 2; es <= 4; es += 2)
      pairs = std::max(pairs, fold_pairs(plan_scan(B, T, D, V, fwd_resident(es)), B, D));
  return pairs * (int64_t)sizeof(float2);
}

extern "C" zrl_status zrl_gated_scan(const void *x, const void *rec, const void *inp,
                                     const float *lam, const float *h0, const uint8_t *resets,
                                     int64_t B, int64_t T, int64_t D, int32_t dtype, float c,
                                     const int64_t *strides, void *h, float *h_last,
                                     float *carry, void *workspace, int64_t workspace_bytes,
                                     void *stream) {
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
  const ScanPlan p = plan_scan(B, T, D, pairs ? 2 : 1, fwd_resident(es));
  if (p.blocks > 0x7fffffff) return seq_fail(ZRL_NOT_SUPPORTED, "gated_scan: B * D too large");
  if (workspace_bytes < zrl_gated_scan_workspace(B, T, D) || !aligned(workspace, 16) ||
      (!workspace && p.slabs > 1))
    return seq_fail(ZRL_INVALID_ARG, "gated_scan: workspace too small or not aligned");
  use_plan(a, p, workspace);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  with_plan(dtype, p, [&](auto t, auto v) {
    using E = decltype(t);
    constexpr int V = decltype(v)::value;
    const dim3 grid((unsigned)p.blocks, (unsigned)p.slab_blocks), threads(32, kWarps);
    if (T == 1) {
      const int64_t per = D / V;
      const int cols = (int)std::min<int64_t>(256, per);
      const int64_t across = (per + cols - 1) / cols, rows = 256 / cols;
      const int64_t down = std::min<int64_t>((B + rows - 1) / rows,
                                             std::max<int64_t>(1, kSms * 4 / across));
      scan_step_kernel<E, V>
          <<<dim3((unsigned)across, (unsigned)down), 256, 0, st>>>(a, cols);
      return;
    }
    if (p.slabs > 1) scan_fold_kernel<E, V, false><<<grid, threads, 0, st>>>(a);
    if (p.slabs > 1) launch_next(scan_kernel<E, V>, grid, threads, 1, st, a);
    else scan_kernel<E, V><<<grid, threads, 0, st>>>(a);
  });
  return seq_launched("gated_scan");
}

extern "C" int64_t zrl_gated_scan_grad_workspace(int64_t B, int64_t T, int64_t D) {
  if (B <= 0 || D <= 0) return 0;
  // dlam's sums, one per row, channel and slab, on top of the first pass's pairs
  int64_t bytes = 0;
  for (int V = 1; V <= 2; ++V) {
    const ScanPlan p = plan_scan(B, T, D, V, kGradResident);
    bytes = std::max(bytes, fold_pairs(p, B, D) * (int64_t)sizeof(float2) +
                                B * D * p.slabs * (int64_t)sizeof(float));
  }
  return bytes;
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
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  ScanTensor ts[] = {{x, 0, &a.xb, &a.xt},     {rec, 2, &a.rb, &a.rt},    {inp, 4, &a.ib, &a.it},
                     {dh, 8, &a.gb, &a.gt},    {dx, 10, &a.dxb, &a.dxt},  {drec, 12, &a.drb, &a.drt},
                     {dinp, 14, &a.dib, &a.dit}};
  bool pairs = false;
  if (!place_tensors(ts, 7, strides, T, D, es, &pairs))
    return seq_fail(ZRL_NOT_SUPPORTED, "gated_scan_grad: a time stride of 2 GiB or more");
  const int V = pairs && es == 2 ? 2 : 1;
  const ScanPlan p = plan_scan(B, T, D, V, kGradResident);
  if (p.blocks > 0x7fffffff)
    return seq_fail(ZRL_NOT_SUPPORTED, "gated_scan_grad: B * D too large");
  use_plan(a, p, workspace);
  a.part = reinterpret_cast<float *>(static_cast<char *>(workspace) +
                                     fold_pairs(p, B, D) * sizeof(float2));
  if (B)
    with_plan(dtype, p, [&](auto t, auto v) {
      using E = decltype(t);
      constexpr int V = decltype(v)::value;
      if constexpr (V * sizeof(E) <= 4) {
        const dim3 grid((unsigned)p.blocks, (unsigned)p.slab_blocks), threads(32, kWarps);
        if (p.slabs > 1) scan_fold_kernel<E, V, true><<<grid, threads, 0, st>>>(a);
        if (p.slabs > 1) launch_next(scan_grad_kernel<E, V>, grid, threads, 1, st, a);
        else scan_grad_kernel<E, V><<<grid, threads, 0, st>>>(a);
      }
    });
  launch_column_sum(a.part, B * p.slabs, D, DlamOut{lam, dlam, c}, st);
  return seq_launched("gated_scan_grad");
}
