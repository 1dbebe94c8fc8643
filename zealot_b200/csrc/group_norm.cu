// group_norm.cu -- group norm over channels-last rows with an activation, and
// its gradient.
//
// x [N, L, C], groups of w = C / G neighbouring channels; per (n, g), over
// L x w elements: mu, var, xh = (x - mu) / sqrt(var + eps); then
// y = act(gamma xh + beta).  Gradient, with dz = dy act'(z):
//   dbeta = sum dz, dgamma = sum dz xh,
//   dx = rstd (gamma dz - mean(gamma dz) - xh mean(gamma dz xh)).
// The kernels are in group_norm_rows.cuh (L = 1) and group_norm_samples.cuh;
// here a call is checked and laid out.
#include <math.h>

#include <algorithm>
#include <initializer_list>
#include <type_traits>

#include "column_sum.cuh"
#include "group_norm_rows.cuh"
#include "group_norm_samples.cuh"

namespace zrl {
namespace {

constexpr int64_t kBatchBytes = 110 << 20;  // of two passes that meet in L2
constexpr int64_t kBlockBytes = 64 << 10;   // shared memory of the block form

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

// A call, and whether its tensors can be taken in vectors.
struct NormShape {
  int64_t N, L, C;
  int32_t G;
  int es;
  bool grad;
  int64_t align;       // bytes that pointers and strides are multiples of: 16, 8, 4 or es
};

// How a call is laid out.
//  lanes:   L = 1: E vectors of 16 bytes to one element a lane, p lanes a
//           group.  About eight channels a lane where the group has them, so
//           that the shuffles of the sums are shared by as many: at w = 25 in
//           fp32, four by eight lanes took 71 us, one by 32 lanes 92 us
//           (98304 x 250 forward, vector by vector; 53 us now).
//  block:   a sample's columns fit a block's shared memory.
//  passes:  the rest.
// A row whose groups are too wide for the lanes of a warp (above 256 channels in fp32
// and 512 in 16 bits on aligned rows, 128 at odd widths) goes to the block form with one
// position, which is made for many: 24576 x 1024 bf16 in one group 316 us forward and
// 378 us with its sums back, where 512 channels take 16 and 49; so are samples of a few
// positions (16384 x 4 x 256 bf16 259 and 309 us).  And the block form leaves its sums per
// sample: a gradient's workspace of 2 C floats for each of N.
struct NormPlan {
  enum { kLanes, kBlock, kPasses } form;
  int vec, E, p, gb, rb, blocks, across;  // lanes
  int cols, parts, stretches, depth;      // samples (depth: blocks over channels)
  int64_t stretch, batch, bytes;          // batch: samples of a launch; shared memory
};

bool plan_lanes(const NormShape &s, NormPlan *p) {
  const int64_t w = s.C / s.G;
  int vec = 16 / s.es;
  while (w % vec || s.align % (vec * s.es)) vec /= 2;
  const int64_t nv = w / vec, most = vec >= 4 ? 2 : 4;
  int64_t E = 1;
  while (E < most && E * vec < 8 && 8 * E < nv) ++E;
  while (E < most && (nv + E - 1) / E > 32) ++E;
  if ((nv + E - 1) / E > 32) return false;
  p->form = NormPlan::kLanes;
  p->vec = vec;
  p->E = (int)E;
  p->p = 1;
  while (p->p < (nv + E - 1) / E) p->p *= 2;
  p->gb = (int)std::min<int64_t>(s.G, kThreads / p->p);
  p->rb = kThreads / (p->gb * p->p);
  p->across = (s.G + p->gb - 1) / p->gb;
  // blocks that stay resident: each loads its gammas, and leaves the gradient's
  // sums, once
  p->blocks = (int)std::max<int64_t>(
      1, std::min<int64_t>((s.N + p->rb - 1) / p->rb, kSms * kLaneBlocks / p->across));
  return p->across <= 65535;
}

// Channels of a block: the whole row where it fits, else as many groups as make
// whole vectors, else a part of one group.
bool plan_columns(const NormShape &s, int vec, int64_t most_channels, NormPlan *p) {
  const int64_t w = s.C / s.G;
  if (s.C % vec || s.align % (vec * s.es)) return false;
  p->vec = vec;
  p->parts = 1;
  if (s.C <= most_channels) {
    p->cols = (int)s.C;
    p->depth = 1;
    return true;
  }
  int64_t unit = 1;
  while (unit * w % vec) unit *= 2;  // vec is a power of two
  const int64_t per = most_channels / w / unit * unit;
  if (per) {
    p->cols = (int)(per * w);
    p->depth = (int)((s.G + per - 1) / per);
    return true;
  }
  if (w % vec || most_channels < (int64_t)kThreads * vec) return false;
  p->cols = kThreads * vec;
  p->parts = (int)((w + p->cols - 1) / p->cols);
  p->depth = s.G * p->parts;
  return true;
}

NormPlan plan_samples(const NormShape &s) {
  NormPlan p{};
  const int64_t tensors = s.grad ? 2 : 1;
  for (int vec = kMaxChannels; vec >= 1; vec /= 2) {
    if (!plan_columns(s, vec, (int64_t)kThreads * vec, &p)) continue;
    // the block form, with columns of 128 bytes or the group if it is wider
    NormPlan b = p;
    const int64_t w = s.C / s.G;
    if (plan_columns(s, vec, std::min<int64_t>((int64_t)kThreads * vec, std::max<int64_t>(128 / s.es, w * vec)), &b) &&
        b.parts == 1 && b.depth <= 65535) {
      const int64_t rows = kThreads / (b.cols / vec);
      b.bytes = (s.L + rows - 1) / rows * kThreads * vec * s.es * tensors;
      if (b.bytes <= kBlockBytes && (s.N * b.depth >= kSms || b.bytes <= kBlockBytes / 4)) {
        b.form = NormPlan::kBlock;
        b.stretches = 1;
        b.stretch = s.L;
        b.batch = std::min<int64_t>(s.N, 65535);
        return b;
      }
    }
    p.form = NormPlan::kPasses;
    const int64_t sample = std::max<int64_t>(1, s.L * s.C * s.es * tensors);
    p.batch = std::max<int64_t>(1, std::min<int64_t>({s.N, (int64_t)65535, kBatchBytes / sample}));
    // one wave of the resident blocks, and some positions for each thread
    const int64_t rows = kThreads / (p.cols / vec);
    const int64_t want =
        std::max<int64_t>(1, kSms * sample_blocks(s.grad) / (p.batch * p.depth));
    const int64_t fit = std::max<int64_t>(1, s.L / (rows * 4));
    p.stretches = (int)std::max<int64_t>(1, std::min<int64_t>({want, fit, (int64_t)512}));
    p.stretch = ((s.L + p.stretches - 1) / p.stretches + rows * 4 - 1) / (rows * 4) * (rows * 4);
    p.stretches = (int)((s.L + p.stretch - 1) / p.stretch);
    return p;
  }
  return p;  // not reached: one channel a vector always fits
}

NormPlan plan_norm(const NormShape &s) {
  NormPlan p{};
  if (s.L == 1 && plan_lanes(s, &p)) return p;
  return plan_samples(s);
}

int64_t workspace_floats(const NormPlan &p, const NormShape &s) {
  if (p.form == NormPlan::kLanes)
    return s.grad ? (int64_t)p.blocks * 2 * s.C : 0;
  if (s.grad)
    return s.N * p.stretches * 2 *
           (s.C + (p.form == NormPlan::kPasses ? (int64_t)s.G * p.parts : 0));
  return p.form == NormPlan::kPasses ? s.N * s.G * p.stretches * p.parts * 2 : 0;
}

template <typename F>
void with_vec(int32_t dtype, int vec, F &&f) {
  using std::integral_constant;
  with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    if (vec == 1) f(t, integral_constant<int, 1>{});
    else if (vec == 2) f(t, integral_constant<int, 2>{});
    else if (vec == 4) f(t, integral_constant<int, 4>{});
    else if constexpr (sizeof(T) == 2) f(t, integral_constant<int, 8>{});
  });
}
template <int VEC, typename F>
void with_e(int E, F &&f) {
  if (E == 1) f(std::integral_constant<int, 1>{});
  else if (E == 2) f(std::integral_constant<int, 2>{});
  else if constexpr (VEC <= 2) {
    if (E == 3) f(std::integral_constant<int, 3>{});
    else f(std::integral_constant<int, 4>{});
  }
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
  a.means = reinterpret_cast<float2 *>(a.part + a.N * p.stretches * 2 * a.C);
  a.wide = aligned(a.gamma, 16) && aligned(a.beta, 16);
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

// The launch error, if any, is left for cudaGetLastError.
void launch_norm(void (*kernel)(NormArgs), dim3 grid, const NormPlan &p, cudaStream_t st,
                 const NormArgs &a) {
  // up to 48 KB, with up to 24 KB of static memory beside it, need no leave.  The limit
  // is the whole context's, so it is always the most that any call takes: a call from
  // another thread never lowers it between here and the launch.
  if (p.bytes > (24 << 10) &&
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           (int)kBlockBytes) != cudaSuccess)
    return;
  kernel<<<grid, kThreads, (size_t)p.bytes, st>>>(a);
}

// What the call's pointers and strides allow.
NormShape shape_of(const NormArgs &a, int es, bool grad,
                   std::initializer_list<const void *> ptrs) {
  NormShape s{a.N, a.L, a.C, a.G, es, grad, 16};
  for (const void *p : ptrs)
    while (!aligned(p, s.align)) s.align /= 2;
  for (int64_t t : {a.sxn, a.syn, grad ? a.sdn : a.syn}) {
    if (a.N > 1)
      while (t * es % s.align) s.align /= 2;
  }
  for (int64_t t : {a.sxl, a.syl, grad ? a.sdl : a.syl})
    if (a.L > 1)
      while (t * es % s.align) s.align /= 2;
  return s;
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
  a.means += n0 * a.G * a.stretches * a.parts;
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
  for (int es : {2, 4})
    for (int64_t align = 16; align >= es; align /= 2) {
      const NormShape s{N, L, C, groups, es, grad != 0, align};
      most = std::max(most, workspace_floats(plan_norm(s), s));
    }
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
  const NormShape shape = shape_of(a, es, false, {x, y});
  const NormPlan p = plan_norm(shape);
  const int64_t need = workspace_floats(p, shape) * (int64_t)sizeof(float);
  if (workspace_bytes < need || !aligned(workspace, 16) || (!workspace && need))
    return seq_fail(ZRL_INVALID_ARG, "group_norm: workspace too small or not aligned");
  use_plan(a, p, workspace);
  with_vec(dtype, p.vec, [&](auto t, auto v) {
    using T = decltype(t);
    constexpr int VEC = decltype(v)::value;
    if (p.form == NormPlan::kLanes) {
      with_e<VEC>(p.E, [&](auto e) {
        norm_rows_kernel<T, VEC, decltype(e)::value>
            <<<dim3((unsigned)p.blocks, (unsigned)p.across), kThreads, 0, st>>>(a);
      });
      return;
    }
    if constexpr (VEC <= kMaxChannels) {
      for (int64_t n0 = 0; n0 < N; n0 += p.batch) {
        const NormArgs b = samples_from(a, n0, es);
        const dim3 grid((unsigned)p.stretches, (unsigned)std::min(p.batch, N - n0),
                        (unsigned)p.depth);
        if (p.form == NormPlan::kBlock) {
          launch_norm(norm_block_kernel<T, VEC>, grid, p, st, b);
          continue;
        }
        norm_stats_kernel<T, VEC><<<grid, kThreads, 0, st>>>(b);
        launch_next(norm_apply_kernel<T, VEC>, grid, dim3(kThreads), 1, st, b);
      }
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
  const NormShape shape = shape_of(a, es, true, {x, dy, dx});
  const NormPlan p = plan_norm(shape);
  if (!workspace || workspace_bytes < workspace_floats(p, shape) * (int64_t)sizeof(float))
    return seq_fail(ZRL_INVALID_ARG, "group_norm_grad: workspace too small");
  use_plan(a, p, workspace);
  int64_t sums = N * p.stretches;  // rows of channel sums
  with_vec(dtype, p.vec, [&](auto t, auto v) {
    using T = decltype(t);
    constexpr int VEC = decltype(v)::value;
    if (p.form == NormPlan::kLanes) {
      with_e<VEC>(p.E, [&](auto e) {
        norm_rows_grad_kernel<T, VEC, decltype(e)::value>
            <<<dim3((unsigned)p.blocks, (unsigned)p.across), kThreads, 0, st>>>(a);
      });
      sums = p.blocks;
      return;
    }
    if constexpr (VEC <= kMaxChannels) {
      for (int64_t n0 = 0; n0 < N; n0 += p.batch) {
        const NormArgs b = samples_from(a, n0, es);
        const dim3 grid((unsigned)p.stretches, (unsigned)std::min(p.batch, N - n0),
                        (unsigned)p.depth);
        if (p.form == NormPlan::kBlock) {
          launch_norm(norm_block_grad_kernel<T, VEC>, grid, p, st, b);
          continue;
        }
        norm_grad_sums_kernel<T, VEC><<<grid, kThreads, 0, st>>>(b);
        launch_next(norm_grad_apply_kernel<T, VEC>, grid, dim3(kThreads), 1, st, b);
      }
    }
  });
  launch_column_sum(a.part, sums, 2 * C, ParamOut{dgamma, dbeta, C}, st);
  return seq_launched("group_norm_grad");
}
