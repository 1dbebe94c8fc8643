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

namespace zrl {
namespace {

// The state at every kChunk-th step is what the gradient starts from when it
// recomputes h.
constexpr int kChunk = 64;

struct ScanArgs {
  const void *x, *rec, *inp, *dh;
  const float *lam, *h0, *dh_last;
  const uint8_t *resets;
  void *h, *dx, *drec, *dinp;
  float *h_last, *carry, *dh0, *part;
  int64_t B, T, D, K;  // K: chunk starts after the first
  int64_t xb, xt, rb, rt, ib, it, zb, zt, hb, ht, gb, gt, dxb, dxt, drb, drt, dib, dit;
  float c;
};

__device__ __forceinline__ float softplus(float v) {
  return fmaxf(v, 0.0f) + log1pf(expf(-fabsf(v)));
}

struct Gate {
  float a, m, si, sr;
};

__device__ __forceinline__ Gate gate(float rec, float inp, float rate, bool reset) {
  Gate g;
  g.sr = 1.0f / (1.0f + expf(-rec));
  g.si = 1.0f / (1.0f + expf(-inp));
  const float la = -rate * g.sr;
  g.a = reset ? 0.0f : expf(la);
  g.m = reset ? 1.0f : sqrtf(-expm1f(2.0f * la));
  return g;
}

// a h + b, with nothing of h where an episode begins
__device__ __forceinline__ float step_state(float a, float h, float b, bool reset) {
  return reset ? b : fmaf(a, h, b);
}

// One thread per (b, d).
template <typename T>
__global__ void __launch_bounds__(128) scan_kernel(const ScanArgs a) {
  for (int64_t e = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; e < a.B * a.D;
       e += (int64_t)gridDim.x * blockDim.x) {
    const int64_t b = e / a.D, d = e - b * a.D;
    const T *x = static_cast<const T *>(a.x) + b * a.xb + d;
    const T *rec = static_cast<const T *>(a.rec) + b * a.rb + d;
    const T *inp = static_cast<const T *>(a.inp) + b * a.ib + d;
    T *out = static_cast<T *>(a.h) + b * a.hb + d;
    const float rate = a.c * softplus(a.lam[d]);
    float h = a.h0 ? a.h0[e] : 0.0f;
    for (int64_t t = 0; t < a.T; ++t) {
      if (a.carry && t && t % kChunk == 0) a.carry[(b * a.K + t / kChunk - 1) * a.D + d] = h;
      const bool reset = a.resets && a.resets[b * a.zb + t * a.zt];
      const Gate g = gate(to_f32(rec[t * a.rt]), to_f32(inp[t * a.it]), rate, reset);
      h = step_state(g.a, h, g.m * g.si * to_f32(x[t * a.xt]), reset);
      out[t * a.ht] = from_f32<T>(h);
    }
    if (a.h_last) a.h_last[e] = h;
  }
}

// One thread per (b, d): chunk by chunk from the end, the states of a chunk
// recomputed from its first.
template <typename T>
__global__ void __launch_bounds__(128) scan_grad_kernel(const ScanArgs a) {
  for (int64_t e = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; e < a.B * a.D;
       e += (int64_t)gridDim.x * blockDim.x) {
    const int64_t b = e / a.D, d = e - b * a.D;
    const T *x = static_cast<const T *>(a.x) + b * a.xb + d;
    const T *rec = static_cast<const T *>(a.rec) + b * a.rb + d;
    const T *inp = static_cast<const T *>(a.inp) + b * a.ib + d;
    const T *dh = static_cast<const T *>(a.dh) + b * a.gb + d;
    T *dx = static_cast<T *>(a.dx) + b * a.dxb + d;
    T *drec = static_cast<T *>(a.drec) + b * a.drb + d;
    T *dinp = static_cast<T *>(a.dinp) + b * a.dib + d;
    const float rate = a.c * softplus(a.lam[d]);
    float g = a.dh_last ? a.dh_last[e] : 0.0f, dl = 0.0f;
    float before[kChunk];
    for (int64_t k = a.K; k >= 0 && a.T; --k) {
      const int64_t t0 = k * kChunk, t1 = min(a.T, t0 + kChunk);
      float h = k ? a.carry[(b * a.K + k - 1) * a.D + d] : (a.h0 ? a.h0[e] : 0.0f);
      for (int64_t t = t0; t < t1; ++t) {
        before[t - t0] = h;
        const bool reset = a.resets && a.resets[b * a.zb + t * a.zt];
        const Gate q = gate(to_f32(rec[t * a.rt]), to_f32(inp[t * a.it]), rate, reset);
        h = step_state(q.a, h, q.m * q.si * to_f32(x[t * a.xt]), reset);
      }
      for (int64_t t = t1 - 1; t >= t0; --t) {
        const bool reset = a.resets && a.resets[b * a.zb + t * a.zt];
        const Gate q = gate(to_f32(rec[t * a.rt]), to_f32(inp[t * a.it]), rate, reset);
        const float xv = to_f32(x[t * a.xt]);
        g += to_f32(dh[t * a.gt]);
        const float inner = q.m > 0.0f ? q.si * xv * q.a * q.a / q.m : 0.0f;
        const float la = reset ? 0.0f : g * (before[t - t0] * q.a - inner);
        dx[t * a.dxt] = from_f32<T>(g * q.m * q.si);
        drec[t * a.drt] = from_f32<T>(-rate * q.sr * (1.0f - q.sr) * la);
        dinp[t * a.dit] = from_f32<T>(g * q.m * xv * q.si * (1.0f - q.si));
        dl += q.sr * la;
        g = reset ? 0.0f : q.a * g;
      }
    }
    if (a.dh0) a.dh0[e] = g;
    a.part[e] = dl;
  }
}

// dlam = -c sigmoid(lam) * (sum over rows), rows folded in order
__global__ void scan_dlam_kernel(const float *part, const float *lam, int64_t B, int64_t D,
                                 float c, float *dlam) {
  const int64_t d = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (d >= D) return;
  double s = 0.0;
  for (int64_t b = 0; b < B; ++b) s += part[b * D + d];
  dlam[d] = (float)(-c * s) / (1.0f + expf(-lam[d]));
}

int64_t chunk_starts(int64_t T) { return T > 0 ? (T - 1) / kChunk : 0; }

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
  const int64_t blocks = std::min<int64_t>((B * D + 127) / 128, (int64_t)1 << 30);
  with_dtype(dtype, [&](auto t) {
    scan_kernel<decltype(t)>
        <<<(unsigned)blocks, 128, 0, static_cast<cudaStream_t>(stream)>>>(a);
  });
  return seq_launched("gated_scan");
}

extern "C" int64_t zrl_gated_scan_grad_workspace(int64_t B, int64_t T, int64_t D) {
  (void)T;
  return B > 0 && D > 0 ? B * D * (int64_t)sizeof(float) : 0;
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
  if (B) {
    const int64_t blocks = std::min<int64_t>((B * D + 127) / 128, (int64_t)1 << 30);
    with_dtype(dtype, [&](auto t) {
      scan_grad_kernel<decltype(t)><<<(unsigned)blocks, 128, 0, st>>>(a);
    });
  }
  scan_dlam_kernel<<<(unsigned)((D + 127) / 128), 128, 0, st>>>(a.part, lam, B, D, c, dlam);
  return seq_launched("gated_scan_grad");
}
