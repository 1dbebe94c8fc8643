// seq_common.cuh -- what the sequence operators (dropout.cu, group_norm.cu,
// gated_scan.cu) share: element types, vector loads and stores that convert
// to and from fp32, and the refusal of bad arguments.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "zrl_internal.h"

namespace zrl {

// Records the calling thread's message (zrl_last_error(NULL)) and returns s.
zrl_status seq_fail(zrl_status s, const char *fmt, ...)
    __attribute__((format(printf, 2, 3)));
// ZRL_OK, or the launch error of the calling thread's last kernel launch.
zrl_status seq_launched(const char *what);

inline int dtype_size(int32_t dt) { return dt == ZRL_F32 ? 4 : 2; }
inline bool dtype_ok(int32_t dt) { return dt == ZRL_F32 || dt == ZRL_BF16 || dt == ZRL_F16; }
inline bool aligned(const void *p, int64_t bytes) {
  return (reinterpret_cast<uintptr_t>(p) % (uintptr_t)bytes) == 0;
}

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
// Outputs are rounded once, to nearest even.
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
template <> __device__ __forceinline__ __half from_f32<__half>(float v) {
  return __float2half_rn(v);
}

// V consecutive elements as one access (V * sizeof(T) in 2, 4, 8, 16 bytes,
// aligned to that).
template <int BYTES> struct RawT;
template <> struct RawT<2> { using type = uint16_t; };
template <> struct RawT<4> { using type = uint32_t; };
template <> struct RawT<8> { using type = uint2; };
template <> struct RawT<16> { using type = uint4; };
template <typename T, int V> using Raw = typename RawT<V * (int)sizeof(T)>::type;

template <typename T, int V>
__device__ __forceinline__ void unpack(const Raw<T, V> &raw, float *out) {
  if constexpr (sizeof(T) == 2 && V >= 2) {
    const uint32_t *w = reinterpret_cast<const uint32_t *>(&raw);
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      if constexpr (sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value) {
        out[2 * i] = __uint_as_float(w[i] << 16);
        out[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      } else {
        const __half2 h = *reinterpret_cast<const __half2 *>(&w[i]);
        const float2 f = __half22float2(h);
        out[2 * i] = f.x;
        out[2 * i + 1] = f.y;
      }
    }
  } else {
    const T *e = reinterpret_cast<const T *>(&raw);
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = to_f32(e[i]);
  }
}

template <typename T, int V>
__device__ __forceinline__ Raw<T, V> pack(const float *in) {
  Raw<T, V> raw;
  if constexpr (sizeof(T) == 2 && V >= 2) {
    uint32_t *w = reinterpret_cast<uint32_t *>(&raw);
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        const __nv_bfloat162 b = __floats2bfloat162_rn(in[2 * i], in[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t *>(&b);
      } else {
        const __half2 h = __floats2half2_rn(in[2 * i], in[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t *>(&h);
      }
    }
  } else {
    T *e = reinterpret_cast<T *>(&raw);
#pragma unroll
    for (int i = 0; i < V; ++i) e[i] = from_f32<T>(in[i]);
  }
  return raw;
}

constexpr float kLog2e = 1.44269504f;

// The special functions' approximate forms: 2^v, 1 / v, 1 / sqrt(v) and sqrt(v)
// within a few units in the last place (PTX's stated bounds), subnormals as zero.
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
__device__ __forceinline__ float root(float v) {
  float r;
  asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
// V channels' values.  Pairs go through the packed fp32 instructions, which
// halve the issue slots of everything but the special functions.
template <int V>
struct Vec {
  float v[V];
  __device__ __forceinline__ float &operator[](int i) { return v[i]; }
  __device__ __forceinline__ const float &operator[](int i) const { return v[i]; }
};
template <int V>
__device__ __forceinline__ Vec<V> all(float c) {
  Vec<V> r;
#pragma unroll
  for (int i = 0; i < V; ++i) r[i] = c;
  return r;
}
template <int V>
__device__ __forceinline__ Vec<V> fma(const Vec<V> &a, const Vec<V> &b, const Vec<V> &c) {
  Vec<V> r;
#pragma unroll
  for (int i = 0; i + 1 < V; i += 2) {
    const float2 f = __ffma2_rn(make_float2(a[i], a[i + 1]), make_float2(b[i], b[i + 1]),
                                make_float2(c[i], c[i + 1]));
    r[i] = f.x, r[i + 1] = f.y;
  }
  if constexpr (V % 2) {
    constexpr int i = V - 1;
    r[i] = fmaf(a[i], b[i], c[i]);
  }
  return r;
}
template <int V>
__device__ __forceinline__ Vec<V> mul(const Vec<V> &a, const Vec<V> &b) {
  Vec<V> r;
#pragma unroll
  for (int i = 0; i + 1 < V; i += 2) {
    const float2 f = __fmul2_rn(make_float2(a[i], a[i + 1]), make_float2(b[i], b[i + 1]));
    r[i] = f.x, r[i + 1] = f.y;
  }
  if constexpr (V % 2) {
    constexpr int i = V - 1;
    r[i] = a[i] * b[i];
  }
  return r;
}
template <int V>
__device__ __forceinline__ Vec<V> add(const Vec<V> &a, const Vec<V> &b) {
  Vec<V> r;
#pragma unroll
  for (int i = 0; i + 1 < V; i += 2) {
    const float2 f = __fadd2_rn(make_float2(a[i], a[i + 1]), make_float2(b[i], b[i + 1]));
    r[i] = f.x, r[i + 1] = f.y;
  }
  if constexpr (V % 2) {
    constexpr int i = V - 1;
    r[i] = a[i] + b[i];
  }
  return r;
}
template <int V>
__device__ __forceinline__ Vec<V> fma(const Vec<V> &a, float b, const Vec<V> &c) {
  return fma(a, all<V>(b), c);
}
template <int V>
__device__ __forceinline__ Vec<V> fma(const Vec<V> &a, const Vec<V> &b, float c) {
  return fma(a, b, all<V>(c));
}
template <int V>
__device__ __forceinline__ Vec<V> fma(const Vec<V> &a, float b, float c) {
  return fma(a, all<V>(b), all<V>(c));
}
template <int V>
__device__ __forceinline__ Vec<V> mul(const Vec<V> &a, float b) {
  return mul(a, all<V>(b));
}
template <int V>
__device__ __forceinline__ Vec<V> add(const Vec<V> &a, float b) {
  return add(a, all<V>(b));
}
template <int V>
__device__ __forceinline__ float sum(const Vec<V> &a) {
  if constexpr (V == 1) {
    return a[0];
  } else if constexpr (V % 2) {
    Vec<V - 1> h;
#pragma unroll
    for (int i = 0; i < V - 1; ++i) h[i] = a[i];
    return sum(h) + a[V - 1];
  } else {
    Vec<V / 2> h, l;
#pragma unroll
    for (int i = 0; i < V / 2; ++i) h[i] = a[i], l[i] = a[i + V / 2];
    return sum(add(h, l));
  }
}
template <typename T, int V>
__device__ __forceinline__ Vec<V> values(const Raw<T, V> &raw) {
  Vec<V> r;
  unpack<T, V>(raw, r.v);
  return r;
}
template <typename T, int V>
__device__ __forceinline__ void load_vec(const T *p, float *out) {
  const Raw<T, V> raw = *reinterpret_cast<const Raw<T, V> *>(p);
  unpack<T, V>(raw, out);
}
template <typename T, int V>
__device__ __forceinline__ void store_vec(T *p, const float *in) {
  *reinterpret_cast<Raw<T, V> *>(p) = pack<T, V>(in);
}

// A kernel that reads what the kernel before it wrote is launched to start while
// that one ends (launch_next): it waits here before it reads or writes any of
// that, and the earlier kernel says near its end that blocks may start.
__device__ __forceinline__ void wait_for_previous() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}
__device__ __forceinline__ void let_next_start() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
// The launch error, if any, is left for cudaGetLastError.
template <typename... P, typename... A>
inline void launch_next(void (*kernel)(P...), dim3 grid, dim3 block, int cluster,
                        cudaStream_t st, A... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = (unsigned)cluster;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  (void)cudaLaunchKernelEx(&cfg, kernel, args...);
}

// Calls f with a value of the element type that dtype names.
template <typename F>
inline void with_dtype(int32_t dtype, F &&f) {
  if (dtype == ZRL_F32) f(float{});
  else if (dtype == ZRL_BF16) f(__nv_bfloat16{});
  else f(__half{});
}

}  // namespace zrl
