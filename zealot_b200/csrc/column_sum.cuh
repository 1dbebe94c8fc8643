// column_sum.cuh -- sums of the columns of a row-major fp32 matrix in a fixed
// order: the last step of a parameter's gradient.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "seq_common.cuh"

namespace zrl {

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
// Stores a value at the same shared-memory place of another block of the cluster.
__device__ __forceinline__ void store_at(float *p, uint32_t rank, float v) {
  uint32_t a = (uint32_t)__cvta_generic_to_shared(p), r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(r), "f"(v) : "memory");
}

// out(column, sum) for every column of part [rows, cols].  A cluster takes 32
// columns: its blocks every ranks-th stretch of 32 rows, their sums meet in the
// first block.  Bound by latency: 4096 x 512 in 4.7 us (1.8 TB/s).
template <typename Out>
__global__ void __launch_bounds__(1024) column_sum_kernel(const float *part, int64_t rows,
                                                          int64_t cols, Out out) {
  __shared__ float buf[32][33];
  __shared__ float whole[8][32];
  const uint32_t ranks = cluster_size(), rank = cluster_rank();
  const int lane = threadIdx.x & 31, wy = threadIdx.x >> 5;
  const int64_t d = (int64_t)(blockIdx.x / ranks) * 32 + lane;
  if (ranks > 1) cluster_barrier();  // every block of the cluster runs
  wait_for_previous();
  float s = 0.0f;
  if (d < cols) {
#pragma unroll 4
    for (int64_t r = (int64_t)rank * 32 + wy; r < rows; r += (int64_t)ranks * 32)
      s += part[r * cols + d];
  }
  buf[wy][lane] = s;
  __syncthreads();
  if (wy == 0) {
    s = 0.0f;
#pragma unroll
    for (int i = 0; i < 32; ++i) s += buf[i][lane];
    if (ranks > 1) store_at(&whole[rank][lane], 0, s);
  }
  if (ranks > 1) {
    cluster_barrier();
    if (wy == 0) {
      s = 0.0f;
      for (uint32_t r = 0; r < ranks; ++r) s += whole[r][lane];
    }
  }
  if (wy == 0 && rank == 0 && d < cols) out(d, s);
}

// After the kernel that wrote part.
template <typename Out>
inline void launch_column_sum(const float *part, int64_t rows, int64_t cols, Out out,
                              cudaStream_t st) {
  const int ranks = rows >= 256 ? 8 : 1;
  launch_next(column_sum_kernel<Out>, dim3((unsigned)((cols + 31) / 32 * ranks)), dim3(1024),
              ranks, st, part, rows, cols, out);
}

}  // namespace zrl
