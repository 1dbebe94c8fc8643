// dropout.cu -- dropout whose mask is a function of (seed, stream, row,
// column) and is drawn again wherever it is needed, forward and backward.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "philox.cuh"
#include "seq_common.cuh"

namespace zrl {
namespace {

struct DropoutArgs {
  const void *x, *residual;
  const int64_t *rows;
  void *y;
  int64_t sx, sr, sy;  // row strides, elements
  int64_t N, row0;     // rows, number of the first (rows == NULL)
  int32_t D, groups;   // columns, groups of 8 columns
  uint32_t drop;       // a lane below this is dropped
  float scale;
  uint2 key;
  uint32_t stream_id;
};

// One thread per group of eight columns.
template <typename T>
__global__ void __launch_bounds__(256) dropout_kernel(const DropoutArgs a) {
  const int64_t total = a.N * a.groups;
  for (int64_t e = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; e < total;
       e += (int64_t)gridDim.x * blockDim.x) {
    const int64_t row = e / a.groups;
    const int g = (int)(e - row * a.groups);
    const int64_t id = a.rows ? a.rows[row] : row;
    const uint4 w = philox4x32_10(
        make_uint4((uint32_t)g, (uint32_t)id, (uint32_t)((uint64_t)id >> 32), a.stream_id),
        a.key);
    const uint32_t word[4] = {w.x, w.y, w.z, w.w};
    const T *x = static_cast<const T *>(a.x) + row * a.sx;
    const T *r = a.residual ? static_cast<const T *>(a.residual) + row * a.sr : nullptr;
    T *y = static_cast<T *>(a.y) + row * a.sy;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int col = g * 8 + j;
      if (col >= a.D) break;
      const uint32_t lane = (word[j / 2] >> (16 * (j & 1))) & 0xffffu;
      float v = lane >= a.drop ? to_f32(x[col]) * a.scale : 0.0f;
      if (r) v += to_f32(r[col]);
      y[col] = from_f32<T>(v);
    }
  }
}

}  // namespace
}  // namespace zrl

using namespace zrl;

extern "C" zrl_status zrl_dropout(const void *x, const void *residual, const int64_t *rows,
                                  int64_t N, int64_t D, int32_t dtype, double p,
                                  uint64_t seed, uint32_t stream_id, const int64_t *strides,
                                  void *y, void *stream) {
  if (N < 0 || D < 0 || D > (int64_t)1 << 30)
    return seq_fail(ZRL_INVALID_ARG, "dropout: N >= 0 and 0 <= D <= 2^30");
  if (!dtype_ok(dtype)) return seq_fail(ZRL_INVALID_ARG, "dropout: unknown dtype %d", dtype);
  if (!(p >= 0.0 && p <= 1.0)) return seq_fail(ZRL_INVALID_ARG, "dropout: p outside [0, 1]");
  if (N == 0 || D == 0) return ZRL_OK;
  if (!x || !y) return seq_fail(ZRL_INVALID_ARG, "dropout: x or y is NULL");
  const int es = dtype_size(dtype);
  if (!aligned(x, es) || !aligned(y, es) || !aligned(residual, es) || !aligned(rows, 8))
    return seq_fail(ZRL_INVALID_ARG, "dropout: a pointer is not aligned to its element");
  DropoutArgs a{};
  a.x = x;
  a.residual = residual;
  a.rows = rows;
  a.y = y;
  a.sx = strides ? strides[0] : D;
  a.sr = strides ? strides[1] : D;
  a.sy = strides ? strides[2] : D;
  if (N > 1 && a.sy < D && a.sy > -D)
    return seq_fail(ZRL_INVALID_ARG, "dropout: rows of y overlap");
  a.N = N;
  a.D = (int32_t)D;
  a.groups = (int32_t)((D + 7) / 8);
  const double drop = nearbyint(65536.0 * p);
  a.drop = (uint32_t)drop;
  a.scale = drop < 65536.0 ? (float)(65536.0 / (65536.0 - drop)) : 0.0f;
  a.key = make_uint2((uint32_t)seed, (uint32_t)(seed >> 32));
  a.stream_id = stream_id;
  const int64_t blocks = std::min<int64_t>((N * a.groups + 255) / 256, 148 * 32);
  with_dtype(dtype, [&](auto t) {
    dropout_kernel<decltype(t)>
        <<<(unsigned)blocks, 256, 0, static_cast<cudaStream_t>(stream)>>>(a);
  });
  return seq_launched("dropout");
}
