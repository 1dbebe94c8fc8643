// dropout.cu -- dropout whose mask is a function of (seed, stream, row,
// column) and is drawn again wherever it is needed, forward and backward.
#include <math.h>

#include <algorithm>
#include <initializer_list>
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
  int64_t N, row0;     // rows of this launch, number of the first (rows == NULL)
  int32_t D, groups;   // columns; groups of 8 columns, or segments
  uint32_t drop;       // a lane below this is dropped
  float scale;
  uint2 key;
  uint32_t stream_id;
  uint32_t magic, shift;  // e / groups = umulhi(e, magic) >> shift, for e < 2^31
};

// Bit j: column j of the group is kept.
__device__ __forceinline__ uint32_t keep_bits(const DropoutArgs &a, int64_t id, uint32_t group) {
  const uint4 w = philox4x32_10(
      make_uint4(group, (uint32_t)id, (uint32_t)((uint64_t)id >> 32), a.stream_id), a.key);
  const uint32_t word[4] = {w.x, w.y, w.z, w.w};
  uint32_t bits = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    bits |= ((word[j] & 0xffffu) >= a.drop ? 1u : 0u) << (2 * j);
    bits |= ((word[j] >> 16) >= a.drop ? 2u : 0u) << (2 * j);
  }
  return bits;
}
__device__ __forceinline__ uint32_t quotient(const DropoutArgs &a, uint32_t e) {
  return a.groups == 1 ? e : __umulhi(e, a.magic) >> a.shift;
}

// Whole groups of eight columns on 16-byte boundaries: a thread per group, one
// generator call and 16-byte accesses (two where elements have four bytes), two
// groups in flight.  The generator is about 60 of the 130 issue slots of a group,
// so that 16-bit data without a residual is bound by them and by memory alike.
// 24576 x 512 bf16 with a residual: 14.0 us (5.4 TB/s); a thread per group with
// scalar accesses took 35.5.
template <typename T, bool RES>
__global__ void __launch_bounds__(256) dropout_vec_kernel(const __grid_constant__ DropoutArgs a) {
  constexpr int H = 16 / (int)sizeof(T), PARTS = 8 / H, U = 2;
  const uint32_t total = (uint32_t)(a.N * a.groups), pace = gridDim.x * 256;
  for (uint32_t e0 = blockIdx.x * 256 + threadIdx.x; e0 < total; e0 += U * pace) {
    Raw<T, H> x[U][PARTS], r[U][PARTS];
    uint32_t row[U], group[U];
    int64_t id[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t e = e0 + u * pace;
      if (e >= total) break;
      row[u] = quotient(a, e);
      group[u] = e - row[u] * a.groups;
      id[u] = a.rows ? a.rows[row[u]] : a.row0 + row[u];
      const T *xp = static_cast<const T *>(a.x) + (int64_t)row[u] * a.sx + group[u] * 8;
      const T *rp = static_cast<const T *>(a.residual) + (int64_t)row[u] * a.sr + group[u] * 8;
#pragma unroll
      for (int i = 0; i < PARTS; ++i) {
        x[u][i] = *reinterpret_cast<const Raw<T, H> *>(xp + i * H);
        if (RES) r[u][i] = *reinterpret_cast<const Raw<T, H> *>(rp + i * H);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (e0 + u * pace >= total) break;
      const uint32_t bits = keep_bits(a, id[u], group[u]);
      T *yp = static_cast<T *>(a.y) + (int64_t)row[u] * a.sy + group[u] * 8;
#pragma unroll
      for (int i = 0; i < PARTS; ++i) {
        Vec<H> v = mul(values<T, H>(x[u][i]), a.scale);
#pragma unroll
        for (int j = 0; j < H; ++j) v[j] = bits >> (i * H + j) & 1 ? v[j] : 0.0f;
        if (RES) v = add(v, values<T, H>(r[u][i]));
        store_vec<T, H>(yp + i * H, v.v);
      }
    }
  }
}

// Any width, stride and alignment: W = 2^WIDE lanes per row and segment of 8 W
// columns.  Lane l of them draws group l; column k W + l takes its bit from
// the lane that has its group, so every access is to neighbouring elements.
// 98304 x 333 f32: 51 us (5.1 TB/s); a thread per group took 146.
template <typename T, int WIDE>
__global__ void __launch_bounds__(256) dropout_kernel(const __grid_constant__ DropoutArgs a) {
  constexpr uint32_t W = 1u << WIDE, at_once = 32u >> WIDE;
  const uint32_t lane = threadIdx.x & 31, q = lane & (W - 1);
  const uint32_t total = (uint32_t)(a.N * a.groups);
  // every lane of a warp takes part in the exchange, with a row or without
  for (uint32_t e0 = (blockIdx.x * 8 + (threadIdx.x >> 5)) * at_once; e0 < total;
       e0 += gridDim.x * 8 * at_once) {
    const uint32_t e = e0 + (lane >> WIDE);
    const bool on = e < total;
    const uint32_t row = on ? quotient(a, e) : 0, segment = on ? e - row * a.groups : 0;
    const int64_t id = a.rows ? a.rows[row] : a.row0 + row;
    const int c0 = segment * 8 * W + q, end = on ? a.D : 0;
    const T *x = static_cast<const T *>(a.x) + (int64_t)row * a.sx + c0;
    const T *r = static_cast<const T *>(a.residual) + (int64_t)row * a.sr + c0;
    T *y = static_cast<T *>(a.y) + (int64_t)row * a.sy + c0;
    T xv[8], rv[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (c0 + (k << WIDE) < end) {
        xv[k] = x[k << WIDE];
        if (a.residual) rv[k] = r[k << WIDE];
      }
    }
    const uint32_t mine = keep_bits(a, id, segment * W + q);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t c = (k << WIDE) + q;  // of the segment
      const uint32_t bits = __shfl_sync(0xffffffffu, mine, (lane - q) + (c >> 3));
      if (c0 + (k << WIDE) < end) {
        float v = bits >> (c & 7) & 1 ? to_f32(xv[k]) * a.scale : 0.0f;
        if (a.residual) v += to_f32(rv[k]);
        y[k << WIDE] = from_f32<T>(v);
      }
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
  a.D = (int32_t)D;
  const double drop = nearbyint(65536.0 * p);
  a.drop = (uint32_t)drop;
  a.scale = drop < 65536.0 ? (float)(65536.0 / (65536.0 - drop)) : 0.0f;
  a.key = make_uint2((uint32_t)seed, (uint32_t)(seed >> 32));
  a.stream_id = stream_id;
  bool vec = D % 8 == 0 && aligned(x, 16) && aligned(y, 16) && aligned(residual, 16);
  for (int64_t st : {a.sx, residual ? a.sr : a.sx, a.sy}) vec = vec && (N == 1 || st * es % 16 == 0);
  // the segment that leaves the fewest lanes without columns, the widest of them
  int wide = 5;
  int64_t best = INT64_MAX;
  for (int w : {5, 4, 3, 1}) {
    const int64_t lanes = (D + (8 << w) - 1) / (8 << w) << w;
    if (lanes < best && (w >= 3 || D <= 8 << w)) best = lanes, wide = w;
  }
  a.groups = (int32_t)(vec ? D / 8 : (D + (8 << wide) - 1) / (8 << wide));
  while ((1u << a.shift) < (uint32_t)a.groups) ++a.shift;
  a.shift = a.shift ? a.shift - 1 : 0;
  a.magic = (uint32_t)((((uint64_t)1 << (32 + a.shift)) + a.groups - 1) / a.groups);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  // launches of fewer than 2^31 groups
  const int64_t most = std::max<int64_t>(1, (((int64_t)1 << 31) - 1) / a.groups);
  for (int64_t n0 = 0; n0 < N; n0 += most) {
    a.N = std::min(most, N - n0);
    a.row0 = n0;
    const int64_t units = vec ? (a.N * a.groups + 255) / 256 : ((a.N * a.groups << wide) + 255) / 256;
    const unsigned blocks = (unsigned)std::min<int64_t>(units, 148 * (vec ? 4 : 16));
    with_dtype(dtype, [&](auto t) {
      using T = decltype(t);
      if (!vec && wide == 5) dropout_kernel<T, 5><<<blocks, 256, 0, st>>>(a);
      else if (!vec && wide == 4) dropout_kernel<T, 4><<<blocks, 256, 0, st>>>(a);
      else if (!vec && wide == 3) dropout_kernel<T, 3><<<blocks, 256, 0, st>>>(a);
      else if (!vec) dropout_kernel<T, 1><<<blocks, 256, 0, st>>>(a);
      else if (residual) dropout_vec_kernel<T, true><<<blocks, 256, 0, st>>>(a);
      else dropout_vec_kernel<T, false><<<blocks, 256, 0, st>>>(a);
    });
    auto on = [&](auto &ptr, int64_t elements, int size) {
      if (ptr) ptr = (std::remove_reference_t<decltype(ptr)>)((char *)ptr + elements * size);
    };
    on(a.x, most * a.sx, es);
    on(a.residual, most * a.sr, es);
    on(a.y, most * a.sy, es);
    on(a.rows, most, 8);
  }
  return seq_launched("dropout");
}
