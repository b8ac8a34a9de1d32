// What the kernels over token rows share (the modulated norm, the sublayer joint, the rotary
// positions): 8-value loads and stores of bf16 or float32 rows, a wave's sum, and the fixed-order
// column sums that finish a vector's gradient.
#pragma once

#include "mlora_common.h"
#include "mlora_host.h"

namespace mlora {

// Eight consecutive values at element offset e of a bf16 or float32 array.
__device__ __forceinline__ void load8(const void *base, bool f32, int64_t e, float (&v)[8]) {
  if (f32) {
    const float *p = static_cast<const float *>(base) + e;
    const f32x4 a = *(const MLORA_GLOBAL f32x4 *)p, b = *(const MLORA_GLOBAL f32x4 *)(p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = a[i], v[i + 4] = b[i];
  } else {
    const u32x4 u = *(const MLORA_GLOBAL u32x4 *)(static_cast<const uint16_t *>(base) + e);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = bf16_to_f32((uint16_t)(i % 2 ? u[i / 2] >> 16 : u[i / 2] & 0xffff));
  }
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) v += __shfl_xor(v, m);
  return v;
}

// v plus its value M lanes across (M = 1, 2, 4, ...: groups of M lanes already hold one value each, so that a
// mirrored half row is as good as an exchange), in the VALU's own lane moves: a shuffle through the LDS unit costs
// some hundred cycles, six of them per sum and several sums per row in a row's critical path.
template <int M>
__device__ __forceinline__ float lanes_add(float v) {
  const uint32_t u = __float_as_uint(v);
  if constexpr (M == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
  } else if constexpr (M == 32) {
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
  } else {
    constexpr int kMove = M == 1 ? 0xB1 : M == 2 ? 0x4E : M == 4 ? 0x141 : 0x140;  // quad pairs, quad halves, mirrors
    return v + __uint_as_float((uint32_t)__builtin_amdgcn_mov_dpp((int)u, kMove, 0xf, 0xf, false));
  }
}

// The sum of N neighbouring lanes (a power of two), in each of them.
template <int N>
__device__ __forceinline__ float lanes_sum(float v) {
  if constexpr (N >= 2) v = lanes_add<1>(v);
  if constexpr (N >= 4) v = lanes_add<2>(v);
  if constexpr (N >= 8) v = lanes_add<4>(v);
  if constexpr (N >= 16) v = lanes_add<8>(v);
  if constexpr (N >= 32) v = lanes_add<16>(v);
  if constexpr (N >= 64) v = lanes_add<32>(v);
  return v;
}

__device__ __forceinline__ void store8_any(void *base, bool f32, int64_t e, const float (&v)[8]) {
  if (f32) {
    float *p = static_cast<float *>(base) + e;
    *(MLORA_GLOBAL f32x4 *)p = f32x4{v[0], v[1], v[2], v[3]};
    *(MLORA_GLOBAL f32x4 *)(p + 4) = f32x4{v[4], v[5], v[6], v[7]};
  } else {
    *(MLORA_GLOBAL u32x4 *)(static_cast<uint16_t *>(base) + e) =
        u32x4{pack2_bf16(v[0], v[1]), pack2_bf16(v[2], v[3]), pack2_bf16(v[4], v[5]), pack2_bf16(v[6], v[7])};
  }
}

// Rows of 16-byte chunks: every row start 16-byte aligned.
inline bool rows_aligned(const void *p, int64_t sb, int64_t st) {
  return aligned16(p) && sb >= 0 && st >= 0 && sb % 8 == 0 && st % 8 == 0;
}

// Column sums of float32 partial rows: out[b, c] = Σ_r src[b·batch_stride + r·row_stride + c], r in a
// fixed order. One launch runs every job (mlora_rows.hip).
struct ColSumJob {
  const float *src;
  void *out;  // [batches, width], float32 or bf16
  int64_t batch_stride, row_stride;
  int32_t rows, batches, width, out_f32;
};

constexpr int kColSumJobs = 4;

struct ColSums {
  int32_t n = 0;
  ColSumJob job[kColSumJobs];
  void add(const ColSumJob &j) { job[n++] = j; }
};

int launch_col_sums(const ColSums &s, hipStream_t stream);

}  // namespace mlora
