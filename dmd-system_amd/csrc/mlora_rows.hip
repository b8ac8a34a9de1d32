// Fixed-order column sums of the partial rows that the row kernels' backward passes leave (mlora_rows.h).
//
// A workgroup owns 64 columns of one output: thread (g, q) adds rows g, g + 16, ... of the columns
// 4q .. 4q + 3 (16-byte loads), then the 16 groups are added in order through LDS. Latency bounds it:
// a few hundred partial rows of a few thousand columns.
#include "mlora_rows.h"

namespace mlora {

constexpr int kColSumCols = 64, kColSumGroups = 16;

__global__ __launch_bounds__(256) void col_sums_kernel(const ColSums s) {
  int blk = blockIdx.x, j = 0;
  for (; j + 1 < s.n; ++j) {
    const int n = s.job[j].batches * ((s.job[j].width + kColSumCols - 1) / kColSumCols);
    if (blk < n) break;
    blk -= n;
  }
  const ColSumJob &a = s.job[j];
  const int per = (a.width + kColSumCols - 1) / kColSumCols;
  const int64_t b = blk / per;
  const int q = threadIdx.x & 15, g = threadIdx.x >> 4;
  const int col = (blk % per) * kColSumCols + 4 * q;
  __shared__ f32x4 red[kColSumGroups][16];
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  if (col < a.width) {
    const MLORA_GLOBAL float *p = gp(a.src) + b * a.batch_stride + g * a.row_stride + col;
    const int64_t step = kColSumGroups * a.row_stride;
#pragma unroll 8
    for (int r = g; r < a.rows; r += kColSumGroups, p += step) acc += *(const MLORA_GLOBAL f32x4 *)p;
  }
  red[g][q] = acc;
  __syncthreads();
  if (g != 0 || col >= a.width) return;
#pragma unroll
  for (int i = 1; i < kColSumGroups; ++i) acc += red[i][q];
  const int64_t e = b * a.width + col;
  if (a.out_f32) {
    *(MLORA_GLOBAL f32x4 *)(static_cast<float *>(a.out) + e) = acc;
  } else {
    *(MLORA_GLOBAL u32x2 *)(static_cast<uint16_t *>(a.out) + e) = u32x2{pack2_bf16(acc[0], acc[1]), pack2_bf16(acc[2], acc[3])};
  }
}

int launch_col_sums(const ColSums &s, hipStream_t stream) {
  int64_t blocks = 0;
  for (int j = 0; j < s.n; ++j)
    blocks += (int64_t)s.job[j].batches * ((s.job[j].width + kColSumCols - 1) / kColSumCols);
  if (blocks == 0) return MLORA_OK;
  if (blocks > INT32_MAX) return MLORA_ERR_LIMIT;
  hipLaunchKernelGGL(col_sums_kernel, dim3((unsigned)blocks), dim3(256), 0, stream, s);
  return launch_status();
}

}  // namespace mlora
