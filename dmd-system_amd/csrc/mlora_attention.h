// What the attention kernels share: their tiles in LDS, fragments, matrix products and masks.
//
// Every product is D[32 x 32] += A[32 x 16] · B[16 x 32] per step (mma16): a lane holds row (or column)
// lane % 32 of an operand and 8 of the step's 16 contraction elements, the half lane / 32 decides which
// (bf16: one v_mfma_f32_32x32x16_bf16; float32: eight v_mfma_f32_32x32x2_f32, one per element). The result
// leaves lane l with column l % 32 and rows 8·(i / 4) + 4·(l / 32) + i % 4, i = 0 .. 15.
//
// The kernels compute transposed tiles, S^T = K·Q^T (or S = Q·K^T in the dK / dV kernel), so that a lane's 16
// results are 16 contraction elements of the *next* product's B operand for the same column: elements
// 8s .. 8s + 7 are step s, in the order perm(h, j) = 16s + 8·(j / 4) + 4h + j % 4. P and dS therefore go
// from one product to the next in registers; the other operand is read from LDS in that order, transposed
// (ds_read_b64_tr_b16 for bf16, single floats for float32).
#pragma once

#include "mlora_common.h"
#include "mlora_host.h"

#include <type_traits>

namespace mlora {

typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));

template <class T>
struct Frag;  // 8 contraction elements of one row or column
template <>
struct Frag<uint16_t> {
  u32x4 v;
};
template <>
struct Frag<float> {
  float v[8];
};

__device__ __forceinline__ f32x16 mma16(const Frag<uint16_t> &a, const Frag<uint16_t> &b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf16x8(a.v), as_bf16x8(b.v), c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma16(const Frag<float> &a, const Frag<float> &b, f32x16 c) {
#pragma unroll
  for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.v[j], b.v[j], c, 0, 0, 0);
  return c;
}

// Results 8s .. 8s + 7 of a 32 x 32 tile as the next product's B operand. bf16: rounded to nearest.
__device__ __forceinline__ void to_frag(const f32x16 &x, int s, Frag<uint16_t> &f) {
#pragma unroll
  for (int j = 0; j < 4; ++j) f.v[j] = pack2_bf16(x[8 * s + 2 * j], x[8 * s + 2 * j + 1]);
}
__device__ __forceinline__ void to_frag(const f32x16 &x, int s, Frag<float> &f) {
#pragma unroll
  for (int j = 0; j < 8; ++j) f.v[j] = x[8 * s + j];
}

// What that rounding left, as a second operand.
__device__ __forceinline__ void rest_frag(const f32x16 &x, int s, const Frag<uint16_t> &f, Frag<uint16_t> &r) {
#pragma unroll
  for (int j = 0; j < 4; ++j)
    r.v[j] = pack2_bf16(x[8 * s + 2 * j] - __uint_as_float(f.v[j] << 16),
                        x[8 * s + 2 * j + 1] - __uint_as_float(f.v[j] & 0xffff0000u));
}

// The other half's value (lane ^ 32): max and sum over the two halves of a column.
__device__ __forceinline__ float half_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float half_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// A tile of ROWS rows of DP elements in LDS (DP: the head dimension padded to 64 or 128; loads past it
// read as zero). Chunk c (16 bytes) of row r is stored at slot c ^ swz(r):
//   16 rows read at one chunk (row fragments) hit 16 slots, every bank once;
//   4 rows x 64 bytes (a transposing bf16 read) fall on 4 different 64-byte groups of the 256-byte bank row;
//   a float32 column read meets the other half's row (4 further down) on the other 128 bytes.
template <class T, int DP>
struct HeadTile {
  static constexpr int E = sizeof(T), RB = DP * E, CH = RB / 16, RPL = 1024 / RB;
  static __device__ __forceinline__ int swz(int r) {
    if constexpr (E == 4) return (((r >> 2) & 1) << 3) | ((r & 3) << 1) | ((r >> 3) & 1);
    else if constexpr (CH == 16) return ((r & 3) << 2) | ((r >> 2) & 3);
    else return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
  }
};

// A lane's addresses for fragment reads of a HeadTile.
template <class T, int DP>
struct FragReader;

// rows<OFF, R0>: rows R0 + lane % 32 (R0 a multiple of 32) of the tile OFF bytes past the reader's base, contraction
// elements 16s + 8h .. + 7 of the row. cols<OFF, R0>: columns 32d + lane % 32, contraction over rows R0 + perm(h, j) (R0 a
// multiple of 16).
template <int DP>
struct FragReader<uint16_t, DP> {
  using Tile = HeadTile<uint16_t, DP>;
  int32_t row[DP / 16];     // LDS address of row lane % 32, chunk of step s
  int32_t col[DP / 32][2];  // transposed: d block, first and second group of four rows
  __device__ __forceinline__ void init(int lane, const MLORA_LDS char *base) {
    const int32_t at = (int32_t)(uintptr_t)base;
    const int r = lane & 31, h = lane >> 5;
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) row[s] = at + r * Tile::RB + (((2 * s + h) ^ Tile::swz(r)) << 4);
    // group g of 16 lanes: columns 16·(g & 1) .. + 15 of the block, rows 4·(g >> 1) + e; lane m = 4e + c of
    // the group addresses row e, columns 4c .. 4c + 3, and receives column m of the four rows
    const int g = lane >> 4, m = lane & 15, e = m >> 2, c = m & 3;
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const int key = 8 * w + 4 * (g >> 1) + e, chunk = 4 * d + 2 * (g & 1) + (c >> 1);
        col[d][w] = at + key * Tile::RB + ((chunk ^ Tile::swz(key)) << 4) + 8 * (c & 1);
      }
  }
  // the other buffer: every address ^ by (the base and the tiles of a buffer within an aligned block of `by` bytes)
  __device__ __forceinline__ void flip(int by) {
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) row[s] ^= by;
#pragma unroll
    for (int d = 0; d < DP / 32; ++d) col[d][0] ^= by, col[d][1] ^= by;
  }
  template <int OFF, int R0>
  __device__ __forceinline__ void rows(int s, Frag<uint16_t> &f) const {
    f.v = *(const lds_u4 *)((const MLORA_LDS char *)(uintptr_t)(uint32_t)row[s] + OFF + R0 * Tile::RB);
  }
  template <int OFF, int R0>
  __device__ __forceinline__ void cols(int d, Frag<uint16_t> &f) const {
    typedef MLORA_LDS bf16x4 lds_b4;
    const MLORA_LDS char *p = (const MLORA_LDS char *)(uintptr_t)(uint32_t)col[d][0] + OFF + R0 * Tile::RB;
    const MLORA_LDS char *r = (const MLORA_LDS char *)(uintptr_t)(uint32_t)col[d][1] + OFF + R0 * Tile::RB;
    const u32x2 x = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_b4 *)p));
    const u32x2 y = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_b4 *)r));
    f.v = u32x4{x[0], x[1], y[0], y[1]};
  }
};

template <int DP>
struct FragReader<float, DP> {
  using Tile = HeadTile<float, DP>;
  int32_t row, col, sw, h, lane32;
  __device__ __forceinline__ void init(int lane, const MLORA_LDS char *base) {
    lane32 = lane & 31, h = lane >> 5, sw = Tile::swz(lane32);
    col = (int32_t)(uintptr_t)base, row = col + lane32 * Tile::RB;
  }
  __device__ __forceinline__ void flip(int by) { row ^= by, col ^= by; }
  template <int OFF, int R0>
  __device__ __forceinline__ void rows(int s, Frag<float> &f) const {
    const MLORA_LDS char *t = (const MLORA_LDS char *)(uintptr_t)(uint32_t)row + OFF + R0 * Tile::RB;
    const f32x4 a = *(const lds_f4 *)(t + (((4 * s + 2 * h) ^ sw) << 4)), b = *(const lds_f4 *)(t + (((4 * s + 2 * h + 1) ^ sw) << 4));
#pragma unroll
    for (int j = 0; j < 4; ++j) f.v[j] = a[j], f.v[j + 4] = b[j];
  }
  template <int OFF, int R0>
  __device__ __forceinline__ void cols(int d, Frag<float> &f) const {
    const MLORA_LDS char *t = (const MLORA_LDS char *)(uintptr_t)(uint32_t)col + OFF;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int r = 8 * (j / 4) + 4 * h + j % 4, chunk = 8 * d + (lane32 >> 2);  // swz(R0 + r) = swz(r)
      f.v[j] = *(const MLORA_LDS float *)(t + (R0 + r) * Tile::RB + ((chunk ^ Tile::swz(r)) << 4) + 4 * (lane32 & 3));
    }
  }
};

// Loads a tile's rows straight into LDS, N of its 1024-byte blocks (RPL rows each) by the calling wave: blocks
// first, first + step, ... Rows that are not live and chunks past the head dimension read as zero (their offset is
// past the buffer), so whatever lies in masked rows never enters a product.
template <class T, int DP, int N>
struct TileLoader {
  using Tile = HeadTile<T, DP>;
  int32_t off[N];  // byte offset of the lane's chunk within the tile's rows; kOOB past the head dimension
  int32_t first, step, r0;
  __device__ __forceinline__ void init(int lane, int first_block, int block_step, int64_t stride, int head_dim) {
    first = first_block, step = block_step, r0 = lane / Tile::CH;
    const int slot = lane % Tile::CH;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int r = (first + i * step) * Tile::RPL + r0, c = slot ^ Tile::swz(r);
      off[i] = c * 16 < head_dim * Tile::E ? (int32_t)(r * stride * Tile::E) + c * 16 : kOOB;
    }
  }
  // base: the tile's first row; live: one bit per row (tiles of at most 64 rows)
  __device__ __forceinline__ void load(const void *base, uint64_t live, MLORA_LDS char *lds) const {
    const auto rsrc = make_rsrc(base, (int64_t)kOOB);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int blk = first + i * step;
      const bool on = (live >> (blk * Tile::RPL + r0)) & 1;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (MLORA_LDS void *)(lds + blk * 1024), 16, on ? off[i] : kOOB, 0, 0, 0);
    }
  }
};

__device__ __forceinline__ uint64_t low_bits(int n) { return n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1; }

constexpr float kLog2e = 1.4426950408889634f;

}  // namespace mlora
