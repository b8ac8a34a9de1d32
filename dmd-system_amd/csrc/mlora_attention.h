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
  __device__ __forceinline__ void load_all(const void *base, MLORA_LDS char *lds) const {  // every row is live
    const auto rsrc = make_rsrc(base, (int64_t)kOOB);
#pragma unroll
    for (int i = 0; i < N; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (MLORA_LDS void *)(lds + (first + i * step) * 1024), 16, off[i], 0, 0, 0);
  }
};

__device__ __forceinline__ uint64_t low_bits(int n) { return n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1; }

constexpr float kLog2e = 1.4426950408889634f;

// 8 elements at base + off, or zeros (base itself is always readable: no branch around the load).
__device__ __forceinline__ void load_frag(const uint16_t *base, int64_t off, bool on, Frag<uint16_t> &f) {
  const u32x4 v = *(const MLORA_GLOBAL u32x4 *)(base + (on ? off : 0));
#pragma unroll
  for (int j = 0; j < 4; ++j) f.v[j] = on ? v[j] : 0;
}
__device__ __forceinline__ void load_frag(const float *base, int64_t off, bool on, Frag<float> &f) {
  const float *p = base + (on ? off : 0);
  const f32x4 a = *(const MLORA_GLOBAL f32x4 *)p, b = *(const MLORA_GLOBAL f32x4 *)(p + 4);
#pragma unroll
  for (int j = 0; j < 4; ++j) f.v[j] = on ? a[j] : 0.f, f.v[j + 4] = on ? b[j] : 0.f;
}

// The running maximum before any key: below every other score, but finite, so that 2^(−inf − m) is 0 and not NaN where
// a block has no live key.
constexpr float kNoMax = -3.4028234664e38f;

// What a row's exponents are relative to: P = 2^((s − a)·c − r), a function of the row's largest product m alone. Near
// zero a = 0 and r = m·c rounded, off by 2^-15 at most, the same for the whole row; far from zero a = m and r = 0, since
// the rounding of m·c would grow with it and end in 2^128 or 0 (at |m·c| of 3e9).
struct RowRef {
  float a, r;
};
constexpr float kFar = 1024.f;
__device__ __forceinline__ RowRef row_ref(float m, float c) {
  const float mc = m * c;
  const bool far = !(fabsf(mc) < kFar);
  return {far ? m : 0.f, far ? 0.f : mc};
}
// 2^(x − y): what sums relative to x become relative to y.
__device__ __forceinline__ float ref_factor(const RowRef &x, const RowRef &y, float c) {
  return __builtin_amdgcn_exp2f(__builtin_fmaf(x.a - y.a, c, x.r - y.r));
}
// The logarithm of a row's sum l relative to row_ref(m): +inf without keys, finite for finite scores.
__device__ __forceinline__ float row_lse(float m, float l, float c) {
  const float mc = fminf(fmaxf(m * c, kNoMax), -kNoMax);
  return l > 0.f ? mc + __builtin_amdgcn_logf(l) : l != l ? l : INFINITY;
}

// The running softmax of NQ x 32 queries (a column per lane and half) against KT keys per step. EXACT: e sums the weights
// before their rounding to bf16, for lse: the backward forms them unrounded, and where a row rests on few keys the two sums
// are up to half a bf16 step apart (a factor of all of its gradients). 16 additions more per 32 x 32 block; l is e elsewhere.
template <class T, int DP, int NQ, int KT, bool EXACT>
struct Softmax {
  static constexpr bool kTwoSums = EXACT && sizeof(T) == 2;
  f32x16 o[NQ][DP / 32];
  Frag<T> q[NQ][DP / 16];
  float m[NQ], l[NQ], e[NQ];  // the largest product so far, the sums relative to row_ref(m)

  __device__ __forceinline__ void init() {
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      m[n] = kNoMax, l[n] = 0.f, e[n] = 0.f;
#pragma unroll
      for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[n][d][i] = 0.f;
    }
  }

  // One tile of keys KOFF bytes from the reader's base, V at VOFF. bits: the keys that count, the same for every lane; or
  // (`masked` then says whether any query lacks one) those of the lane's queries.
  template <int KOFF, int VOFF>
  __device__ __forceinline__ void step(const FragReader<T, DP> &fr, uint64_t bits, float c, int lane) {
    uint64_t all[NQ];
#pragma unroll
    for (int n = 0; n < NQ; ++n) all[n] = bits;
    step<KOFF, VOFF>(fr, bits != low_bits(KT), all, c, lane);
  }
  template <int KOFF, int VOFF>
  __device__ __forceinline__ void step(const FragReader<T, DP> &fr, bool masked, const uint64_t (&bits)[NQ], float c, int lane) {
    constexpr int NB = KT / 32;
    f32x16 s[NQ][NB];
#pragma unroll
    for (int n = 0; n < NQ; ++n)
#pragma unroll
      for (int kb = 0; kb < NB; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[n][kb][i] = 0.f;
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks)  // the blocks' sums in turn: a sum waits for its last product
      static_for<NB>([&](auto kb) __attribute__((always_inline)) {
        Frag<T> kf;
        fr.template rows<KOFF, 32 * decltype(kb)::value>(ks, kf);
#pragma unroll
        for (int n = 0; n < NQ; ++n) s[n][kb] = mma16(kf, q[n][ks], s[n][kb]);
        return true;
      });
    if (masked) {
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        const uint64_t mine = bits[n] >> (4 * (lane >> 5));
#pragma unroll
        for (int kb = 0; kb < NB; ++kb)
#pragma unroll
          for (int i = 0; i < 16; ++i)
            s[n][kb][i] = (mine >> (32 * kb + 8 * (i / 4) + i % 4)) & 1 ? s[n][kb][i] : -INFINITY;
      }
    }
    Frag<T> p[NQ][KT / 16];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      float mx = s[n][0][0];
#pragma unroll
      for (int kb = 0; kb < NB; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[n][kb][i]);
      mx = half_max(mx);
      RowRef ref = row_ref(m[n], c);
      if (__any(__builtin_fmaf(mx - ref.a, c, -ref.r) > 8.f)) {
        m[n] = fmaxf(m[n], mx);
        const RowRef up = row_ref(m[n], c);
        const float f = ref_factor(ref, up, c);
        ref = up;
        l[n] *= f, e[n] *= f;
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
#pragma unroll
          for (int i = 0; i < 16; ++i) o[n][d][i] *= f;
      }
      if (__any(ref.a != 0.f)) {
#pragma unroll
        for (int kb = 0; kb < NB; ++kb)
#pragma unroll
          for (int i = 0; i < 16; ++i) s[n][kb][i] -= ref.a;
      }
#pragma unroll
      for (int kb = 0; kb < NB; ++kb) {
#pragma unroll
        for (int i = 0; i < 16; ++i) s[n][kb][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[n][kb][i], c, -ref.r));
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) to_frag(s[n][kb], ks, p[n][2 * kb + ks]);
        if constexpr (kTwoSums) {
          float t[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) t[i] = (s[n][kb][i] + s[n][kb][4 + i]) + (s[n][kb][8 + i] + s[n][kb][12 + i]);
          e[n] += (t[0] + t[1]) + (t[2] + t[3]);
        }
      }
      l[n] += frag_sum(p[n]);
    }
    static_for<KT / 16>([&](auto ks) __attribute__((always_inline)) {
#pragma unroll
      for (int d = 0; d < DP / 32; ++d) {
        Frag<T> vf;
        fr.template cols<VOFF, 16 * decltype(ks)::value>(d, vf);
#pragma unroll
        for (int n = 0; n < NQ; ++n) o[n][d] = mma16(vf, p[n][ks], o[n][d]);
      }
      return true;
    });
  }

  // The row's whole sums over both halves; f: what makes O a sum of weights that add up to e where they added up to l.
  __device__ __forceinline__ float sums(int n, float &f) {
    const float lw = half_sum(l[n]);
    f = 1.f;
    if constexpr (!kTwoSums) return lw;
    const float ew = half_sum(e[n]);
    if (lw > 0.f) f = ew / lw;
    return lw > 0.f ? ew : lw;
  }

  // The sum of the weights as the product with V sees them (bf16: two per v_dot2_f32_bf16 with ones).
  static __device__ __forceinline__ float frag_sum(const Frag<T> (&p)[KT / 16]) {
    float t = 0.f;
#pragma unroll
    for (int ks = 0; ks < KT / 16; ++ks) {
      if constexpr (sizeof(T) == 2) {
        const auto ones = __builtin_bit_cast(bf16x2, 0x3f803f80u);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          t = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, (uint32_t)p[ks].v[j]), ones, t, false);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) t += p[ks].v[j];
      }
    }
    return t;
  }
};

// Writes NQ x 32 rows of the O^T registers (times f[n]) to base, row r at element at_row(r) of it. The halves of a column hold alternating groups of
// four channels; they swap groups, so that a lane has eight neighbouring channels: one 16-byte store of bf16.
template <class T, int DP, int NQ, class At>
__device__ __forceinline__ void store_rows(T *base, const f32x16 (&o)[NQ][DP / 32], const float (&f)[NQ], int row0, int rows,
                                           At &&at_row, int D, int lane) {
  auto swap = [](uint32_t &x, uint32_t &y) __attribute__((always_inline)) {
    const auto r = __builtin_amdgcn_permlane32_swap(x, y, false, false);
    x = r[0], y = r[1];
  };
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int r = row0 + 32 * n + (lane & 31);
    T *p = base + at_row(min(r, rows - 1)) + 8 * (lane >> 5);
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
      for (int i = 0; i < 4; i += 2) {
        const int at = 32 * d + 8 * i + 8 * (lane >> 5);  // the head dimension is a multiple of 8
        uint32_t x[4], y[4];
        if constexpr (sizeof(T) == 2) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            x[j] = pack2_bf16(o[n][d][4 * i + 2 * j] * f[n], o[n][d][4 * i + 2 * j + 1] * f[n]);
            y[j] = pack2_bf16(o[n][d][4 * i + 4 + 2 * j] * f[n], o[n][d][4 * i + 5 + 2 * j] * f[n]);
            swap(x[j], y[j]);
          }
          if (r < rows && at < D) *(MLORA_GLOBAL u32x4 *)(p + 32 * d + 8 * i) = u32x4{x[0], x[1], y[0], y[1]};
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            x[j] = __float_as_uint(o[n][d][4 * i + j] * f[n]), y[j] = __float_as_uint(o[n][d][4 * i + 4 + j] * f[n]);
            swap(x[j], y[j]);
          }
          if (r < rows && at < D) {
            *(MLORA_GLOBAL u32x4 *)(p + 32 * d + 8 * i) = u32x4{x[0], x[1], x[2], x[3]};
            *(MLORA_GLOBAL u32x4 *)(p + 32 * d + 8 * i + 4) = u32x4{y[0], y[1], y[2], y[3]};
          }
        }
      }
  }
}

template <class T>
struct AttnTile {
  static constexpr int KT = sizeof(T) == 2 ? 64 : 32;  // keys per tile: 16 KB of K and of V at 128 channels
};

}  // namespace mlora
