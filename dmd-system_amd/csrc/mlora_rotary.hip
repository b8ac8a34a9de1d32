// Rotary positions with several axes (time, height, width, ...) for the heads of q and k, with the
// RMSNorm that precedes them:
//
//   n = x · r · w,  r = 1 / sqrt(mean(x²) + eps)    over the token's whole row [H·D] or over each head [D];
//                                                   n = x without a norm
//   pair i of a head (elements 2i, 2i + 1, or i, i + D/2) belongs to one axis c, where it has the
//   frequency f_i:   φ = position[b, t, c] · f_i,   (a, b) -> (a cos φ − b sin φ, a sin φ + b cos φ)
//
// Backward: the upstream gradient is turned by −φ (g'), then, with n̂ = x·r:
//   dw = Σ_tokens g'·n̂ (summed over the heads too for a per-head weight);  h = g'·w;
//   dx = r·(h − n̂·mean(h·n̂))
//
// Angles: φ / 2π = position · (f_i / 2π) is formed and reduced to [−1/2, 1/2] in 64 bits (a position of
// thousands times a 32-bit frequency would lose the low bits of the angle), then one 32-bit sincospi. No
// tables: any position, whole or fractional, costs the same, and a token's D/2 angles are shared by all its
// heads, so the 64 fp64 products and sincos per row hide behind the row's loads (3 KB in and out at
// 12 heads of 128).
//
// HBM-bound: 2 x 32760 tokens, q and k of 12 heads of 128, bf16, normed over the row: forward 181 us for 805 MB
// (4.4 TB/s), backward 291 for 1208 MB (4.2 TB/s); one frame of 1560 tokens 10 us for 19 MB: a row per wave, whose loads,
// sum, angles and stores wait for each other, of which a launch is 3 to 4.
//
// A unit is 8 pairs (16 values: two 16-byte loads of bf16): chunks 2j and 2j + 1 of a head, or chunks j and
// j + D/16 where halves are paired. WPR waves hold a row's units, NU per lane; a wave writes
// its row's angles to its own LDS corner and reads them back per unit (no barrier). A workgroup takes
// `chunk` consecutive tokens of one tensor (blockIdx.y: q or k); the weight gradient stays in registers
// over them and leaves as one partial row per workgroup, added in a fixed order.
#include "mlora_common.h"
#include "mlora_host.h"
#include "mlora_rows.h"

#include <cmath>

namespace mlora {

constexpr int kRotMaxWidth = 8192, kRotMaxHeadDim = 256, kRotMaxPairs = kRotMaxHeadDim / 2;
constexpr int kRotWaves = 4, kRotMaxTensors = 2;
enum { kRotNormNone = 0, kRotNormHead = 1, kRotNormRow = 2 };
enum { kPosI32 = 0, kPosI64 = 1, kPosF32 = 2 };

struct RotTensor {
  const void *x, *g, *w;
  void *y;         // the output, or dx: contiguous
  float *partial;  // backward with a weight: [workgroups, width or D]
  int64_t x_sb, x_st, x_sh, g_sb, g_st, g_sh;
  int32_t heads;
};

struct RotArgs {
  RotTensor t[kRotMaxTensors];
  const void *pos;
  int64_t pos_sb, pos_st;  // 0 batch stride: shared
  int32_t tokens, rows, head_dim, chunk;
  int32_t pos_type, norm, halves, w_f32;
  float eps;
  double turns[kRotMaxPairs];  // f_i / 2π
  uint8_t axis[kRotMaxPairs];
};

// A position as it lies in memory, and its value.
__device__ __forceinline__ uint64_t load_pos(const RotArgs &a, int64_t o) {
  if (a.pos_type == kPosI64) return static_cast<const uint64_t *>(a.pos)[o];
  return static_cast<const uint32_t *>(a.pos)[o];
}
__device__ __forceinline__ double pos_value(const RotArgs &a, uint64_t p) {
  if (a.pos_type == kPosI64) return (double)(int64_t)p;
  return a.pos_type == kPosI32 ? (double)(int32_t)p : (double)__uint_as_float((uint32_t)p);
}

// A unit's two chunks as they lie in memory, to be asked for a row ahead.
template <bool F32>
struct RawUnit {
  u32x4 r[2][F32 ? 2 : 1];
  __device__ __forceinline__ void load(const void *p, int64_t e0, int64_t e1, bool on) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int64_t e = h ? e1 : e0;
      if constexpr (F32) {
        const float *q = static_cast<const float *>(p) + e;
        r[h][0] = on ? *(const MLORA_GLOBAL u32x4 *)q : u32x4{0, 0, 0, 0};
        r[h][1] = on ? *(const MLORA_GLOBAL u32x4 *)(q + 4) : u32x4{0, 0, 0, 0};
      } else {
        r[h][0] = on ? *(const MLORA_GLOBAL u32x4 *)(static_cast<const uint16_t *>(p) + e) : u32x4{0, 0, 0, 0};
      }
    }
  }
  __device__ __forceinline__ void unpack(float (&v)[16]) const {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      if constexpr (F32) v[i] = __uint_as_float(r[i / 8][i % 8 / 4][i % 4]);
      else v[i] = __uint_as_float(i % 2 ? r[i / 8][0][i % 8 / 2] & 0xffff0000u : r[i / 8][0][i % 8 / 2] << 16);
    }
  }
};

// BWD: g is turned back and, with a norm, taken through it; else x is normed and turned.
template <int NU, int WPR, bool F32, bool HALVES, bool NORM, bool BWD>
__global__ __launch_bounds__(64 * kRotWaves) void rotary_kernel(const RotArgs a) {
  constexpr int STREAMS = kRotWaves / WPR, UNITS = NU * WPR * 64;
  __shared__ float2 angles[kRotWaves][kRotMaxPairs];  // (cos, sin) of the wave's row
  __shared__ float red[4][kRotWaves];
  __shared__ float unit_part[2][NORM ? STREAMS * UNITS : 1];
  __shared__ float sums[NORM && BWD ? UNITS * 16 : 1];
  const RotTensor &x = a.t[blockIdx.y];
  const int wave = wave_id(), lane = threadIdx.x & 63, sub = wave % WPR, stream = wave / WPR;
  const int D = a.head_dim, pairs = D / 2, uph = D / 16;  // units per head
  const int units = x.heads * uph, width = x.heads * D;
  const int r0 = blockIdx.x * a.chunk, r1 = min(r0 + a.chunk, a.rows);
  const float inv = 1.0f / (float)(a.norm == kRotNormHead ? D : width);
  double turn[2];  // of pairs lane and lane + 64
  int ax[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int p = min(lane + 64 * i, pairs - 1);
    turn[i] = a.turns[p], ax[i] = a.axis[p];
  }
  int head[NU], j8[NU], e0[NU], e1[NU];  // a unit's head, its first pair, its two chunks' elements in the head
  float w[NORM ? NU : 1][16], acc[NORM && BWD ? NU : 1][16];
#pragma unroll
  for (int k = 0; k < NU; ++k) {
    const int u = lane + 64 * (k * WPR + sub), j = u % uph;
    head[k] = u / uph, j8[k] = 8 * j;
    e0[k] = HALVES ? 8 * j : 16 * j, e1[k] = HALVES ? 8 * (j + uph) : 16 * j + 8;
    if constexpr (NORM) {
      float lo[8] = {}, hi[8] = {};
      if (u < units) {
        const int64_t o = a.norm == kRotNormHead ? 0 : (int64_t)head[k] * D;
        load8(x.w, a.w_f32, o + e0[k], lo), load8(x.w, a.w_f32, o + e1[k], hi);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) w[k][i] = lo[i], w[k][i + 8] = hi[i];
      if constexpr (BWD) {
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[k][i] = 0.f;
      }
    }
  }
  int slot = 0;  // an LDS slot of `over` is written again only after a barrier that follows its reads
  // v[k] <- the sum of v over the row, or over unit k's head, in a fixed order
  auto over = [&](float (&v)[NU]) __attribute__((always_inline)) {
    if (a.norm == kRotNormRow) {
      float s = 0.f;
#pragma unroll
      for (int k = 0; k < NU; ++k) s += v[k];
      s = lanes_sum<64>(s);
      if constexpr (WPR > 1) {
        if (lane == 0) red[slot][wave] = s;
        __syncthreads();
        s = red[slot][stream * WPR];
#pragma unroll
        for (int q = 1; q < WPR; ++q) s += red[slot][stream * WPR + q];
        slot ^= 1;
      }
#pragma unroll
      for (int k = 0; k < NU; ++k) v[k] = s;
    } else if (64 % uph == 0) {  // a head's units are neighbouring lanes
#pragma unroll
      for (int k = 0; k < NU; ++k) {
        if (uph >= 2) v[k] = lanes_add<1>(v[k]);
        if (uph >= 4) v[k] = lanes_add<2>(v[k]);
        if (uph >= 8) v[k] = lanes_add<4>(v[k]);
        if (uph >= 16) v[k] = lanes_add<8>(v[k]);
      }
    } else {  // heads run across lanes, units and waves
      float *part = unit_part[slot] + stream * UNITS;
#pragma unroll
      for (int k = 0; k < NU; ++k) part[lane + 64 * (k * WPR + sub)] = v[k];
      __syncthreads();
#pragma unroll
      for (int k = 0; k < NU; ++k) {
        if (lane + 64 * (k * WPR + sub) >= units) continue;
        float s = 0.f;
        for (int i = 0; i < uph; ++i) s += part[head[k] * uph + i];
        v[k] = s;
      }
      slot ^= 1;
    }
  };
  // the next row's loads under this row's work (float32 rows are twice the registers: their waves do more)
  constexpr bool kAhead = !F32;
  RawUnit<F32> rv[!BWD || NORM ? NU : 1], rg[BWD ? NU : 1];
  uint64_t pos[2];
  auto load = [&](int r) __attribute__((always_inline)) {
    const bool live = r < r1;
    const int rc = min(r, a.rows - 1);
    const int64_t b = rc / a.tokens, t = rc % a.tokens;
#pragma unroll
    for (int i = 0; i < 2; ++i) pos[i] = load_pos(a, b * a.pos_sb + t * a.pos_st + ax[i]);
#pragma unroll
    for (int k = 0; k < NU; ++k) {
      const bool on = live && lane + 64 * (k * WPR + sub) < units;
      if constexpr (!BWD || NORM) {
        const int64_t e = b * x.x_sb + t * x.x_st + head[k] * x.x_sh;
        rv[k].load(x.x, e + e0[k], e + e1[k], on);
      }
      if constexpr (BWD) {
        const int64_t e = b * x.g_sb + t * x.g_st + head[k] * x.g_sh;
        rg[k].load(x.g, e + e0[k], e + e1[k], on);
      }
    }
  };
  if constexpr (kAhead) load(r0 + stream);
  // every stream runs the same number of rows, so that every wave meets the same barriers
  for (int r = r0 + stream; r - stream < r1; r += STREAMS) {
    const bool live = r < r1;
    if constexpr (!kAhead) load(r);
    float v[NU][16], g[BWD ? NU : 1][16];
#pragma unroll
    for (int k = 0; k < NU; ++k) {
      if constexpr (!BWD || NORM) rv[k].unpack(v[k]);
      if constexpr (BWD) rg[k].unpack(g[k]);
    }
    double phi[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) phi[i] = pos_value(a, pos[i]) * turn[i];
    if constexpr (kAhead) load(r + STREAMS);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (lane + 64 * i >= pairs) break;
      float s, c;
      sincospif(2.0f * (float)(phi[i] - __builtin_rint(phi[i])), &s, &c);
      angles[wave][lane + 64 * i] = float2{c, BWD ? -s : s};
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    auto turned = [&](float (&o)[16], int k) __attribute__((always_inline)) {
#pragma unroll
      for (int p = 0; p < 8; ++p) {
        const float2 cs = angles[wave][j8[k] + p];
        float &a0 = o[HALVES ? p : 2 * p], &b0 = o[HALVES ? p + 8 : 2 * p + 1];
        const float va = a0, vb = b0;
        a0 = va * cs.x - vb * cs.y, b0 = va * cs.y + vb * cs.x;
      }
    };
    float rstd[NU];
    if constexpr (NORM) {
#pragma unroll
      for (int k = 0; k < NU; ++k) {
        rstd[k] = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) rstd[k] += v[k][i] * v[k][i];
      }
      over(rstd);
#pragma unroll
      for (int k = 0; k < NU; ++k) {
        rstd[k] = 1.0f / __fsqrt_rn(rstd[k] * inv + a.eps);
#pragma unroll
        for (int i = 0; i < 16; ++i) v[k][i] *= rstd[k];
      }
    }
    if constexpr (!BWD) {
#pragma unroll
      for (int k = 0; k < NU; ++k) {
        if constexpr (NORM) {
#pragma unroll
          for (int i = 0; i < 16; ++i) v[k][i] *= w[k][i];
        }
        turned(v[k], k);
      }
    } else {
#pragma unroll
      for (int k = 0; k < NU; ++k) turned(g[k], k);
      if constexpr (NORM) {
        float m[NU];
#pragma unroll
        for (int k = 0; k < NU; ++k) {
          m[k] = 0.f;
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            acc[k][i] += g[k][i] * v[k][i];
            g[k][i] *= w[k][i];
            m[k] += g[k][i] * v[k][i];
          }
        }
        over(m);
#pragma unroll
        for (int k = 0; k < NU; ++k)
#pragma unroll
          for (int i = 0; i < 16; ++i) g[k][i] = rstd[k] * (g[k][i] - v[k][i] * (m[k] * inv));
      }
    }
#pragma unroll
    for (int k = 0; k < NU; ++k) {
      if (!live || lane + 64 * (k * WPR + sub) >= units || x.y == nullptr) continue;
      const int64_t e = ((int64_t)r * x.heads + head[k]) * D;
      const float(&o)[16] = BWD ? g[BWD ? k : 0] : v[k];
      float lo[8], hi[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) lo[i] = o[i], hi[i] = o[i + 8];
      store8_any(x.y, F32, e + e0[k], lo), store8_any(x.y, F32, e + e1[k], hi);
    }
  }
  if constexpr (NORM && BWD) {
    if (x.partial == nullptr) return;
    // the streams' sums in stream order, then one partial row (summed over the heads for a per-head weight)
#pragma unroll
    for (int q = 0; q < STREAMS; ++q) {
      if (stream == q) {
#pragma unroll
        for (int k = 0; k < NU; ++k) {
          if (lane + 64 * (k * WPR + sub) >= units) continue;
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            float &dst = sums[head[k] * D + (i < 8 ? e0[k] + i : e1[k] + i - 8)];
            dst = q > 0 ? dst + acc[k][i] : acc[k][i];
          }
        }
      }
      __syncthreads();
    }
    const int n = a.norm == kRotNormHead ? D : width, heads = a.norm == kRotNormHead ? x.heads : 1;
    for (int e = threadIdx.x; e < n; e += 64 * kRotWaves) {
      float s = 0.f;
      for (int h = 0; h < heads; ++h) s += sums[h * D + e];
      x.partial[(int64_t)blockIdx.x * n + e] = s;
    }
  }
}

struct RotTile {
  int nu, wpr;
};
static RotTile rot_tile(int64_t width) {
  const int n = (int)((width / 16 + 63) / 64);  // units per lane of one wave
  if (n <= 2) return {n, 1};
  return {2, n <= 4 ? 2 : 4};
}

// Tokens per workgroup (a multiple of the rows in flight): what leaves about `most` workgroups, of all tensors.
// 2 x 32760 tokens, q and k of 12 x 128, bf16: forward 199 us at 1024, 183 at 2048, 181 at 4096, 180 at 8192, 253 at
// 32768; backward, whose workgroups leave partial sums of the weights, 377 at 256 (half the chip's places), 291 at
// 512, 366 at 768, 297 at 1024.
static int64_t rot_chunk(int64_t rows, int64_t width, int64_t most) {
  const int64_t streams = kRotWaves / rot_tile(width).wpr, n = (rows + most - 1) / most;
  return (n + streams - 1) / streams * streams;
}
constexpr int64_t kRotMostFwd = 4096, kRotMostBwd = 512;

static int64_t max_width(const int32_t *heads, int n, int64_t D) {
  int64_t w = 0;
  for (int i = 0; i < n; ++i) w = heads[i] * D > w ? heads[i] * D : w;
  return w;
}

template <bool NORM, bool BWD>
static int launch_rotary(const RotArgs &a, int n, int64_t width, bool f32, hipStream_t s) {
  const RotTile tile = rot_tile(width);
  const dim3 grid((unsigned)((a.rows + a.chunk - 1) / a.chunk), (unsigned)n), block(64 * kRotWaves);
  auto go = [&](auto nu, auto wpr) {
    constexpr int NU = decltype(nu)::value, WPR = decltype(wpr)::value;
    if (f32 && a.halves) hipLaunchKernelGGL((rotary_kernel<NU, WPR, true, true, NORM, BWD>), grid, block, 0, s, a);
    else if (f32) hipLaunchKernelGGL((rotary_kernel<NU, WPR, true, false, NORM, BWD>), grid, block, 0, s, a);
    else if (a.halves) hipLaunchKernelGGL((rotary_kernel<NU, WPR, false, true, NORM, BWD>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((rotary_kernel<NU, WPR, false, false, NORM, BWD>), grid, block, 0, s, a);
  };
  using std::integral_constant;
  if (tile.nu == 1) go(integral_constant<int, 1>{}, integral_constant<int, 1>{});
  else if (tile.wpr == 1) go(integral_constant<int, 2>{}, integral_constant<int, 1>{});
  else if (tile.wpr == 2) go(integral_constant<int, 2>{}, integral_constant<int, 2>{});
  else go(integral_constant<int, 2>{}, integral_constant<int, 4>{});
  return launch_status();
}

// Checks shared by both directions; fills the tensors' inputs and the angles.
static int rotary_args(RotArgs &a, const void *const *xs, const void *const *ws, const int64_t *x_strides,
                       const int32_t *heads, int n, int dtype, int w_dtype, int norm, float eps, const void *pos,
                       int pos_type, int64_t pos_sb, int64_t pos_st, const double *turns, const int32_t *axis,
                       int64_t n_axes, int halves, int64_t batches, int64_t tokens, int64_t head_dim) {
  if (n < 1 || n > kRotMaxTensors || xs == nullptr || x_strides == nullptr || heads == nullptr || turns == nullptr ||
      axis == nullptr)
    return MLORA_ERR_INVALID;
  if (batches < 0 || tokens < 0 || n_axes < 1) return MLORA_ERR_INVALID;
  if ((dtype != MLORA_BF16 && dtype != MLORA_F32) || (w_dtype != MLORA_BF16 && w_dtype != MLORA_F32))
    return MLORA_ERR_UNSUPPORTED;
  if (norm < kRotNormNone || norm > kRotNormRow || pos_type < kPosI32 || pos_type > kPosF32) return MLORA_ERR_INVALID;
  if (norm != kRotNormNone && !(eps > 0.f && eps < INFINITY)) return MLORA_ERR_INVALID;
  if (head_dim < 16 || head_dim % 16 != 0 || head_dim > kRotMaxHeadDim) return MLORA_ERR_UNSUPPORTED;
  if (batches > 0 && tokens > (INT32_MAX - 65536) / batches) return MLORA_ERR_LIMIT;
  a = RotArgs{};
  for (int i = 0; i < n; ++i) {
    if (heads[i] < 1) return MLORA_ERR_INVALID;
    if (heads[i] > kRotMaxWidth / head_dim) return MLORA_ERR_LIMIT;
    RotTensor &t = a.t[i];
    t.x = xs[i], t.w = norm != kRotNormNone && ws != nullptr ? ws[i] : nullptr;
    t.x_sb = x_strides[3 * i], t.x_st = x_strides[3 * i + 1], t.x_sh = x_strides[3 * i + 2], t.heads = heads[i];
    if (batches * tokens == 0) continue;
    if (t.x == nullptr || (norm != kRotNormNone && t.w == nullptr)) return MLORA_ERR_INVALID;
    if (!rows_aligned(t.x, t.x_sb, t.x_st) || t.x_sh < 0 || t.x_sh % 8 != 0 || !aligned16(t.w)) return MLORA_ERR_UNSUPPORTED;
  }
  for (int p = 0; p < head_dim / 2; ++p) {
    if (axis[p] < 0 || axis[p] >= n_axes || axis[p] > 255 || !(turns[p] > -INFINITY && turns[p] < INFINITY))
      return MLORA_ERR_INVALID;
    a.turns[p] = turns[p], a.axis[p] = (uint8_t)axis[p];
  }
  if (batches * tokens > 0 && (pos == nullptr || pos_sb < 0 || pos_st < 0)) return MLORA_ERR_INVALID;
  a.pos = pos, a.pos_sb = pos_sb, a.pos_st = pos_st, a.pos_type = pos_type;
  a.tokens = (int32_t)tokens, a.rows = (int32_t)(batches * tokens), a.head_dim = (int32_t)head_dim;
  a.norm = norm, a.halves = halves != 0, a.w_f32 = w_dtype == MLORA_F32, a.eps = eps;
  return MLORA_OK;
}

}  // namespace mlora

using namespace mlora;

extern "C" int mlora_rotary_turns(const int32_t *axis_dims, int32_t n_axes, double theta, double *turns, int32_t *axis) {
  if (axis_dims == nullptr || turns == nullptr || axis == nullptr || n_axes < 1 || n_axes > 255) return MLORA_ERR_INVALID;
  if (!(theta > 0.0 && theta < INFINITY)) return MLORA_ERR_INVALID;
  int64_t total = 0;
  for (int c = 0; c < n_axes; ++c) {
    if (axis_dims[c] < 0 || axis_dims[c] % 2 != 0) return MLORA_ERR_INVALID;
    total += axis_dims[c];
  }
  if (total > kRotMaxHeadDim) return MLORA_ERR_LIMIT;
  int p = 0;
  for (int c = 0; c < n_axes; ++c)
    for (int i = 0; i < axis_dims[c] / 2; ++i, ++p) {
      turns[p] = std::pow(theta, -2.0 * i / axis_dims[c]) / (2.0 * M_PI);
      axis[p] = c;
    }
  return MLORA_OK;
}

extern "C" int mlora_rotary_axes(const void *const *xs, void *const *ys, const void *const *ws, const int64_t *x_strides,
                                 const int32_t *heads, int n, int dtype, int w_dtype, int norm, float eps,
                                 const void *pos, int pos_type, int64_t pos_sb, int64_t pos_st, const double *turns,
                                 const int32_t *axis, int64_t n_axes, int halves, int64_t batches, int64_t tokens,
                                 int64_t head_dim, void *stream) {
  RotArgs a;
  int st = rotary_args(a, xs, ws, x_strides, heads, n, dtype, w_dtype, norm, eps, pos, pos_type, pos_sb, pos_st, turns,
                       axis, n_axes, halves, batches, tokens, head_dim);
  if (st || a.rows == 0) return st;
  if (ys == nullptr) return MLORA_ERR_INVALID;
  for (int i = 0; i < n; ++i) {
    if (ys[i] == nullptr) return MLORA_ERR_INVALID;
    if (!aligned16(ys[i])) return MLORA_ERR_UNSUPPORTED;
    a.t[i].y = ys[i];
  }
  const int64_t width = max_width(heads, n, head_dim);
  a.chunk = (int32_t)rot_chunk(a.rows, width, kRotMostFwd / n);
  hipStream_t s = static_cast<hipStream_t>(stream);
  return norm == kRotNormNone ? launch_rotary<false, false>(a, n, width, dtype == MLORA_F32, s)
                              : launch_rotary<true, false>(a, n, width, dtype == MLORA_F32, s);
}

extern "C" int64_t mlora_rotary_axes_backward_workspace_bytes(const int32_t *heads, int n, int norm, int64_t batches,
                                                              int64_t tokens, int64_t head_dim) {
  if (heads == nullptr || n < 1 || n > kRotMaxTensors || batches < 0 || tokens < 0 || head_dim < 1) return MLORA_ERR_INVALID;
  if (batches > 0 && tokens > (INT32_MAX - 65536) / batches) return MLORA_ERR_LIMIT;
  const int64_t rows = batches * tokens;
  if (norm == kRotNormNone || rows == 0) return 0;
  int64_t values = 0;
  for (int i = 0; i < n; ++i) {
    if (heads[i] < 1) return MLORA_ERR_INVALID;
    if (heads[i] > kRotMaxWidth / head_dim) return MLORA_ERR_LIMIT;
    values += norm == kRotNormHead ? head_dim : heads[i] * head_dim;
  }
  const int64_t chunk = rot_chunk(rows, max_width(heads, n, head_dim), kRotMostBwd / n);
  return (rows + chunk - 1) / chunk * values * (int64_t)sizeof(float);
}

extern "C" int mlora_rotary_axes_backward(const void *const *xs, const void *const *gs, void *const *dxs,
                                          const void *const *ws, void *const *dws, const int64_t *x_strides,
                                          const int64_t *g_strides, const int32_t *heads, int n, int dtype, int w_dtype,
                                          int norm, float eps, const void *pos, int pos_type, int64_t pos_sb,
                                          int64_t pos_st, const double *turns, const int32_t *axis, int64_t n_axes,
                                          int halves, void *workspace, int64_t workspace_bytes, int64_t batches,
                                          int64_t tokens, int64_t head_dim, void *stream) {
  RotArgs a;
  // without a norm the input is not read: its place is taken by the gradient's
  int st = rotary_args(a, norm == kRotNormNone ? gs : xs, ws, norm == kRotNormNone ? g_strides : x_strides, heads, n,
                       dtype, w_dtype, norm, eps, pos, pos_type, pos_sb, pos_st, turns, axis, n_axes, halves, batches,
                       tokens, head_dim);
  if (st) return st;
  if (gs == nullptr || g_strides == nullptr || dxs == nullptr) return MLORA_ERR_INVALID;
  bool sums = false;
  for (int i = 0; i < n; ++i) {
    RotTensor &t = a.t[i];
    if (dws != nullptr && dws[i] != nullptr) {
      if (norm == kRotNormNone) return MLORA_ERR_INVALID;
      if (!aligned16(dws[i])) return MLORA_ERR_UNSUPPORTED;
      sums = true;
    }
    t.g = gs[i], t.g_sb = g_strides[3 * i], t.g_st = g_strides[3 * i + 1], t.g_sh = g_strides[3 * i + 2], t.y = dxs[i];
    if (a.rows == 0) continue;
    if (t.g == nullptr) return MLORA_ERR_INVALID;
    if (!rows_aligned(t.g, t.g_sb, t.g_st) || t.g_sh < 0 || t.g_sh % 8 != 0 || !aligned16(t.y)) return MLORA_ERR_UNSUPPORTED;
  }
  const int64_t width = max_width(heads, n, head_dim);
  hipStream_t s = static_cast<hipStream_t>(stream);
  int64_t blocks = 0;
  float *p = static_cast<float *>(workspace);
  ColSums cs;
  if (a.rows > 0) {
    a.chunk = (int32_t)rot_chunk(a.rows, width, kRotMostBwd / n);
    blocks = (a.rows + a.chunk - 1) / a.chunk;
    if (sums) {
      const int64_t need = mlora_rotary_axes_backward_workspace_bytes(heads, n, norm, batches, tokens, head_dim);
      if (p == nullptr || workspace_bytes < need) return MLORA_ERR_WORKSPACE;
      if (!aligned16(p)) return MLORA_ERR_UNSUPPORTED;
    }
  }
  for (int i = 0; i < n && sums; ++i) {
    const int64_t wn = norm == kRotNormHead ? head_dim : heads[i] * head_dim;
    if (dws[i] == nullptr) continue;
    a.t[i].partial = p;
    cs.add({p, dws[i], 0, wn, (int32_t)blocks, 1, (int32_t)wn, w_dtype == MLORA_F32});
    if (a.rows > 0) p += blocks * wn;
  }
  if (a.rows > 0) {
    st = norm == kRotNormNone ? launch_rotary<false, true>(a, n, width, dtype == MLORA_F32, s)
                              : launch_rotary<true, true>(a, n, width, dtype == MLORA_F32, s);
    if (st) return st;
  }
  return sums ? launch_col_sums(cs, s) : MLORA_OK;
}
