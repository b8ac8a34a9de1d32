// Attention of q to an encoder's keys and values of another length, forward:
//
//   s_j = scale · q·k_j over the sample's live keys (its first key_lengths[b], those with key_mask set);
//   out = Σ_j p_j v_j with p = softmax(s);  a query without a live key gets zeros.
//
// One pass over the keys with a running maximum m and sum l per query (base 2: s' = s·scale·log2 e):
//   P = 2^(s' − m),  l = Σ P,  O = Σ P·V;  out = O / l,  lse = m + log2 l (what the backward needs; +inf
// for a query without keys, so that every 2^(s' − lse) is 0). The running maximum is raised only when a tile's
// exceeds it by more than 2^8 (P then stays below 2^8, far from any limit, and rounding is relative), so the
// rescaling of O is a rare branch. bf16: P is rounded to bf16 for the product with V, and l sums the rounded
// values, so that the weights that multiply V add up to one. Everything else is float32.
//
// Rows: the G = heads / kv_heads query heads that share a key head are packed, row r = g·Lq + i, so that shared
// keys are read once for all of them.
#include "mlora_attention.h"

namespace mlora {

struct AttnArgs {
  const void *q, *k, *v;
  void *out;          // [B, Lq, H, D] contiguous
  float *lse;         // [B, H, Lq]
  const int32_t *lengths;
  const uint8_t *mask;
  float *part_o, *part_ml;  // splits: [splits][B·Hk·rows][D] sums and [splits][B·Hk·rows][2] (m, l)
  int64_t q_sb, q_sl, q_sh, k_sb, k_sl, k_sh, v_sb, v_sl, v_sh, mask_sb;
  int32_t batches, Lq, Lk, H, Hk, G, D, rows, row_tiles, splits, split_tiles;
  float c;            // scale · log2 e
};

// A sample's live keys, 64 (or KT) at a time.
template <int KT>
struct KeyMask {
  const uint8_t *mask;  // null: no mask
  int len;
  __device__ __forceinline__ int byte(int tile, int lane) const {  // of key tile·KT + lane
    const int key = tile * KT + lane;
    return mask != nullptr && lane < KT && key < len ? mask[key] : 1;
  }
  __device__ __forceinline__ uint64_t bits(int tile, int lane_byte) const {
    uint64_t b = low_bits(min(len - tile * KT, KT));
    if (mask != nullptr) b &= __ballot(lane_byte != 0);
    return b;
  }
};

__device__ __forceinline__ int sample_keys(const AttnArgs &a, int b) {
  return a.lengths == nullptr ? a.Lk : min(max(a.lengths[b], 0), a.Lk);
}

__device__ __forceinline__ void load_frag(const uint16_t *p, bool on, Frag<uint16_t> &f) {
  f.v = on ? *(const MLORA_GLOBAL u32x4 *)p : u32x4{0, 0, 0, 0};
}
__device__ __forceinline__ void load_frag(const float *p, bool on, Frag<float> &f) {
  const f32x4 z = {0.f, 0.f, 0.f, 0.f};
  const f32x4 a = on ? *(const MLORA_GLOBAL f32x4 *)p : z, b = on ? *(const MLORA_GLOBAL f32x4 *)(p + 4) : z;
#pragma unroll
  for (int j = 0; j < 4; ++j) f.v[j] = a[j], f.v[j + 4] = b[j];
}

// The running softmax of NQ x 32 queries (a column per lane and half) against KT keys per step.
template <class T, int DP, int NQ, int KT>
struct Softmax {
  f32x16 o[NQ][DP / 32];
  Frag<T> q[NQ][DP / 16];
  float m[NQ], l[NQ];

  __device__ __forceinline__ void init() {
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      m[n] = -INFINITY, l[n] = 0.f;
#pragma unroll
      for (int d = 0; d < DP / 32; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[n][d][i] = 0.f;
    }
  }

  // One tile of keys in LDS with at least one live bit.
  __device__ __forceinline__ void step(const FragReader<T, DP> &fr, const MLORA_LDS char *kt, const MLORA_LDS char *vt,
                                       uint64_t bits, float c, int lane) {
    constexpr int NB = KT / 32;
    f32x16 s[NQ][NB];
#pragma unroll
    for (int kb = 0; kb < NB; ++kb) {
#pragma unroll
      for (int n = 0; n < NQ; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[n][kb][i] = 0.f;
#pragma unroll
      for (int ks = 0; ks < DP / 16; ++ks) {
        Frag<T> kf;
        fr.rows(kt, 32 * kb, ks, kf);
#pragma unroll
        for (int n = 0; n < NQ; ++n) s[n][kb] = mma16(kf, q[n][ks], s[n][kb]);
      }
    }
    if (bits != low_bits(KT)) {
      const uint64_t mine = bits >> (4 * (lane >> 5));
#pragma unroll
      for (int kb = 0; kb < NB; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const bool on = (mine >> (32 * kb + 8 * (i / 4) + i % 4)) & 1;
#pragma unroll
          for (int n = 0; n < NQ; ++n) s[n][kb][i] = on ? s[n][kb][i] : -INFINITY;
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
      mx = half_max(mx) * c;
      if (__any(mx > m[n] + 8.f)) {
        const float to = fmaxf(m[n], mx), f = __builtin_amdgcn_exp2f(m[n] - to);
        m[n] = to;
        l[n] *= f;
#pragma unroll
        for (int d = 0; d < DP / 32; ++d)
#pragma unroll
          for (int i = 0; i < 16; ++i) o[n][d][i] *= f;
      }
#pragma unroll
      for (int kb = 0; kb < NB; ++kb) {
#pragma unroll
        for (int i = 0; i < 16; ++i) s[n][kb][i] = __builtin_amdgcn_exp2f(s[n][kb][i] * c - m[n]);
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) to_frag(s[n][kb], ks, p[n][2 * kb + ks]);
      }
      l[n] += frag_sum(p[n]);
    }
#pragma unroll
    for (int ks = 0; ks < KT / 16; ++ks)
#pragma unroll
      for (int d = 0; d < DP / 32; ++d) {
        Frag<T> vf;
        fr.cols(vt, 16 * ks, d, vf);
#pragma unroll
        for (int n = 0; n < NQ; ++n) o[n][d] = mma16(vf, p[n][ks], o[n][d]);
      }
  }

  // The sum of the weights as the product with V sees them.
  static __device__ __forceinline__ float frag_sum(const Frag<T> (&p)[KT / 16]) {
    float t = 0.f;
#pragma unroll
    for (int ks = 0; ks < KT / 16; ++ks) {
      if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          t += __uint_as_float(p[ks].v[j] << 16);
          t += __uint_as_float(p[ks].v[j] & 0xffff0000u);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) t += p[ks].v[j];
      }
    }
    return t;
  }
};

// Rows of an attention call: address of row r of (b, kv head), in elements.
__device__ __forceinline__ int64_t row_at(int r, int Lq, int64_t sl, int64_t sh) {
  const int g = r / Lq, i = r - g * Lq;
  return g * sh + i * sl;
}

// Writes NQ x 32 rows of the O^T registers (times f[n]) to out, 8 or 16 bytes per lane and store.
template <class T, int DP, int NQ>
__device__ __forceinline__ void store_rows(T *base, const f32x16 (&o)[NQ][DP / 32], const float (&f)[NQ], int row0, int rows,
                                           int Lq, int64_t sl, int64_t sh, int D, int lane) {
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int r = row0 + 32 * n + (lane & 31);
    if (r >= rows) continue;
    T *p = base + row_at(r, Lq, sl, sh) + 4 * (lane >> 5);
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int at = 32 * d + 8 * i;
        if (at >= D) continue;  // the head dimension is a multiple of 8
        const float x0 = o[n][d][4 * i] * f[n], x1 = o[n][d][4 * i + 1] * f[n], x2 = o[n][d][4 * i + 2] * f[n],
                    x3 = o[n][d][4 * i + 3] * f[n];
        if constexpr (sizeof(T) == 2) *(MLORA_GLOBAL u32x2 *)(p + at) = u32x2{pack2_bf16(x0, x1), pack2_bf16(x2, x3)};
        else *(MLORA_GLOBAL f32x4 *)(p + at) = f32x4{x0, x1, x2, x3};
      }
  }
}

template <class T>
struct AttnTile {
  static constexpr int KT = sizeof(T) == 2 ? 64 : 32;  // keys per tile: 16 KB of K and of V at 128 channels
};

// Four waves of NQ x 32 rows each against the same key tiles, two buffers of K and V in LDS: tile t + 1 loads
// while tile t is multiplied; one barrier per tile.
template <class T, int DP, int NQ>
__global__ __launch_bounds__(256, NQ == 1 ? 2 : 1) void attn_fwd_kernel(const AttnArgs a) {
  constexpr int KT = AttnTile<T>::KT;
  using Tile = HeadTile<T, DP>;
  constexpr int TB = KT * Tile::RB, N = TB / 1024 / 4;
  __shared__ u32x4 smem[4 * TB / 16];  // K, V of buffer 0, K, V of buffer 1
  MLORA_LDS char *lds = (MLORA_LDS char *)smem;
  const int wave = wave_id(), lane = threadIdx.x & 63;
  int id = xcd_contiguous(blockIdx.x, gridDim.x);  // one key head's row tiles stay on one XCD's L2
  const int rt = id % a.row_tiles;
  id /= a.row_tiles;
  const int sp = id % a.splits;
  id /= a.splits;
  const int hk = id % a.Hk, b = id / a.Hk;
  const KeyMask<KT> km{a.mask == nullptr ? nullptr : a.mask + b * a.mask_sb, sample_keys(a, b)};
  const int t0 = sp * a.split_tiles, t1 = min(t0 + a.split_tiles, (km.len + KT - 1) / KT);
  const T *kp = static_cast<const T *>(a.k) + b * a.k_sb + hk * a.k_sh;
  const T *vp = static_cast<const T *>(a.v) + b * a.v_sb + hk * a.v_sh;
  TileLoader<T, DP, N> kl, vl;
  kl.init(lane, wave, 4, a.k_sl, a.D), vl.init(lane, wave, 4, a.v_sl, a.D);
  auto stage = [&](int t, int buf, uint64_t bits) __attribute__((always_inline)) {
    kl.load(kp + (int64_t)t * KT * a.k_sl, bits, lds + buf * 2 * TB);
    vl.load(vp + (int64_t)t * KT * a.v_sl, bits, lds + buf * 2 * TB + TB);
  };
  uint64_t bits = 0, next = 0;
  if (t0 < t1) {
    bits = km.bits(t0, km.byte(t0, lane));
    stage(t0, 0, bits);
    next = km.bits(t0 + 1, km.byte(t0 + 1, lane));
  }
  FragReader<T, DP> fr;
  fr.init(lane);
  Softmax<T, DP, NQ, KT> sm;
  sm.init();
  const int row0 = (rt * 4 + wave) * 32 * NQ;
  const T *qp = static_cast<const T *>(a.q) + b * a.q_sb + (int64_t)hk * a.G * a.q_sh;
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const T *p = qp + row_at(min(row0 + 32 * n + (lane & 31), a.rows - 1), a.Lq, a.q_sl, a.q_sh);
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) {
      const int d = 16 * s + 8 * (lane >> 5);
      load_frag(p + d, d < a.D, sm.q[n][s]);
    }
  }
  auto turn = [&](auto buf, int t) __attribute__((always_inline)) {
    constexpr int B = decltype(buf)::value;
    wait_vmcnt<0>();
    lds_pipeline_barrier();  // tile t is in LDS, and every wave has read tile t - 1
    int byte = 1;
    if (t + 1 < t1) {
      stage(t + 1, B ^ 1, next);
      byte = km.byte(t + 2, lane);
    }
    if (bits != 0) sm.step(fr, lds + B * 2 * TB, lds + B * 2 * TB + TB, bits, a.c, lane);
    bits = next;
    next = km.bits(t + 2, byte);
  };
  for (int t = t0; t < t1; t += 2) {
    turn(std::integral_constant<int, 0>{}, t);
    if (t + 1 < t1) turn(std::integral_constant<int, 1>{}, t + 1);
  }
  const int64_t head_rows = ((int64_t)b * a.Hk + hk) * a.rows;
  if (a.splits > 1) {
    const int64_t all = (int64_t)a.batches * a.Hk * a.rows, first = sp * all + head_rows;
    float one[NQ];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      one[n] = 1.f;
      const float l = half_sum(sm.l[n]);
      const int r = row0 + 32 * n + lane;
      if (lane < 32 && r < a.rows) *(float2 *)(a.part_ml + 2 * (first + r)) = float2{sm.m[n], l};
    }
    store_rows<float, DP, NQ>(a.part_o + first * a.D, sm.o, one, row0, a.rows, a.rows, a.D, 0, a.D, lane);
    return;
  }
  float inv[NQ];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const float l = half_sum(sm.l[n]);
    inv[n] = l > 0.f || l != l ? 1.0f / l : 0.f;
    const int r = row0 + 32 * n + lane;
    if (lane < 32 && r < a.rows) a.lse[head_rows + r] = l > 0.f ? sm.m[n] + __builtin_amdgcn_logf(l) : l != l ? l : INFINITY;
  }
  T *op = static_cast<T *>(a.out) + ((int64_t)b * a.Lq * a.H + (int64_t)hk * a.G) * a.D;
  store_rows<T, DP, NQ>(op, sm.o, inv, row0, a.rows, a.Lq, (int64_t)a.H * a.D, a.D, a.D, lane);
}

// Few rows (at most 32 NQ per key head): the NW waves take different key tiles, each with its own buffers (no
// barrier in the loop), and their running softmaxes are joined through LDS. Bound by the reading of K and V.
template <class T, int DP>
struct FewTile {
  static constexpr int KT = 32, NW = sizeof(T) * DP == 512 ? 2 : 4;  // 128 KB of LDS at most
};

template <class T, int DP, int NQ>
__global__ __launch_bounds__((64 * FewTile<T, DP>::NW), 1) void attn_few_kernel(const AttnArgs a) {
  constexpr int KT = FewTile<T, DP>::KT, NW = FewTile<T, DP>::NW, ND = DP / 32;
  using Tile = HeadTile<T, DP>;
  constexpr int TB = KT * Tile::RB, N = TB / 1024;
  static_assert(NW * NQ * ND * 4 * 64 * 16 <= 4 * TB * NW, "the waves' sums fit the buffers");
  __shared__ u32x4 smem[4 * TB * NW / 16];
  __shared__ float2 ml[NW][NQ][32];
  const int wave = wave_id(), lane = threadIdx.x & 63;
  MLORA_LDS char *lds = (MLORA_LDS char *)smem + wave * 4 * TB;
  int id = blockIdx.x;
  const int sp = id % a.splits;
  id /= a.splits;
  const int hk = id % a.Hk, b = id / a.Hk;
  const KeyMask<KT> km{a.mask == nullptr ? nullptr : a.mask + b * a.mask_sb, sample_keys(a, b)};
  const int t0 = sp * a.split_tiles + wave, t1 = min((sp + 1) * a.split_tiles, (km.len + KT - 1) / KT);
  const T *kp = static_cast<const T *>(a.k) + b * a.k_sb + hk * a.k_sh;
  const T *vp = static_cast<const T *>(a.v) + b * a.v_sb + hk * a.v_sh;
  TileLoader<T, DP, N> kl, vl;
  kl.init(lane, 0, 1, a.k_sl, a.D), vl.init(lane, 0, 1, a.v_sl, a.D);
  auto stage = [&](int t, int buf, uint64_t bits) __attribute__((always_inline)) {
    kl.load(kp + (int64_t)t * KT * a.k_sl, bits, lds + buf * 2 * TB);
    vl.load(vp + (int64_t)t * KT * a.v_sl, bits, lds + buf * 2 * TB + TB);
  };
  uint64_t bits = 0, next = 0;
  if (t0 < t1) {
    bits = km.bits(t0, km.byte(t0, lane));
    stage(t0, 0, bits);
    next = km.bits(t0 + NW, km.byte(t0 + NW, lane));
  }
  FragReader<T, DP> fr;
  fr.init(lane);
  Softmax<T, DP, NQ, KT> sm;
  sm.init();
  const T *qp = static_cast<const T *>(a.q) + b * a.q_sb + (int64_t)hk * a.G * a.q_sh;
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const T *p = qp + row_at(min(32 * n + (lane & 31), a.rows - 1), a.Lq, a.q_sl, a.q_sh);
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) {
      const int d = 16 * s + 8 * (lane >> 5);
      load_frag(p + d, d < a.D, sm.q[n][s]);
    }
  }
  auto turn = [&](auto buf, int t) __attribute__((always_inline)) {
    constexpr int B = decltype(buf)::value;
    wait_vmcnt<0>();  // tile t is in this wave's buffer
    asm volatile("" ::: "memory");
    int byte = 1;
    if (t + NW < t1) {
      stage(t + NW, B ^ 1, next);
      byte = km.byte(t + 2 * NW, lane);
    }
    if (bits != 0) sm.step(fr, lds + B * 2 * TB, lds + B * 2 * TB + TB, bits, a.c, lane);
    bits = next;
    next = km.bits(t + 2 * NW, byte);
  };
  for (int t = t0; t < t1; t += 2 * NW) {
    turn(std::integral_constant<int, 0>{}, t);
    if (t + NW < t1) turn(std::integral_constant<int, 1>{}, t + NW);
  }
  // join the waves: every wave leaves its sums, then sums its share of the 32 x 32 tiles over the waves
  float l[NQ];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    l[n] = half_sum(sm.l[n]);
    if (lane < 32) ml[wave][n][lane] = float2{sm.m[n], l[n]};
  }
  __syncthreads();
  f32x4 *sums = (f32x4 *)smem;
#pragma unroll
  for (int n = 0; n < NQ; ++n)
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        sums[(((wave * NQ + n) * ND + d) * 4 + i) * 64 + lane] =
            f32x4{sm.o[n][d][4 * i], sm.o[n][d][4 * i + 1], sm.o[n][d][4 * i + 2], sm.o[n][d][4 * i + 3]};
  __syncthreads();
  const int64_t head_rows = ((int64_t)b * a.Hk + hk) * a.rows, all = (int64_t)a.batches * a.Hk * a.rows;
  T *op = static_cast<T *>(a.out) + ((int64_t)b * a.Lq * a.H + (int64_t)hk * a.G) * a.D;
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int r = 32 * n + (lane & 31);
    float m = -INFINITY, lsum = 0.f, w[NW];
#pragma unroll
    for (int q = 0; q < NW; ++q) m = fmaxf(m, ml[q][n][lane & 31].x);
#pragma unroll
    for (int q = 0; q < NW; ++q) {
      const float2 v = ml[q][n][lane & 31];
      w[q] = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(v.x - m);
      lsum += w[q] * v.y;
    }
    const float inv = a.splits > 1 ? 1.f : lsum > 0.f || lsum != lsum ? 1.0f / lsum : 0.f;
    if (wave == 0 && lane < 32 && r < a.rows) {
      if (a.splits > 1) *(float2 *)(a.part_ml + 2 * (sp * all + head_rows + r)) = float2{m, lsum};
      else a.lse[head_rows + r] = lsum > 0.f ? m + __builtin_amdgcn_logf(lsum) : lsum != lsum ? lsum : INFINITY;
    }
    const int64_t at = row_at(min(r, a.rows - 1), a.Lq, (int64_t)a.H * a.D, a.D);
    for (int u = wave; u < 4 * ND; u += NW) {  // 4 consecutive channels per lane
      f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int q = 0; q < NW; ++q) o += w[q] * sums[((q * NQ + n) * 4 * ND + u) * 64 + lane];
      const int ch = 32 * (u / 4) + 8 * (u % 4) + 4 * (lane >> 5);
      if (r >= a.rows || ch >= a.D) continue;
      o *= inv;
      if (a.splits > 1) *(MLORA_GLOBAL f32x4 *)(a.part_o + (sp * all + head_rows + r) * a.D + ch) = o;
      else if constexpr (sizeof(T) == 2) *(MLORA_GLOBAL u32x2 *)(op + at + ch) = u32x2{pack2_bf16(o[0], o[1]), pack2_bf16(o[2], o[3])};
      else *(MLORA_GLOBAL f32x4 *)(op + at + ch) = o;
    }
  }
}

// Joins the splits of a row: weights 2^(m_s − max m).
template <class T>
__global__ __launch_bounds__(256) void attn_join_kernel(const AttnArgs a) {
  const int64_t all = (int64_t)a.batches * a.Hk * a.rows;
  const int per = 256 / 32;
  const int64_t row = (int64_t)blockIdx.x * per + threadIdx.x / 32;
  if (row >= all) return;
  const int at = threadIdx.x % 32;
  float m = -INFINITY;
  for (int s = 0; s < a.splits; ++s) m = fmaxf(m, a.part_ml[2 * (s * all + row)]);
  float l = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < a.splits; ++s) {
    const float2 ml = *(const float2 *)(a.part_ml + 2 * (s * all + row));
    const float w = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml.x - m);
    l += w * ml.y;
    if (4 * at < a.D) o += w * *(const MLORA_GLOBAL f32x4 *)(a.part_o + (s * all + row) * a.D + 4 * at);
  }
  const float inv = l > 0.f || l != l ? 1.0f / l : 0.f;
  if (at == 0) a.lse[row] = l > 0.f ? m + __builtin_amdgcn_logf(l) : l != l ? l : INFINITY;
  if (4 * at >= a.D) return;
  const int r = (int)(row % a.rows), hk = (int)(row / a.rows % a.Hk), b = (int)(row / a.rows / a.Hk);
  T *p = static_cast<T *>(a.out) + ((int64_t)b * a.Lq * a.H + (int64_t)hk * a.G) * a.D +
         row_at(r, a.Lq, (int64_t)a.H * a.D, a.D) + 4 * at;
  o *= inv;
  if constexpr (sizeof(T) == 2) *(MLORA_GLOBAL u32x2 *)p = u32x2{pack2_bf16(o[0], o[1]), pack2_bf16(o[2], o[3])};
  else *(MLORA_GLOBAL f32x4 *)p = o;
}

// ------------------------------------------------------------------ backward
//
//   P = 2^(s' − lse),  delta = Σ_d do·out,  dP = do·Vᵀ,  dS = P·(dP − delta)
//   dq = scale · dS·K,   dk = scale · dSᵀ·q,   dv = Pᵀ·do
// Two kernels form P again: one owns query rows (dq, and delta on the way), one owns keys (dk, dv). That
// is 7 products instead of 5, and no atomics: every sum has a fixed order. bf16: P and dS are rounded to bf16
// as operands of the products that follow.

struct AttnBwdArgs {
  AttnArgs f;
  const void *o, *g;  // the output [B, Lq, H, D] contiguous, and its gradient
  void *dq, *dk, *dv;  // contiguous
  float *delta;        // [B, H, Lq]
  f32x4 *part;         // dk / dv splits, in register order
  int64_t g_sb, g_sl, g_sh;
  float scale;
  int32_t key_blocks, q_tiles, head_q_tiles, q_splits, q_split_tiles;
};

template <class T, int DP>
__global__ __launch_bounds__(256, sizeof(T) == 2 ? 2 : 1) void attn_dq_kernel(const AttnBwdArgs ba) {
  const AttnArgs &a = ba.f;
  constexpr int KT = AttnTile<T>::KT, ND = DP / 32;
  using Tile = HeadTile<T, DP>;
  constexpr int TB = KT * Tile::RB, N = TB / 1024 / 4;
  __shared__ u32x4 smem[4 * TB / 16];
  MLORA_LDS char *lds = (MLORA_LDS char *)smem;
  const int wave = wave_id(), lane = threadIdx.x & 63;
  int id = xcd_contiguous(blockIdx.x, gridDim.x);
  const int rt = id % a.row_tiles;
  id /= a.row_tiles;
  const int hk = id % a.Hk, b = id / a.Hk;
  const KeyMask<KT> km{a.mask == nullptr ? nullptr : a.mask + b * a.mask_sb, sample_keys(a, b)};
  const int t1 = (km.len + KT - 1) / KT;
  const T *kp = static_cast<const T *>(a.k) + b * a.k_sb + hk * a.k_sh;
  const T *vp = static_cast<const T *>(a.v) + b * a.v_sb + hk * a.v_sh;
  TileLoader<T, DP, N> kl, vl;
  kl.init(lane, wave, 4, a.k_sl, a.D), vl.init(lane, wave, 4, a.v_sl, a.D);
  auto stage = [&](int t, int buf, uint64_t bits) __attribute__((always_inline)) {
    kl.load(kp + (int64_t)t * KT * a.k_sl, bits, lds + buf * 2 * TB);
    vl.load(vp + (int64_t)t * KT * a.v_sl, bits, lds + buf * 2 * TB + TB);
  };
  uint64_t bits = 0, next = 0;
  if (t1 > 0) {
    bits = km.bits(0, km.byte(0, lane));
    stage(0, 0, bits);
    next = km.bits(1, km.byte(1, lane));
  }
  FragReader<T, DP> fr;
  fr.init(lane);
  const int row0 = (rt * 4 + wave) * 32, r = row0 + (lane & 31), rc = min(r, a.rows - 1);
  const int64_t head_rows = ((int64_t)b * a.Hk + hk) * a.rows;
  const int64_t oat = ((int64_t)b * a.Lq * a.H + (int64_t)hk * a.G) * a.D;
  Frag<T> q[DP / 16], g[DP / 16];
  float delta = 0.f;
  {
    const T *qp = static_cast<const T *>(a.q) + b * a.q_sb + (int64_t)hk * a.G * a.q_sh + row_at(rc, a.Lq, a.q_sl, a.q_sh);
    const T *gp_ = static_cast<const T *>(ba.g) + b * ba.g_sb + (int64_t)hk * a.G * ba.g_sh + row_at(rc, a.Lq, ba.g_sl, ba.g_sh);
    const T *op = static_cast<const T *>(ba.o) + oat + row_at(rc, a.Lq, (int64_t)a.H * a.D, a.D);
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) {
      const int d = 16 * s + 8 * (lane >> 5);
      Frag<T> of;
      load_frag(qp + d, d < a.D, q[s]);
      load_frag(gp_ + d, d < a.D, g[s]);
      load_frag(op + d, d < a.D, of);
      if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          delta += __uint_as_float(g[s].v[j] << 16) * __uint_as_float(of.v[j] << 16);
          delta += __uint_as_float(g[s].v[j] & 0xffff0000u) * __uint_as_float(of.v[j] & 0xffff0000u);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) delta += g[s].v[j] * of.v[j];
      }
    }
  }
  delta = half_sum(delta);
  if (lane < 32 && r < a.rows) ba.delta[head_rows + r] = delta;
  const float lse = a.lse[head_rows + rc];
  f32x16 dq[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) dq[d][i] = 0.f;
  auto step = [&](const MLORA_LDS char *kt, const MLORA_LDS char *vt, uint64_t bits) __attribute__((always_inline)) {
#pragma unroll
    for (int kb = 0; kb < KT / 32; ++kb) {
      f32x16 s, dp;
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = 0.f, dp[i] = 0.f;
#pragma unroll
      for (int ks = 0; ks < DP / 16; ++ks) {
        Frag<T> kf, vf;
        fr.rows(kt, 32 * kb, ks, kf);
        s = mma16(kf, q[ks], s);
        fr.rows(vt, 32 * kb, ks, vf);
        dp = mma16(vf, g[ks], dp);
      }
      if (bits != low_bits(KT)) {
        const uint64_t mine = bits >> (4 * (lane >> 5));
#pragma unroll
        for (int i = 0; i < 16; ++i) s[i] = (mine >> (32 * kb + 8 * (i / 4) + i % 4)) & 1 ? s[i] : -INFINITY;
      }
      Frag<T> ds[2];
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = __builtin_amdgcn_exp2f(s[i] * a.c - lse) * (dp[i] - delta);
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        to_frag(s, ks, ds[ks]);
#pragma unroll
        for (int d = 0; d < ND; ++d) {
          Frag<T> kf;
          fr.cols(kt, 32 * kb + 16 * ks, d, kf);
          dq[d] = mma16(kf, ds[ks], dq[d]);
        }
      }
    }
  };
  auto turn = [&](auto buf, int t) __attribute__((always_inline)) {
    constexpr int B = decltype(buf)::value;
    wait_vmcnt<0>();
    lds_pipeline_barrier();  // tile t is in LDS, and every wave has read tile t - 1
    int byte = 1;
    if (t + 1 < t1) {
      stage(t + 1, B ^ 1, next);
      byte = km.byte(t + 2, lane);
    }
    if (bits != 0) step(lds + B * 2 * TB, lds + B * 2 * TB + TB, bits);
    bits = next;
    next = km.bits(t + 2, byte);
  };
  for (int t = 0; t < t1; t += 2) {
    turn(std::integral_constant<int, 0>{}, t);
    if (t + 1 < t1) turn(std::integral_constant<int, 1>{}, t + 1);
  }
  const float f[1] = {ba.scale};
  f32x16 o[1][ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) o[0][d] = dq[d];
  store_rows<T, DP, 1>(static_cast<T *>(ba.dq) + oat, o, f, row0, a.rows, a.Lq, (int64_t)a.H * a.D, a.D, a.D, lane);
}

// Four waves own 32 NK keys each (K and V fragments in registers) and share tiles of QT query rows of one head
// in LDS, double-buffered: q, the output's gradient, lse and delta.
template <class T, int DP, int NK>
__global__ __launch_bounds__(256, 1) void attn_dkv_kernel(const AttnBwdArgs ba) {
  const AttnArgs &a = ba.f;
  constexpr int QT = AttnTile<T>::KT, ND = DP / 32;
  using Tile = HeadTile<T, DP>;
  constexpr int TB = QT * Tile::RB, N = TB / 1024 / 4;
  __shared__ u32x4 smem[4 * TB / 16];
  __shared__ f32x4 stats[2][2][QT / 4];  // buffer; lse, delta
  MLORA_LDS char *lds = (MLORA_LDS char *)smem;
  const int wave = wave_id(), lane = threadIdx.x & 63;
  int id = xcd_contiguous(blockIdx.x, gridDim.x);
  const int kb = id % ba.key_blocks;
  id /= ba.key_blocks;
  const int sp = id % ba.q_splits;
  id /= ba.q_splits;
  const int hk = id % a.Hk, b = id / a.Hk;
  const int len = sample_keys(a, b);
  const int key0 = (kb * 4 + wave) * 32 * NK;
  const uint8_t *mask = a.mask == nullptr ? nullptr : a.mask + b * a.mask_sb;
  Frag<T> k[NK][DP / 16], v[NK][DP / 16];
  bool live[NK];
#pragma unroll
  for (int n = 0; n < NK; ++n) {
    const int key = key0 + 32 * n + (lane & 31);
    live[n] = key < len && (mask == nullptr || mask[key] != 0);
    const int64_t at = live[n] ? key : 0;
    const T *kp = static_cast<const T *>(a.k) + b * a.k_sb + hk * a.k_sh + at * a.k_sl;
    const T *vp = static_cast<const T *>(a.v) + b * a.v_sb + hk * a.v_sh + at * a.v_sl;
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) {
      const int d = 16 * s + 8 * (lane >> 5);
      load_frag(kp + d, live[n] && d < a.D, k[n][s]);
      load_frag(vp + d, live[n] && d < a.D, v[n][s]);
    }
  }
  f32x16 dk[NK][ND], dv[NK][ND];
#pragma unroll
  for (int n = 0; n < NK; ++n)
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) dk[n][d][i] = 0.f, dv[n][d][i] = 0.f;
  const int t0 = sp * ba.q_split_tiles;
  const int t1 = kb * 128 * NK >= len ? 0 : min(t0 + ba.q_split_tiles, ba.q_tiles);  // no key at all: zeros
  TileLoader<T, DP, N> ql, gl;
  ql.init(lane, wave, 4, a.q_sl, a.D), gl.init(lane, wave, 4, ba.g_sl, a.D);
  const int64_t head_rows = ((int64_t)b * a.Hk + hk) * a.rows;
  FragReader<T, DP> fr;
  fr.init(lane);
  // a tile's rows into LDS; returns lse (threads 0 .. QT - 1) or delta (QT .. 2 QT - 1) of the thread's row
  auto stage = [&](int t, int buf) __attribute__((always_inline)) -> float {
    const int g = t / ba.head_q_tiles, i0 = (t - g * ba.head_q_tiles) * QT, h = hk * a.G + g;
    const uint64_t rows = low_bits(min(a.Lq - i0, QT));
    ql.load(static_cast<const T *>(a.q) + b * a.q_sb + h * a.q_sh + i0 * a.q_sl, rows, lds + buf * 2 * TB);
    gl.load(static_cast<const T *>(ba.g) + b * ba.g_sb + h * ba.g_sh + i0 * ba.g_sl, rows, lds + buf * 2 * TB + TB);
    const int i = threadIdx.x % QT;
    const float *src = threadIdx.x < QT ? a.lse : ba.delta;
    float x = threadIdx.x < QT ? INFINITY : 0.f;  // rows behind the last: P = 0
    if (threadIdx.x < 2 * QT && i0 + i < a.Lq) x = src[head_rows + (int64_t)g * a.Lq + i0 + i];
    return x;
  };
  auto keep = [&](int buf, float x) __attribute__((always_inline)) {
    if (threadIdx.x < 2 * QT) ((float *)stats[buf][threadIdx.x / QT])[threadIdx.x % QT] = x;
  };
  auto step = [&](const MLORA_LDS char *qt, const MLORA_LDS char *gt, int buf) __attribute__((always_inline)) {
#pragma unroll
    for (int qb = 0; qb < QT / 32; ++qb) {
      f32x16 s[NK], dp[NK];
#pragma unroll
      for (int n = 0; n < NK; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[n][i] = 0.f, dp[n][i] = 0.f;
#pragma unroll
      for (int ks = 0; ks < DP / 16; ++ks) {
        Frag<T> f;
        fr.rows(qt, 32 * qb, ks, f);
#pragma unroll
        for (int n = 0; n < NK; ++n) s[n] = mma16(f, k[n][ks], s[n]);
      }
#pragma unroll
      for (int ks = 0; ks < DP / 16; ++ks) {
        Frag<T> f;
        fr.rows(gt, 32 * qb, ks, f);
#pragma unroll
        for (int n = 0; n < NK; ++n) dp[n] = mma16(f, v[n][ks], dp[n]);
      }
      Frag<T> pf[NK][2], df[NK][2];
#pragma unroll
      for (int i4 = 0; i4 < 4; ++i4) {
        const f32x4 lse = stats[buf][0][8 * qb + 2 * i4 + (lane >> 5)], delta = stats[buf][1][8 * qb + 2 * i4 + (lane >> 5)];
#pragma unroll
        for (int n = 0; n < NK; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float p = __builtin_amdgcn_exp2f(s[n][4 * i4 + j] * a.c - lse[j]);
            s[n][4 * i4 + j] = p;
            dp[n][4 * i4 + j] = p * (dp[n][4 * i4 + j] - delta[j]);
          }
      }
#pragma unroll
      for (int n = 0; n < NK; ++n)
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) to_frag(s[n], ks, pf[n][ks]), to_frag(dp[n], ks, df[n][ks]);
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
#pragma unroll
        for (int d = 0; d < ND; ++d) {
          Frag<T> f;
          fr.cols(gt, 32 * qb + 16 * ks, d, f);
#pragma unroll
          for (int n = 0; n < NK; ++n) dv[n][d] = mma16(f, pf[n][ks], dv[n][d]);
        }
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
#pragma unroll
        for (int d = 0; d < ND; ++d) {
          Frag<T> f;
          fr.cols(qt, 32 * qb + 16 * ks, d, f);
#pragma unroll
          for (int n = 0; n < NK; ++n) dk[n][d] = mma16(f, df[n][ks], dk[n][d]);
        }
    }
  };
  if (t0 < t1) keep(0, stage(t0, 0));
  auto turn = [&](auto buf, int t) __attribute__((always_inline)) {
    constexpr int B = decltype(buf)::value;
    wait_vmcnt<0>();
    lds_pipeline_barrier();  // tile t is in LDS, and every wave has read tile t - 1
    float x = 0.f;
    if (t + 1 < t1) x = stage(t + 1, B ^ 1);
    step(lds + B * 2 * TB, lds + B * 2 * TB + TB, B);
    if (t + 1 < t1) keep(B ^ 1, x);
  };
  for (int t = t0; t < t1; t += 2) {
    turn(std::integral_constant<int, 0>{}, t);
    if (t + 1 < t1) turn(std::integral_constant<int, 1>{}, t + 1);
  }
  float fk[NK], fv[NK];
#pragma unroll
  for (int n = 0; n < NK; ++n) {  // a masked key's column holds whatever its zeroed fragments gave
    fk[n] = ba.scale, fv[n] = 1.f;
    if (!live[n]) {
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) dk[n][d][i] = 0.f, dv[n][d][i] = 0.f;
    }
  }
  if (ba.q_splits > 1) {
    f32x4 *p = ba.part + (((((int64_t)sp * a.batches + b) * a.Hk + hk) * ba.key_blocks + kb) * 4 + wave) * (2 * NK * ND * 4 * 64) + lane;
#pragma unroll
    for (int n = 0; n < NK; ++n)
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          *(MLORA_GLOBAL f32x4 *)(p + ((n * ND + d) * 4 + i) * 64) =
              f32x4{dk[n][d][4 * i], dk[n][d][4 * i + 1], dk[n][d][4 * i + 2], dk[n][d][4 * i + 3]};
          *(MLORA_GLOBAL f32x4 *)(p + (((NK + n) * ND + d) * 4 + i) * 64) =
              f32x4{dv[n][d][4 * i], dv[n][d][4 * i + 1], dv[n][d][4 * i + 2], dv[n][d][4 * i + 3]};
        }
    return;
  }
  const int64_t at = ((int64_t)b * a.Lk * a.Hk + hk) * a.D;
  store_rows<T, DP, NK>(static_cast<T *>(ba.dk) + at, dk, fk, key0, a.Lk, a.Lk, (int64_t)a.Hk * a.D, 0, a.D, lane);
  store_rows<T, DP, NK>(static_cast<T *>(ba.dv) + at, dv, fv, key0, a.Lk, a.Lk, (int64_t)a.Hk * a.D, 0, a.D, lane);
}

// Adds the splits of dk and dv in split order and writes them out.
template <class T, int DP, int NK>
__global__ __launch_bounds__(256) void attn_dkv_join_kernel(const AttnBwdArgs ba) {
  const AttnArgs &a = ba.f;
  constexpr int ND = DP / 32;
  const int64_t per = (int64_t)a.batches * a.Hk * ba.key_blocks * 4 * 2 * NK * ND * 4 * 64;
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (e >= per) return;
  f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = 0; s < ba.q_splits; ++s) x += *(const MLORA_GLOBAL f32x4 *)(ba.part + s * per + e);
  int64_t u = e / 64;
  const int lane = (int)(e % 64), i = (int)(u % 4), d = (int)(u / 4 % ND), n = (int)(u / 4 / ND % NK), which = (int)(u / 4 / ND / NK % 2);
  u /= 4 * ND * NK * 2;  // (b, hk, key block, wave)
  const int64_t wave_block = u % (4 * ba.key_blocks), bh = u / (4 * ba.key_blocks);
  const int64_t key = wave_block * 32 * NK + 32 * n + (lane & 31);
  const int ch = 32 * d + 8 * i + 4 * (lane >> 5);
  if (key >= a.Lk || ch >= a.D) return;
  T *p = static_cast<T *>(which ? ba.dv : ba.dk) + ((bh / a.Hk * a.Lk + key) * a.Hk + bh % a.Hk) * a.D + ch;
  if (!which) x *= ba.scale;
  if constexpr (sizeof(T) == 2) *(MLORA_GLOBAL u32x2 *)p = u32x2{pack2_bf16(x[0], x[1]), pack2_bf16(x[2], x[3])};
  else *(MLORA_GLOBAL f32x4 *)p = x;
}

// The kernels are named here because hipcc's host pass does not instantiate a kernel that holds generic lambdas
// from a launch inside one.
#define MLORA_ATTN(T, DP)                                        \
  template __global__ void attn_fwd_kernel<T, DP, 1>(const AttnArgs); \
  template __global__ void attn_few_kernel<T, DP, 1>(const AttnArgs); \
  template __global__ void attn_few_kernel<T, DP, 2>(const AttnArgs); \
  template __global__ void attn_dq_kernel<T, DP>(const AttnBwdArgs);  \
  template __global__ void attn_dkv_kernel<T, DP, 1>(const AttnBwdArgs);
MLORA_ATTN(uint16_t, 64)
MLORA_ATTN(uint16_t, 128)
MLORA_ATTN(float, 64)
MLORA_ATTN(float, 128)
#undef MLORA_ATTN
template __global__ void attn_dkv_kernel<uint16_t, 64, 2>(const AttnBwdArgs);

// ------------------------------------------------------------------ host

constexpr int kAttnMaxHeadDim = 128, kFewRows = 64;

struct AttnPlan {
  bool few;
  int nq;  // 32-row blocks per wave
  int64_t row_tiles, splits, split_tiles;
};

// How a forward is cut: few rows per key head run waves over different keys, more rows 128 per workgroup;
// the keys are split where that leaves less than a workgroup for every compute unit and there are enough of them.
static AttnPlan attn_plan(int64_t batches, int64_t rows, int64_t Lk, int64_t Hk, int64_t D, bool f32) {
  AttnPlan p{};
  p.few = rows <= kFewRows;
  const int64_t waves = p.few && f32 && D > 64 ? 2 : 4;
  const int64_t kt = p.few || f32 ? 32 : 64, tiles = (Lk + kt - 1) / kt;
  p.nq = p.few && rows > 32 ? 2 : 1;
  p.row_tiles = p.few ? 1 : (rows + 127) / 128;
  const int64_t groups = batches * Hk * p.row_tiles;
  const int64_t least = p.few ? 4 * waves : 8;  // tiles that a split is worth its join for
  int64_t splits = groups > 0 && groups < 256 ? 256 / groups : 1;
  if (splits > tiles / least) splits = tiles / least;
  if (splits < 1) splits = 1;
  p.split_tiles = (tiles + splits - 1) / splits;
  if (p.split_tiles < 1) p.split_tiles = 1;
  p.splits = tiles > 0 ? (tiles + p.split_tiles - 1) / p.split_tiles : 1;
  return p;
}

static int64_t attn_part_floats(const AttnPlan &p, int64_t batches, int64_t Hk, int64_t rows, int64_t D) {
  return p.splits > 1 ? p.splits * batches * Hk * rows * (D + 2) : 0;
}

struct DkvPlan {
  int nk;
  int64_t key_blocks, q_tiles, head_q_tiles, splits, split_tiles;
};

// dk / dv: 128 nk keys per workgroup; the query rows are split where the keys alone leave compute units idle.
static DkvPlan dkv_plan(int64_t batches, int64_t Lq, int64_t Lk, int64_t Hk, int64_t G, int64_t D, bool f32) {
  DkvPlan p{};
  const int64_t qt = f32 ? 32 : 64;
  p.nk = !f32 && D <= 64 && Lk > 128 ? 2 : 1;
  p.key_blocks = (Lk + 128 * p.nk - 1) / (128 * p.nk);
  p.head_q_tiles = (Lq + qt - 1) / qt;
  p.q_tiles = G * p.head_q_tiles;
  const int64_t groups = batches * Hk * p.key_blocks;
  int64_t splits = groups > 0 && groups < 256 ? 256 / groups : 1;
  if (splits > p.q_tiles / 4) splits = p.q_tiles / 4;
  if (splits < 1) splits = 1;
  p.split_tiles = (p.q_tiles + splits - 1) / splits;
  if (p.split_tiles < 1) p.split_tiles = 1;
  p.splits = p.q_tiles > 0 ? (p.q_tiles + p.split_tiles - 1) / p.split_tiles : 1;
  return p;
}

static int64_t dkv_part_bytes(const DkvPlan &p, int64_t batches, int64_t Hk, int64_t D) {
  const int64_t nd = D > 64 ? 4 : 2;
  return p.splits > 1 ? p.splits * batches * Hk * p.key_blocks * 4 * 2 * p.nk * nd * 4 * 64 * 16 : 0;
}

// Sizes and types shared by every entry. MLORA_OK, or the status.
static int attn_sizes(int dtype, int64_t B, int64_t Lq, int64_t Lk, int64_t H, int64_t Hk, int64_t D) {
  if (dtype != MLORA_BF16 && dtype != MLORA_F32) return MLORA_ERR_UNSUPPORTED;
  if (B < 0 || Lq < 0 || Lk < 0 || H < 1 || Hk < 1 || H % Hk != 0) return MLORA_ERR_INVALID;
  if (D < 8 || D % 8 != 0 || D > kAttnMaxHeadDim) return MLORA_ERR_UNSUPPORTED;
  const int64_t most = INT32_MAX - 65536;
  if (H > most || Lk > most || (Lq > 0 && H > most / Lq)) return MLORA_ERR_LIMIT;  // rows per key head
  // workgroups: one per (sample, key head, 128 rows or keys), splits only below 256 of them
  const int64_t blocks = (H / Hk * Lq + 127) / 128 + (Lk + 127) / 128 + 256;
  if (B > 0 && (Hk > most / B || blocks > most / (B * Hk))) return MLORA_ERR_LIMIT;
  return MLORA_OK;
}

// A [B, L, heads, D] operand: 16-byte aligned heads, token strides whose tiles stay within 32-bit offsets.
static int check_heads(const void *p, int64_t sb, int64_t sl, int64_t sh, bool empty) {
  if (empty) return MLORA_OK;
  if (p == nullptr) return MLORA_ERR_INVALID;
  if (!aligned16(p) || sb < 0 || sl < 0 || sh < 0 || sb % 8 != 0 || sl % 8 != 0 || sh % 8 != 0) return MLORA_ERR_UNSUPPORTED;
  if (sl >= (int64_t)1 << 22) return MLORA_ERR_LIMIT;  // 64 rows of 2^22 floats: 2^30 bytes
  return MLORA_OK;
}

static int attn_args(AttnArgs &a, const void *q, const int64_t *qs, const void *k, const int64_t *ks, const void *v,
                     const int64_t *vs, int dtype, const int32_t *lengths, const uint8_t *mask, int64_t mask_sb,
                     float scale, const float *lse, int64_t B, int64_t Lq, int64_t Lk, int64_t H, int64_t Hk, int64_t D) {
  int st = attn_sizes(dtype, B, Lq, Lk, H, Hk, D);
  if (st) return st;
  if (!(scale > 0.f && scale < INFINITY) || qs == nullptr || ks == nullptr || vs == nullptr || mask_sb < 0)
    return MLORA_ERR_INVALID;
  st = check_heads(q, qs[0], qs[1], qs[2], B * Lq == 0);
  if (!st) st = check_heads(k, ks[0], ks[1], ks[2], B * Lk == 0);
  if (!st) st = check_heads(v, vs[0], vs[1], vs[2], B * Lk == 0);
  if (st) return st;
  if (B * Lq > 0 && lse == nullptr) return MLORA_ERR_INVALID;
  a = AttnArgs{};
  a.q = q, a.k = k, a.v = v, a.lse = const_cast<float *>(lse), a.lengths = lengths, a.mask = mask, a.mask_sb = mask_sb;
  a.q_sb = qs[0], a.q_sl = qs[1], a.q_sh = qs[2], a.k_sb = ks[0], a.k_sl = ks[1], a.k_sh = ks[2];
  a.v_sb = vs[0], a.v_sl = vs[1], a.v_sh = vs[2];
  a.batches = (int32_t)B, a.Lq = (int32_t)Lq, a.Lk = (int32_t)Lk, a.H = (int32_t)H, a.Hk = (int32_t)Hk;
  a.G = (int32_t)(H / Hk), a.D = (int32_t)D, a.rows = (int32_t)(H / Hk * Lq), a.c = scale * kLog2e;
  a.splits = 1;
  return MLORA_OK;
}

template <class F>
static void with_head(bool f32, int64_t D, F &&f) {
  using std::integral_constant;
  auto small = integral_constant<int, 64>{};
  auto large = integral_constant<int, 128>{};
  if (f32 && D <= 64) f(float{}, small);
  else if (f32) f(float{}, large);
  else if (D <= 64) f(uint16_t{}, small);
  else f(uint16_t{}, large);
}

}  // namespace mlora

using namespace mlora;

extern "C" int64_t mlora_cross_attention_workspace_bytes(int dtype, int64_t B, int64_t Lq, int64_t Lk, int64_t H,
                                                         int64_t Hk, int64_t D) {
  const int st = attn_sizes(dtype, B, Lq, Lk, H, Hk, D);
  if (st) return st;
  const int64_t rows = H / Hk * Lq;
  return attn_part_floats(attn_plan(B, rows, Lk, Hk, D, dtype == MLORA_F32), B, Hk, rows, D) * (int64_t)sizeof(float);
}

extern "C" int mlora_cross_attention(const void *q, const int64_t *q_strides, const void *k, const int64_t *k_strides,
                                     const void *v, const int64_t *v_strides, int dtype, const int32_t *key_lengths,
                                     const uint8_t *key_mask, int64_t key_mask_stride_b, float scale, void *out,
                                     float *lse, void *workspace, int64_t workspace_bytes, int64_t B, int64_t Lq,
                                     int64_t Lk, int64_t H, int64_t Hk, int64_t D, void *stream) {
  AttnArgs a;
  int st = attn_args(a, q, q_strides, k, k_strides, v, v_strides, dtype, key_lengths, key_mask, key_mask_stride_b, scale,
                     lse, B, Lq, Lk, H, Hk, D);
  if (st || B * Lq == 0) return st;
  if (out == nullptr) return MLORA_ERR_INVALID;
  if (!aligned16(out) || (reinterpret_cast<uintptr_t>(lse) & 3u) != 0) return MLORA_ERR_UNSUPPORTED;
  const bool f32 = dtype == MLORA_F32;
  const AttnPlan p = attn_plan(B, a.rows, Lk, Hk, D, f32);
  const int64_t floats = attn_part_floats(p, B, Hk, a.rows, D);
  if (floats > 0) {
    if (workspace == nullptr || workspace_bytes < floats * (int64_t)sizeof(float)) return MLORA_ERR_WORKSPACE;
    if (!aligned16(workspace)) return MLORA_ERR_UNSUPPORTED;
  }
  a.out = out, a.row_tiles = (int32_t)p.row_tiles, a.splits = (int32_t)p.splits, a.split_tiles = (int32_t)p.split_tiles;
  a.part_o = static_cast<float *>(workspace);
  a.part_ml = a.part_o + p.splits * B * Hk * a.rows * D;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 grid((unsigned)(B * Hk * p.row_tiles * p.splits));
  with_head(f32, D, [&](auto t, auto dp) {
    using T = decltype(t);
    constexpr int DP = decltype(dp)::value;
    if (p.few && p.nq == 1) hipLaunchKernelGGL((attn_few_kernel<T, DP, 1>), grid, dim3(64 * FewTile<T, DP>::NW), 0, s, a);
    else if (p.few) hipLaunchKernelGGL((attn_few_kernel<T, DP, 2>), grid, dim3(64 * FewTile<T, DP>::NW), 0, s, a);
    else hipLaunchKernelGGL((attn_fwd_kernel<T, DP, 1>), grid, dim3(256), 0, s, a);
  });
  st = launch_status();
  if (st || p.splits == 1) return st;
  const dim3 joins((unsigned)((B * Hk * a.rows + 7) / 8));
  if (f32) hipLaunchKernelGGL(attn_join_kernel<float>, joins, dim3(256), 0, s, a);
  else hipLaunchKernelGGL(attn_join_kernel<uint16_t>, joins, dim3(256), 0, s, a);
  return launch_status();
}

extern "C" int64_t mlora_cross_attention_backward_workspace_bytes(int dtype, int64_t B, int64_t Lq, int64_t Lk, int64_t H,
                                                                  int64_t Hk, int64_t D) {
  const int st = attn_sizes(dtype, B, Lq, Lk, H, Hk, D);
  if (st) return st;
  // delta, rounded up to whole 16-byte vectors, then the splits of dk and dv
  return (B * H * Lq + 3) / 4 * 16 + dkv_part_bytes(dkv_plan(B, Lq, Lk, Hk, H / Hk, D, dtype == MLORA_F32), B, Hk, D);
}

extern "C" int mlora_cross_attention_backward(const void *q, const int64_t *q_strides, const void *k,
                                              const int64_t *k_strides, const void *v, const int64_t *v_strides, int dtype,
                                              const int32_t *key_lengths, const uint8_t *key_mask,
                                              int64_t key_mask_stride_b, float scale, const void *out, const float *lse,
                                              const void *g, const int64_t *g_strides, void *dq, void *dk, void *dv,
                                              void *workspace, int64_t workspace_bytes, int64_t B, int64_t Lq, int64_t Lk,
                                              int64_t H, int64_t Hk, int64_t D, void *stream) {
  AttnBwdArgs ba{};
  int st = attn_args(ba.f, q, q_strides, k, k_strides, v, v_strides, dtype, key_lengths, key_mask, key_mask_stride_b,
                     scale, lse, B, Lq, Lk, H, Hk, D);
  if (st || B == 0) return st;
  if (g_strides == nullptr) return MLORA_ERR_INVALID;
  st = check_heads(g, g_strides[0], g_strides[1], g_strides[2], Lq == 0);
  if (st) return st;
  if ((Lq > 0 && (out == nullptr || dq == nullptr)) || (Lk > 0 && (dk == nullptr || dv == nullptr))) return MLORA_ERR_INVALID;
  for (const void *p : {out, (const void *)dq, (const void *)dk, (const void *)dv})
    if (!aligned16(p)) return MLORA_ERR_UNSUPPORTED;
  const bool f32 = dtype == MLORA_F32;
  if (workspace_bytes < mlora_cross_attention_backward_workspace_bytes(dtype, B, Lq, Lk, H, Hk, D) ||
      (workspace == nullptr && workspace_bytes > 0))
    return MLORA_ERR_WORKSPACE;
  if (!aligned16(workspace)) return MLORA_ERR_UNSUPPORTED;
  AttnArgs &a = ba.f;
  const DkvPlan p = dkv_plan(B, Lq, Lk, Hk, a.G, D, f32);
  ba.o = out, ba.g = g, ba.g_sb = g_strides[0], ba.g_sl = g_strides[1], ba.g_sh = g_strides[2], ba.scale = scale;
  ba.dq = dq, ba.dk = dk, ba.dv = dv, ba.delta = static_cast<float *>(workspace);
  ba.part = static_cast<f32x4 *>(workspace) + (B * H * Lq + 3) / 4;
  ba.key_blocks = (int32_t)p.key_blocks, ba.q_tiles = (int32_t)p.q_tiles, ba.head_q_tiles = (int32_t)p.head_q_tiles;
  ba.q_splits = (int32_t)p.splits, ba.q_split_tiles = (int32_t)p.split_tiles;
  a.row_tiles = (int32_t)((a.rows + 127) / 128);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (Lq > 0) {
    with_head(f32, D, [&](auto t, auto dp) {
      hipLaunchKernelGGL((attn_dq_kernel<decltype(t), decltype(dp)::value>), dim3((unsigned)(B * Hk * a.row_tiles)),
                         dim3(256), 0, s, ba);
    });
    st = launch_status();
    if (st) return st;
  }
  if (Lk == 0) return MLORA_OK;
  const dim3 grid((unsigned)(B * Hk * p.key_blocks * p.splits));
  const int64_t vectors = B * Hk * p.key_blocks * 4 * 2 * p.nk * (D > 64 ? 4 : 2) * 4 * 64;
  with_head(f32, D, [&](auto t, auto dp) {
    using T = decltype(t);
    constexpr int DP = decltype(dp)::value;
    auto run = [&](auto nk) {
      constexpr int NK = decltype(nk)::value;
      hipLaunchKernelGGL((attn_dkv_kernel<T, DP, NK>), grid, dim3(256), 0, s, ba);
      if (p.splits > 1)
        hipLaunchKernelGGL((attn_dkv_join_kernel<T, DP, NK>), dim3((unsigned)((vectors + 255) / 256)), dim3(256), 0, s, ba);
    };
    if constexpr (sizeof(T) == 2 && DP == 64) {
      if (p.nk == 2) return run(std::integral_constant<int, 2>{});
    }
    run(std::integral_constant<int, 1>{});
  });
  return launch_status();
}
