// Attention of q to an encoder's keys and values of another length. Forward:
//
//   s_j = scale · q·k_j over the sample's live keys (its first key_lengths[b], those with key_mask set);
//   out = Σ_j p_j v_j with p = softmax(s);  a query without a live key gets zeros.
//
// One pass over the keys with a running maximum m (of the products themselves) and sum l per query, c = scale·log2 e:
//   P = 2^(s·c − m·c),  l = Σ P,  O = Σ P·V;  out = O / l,  lse = m·c + log2 l (+inf for a query without keys, so
// that every 2^(s·c − lse) is 0). The running maximum is raised only when a tile's exceeds it by a factor of more
// than 2^8 (P then stays below 2^8, far from any limit, and rounding is relative), so the rescaling of O is a rare
// branch. Scores of any finite size count by their differences (RowRef): where |m·c| is small, the exponent is one fma
// whose constant's rounding all weights of the row share; from 2^10 on s − m is formed first, which is exact where
// it matters, and the backward, whose lse would have lost log2 l, measures m and l once more. bf16: P is rounded to bf16 for the product with V, and l sums the rounded
// values, so that the weights that multiply V add up to one. Everything else is float32.
//
// Rows: the G = heads / kv_heads query heads that share a key head are packed, row r = g·Lq + i, so that shared
// keys are read once for all of them.
//
// Products are of transposed tiles (Sᵀ = K·Qᵀ, Oᵀ = Vᵀ·Pᵀ): a column of a 32 x 32 result is a query, its softmax
// needs one exchange between two lanes, and the result's registers are the next product's operand as they lie.
//
// What bounds it, bf16 with 128 channels: a 32 x 32 block of scores costs the SIMD's matrix core 16 products of
// 32 cycles and its vector unit about as many cycles (16 exp2 at a quarter of the rate, the maximum, fma, packing);
// the two waves of a SIMD overlap the two only in part. dk / dv has fewer vector instructions per product (4.3; forward 7.6,
// dq 6.8) but two LDS reads (1.5, 1.3), since every fragment it reads feeds one product, and it spills six registers. Counters at
// 2 x 32760 rows x 512 keys, 12 heads: matrix cores busy 34 % of the cycles forward, 37 % in dq, 46 % in dk / dv, no
// LDS bank conflict. Measured there, averages of 20 calls (minima): forward 302 us (275; 680 TFLOP/s), dq 425 (392;
// 730), dk / dv 470 (424; 880). 16380 rows x 4096 keys: forward 433 us (950), dq 562 (1100). Few rows are bound by
// reading K and V: 48 rows per key head x 65520 keys, 8 key heads, 268 MB: 52 us, 5.1 TB/s, and 5 us for the join of
// its 32 splits.
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
  int32_t batches, Lq, Lk, H, Hk, G, D, rows, row_tiles, turns, splits, split_tiles;
  float c;            // scale · log2 e
};

// How many of 16 mask bytes are set, without the first `skip`.
typedef uint32_t unaligned_u4 __attribute__((ext_vector_type(4), aligned(1)));
__device__ __forceinline__ int live_bytes(const u32x4 &v, int skip) {
  int n = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t set = (((v[j] & 0x7f7f7f7fu) + 0x7f7f7f7fu) | v[j]) & 0x80808080u;  // a byte's top bit: it is not 0
    n += __popc(set & (uint32_t)(0xffffffffull << (8 * min(max(skip - 4 * j, 0), 4))));
  }
  return n;
}

// A sample's live keys, 64 (or KT) at a time.
template <int KT>
struct KeyMask {
  const uint8_t *mask;  // null: no mask
  int len;              // keys from here on do not count (the sample's length, or the split's end before it)
  __device__ __forceinline__ int byte(int tile, int lane) const {  // of key tile·KT + lane
    if (mask == nullptr) return 1;
    return mask[max(min(tile * KT + (lane & (KT - 1)), len - 1), 0)];
  }
  __device__ __forceinline__ uint64_t bits(int tile, int lane_byte) const {
    uint64_t b = low_bits(min(len - tile * KT, KT));
    if (mask != nullptr) {
      asm volatile("" : "+v"(lane_byte));  // looked at here and not where it was loaded
      b &= __ballot(lane_byte != 0);
    }
    return b;
  }
};

__device__ __forceinline__ int sample_keys(const AttnArgs &a, int b) {
  return a.lengths == nullptr ? a.Lk : min(max(a.lengths[b], 0), a.Lk);
}

// Rows of an attention call: address of row r of (b, kv head), in elements.
__device__ __forceinline__ int64_t row_at(int r, int Lq, int64_t sl, int64_t sh) {
  const int g = r / Lq, i = r - g * Lq;
  return g * sh + i * sl;
}

// Four waves of 32 rows each against the same key tiles, two buffers of K and V in LDS: tile t + 1 loads while tile
// t is multiplied; one barrier per tile. A workgroup takes `turns` row tiles of one head in a row: the key tiles
// go on loading from one to the next, and the next rows' q arrives under the present ones' products (with one row
// tile per workgroup and 512 keys, every workgroup waits for q and its first keys, in step with all others).
template <class T, int DP, bool EXACT>
__global__ __launch_bounds__(256, sizeof(T) == 2 ? 2 : 1) void attn_fwd_kernel(const AttnArgs a) {
  constexpr int KT = AttnTile<T>::KT;
  using Tile = HeadTile<T, DP>;
  constexpr int TB = KT * Tile::RB, N = TB / 1024 / 4;
  __shared__ u32x4 smem[4 * TB / 16];  // K, V of buffer 0, K, V of buffer 1
  MLORA_LDS char *lds = (MLORA_LDS char *)smem;
  const int wave = wave_id(), lane = threadIdx.x & 63;
  int id = blockIdx.x;  // heads first: rows of all heads are read together, whole token rows of memory
  const int hk = id % a.Hk;
  id /= a.Hk;
  const int groups = (a.row_tiles + a.turns - 1) / a.turns;
  const int rt0 = id % groups * a.turns, rt1 = min(rt0 + a.turns, a.row_tiles);
  id /= groups;
  const int sp = id % a.splits, b = id / a.splits;
  const int t0 = sp * a.split_tiles;
  const int end = (int)min((int64_t)(t0 + a.split_tiles) * KT, (int64_t)sample_keys(a, b)), t1 = (end + KT - 1) / KT;
  const KeyMask<KT> km{a.mask == nullptr ? nullptr : a.mask + b * a.mask_sb, end};
  const T *kp = static_cast<const T *>(a.k) + b * a.k_sb + hk * a.k_sh;
  const T *vp = static_cast<const T *>(a.v) + b * a.v_sb + hk * a.v_sh;
  TileLoader<T, DP, N> kl, vl;
  kl.init(lane, wave, 4, a.k_sl, a.D), vl.init(lane, wave, 4, a.v_sl, a.D);
  auto stage = [&](int t, int buf, uint64_t bits) __attribute__((always_inline)) {
    kl.load(kp + (int64_t)t * KT * a.k_sl, bits, lds + buf * 2 * TB);
    vl.load(vp + (int64_t)t * KT * a.v_sl, bits, lds + buf * 2 * TB + TB);
  };
  auto after = [&](int t) __attribute__((always_inline)) { return t + 1 < t1 ? t + 1 : t0; };  // the tiles go round
  uint64_t bits = 0, next = 0;
  if (t0 < t1) {
    bits = km.bits(t0, km.byte(t0, lane));
    stage(t0, 0, bits);
    next = km.bits(after(t0), km.byte(after(t0), lane));
  }
  FragReader<T, DP> fr;
  fr.init(lane, lds);
  Softmax<T, DP, 1, KT, EXACT> sm;
  const T *qp = static_cast<const T *>(a.q) + b * a.q_sb + (int64_t)hk * a.G * a.q_sh;
  Frag<T> qn[DP / 16];
  auto load_q = [&](int rt) __attribute__((always_inline)) {
    const T *p = qp + row_at(min((rt * 4 + wave) * 32 + (lane & 31), a.rows - 1), a.Lq, a.q_sl, a.q_sh);
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) {
      const int d = 16 * s + 8 * (lane >> 5);
      load_frag(p, d, d < a.D, qn[s]);
    }
  };
  load_q(rt0);
  const int64_t head_rows = ((int64_t)b * a.Hk + hk) * a.rows, all = (int64_t)a.batches * a.Hk * a.rows;
  T *op = static_cast<T *>(a.out) + ((int64_t)b * a.Lq * a.H + (int64_t)hk * a.G) * a.D;
  constexpr int kLoadsQ = DP / 16 * sizeof(T) / 2;
  int buf = 0;
  for (int rt = rt0; rt < rt1; ++rt) {
    sm.init();
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) sm.q[0][s] = qn[s];
    for (int t = t0; t < t1; ++t) {
      // the tile's loads: the next rows' q, asked for behind them, need not be there yet; at the first tile of later
      // rows they were waited for before the stores, which nothing waits for
      if (t == t0 + 1) wait_vmcnt<kLoadsQ>();
      else if (t > t0 || rt == rt0) wait_vmcnt<0>();
      lds_pipeline_barrier();  // tile t is in LDS, and every wave has read the tile before it
      buf ^= 1;
      stage(after(t), buf, rt + 1 < rt1 || t + 1 < t1 ? next : 0);  // behind the last one nothing is read
      const int byte = km.byte(after(after(t)), lane);
      if (t == t0) {  // kept between the tile's loads and the next wait, which counts them
        asm volatile("" ::: "memory");
        load_q(min(rt + 1, rt1 - 1));
        asm volatile("" ::: "memory");
      }
      if (bits != 0) sm.template step<0, TB>(fr, bits, a.c, lane);
      fr.flip(2 * TB);
      bits = next;
      next = km.bits(after(after(t)), byte);
    }
    const int row0 = (rt * 4 + wave) * 32, r = row0 + (lane & 31);
    float f[1];
    const float l = sm.sums(0, f[0]);
    if (t1 - t0 == 1) wait_vmcnt<kLoadsQ>();  // the next rows' first tile
    else wait_vmcnt<0>();
    if (a.splits > 1) {
      const int64_t first = sp * all + head_rows;
      if (lane < 32 && r < a.rows) *(float2 *)(a.part_ml + 2 * (first + r)) = float2{sm.m[0], l};
      store_rows<float, DP, 1>(a.part_o + first * a.D, sm.o, f, row0, a.rows, [&](int r) { return (int64_t)r * a.D; }, a.D, lane);
    } else {
      const float inv[1] = {l > 0.f || l != l ? f[0] / l : 0.f};
      if (lane < 32 && r < a.rows) a.lse[head_rows + r] = row_lse(sm.m[0], l, a.c);
      store_rows<T, DP, 1>(op, sm.o, inv, row0, a.rows, [&](int r) { return row_at(r, a.Lq, (int64_t)a.H * a.D, a.D); }, a.D, lane);
    }
  }
  wait_vmcnt<0>();
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
  // one array, so that the readers' buffers start at multiples of 4 TB; (m, l) of [wave][n][query] behind them
  __shared__ u32x4 smem[4 * TB * NW / 16 + NW * NQ * 16];
  float2 (&ml)[NW][NQ][32] = *(float2 (*)[NW][NQ][32])(smem + 4 * TB * NW / 16);
  const int wave = wave_id(), lane = threadIdx.x & 63;
  MLORA_LDS char *lds = (MLORA_LDS char *)smem + wave * 4 * TB;
  int id = blockIdx.x;
  const int sp = id % a.splits;
  id /= a.splits;
  const int hk = id % a.Hk, b = id / a.Hk;
  const int t0 = sp * a.split_tiles + wave;
  const int end = (int)min((int64_t)(sp + 1) * a.split_tiles * KT, (int64_t)sample_keys(a, b)), t1 = (end + KT - 1) / KT;
  const KeyMask<KT> km{a.mask == nullptr ? nullptr : a.mask + b * a.mask_sb, end};
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
  fr.init(lane, lds);
  Softmax<T, DP, NQ, KT, true> sm;  // bound by K and V: the second sum costs nothing
  sm.init();
  const T *qp = static_cast<const T *>(a.q) + b * a.q_sb + (int64_t)hk * a.G * a.q_sh;
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const T *p = qp + row_at(min(32 * n + (lane & 31), a.rows - 1), a.Lq, a.q_sl, a.q_sh);
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) {
      const int d = 16 * s + 8 * (lane >> 5);
      load_frag(p, d, d < a.D, sm.q[n][s]);
    }
  }
  auto turn = [&](auto buf, int t) __attribute__((always_inline)) {
    constexpr int B = decltype(buf)::value;
    wait_vmcnt<0>();  // tile t is in this wave's buffer
    asm volatile("" ::: "memory");
    stage(t + NW, 1 - B, next);  // past the last tile: no live row, nothing is read
    const int byte = km.byte(t + 2 * NW, lane);
    if (bits != 0) sm.template step<2 * B * TB, 2 * B * TB + TB>(fr, bits, a.c, lane);
    bits = next;
    next = km.bits(t + 2 * NW, byte);
  };
  for (int t = t0; t < t1; t += 2 * NW) {
    turn(std::integral_constant<int, 0>{}, t);
    if (t + NW < t1) turn(std::integral_constant<int, 1>{}, t + NW);
  }
  wait_vmcnt<0>();
  // join the waves: every wave leaves its sums, then sums its share of the 32 x 32 tiles over the waves
  float f[NQ];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const float l = sm.sums(n, f[n]);
    if (lane < 32) ml[wave][n][lane] = float2{sm.m[n], l};
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
            f32x4{sm.o[n][d][4 * i], sm.o[n][d][4 * i + 1], sm.o[n][d][4 * i + 2], sm.o[n][d][4 * i + 3]} * f[n];
  __syncthreads();
  const int64_t head_rows = ((int64_t)b * a.Hk + hk) * a.rows, all = (int64_t)a.batches * a.Hk * a.rows;
  T *op = static_cast<T *>(a.out) + ((int64_t)b * a.Lq * a.H + (int64_t)hk * a.G) * a.D;
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int r = 32 * n + (lane & 31);
    float m = kNoMax, lsum = 0.f, w[NW];
#pragma unroll
    for (int q = 0; q < NW; ++q) m = fmaxf(m, ml[q][n][lane & 31].x);
    const RowRef top = row_ref(m, a.c);
#pragma unroll
    for (int q = 0; q < NW; ++q) {
      const float2 v = ml[q][n][lane & 31];
      w[q] = ref_factor(row_ref(v.x, a.c), top, a.c);
      lsum += w[q] * v.y;
    }
    const float inv = a.splits > 1 ? 1.f : lsum > 0.f || lsum != lsum ? 1.0f / lsum : 0.f;
    if (wave == 0 && lane < 32 && r < a.rows) {
      if (a.splits > 1) *(float2 *)(a.part_ml + 2 * (sp * all + head_rows + r)) = float2{m, lsum};
      else a.lse[head_rows + r] = row_lse(m, lsum, a.c);
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

// Joins the splits of a row, one workgroup per row: weights 2^((m_s − max m)·c). Eight groups of 32 lanes (4 channels
// each) take every eighth split, and their sums are added in order through LDS.
template <class T>
__global__ __launch_bounds__(256) void attn_join_kernel(const AttnArgs a) {
  __shared__ f32x4 sums[8][32];
  __shared__ float ls[8];
  const int64_t all = (int64_t)a.batches * a.Hk * a.rows, row = blockIdx.x;
  const int at = threadIdx.x % 32, g = threadIdx.x / 32;
  float m = kNoMax;
  for (int s = at; s < a.splits; s += 32) m = fmaxf(m, a.part_ml[2 * (s * all + row)]);
#pragma unroll
  for (int i = 16; i >= 1; i >>= 1) m = fmaxf(m, __shfl_xor(m, i));
  const RowRef top = row_ref(m, a.c);
  float l = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = g; s < a.splits; s += 8) {
    const float2 ml = *(const float2 *)(a.part_ml + 2 * (s * all + row));
    const float w = ref_factor(row_ref(ml.x, a.c), top, a.c);
    l += w * ml.y;
    if (4 * at < a.D) o += w * *(const MLORA_GLOBAL f32x4 *)(a.part_o + (s * all + row) * a.D + 4 * at);
  }
  sums[g][at] = o;
  if (at == 0) ls[g] = l;
  __syncthreads();
  if (g != 0) return;
#pragma unroll
  for (int i = 1; i < 8; ++i) o += sums[i][at], l += ls[i];
  const float inv = l > 0.f || l != l ? 1.0f / l : 0.f;
  if (at == 0) a.lse[row] = row_lse(m, l, a.c);
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
//   P = 2^(s·c − lse),  delta = Σ_d do·out,  dP = do·Vᵀ,  dS = P·(dP − delta)
//   dq = scale · dS·K,   dk = scale · dSᵀ·q,   dv = Pᵀ·do
// Two kernels form P again: one owns query rows (dq, and delta on the way), one owns keys (dk, dv). That
// is 7 products instead of 5, and no atomics: every sum has a fixed order. One kernel for all three would write and
// add up float32 parts of dq per 256 keys (402 MB each at 2 x 32760 rows of 12 x 128: more time than its
// two products). bf16: P and dS are rounded to bf16 as operands of the products that follow: half a step each,
// 1.7e-3 of dq, dk and dv in the mean square where few rows add up, as much as their own rounding. FINE: what the
// rounding left is a second operand, and the forward's lse holds the weights' sum before their rounding. Then the
// gradients' own rounding remains, and beyond 64 live keys delta's from the rounded out: relative to |do| |out|, little where
// out averages many values, up to half a step where one key has nearly all the weight (dq's error at 512 keys 2.4e-3 ->
// 1.7e-3). At 2 x 32760 rows x 512 keys, 12 heads of 128, that costs dq 414 -> 456 us and dk alone 460 -> 617:
// it is done up to 2^30 products of scores and channels of one sample, whatever the batch, so that a sample's gradients do
// not depend on what it is batched with. Below that line it costs a backward a tenth to a fifth (500 x 512, 12 heads
// of 128: 49 -> 59 us; with the forward 64 of them 706 -> 846; 1000 x 1000, 8 of 64: 41 -> 44), and single rows of a
// long cache a quarter (4 x 1 x 58981 keys, 40 heads on 4 of 64: 407 -> 513 us): it is there that dv, a sum of few rows,
// has the most to lose.

struct AttnBwdArgs {
  AttnArgs f;
  const void *o, *g;  // the output [B, Lq, H, D] contiguous, and its gradient
  void *dq, *dk, *dv;  // contiguous
  float *stats;        // [3][B·H·Lq]: x, delta and a of every row, P = 2^((s − a)·c − x): a = 0 and x = lse, but far from
                       // zero a = m and x = log2 l
  f32x4 *part;         // splits of dq, then of dk and dv, in register order
  int64_t g_sb, g_sl, g_sh;
  float scale;
  int32_t key_blocks, q_tiles, head_q_tiles, q_splits, q_split_tiles;  // dk / dv; dq's splits are f's
};

template <class T, int DP, int NW, bool FINE>
__global__ __launch_bounds__((64 * NW), (sizeof(T) == 2 ? 2 : 1)) void attn_dq_kernel(const AttnBwdArgs ba) {
  const AttnArgs &a = ba.f;
  constexpr int KT = AttnTile<T>::KT, ND = DP / 32;
  using Tile = HeadTile<T, DP>;
  constexpr int TB = KT * Tile::RB, N = TB / 1024 / NW;
  __shared__ u32x4 smem[4 * TB / 16];
  MLORA_LDS char *lds = (MLORA_LDS char *)smem;
  const int wave = wave_id(), lane = threadIdx.x & 63;
  int id = blockIdx.x;  // heads first: rows of all heads are read together, whole token rows of memory
  const int hk = id % a.Hk;
  id /= a.Hk;
  const int rt = id % a.row_tiles;
  id /= a.row_tiles;
  const int b = id % a.batches, sp = id / a.batches;
  const int t0 = sp * a.split_tiles, keys = sample_keys(a, b);
  const int end = (int)min((int64_t)(t0 + a.split_tiles) * KT, (int64_t)keys), t1 = (end + KT - 1) / KT;
  const uint8_t *mask = a.mask == nullptr ? nullptr : a.mask + b * a.mask_sb;
  const T *kp = static_cast<const T *>(a.k) + b * a.k_sb + hk * a.k_sh;
  const T *vp = static_cast<const T *>(a.v) + b * a.v_sb + hk * a.v_sh;
  TileLoader<T, DP, N> kl, vl;
  kl.init(lane, wave, NW, a.k_sl, a.D), vl.init(lane, wave, NW, a.v_sl, a.D);
  auto stage = [&](int t, int buf, uint64_t bits) __attribute__((always_inline)) {
    kl.load(kp + (int64_t)t * KT * a.k_sl, bits, lds + buf * 2 * TB);
    vl.load(vp + (int64_t)t * KT * a.v_sl, bits, lds + buf * 2 * TB + TB);
  };
  uint64_t bits = 0, next = 0;
  auto start = [&](const KeyMask<KT> &km, int first, int second) __attribute__((always_inline)) {
    bits = km.bits(first, km.byte(first, lane));
    stage(first, 0, bits);
    next = km.bits(second, km.byte(second, lane));
  };
  FragReader<T, DP> fr;
  fr.init(lane, lds);
  // body(live bits) for the tiles first .. last - 1 after start(first); tile `last` is asked for too: without live keys
  auto sweep = [&](const KeyMask<KT> &km, int first, int last, auto tile, auto body) __attribute__((always_inline)) {
    for (int t = first; t < last; ++t) {
      wait_vmcnt<0>();
      lds_pipeline_barrier();  // tile t is in LDS, and every wave has read tile t - 1
      stage(tile(t + 1), (t + 1 - first) & 1, next);  // past the last tile: no live row, nothing is read
      const int byte = km.byte(tile(t + 2), lane);
      if (bits != 0) body(bits);
      fr.flip(2 * TB);
      bits = next;
      next = km.bits(tile(t + 2), byte);
    }
    wait_vmcnt<0>();
  };
  auto same = [](int t) __attribute__((always_inline)) { return t; };
  const int row0 = (rt * NW + wave) * 32, r = row0 + (lane & 31), rc = min(r, a.rows - 1);
  const int64_t head_rows = ((int64_t)b * a.Hk + hk) * a.rows;
  float wg_lse[NW / 2];  // of all the workgroup's rows, in every wave: asked for first, looked at below
#pragma unroll
  for (int i = 0; i < NW / 2; ++i) wg_lse[i] = a.lse[head_rows + min(rt * NW * 32 + 64 * i + lane, a.rows - 1)];
  if (t0 < t1) start(KeyMask<KT>{mask, end}, t0, t0 + 1);
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
      load_frag(qp, d, d < a.D, q[s]);
      load_frag(gp_, d, d < a.D, g[s]);
      load_frag(op, d, d < a.D, of);
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
  float x = a.lse[head_rows + rc], shift = 0.f;  // P = 2^((s − shift)·c − x)
  auto scores = [&](auto block, uint64_t bits, f32x16 &s, f32x16 &dp) __attribute__((always_inline)) {  // S and dP
    constexpr int kb = decltype(block)::value;
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = 0.f, dp[i] = 0.f;
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks) {
      Frag<T> kf, vf;
      fr.template rows<0, 32 * kb>(ks, kf);
      s = mma16(kf, q[ks], s);
      fr.template rows<TB, 32 * kb>(ks, vf);
      dp = mma16(vf, g[ks], dp);
    }
    if (bits != low_bits(KT)) {
      const uint64_t mine = bits >> (4 * (lane >> 5));
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = (mine >> (32 * kb + 8 * (i / 4) + i % 4)) & 1 ? s[i] : -INFINITY;
    }
  };
  // Few live keys, and roundings to bf16 do not average away: out's tells in delta, the weights' in their sum (2 to 5
  // keys: 1.4e-3 to 4e-3 of dq and dk, as much and more than the gradients' own). Then x and delta are measured too. From
  // 65 keys on delta's share is below a third of that. The keys are counted up to there, with length and mask; lane i
  // keeps the i-th tile that has one. The measuring takes 2 us of a small backward (2 x 1560 rows, 12 heads of 128, 5 of 512
  // keys: 52 -> 54 us) and 2 per tile where the keys lie far apart (40 of 65520, 16 rows, 24 heads on 8: 124 -> 241); its
  // presence costs dq 3 % where it does not run but tiles are few (2 x 32760 x 512: 383 -> 395).
  int live = 0, live_tiles = 0, list = 0;
  if constexpr (sizeof(T) == 2) {
    if (mask == nullptr || keys <= KT) {
      live = keys, live_tiles = 1;
    } else {
      // 16 keys per lane and load, unaligned; the row's last load begins at keys − 16 and leaves out what came before
      constexpr int kAtOnce = 4;
      for (int k0 = 0; k0 < keys && live <= KT; k0 += kAtOnce * 1024) {
        u32x4 bytes[kAtOnce];
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j) bytes[j] = *(const unaligned_u4 *)(mask + min(k0 + 1024 * j + 16 * lane, keys - 16));
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j) {
          const int key = k0 + 1024 * j + 16 * lane;
          const int n = live_bytes(bytes[j], max(key - (keys - 16), 0));
          const uint64_t on = __ballot(n != 0);
          if (on == 0) continue;
#pragma unroll
          for (int bit = 0; bit < 5; ++bit) live += __popcll(__ballot((n >> bit) & 1)) << bit;
          if (live > KT) break;
          for (int t = 0; t < 16; ++t)  // four lanes hold a tile
            if ((on >> (4 * t)) & 15) {
              if (lane == live_tiles) list = k0 / KT + 16 * j + t;
              ++live_tiles;
            }
        }
      }
    }
  }
  const bool few = sizeof(T) == 2 && live > 0 && live <= KT;
  // Rows far from zero, whose lse says nothing of log2 l: their maximum, sum and delta are measured over all keys of
  // the sample. The workgroup's waves share the tiles, so that they all do.
  bool far = false;
#pragma unroll
  for (int i = 0; i < NW / 2; ++i) far |= fabsf(wg_lse[i]) >= kFar && fabsf(wg_lse[i]) < INFINITY;
  if (few || __any(far)) {
    float m = kNoMax, l = 0.f, pd = 0.f;
    const KeyMask<KT> km{mask, keys};
    const int tiles = (keys + KT - 1) / KT, n = few ? live_tiles : tiles;
    auto tile = [&](int i) __attribute__((always_inline)) { return i >= n ? tiles : few ? __builtin_amdgcn_readlane(list, i) : i; };
    const bool there = n == 1 && tile(0) == t0 && t0 < t1;  // the only tile is this split's first
    const uint64_t first = bits;
    if (!there) {
      wait_vmcnt<0>();
      lds_pipeline_barrier();  // what is on its way into the buffers has arrived
      start(km, tile(0), tile(1));
    }
    sweep(km, 0, n, tile, [&](uint64_t bits) __attribute__((always_inline)) {
      static_for<KT / 32>([&](auto block) __attribute__((always_inline)) {
        f32x16 s, dp;
        scores(block, bits, s, dp);
        float mx = s[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) mx = fmaxf(mx, s[i]);
        mx = fmaxf(m, half_max(mx));
        const float f = __builtin_amdgcn_exp2f((m - mx) * a.c);
        m = mx, l *= f, pd *= f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float p = __builtin_amdgcn_exp2f((s[i] - m) * a.c);
          l += p, pd += p * dp[i];
        }
        return true;
      });
    });
    if (n & 1) fr.flip(2 * TB);
    lds_pipeline_barrier();  // every wave has read the last tile
    if (there) bits = first, next = 0;  // it lies in the first buffer still, and no other tile has a key
    else if (t0 < t1) start(KeyMask<KT>{mask, end}, t0, t0 + 1);
    l = half_sum(l), pd = half_sum(pd);
    if (l > 0.f) {
      const RowRef ref = row_ref(m, a.c);
      const float ll = __builtin_amdgcn_logf(l);
      shift = ref.a, x = ref.a != 0.f ? ll : __builtin_fmaf(m, a.c, ll), delta = pd / l;
    } else {
      x = l != l ? l : INFINITY;
    }
  }
  f32x16 dq[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) dq[d][i] = 0.f;
  auto step = [&](auto shifted, uint64_t bits) __attribute__((always_inline)) {
    static_for<KT / 32>([&](auto block) __attribute__((always_inline)) {
      constexpr int kb = decltype(block)::value;
      f32x16 s, dp;
      scores(block, bits, s, dp);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float ds = decltype(shifted)::value ? s[i] - shift : s[i];
        s[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(ds, a.c, -x)) * (dp[i] - delta);
      }
      static_for<2>([&](auto ks) __attribute__((always_inline)) {
        Frag<T> ds, rest;
        to_frag(s, ks, ds);
        if constexpr (FINE) rest_frag(s, ks, ds, rest);
#pragma unroll
        for (int d = 0; d < ND; ++d) {
          Frag<T> kf;
          fr.template cols<0, 32 * kb + 16 * decltype(ks)::value>(d, kf);
          dq[d] = mma16(kf, ds, dq[d]);
          if constexpr (FINE) dq[d] = mma16(kf, rest, dq[d]);
        }
        return true;
      });
      return true;
    });
  };
  // a loop each: a branch between a block's products and its exponentials would keep the next block's out of them
  const KeyMask<KT> km{mask, end};
  if (__any(shift != 0.f)) sweep(km, t0, t1, same, [&](uint64_t bits) __attribute__((always_inline)) { step(std::true_type{}, bits); });
  else sweep(km, t0, t1, same, [&](uint64_t bits) __attribute__((always_inline)) { step(std::false_type{}, bits); });
  if (lane < 32 && r < a.rows && sp == 0) {
    const int64_t all = (int64_t)a.batches * a.Hk * a.rows;
    float *p = ba.stats + head_rows + r;
    p[0] = x, p[all] = delta, p[2 * all] = shift;
  }
  if (a.splits > 1) {
    f32x4 *p = ba.part + ((((int64_t)sp * a.batches + b) * a.row_tiles + rt) * a.Hk + hk) * (NW * ND * 4 * 64) + wave * (ND * 4 * 64) + lane;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *(MLORA_GLOBAL f32x4 *)(p + (d * 4 + i) * 64) = f32x4{dq[d][4 * i], dq[d][4 * i + 1], dq[d][4 * i + 2], dq[d][4 * i + 3]};
    return;
  }
  const float f[1] = {ba.scale};
  f32x16 o[1][ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) o[0][d] = dq[d];
  store_rows<T, DP, 1>(static_cast<T *>(ba.dq) + oat, o, f, row0, a.rows,
                       [&](int r) { return row_at(r, a.Lq, (int64_t)a.H * a.D, a.D); }, a.D, lane);
}

// Adds the splits of dq in split order and writes them out.
template <class T, int DP, int NW>
__global__ __launch_bounds__(256) void attn_dq_join_kernel(const AttnBwdArgs ba) {
  const AttnArgs &a = ba.f;
  constexpr int ND = DP / 32;
  const int64_t per = (int64_t)a.batches * a.row_tiles * a.Hk * NW * ND * 4 * 64;
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;  // per is a multiple of 256
  int64_t u = e / 64;
  const int lane = (int)(e % 64), i = (int)(u % 4), d = (int)(u / 4 % ND), wave = (int)(u / 4 / ND % NW);
  u /= 4 * ND * NW;  // (b, row tile, hk)
  const int hk = (int)(u % a.Hk), r = (int)(u / a.Hk % a.row_tiles) * (32 * NW) + wave * 32 + (lane & 31);
  const int64_t b = u / a.Hk / a.row_tiles;
  const int ch = 32 * d + 8 * i + 4 * (lane >> 5);
  if (r >= a.rows || ch >= a.D) return;
  f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = 0; s < a.splits; ++s) x += *(const MLORA_GLOBAL f32x4 *)(ba.part + s * per + e);
  x *= ba.scale;
  T *p = static_cast<T *>(ba.dq) + (b * a.Lq * a.H + (int64_t)hk * a.G) * a.D + row_at(r, a.Lq, (int64_t)a.H * a.D, a.D) + ch;
  if constexpr (sizeof(T) == 2) *(MLORA_GLOBAL u32x2 *)p = u32x2{pack2_bf16(x[0], x[1]), pack2_bf16(x[2], x[3])};
  else *(MLORA_GLOBAL f32x4 *)p = x;
}

// NW waves own 32 keys each (K fragments in registers; V in LDS for bf16, whose two waves per SIMD leave no room
// for them) and share tiles of QT query rows of one head in LDS, double-buffered: q, the output's gradient and the rows'
// x, delta and a (the last read only in a tile that has one: a flag per buffer says so).
template <class T, int DP, int NW>
struct DkvTile {  // query rows per tile: half as many where that leaves room for another workgroup
  static constexpr int QT = sizeof(T) == 2 && !(DP == 128 && NW == 4) ? 64 : 32;
};

template <class T, int DP, int NW, bool FINE>
__global__ __launch_bounds__((64 * NW), (sizeof(T) == 2 ? 2 : 1)) void attn_dkv_kernel(const AttnBwdArgs ba) {
  const AttnArgs &a = ba.f;
  constexpr int QT = DkvTile<T, DP, NW>::QT, ND = DP / 32, NS = DP / 16;
  constexpr bool VLDS = sizeof(T) == 2;
  using Tile = HeadTile<T, DP>;
  constexpr int TB = QT * Tile::RB, N = TB / 1024 / NW, VB = VLDS ? 32 * Tile::RB : 0;
  // one array, so that the readers' buffers start at a multiple of 4 TB; then V, then x, delta and a per buffer and a flag
  // for each
  static_assert(64 * NW >= 3 * QT, "a thread loads one of a row's three values");
  __shared__ u32x4 smem[(4 * TB + NW * VB) / 16 + 3 * QT / 2 + 1];
  f32x4 (&stats)[2][3][QT / 4] = *(f32x4 (*)[2][3][QT / 4])(smem + (4 * TB + NW * VB) / 16);
  int *tile_far = (int *)(smem + (4 * TB + NW * VB) / 16 + 3 * QT / 2);
  MLORA_LDS char *lds = (MLORA_LDS char *)smem;
  const int wave = wave_id(), lane = threadIdx.x & 63;
  int id = blockIdx.x;  // heads first, as above
  const int hk = id % a.Hk;
  id /= a.Hk;
  const int kb = id % ba.key_blocks;
  id /= ba.key_blocks;
  const int sp = id % ba.q_splits, b = id / ba.q_splits;
  const int len = sample_keys(a, b);
  const int key0 = (kb * NW + wave) * 32, key = key0 + (lane & 31);
  const uint8_t *mask = a.mask == nullptr ? nullptr : a.mask + b * a.mask_sb;
  const bool live = key < len && (mask == nullptr || mask[key] != 0);
  const uint64_t live_bits = __ballot(live) & 0xffffffffull;
  const T *kp = static_cast<const T *>(a.k) + b * a.k_sb + hk * a.k_sh;
  const T *vp = static_cast<const T *>(a.v) + b * a.v_sb + hk * a.v_sh;
  Frag<T> k[NS], v[VLDS ? 1 : NS];
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    const int d = 16 * s + 8 * (lane >> 5);
    load_frag(kp, key * a.k_sl + d, live && d < a.D, k[s]);
    if constexpr (!VLDS) load_frag(vp, key * a.v_sl + d, live && d < a.D, v[s]);
  }
  MLORA_LDS char *vt = lds + 4 * TB + wave * VB;
  if constexpr (VLDS) {
    TileLoader<T, DP, VB / 1024> vl;
    vl.init(lane, 0, 1, a.v_sl, a.D);
    vl.load(vp + (int64_t)key0 * a.v_sl, live_bits, vt);
  }
  f32x16 dk[1][ND], dv[1][ND];
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) dk[0][d][i] = 0.f, dv[0][d][i] = 0.f;
  const int t0 = sp * ba.q_split_tiles;
  const int t1 = kb * 32 * NW >= len ? 0 : min(t0 + ba.q_split_tiles, ba.q_tiles);  // no key at all: zeros
  TileLoader<T, DP, N> ql, gl;
  ql.init(lane, wave, NW, a.q_sl, a.D), gl.init(lane, wave, NW, ba.g_sl, a.D);
  const int64_t head_rows = ((int64_t)b * a.Hk + hk) * a.rows, all = (int64_t)a.batches * a.Hk * a.rows;
  FragReader<T, DP> fr, vr;
  fr.init(lane, lds), vr.init(lane, vt);
  // a tile's rows into LDS; returns x (threads 0 .. QT - 1), delta (QT .. 2 QT - 1) or a (.. 3 QT - 1) of the thread's row
  auto stage = [&](int t, int buf) __attribute__((always_inline)) -> float {
    const int g = t / ba.head_q_tiles, i0 = (t - g * ba.head_q_tiles) * QT, h = hk * a.G + g;
    const uint64_t rows = t < t1 ? low_bits(min(a.Lq - i0, QT)) : 0;  // past the last tile: nothing is read
    ql.load(static_cast<const T *>(a.q) + b * a.q_sb + h * a.q_sh + i0 * a.q_sl, rows, lds + buf * 2 * TB);
    gl.load(static_cast<const T *>(ba.g) + b * ba.g_sb + h * ba.g_sh + i0 * ba.g_sl, rows, lds + buf * 2 * TB + TB);
    const int i = threadIdx.x % QT, which = threadIdx.x / QT;
    float x = which == 0 ? INFINITY : 0.f;  // rows behind the last: P = 0
    if (which < 3 && t < t1 && i0 + i < a.Lq) x = ba.stats[which * all + head_rows + (int64_t)g * a.Lq + i0 + i];
    return x;
  };
  auto keep = [&](int buf, float x) __attribute__((always_inline)) {
    if (threadIdx.x < 3 * QT) ((float *)stats[buf][threadIdx.x / QT])[threadIdx.x % QT] = x;
    const bool far = __any(threadIdx.x / QT == 2 && x != 0.f);  // the threads with a's are lanes of one wave
    if (threadIdx.x == 2 * QT) tile_far[buf] = far;
  };
  auto step = [&](int buf) __attribute__((always_inline)) {
    const int far = __builtin_amdgcn_readfirstlane(tile_far[buf]);  // a scalar: kept in a vector register it spills (+10 %)
    static_for<QT / 32>([&](auto block) __attribute__((always_inline)) {
      constexpr int qb = decltype(block)::value;
      __builtin_amdgcn_sched_barrier(0);  // between the phases too: interleaved, they spill
      f32x16 s, dp;
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = 0.f, dp[i] = 0.f;
#pragma unroll
      for (int ks = 0; ks < NS; ++ks) {  // the two sums in turn: a sum waits for its last product
        Frag<T> qf, gf, vf;
        fr.template rows<0, 32 * qb>(ks, qf);
        s = mma16(qf, k[ks], s);
        fr.template rows<TB, 32 * qb>(ks, gf);
        if constexpr (VLDS) vr.template rows<0, 0>(ks, vf);
        else vf = v[ks];
        dp = mma16(gf, vf, dp);
      }
      __builtin_amdgcn_sched_barrier(0);
      if (far) {
#pragma unroll
        for (int i4 = 0; i4 < 4; ++i4) {
          const f32x4 shift = stats[buf][2][8 * qb + 2 * i4 + (lane >> 5)];
#pragma unroll
          for (int j = 0; j < 4; ++j) s[4 * i4 + j] -= shift[j];
        }
      }
#pragma unroll
      for (int i4 = 0; i4 < 4; ++i4) {
        const f32x4 x = stats[buf][0][8 * qb + 2 * i4 + (lane >> 5)], delta = stats[buf][1][8 * qb + 2 * i4 + (lane >> 5)];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[4 * i4 + j], a.c, -x[j]));
          s[4 * i4 + j] = p;
          dp[4 * i4 + j] = p * (dp[4 * i4 + j] - delta[j]);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      static_for<2>([&](auto ks) __attribute__((always_inline)) {
        Frag<T> pf, rest;
        to_frag(s, ks, pf);
        if constexpr (FINE) rest_frag(s, ks, pf, rest);
#pragma unroll
        for (int d = 0; d < ND; ++d) {
          Frag<T> f;
          fr.template cols<TB, 32 * qb + 16 * decltype(ks)::value>(d, f);
          dv[0][d] = mma16(f, pf, dv[0][d]);
          if constexpr (FINE) dv[0][d] = mma16(f, rest, dv[0][d]);
        }
        return true;
      });
      static_for<2>([&](auto ks) __attribute__((always_inline)) {
        Frag<T> df, rest;
        to_frag(dp, ks, df);
        if constexpr (FINE) rest_frag(dp, ks, df, rest);
#pragma unroll
        for (int d = 0; d < ND; ++d) {
          Frag<T> f;
          fr.template cols<0, 32 * qb + 16 * decltype(ks)::value>(d, f);
          dk[0][d] = mma16(f, df, dk[0][d]);
          if constexpr (FINE) dk[0][d] = mma16(f, rest, dk[0][d]);
        }
        return true;
      });
      return true;
    });
  };
  if (t0 < t1) keep(0, stage(t0, 0));
  for (int t = t0; t < t1; ++t) {
    const int buf = (t - t0) & 1;
    wait_vmcnt<0>();
    lds_pipeline_barrier();  // tile t is in LDS, and every wave has read tile t - 1
    const float x = stage(t + 1, buf ^ 1);
    if (live_bits != 0) step(buf);
    keep(buf ^ 1, x);
    fr.flip(2 * TB);
  }
  wait_vmcnt<0>();
  if (!live) {  // a masked key's column holds whatever its zeroed fragments gave
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) dk[0][d][i] = 0.f, dv[0][d][i] = 0.f;
  }
  if (ba.q_splits > 1) {
    f32x4 *p = ba.part + (((((int64_t)sp * a.batches + b) * a.Hk + hk) * ba.key_blocks + kb) * NW + wave) * (2 * ND * 4 * 64) + lane;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        *(MLORA_GLOBAL f32x4 *)(p + (d * 4 + i) * 64) = f32x4{dk[0][d][4 * i], dk[0][d][4 * i + 1], dk[0][d][4 * i + 2], dk[0][d][4 * i + 3]};
        *(MLORA_GLOBAL f32x4 *)(p + ((ND + d) * 4 + i) * 64) = f32x4{dv[0][d][4 * i], dv[0][d][4 * i + 1], dv[0][d][4 * i + 2], dv[0][d][4 * i + 3]};
      }
    return;
  }
  const int64_t at = ((int64_t)b * a.Lk * a.Hk + hk) * a.D;
  const float fk[1] = {ba.scale}, fv[1] = {1.f};
  auto key_at = [&](int key) { return (int64_t)key * a.Hk * a.D; };
  store_rows<T, DP, 1>(static_cast<T *>(ba.dk) + at, dk, fk, key0, a.Lk, key_at, a.D, lane);
  store_rows<T, DP, 1>(static_cast<T *>(ba.dv) + at, dv, fv, key0, a.Lk, key_at, a.D, lane);
}

// Adds the splits of dk and dv in split order and writes them out.
template <class T, int DP, int NW>
__global__ __launch_bounds__(256) void attn_dkv_join_kernel(const AttnBwdArgs ba) {
  const AttnArgs &a = ba.f;
  constexpr int ND = DP / 32;
  const int64_t per = (int64_t)a.batches * a.Hk * ba.key_blocks * NW * 2 * ND * 4 * 64;
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (e >= per) return;
  f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = 0; s < ba.q_splits; ++s) x += *(const MLORA_GLOBAL f32x4 *)(ba.part + s * per + e);
  int64_t u = e / 64;
  const int lane = (int)(e % 64), i = (int)(u % 4), d = (int)(u / 4 % ND), which = (int)(u / 4 / ND % 2);
  u /= 4 * ND * 2;  // (b, hk, key block, wave)
  const int64_t key = u % (NW * ba.key_blocks) * 32 + (lane & 31), bh = u / (NW * ba.key_blocks);
  const int ch = 32 * d + 8 * i + 4 * (lane >> 5);
  if (key >= a.Lk || ch >= a.D) return;
  T *p = static_cast<T *>(which ? ba.dv : ba.dk) + ((bh / a.Hk * a.Lk + key) * a.Hk + bh % a.Hk) * a.D + ch;
  if (!which) x *= ba.scale;
  if constexpr (sizeof(T) == 2) *(MLORA_GLOBAL u32x2 *)p = u32x2{pack2_bf16(x[0], x[1]), pack2_bf16(x[2], x[3])};
  else *(MLORA_GLOBAL f32x4 *)p = x;
}

// The kernels are named here because hipcc's host pass does not instantiate a kernel that holds generic lambdas
// from a launch inside one.
#define MLORA_ATTN(T, DP)                                                       \
  template __global__ void attn_fwd_kernel<T, DP, false>(const AttnArgs);       \
  template __global__ void attn_few_kernel<T, DP, 1>(const AttnArgs);           \
  template __global__ void attn_dq_kernel<T, DP, 4, false>(const AttnBwdArgs);  \
  template __global__ void attn_dkv_kernel<T, DP, 4, false>(const AttnBwdArgs);
MLORA_ATTN(uint16_t, 64)
MLORA_ATTN(uint16_t, 128)
MLORA_ATTN(float, 64)
MLORA_ATTN(float, 128)
#undef MLORA_ATTN
template __global__ void attn_fwd_kernel<uint16_t, 64, true>(const AttnArgs);
template __global__ void attn_fwd_kernel<uint16_t, 128, true>(const AttnArgs);
template __global__ void attn_few_kernel<uint16_t, 64, 2>(const AttnArgs);
template __global__ void attn_few_kernel<uint16_t, 128, 2>(const AttnArgs);
template __global__ void attn_few_kernel<float, 64, 2>(const AttnArgs);
template __global__ void attn_dkv_kernel<uint16_t, 128, 8, false>(const AttnBwdArgs);
template __global__ void attn_dq_kernel<uint16_t, 64, 4, true>(const AttnBwdArgs);
template __global__ void attn_dq_kernel<uint16_t, 128, 4, true>(const AttnBwdArgs);
template __global__ void attn_dq_kernel<float, 64, 2, false>(const AttnBwdArgs);
template __global__ void attn_dq_kernel<float, 128, 2, false>(const AttnBwdArgs);
template __global__ void attn_dkv_kernel<float, 64, 2, false>(const AttnBwdArgs);
template __global__ void attn_dkv_kernel<float, 128, 2, false>(const AttnBwdArgs);
template __global__ void attn_dkv_kernel<uint16_t, 64, 4, true>(const AttnBwdArgs);
template __global__ void attn_dkv_kernel<uint16_t, 128, 4, true>(const AttnBwdArgs);
template __global__ void attn_dkv_kernel<uint16_t, 128, 8, true>(const AttnBwdArgs);

// ------------------------------------------------------------------ host

constexpr int kAttnMaxHeadDim = 128;

struct AttnPlan {
  bool few;
  int nq;  // 32-row blocks per wave
  int64_t row_tiles, turns, splits, split_tiles;
};

// Row tiles per workgroup: up to 4 where few key tiles leave a workgroup mostly waiting for its first loads and
// at least 1024 workgroups (two for every place) remain. 2 x 32760 rows of 12 heads of 128: 512 keys 285 us with
// one, 263 with four; 64 keys 141 and 120; 1024 keys 494 and 451; at 4096 keys one row's tile is best (819, 909; minima).
static int64_t row_turns(int64_t tiles, int64_t key_tiles) {
  const int64_t most = key_tiles <= 16 ? 4 : 1, turns = tiles / 1024;
  return turns < 1 ? 1 : turns > most ? most : turns;
}

// How a forward is cut: few rows per key head run waves over different keys, more rows 128 per workgroup;
// the keys are split where that leaves less than a workgroup for every compute unit and there are enough of them:
// a float32 tile takes about as long as a join, a bf16 tile a sixth of it (2 x 64 rows x 512 keys, 12 heads of 128,
// float32: 47 us where a split takes 8 tiles at least, 31 with 4, 23 with 2; bf16 14.7, 16.3 and 15.6). 129 to 255
// workgroups stay whole, and a second place per compute unit, which bf16 and float32 up to 64 channels have, is not
// counted: one frame of 1560 rows, 12 heads of 128, is 156 workgroups (9360 keys 245 us, 62 at the matrix cores' rate;
// 32760 keys 799 and 217).
static AttnPlan attn_plan(int64_t batches, int64_t rows, int64_t Lk, int64_t Hk, int64_t D, bool f32) {
  AttnPlan p{};
  p.few = rows <= (f32 && D > 64 ? 32 : 64);
  const int64_t waves = p.few && f32 && D > 64 ? 2 : 4;
  const int64_t kt = p.few || f32 ? 32 : 64, tiles = (Lk + kt - 1) / kt;
  p.nq = p.few && rows > 32 ? 2 : 1;
  p.row_tiles = p.few ? 1 : (rows + 127) / 128;
  p.turns = p.few ? 1 : row_turns(batches * Hk * p.row_tiles, tiles);
  const int64_t groups = batches * Hk * p.row_tiles;
  const int64_t least = p.few ? (f32 ? waves : 4 * waves) : f32 ? 2 : 8;  // tiles that a split is worth its join for
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

struct DqPlan {
  int nw;  // waves per workgroup, 32 rows each
  int64_t row_tiles, splits, split_tiles;
};

// dq: 32 nw rows per workgroup, two waves for up to 64 float32 rows (a wave without rows holds its SIMD's one
// place: 4 x 2 rows x 4779 keys, 12 heads of 128: the backward 433 us with four, 335 with two). The keys are
// split where the rows alone leave places for workgroups free (bf16, 300 rows x 8192 keys, 8 heads of 128: the
// backward takes 72 us, unsplit 226), four tiles at least to a split for bf16, one for float32 (200 rows x 300
// keys, 16 heads of 64: bf16 20 us, with one tile 24; float32 41, with four 66).
static DqPlan dq_plan(int64_t batches, int64_t rows, int64_t Lk, int64_t Hk, bool f32) {
  DqPlan p{};
  p.nw = f32 && rows <= 64 ? 2 : 4;
  p.row_tiles = (rows + 32 * p.nw - 1) / (32 * p.nw);
  const int64_t kt = f32 ? AttnTile<float>::KT : AttnTile<uint16_t>::KT, tiles = (Lk + kt - 1) / kt;
  const int64_t groups = batches * Hk * p.row_tiles, most = f32 && p.nw == 4 ? 256 : 512;
  int64_t splits = groups > 0 && groups < most ? most / groups : 1;
  const int64_t least = f32 ? 1 : 4;
  if (splits > tiles / least) splits = tiles / least;
  if (splits < 1) splits = 1;
  p.split_tiles = (tiles + splits - 1) / splits;
  if (p.split_tiles < 1) p.split_tiles = 1;
  p.splits = tiles > 0 ? (tiles + p.split_tiles - 1) / p.split_tiles : 1;
  return p;
}

// 16-byte vectors of one split of dq, in register order.
static int64_t dq_vectors(const DqPlan &p, int64_t batches, int64_t Hk, int64_t D) {
  return batches * p.row_tiles * Hk * p.nw * (D > 64 ? 4 : 2) * 4 * 64;
}

struct DkvPlan {
  int nw;  // waves per workgroup, 32 keys each
  int64_t key_blocks, q_tiles, head_q_tiles, splits, split_tiles;
};

// dk / dv: 32 nw keys per workgroup. float32 takes 2 waves where they hold all keys: a wave without keys holds
// its SIMD's one place until its workgroup ends (3 x 3074 rows x 12 keys, 40 heads of 80: 527 us with 4 waves,
// 322 with 2; bf16, with two waves per SIMD, gains nothing: the backward of 2 x 8000 x 64, 16 heads of 64, 65
// and 75). The query rows are split where the keys alone leave compute units idle, with dq's least numbers of
// tiles. Where a compute unit holds one workgroup, also beyond 256 of them: a last round that is nearly empty
// costs as much as a full one. The number of splits is the one with the least estimated time, of the rounds at
// 4 TFLOP/s (float32: 0.45) per compute unit and of writing and reading the splits at 5 TB/s (32760 rows x 4096
// keys, 12 heads of 128, bf16, 192 workgroups unsplit: the backward 2911 us, with 4 splits 2699; 8192 x 8192,
// 10 heads, 320 workgroups: 1415 and 1263; float32, 2 x 32760 x 512, 12 heads: 8465 and 7085).
static DkvPlan dkv_plan(int64_t batches, int64_t Lq, int64_t Lk, int64_t Hk, int64_t G, int64_t D, bool f32) {
  DkvPlan p{};
  p.nw = f32 ? (Lk <= 64 ? 2 : 4) : D > 64 && Lk > 128 ? 8 : 4;
  const int64_t qt = f32 || (D > 64 && p.nw == 4) ? 32 : 64, dp = D > 64 ? 128 : 64;
  p.key_blocks = (Lk + 32 * p.nw - 1) / (32 * p.nw);
  p.head_q_tiles = (Lq + qt - 1) / qt;
  p.q_tiles = G * p.head_q_tiles;
  const int64_t groups = batches * Hk * p.key_blocks;
  const int64_t most_splits = p.q_tiles / (f32 ? 1 : 4);
  int64_t splits = 1;
  if (!f32 && p.nw == 4) {
    if (groups > 0 && groups < 512) splits = 512 / groups;  // two workgroups per compute unit
    if (splits > most_splits) splits = most_splits;
  } else if (groups > 0) {
    const int64_t places = p.nw == 2 ? 512 : 256;
    const double tile_us = 8e-6 * (double)(qt * 32 * p.nw * dp) / (f32 ? 0.45 : 4.0) * (double)places / 256.0;
    const double split_us = (double)(groups * p.nw * 64 * dp) * 4.0 * 2.0 / 5e6;  // dk and dv, out and in
    double best = 0.0;
    for (int64_t n = 1; n <= most_splits && n * groups <= 2048; ++n) {  // 512 MB of splits at most
      const double us = (double)((groups * n + places - 1) / places * ((p.q_tiles + n - 1) / n)) * tile_us + (n > 1 ? (double)n * split_us : 0.0);
      if (n == 1 || us < 0.97 * best) best = us, splits = n;
    }
  }
  if (splits < 1) splits = 1;
  p.split_tiles = (p.q_tiles + splits - 1) / splits;
  if (p.split_tiles < 1) p.split_tiles = 1;
  p.splits = p.q_tiles > 0 ? (p.q_tiles + p.split_tiles - 1) / p.split_tiles : 1;
  return p;
}

// 16-byte vectors of one split of dk and dv, in register order.
static int64_t dkv_vectors(const DkvPlan &p, int64_t batches, int64_t Hk, int64_t D) {
  return batches * Hk * p.key_blocks * p.nw * 2 * (D > 64 ? 4 : 2) * 4 * 64;
}

// The splits of dq, and after they are joined those of dk and dv in the same place.
static int64_t bwd_part_bytes(const DqPlan &q, const DkvPlan &p, int64_t batches, int64_t Hk, int64_t D) {
  const int64_t dq = q.splits > 1 ? q.splits * dq_vectors(q, batches, Hk, D) * 16 : 0;
  const int64_t dkv = p.splits > 1 ? p.splits * dkv_vectors(p, batches, Hk, D) * 16 : 0;
  return dq > dkv ? dq : dkv;
}

// Whether the backward's products take P and dS in two bf16 parts, and the forward's lse the sum that goes with them: a
// matter of one sample's sizes, so that its gradients do not depend on the batch it is in.
static bool fine_call(int64_t H, int64_t Lq, int64_t Lk, int64_t D) {
  return (double)H * (double)Lq * (double)Lk * (double)D <= 1073741824.0;
}

// Sizes and types shared by every entry. MLORA_OK, or the status.
static int attn_sizes(int dtype, int64_t B, int64_t Lq, int64_t Lk, int64_t H, int64_t Hk, int64_t D) {
  if (dtype != MLORA_BF16 && dtype != MLORA_F32) return MLORA_ERR_UNSUPPORTED;
  if (B < 0 || Lq < 0 || Lk < 0 || H < 1 || Hk < 1 || H % Hk != 0) return MLORA_ERR_INVALID;
  if (D < 8 || D % 8 != 0 || D > kAttnMaxHeadDim) return MLORA_ERR_UNSUPPORTED;
  const int64_t most = INT32_MAX - 65536;
  if (H > most || Lk > most || (Lq > 0 && H > most / Lq)) return MLORA_ERR_LIMIT;  // rows per key head
  // workgroups: one per (sample, key head, 128 rows or keys), splits up to 2048 of them
  const int64_t blocks = (H / Hk * Lq + 127) / 128 + (Lk + 127) / 128 + 2048;
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
  if (!(scale > 0.f && scale * kLog2e < INFINITY) || qs == nullptr || ks == nullptr || vs == nullptr || mask_sb < 0)
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
  a.out = out, a.row_tiles = (int32_t)p.row_tiles, a.turns = (int32_t)p.turns, a.splits = (int32_t)p.splits, a.split_tiles = (int32_t)p.split_tiles;
  a.part_o = static_cast<float *>(workspace);
  a.part_ml = a.part_o + p.splits * B * Hk * a.rows * D;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const dim3 grid((unsigned)(B * Hk * ((p.row_tiles + p.turns - 1) / p.turns) * p.splits));
  with_head(f32, D, [&](auto t, auto dp) {
    using T = decltype(t);
    constexpr int DP = decltype(dp)::value;
    if (p.few && p.nq == 1) hipLaunchKernelGGL((attn_few_kernel<T, DP, 1>), grid, dim3(64 * FewTile<T, DP>::NW), 0, s, a);
    else if (!p.few) {
      if constexpr (sizeof(T) == 2) {
        if (fine_call(H, Lq, Lk, D)) {
          hipLaunchKernelGGL((attn_fwd_kernel<T, DP, true>), grid, dim3(256), 0, s, a);
          return;
        }
      }
      hipLaunchKernelGGL((attn_fwd_kernel<T, DP, false>), grid, dim3(256), 0, s, a);
    }
    else if constexpr (sizeof(T) * DP < 512)
      hipLaunchKernelGGL((attn_few_kernel<T, DP, 2>), grid, dim3(64 * FewTile<T, DP>::NW), 0, s, a);
  });
  st = launch_status();
  if (st || p.splits == 1) return st;
  const dim3 joins((unsigned)(B * Hk * a.rows));
  if (f32) hipLaunchKernelGGL(attn_join_kernel<float>, joins, dim3(256), 0, s, a);
  else hipLaunchKernelGGL(attn_join_kernel<uint16_t>, joins, dim3(256), 0, s, a);
  return launch_status();
}

extern "C" int64_t mlora_cross_attention_backward_workspace_bytes(int dtype, int64_t B, int64_t Lq, int64_t Lk, int64_t H,
                                                                  int64_t Hk, int64_t D) {
  const int st = attn_sizes(dtype, B, Lq, Lk, H, Hk, D);
  if (st) return st;
  // three values of every row, rounded up to whole 16-byte vectors, then the splits
  const bool f32 = dtype == MLORA_F32;
  return (3 * B * H * Lq + 3) / 4 * 16 +
         bwd_part_bytes(dq_plan(B, H / Hk * Lq, Lk, Hk, f32), dkv_plan(B, Lq, Lk, Hk, H / Hk, D, f32), B, Hk, D);
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
  ba.dq = dq, ba.dk = dk, ba.dv = dv, ba.stats = static_cast<float *>(workspace);
  ba.part = static_cast<f32x4 *>(workspace) + (3 * B * H * Lq + 3) / 4;
  ba.key_blocks = (int32_t)p.key_blocks, ba.q_tiles = (int32_t)p.q_tiles, ba.head_q_tiles = (int32_t)p.head_q_tiles;
  ba.q_splits = (int32_t)p.splits, ba.q_split_tiles = (int32_t)p.split_tiles;
  const DqPlan qp = dq_plan(B, a.rows, Lk, Hk, f32);
  a.row_tiles = (int32_t)qp.row_tiles, a.splits = (int32_t)qp.splits, a.split_tiles = (int32_t)qp.split_tiles;
  const bool fine = fine_call(H, Lq, Lk, D);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (Lq > 0) {
    with_head(f32, D, [&](auto t, auto dp) {
      using T = decltype(t);
      constexpr int DP = decltype(dp)::value;
      const dim3 grid((unsigned)(B * Hk * a.row_tiles * qp.splits)), joins((unsigned)(dq_vectors(qp, B, Hk, D) / 256));
      if constexpr (sizeof(T) == 4) {
        if (qp.nw == 2) {
          hipLaunchKernelGGL((attn_dq_kernel<T, DP, 2, false>), grid, dim3(128), 0, s, ba);
          if (qp.splits > 1) hipLaunchKernelGGL((attn_dq_join_kernel<T, DP, 2>), joins, dim3(256), 0, s, ba);
          return;
        }
      } else if (fine) {
        hipLaunchKernelGGL((attn_dq_kernel<T, DP, 4, true>), grid, dim3(256), 0, s, ba);
      }
      if (sizeof(T) == 4 || !fine) hipLaunchKernelGGL((attn_dq_kernel<T, DP, 4, false>), grid, dim3(256), 0, s, ba);
      if (qp.splits > 1) hipLaunchKernelGGL((attn_dq_join_kernel<T, DP, 4>), joins, dim3(256), 0, s, ba);
    });
    st = launch_status();
    if (st) return st;
  }
  if (Lk == 0) return MLORA_OK;
  const dim3 grid((unsigned)(B * Hk * p.key_blocks * p.splits));
  const dim3 joins((unsigned)((dkv_vectors(p, B, Hk, D) + 255) / 256));
  with_head(f32, D, [&](auto t, auto dp) {
    using T = decltype(t);
    constexpr int DP = decltype(dp)::value;
    if constexpr (sizeof(T) == 2 && DP == 128) {
      if (p.nw == 8) {
        if (fine) hipLaunchKernelGGL((attn_dkv_kernel<T, DP, 8, true>), grid, dim3(512), 0, s, ba);
        else hipLaunchKernelGGL((attn_dkv_kernel<T, DP, 8, false>), grid, dim3(512), 0, s, ba);
        if (p.splits > 1) hipLaunchKernelGGL((attn_dkv_join_kernel<T, DP, 8>), joins, dim3(256), 0, s, ba);
        return;
      }
    }
    auto go = [&](auto nw) {
      constexpr int NW = decltype(nw)::value;
      if constexpr (sizeof(T) == 2) {
        if (fine) hipLaunchKernelGGL((attn_dkv_kernel<T, DP, NW, true>), grid, dim3(64 * NW), 0, s, ba);
        else hipLaunchKernelGGL((attn_dkv_kernel<T, DP, NW, false>), grid, dim3(64 * NW), 0, s, ba);
      } else {
        hipLaunchKernelGGL((attn_dkv_kernel<T, DP, NW, false>), grid, dim3(64 * NW), 0, s, ba);
      }
      if (p.splits > 1) hipLaunchKernelGGL((attn_dkv_join_kernel<T, DP, NW>), joins, dim3(256), 0, s, ba);
    };
    if constexpr (sizeof(T) == 4) {
      if (p.nw == 2) return go(std::integral_constant<int, 2>{});
    }
    go(std::integral_constant<int, 4>{});
  });
  return launch_status();
}
