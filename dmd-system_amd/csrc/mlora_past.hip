// Attention of a stream's tokens to their own past: a window, the first tokens, a prefix that samples share.
//
// A query at position p of a sample with n keys, chunks of C tokens, a window of W and S sinks sees its sample's keys
//   j < min(e, n) with j >= e − W or j < S,   e = (⌊p / C⌋ + 1)·C the end of its chunk,
// and all keys of its group's prefix. out = Σ_j P_j v_j, P = softmax(scale · q·k_j) over the keys that it sees; queries
// with p < 0 or p >= n belong to no token and get zeros.
//
// One pass over the key tiles that some row of a workgroup sees: the prefix's, the sinks', then the window's from its first
// tile on, with a running maximum and sum per row (Softmax). Everything between them is never read. Only the tiles at the edges of
// a wave's rows need masks; keys that no row of the workgroup sees are loaded as zeros, whatever lies there.
//
// Rows: the G = heads / kv_heads query heads that share a key head are packed token by token, row r = i·G + g of token i,
// so that 32 rows are 32 / G neighbouring tokens and see almost the same keys.
#include "mlora_attention.h"

#include <algorithm>

namespace mlora {

struct PastArgs {
  const void *q, *k, *v, *pk, *pv;
  void *out;        // [B, Lq, H, D] contiguous
  uint16_t *rest;   // bf16 and a backward to come: what out's rounding left, [B, Lq, H, D]
  float *stats;     // a backward to come: [2][B·Hk·rows], x and a of every row: P = 2^((s − a)·c − x)
  const int32_t *lengths, *starts, *prefix_lengths;
  float *part_o, *part_ml;  // [slots][B·Hk·rows][D] sums and [slots][B·Hk·rows][2] (m, l)
  int64_t q_sb, q_sl, q_sh, k_sb, k_sl, k_sh, v_sb, v_sl, v_sh, pk_sb, pk_sl, pk_sh, pv_sb, pv_sl, pv_sh;
  int32_t B, Lq, Lk, H, Hk, G, D, Lp, each;  // each: samples per prefix
  int32_t window, sinks, chunk, first, from_end, rows;
  int32_t packed_blocks;  // workgroups at the grid's start that take the prefix alone, for the rows of all its samples
  int32_t packed_tiles, packed_splits, row_tiles, splits, slots;
  int32_t with_prefix;    // the other workgroups take the prefix too
  float c;                // scale · log2 e
};

constexpr int kEver = 1 << 30;  // past every position; lengths, windows and chunks are limited so that sums of two stay in int32

struct Sample {
  int n, start;  // its keys; the position of its first query
};
__device__ __forceinline__ Sample sample_of(const PastArgs &a, int b) {
  Sample s;
  s.n = a.lengths == nullptr ? a.Lk : min(max(a.lengths[b], 0), a.Lk);
  const int first = a.starts != nullptr ? a.starts[b] : a.from_end ? s.n - a.Lq : a.first;
  s.start = min(max(first, -a.Lq), a.Lk);  // beyond these no query has a token
  return s;
}
__device__ __forceinline__ Sample uniform(const Sample &s) {
  return {__builtin_amdgcn_readfirstlane(s.n), __builtin_amdgcn_readfirstlane(s.start)};
}
__device__ __forceinline__ int prefix_keys(const PastArgs &a, int group) {
  if (a.prefix_lengths == nullptr) return a.Lp;
  return __builtin_amdgcn_readfirstlane(min(max(a.prefix_lengths[group], 0), a.Lp));
}

// The own keys [lo, hi) that a token sees beside the sinks; lo may be negative.
struct Span {
  int lo, hi;
};
__device__ __forceinline__ Span span_of(const PastArgs &a, int n, int p) {
  const int end = (int)((uint32_t)p / (uint32_t)a.chunk + 1) * a.chunk;
  return {end - a.window, min(end, n)};
}

// The key tiles that the tokens pa .. pb of a sample see, in the order they are taken.
template <int KT>
struct KeyTiles {
  int plen, lo, hi, sink_end;       // prefix keys; own keys [lo, hi) and [0, sink_end)
  int np, ns, w0, count;            // tiles of the prefix, of the sinks before tile w0, all
  __device__ __forceinline__ void init(const PastArgs &a, int plen_, int n, int pa, int pb) {
    plen = pa <= pb ? plen_ : 0, np = (plen + KT - 1) / KT, lo = hi = sink_end = ns = w0 = 0, count = np;
    if (pa > pb || n == 0) return;
    lo = max(span_of(a, n, pa).lo, 0), hi = span_of(a, n, pb).hi, sink_end = min(a.sinks, hi);
    w0 = lo / KT, ns = min((sink_end + KT - 1) / KT, w0);
    count = np + ns + (hi + KT - 1) / KT - w0;
  }
  __device__ __forceinline__ bool own(int t) const { return t >= np; }
  __device__ __forceinline__ int key0(int t) const {
    const int u = t - np;
    return (u < 0 ? t : u < ns ? u : w0 + u - ns) * KT;
  }
  // the tile's keys that some row may see; none past the last tile
  __device__ __forceinline__ uint64_t bits(int t, int end) const {
    const int k0 = key0(t);
    const uint64_t b = t < np ? low_bits(plen - k0) : low_bits(hi - k0) & (~low_bits(lo - k0) | low_bits(sink_end - k0));
    return t < end ? b & low_bits(KT) : 0;
  }
};

// What the rows of one wave (or 32 of them) see of an own tile.
struct WaveRows {
  int none;              // no row belongs to a token
  int lo_a, hi_a, lo_b, hi_b;  // the spans of the first and the last token
  __device__ __forceinline__ void init(const PastArgs &a, const Sample &s, int r0, int r1) {  // rows r0 .. r1 - 1
    const int pa = max(s.start + r0 / a.G, 0), pb = min(s.start + (r1 - 1) / a.G, s.n - 1);
    none = r0 >= r1 || pa > pb;
    if (none) return;
    const Span x = span_of(a, s.n, pa), y = span_of(a, s.n, pb);
    lo_a = x.lo, hi_a = x.hi, lo_b = y.lo, hi_b = y.hi;
  }
  __device__ __forceinline__ bool nothing(const PastArgs &a, int k0, int KT) const {
    return k0 >= hi_b || (k0 + KT <= lo_a && k0 >= a.sinks);
  }
  __device__ __forceinline__ bool everything(const PastArgs &a, int k0, int KT) const {
    return k0 + KT <= hi_a && (k0 >= lo_b || k0 + KT <= a.sinks);
  }
};

// A lane's row.
struct Row {
  int b, i, g;   // sample, token, head within the key head's
  int lo, hi;    // its span
  bool on;       // it belongs to a token
  int64_t at;    // (sample, key head, row)
  __device__ __forceinline__ uint64_t bits(const PastArgs &a, int k0) const {
    return low_bits(hi - k0) & (~low_bits(lo - k0) | low_bits(a.sinks - k0));
  }
};
// Row r (of `rows`) of sample b, or of the samples of group b one after the other.
__device__ __forceinline__ Row row_of(const PastArgs &a, bool packed, int b, int hk, int r, int rows, const Sample &s) {
  Row x;
  const int rc = min(r, rows - 1);
  int in = rc;
  x.b = b;
  Sample mine = s;
  if (packed) {
    x.b = b * a.each + rc / a.rows, in = rc % a.rows;
    mine = sample_of(a, x.b);
  }
  x.i = in / a.G, x.g = in - x.i * a.G;
  const int p = mine.start + x.i;
  x.on = r < rows && p >= 0 && p < mine.n;
  x.at = ((int64_t)x.b * a.Hk + hk) * a.rows + in;
  const Span w = span_of(a, mine.n, max(p, 0));
  x.lo = x.on ? w.lo : 0, x.hi = x.on ? w.hi : 0;
  return x;
}
// Its place in a [B, Lq, H, D] tensor.
__device__ __forceinline__ int64_t row_place(const PastArgs &a, const Row &x, int hk, int64_t sb, int64_t sl, int64_t sh) {
  return x.b * sb + x.i * sl + (int64_t)(hk * a.G + x.g) * sh;
}

// Which rows a workgroup takes, and which share of their key tiles.
struct Job {
  bool packed;
  int hk, rt, b, slot, rows;
  int sp, splits;
  __device__ __forceinline__ void init(const PastArgs &a, int id) {
    packed = id < a.packed_blocks;
    if (!packed) id -= a.packed_blocks;
    const int tiles = packed ? a.packed_tiles : a.row_tiles;
    splits = packed ? a.packed_splits : a.splits;
    rows = packed ? a.each * a.rows : a.rows;
    hk = id % a.Hk, id /= a.Hk;  // heads first: rows of all heads are read together, whole token rows of memory
    rt = tiles - 1 - id % tiles, id /= tiles;  // the last rows see the most keys
    sp = id % splits, b = id / splits;
    slot = packed ? sp : a.packed_splits + sp;
  }
  __device__ __forceinline__ int share(int count, int s) const { return (int)((int64_t)count * s / splits); }
};

// Writes 32 rows of the O^T registers: the lane's row at base + at.
template <class T, int DP>
__device__ __forceinline__ void store_row(T *base, int64_t at, bool on, const f32x16 (&o)[1][DP / 32], float f, int D, int lane) {
  const float fs[1] = {f};
  store_rows<T, DP, 1>(base, o, fs, on ? 0 : 1, 1, [&](int) { return at; }, D, lane & 32);
}

// The rows of a wave that are done: out, what its rounding left, and the statistics for the backward.
template <class T, int DP>
__device__ __forceinline__ void finish_rows(const PastArgs &a, const Row &x, bool there, int hk, f32x16 (&o)[1][DP / 32], float inv,
                                            float m, float l, int lane) {
  const int64_t at = row_place(a, x, hk, (int64_t)a.Lq * a.H * a.D, (int64_t)a.H * a.D, a.D);
  if (__any(!x.on)) {  // whatever v held
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[0][d][i] = x.on ? o[0][d][i] : 0.f;
  }
  store_row<T, DP>(static_cast<T *>(a.out), at, there, o, inv, a.D, lane);
  if (a.stats == nullptr) return;
  const int64_t all = (int64_t)a.B * a.Hk * a.rows;
  if (lane < 32 && there) {
    const RowRef ref = row_ref(m, a.c);
    const bool some = l > 0.f;
    a.stats[x.at] = some ? ref.r + __builtin_amdgcn_logf(l) : l != l ? l : INFINITY;
    a.stats[all + x.at] = some ? ref.a : 0.f;
  }
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int d = 0; d < DP / 32; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float y = o[0][d][i] * inv;
        o[0][d][i] = y - bf16_to_f32(f32_to_bf16_rne(y));
      }
    store_row<uint16_t, DP>(a.rest, at, there, o, 1.f, a.D, lane);
  }
}

// Tiles of bf16 rows padded to 128 channels, laid out so that a lane's fragment addresses are one register and constants: 1024 bytes
// hold four rows, 64 bytes of each after the other, and blocks of four rows lie 1040 bytes apart: 16 rows read at one chunk, and
// the 4 rows x 64 bytes of a transposing read, meet every bank once. HeadTile's swizzle takes 24 address registers in dk / dv, which
// then has none left to read an operand ahead of its product.
template <int DP>
struct PastTile {
  static constexpr int BLOCK = 1024, ROWS = 8, ROW = 128;
  template <int RT>
  static constexpr int bytes() { return RT * ROW; }
};
template <>
struct PastTile<128> {
  static constexpr int BLOCK = 1040, ROWS = 4;
  template <int RT>
  static constexpr int bytes() { return RT / 4 * 1040; }
};

template <int DP>
struct PastReader {
  FragReader<uint16_t, DP> fr;
  __device__ __forceinline__ void init(int lane, const MLORA_LDS char *base) { fr.init(lane, base); }
  __device__ __forceinline__ void move(int by) {
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) fr.row[s] += by;
#pragma unroll
    for (int d = 0; d < DP / 32; ++d) fr.col[d][0] += by, fr.col[d][1] += by;
  }
  template <int OFF, int R0>
  __device__ __forceinline__ void rows(int s, Frag<uint16_t> &f) const { fr.template rows<OFF, R0>(s, f); }
  template <int OFF, int R0>
  __device__ __forceinline__ void cols(int d, Frag<uint16_t> &f) const { fr.template cols<OFF, R0>(d, f); }
};
template <>
struct PastReader<128> {
  int32_t row, col;
  __device__ __forceinline__ void init(int lane, const MLORA_LDS char *base) {
    const int at = (int)(uintptr_t)base, r = lane & 31, g = lane >> 4, m = lane & 15;
    row = at + (r >> 2) * 1040 + (r & 3) * 64 + (lane >> 5) * 16;
    col = at + (g >> 1) * 1040 + (m >> 2) * 64 + (2 * (g & 1) + ((m & 3) >> 1)) * 16 + 8 * (m & 1);
  }
  __device__ __forceinline__ void move(int by) { row += by, col += by; }
  template <int OFF, int R0>
  __device__ __forceinline__ void rows(int s, Frag<uint16_t> &f) const {
    f.v = *(const lds_u4 *)((const MLORA_LDS char *)(uintptr_t)(uint32_t)row + OFF + R0 / 4 * 1040 + s / 2 * 256 + s % 2 * 32);
  }
  template <int OFF, int R0>
  __device__ __forceinline__ void cols(int d, Frag<uint16_t> &f) const {
    typedef MLORA_LDS bf16x4 lds_b4;
    const MLORA_LDS char *p = (const MLORA_LDS char *)(uintptr_t)(uint32_t)col + OFF + R0 / 4 * 1040 + d * 256;
    const u32x2 x = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_b4 *)p));
    const u32x2 y = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_b4 *)(p + 2 * 1040)));
    f.v = u32x4{x[0], x[1], y[0], y[1]};
  }
};

// TileLoader for them: N of a tile's blocks by the calling wave.
template <int DP, int N>
struct PastLoader {
  static constexpr int ROWS = PastTile<DP>::ROWS;
  int32_t off[N], first, step, r0;
  __device__ __forceinline__ void init(int lane, int first_block, int block_step, int64_t stride, int head_dim) {
    first = first_block, step = block_step, r0 = DP == 128 ? (lane >> 2) & 3 : lane / 8;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int r = (first + i * step) * ROWS + r0;
      const int c = DP == 128 ? (lane >> 4) * 4 + (lane & 3) : (lane % 8) ^ HeadTile<uint16_t, 64>::swz(r);
      off[i] = c * 8 < head_dim ? (int32_t)(r * stride * 2) + c * 16 : kOOB;
    }
  }
  __device__ __forceinline__ void load(const void *base, uint64_t live, MLORA_LDS char *lds) const {
    const auto rsrc = make_rsrc(base, (int64_t)kOOB);
    const bool all = live == ~0ull;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int blk = first + i * step;
      const bool on = all || ((live >> (blk * ROWS + r0)) & 1);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (MLORA_LDS void *)(lds + blk * PastTile<DP>::BLOCK), 16, on ? off[i] : kOOB, 0, 0, 0);
    }
  }
};

// use(i, f) for i = 0 .. N - 1 with f as read(i) gave it, each read AHEAD uses before. The compiler alone reads an operand right before
// its product and waits for it.
template <int N, int AHEAD, class Read, class Use>
__device__ __forceinline__ void read_ahead(Read &&read, Use &&use) {
  using F = decltype(read(std::integral_constant<int, 0>{}));
  F ring[AHEAD + 1];
  static_for<(AHEAD < N ? AHEAD : N)>([&](auto i) __attribute__((always_inline)) {
    ring[decltype(i)::value] = read(i);
    return true;
  });
  static_for<N>([&](auto i) __attribute__((always_inline)) {
    constexpr int I = decltype(i)::value;
    if constexpr (I + AHEAD < N) ring[(I + AHEAD) % (AHEAD + 1)] = read(std::integral_constant<int, I + AHEAD>{});
    use(i, ring[I % (AHEAD + 1)]);
    __builtin_amdgcn_sched_barrier(0);
    return true;
  });
}

// Four waves of 32 rows each against the same key tiles, two buffers of K and V in LDS: tile t + 1 loads while tile
// t is multiplied; one barrier per tile.
template <int DP>
__global__ __launch_bounds__(256, 2) void past_fwd_kernel(const PastArgs a) {
  using T = uint16_t;
  constexpr int KT = AttnTile<T>::KT;
  using Tile = HeadTile<T, DP>;
  constexpr int TB = KT * Tile::RB, N = TB / 1024 / 4;
  __shared__ u32x4 smem[4 * TB / 16];  // K, V of buffer 0, K, V of buffer 1
  MLORA_LDS char *lds = (MLORA_LDS char *)smem;
  const int wave = wave_id(), lane = threadIdx.x & 63;
  Job job;
  job.init(a, blockIdx.x);
  const int hk = job.hk, r0 = job.rt * 128, group = job.packed ? job.b : job.b / a.each;
  Sample s{1, 0};
  KeyTiles<KT> tiles;
  WaveRows wr;
  wr.none = 0;
  if (job.packed) {
    tiles.init(a, prefix_keys(a, group), 0, 0, 0);
  } else {
    s = uniform(sample_of(a, job.b));
    tiles.init(a, a.with_prefix ? prefix_keys(a, group) : 0, s.n, max(s.start + r0 / a.G, 0),
               min(s.start + min(r0 + 127, a.rows - 1) / a.G, s.n - 1));
    wr.init(a, s, r0 + wave * 32, min(r0 + wave * 32 + 32, a.rows));
  }
  const int t0 = job.share(tiles.count, job.sp), t1 = job.share(tiles.count, job.sp + 1);
  const T *kp = static_cast<const T *>(a.k) + job.b * a.k_sb + hk * a.k_sh, *vp = static_cast<const T *>(a.v) + job.b * a.v_sb + hk * a.v_sh;
  const T *pkp = static_cast<const T *>(a.pk) + group * a.pk_sb + hk * a.pk_sh, *pvp = static_cast<const T *>(a.pv) + group * a.pv_sb + hk * a.pv_sh;
  TileLoader<T, DP, N> kl, vl;
  bool own = false;
  auto aim = [&](bool o) __attribute__((always_inline)) {
    own = o;
    kl.init(lane, wave, 4, o ? a.k_sl : a.pk_sl, a.D), vl.init(lane, wave, 4, o ? a.v_sl : a.pv_sl, a.D);
  };
  auto stage = [&](int t, int buf) __attribute__((always_inline)) {
    const bool o = tiles.own(t);
    if (o != own) aim(o);  // at the end of the prefix
    const int64_t k0 = tiles.key0(t);
    const uint64_t bits = tiles.bits(t, t1);  // behind the last one nothing is read
    kl.load(o ? kp + k0 * a.k_sl : pkp + k0 * a.pk_sl, bits, lds + buf * 2 * TB);
    vl.load(o ? vp + k0 * a.v_sl : pvp + k0 * a.pv_sl, bits, lds + buf * 2 * TB + TB);
  };
  aim(tiles.own(t0));
  if (t0 < t1) stage(t0, 0);
  FragReader<T, DP> fr;
  fr.init(lane, lds);
  Softmax<T, DP, 1, KT, true> sm;
  sm.init();
  const Row x = row_of(a, job.packed, job.b, hk, r0 + wave * 32 + (lane & 31), job.rows, s);
  const bool there = r0 + wave * 32 + (lane & 31) < job.rows;
  {
    const T *p = static_cast<const T *>(a.q) + row_place(a, x, hk, a.q_sb, a.q_sl, a.q_sh);
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks) {
      const int d = 16 * ks + 8 * (lane >> 5);
      load_frag(p, d, x.on && d < a.D, sm.q[0][ks]);
    }
  }
  for (int t = t0; t < t1; ++t) {
    wait_vmcnt<0>();
    lds_pipeline_barrier();  // tile t is in LDS, and every wave has read the tile before it
    stage(t + 1, (t + 1 - t0) & 1);
    const int k0 = tiles.key0(t);
    const bool o = tiles.own(t);
    if (!wr.none && !(o && wr.nothing(a, k0, KT))) {
      const uint64_t all = tiles.bits(t, t1);
      uint64_t bits[1] = {all};
      bool masked = all != low_bits(KT);
      if (o && !wr.everything(a, k0, KT)) masked = true, bits[0] = x.bits(a, k0);
      sm.template step<0, TB>(fr, masked, bits, a.c, lane);
    }
    fr.flip(2 * TB);
  }
  wait_vmcnt<0>();
  float f;
  const float l = sm.sums(0, f);
  if (a.slots > 1) {
    const int64_t first = job.slot * ((int64_t)a.B * a.Hk * a.rows);
    if (lane < 32 && there) *(float2 *)(a.part_ml + 2 * (first + x.at)) = x.on ? float2{sm.m[0], l} : float2{kNoMax, 0.f};
    store_row<float, DP>(a.part_o + first * a.D, x.at * a.D, there, sm.o, f, a.D, lane);
  } else {
    const bool some = x.on && (l > 0.f || l != l);
    finish_rows<T, DP>(a, x, there, hk, sm.o, some ? f / l : 0.f, sm.m[0], x.on ? l : 0.f, lane);
  }
}

// ---------------------------------------------------------------- few rows
//
// Blocks of 16 rows on 16 x 16 products: D[16 x 16] += A[16 x 32] B[32 x 16], a lane holds row (or column) lane % 16 and 8 of the
// step's 32 contraction elements, its quarter lane / 16 decides which; the result leaves it column lane % 16 and rows
// 4·(lane / 16) + i. S^T = K·Q^T of 16 keys leaves a lane four keys of its query; two such blocks are the eight
// contraction elements of O^T += V^T·P^T, keys 4g + j and 16 + 4g + j of 32.
__device__ __forceinline__ f32x4 mma32(const Frag<uint16_t> &a, const Frag<uint16_t> &b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(a.v), as_bf16x8(b.v), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma4(float a, float b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }
// over the four quarters of a column
__device__ __forceinline__ float quarter_max(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return half_max(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
__device__ __forceinline__ float quarter_sum(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return half_sum(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

// A lane's addresses for such fragments of a HeadTile. keys: row R0 + lane % 16, elements 32s + 8·(lane / 16) .. + 7; values: column
// 16d + lane % 16 of the 32 rows in the order above.
template <class T, int DP>
struct FewReader;
template <int DP>
struct FewReader<uint16_t, DP> {
  using Tile = HeadTile<uint16_t, DP>;
  int32_t row[DP / 32], col[DP / 16];
  __device__ __forceinline__ void init(int lane, const MLORA_LDS char *base) {
    const int32_t at = (int32_t)(uintptr_t)base;
    const int r = lane & 15, g = lane >> 4;
#pragma unroll
    for (int s = 0; s < DP / 32; ++s) row[s] = at + r * Tile::RB + (((4 * s + g) ^ Tile::swz(r)) << 4);
    const int key = 4 * g + (r >> 2), c = r & 3;
#pragma unroll
    for (int d = 0; d < DP / 16; ++d) col[d] = at + key * Tile::RB + (((2 * d + (c >> 1)) ^ Tile::swz(key)) << 4) + 8 * (c & 1);
  }
  template <int OFF, int R0>  // swz(r + 16) = swz(r)
  __device__ __forceinline__ void keys(int s, Frag<uint16_t> &f) const {
    f.v = *(const lds_u4 *)((const MLORA_LDS char *)(uintptr_t)(uint32_t)row[s] + OFF + R0 * Tile::RB);
  }
  template <int OFF>
  __device__ __forceinline__ void values(int d, Frag<uint16_t> &f) const {
    typedef MLORA_LDS bf16x4 lds_b4;
    const MLORA_LDS char *p = (const MLORA_LDS char *)(uintptr_t)(uint32_t)col[d] + OFF;
    const u32x2 x = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_b4 *)p));
    const u32x2 y = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds_b4 *)(p + 16 * Tile::RB)));
    f.v = u32x4{x[0], x[1], y[0], y[1]};
  }
};
template <int DP>
struct FewReader<float, DP> {
  using Tile = HeadTile<float, DP>;
  int32_t row[2], val[4], sw;
  __device__ __forceinline__ void init(int lane, const MLORA_LDS char *base) {
    const int r = lane & 15, g = lane >> 4, at = (int32_t)(uintptr_t)base;
    sw = Tile::swz(r) ^ (2 * g);
    row[0] = at + r * Tile::RB, row[1] = row[0] + 16 * Tile::RB;
#pragma unroll
    for (int j = 0; j < 4; ++j) val[j] = at + (4 * g + j) * Tile::RB + ((r ^ Tile::swz(4 * g + j)) << 4);
  }
  template <int OFF, int R0>  // swz(r + 16) = swz(r)
  __device__ __forceinline__ void keys(int s, Frag<float> &f) const {
    const MLORA_LDS char *t = (const MLORA_LDS char *)(uintptr_t)(uint32_t)row[R0 / 16] + OFF;
    const f32x4 a = *(const lds_f4 *)(t + (((8 * s) ^ sw) << 4)), b = *(const lds_f4 *)(t + (((8 * s + 1) ^ sw) << 4));
#pragma unroll
    for (int j = 0; j < 4; ++j) f.v[j] = a[j], f.v[j + 4] = b[j];
  }
  // channels 64h + 4·(lane % 16) .. + 3 of row 16·(j / 4) + 4·(lane / 16) + j % 4: element i is the operand of channels 64h + 4m + i, m the
  // result's row
  template <int OFF>
  __device__ __forceinline__ f32x4 value4(int j, int h) const {
    return *(const lds_f4 *)((const MLORA_LDS char *)(uintptr_t)(uint32_t)val[j % 4] + OFF + j / 4 * 16 * Tile::RB + 256 * h);
  }
};

// s[n][b] += rows 16b .. of the tile at OFF times the NC x 16 columns of x.
template <int OFF, int DP, int NC>
__device__ __forceinline__ void few_scores(const FewReader<uint16_t, DP> &fr, const Frag<uint16_t> (&x)[NC][DP / 32], f32x4 (&s)[NC][2]) {
#pragma unroll
  for (int ks = 0; ks < DP / 32; ++ks)
    static_for<2>([&](auto kb) __attribute__((always_inline)) {
      Frag<uint16_t> kf;
      fr.template keys<OFF, 16 * decltype(kb)::value>(ks, kf);
#pragma unroll
      for (int n = 0; n < NC; ++n) s[n][kb] = mma32(kf, x[n][ks], s[n][kb]);
      return true;
    });
}
template <int OFF, int DP, int NC>
__device__ __forceinline__ void few_scores(const FewReader<float, DP> &fr, const Frag<float> (&x)[NC][DP / 32], f32x4 (&s)[NC][2]) {
#pragma unroll
  for (int ks = 0; ks < DP / 32; ++ks) {
    Frag<float> kf[2];
    fr.template keys<OFF, 0>(ks, kf[0]);
    fr.template keys<OFF, 16>(ks, kf[1]);
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int n = 0; n < NC; ++n) s[n][kb] = mma4(kf[kb].v[j], x[n][ks].v[j], s[n][kb]);
  }
}

// o[n] += the tile at OFF, transposed, times p[n].
template <int OFF, int DP, int NC>
__device__ __forceinline__ void few_weigh(const FewReader<uint16_t, DP> &fr, const Frag<uint16_t> (&p)[NC], f32x4 (&o)[NC][DP / 16]) {
#pragma unroll
  for (int d = 0; d < DP / 16; ++d) {
    Frag<uint16_t> vf;
    fr.template values<OFF>(d, vf);
#pragma unroll
    for (int n = 0; n < NC; ++n) o[n][d] = mma32(vf, p[n], o[n][d]);
  }
}
template <int OFF, int DP, int NC>
__device__ __forceinline__ void few_weigh(const FewReader<float, DP> &fr, const Frag<float> (&p)[NC], f32x4 (&o)[NC][DP / 16]) {
#pragma unroll
  for (int j = 0; j < 8; ++j)
#pragma unroll
    for (int h = 0; h < DP / 64; ++h) {
      const f32x4 v = fr.template value4<OFF>(j, h);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int n = 0; n < NC; ++n) o[n][4 * h + i] = mma4(v[i], p[n].v[j], o[n][4 * h + i]);
    }
}

// Four channels that follow each other, few_channel(d) .. + 3, of a lane's column of such sums, d < DP / 16.
template <class T, int ND>
__device__ __forceinline__ f32x4 few_vector(const f32x4 (&o)[ND], int d) {
  if constexpr (sizeof(T) == 2) return o[d];
  else return f32x4{o[d & ~3][d & 3], o[(d & ~3) + 1][d & 3], o[(d & ~3) + 2][d & 3], o[(d & ~3) + 3][d & 3]};
}
template <class T>
__device__ __forceinline__ int few_channel(int d, int lane) {
  return sizeof(T) == 2 ? 16 * d + 4 * (lane >> 4) : 64 * (d >> 2) + 16 * (lane >> 4) + 4 * (d & 3);
}

// The running softmax of NC x 16 rows against 32 keys per step, as Softmax does it (two sums: e of the weights before their
// rounding to bf16, l of what the product with V sees).
template <class T, int DP, int NC>
struct FewSoftmax {
  static constexpr int ND = DP / 16, NS = DP / 32;
  f32x4 o[NC][ND];
  Frag<T> q[NC][NS];
  float m[NC], l[NC], e[NC];

  __device__ __forceinline__ void init() {
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      m[n] = kNoMax, l[n] = 0.f, e[n] = 0.f;
#pragma unroll
      for (int d = 0; d < ND; ++d) o[n][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
  }

  template <int KOFF, int VOFF>
  __device__ __forceinline__ void step(const FewReader<T, DP> &fr, bool masked, const uint32_t (&bits)[NC], float c, int lane) {
    f32x4 s[NC][2];
#pragma unroll
    for (int n = 0; n < NC; ++n) s[n][0] = s[n][1] = f32x4{0.f, 0.f, 0.f, 0.f};
    few_scores<KOFF, DP, NC>(fr, q, s);
    if (masked) {
#pragma unroll
      for (int n = 0; n < NC; ++n) {
        const uint32_t mine = bits[n] >> (4 * (lane >> 4));
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[n][kb][i] = (mine >> (16 * kb + i)) & 1 ? s[n][kb][i] : -INFINITY;
      }
    }
    Frag<T> p[NC];
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      float mx = fmaxf(fmaxf(fmaxf(s[n][0][0], s[n][0][1]), fmaxf(s[n][0][2], s[n][0][3])),
                       fmaxf(fmaxf(s[n][1][0], s[n][1][1]), fmaxf(s[n][1][2], s[n][1][3])));
      mx = quarter_max(mx);
      RowRef ref = row_ref(m[n], c);
      if (__any(__builtin_fmaf(mx - ref.a, c, -ref.r) > 8.f)) {
        m[n] = fmaxf(m[n], mx);
        const RowRef up = row_ref(m[n], c);
        const float f = ref_factor(ref, up, c);
        ref = up;
        l[n] *= f, e[n] *= f;
#pragma unroll
        for (int d = 0; d < ND; ++d) o[n][d] *= f;
      }
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[n][kb][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[n][kb][i] - ref.a, c, -ref.r));
      if constexpr (sizeof(T) == 2) {
        const auto ones = __builtin_bit_cast(bf16x2, 0x3f803f80u);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          p[n].v[j] = pack2_bf16(s[n][j / 2][2 * (j % 2)], s[n][j / 2][2 * (j % 2) + 1]);
          l[n] = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, (uint32_t)p[n].v[j]), ones, l[n], false);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) p[n].v[j] = s[n][j / 4][j % 4];
      }
      const f32x4 t = s[n][0] + s[n][1];
      e[n] += (t[0] + t[1]) + (t[2] + t[3]);
    }
    few_weigh<VOFF, DP, NC>(fr, p, o);
  }

  __device__ __forceinline__ float sums(int n, float &f) {
    const float ew = quarter_sum(e[n]);
    f = 1.f;
    if constexpr (sizeof(T) == 4) return ew;
    const float lw = quarter_sum(l[n]);
    if (lw > 0.f) f = ew / lw;
    return lw > 0.f ? ew : lw;
  }
};

// A workgroup's key tiles of K and V on their way into LDS, N blocks of 1024 bytes of either by the calling wave.
template <class T, int DP, int KT, int N>
struct TileStream {
  const T *kp, *vp, *pkp, *pvp;
  TileLoader<T, DP, N> kl, vl;
  int end;
  bool own;
  __device__ __forceinline__ void aim(const PastArgs &a, int wave, int waves, int lane, bool o) {
    own = o;
    kl.init(lane, wave, waves, o ? a.k_sl : a.pk_sl, a.D), vl.init(lane, wave, waves, o ? a.v_sl : a.pv_sl, a.D);
  }
  __device__ __forceinline__ void init(const PastArgs &a, int b, int group, int hk, int wave, int waves, int lane, const KeyTiles<KT> &tiles, int t0, int t1) {
    kp = static_cast<const T *>(a.k) + b * a.k_sb + hk * a.k_sh, vp = static_cast<const T *>(a.v) + b * a.v_sb + hk * a.v_sh;
    pkp = static_cast<const T *>(a.pk) + group * a.pk_sb + hk * a.pk_sh, pvp = static_cast<const T *>(a.pv) + group * a.pv_sb + hk * a.pv_sh;
    end = t1;
    aim(a, wave, waves, lane, tiles.own(t0));
  }
  __device__ __forceinline__ void stage(const PastArgs &a, const KeyTiles<KT> &tiles, int t, MLORA_LDS char *to) {
    constexpr int TB = KT * HeadTile<T, DP>::RB;
    const bool o = tiles.own(t);
    if (o != own) aim(a, kl.first, kl.step, threadIdx.x & 63, o);  // at the end of the prefix
    const int64_t k0 = tiles.key0(t);
    const uint64_t bits = tiles.bits(t, end);
    const T *k = o ? kp + k0 * a.k_sl : pkp + k0 * a.pk_sl, *v = o ? vp + k0 * a.v_sl : pvp + k0 * a.pv_sl;
    if (bits == low_bits(KT)) kl.load_all(k, to), vl.load_all(v, to + TB);
    else kl.load(k, bits, to), vl.load(v, bits, to + TB);
  }
};

// A row as a column operand of 16 x 16 products.
template <class T, int DP>
__device__ __forceinline__ void load_row(const T *p, bool on, int D, int lane, Frag<T> (&f)[DP / 32]) {
#pragma unroll
  for (int ks = 0; ks < DP / 32; ++ks) {
    const int d = 32 * ks + 8 * (lane >> 4);
    load_frag(p, d, on && d < D, f[ks]);
  }
}

// Few rows (16 NC per workgroup): the waves take different key tiles, each with its own buffer (no barrier in the loop; two
// waves per SIMD, one multiplies while the other waits), and their running softmaxes are joined through LDS. Bound by the reading
// of K and V where they are long (65520 keys, 8 key heads of 128: 46 us, 5.9 TB/s, much of it out of the 256 MB cache), by a launch and one chain of loads,
// products and the join where they are short (32 keys 5.4 us, 260 keys of 64 channels 6.1). On 32 x 32 products, four waves with two
// buffers each: 51, 7.7 and 8.3.
// float32 takes any number of rows this way (waves of 32 rows that share tiles behind a barrier: 1573 tokens, window 257, 12 heads of
// 64: 46 us, here 30; 524 rows on 646 keys 32 and 21): the matrix core takes 2048 cycles for 32 rows by 32 keys by 64 channels, so
// that reading the tiles again costs less than waiting. f32_waves chooses between NW and half or a quarter of it.
template <class T, int DP>
constexpr int kFewWaves = sizeof(T) * DP == 512 ? 4 : 8;

template <class T, int DP, int NC, int NW>
__global__ __launch_bounds__((64 * NW), (kFewWaves<T, DP> / 4)) void past_few_kernel(const PastArgs a) {
  constexpr int KT = 32, ND = DP / 16;
  using Tile = HeadTile<T, DP>;
  constexpr int TB = KT * Tile::RB, N = TB / 1024;
  static_assert(NC * ND * 64 * 16 <= 2 * TB, "a wave's sums fit its buffers");
  // one array, (m, l) of [wave][n][query] behind them
  __shared__ u32x4 smem[2 * TB * NW / 16 + NW * NC * 8];
  float2 (&ml)[NW][NC][16] = *(float2 (*)[NW][NC][16])(smem + 2 * TB * NW / 16);
  const int wave = wave_id(), lane = threadIdx.x & 63;
  MLORA_LDS char *lds = (MLORA_LDS char *)smem + wave * 2 * TB;
  Job job;
  job.init(a, blockIdx.x);
  const int hk = job.hk, r0 = job.rt * 16 * NC, group = job.packed ? job.b : job.b / a.each;
  Sample s{1, 0};
  KeyTiles<KT> tiles;
  WaveRows wr;
  wr.none = 0;
  if (job.packed) {
    tiles.init(a, prefix_keys(a, group), 0, 0, 0);
  } else {
    s = uniform(sample_of(a, job.b));
    tiles.init(a, a.with_prefix ? prefix_keys(a, group) : 0, s.n, max(s.start + r0 / a.G, 0),
               min(s.start + min(r0 + 16 * NC - 1, a.rows - 1) / a.G, s.n - 1));
    wr.init(a, s, r0, min(r0 + 16 * NC, a.rows));
  }
  const int t1 = job.share(tiles.count, job.sp + 1), t0 = min(job.share(tiles.count, job.sp) + wave, t1);
  TileStream<T, DP, KT, N> in;
  in.init(a, job.b, group, hk, 0, 1, lane, tiles, t0, t1);
  if (t0 < t1) in.stage(a, tiles, t0, lds);
  FewReader<T, DP> fr;
  fr.init(lane, lds);
  FewSoftmax<T, DP, NC> sm;
  sm.init();
  Row x[NC];
  bool there[NC];
#pragma unroll
  for (int n = 0; n < NC; ++n) {
    x[n] = row_of(a, job.packed, job.b, hk, r0 + 16 * n + (lane & 15), job.rows, s);
    there[n] = r0 + 16 * n + (lane & 15) < job.rows;
    load_row<T, DP>(static_cast<const T *>(a.q) + row_place(a, x[n], hk, a.q_sb, a.q_sl, a.q_sh), x[n].on, a.D, lane, sm.q[n]);
  }
  for (int t = t0; t < t1; t += NW) {
    wait_vmcnt<0>();  // tile t is in this wave's buffer
    asm volatile("" ::: "memory");
    const int k0 = tiles.key0(t);
    const bool o = tiles.own(t);
    const uint32_t all = (uint32_t)tiles.bits(t, t1);
    uint32_t bits[NC];
    bool masked = all != ~0u;
    const bool rows = o && !wr.everything(a, k0, KT);
    masked |= rows;
#pragma unroll
    for (int n = 0; n < NC; ++n) bits[n] = rows ? (uint32_t)x[n].bits(a, k0) : all;
    sm.template step<0, TB>(fr, masked, bits, a.c, lane);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the buffer is read
    if (t + NW < t1) in.stage(a, tiles, t + NW, lds);
  }
  // join the waves: every wave leaves its sums, then sums its share of the 16 x 16 tiles over the waves
  float f[NC];
#pragma unroll
  for (int n = 0; n < NC; ++n) {
    const float l = sm.sums(n, f[n]);
    if (lane < 16) ml[wave][n][lane] = float2{sm.m[n], l};
  }
  f32x4 *mine = (f32x4 *)smem + wave * 2 * TB / 16;
#pragma unroll
  for (int n = 0; n < NC; ++n)
#pragma unroll
    for (int d = 0; d < ND; ++d) mine[(n * ND + d) * 64 + lane] = few_vector<T, ND>(sm.o[n], d) * f[n];
  __syncthreads();
  const int64_t all = (int64_t)a.B * a.Hk * a.rows;
#pragma unroll
  for (int n = 0; n < NC; ++n) {
    float m = kNoMax, lsum = 0.f, w[NW];
#pragma unroll
    for (int q = 0; q < NW; ++q) m = fmaxf(m, ml[q][n][lane & 15].x);
    const RowRef top = row_ref(m, a.c);
#pragma unroll
    for (int q = 0; q < NW; ++q) {
      const float2 v = ml[q][n][lane & 15];
      w[q] = ref_factor(row_ref(v.x, a.c), top, a.c);
      lsum += w[q] * v.y;
    }
    if (!x[n].on) lsum = 0.f;
    const bool some = lsum > 0.f || lsum != lsum;
    const float inv = a.slots > 1 ? 1.f : some ? 1.0f / lsum : 0.f;
    if (wave == 0 && lane < 16 && there[n]) {
      if (a.slots > 1) *(float2 *)(a.part_ml + 2 * (job.slot * all + x[n].at)) = float2{some ? m : kNoMax, lsum};
      else if (a.stats != nullptr) {
        a.stats[x[n].at] = lsum > 0.f ? top.r + __builtin_amdgcn_logf(lsum) : lsum != lsum ? lsum : INFINITY;
        a.stats[all + x[n].at] = lsum > 0.f ? top.a : 0.f;
      }
    }
    const int64_t at = row_place(a, x[n], hk, (int64_t)a.Lq * a.H * a.D, (int64_t)a.H * a.D, a.D);
    for (int d = wave; d < ND; d += NW) {  // 4 consecutive channels per lane
      f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int q = 0; q < NW; ++q) o += w[q] * ((const f32x4 *)smem + q * 2 * TB / 16)[(n * ND + d) * 64 + lane];
      const int ch = few_channel<T>(d, lane);
      if (!there[n] || ch >= a.D) continue;
      o *= inv;
      if (!some) o = f32x4{0.f, 0.f, 0.f, 0.f};
      if (a.slots > 1) *(MLORA_GLOBAL f32x4 *)(a.part_o + (job.slot * all + x[n].at) * a.D + ch) = o;
      else if constexpr (sizeof(T) == 2) {
        *(MLORA_GLOBAL u32x2 *)(static_cast<T *>(a.out) + at + ch) = u32x2{pack2_bf16(o[0], o[1]), pack2_bf16(o[2], o[3])};
        if (a.stats != nullptr) {
#pragma unroll
          for (int j = 0; j < 4; ++j) o[j] -= bf16_to_f32(f32_to_bf16_rne(o[j]));
          *(MLORA_GLOBAL u32x2 *)(a.rest + at + ch) = u32x2{pack2_bf16(o[0], o[1]), pack2_bf16(o[2], o[3])};
        }
      } else *(MLORA_GLOBAL f32x4 *)(static_cast<T *>(a.out) + at + ch) = o;
    }
  }
}

// Writes a joined row, four channels per lane `at` of 32: its sums o and l relative to top.
template <class T>
__device__ __forceinline__ void write_joined(const PastArgs &a, int64_t all, int64_t row, int at, f32x4 o, float l, const RowRef &top) {
  if (at == 0 && a.stats != nullptr) {
    a.stats[row] = l > 0.f ? top.r + __builtin_amdgcn_logf(l) : l != l ? l : INFINITY;
    a.stats[all + row] = l > 0.f ? top.a : 0.f;
  }
  if (4 * at >= a.D) return;
  const int r = (int)(row % a.rows), hk = (int)(row / a.rows % a.Hk);
  const int64_t b = row / a.rows / a.Hk;
  const int64_t place = (b * a.Lq + r / a.G) * a.H * a.D + (int64_t)(hk * a.G + r % a.G) * a.D + 4 * at;
  o *= l > 0.f || l != l ? 1.0f / l : 0.f;
  T *p = static_cast<T *>(a.out) + place;
  if constexpr (sizeof(T) == 2) {
    *(MLORA_GLOBAL u32x2 *)p = u32x2{pack2_bf16(o[0], o[1]), pack2_bf16(o[2], o[3])};
    if (a.stats == nullptr) return;
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] -= bf16_to_f32(f32_to_bf16_rne(o[j]));
    *(MLORA_GLOBAL u32x2 *)(a.rest + place) = u32x2{pack2_bf16(o[0], o[1]), pack2_bf16(o[2], o[3])};
  } else *(MLORA_GLOBAL f32x4 *)p = o;
}

// Joins up to eight shares of a row, weights 2^((m_s − max m)·c): 32 lanes per row, every share's sums asked for before any is used
// (18720 rows of three shares 7.6 us; with a workgroup per row 18.8).
template <class T>
__global__ __launch_bounds__(256) void past_join_rows_kernel(const PastArgs a) {
  constexpr int MOST = 8;
  const int64_t all = (int64_t)a.B * a.Hk * a.rows, row = (int64_t)blockIdx.x * 8 + threadIdx.x / 32;
  const int at = threadIdx.x % 32, ch = min(4 * at, a.D - 4);
  if (row >= all) return;
  float2 ml[MOST];
  f32x4 part[MOST];
#pragma unroll
  for (int s = 0; s < MOST; ++s) {
    if (s >= a.slots) break;
    ml[s] = *(const float2 *)(a.part_ml + 2 * (s * all + row));
    part[s] = *(const MLORA_GLOBAL f32x4 *)(a.part_o + (s * all + row) * a.D + ch);
  }
  float m = kNoMax, l = 0.f;
#pragma unroll
  for (int s = 0; s < MOST; ++s)
    if (s < a.slots) m = fmaxf(m, ml[s].x);
  const RowRef top = row_ref(m, a.c);
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int s = 0; s < MOST; ++s) {
    if (s >= a.slots) break;
    const float w = ref_factor(row_ref(ml[s].x, a.c), top, a.c);
    l += w * ml[s].y;
    if (ml[s].y != 0.f) o += w * part[s];
  }
  write_joined<T>(a, all, row, at, o, l, top);
}

// Joins more shares of a row, one workgroup per row: weights 2^((m_s − max m)·c). Eight groups of 32 lanes (4 channels
// each) take every eighth share, and their sums are added in order through LDS.
template <class T>
__global__ __launch_bounds__(256) void past_join_kernel(const PastArgs a) {
  __shared__ f32x4 sums[8][32];
  __shared__ float ls[8];
  const int64_t all = (int64_t)a.B * a.Hk * a.rows, row = blockIdx.x;
  const int at = threadIdx.x % 32, g = threadIdx.x / 32, ch = min(4 * at, a.D - 4);
  float m = kNoMax;
  for (int s = at; s < a.slots; s += 32) m = fmaxf(m, a.part_ml[2 * (s * all + row)]);
#pragma unroll
  for (int i = 16; i >= 1; i >>= 1) m = fmaxf(m, __shfl_xor(m, i));
  const RowRef top = row_ref(m, a.c);
  float l = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = g; s < a.slots; s += 8) {
    const float2 ml = *(const float2 *)(a.part_ml + 2 * (s * all + row));
    const f32x4 part = *(const MLORA_GLOBAL f32x4 *)(a.part_o + (s * all + row) * a.D + ch);  // both loads before either is used
    const float w = ref_factor(row_ref(ml.x, a.c), top, a.c);
    l += w * ml.y;
    if (ml.y != 0.f) o += w * part;
  }
  sums[g][at] = o;
  if (at == 0) ls[g] = l;
  __syncthreads();
  if (g != 0) return;
  l = ls[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) o += sums[i][at], l += ls[i];
  write_joined<T>(a, all, row, at, o, l, top);
}

// ------------------------------------------------------------------ backward
//
//   P = 2^((s − a)·c − x),  delta = Σ_d do·(out + rest),  dP = do·Vᵀ,  dS = P·(dP − delta)
//   dq = scale · dS·K,   dk = scale · dSᵀ·q,   dv = Pᵀ·do
// Two kernels form P again: one owns query rows (dq, and delta on the way), one owns keys (dk, dv; a prefix's keys meet
// the rows of all its samples). That is 7 products instead of 5, and no atomics: every sum has a fixed order. rest holds what
// the rounding of out to bf16 left, so that delta is as good as float32 sums: a row that rests on one key has dS = 0, and
// half a bf16 step of out in delta would be its whole gradient. P and dS are rounded to bf16 as operands of the
// products that follow: half a step each.

struct PastBwdArgs {
  PastArgs f;
  const void *g;             // the output's gradient
  void *dq, *dk, *dv, *dpk, *dpv;  // contiguous
  float *delta;              // [B·Hk·rows]
  f32x4 *part;               // shares of dq, then of dk and dv, in register order
  int64_t g_sb, g_sl, g_sh;
  float scale;
  int32_t key_blocks, prefix_blocks, sink_blocks;  // of 32 NW keys: all own ones, the prefix's, those with a sink
  int32_t prefix_splits, sink_splits, own_splits;
  int64_t sink_part, own_part;  // where a class's shares begin, in 16-byte vectors
};

template <int DP>
__global__ __launch_bounds__(256, 2) void past_dq_kernel(const PastBwdArgs ba) {
  using T = uint16_t;
  const PastArgs &a = ba.f;
  constexpr int KT = AttnTile<T>::KT, ND = DP / 32;
  using Tile = HeadTile<T, DP>;
  constexpr int TB = KT * Tile::RB, N = TB / 1024 / 4;
  __shared__ u32x4 smem[4 * TB / 16];
  MLORA_LDS char *lds = (MLORA_LDS char *)smem;
  const int wave = wave_id(), lane = threadIdx.x & 63;
  Job job;
  job.init(a, blockIdx.x);
  const int hk = job.hk, r0 = job.rt * 128, group = job.b / a.each;
  const Sample s = uniform(sample_of(a, job.b));
  KeyTiles<KT> tiles;
  WaveRows wr;
  tiles.init(a, a.with_prefix ? prefix_keys(a, group) : 0, s.n, max(s.start + r0 / a.G, 0),
             min(s.start + min(r0 + 127, a.rows - 1) / a.G, s.n - 1));
  wr.init(a, s, r0 + wave * 32, min(r0 + wave * 32 + 32, a.rows));
  const int t0 = job.share(tiles.count, job.sp), t1 = job.share(tiles.count, job.sp + 1);
  const T *kp = static_cast<const T *>(a.k) + job.b * a.k_sb + hk * a.k_sh, *vp = static_cast<const T *>(a.v) + job.b * a.v_sb + hk * a.v_sh;
  const T *pkp = static_cast<const T *>(a.pk) + group * a.pk_sb + hk * a.pk_sh, *pvp = static_cast<const T *>(a.pv) + group * a.pv_sb + hk * a.pv_sh;
  TileLoader<T, DP, N> kl, vl;
  bool own = false;
  auto aim = [&](bool o) __attribute__((always_inline)) {
    own = o;
    kl.init(lane, wave, 4, o ? a.k_sl : a.pk_sl, a.D), vl.init(lane, wave, 4, o ? a.v_sl : a.pv_sl, a.D);
  };
  auto stage = [&](int t, int buf) __attribute__((always_inline)) {
    const bool o = tiles.own(t);
    if (o != own) aim(o);
    const int64_t k0 = tiles.key0(t);
    const uint64_t bits = tiles.bits(t, t1);
    kl.load(o ? kp + k0 * a.k_sl : pkp + k0 * a.pk_sl, bits, lds + buf * 2 * TB);
    vl.load(o ? vp + k0 * a.v_sl : pvp + k0 * a.pv_sl, bits, lds + buf * 2 * TB + TB);
  };
  aim(tiles.own(t0));
  if (t0 < t1) stage(t0, 0);
  FragReader<T, DP> fr;
  fr.init(lane, lds);
  const Row row = row_of(a, false, job.b, hk, r0 + wave * 32 + (lane & 31), a.rows, s);
  const bool there = r0 + wave * 32 + (lane & 31) < a.rows;
  const int64_t all = (int64_t)a.B * a.Hk * a.rows;
  const int64_t oat = row_place(a, row, hk, (int64_t)a.Lq * a.H * a.D, (int64_t)a.H * a.D, a.D);
  Frag<T> q[DP / 16], g[DP / 16];
  float delta = 0.f;
  {
    const T *qp = static_cast<const T *>(a.q) + row_place(a, row, hk, a.q_sb, a.q_sl, a.q_sh);
    const T *gp_ = static_cast<const T *>(ba.g) + row_place(a, row, hk, ba.g_sb, ba.g_sl, ba.g_sh);
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks) {
      const int d = 16 * ks + 8 * (lane >> 5);
      const bool on = row.on && d < a.D;
      Frag<T> of;
      load_frag(qp, d, on, q[ks]);
      load_frag(gp_, d, on, g[ks]);
      load_frag(static_cast<const T *>(a.out) + oat, d, on, of);
      Frag<T> rf;
      load_frag(a.rest + oat, d, on, rf);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        delta += __uint_as_float(g[ks].v[j] << 16) * (__uint_as_float(of.v[j] << 16) + __uint_as_float(rf.v[j] << 16));
        delta += __uint_as_float(g[ks].v[j] & 0xffff0000u) * (__uint_as_float(of.v[j] & 0xffff0000u) + __uint_as_float(rf.v[j] & 0xffff0000u));
      }
    }
  }
  delta = half_sum(delta);
  const float x = row.on ? a.stats[row.at] : INFINITY, shift = row.on ? a.stats[all + row.at] : 0.f;
  if (job.sp == 0 && lane < 32 && there) ba.delta[row.at] = delta;
  const bool shifted = __any(shift != 0.f);
  f32x16 dq[1][ND];
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) dq[0][d][i] = 0.f;
  for (int t = t0; t < t1; ++t) {
    wait_vmcnt<0>();
    lds_pipeline_barrier();  // tile t is in LDS, and every wave has read the tile before it
    stage(t + 1, (t + 1 - t0) & 1);
    const int k0 = tiles.key0(t);
    const bool o = tiles.own(t);
    if (!wr.none && !(o && wr.nothing(a, k0, KT))) {
      uint64_t bits = tiles.bits(t, t1);
      bool masked = bits != low_bits(KT);
      if (o && !wr.everything(a, k0, KT)) masked = true, bits = row.bits(a, k0);
      static_for<KT / 32>([&](auto block) __attribute__((always_inline)) {
        constexpr int kb = decltype(block)::value;
        f32x16 sc, dp;
#pragma unroll
        for (int i = 0; i < 16; ++i) sc[i] = 0.f, dp[i] = 0.f;
#pragma unroll
        for (int ks = 0; ks < DP / 16; ++ks) {
          Frag<T> kf, vf;
          fr.template rows<0, 32 * kb>(ks, kf);
          sc = mma16(kf, q[ks], sc);
          fr.template rows<TB, 32 * kb>(ks, vf);
          dp = mma16(vf, g[ks], dp);
        }
        if (masked) {
          const uint64_t mine = bits >> (4 * (lane >> 5));
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const bool on = (mine >> (32 * kb + 8 * (i / 4) + i % 4)) & 1;
            sc[i] = on ? sc[i] : -INFINITY, dp[i] = on ? dp[i] : 0.f;
          }
        }
        if (shifted) {
#pragma unroll
          for (int i = 0; i < 16; ++i) sc[i] -= shift;
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) sc[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[i], a.c, -x)) * (dp[i] - delta);
        static_for<2>([&](auto ks) __attribute__((always_inline)) {
          Frag<T> ds;
          to_frag(sc, ks, ds);
#pragma unroll
          for (int d = 0; d < ND; ++d) {
            Frag<T> kf;
            fr.template cols<0, 32 * kb + 16 * decltype(ks)::value>(d, kf);
            dq[0][d] = mma16(kf, ds, dq[0][d]);
          }
          return true;
        });
        return true;
      });
    }
    fr.flip(2 * TB);
  }
  wait_vmcnt<0>();
  if (__any(!row.on)) {
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) dq[0][d][i] = row.on ? dq[0][d][i] : 0.f;
  }
  if (a.splits > 1) {
    f32x4 *p = ba.part + ((((int64_t)job.sp * a.B + job.b) * a.row_tiles + job.rt) * a.Hk + hk) * (4 * ND * 4 * 64) + wave * (ND * 4 * 64) + lane;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *(MLORA_GLOBAL f32x4 *)(p + (d * 4 + i) * 64) = f32x4{dq[0][d][4 * i], dq[0][d][4 * i + 1], dq[0][d][4 * i + 2], dq[0][d][4 * i + 3]};
    return;
  }
  store_row<T, DP>(static_cast<T *>(ba.dq), oat, there, dq, ba.scale, a.D, lane);
}

// Adds the shares of dq in order and writes them out. bf16: in the order of its kernel's registers; float32: rows in order.
template <class T, int DP>
__global__ __launch_bounds__(256) void past_dq_join_kernel(const PastBwdArgs ba) {
  const PastArgs &a = ba.f;
  constexpr int ND = DP / 32;
  const int64_t per = sizeof(T) == 2 ? (int64_t)a.B * a.row_tiles * a.Hk * 4 * ND * 4 * 64 : (int64_t)a.B * a.Hk * a.rows * (a.D / 4);
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  int hk, r, ch;
  int64_t b;
  if constexpr (sizeof(T) == 2) {  // per is a multiple of 256
    int64_t u = e / 64;
    const int lane = (int)(e % 64), i = (int)(u % 4), d = (int)(u / 4 % ND), wave = (int)(u / 4 / ND % 4);
    u /= 4 * ND * 4;  // (b, row tile, hk)
    hk = (int)(u % a.Hk), r = (int)(u / a.Hk % a.row_tiles) * 128 + wave * 32 + (lane & 31);
    b = u / a.Hk / a.row_tiles, ch = 32 * d + 8 * i + 4 * (lane >> 5);
    if (r >= a.rows || ch >= a.D) return;
  } else {
    if (e >= per) return;
    const int64_t u = e / (a.D / 4);
    ch = (int)(e % (a.D / 4)) * 4, r = (int)(u % a.rows), hk = (int)(u / a.rows % a.Hk), b = u / a.rows / a.Hk;
  }
  f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = 0; s < a.splits; ++s) x += *(const MLORA_GLOBAL f32x4 *)(ba.part + s * per + e);
  x *= ba.scale;
  T *p = static_cast<T *>(ba.dq) + (b * a.Lq + r / a.G) * a.H * a.D + (int64_t)(hk * a.G + r % a.G) * a.D + ch;
  if constexpr (sizeof(T) == 2) *(MLORA_GLOBAL u32x2 *)p = u32x2{pack2_bf16(x[0], x[1]), pack2_bf16(x[2], x[3])};
  else *(MLORA_GLOBAL f32x4 *)p = x;
}

constexpr int kF32Keys = 32;  // of a workgroup in float32

// A workgroup of dk / dv: which keys, and which share of the rows that see them. Blocks of the prefix come first, then those
// that hold a sink (both meet many rows and are shared out), then the other own ones.
struct KeyJob {
  int prefix, block, o, hk, sp, splits;
  int64_t part;  // index of the first share's tile in its class
  __device__ __forceinline__ void init(const PastBwdArgs &ba, int id) {
    const PastArgs &a = ba.f;
    const int groups = a.B / a.each;
    const int np = groups * a.Hk * ba.prefix_blocks * ba.prefix_splits, ns = a.B * a.Hk * ba.sink_blocks * ba.sink_splits;
    prefix = id < np;
    const bool sink = !prefix && id < np + ns;
    id -= prefix ? 0 : sink ? np : np + ns;
    const int first = prefix || sink ? 0 : ba.sink_blocks;
    const int blocks = prefix ? ba.prefix_blocks : sink ? ba.sink_blocks : ba.key_blocks - ba.sink_blocks;
    splits = prefix ? ba.prefix_splits : sink ? ba.sink_splits : ba.own_splits;
    hk = id % a.Hk, id /= a.Hk;
    block = id % blocks, id /= blocks;
    sp = id % splits, o = id / splits;
    part = (prefix ? 0 : sink ? ba.sink_part : ba.own_part);
    items = (int64_t)(prefix ? groups : a.B) * a.Hk * blocks;
    item = ((int64_t)o * a.Hk + hk) * blocks + block;
    block += first;
  }
  int64_t items, item;
};

// bf16: KW waves own 32 keys each (K fragments in registers; V in LDS, two waves per SIMD leave no room for it) and share tiles of query
// rows of one head in LDS: q, the output's gradient and the rows' x, delta and a, NB buffers, so that a tile has NB - 1 others' time to
// arrive in. RG 2: two such groups take half of every tile's rows each and add their sums at the end, so that half the keys
// fill a compute unit.
template <int DP, int RG>
constexpr int kDkvBuffers = DP == 128 && RG == 1 ? 2 : 3;

template <int DP, int KW, int RG>
__global__ __launch_bounds__((64 * KW * RG), 2) void past_dkv_kernel(const PastBwdArgs ba) {
  using T = uint16_t;
  const PastArgs &a = ba.f;
  constexpr int NW = KW * RG, QT = 64, NB = kDkvBuffers<DP, RG>, ND = DP / 32, NS = DP / 16;
  using Tile = PastTile<DP>;
  constexpr int TB = Tile::template bytes<QT>(), N = QT / Tile::ROWS / NW, VB = Tile::template bytes<32>();
  static_assert(NW >= 4 && (NB - 2) * (2 * N + 1) < 64, "a wave for each of a row's values; the loads on their way");
  // q and the output's gradient of every buffer; V; x, delta and a (and nothing) of every buffer's rows
  constexpr int ST = 4 * 256;
  __shared__ u32x4 smem[(NB * (2 * TB + ST) + KW * VB) / 16];
  MLORA_LDS char *lds = (MLORA_LDS char *)smem;
  const int wave = wave_id(), kw = wave % KW, rg = wave / KW, lane = threadIdx.x & 63;
  KeyJob job;
  job.init(ba, blockIdx.x);
  const int hk = job.hk;
  Sample s{0, 0};
  if (!job.prefix) s = uniform(sample_of(a, job.o));
  const int len = job.prefix ? prefix_keys(a, job.o) : s.n;
  const int key0 = (job.block * KW + kw) * 32, key = key0 + (lane & 31);
  const bool live = key < len;
  const uint64_t live_bits = low_bits(min(len - key0, 32));
  const T *kp = static_cast<const T *>(job.prefix ? a.pk : a.k) + job.o * (job.prefix ? a.pk_sb : a.k_sb) + hk * (job.prefix ? a.pk_sh : a.k_sh);
  const T *vp = static_cast<const T *>(job.prefix ? a.pv : a.v) + job.o * (job.prefix ? a.pv_sb : a.v_sb) + hk * (job.prefix ? a.pv_sh : a.v_sh);
  const int64_t k_sl = job.prefix ? a.pk_sl : a.k_sl, v_sl = job.prefix ? a.pv_sl : a.v_sl;
  Frag<T> k[NS];
#pragma unroll
  for (int ks = 0; ks < NS; ++ks) {
    const int d = 16 * ks + 8 * (lane >> 5);
    load_frag(kp, key * k_sl + d, live && d < a.D, k[ks]);
  }
  MLORA_LDS char *vt = lds + NB * 2 * TB + kw * VB, *values = lds + NB * 2 * TB + KW * VB;
  if (rg == 0) {
    PastLoader<DP, 32 / Tile::ROWS> vl;
    vl.init(lane, 0, 1, v_sl, a.D);
    vl.load(vp + (int64_t)key0 * v_sl, live_bits, vt);
  }
  f32x16 dk[1][ND], dv[1][ND];
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) dk[0][d][i] = 0.f, dv[0][d][i] = 0.f;
  // the tokens whose rows see a key: those from the key's chunk on, to the last whose window reaches it (positions)
  auto from = [&](int j) __attribute__((always_inline)) { return (int)((uint32_t)j / (uint32_t)a.chunk) * a.chunk; };
  auto to = [&](int j) __attribute__((always_inline)) {
    return job.prefix || j < a.sinks ? kEver : (int)((uint32_t)(j + a.window) / (uint32_t)a.chunk) * a.chunk;
  };
  const int bk0 = job.block * KW * 32, bk1 = min(bk0 + KW * 32, len) - 1;  // the block's keys
  int i0 = 0, i1 = bk0 < len ? a.Lq : 0;  // the block's tokens, of an own block
  if (!job.prefix && bk0 < len) {
    const int last = bk0 < a.sinks ? kEver : to(bk1);
    i0 = max(from(bk0) - s.start, 0), i1 = max(min(min(last, s.n) - s.start, a.Lq), i0);
  }
  const int tile0 = i0 / QT, head_tiles = max((i1 + QT - 1) / QT - tile0, 0), tiles = head_tiles * a.G * (job.prefix ? a.each : 1);
  const int t0 = (int)((int64_t)tiles * job.sp / job.splits), t1 = (int)((int64_t)tiles * (job.sp + 1) / job.splits);
  // rows of the wave's keys: all of them see tokens [full_a, full_b), none of them any outside [some_a, some_b)
  int full_a = 0, full_b = kEver, some_a = 0, some_b = kEver, mine_a = 0, mine_b = kEver;
  if (!job.prefix && key0 < len) {
    const int k1 = min(key0 + 31, len - 1), k2 = max(key0, min(a.sinks, k1));
    some_a = from(key0), full_a = from(k1), full_b = to(k2), some_b = key0 < a.sinks ? kEver : to(k1);
    mine_a = from(key), mine_b = to(key);
  }
  PastLoader<DP, N> ql, gl;
  ql.init(lane, wave, NW, a.q_sl, a.D), gl.init(lane, wave, NW, ba.g_sl, a.D);
  const int64_t all = (int64_t)a.B * a.Hk * a.rows;
  PastReader<DP> fr, vr;
  fr.init(lane, lds + rg * Tile::template bytes<32>()), vr.init(lane, vt);
  // the tile to load next: its place in its head, the head and the sample (of a prefix's group)
  int tile = head_tiles > 0 ? t0 % head_tiles : 0, head = head_tiles > 0 ? t0 / head_tiles % a.G : 0;
  int member = job.prefix && head_tiles > 0 ? t0 / head_tiles / a.G : 0, loaded = t0;
  uint64_t rows[NB];  // of the tiles from the one at work on: those that are tokens
  int place[NB];      // and the position of the first
#pragma unroll
  for (int i = 0; i < NB; ++i) rows[i] = 0, place[i] = 0;
  auto stage = [&](int buf) __attribute__((always_inline)) {
    const int b = job.prefix ? job.o * a.each + member : job.o, i = (tile0 + tile) * QT, h = hk * a.G + head;
    uint64_t live = 0;
    if (loaded < t1) {
      const Sample ks = job.prefix ? uniform(sample_of(a, b)) : s;
      live = low_bits(min(min(a.Lq, ks.n - ks.start) - i, QT)) & ~low_bits(-ks.start - i);
      place[NB - 1] = ks.start + i;
    }
    rows[NB - 1] = live;
    // behind the last tile nothing is read; every stage has the same number of loads
    const int at = loaded < t1 ? i : 0, from_b = loaded < t1 ? b : job.prefix ? job.o * a.each : job.o;
    ql.load(static_cast<const T *>(a.q) + from_b * a.q_sb + h * a.q_sh + at * a.q_sl, live, lds + buf * 2 * TB);
    gl.load(static_cast<const T *>(ba.g) + from_b * ba.g_sb + h * ba.g_sh + at * ba.g_sl, live, lds + buf * 2 * TB + TB);
    const int which = min(wave, 3);
    const float *x = (which == 1 ? ba.delta : a.stats + (which == 2 ? all : 0)) + ((int64_t)from_b * a.Hk + hk) * a.rows + (int64_t)at * a.G + head;
    const bool on = which < 3 && ((live >> lane) & 1);  // the others read as zero: they are masked
    __builtin_amdgcn_raw_ptr_buffer_load_lds(make_rsrc(x, (int64_t)kOOB), (MLORA_LDS void *)(values + buf * ST + which * 256), 4,
                                             on ? lane * a.G * 4 : kOOB, 0, 0, 0);
    ++loaded;
    if (++tile == head_tiles) {
      tile = 0;
      if (++head == a.G) head = 0, ++member;
    }
  };
  auto step = [&](int buf, int p0) __attribute__((always_inline)) {  // p0: the position of the tile's first token
    if (!job.prefix && (p0 + QT <= some_a || p0 >= some_b)) return;
    // rows that are no tokens too: a key that none of the tokens sees may hold anything
    const bool masked = rows[0] != low_bits(QT) || (!job.prefix && (p0 < full_a || p0 + QT > full_b));
    uint64_t mine = rows[0];
    const MLORA_LDS char *val = values + buf * ST;
    if (masked && !job.prefix) mine &= low_bits(mine_b - p0) & ~low_bits(mine_a - p0);
    mine >>= 4 * (lane >> 5) + 32 * rg;
    static_for<QT / 32 / RG>([&](auto block) __attribute__((always_inline)) {
      constexpr int qb = decltype(block)::value;
      const int at = 8 * (qb + rg) + (lane >> 5);  // of the rows' x, delta and a
      __builtin_amdgcn_sched_barrier(0);  // between the phases too: interleaved, they spill
      f32x16 sc, dp;
#pragma unroll
      for (int i = 0; i < 16; ++i) sc[i] = 0.f, dp[i] = 0.f;
      struct Three {
        Frag<T> q, g, v;
      };
      read_ahead<NS, 2>(
          [&](auto ks) __attribute__((always_inline)) {
            Three f;
            fr.template rows<0, 32 * qb>(ks, f.q);
            fr.template rows<TB, 32 * qb>(ks, f.g);
            vr.template rows<0, 0>(ks, f.v);
            return f;
          },
          [&](auto ks, const Three &f) __attribute__((always_inline)) {  // the two sums in turn: a sum waits for its last product
            sc = mma16(f.q, k[ks], sc);
            dp = mma16(f.g, f.v, dp);
          });
      if (masked) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const bool on = (mine >> (32 * qb + 8 * (i / 4) + i % 4)) & 1;
          sc[i] = on ? sc[i] : -INFINITY, dp[i] = on ? dp[i] : 0.f;
        }
      }
#pragma unroll
      for (int i4 = 0; i4 < 4; ++i4) {
        const f32x4 x = *(const lds_f4 *)(val + 0 + 16 * (at + 2 * i4)), delta = *(const lds_f4 *)(val + 256 + 16 * (at + 2 * i4));
        const f32x4 shift = *(const lds_f4 *)(val + 512 + 16 * (at + 2 * i4));
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[4 * i4 + j] - shift[j], a.c, -x[j]));
          sc[4 * i4 + j] = p;
          dp[4 * i4 + j] = p * (dp[4 * i4 + j] - delta[j]);
        }
      }
      Frag<T> pf[2], df[2];
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) to_frag(sc, ks, pf[ks]), to_frag(dp, ks, df[ks]);
      __builtin_amdgcn_sched_barrier(0);
      read_ahead<4 * ND, 3>(
          [&](auto u) __attribute__((always_inline)) {
            constexpr int U = decltype(u)::value, VALUE = U / (2 * ND), KS = U / ND % 2;
            Frag<T> f;
            fr.template cols<VALUE ? 0 : TB, 32 * qb + 16 * KS>(U % ND, f);
            return f;
          },
          [&](auto u, const Frag<T> &f) __attribute__((always_inline)) {
            constexpr int U = decltype(u)::value, KS = U / ND % 2;
            if constexpr (U / (2 * ND) == 0) dv[0][U % ND] = mma16(f, pf[KS], dv[0][U % ND]);
            else dk[0][U % ND] = mma16(f, df[KS], dk[0][U % ND]);
          });
      return true;
    });
  };
  auto shift = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i + 1 < NB; ++i) rows[i] = rows[i + 1], place[i] = place[i + 1];
  };
  if (t0 < t1) {
#pragma unroll
    for (int i = 0; i < NB - 1; ++i) shift(), stage(i);
    shift();
  }
  int buf = 0;
  for (int t = t0; t < t1; ++t) {
    wait_vmcnt<(NB - 2) * (2 * N + 1)>();
    lds_pipeline_barrier();  // tile t is in LDS, and every wave has read tile t - 1
    stage(buf == 0 ? NB - 1 : buf - 1);
    if (key0 < len) step(buf, place[0]);
    shift();
    fr.move(buf == NB - 1 ? -(NB - 1) * 2 * TB : 2 * TB);
    buf = buf == NB - 1 ? 0 : buf + 1;
  }
  wait_vmcnt<0>();
  if (!live) {  // a column of keys that are none holds whatever its zeroed fragments gave
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) dk[0][d][i] = 0.f, dv[0][d][i] = 0.f;
  }
  if constexpr (RG == 2) {  // the first group has dk, the second dv
    static_assert(KW * ND * 4 * 64 <= NB * 2 * TB / 16, "the sums fit the buffers");
    f32x4 *to = (f32x4 *)smem + kw * (ND * 4 * 64) + lane;
    auto hand = [&](const f32x16 (&x)[1][ND]) __attribute__((always_inline)) {
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) to[(d * 4 + i) * 64] = f32x4{x[0][d][4 * i], x[0][d][4 * i + 1], x[0][d][4 * i + 2], x[0][d][4 * i + 3]};
    };
    auto take = [&](f32x16 (&x)[1][ND]) __attribute__((always_inline)) {
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const f32x4 y = to[(d * 4 + i) * 64];
#pragma unroll
          for (int j = 0; j < 4; ++j) x[0][d][4 * i + j] += y[j];
        }
    };
    __syncthreads();
    if (rg == 1) hand(dk);
    __syncthreads();
    if (rg == 0) take(dk);
    __syncthreads();
    if (rg == 0) hand(dv);
    __syncthreads();
    if (rg == 1) take(dv);
  }
  const bool has_dk = RG == 1 || rg == 0, has_dv = RG == 1 || rg == 1;
  if (job.splits > 1) {
    f32x4 *p = ba.part + job.part + ((job.sp * job.items + job.item) * KW + kw) * (2 * ND * 4 * 64) + lane;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (has_dk) *(MLORA_GLOBAL f32x4 *)(p + (d * 4 + i) * 64) = f32x4{dk[0][d][4 * i], dk[0][d][4 * i + 1], dk[0][d][4 * i + 2], dk[0][d][4 * i + 3]};
        if (has_dv) *(MLORA_GLOBAL f32x4 *)(p + ((ND + d) * 4 + i) * 64) = f32x4{dv[0][d][4 * i], dv[0][d][4 * i + 1], dv[0][d][4 * i + 2], dv[0][d][4 * i + 3]};
      }
    return;
  }
  const int L = job.prefix ? a.Lp : a.Lk;
  const int64_t at = ((int64_t)job.o * L * a.Hk + hk) * a.D;
  const float fk[1] = {ba.scale}, fv[1] = {1.f};
  auto key_at = [&](int key) { return (int64_t)key * a.Hk * a.D; };
  if (has_dk) store_rows<T, DP, 1>(static_cast<T *>(job.prefix ? ba.dpk : ba.dk) + at, dk, fk, key0, L, key_at, a.D, lane);
  if (has_dv) store_rows<T, DP, 1>(static_cast<T *>(job.prefix ? ba.dpv : ba.dv) + at, dv, fv, key0, L, key_at, a.D, lane);
}

// Adds the shares of the key blocks of all classes that have several (the prefix's, those with a sink, the others) in order and
// writes them out; which: its workgroups of each class. bf16: a share is in the order of its kernel's registers, [wave][dk, dv][..];
// float32: [key][dk, dv][D].
struct JoinBlocks {
  int64_t upto[3];  // workgroups up to the end of each class
};
template <class T, int DP, int KW>
__global__ __launch_bounds__(256) void past_dkv_join_kernel(const PastBwdArgs ba, const JoinBlocks which) {
  const PastArgs &a = ba.f;
  constexpr int ND = DP / 32, KEYS = sizeof(T) == 2 ? 32 * KW : kF32Keys;
  const int64_t id = blockIdx.x;
  const int cls = id < which.upto[0] ? 0 : id < which.upto[1] ? 1 : 2;
  const bool prefix = cls == 0;
  const int blocks = prefix ? ba.prefix_blocks : cls == 1 ? ba.sink_blocks : ba.key_blocks - ba.sink_blocks;
  const int splits = prefix ? ba.prefix_splits : cls == 1 ? ba.sink_splits : ba.own_splits;
  const f32x4 *part = ba.part + (prefix ? 0 : cls == 1 ? ba.sink_part : ba.own_part);
  const int64_t items = (int64_t)(prefix ? a.B / a.each : a.B) * a.Hk * blocks;
  const int64_t per = items * (sizeof(T) == 2 ? KW * 2 * ND * 4 * 64 : KEYS * (a.D / 2));
  const int64_t e = (id - (cls == 0 ? 0 : which.upto[cls - 1])) * 256 + threadIdx.x;
  if (e >= per) return;
  f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = 0; s < splits; ++s) x += *(const MLORA_GLOBAL f32x4 *)(part + s * per + e);
  int64_t u;
  int in, ch, value;  // key within the block
  if constexpr (sizeof(T) == 2) {
    u = e / 64;
    const int lane = (int)(e % 64), i = (int)(u % 4), d = (int)(u / 4 % ND);
    value = (int)(u / 4 / ND % 2), u /= 4 * ND * 2;
    in = (int)(u % KW) * 32 + (lane & 31), ch = 32 * d + 8 * i + 4 * (lane >> 5), u /= KW;
  } else {
    u = e / (a.D / 4), ch = (int)(e % (a.D / 4)) * 4;
    value = (int)(u % 2), u /= 2, in = (int)(u % KEYS), u /= KEYS;
  }
  const int64_t key = (u % blocks + (cls == 2 ? ba.sink_blocks : 0)) * KEYS + in, bh = u / blocks;
  const int L = prefix ? a.Lp : a.Lk;
  if (key >= L || ch >= a.D) return;
  void *base = value ? (prefix ? ba.dpv : ba.dv) : prefix ? ba.dpk : ba.dk;
  T *p = static_cast<T *>(base) + ((bh / a.Hk * L + key) * a.Hk + bh % a.Hk) * a.D + ch;
  if (!value) x *= ba.scale;
  if constexpr (sizeof(T) == 2) *(MLORA_GLOBAL u32x2 *)p = u32x2{pack2_bf16(x[0], x[1]), pack2_bf16(x[2], x[3])};
  else *(MLORA_GLOBAL f32x4 *)p = x;
}

// ---------------------------------------------------------------- backward, float32
//
// As the forward of few rows: 32 rows (or keys) per workgroup, the waves take different tiles and their sums are joined through LDS.
// A product of 32 x 32 x 64 channels holds the matrix core for 2048 cycles, so that reading the tiles again for every 32 rows
// costs less than it would in bf16.
template <int DP, int NW>
__global__ __launch_bounds__((64 * NW), (kFewWaves<float, DP> / 4)) void past_dq_f32_kernel(const PastBwdArgs ba) {
  const PastArgs &a = ba.f;
  using Tile = HeadTile<float, DP>;
  constexpr int KT = 32, ND = DP / 16, NS = DP / 32, TB = KT * Tile::RB;
  static_assert(2 * ND * 64 * 16 <= 2 * TB, "a wave's sums fit its buffer");
  __shared__ u32x4 smem[2 * TB * NW / 16];
  const int wave = wave_id(), lane = threadIdx.x & 63;
  MLORA_LDS char *lds = (MLORA_LDS char *)smem + wave * 2 * TB;
  Job job;
  job.init(a, blockIdx.x);
  const int hk = job.hk, r0 = job.rt * 32, group = job.b / a.each;
  const Sample s = uniform(sample_of(a, job.b));
  KeyTiles<KT> tiles;
  WaveRows wr;
  tiles.init(a, a.with_prefix ? prefix_keys(a, group) : 0, s.n, max(s.start + r0 / a.G, 0), min(s.start + min(r0 + 31, a.rows - 1) / a.G, s.n - 1));
  wr.init(a, s, r0, min(r0 + 32, a.rows));
  const int t1 = job.share(tiles.count, job.sp + 1), t0 = min(job.share(tiles.count, job.sp) + wave, t1);
  TileStream<float, DP, KT, TB / 1024> in;
  in.init(a, job.b, group, hk, 0, 1, lane, tiles, t0, t1);
  if (t0 < t1) in.stage(a, tiles, t0, lds);
  FewReader<float, DP> fr;
  fr.init(lane, lds);
  Row x[2];
  Frag<float> q[2][NS], g[2][NS];
  float delta[2], ref[2], shift[2];
  f32x4 dq[2][ND];
  const int64_t all = (int64_t)a.B * a.Hk * a.rows;
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    x[n] = row_of(a, false, job.b, hk, r0 + 16 * n + (lane & 15), a.rows, s);
    const bool on = x[n].on;
    Frag<float> o[NS];
    load_row<float, DP>(static_cast<const float *>(a.q) + row_place(a, x[n], hk, a.q_sb, a.q_sl, a.q_sh), on, a.D, lane, q[n]);
    load_row<float, DP>(static_cast<const float *>(ba.g) + row_place(a, x[n], hk, ba.g_sb, ba.g_sl, ba.g_sh), on, a.D, lane, g[n]);
    load_row<float, DP>(static_cast<const float *>(a.out) + row_place(a, x[n], hk, (int64_t)a.Lq * a.H * a.D, (int64_t)a.H * a.D, a.D), on, a.D, lane, o);
    ref[n] = on ? a.stats[x[n].at] : INFINITY, shift[n] = on ? a.stats[all + x[n].at] : 0.f;
    delta[n] = 0.f;
#pragma unroll
    for (int ks = 0; ks < NS; ++ks)
#pragma unroll
      for (int j = 0; j < 8; ++j) delta[n] += g[n][ks].v[j] * o[ks].v[j];
    delta[n] = quarter_sum(delta[n]);
    if (job.sp == 0 && wave == 0 && lane < 16 && r0 + 16 * n + lane < a.rows) ba.delta[x[n].at] = delta[n];
#pragma unroll
    for (int d = 0; d < ND; ++d) dq[n][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  for (int t = t0; t < t1; t += NW) {
    wait_vmcnt<0>();  // tile t is in this wave's buffer
    asm volatile("" ::: "memory");
    const int k0 = tiles.key0(t);
    const bool o = tiles.own(t), rows = o && !wr.everything(a, k0, KT);
    const uint32_t bits = (uint32_t)tiles.bits(t, t1);
    f32x4 sc[2][2], dp[2][2];
#pragma unroll
    for (int n = 0; n < 2; ++n) sc[n][0] = sc[n][1] = dp[n][0] = dp[n][1] = f32x4{0.f, 0.f, 0.f, 0.f};
    few_scores<0, DP, 2>(fr, q, sc);
    few_scores<TB, DP, 2>(fr, g, dp);
    Frag<float> ds[2];
    const bool masked = rows || bits != ~0u;
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      const uint32_t mine = (rows ? (uint32_t)x[n].bits(a, k0) : bits) >> (4 * (lane >> 4));
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float y = sc[n][j / 4][j % 4], z = dp[n][j / 4][j % 4];
        if (masked && !((mine >> (16 * (j / 4) + j % 4)) & 1)) y = -INFINITY, z = 0.f;
        ds[n].v[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(y - shift[n], a.c, -ref[n])) * (z - delta[n]);
      }
    }
    few_weigh<0, DP, 2>(fr, ds, dq);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // and read
    if (t + NW < t1) in.stage(a, tiles, t + NW, lds);
  }
  f32x4 *mine = (f32x4 *)smem + wave * (2 * TB / 16);
#pragma unroll
  for (int n = 0; n < 2; ++n)
#pragma unroll
    for (int d = 0; d < ND; ++d) mine[(n * ND + d) * 64 + lane] = few_vector<float, ND>(dq[n], d);
  __syncthreads();
  for (int u = wave; u < 2 * ND; u += NW) {
    const int n = u / ND, d = u % ND, ch = few_channel<float>(d, lane), r = r0 + 16 * n + (lane & 15);
    f32x4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < NW; ++w) y += ((const f32x4 *)smem + w * (2 * TB / 16))[u * 64 + lane];
    if (r >= a.rows || ch >= a.D) continue;
    const Row &xr = n == 0 ? x[0] : x[1];
    if (!xr.on) y = f32x4{0.f, 0.f, 0.f, 0.f};
    if (a.splits > 1) ba.part[(job.sp * all + xr.at) * (a.D / 4) + ch / 4] = y;
    else *(MLORA_GLOBAL f32x4 *)(static_cast<float *>(ba.dq) + row_place(a, xr, hk, (int64_t)a.Lq * a.H * a.D, (int64_t)a.H * a.D, a.D) + ch) = y * ba.scale;
  }
}

template <int DP, int NW>
__global__ __launch_bounds__((64 * NW), (kFewWaves<float, DP> / 4)) void past_dkv_f32_kernel(const PastBwdArgs ba) {
  const PastArgs &a = ba.f;
  using Tile = HeadTile<float, DP>;
  constexpr int QT = 32, ND = DP / 16, NS = DP / 32, TB = QT * Tile::RB, N = TB / 1024;
  static_assert(2 * ND * 64 * 16 <= 2 * TB, "half of a wave's sums fit its buffer");
  __shared__ u32x4 smem[2 * TB * NW / 16 + NW * 24];  // q and the output's gradient of every wave; x, delta and a of its rows
  const int wave = wave_id(), lane = threadIdx.x & 63;
  MLORA_LDS char *lds = (MLORA_LDS char *)smem + wave * 2 * TB;
  float *stats = (float *)(smem + 2 * TB * NW / 16 + wave * 24);  // [3][32]
  KeyJob job;
  job.init(ba, blockIdx.x);
  const int hk = job.hk;
  Sample s{0, 0};
  if (!job.prefix) s = uniform(sample_of(a, job.o));
  const int len = job.prefix ? prefix_keys(a, job.o) : s.n, key0 = job.block * kF32Keys;
  const float *kp = static_cast<const float *>(job.prefix ? a.pk : a.k) + job.o * (job.prefix ? a.pk_sb : a.k_sb) + hk * (job.prefix ? a.pk_sh : a.k_sh);
  const float *vp = static_cast<const float *>(job.prefix ? a.pv : a.v) + job.o * (job.prefix ? a.pv_sb : a.v_sb) + hk * (job.prefix ? a.pv_sh : a.v_sh);
  const int64_t k_sl = job.prefix ? a.pk_sl : a.k_sl, v_sl = job.prefix ? a.pv_sl : a.v_sl;
  // the tokens whose rows see a key, as in the bf16 kernel
  auto from = [&](int j) __attribute__((always_inline)) { return (int)((uint32_t)j / (uint32_t)a.chunk) * a.chunk; };
  auto to = [&](int j) __attribute__((always_inline)) {
    return job.prefix || j < a.sinks ? kEver : (int)((uint32_t)(j + a.window) / (uint32_t)a.chunk) * a.chunk;
  };
  const int last_key = min(key0 + kF32Keys, len) - 1;
  int i0 = 0, i1 = key0 < len ? a.Lq : 0, full_a = 0, full_b = kEver;
  if (!job.prefix && key0 < len) {
    const int last = key0 < a.sinks ? kEver : to(last_key);
    i0 = max(from(key0) - s.start, 0), i1 = max(min(min(last, s.n) - s.start, a.Lq), i0);
    full_a = from(last_key), full_b = to(max(key0, min(a.sinks, last_key)));
  }
  const int tile0 = i0 / QT, head_tiles = max((i1 + QT - 1) / QT - tile0, 0), tiles = head_tiles * a.G * (job.prefix ? a.each : 1);
  const int t1 = (int)((int64_t)tiles * (job.sp + 1) / job.splits), t0 = min((int)((int64_t)tiles * job.sp / job.splits) + wave, t1);
  TileLoader<float, DP, N> ql, gl;
  ql.init(lane, 0, 1, a.q_sl, a.D), gl.init(lane, 0, 1, ba.g_sl, a.D);
  const int64_t all = (int64_t)a.B * a.Hk * a.rows;
  uint32_t rows = 0;  // the rows on their way that are tokens
  int p0 = 0;         // the position of the first
  float x = 0.f, y = 0.f, z = 0.f;  // of lane's row: x, delta, a
  auto stage = [&](int t) __attribute__((always_inline)) {
    const int h = t / head_tiles, m = h / a.G, b = job.prefix ? job.o * a.each + m : job.o, i = (tile0 + t - h * head_tiles) * QT;
    const Sample ks = job.prefix ? uniform(sample_of(a, b)) : s;
    const int head = h - m * a.G;
    const uint64_t live = low_bits(min(min(a.Lq, ks.n - ks.start) - i, QT)) & ~low_bits(-ks.start - i);
    rows = (uint32_t)live, p0 = ks.start + i;
    const float *q = static_cast<const float *>(a.q) + b * a.q_sb + (hk * a.G + head) * a.q_sh + i * a.q_sl;
    const float *g = static_cast<const float *>(ba.g) + b * ba.g_sb + (hk * a.G + head) * ba.g_sh + i * ba.g_sl;
    if (live == low_bits(QT)) ql.load_all(q, lds), gl.load_all(g, lds + TB);
    else ql.load(q, live, lds), gl.load(g, live, lds + TB);
    const int64_t at = ((int64_t)b * a.Hk + hk) * a.rows + (int64_t)(i + (lane & 31)) * a.G + head;
    const bool on = (rows >> (lane & 31)) & 1;
    x = on ? a.stats[at] : INFINITY, y = on ? ba.delta[at] : 0.f, z = on ? a.stats[all + at] : 0.f;  // rows without a token: P = 0
  };
  if (t0 < t1) stage(t0);
  Frag<float> k[2][NS], v[2][NS];
  f32x4 dk[2][ND], dv[2][ND];
  int mine_a[2], mine_b[2];
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    const int64_t key = key0 + 16 * n + (lane & 15);
    const bool live = key < len;
    load_row<float, DP>(kp + (live ? key * k_sl : 0), live, a.D, lane, k[n]);
    load_row<float, DP>(vp + (live ? key * v_sl : 0), live, a.D, lane, v[n]);
    mine_a[n] = job.prefix ? 0 : from((int)key), mine_b[n] = to((int)key);
#pragma unroll
    for (int d = 0; d < ND; ++d) dk[n][d] = dv[n][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  FewReader<float, DP> fr;
  fr.init(lane, lds);
  for (int t = t0; t < t1; t += NW) {
    wait_vmcnt<0>();  // tile t is in this wave's buffer
    if (lane < 32) stats[lane] = x, stats[32 + lane] = y, stats[64 + lane] = z;
    asm volatile("" ::: "memory");
    // rows that are no tokens too: a key that none of the tokens sees may hold anything
    const bool part = !job.prefix && (p0 < full_a || p0 + QT > full_b), masked = part || rows != ~0u;
    f32x4 sc[2][2], dp[2][2];
#pragma unroll
    for (int n = 0; n < 2; ++n) sc[n][0] = sc[n][1] = dp[n][0] = dp[n][1] = f32x4{0.f, 0.f, 0.f, 0.f};
    few_scores<0, DP, 2>(fr, k, sc);
    few_scores<TB, DP, 2>(fr, v, dp);
    Frag<float> pf[2], df[2];
    uint32_t mine[2];
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      mine[n] = rows;
      if (part) mine[n] &= (uint32_t)(low_bits(mine_b[n] - p0) & ~low_bits(mine_a[n] - p0));
      mine[n] >>= 4 * (lane >> 4);
    }
#pragma unroll
    for (int qb = 0; qb < 2; ++qb) {
      const int r = 16 * qb + 4 * (lane >> 4);
      const f32x4 ref = *(const f32x4 *)(stats + r), delta = *(const f32x4 *)(stats + 32 + r), shift = *(const f32x4 *)(stats + 64 + r);
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float u = sc[n][qb][i], w = dp[n][qb][i];
          if (masked && !((mine[n] >> (16 * qb + i)) & 1)) u = -INFINITY, w = 0.f;
          const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(u - shift[i], a.c, -ref[i]));
          pf[n].v[4 * qb + i] = p, df[n].v[4 * qb + i] = p * (w - delta[i]);
        }
    }
    few_weigh<TB, DP, 2>(fr, pf, dv);
    few_weigh<0, DP, 2>(fr, df, dk);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // and read
    if (t + NW < t1) stage(t + NW);
  }
  // the waves' sums, dk and then dv, through the buffers
  const int L = job.prefix ? a.Lp : a.Lk;
#pragma unroll
  for (int value = 0; value < 2; ++value) {
    __syncthreads();
    f32x4 *to_sum = (f32x4 *)smem + wave * (2 * TB / 16);
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int d = 0; d < ND; ++d) to_sum[(n * ND + d) * 64 + lane] = few_vector<float, ND>(value ? dv[n] : dk[n], d);
    __syncthreads();
    for (int u = wave; u < 2 * ND; u += NW) {
      const int in = 16 * (u / ND) + (lane & 15), ch = few_channel<float>(u % ND, lane);
      const int64_t key = key0 + in;
      f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < NW; ++w) sum += ((const f32x4 *)smem + w * (2 * TB / 16))[u * 64 + lane];
      if (ch >= a.D) continue;
      if (key >= len) sum = f32x4{0.f, 0.f, 0.f, 0.f};  // whatever its zeroed fragments gave
      if (job.splits > 1) {
        ba.part[job.part + (((job.sp * job.items + job.item) * kF32Keys + in) * 2 + value) * (a.D / 4) + ch / 4] = sum;
      } else if (key < L) {
        float *p = static_cast<float *>(value ? (job.prefix ? ba.dpv : ba.dv) : job.prefix ? ba.dpk : ba.dk);
        *(MLORA_GLOBAL f32x4 *)(p + ((job.o * (int64_t)L + key) * a.Hk + hk) * a.D + ch) = value ? sum : sum * ba.scale;
      }
    }
  }
}

// The kernels are named here because hipcc's host pass does not instantiate a kernel that holds generic lambdas
// from a launch inside one.
#define MLORA_PAST(DP)                                                                           \
  template __global__ void past_fwd_kernel<DP>(const PastArgs);                                  \
  template __global__ void past_few_kernel<uint16_t, DP, 1, 8>(const PastArgs);                  \
  template __global__ void past_few_kernel<uint16_t, DP, 2, 8>(const PastArgs);                  \
  template __global__ void past_few_kernel<float, DP, 1, kFewWaves<float, DP>>(const PastArgs); \
  template __global__ void past_dq_kernel<DP>(const PastBwdArgs);                                \
  template __global__ void past_dkv_kernel<DP, 4, DP / 64>(const PastBwdArgs);
#define MLORA_PAST_F32(DP, NW)                                             \
  template __global__ void past_few_kernel<float, DP, 2, NW>(const PastArgs); \
  template __global__ void past_dq_f32_kernel<DP, NW>(const PastBwdArgs);
MLORA_PAST(64)
MLORA_PAST(128)
MLORA_PAST_F32(64, 8)
MLORA_PAST_F32(64, 4)
MLORA_PAST_F32(64, 2)
MLORA_PAST_F32(128, 4)
MLORA_PAST_F32(128, 2)
#undef MLORA_PAST
#undef MLORA_PAST_F32
template __global__ void past_dkv_f32_kernel<64, 8>(const PastBwdArgs);
template __global__ void past_dkv_f32_kernel<64, 4>(const PastBwdArgs);
template __global__ void past_dkv_f32_kernel<128, 4>(const PastBwdArgs);
template __global__ void past_dkv_f32_kernel<128, 2>(const PastBwdArgs);
template __global__ void past_dkv_kernel<128, 8, 1>(const PastBwdArgs);

// ------------------------------------------------------------------ host

constexpr int64_t kPastMostTokens = 1 << 28, kPastMostBlocks = INT32_MAX - 65536;

static int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
static int64_t between(int64_t x, int64_t lo, int64_t hi) { return x < lo ? lo : x > hi ? hi : x; }

// A call's sizes with options brought into the range where they differ, or a status.
struct PastSizes {
  bool f32;
  int64_t B, Lq, Lk, H, Hk, G, D, groups, each, Lp, rows, window, sinks, chunk, first;
};

static int past_sizes(PastSizes &z, const mlora_past_shape *s) {
  if (s == nullptr) return MLORA_ERR_INVALID;
  if (s->dtype != MLORA_BF16 && s->dtype != MLORA_F32) return MLORA_ERR_UNSUPPORTED;
  if (s->B < 0 || s->Lq < 0 || s->Lk < 0 || s->H < 1 || s->Hk < 1 || s->H % s->Hk != 0) return MLORA_ERR_INVALID;
  if (s->D < 8 || s->D % 8 != 0 || s->D > 128) return MLORA_ERR_UNSUPPORTED;
  if (s->window < 0 || s->sinks < 0 || s->chunk < 1 || (s->window > 0 && s->window < s->chunk)) return MLORA_ERR_INVALID;
  if (s->groups < 0 || s->Lp < 0 || (s->groups == 0 && s->Lp > 0) || (s->groups > 0 && s->B % s->groups != 0)) return MLORA_ERR_INVALID;
  if (!(s->scale > 0.f && s->scale * kLog2e < INFINITY)) return MLORA_ERR_INVALID;
  z.f32 = s->dtype == MLORA_F32;
  z.B = s->B, z.Lq = s->Lq, z.Lk = s->Lk, z.H = s->H, z.Hk = s->Hk, z.D = s->D, z.G = s->H / s->Hk, z.Lp = s->Lp;
  if (z.Lq > kPastMostTokens || z.Lk > kPastMostTokens || z.Lp > kPastMostTokens || z.H > 65536) return MLORA_ERR_LIMIT;
  z.groups = s->groups > 0 ? s->groups : z.B, z.each = z.groups > 0 ? z.B / z.groups : 1;
  z.rows = z.G * z.Lq;
  // workgroups: one per (sample, key head, 32 rows or keys at least), a few thousand shares beside them; rows of a group. What a launch
  // takes is checked of each (launch_fits)
  const int64_t most = kPastMostBlocks, blocks = ceil_div(z.rows, 32) + ceil_div(z.Lk, 32) + ceil_div(z.Lp, 32) + 1;
  if (z.rows > most || (z.B > 0 && (z.Hk > most / z.B || blocks > most / (z.B * z.Hk) || z.rows > most / z.B))) return MLORA_ERR_LIMIT;
  z.chunk = between(s->chunk, 1, z.Lk > 1 ? z.Lk : 1);  // from there on all keys are one chunk
  z.window = s->window > 0 ? between(s->window, z.chunk, z.Lk + z.chunk) : z.Lk + z.chunk;
  z.sinks = between(s->sinks, 0, z.Lk);
  z.first = between(s->first, -z.Lq, z.Lk);
  return MLORA_OK;
}

// Key tiles of kt keys that `rows` neighbouring rows of a sample see at most, the prefix aside.
static int64_t own_tiles(const PastSizes &z, int64_t rows, int64_t kt) {
  const int64_t all = ceil_div(z.Lk, kt), some = ceil_div(z.window + z.chunk + rows / z.G, kt) + 1 + ceil_div(z.sinks, kt);
  return some < all ? some : all;
}

// How a forward is cut. Up to 64 rows per key head, and all of them in float32, run waves over different keys, 32 rows per workgroup;
// more rows 128 per workgroup. Up to 64 rows of samples that share a prefix take it together, in workgroups of its own: then
// all shares are joined. Keys are shared out where there is less than a workgroup for every compute unit.
struct PastPlan {
  bool few, packed, packed_few;
  int waves;  // of few rows
  int64_t packed_tiles, packed_splits, row_tiles, splits, slots;
};

// How many waves a float32 workgroup has: `items` workgroups whose waves share `tiles` tiles. A tile waits for its loads, so that it
// takes a SIMD's one wave as long as two; fewer waves leave room for more workgroups on a compute unit. Measured as all / half / a quarter
// of the waves, us of the forward of 64 channels (the backward's dq goes the same way):
//   half above 256 workgroups: 200 of 12 tiles 14.0 / 14.3 / 19.3, 296 of 12 23.9 / 18.4 / 23.8, 448 of 26 40.8 / 35.5 / 59.0;
//   a quarter from 513 to 1024, which halves take in two rounds and quarters in one, where tiles are few: 600 of 8 31.9 / 24.2 / 22.0, 896 of
//   12 50.7 / 40.3 / 31.9, 1024 of 12 50.6 / 40.3 / 32.3 (544 of 12 loses: 32.0 / 26.8 / 30.5). Not where they are many: 600 of 18 44.3 / 36.6 / 43.1,
//   696 of 26 59.7 / 53.3 / 60.1, though a full second round would gain there too (1024 of 26 79.0 / 67.4 / 62.1).
// 128 channels, all / half of four: 296 of 5 25.0 / 19.8, 448 of 26 77.0 / 69.9, 2048 of 12 183.9 / 143.3. Where a half's second workgroup per unit
// is missing on most units and tiles are many, all would be faster: 296 of 26 41.6 / 67.1.
static int f32_waves(int64_t D, int64_t items, int64_t tiles) {
  const int most = D > 64 ? 4 : 8;
  if (items <= 256) return most;
  return D <= 64 && items > 512 && items <= 1024 && tiles <= 16 ? most / 4 : most / 2;
}

// Into how many shares the key tiles of `items` workgroups of 128 rows are cut, two of which share a compute unit: what takes least
// time, in microseconds. A tile of 64 keys takes 1.5 where a workgroup has the unit for itself and 2.0 where two share it (128
// channels; the ratio is what counts), a share one and a half tiles more for its start; its sums are written, read and joined by
// another launch (the forward's, row by row, at 4 TB/s, dq's, as they lie in registers, at 8). A frame of 1560 tokens on nine
// others, 12 heads (156 workgroups of 244 tiles): 381 us in one share, 188 in three; on 14040 keys that two samples share (312) 478
// and 362; by itself (156 of 25) 46 and 50: under 7 % it is not worth the launch.
static int64_t wide_shares(int64_t items, int64_t tiles, int64_t floats, double bytes_per_us) {
  int64_t best = 1;
  double least = 0;
  for (int64_t n = 1; n <= 16 && (n == 1 || tiles >= 8 * n); ++n) {
    const int64_t blocks = items * n, left = blocks % 512;
    double t = (2.0 * (double)(blocks / 512) + (left == 0 ? 0.0 : left <= 256 ? 1.5 : 2.0)) * ((double)ceil_div(tiles, n) + 1.5);
    if (n > 1) t += 5.0 + (double)blocks * (double)floats * 8 / bytes_per_us;
    if (n == 1 || t < 0.93 * least) least = t, best = n;
  }
  return best;
}

static PastPlan past_plan(const PastSizes &z) {
  PastPlan p{};
  const int waves = z.f32 && z.D > 64 ? 4 : 8;
  const int64_t few_rows = z.f32 ? INT64_MAX : 64, e = z.f32 ? 4 : 2;
  p.few = z.rows <= few_rows;
  p.packed = z.rows <= 64 && z.each > 1 && z.groups * (z.each - 1) * z.Lp * z.Hk * z.D * 2 * e > (16 << 20);
  p.row_tiles = ceil_div(z.rows, p.few ? 32 : 128);
  auto share = [&](int64_t items, int64_t tiles, bool few) -> int64_t {
    if (items <= 0) return 1;
    if (!few) return wide_shares(items, tiles, 128 * z.D, 4e6);
    // tiles that a share is worth its join for: one per wave (1024 keys in 4 shares 10.1 us, in 2 11.8, in one 11.3), from four per
    // wave on (576 keys in 2 shares 10.0 us, in one 7.2)
    return between(256 / items, 1, between(tiles < 4 * waves ? 1 : tiles / waves, 1, 64));
  };
  const int64_t kt = p.few || z.f32 ? 32 : 64;
  const int64_t prefix_tiles = p.packed ? 0 : ceil_div(z.Lp, kt);
  p.splits = share(z.B * z.Hk * p.row_tiles, own_tiles(z, p.few ? 32 : 128, kt) + prefix_tiles, p.few);
  if (p.packed) {
    const int64_t rows = z.each * z.rows;
    p.packed_few = rows <= few_rows;
    p.packed_tiles = ceil_div(rows, p.packed_few ? 32 : 128);
    p.packed_splits = share(z.groups * z.Hk * p.packed_tiles, ceil_div(z.Lp, p.packed_few || z.f32 ? 32 : 64), p.packed_few);
  }
  p.slots = p.splits + p.packed_splits;
  p.waves = waves;
  if (z.f32) {
    const int64_t own = z.B * z.Hk * p.row_tiles * p.splits, packed = z.groups * z.Hk * p.packed_tiles * p.packed_splits;
    p.waves = f32_waves(z.D, own + packed, ceil_div(own_tiles(z, 32, kt) + prefix_tiles, p.splits));
  }
  return p;
}

static int64_t past_floats(const PastPlan &p, const PastSizes &z) {
  return p.slots > 1 ? p.slots * ceil_div(z.B * z.Hk * z.rows * (z.D + 2), 4) * 4 : 0;
}

// HIP launches fewer than 2^32 work items (threads: a power of two).
static bool launch_fits(int64_t blocks, int64_t threads) { return blocks < ((int64_t)1 << 32) / threads; }

static int64_t packed_blocks(const PastPlan &p, const PastSizes &z) { return z.groups * z.Hk * p.packed_tiles * p.packed_splits; }
static int64_t own_blocks(const PastPlan &p, const PastSizes &z) { return z.B * z.Hk * p.row_tiles * p.splits; }

// Whether the rows of a few-row launch fit one block of 16.
static bool one_block(const PastPlan &p, const PastSizes &z) { return (p.packed_few ? z.each * z.rows : z.rows) <= 16; }

// A row's shares are joined by 32 lanes, or by a workgroup where they are many or rows are few.
static bool join_by_lanes(const PastPlan &p, const PastSizes &z) {  // 64 rows of 8 shares 16.7 us with the forward, by a workgroup per row 16.2
  return p.slots <= (z.B * z.Hk * z.rows < 1024 ? 4 : 8);
}

static int past_limit(const PastPlan &p, const PastSizes &z) {
  const int64_t rows = z.B * z.Hk * z.rows, most = z.f32 && z.D > 64 ? 4 : 8;
  bool fits = p.few ? launch_fits(own_blocks(p, z) + (p.packed_few ? packed_blocks(p, z) : 0), 64 * (one_block(p, z) ? most : p.waves))
                    : launch_fits(own_blocks(p, z), 256);
  if (p.packed && !p.packed_few) fits = fits && launch_fits(packed_blocks(p, z), 256);
  if (p.slots > 1) fits = fits && launch_fits(join_by_lanes(p, z) ? ceil_div(rows, 8) : rows, 256);
  return fits ? MLORA_OK : MLORA_ERR_LIMIT;
}

struct PastBwdPlan {
  int kw;       // waves of dk / dv over different keys, 32 each
  int64_t row_tiles, splits;
  int64_t key_blocks, prefix_blocks, sink_blocks, prefix_splits, sink_splits, own_splits;
  int64_t prefix_vectors, sink_vectors, own_vectors;  // 16-byte vectors of all shares of a class, 0 where it has one
  int64_t dq_vectors;                                 // of one share of dq
  double cost;  // of dk / dv, to choose by
  int dq_waves;  // float32
};

static PastBwdPlan past_bwd_plan(const PastSizes &z) {
  PastBwdPlan p{};
  const int64_t kt = z.f32 ? 32 : 64, dp = z.D > 64 ? 128 : 64;
  const int64_t row_tile = z.f32 ? 32 : 128;
  p.row_tiles = ceil_div(z.rows, row_tile);
  const int64_t items = z.B * z.Hk * p.row_tiles, tiles = own_tiles(z, row_tile, kt) + ceil_div(z.Lp, kt);
  p.splits = items <= 0 ? 1 : !z.f32 ? wide_shares(items, tiles, 128 * dp, 8e6) : between(256 / items, 1, between(tiles / 8, 1, 64));
  p.dq_vectors = z.f32 ? z.B * z.Hk * z.rows * (z.D / 4) : items * 4 * (dp / 32) * 4 * 64;
  p.dq_waves = f32_waves(z.D, items * p.splits, ceil_div(tiles, p.splits));
  const bool bounded = z.window < z.Lk;
  auto plan = [&](int kw, double finer) {
    PastBwdPlan c = p;
    c.kw = kw;
    const int64_t qt = z.f32 ? 32 : 64, keys = z.f32 ? kF32Keys : 32 * kw;
    c.key_blocks = ceil_div(z.Lk, keys), c.prefix_blocks = ceil_div(z.Lp, keys);
    c.sink_blocks = bounded ? between(ceil_div(z.sinks, keys), 0, c.key_blocks) : 0;  // without a window all blocks are alike
    const int64_t head_tiles = ceil_div(z.Lq, qt), seen = z.window + z.chunk + keys;
    const int64_t work[3] = {z.each * z.G * head_tiles, z.G * head_tiles, z.G * (bounded && seen < z.Lq ? ceil_div(seen, qt) + 1 : head_tiles)};
    const int64_t items[3] = {z.groups * z.Hk * c.prefix_blocks, z.B * z.Hk * c.sink_blocks, z.B * z.Hk * (c.key_blocks - c.sink_blocks)};
    const int64_t total = items[0] * work[0] + items[1] * work[1] + items[2] * work[2];
    const int64_t slots = z.f32 ? 1024 : z.D > 64 ? 256 : 512, least = z.f32 ? 8 : 4;
    const int64_t target = std::max((int64_t)(finer * (double)ceil_div(total, slots)), least);
    int64_t splits[3], blocks = 0, longest = 0;
    for (int i = 0; i < 3; ++i) {
      splits[i] = items[i] > 0 ? between(work[i] / target, 1, 64) : 1;
      blocks += items[i] * splits[i];
      if (items[i] > 0) longest = std::max(longest, ceil_div(work[i], splits[i]));
    }
    c.prefix_splits = splits[0], c.sink_splits = splits[1], c.own_splits = splits[2];
    const int64_t per = z.f32 ? keys * (z.D / 2) : kw * 2 * (dp / 32) * 4 * 64;
    c.prefix_vectors = splits[0] > 1 ? items[0] * splits[0] * per : 0;
    c.sink_vectors = splits[1] > 1 ? items[1] * splits[1] * per : 0;
    c.own_vectors = splits[2] > 1 ? items[2] * splits[2] * per : 0;
    // in tiles of 256 keys by 64 rows, 2.4 us each: as long as the longest share, or full rounds of 256 workgroups and half of it; three
    // tiles for a workgroup's start and end, the shares' sums at 6 TB/s. Of whole sequences the later keys are seen by fewer tokens.
    const double shares = (double)(c.prefix_vectors + c.sink_vectors + c.own_vectors) * 32 / 6e6 / 2.4;
    const double part = z.Lq == z.Lk && z.Lk > 0 ? 1.0 - 0.5 * (double)std::max<int64_t>(std::min(seen, z.Lk) - z.chunk, 0) / (double)z.Lk : 1.0;
    const double all = (double)(items[0] * work[0] + items[1] * work[1]) + part * (double)(items[2] * work[2]) + 3.0 * (double)blocks;
    c.cost = (blocks <= slots ? (double)longest + 3.0 : std::max((double)longest + 3.0, all / (double)slots + 0.5 * (double)longest)) *
                 (kw == 8 ? 1.0 : 0.66) + shares + (shares > 0 ? 2.0 : 0.0);
    return c;
  };
  // float32 and up to 64 channels: even parts. Finer ones (0.8 and 0.6 of an even part), us of the backward: 2 x 4096 tokens, window 1024,
  // 16 / 4 heads of 64 233, 205 and 217, 4096 tokens without a window, 12 heads 224, 225 and 190; but 2 x 1024, 16 / 4 heads 66, 77 and 75, a frame of
  // 1560, 12 heads 72, 80 and 81; float32, the same frame of 128 channels 840, 756 and 756, 2 x 2048, 8 / 2 heads 288, 310 and 308. The cost
  // below is of tiles of 128 channels in bf16 and does not tell these apart.
  if (z.f32 || z.D <= 64) return plan(4, 1.0);
  // 256 keys per workgroup, or 128 whose tiles take 0.66 of the time (a barrier per 32 rows of a wave): 32760 keys, 12 heads, in one 4.7 ms,
  // in the other 5.4; 4096 keys without a window, 12 heads, 240 us and 165. Shares of an even part of the work,
  // or finer ones (two samples of 4096 and 2777 tokens, window 1024, 16 / 4 heads: 160 workgroups 270 us, in finer shares 165).
  PastBwdPlan best = plan(8, 1.0);
  for (int kw : {8, 4})
    for (double finer : {1.0, 0.8, 0.6}) {
      const PastBwdPlan c = plan(kw, finer);
      if (c.cost < 0.97 * best.cost) best = c;
    }
  return best;
}

// The rows' deltas, then the shares of dq, and after they are joined those of dk and dv in the same place.
static int64_t past_bwd_bytes(const PastBwdPlan &p, const PastSizes &z) {
  const int64_t dq = p.splits > 1 ? p.splits * p.dq_vectors : 0, dkv = p.prefix_vectors + p.sink_vectors + p.own_vectors;
  return (ceil_div(z.B * z.Hk * z.rows, 4) + (dq > dkv ? dq : dkv)) * 16;
}

// The workgroups of dk / dv, over all classes, and the work items of one; the vectors of a class's share, 0 where it has one.
static int64_t dkv_blocks(const PastBwdPlan &p, const PastSizes &z) {
  return z.groups * z.Hk * p.prefix_blocks * p.prefix_splits + z.B * z.Hk * (p.sink_blocks * p.sink_splits + (p.key_blocks - p.sink_blocks) * p.own_splits);
}
static int64_t dkv_threads(const PastBwdPlan &p, const PastSizes &z) {
  if (z.f32) return (z.D > 64 ? 256 : 512) / (dkv_blocks(p, z) > 256 ? 2 : 1);
  return p.kw == 8 || z.D > 64 ? 512 : 256;
}
static int64_t dkv_join_blocks(const PastBwdPlan &p, int64_t (&upto)[3]) {
  const int64_t vectors[3] = {p.prefix_vectors, p.sink_vectors, p.own_vectors}, splits[3] = {p.prefix_splits, p.sink_splits, p.own_splits};
  int64_t blocks = 0;
  for (int c = 0; c < 3; ++c) upto[c] = blocks += splits[c] > 1 ? ceil_div(vectors[c] / splits[c], 256) : 0;
  return blocks;
}
static int past_bwd_limit(const PastBwdPlan &p, const PastSizes &z) {
  int64_t upto[3];
  const bool fits = launch_fits(z.B * z.Hk * p.row_tiles * p.splits, z.f32 ? 64 * p.dq_waves : 256) &&
                    (p.splits == 1 || launch_fits(ceil_div(p.dq_vectors, 256), 256)) && launch_fits(dkv_blocks(p, z), dkv_threads(p, z)) &&
                    launch_fits(dkv_join_blocks(p, upto), 256);
  return fits ? MLORA_OK : MLORA_ERR_LIMIT;
}

// A [B, L, heads, D] operand: 16-byte aligned heads, token strides whose tiles stay within 32-bit offsets.
static int past_operand(const void *p, const int64_t *st, bool empty) {
  if (empty) return MLORA_OK;
  if (p == nullptr) return MLORA_ERR_INVALID;
  if (!aligned16(p) || st[0] < 0 || st[1] < 0 || st[2] < 0 || st[0] % 8 != 0 || st[1] % 8 != 0 || st[2] % 8 != 0) return MLORA_ERR_UNSUPPORTED;
  if (st[1] >= (int64_t)1 << 22) return MLORA_ERR_LIMIT;  // 64 rows of 2^22 floats: 2^30 bytes
  return MLORA_OK;
}

static int past_args(PastArgs &a, const PastSizes &z, const mlora_past_shape *s, const void *q, const void *k, const void *v,
                     const void *pk, const void *pv, const int32_t *lengths, const int32_t *starts, const int32_t *prefix_lengths) {
  int st = past_operand(q, s->q_strides, z.B * z.Lq == 0);
  if (!st) st = past_operand(k, s->k_strides, z.B * z.Lk == 0);
  if (!st) st = past_operand(v, s->v_strides, z.B * z.Lk == 0);
  if (!st) st = past_operand(pk, s->pk_strides, z.groups * z.Lp == 0);
  if (!st) st = past_operand(pv, s->pv_strides, z.groups * z.Lp == 0);
  if (st) return st;
  a = PastArgs{};
  a.q = q, a.k = k, a.v = v, a.pk = pk, a.pv = pv, a.lengths = lengths, a.starts = starts, a.prefix_lengths = prefix_lengths;
  a.q_sb = s->q_strides[0], a.q_sl = s->q_strides[1], a.q_sh = s->q_strides[2];
  a.k_sb = s->k_strides[0], a.k_sl = s->k_strides[1], a.k_sh = s->k_strides[2];
  a.v_sb = s->v_strides[0], a.v_sl = s->v_strides[1], a.v_sh = s->v_strides[2];
  a.pk_sb = s->pk_strides[0], a.pk_sl = s->pk_strides[1], a.pk_sh = s->pk_strides[2];
  a.pv_sb = s->pv_strides[0], a.pv_sl = s->pv_strides[1], a.pv_sh = s->pv_strides[2];
  a.B = (int32_t)z.B, a.Lq = (int32_t)z.Lq, a.Lk = (int32_t)z.Lk, a.H = (int32_t)z.H, a.Hk = (int32_t)z.Hk, a.G = (int32_t)z.G;
  a.D = (int32_t)z.D, a.Lp = (int32_t)z.Lp, a.each = (int32_t)z.each, a.rows = (int32_t)z.rows;
  a.window = (int32_t)z.window, a.sinks = (int32_t)z.sinks, a.chunk = (int32_t)z.chunk, a.first = (int32_t)z.first;
  a.from_end = s->from_end != 0, a.c = s->scale * kLog2e, a.with_prefix = z.Lp > 0, a.splits = 1;
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

// f with a workgroup's waves: bf16 has one number.
template <class T, int DP, class F>
static void with_waves(int waves, F &&f) {
  constexpr int most = kFewWaves<T, DP>;
  if constexpr (sizeof(T) == 4) {
    if (waves == most / 2) return f(std::integral_constant<int, most / 2>{});
    if constexpr (most == 8) {
      if (waves == 2) return f(std::integral_constant<int, 2>{});
    }
  }
  f(std::integral_constant<int, most>{});
}

}  // namespace mlora

using namespace mlora;

extern "C" int64_t mlora_past_attention_workspace_bytes(const mlora_past_shape *shape) {
  PastSizes z;
  int st = past_sizes(z, shape);
  if (st) return st;
  const PastPlan p = past_plan(z);
  st = past_limit(p, z);
  return st ? st : past_floats(p, z) * (int64_t)sizeof(float);
}

extern "C" int mlora_past_attention(const mlora_past_shape *shape, const void *q, const void *k, const void *v, const void *pk,
                                    const void *pv, const int32_t *key_lengths, const int32_t *query_start,
                                    const int32_t *prefix_lengths, void *out, void *rest, float *stats, void *workspace,
                                    int64_t workspace_bytes, void *stream) {
  PastSizes z;
  int st = past_sizes(z, shape);
  if (st) return st;
  PastArgs a;
  st = past_args(a, z, shape, q, k, v, pk, pv, key_lengths, query_start, prefix_lengths);
  if (st || z.B * z.Lq == 0) return st;
  if (out == nullptr || (stats != nullptr && !z.f32 && rest == nullptr)) return MLORA_ERR_INVALID;
  if (!aligned16(out) || !aligned16(rest) || (reinterpret_cast<uintptr_t>(stats) & 3u) != 0) return MLORA_ERR_UNSUPPORTED;
  const PastPlan p = past_plan(z);
  st = past_limit(p, z);
  if (st) return st;
  const int64_t floats = past_floats(p, z);
  if (floats > 0) {
    if (workspace == nullptr || workspace_bytes < floats * (int64_t)sizeof(float)) return MLORA_ERR_WORKSPACE;
    if (!aligned16(workspace)) return MLORA_ERR_UNSUPPORTED;
  }
  a.out = out, a.rest = static_cast<uint16_t *>(rest), a.stats = stats;
  a.part_o = static_cast<float *>(workspace);
  a.part_ml = a.part_o + p.slots * z.B * z.Hk * z.rows * z.D;
  a.row_tiles = (int32_t)p.row_tiles, a.splits = (int32_t)p.splits, a.slots = (int32_t)p.slots;
  a.packed_tiles = (int32_t)p.packed_tiles, a.packed_splits = (int32_t)p.packed_splits;
  const int64_t packed = packed_blocks(p, z), blocks = own_blocks(p, z);
  if (p.packed) a.with_prefix = 0;
  hipStream_t s = static_cast<hipStream_t>(stream);
  with_head(z.f32, z.D, [&](auto t, auto dp) {
    using T = decltype(t);
    constexpr int DP = decltype(dp)::value;
    if constexpr (sizeof(T) == 2) {
      if (!p.few) {
        hipLaunchKernelGGL(past_fwd_kernel<DP>, dim3((unsigned)blocks), dim3(256), 0, s, a);
        return;
      }
      if (p.packed && !p.packed_few) {  // the prefix's workgroups are of the other kernel
        a.packed_blocks = (int32_t)packed;
        hipLaunchKernelGGL(past_fwd_kernel<DP>, dim3((unsigned)packed), dim3(256), 0, s, a);
      }
    }
    a.packed_blocks = p.packed_few ? (int32_t)packed : 0;
    const dim3 grid((unsigned)(blocks + a.packed_blocks));
    constexpr int most = kFewWaves<T, DP>;
    if (one_block(p, z)) {
      hipLaunchKernelGGL((past_few_kernel<T, DP, 1, most>), grid, dim3(64 * most), 0, s, a);
      return;
    }
    with_waves<T, DP>(p.waves, [&](auto nw) {
      hipLaunchKernelGGL((past_few_kernel<T, DP, 2, decltype(nw)::value>), grid, dim3(64 * decltype(nw)::value), 0, s, a);
    });
  });
  st = launch_status();
  if (st || p.slots == 1) return st;
  const int64_t rows = z.B * z.Hk * z.rows;
  if (join_by_lanes(p, z)) {
    const dim3 joins((unsigned)ceil_div(rows, 8));
    if (z.f32) hipLaunchKernelGGL(past_join_rows_kernel<float>, joins, dim3(256), 0, s, a);
    else hipLaunchKernelGGL(past_join_rows_kernel<uint16_t>, joins, dim3(256), 0, s, a);
  } else {
    const dim3 joins((unsigned)rows);
    if (z.f32) hipLaunchKernelGGL(past_join_kernel<float>, joins, dim3(256), 0, s, a);
    else hipLaunchKernelGGL(past_join_kernel<uint16_t>, joins, dim3(256), 0, s, a);
  }
  return launch_status();
}

extern "C" int64_t mlora_past_attention_backward_workspace_bytes(const mlora_past_shape *shape) {
  PastSizes z;
  int st = past_sizes(z, shape);
  if (st) return st;
  const PastBwdPlan p = past_bwd_plan(z);
  st = past_bwd_limit(p, z);
  return st ? st : past_bwd_bytes(p, z);
}

extern "C" int mlora_past_attention_backward(const mlora_past_shape *shape, const void *q, const void *k, const void *v,
                                             const void *pk, const void *pv, const int32_t *key_lengths,
                                             const int32_t *query_start, const int32_t *prefix_lengths, const void *out,
                                             const void *rest, const float *stats, const void *g, const int64_t *g_strides,
                                             void *dq, void *dk, void *dv, void *dpk, void *dpv, void *workspace,
                                             int64_t workspace_bytes, void *stream) {
  PastSizes z;
  int st = past_sizes(z, shape);
  if (st) return st;
  PastBwdArgs ba{};
  PastArgs &a = ba.f;
  st = past_args(a, z, shape, q, k, v, pk, pv, key_lengths, query_start, prefix_lengths);
  if (st || z.B == 0) return st;
  if (g_strides == nullptr) return MLORA_ERR_INVALID;
  st = past_operand(g, g_strides, z.Lq == 0);
  if (st) return st;
  if ((z.Lq > 0 && (out == nullptr || stats == nullptr || dq == nullptr || (!z.f32 && rest == nullptr))) ||
      (z.Lk > 0 && (dk == nullptr || dv == nullptr)) || (z.groups * z.Lp > 0 && (dpk == nullptr || dpv == nullptr)))
    return MLORA_ERR_INVALID;
  for (const void *p : {out, rest, (const void *)dq, (const void *)dk, (const void *)dv, (const void *)dpk, (const void *)dpv})
    if (!aligned16(p)) return MLORA_ERR_UNSUPPORTED;
  const PastBwdPlan p = past_bwd_plan(z);
  st = past_bwd_limit(p, z);
  if (st) return st;
  if (workspace_bytes < past_bwd_bytes(p, z) || (workspace == nullptr && workspace_bytes > 0)) return MLORA_ERR_WORKSPACE;
  if (!aligned16(workspace)) return MLORA_ERR_UNSUPPORTED;
  a.out = const_cast<void *>(out), a.rest = static_cast<uint16_t *>(const_cast<void *>(rest)), a.stats = const_cast<float *>(stats);
  a.row_tiles = (int32_t)p.row_tiles, a.splits = (int32_t)p.splits, a.slots = (int32_t)p.splits;
  ba.g = g, ba.g_sb = g_strides[0], ba.g_sl = g_strides[1], ba.g_sh = g_strides[2], ba.scale = shape->scale;
  ba.dq = dq, ba.dk = dk, ba.dv = dv, ba.dpk = dpk, ba.dpv = dpv, ba.delta = static_cast<float *>(workspace);
  ba.part = static_cast<f32x4 *>(workspace) + ceil_div(z.B * z.Hk * z.rows, 4);
  ba.key_blocks = (int32_t)p.key_blocks, ba.prefix_blocks = (int32_t)p.prefix_blocks, ba.sink_blocks = (int32_t)p.sink_blocks;
  ba.prefix_splits = (int32_t)p.prefix_splits, ba.sink_splits = (int32_t)p.sink_splits, ba.own_splits = (int32_t)p.own_splits;
  ba.sink_part = p.prefix_vectors, ba.own_part = p.prefix_vectors + p.sink_vectors;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (z.Lq > 0) {
    with_head(z.f32, z.D, [&](auto t, auto dp) {
      using T = decltype(t);
      constexpr int DP = decltype(dp)::value;
      const dim3 grid((unsigned)(z.B * z.Hk * p.row_tiles * p.splits));
      if constexpr (sizeof(T) == 2) hipLaunchKernelGGL(past_dq_kernel<DP>, grid, dim3(256), 0, s, ba);
      else with_waves<T, DP>(p.dq_waves, [&](auto nw) {
        hipLaunchKernelGGL((past_dq_f32_kernel<DP, decltype(nw)::value>), grid, dim3(64 * decltype(nw)::value), 0, s, ba);
      });
      if (p.splits > 1) hipLaunchKernelGGL((past_dq_join_kernel<T, DP>), dim3((unsigned)ceil_div(p.dq_vectors, 256)), dim3(256), 0, s, ba);
    });
    st = launch_status();
    if (st) return st;
  }
  const int64_t blocks = dkv_blocks(p, z);
  if (blocks == 0) return MLORA_OK;
  JoinBlocks joins;
  const int64_t join_blocks = dkv_join_blocks(p, joins.upto);
  with_head(z.f32, z.D, [&](auto t, auto dp) {
    using T = decltype(t);
    constexpr int DP = decltype(dp)::value;
    auto go = [&](auto kw) {
      constexpr int KW = decltype(kw)::value, RG = KW == 4 ? DP / 64 : 1;
      if constexpr (sizeof(T) == 2) hipLaunchKernelGGL((past_dkv_kernel<DP, KW, RG>), dim3((unsigned)blocks), dim3(64 * KW * RG), 0, s, ba);
      else if (blocks > 256) hipLaunchKernelGGL((past_dkv_f32_kernel<DP, kFewWaves<T, DP> / 2>), dim3((unsigned)blocks), dim3(32 * kFewWaves<T, DP>), 0, s, ba);
      else hipLaunchKernelGGL((past_dkv_f32_kernel<DP, kFewWaves<T, DP>>), dim3((unsigned)blocks), dim3(64 * kFewWaves<T, DP>), 0, s, ba);
      if (join_blocks > 0) hipLaunchKernelGGL((past_dkv_join_kernel<T, DP, KW>), dim3((unsigned)join_blocks), dim3(256), 0, s, ba, joins);
    };
    if constexpr (sizeof(T) == 2 && DP == 128) {
      if (p.kw == 8) return go(std::integral_constant<int, 8>{});
    }
    go(std::integral_constant<int, 4>{});
  });
  return launch_status();
}
