// What joins two sublayers of a DiT block, in one pass over the rows:
//
//   p  = N_post(y) · w_post            the sublayer's output, normed if the block norms after it (else p = y)
//   u  = α · x + gate · p              the residual stream, written as x1 in its own type
//   out = N(u) · m + shift             the next sublayer's input, m = 1 + scale (a modulation) or scale (a weight)
//
// N is a LayerNorm (mean removed) or an RMSNorm of the row. x / x1 are bf16 or float32, y / out bf16 or
// float32; the vectors gate, scale, shift [B, W] or shared [W], w_post [W]. Everything between the loads
// and the one rounding of each output is float32; N reads u before its rounding to x1's type.
//
// Backward, with û = N(u), r = 1 / σ(u), p̂ = N_post(y), and the upstream gradients gx of x1 and go of out:
//   h  = go · m;  du = gx + r·(h − mean(h)·[layer] − û·mean(h·û))
//   dx = α·du;  dp = gate·du;  q = dp·w_post;  dy = r_post·(q − mean(q)·[layer] − p̂·mean(q·p̂))   (or dp)
//   dgate = Σ du·p;  dscale = Σ go·û;  dshift = Σ go;  dw_post = Σ dp·p̂          over the tokens
// u and its statistics are formed again from x and y: dgate needs y anyway, so reading x in place of a
// stored x1 costs nothing and keeps û exact.
//
// dgate and dw_post are one sum, S = Σ du·p̂ per channel: dgate = w_post·S, dw_post = gate·S (gate is the
// workgroup's sample's), multiplied behind the rows.
//
// Both passes are HBM-bound and run at what a large copy reaches (4.9 TB/s): 2 x 32760 rows of 1536, float32 stream,
// bf16 y, every vector's gradient: 219 us forward (604 MB in, 604 MB out), 378 backward; 2 x 11040 rows of
// 5120, bf16, normed on both sides: 159 and 291. A row is held in registers by WPR waves (8 values per lane and
// chunk). A workgroup takes `chunk` rows of one sample; the backward's column sums stay in registers over
// those rows, are added over the workgroup's rows in flight through LDS, and leave as one partial row
// per workgroup (fixed order, no atomics).
#include "mlora_common.h"
#include "mlora_host.h"
#include "mlora_rows.h"

namespace mlora {

constexpr int kJointMaxWidth = 8192;
enum { kNormLayer = 0, kNormRms = 1 };
enum { kVecGate = 0, kVecMult = 1, kVecShift = 2, kVecPost = 3, kVecs = 4 };

struct JointArgs {
  const void *x, *y;
  void *x1, *out;                                      // contiguous
  const void *gate, *scale, *shift, *post_w;           // null: 1, (1 or no offset), 0, 1
  int64_t x_sb, x_st, y_sb, y_st, gate_sb, scale_sb, shift_sb;  // element strides
  int32_t tokens, width, n_chunks, chunk;
  int32_t gate_f32, scale_f32, shift_f32, post_f32;
  int32_t norm, post, unit_offset;                     // post: -1 none, else kNormLayer / kNormRms
  float alpha, eps;
};

struct JointBwdArgs {
  JointArgs f;
  const void *gx, *go;  // null: zero
  int64_t gx_sb, gx_st, go_sb, go_st;
  void *dx, *dy;        // contiguous
  float *partial;       // [batches, n_chunks, kVecs, width]
};

// The sums of a row held by WPR of the workgroup's NW waves, added in wave order.
template <int WPR, int NW>
struct RowSum {
  float (*red)[2][NW];  // four slots: a slot is written again only after two more barriers
  int wave, first, slot = 0;
  __device__ __forceinline__ void operator()(float &a, float &b) {
    a = lanes_sum<64>(a), b = lanes_sum<64>(b);
    if constexpr (WPR > 1) {
      if ((threadIdx.x & 63) == 0) red[slot][0][wave] = a, red[slot][1][wave] = b;
      __syncthreads();
      a = red[slot][0][first], b = red[slot][1][first];
#pragma unroll
      for (int w = 1; w < WPR; ++w) a += red[slot][0][first + w], b += red[slot][1][first + w];
      slot = (slot + 1) & 3;
    }
  }
  __device__ __forceinline__ float operator()(float a) {
    a = lanes_sum<64>(a);
    if constexpr (WPR > 1) {
      if ((threadIdx.x & 63) == 0) red[slot][0][wave] = a;
      __syncthreads();
      a = red[slot][0][first];
#pragma unroll
      for (int w = 1; w < WPR; ++w) a += red[slot][0][first + w];
      slot = (slot + 1) & 3;
    }
    return a;
  }
};

// The sample's vectors: gate, m, shift, w_post, formed from their sources (ones or zeros where there is none).
// LDS: copied once per workgroup, values 8c .. 8c + 3 of vector v at [v][0][c], 8c + 4 .. 8c + 7 at [v][1][c]
// (two conflict-free 16-byte reads per chunk): for rows of one wave, four of which share them. Rows of several
// waves are wide and have a workgroup each: its lanes read what they need into registers once (2 x 11040 rows
// of 5120 normed on both sides, bf16: backward 291 us; 418 with the vectors read from the caches for every row, 740
// from LDS, which they would fill).
template <bool LDS>
struct Vectors {
  const JointArgs &a;
  int64_t b;
  f32x4 *base;
  int nchunks;
  __device__ __forceinline__ f32x4 *at(int v) const { return base + (int64_t)v * 2 * nchunks; }
  __device__ __forceinline__ void source(int v, int c, float (&o)[8]) const {
    const void *p = v == kVecGate ? a.gate : v == kVecMult ? a.scale : v == kVecShift ? a.shift : a.post_w;
    const bool f32 = v == kVecGate ? a.gate_f32 : v == kVecMult ? a.scale_f32 : v == kVecShift ? a.shift_f32 : a.post_f32;
    const int64_t off = v == kVecGate ? a.gate_sb : v == kVecMult ? a.scale_sb : v == kVecShift ? a.shift_sb : 0;
    if (p == nullptr) {
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = v == kVecShift ? 0.f : 1.f;
      return;
    }
    load8(p, f32, b * off + 8 * c, o);
    if (v == kVecMult && a.unit_offset) {
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] += 1.f;
    }
  }
  __device__ __forceinline__ void read(int v, int c, float (&o)[8]) const {
    if constexpr (LDS) {
      const f32x4 x = at(v)[c], y = at(v)[nchunks + c];
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = x[i], o[i + 4] = y[i];
    } else {
      source(v, c, o);
    }
  }
  __device__ __forceinline__ void fill() const {
    if constexpr (LDS) {
#pragma unroll
      for (int v = 0; v < kVecs; ++v)
        for (int c = threadIdx.x; c < nchunks; c += blockDim.x) {
          float t[8];
          source(v, c, t);
          at(v)[c] = f32x4{t[0], t[1], t[2], t[3]};
          at(v)[nchunks + c] = f32x4{t[4], t[5], t[6], t[7]};
        }
    }
  }
};

// v <- N(v) for the row's values (zeros past the width); returns 1 / σ.
template <int NCH, int WPR, class Sum>
__device__ __forceinline__ float norm_row(float (&v)[NCH][8], int c0, int nchunks, int kind, float inv_w, float eps,
                                          Sum &sum) {
  if (kind == kNormLayer) {
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < NCH; ++k)
#pragma unroll
      for (int i = 0; i < 8; ++i) s += v[k][i];
    const float mean = sum(s) * inv_w;
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      const bool in = c0 + 64 * WPR * k < nchunks;
#pragma unroll
      for (int i = 0; i < 8; ++i) v[k][i] = in ? v[k][i] - mean : 0.f;
    }
  }
  float s = 0.f;
#pragma unroll
  for (int k = 0; k < NCH; ++k)
#pragma unroll
    for (int i = 0; i < 8; ++i) s += v[k][i] * v[k][i];
  const float r = 1.0f / __fsqrt_rn(sum(s) * inv_w + eps);
#pragma unroll
  for (int k = 0; k < NCH; ++k)
#pragma unroll
    for (int i = 0; i < 8; ++i) v[k][i] *= r;
  return r;
}

// A row's chunks as they lie in memory, to be asked for a row ahead.
template <int NCH, int WPR, bool F32>
struct RawRow {
  u32x4 r[NCH][F32 ? 2 : 1];
  __device__ __forceinline__ void load(const void *p, int64_t o, int c0, int nchunks, bool live) {
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      const int c = c0 + 64 * WPR * k;
      const bool on = live && c < nchunks;
      if constexpr (F32) {
        const float *q = static_cast<const float *>(p) + o + 8 * c;
        r[k][0] = on ? *(const MLORA_GLOBAL u32x4 *)q : u32x4{0, 0, 0, 0};
        r[k][1] = on ? *(const MLORA_GLOBAL u32x4 *)(q + 4) : u32x4{0, 0, 0, 0};
      } else {
        r[k][0] = on ? *(const MLORA_GLOBAL u32x4 *)(static_cast<const uint16_t *>(p) + o + 8 * c) : u32x4{0, 0, 0, 0};
      }
    }
  }
  __device__ __forceinline__ void unpack(float (&v)[NCH][8]) const {
#pragma unroll
    for (int k = 0; k < NCH; ++k)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if constexpr (F32) v[k][i] = __uint_as_float(r[k][i / 4][i % 4]);
        else v[k][i] = __uint_as_float(i % 2 ? r[k][0][i / 2] & 0xffff0000u : r[k][0][i / 2] << 16);
      }
  }
};

template <int NCH, int WPR, int NW, bool XF32, bool YF32>
__global__ __launch_bounds__(64 * NW) void joint_kernel(const JointArgs a) {
  constexpr int STREAMS = NW / WPR;
  constexpr bool kAhead = WPR > 1, kHeld = WPR > 1;
  __shared__ float red[4][2][NW];
  extern __shared__ f32x4 dyn[];
  const int wave = wave_id(), lane = threadIdx.x & 63, stream = wave / WPR;
  const int c0 = lane + 64 * (wave % WPR), nchunks = a.width / 8;
  const int64_t b = blockIdx.x / a.n_chunks;
  const int t0 = (blockIdx.x % a.n_chunks) * a.chunk, t1 = min(t0 + a.chunk, a.tokens);
  const float inv_w = 1.0f / (float)a.width;
  const Vectors<WPR == 1> vec{a, b, dyn, nchunks};
  vec.fill();
  RowSum<WPR, NW> sum{red, wave, stream * WPR};
  __syncthreads();
  float gw[kHeld ? NCH : 1][8], mult[kHeld ? NCH : 1][8], shift[kHeld ? NCH : 1][8];
  auto read_gw = [&](int c, float (&g)[8]) __attribute__((always_inline)) {  // gate · w_post
    vec.read(kVecGate, c, g);
    if (a.post < 0) return;
    float w[8];
    vec.read(kVecPost, c, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) g[i] *= w[i];
  };
  if constexpr (kHeld) {
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      const int c = min(c0 + 64 * WPR * k, nchunks - 1);
      read_gw(c, gw[k]);
      vec.read(kVecMult, c, mult[k]);
      vec.read(kVecShift, c, shift[k]);
    }
  }
  RawRow<NCH, WPR, XF32> rx;
  RawRow<NCH, WPR, YF32> ry;
  auto load = [&](int t) __attribute__((always_inline)) {
    rx.load(a.x, b * a.x_sb + t * a.x_st, c0, nchunks, t < t1);
    ry.load(a.y, b * a.y_sb + t * a.y_st, c0, nchunks, t < t1);
  };
  if constexpr (kAhead) load(t0 + stream);
  // every stream runs the same number of rows, so that every wave meets the same barriers
  for (int t = t0 + stream; t - stream < t1; t += STREAMS) {
    const bool live = t < t1;
    float u[NCH][8], p[NCH][8];
    if constexpr (!kAhead) load(t);
    rx.unpack(u), ry.unpack(p);
    if constexpr (kAhead) load(t + STREAMS);
    if (a.post >= 0) norm_row<NCH, WPR>(p, c0, nchunks, a.post, inv_w, a.eps, sum);
    const int64_t row = (b * a.tokens + t) * a.width;
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      const int c = c0 + 64 * WPR * k;
      if (c >= nchunks) break;
      float g[8];
      if constexpr (!kHeld) read_gw(c, g);
#pragma unroll
      for (int i = 0; i < 8; ++i) u[k][i] = a.alpha * u[k][i] + (kHeld ? gw[kHeld ? k : 0][i] : g[i]) * p[k][i];
      if (live) store8_any(a.x1, XF32, row + 8 * c, u[k]);
    }
    norm_row<NCH, WPR>(u, c0, nchunks, a.norm, inv_w, a.eps, sum);
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      const int c = c0 + 64 * WPR * k;
      if (!live || c >= nchunks) break;
      float m[8], h[8], o[8];
      if constexpr (!kHeld) vec.read(kVecMult, c, m), vec.read(kVecShift, c, h);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        o[i] = (kHeld ? shift[kHeld ? k : 0][i] : h[i]) + u[k][i] * (kHeld ? mult[kHeld ? k : 0][i] : m[i]);
      store8_any(a.out, YF32, row + 8 * c, o);
    }
  }
}

// SUMS: some vector's gradient is wanted; POST: the sublayer's output is normed (its two extra arrays
// would otherwise cost registers that the plain joint uses for waves).
template <int NCH, int WPR, int NW, bool XF32, bool YF32, bool SUMS, bool POST>
__global__ __launch_bounds__(64 * NW) void joint_backward_kernel(const JointBwdArgs ba) {
  const JointArgs &a = ba.f;
  constexpr int STREAMS = NW / WPR, NV = POST ? 4 : 3;
  constexpr bool kAhead = WPR > 1;  // the next row's loads under this row's sums and barriers
  constexpr bool kHeld = WPR > 1;
  __shared__ float red[4][2][NW];
  extern __shared__ f32x4 dyn[];  // the vectors; after the rows, one partial row of each sum
  const int wave = wave_id(), lane = threadIdx.x & 63, stream = wave / WPR;
  const int c0 = lane + 64 * (wave % WPR), nchunks = a.width / 8;
  const int64_t b = blockIdx.x / a.n_chunks;
  const int t0 = (blockIdx.x % a.n_chunks) * a.chunk, t1 = min(t0 + a.chunk, a.tokens);
  const float inv_w = 1.0f / (float)a.width;
  const Vectors<WPR == 1> vec{a, b, dyn, nchunks};
  vec.fill();
  RowSum<WPR, NW> sum{red, wave, stream * WPR};
  float acc[SUMS ? 3 : 1][NCH][8];  // Σ du·p̂ (dgate = w_post times it, dw_post = gate times it), dscale, dshift
#pragma unroll
  for (int v = 0; v < (SUMS ? 3 : 1); ++v)
#pragma unroll
    for (int k = 0; k < NCH; ++k)
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[v][k][i] = 0.f;
  __syncthreads();
  auto read_gw = [&](int c, float (&g)[8]) __attribute__((always_inline)) {  // gate · w_post
    vec.read(kVecGate, c, g);
    if constexpr (POST) {
      float w[8];
      vec.read(kVecPost, c, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) g[i] *= w[i];
    }
  };
  float gw[kHeld ? NCH : 1][8], mult[kHeld ? NCH : 1][8];
  if constexpr (kHeld) {
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      const int c = min(c0 + 64 * WPR * k, nchunks - 1);
      read_gw(c, gw[k]);
      vec.read(kVecMult, c, mult[k]);
    }
  }
  RawRow<NCH, WPR, XF32> rx, rgx;
  RawRow<NCH, WPR, YF32> ry, rgo;
  auto load = [&](int t) __attribute__((always_inline)) {
    rx.load(a.x, b * a.x_sb + t * a.x_st, c0, nchunks, t < t1);
    ry.load(a.y, b * a.y_sb + t * a.y_st, c0, nchunks, t < t1);
    rgo.load(ba.go, b * ba.go_sb + t * ba.go_st, c0, nchunks, t < t1 && ba.go != nullptr);
    rgx.load(ba.gx, b * ba.gx_sb + t * ba.gx_st, c0, nchunks, t < t1 && ba.gx != nullptr);
  };
  if constexpr (kAhead) load(t0 + stream);
  for (int t = t0 + stream; t - stream < t1; t += STREAMS) {
    const bool live = t < t1;
    float u[NCH][8], p[NCH][8], go[NCH][8], d[NCH][8];
    if constexpr (!kAhead) load(t);
    rx.unpack(u), ry.unpack(p), rgo.unpack(go), rgx.unpack(d);
    if constexpr (kAhead) load(t + STREAMS);
    float rp = 1.f;
    if constexpr (POST) rp = norm_row<NCH, WPR>(p, c0, nchunks, a.post, inv_w, a.eps, sum);  // p holds p̂
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      const int c = c0 + 64 * WPR * k;
      if (c >= nchunks) break;
      float g[8];
      if constexpr (!kHeld) read_gw(c, g);
#pragma unroll
      for (int i = 0; i < 8; ++i) u[k][i] = a.alpha * u[k][i] + (kHeld ? gw[kHeld ? k : 0][i] : g[i]) * p[k][i];
    }
    const float r = norm_row<NCH, WPR>(u, c0, nchunks, a.norm, inv_w, a.eps, sum);  // u holds û
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      const int c = c0 + 64 * WPR * k;
      if (c >= nchunks) break;
      float m[8];
      if constexpr (!kHeld) vec.read(kVecMult, c, m);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if constexpr (SUMS) acc[1][k][i] += go[k][i] * u[k][i], acc[2][k][i] += go[k][i];
        go[k][i] *= kHeld ? mult[kHeld ? k : 0][i] : m[i];  // h
        s1 += go[k][i];
        s2 += go[k][i] * u[k][i];
      }
    }
    sum(s1, s2);
    s1 = a.norm == kNormLayer ? s1 * inv_w : 0.f;
    s2 *= inv_w;
    float q1 = 0.f, q2 = 0.f;
    const int64_t row = (b * a.tokens + t) * a.width;
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      const int c = c0 + 64 * WPR * k;
      if (c >= nchunks) break;
      float g[8];
      if constexpr (!kHeld) read_gw(c, g);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float du = d[k][i] + r * (go[k][i] - s1 - u[k][i] * s2);
        d[k][i] = du;
        if constexpr (SUMS) acc[0][k][i] += du * p[k][i];
        go[k][i] = (kHeld ? gw[kHeld ? k : 0][i] : g[i]) * du;  // dp, or q
        if constexpr (POST) q1 += go[k][i], q2 += go[k][i] * p[k][i];
      }
      if (live && ba.dx != nullptr) {
        float o[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i] = a.alpha * d[k][i];
        store8_any(ba.dx, XF32, row + 8 * c, o);
      }
    }
    if constexpr (POST) {
      sum(q1, q2);
      q1 = a.post == kNormLayer ? q1 * inv_w : 0.f;
      q2 *= inv_w;
    }
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      const int c = c0 + 64 * WPR * k;
      if (!live || ba.dy == nullptr || c >= nchunks) break;
      if constexpr (POST) {
#pragma unroll
        for (int i = 0; i < 8; ++i) go[k][i] = rp * (go[k][i] - q1 - p[k][i] * q2);
      }
      store8_any(ba.dy, YF32, row + 8 * c, go[k]);
    }
  }
  if constexpr (SUMS) {
    float post[POST ? NCH : 1][8];  // dw_post
    if constexpr (POST) {
#pragma unroll
      for (int k = 0; k < NCH; ++k) {
        const int c = min(c0 + 64 * WPR * k, nchunks - 1);
        float g[8], w[8];
        vec.read(kVecGate, c, g);
        vec.read(kVecPost, c, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) post[k][i] = acc[0][k][i] * g[i], acc[0][k][i] *= w[i];
      }
    }
    auto total = [&](int v, int k, int i) __attribute__((always_inline)) { return v == kVecPost ? post[POST ? k : 0][i] : acc[v < 3 ? v : 0][k][i]; };
    float *out = ba.partial + (int64_t)blockIdx.x * kVecs * a.width;
    if constexpr (STREAMS > 1) {  // the streams' sums, added in stream order in the vectors' place
      __syncthreads();
#pragma unroll
      for (int w = 0; w < STREAMS; ++w) {
        if (stream == w) {
#pragma unroll
          for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int k = 0; k < NCH; ++k) {
              const int c = c0 + 64 * WPR * k;
              if (c >= nchunks) break;
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                f32x4 s = f32x4{total(v, k, 4 * h), total(v, k, 4 * h + 1), total(v, k, 4 * h + 2), total(v, k, 4 * h + 3)};
                f32x4 &dst = vec.at(v)[h * nchunks + c];
                if (w > 0) s += dst;
                dst = s;
              }
            }
        }
        __syncthreads();
      }
      for (int e = threadIdx.x; e < NV * 2 * nchunks; e += 64 * NW) {
        const int v = e / (2 * nchunks), h = e % 2, c = e / 2 % nchunks;
        *(MLORA_GLOBAL f32x4 *)(out + v * a.width + 8 * c + 4 * h) = vec.at(v)[h * nchunks + c];
      }
    } else {
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int k = 0; k < NCH; ++k) {
          const int c = c0 + 64 * WPR * k;
          float t[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) t[i] = total(v, k, i);
          if (c < nchunks) store8_any(out, true, v * a.width + 8 * c, t);
        }
    }
  }
}

// Rows per workgroup (a multiple of the rows in flight): what leaves about `most` workgroups. Forward: many, so that
// the last ones end together, but each copies or reads the vectors (2 x 32760 rows of 1536 / 2 x 11040 of 5120:
// 2048 workgroups 234 / 169 us, 4096 228 / 164, 8192 219 / 159, 16384 212 / 174). Backward: those that run at
// once, since each leaves a partial row of every sum (half or twice as many: 315 and 322 us against 321).
static int joint_chunk(int64_t batches, int64_t tokens, int streams, int64_t most) {
  const int64_t per_sample = batches < most ? most / batches : 1;
  const int64_t rows = (tokens + per_sample - 1) / per_sample;
  return (int)((rows + streams - 1) / streams * streams);
}
constexpr int64_t kJointMostFwd = 8192, kJointWavesBwd = 2048;

// A row's waves and chunks per lane. Rows of more than one wave have a workgroup each; with three chunks per lane
// there, the backward's sums would leave one wave per SIMD (2 x 11040 rows of 5120, bf16: 342 us with three chunks
// on four waves, 291 with two on eight).
struct JointTile {
  int nch, wpr, nw;
};
static JointTile joint_tile(int64_t width) {
  const int n = (int)((width / 8 + 63) / 64);  // chunks of 8 values per lane of one wave
  if (n <= 3) return {n, 1, 4};
  const int waves = n <= 4 ? 2 : n <= 8 ? 4 : 8;
  return {2, waves, waves};
}

// f(nch, wpr, nw) with the tile's values as integral constants.
template <class F>
static void with_tile(const JointTile &t, F &&f) {
  using std::integral_constant;
  auto one = integral_constant<int, 1>{};
  auto two = integral_constant<int, 2>{};
  auto three = integral_constant<int, 3>{};
  auto four = integral_constant<int, 4>{};
  auto eight = integral_constant<int, 8>{};
  if (t.wpr == 1) {
    if (t.nch == 1) f(one, one, four);
    else if (t.nch == 2) f(two, one, four);
    else f(three, one, four);
  } else if (t.wpr == 2) {
    f(two, two, two);
  } else if (t.wpr == 4) {
    f(two, four, four);
  } else {
    f(two, eight, eight);
  }
}

// Workgroups of the backward that run at once: eight waves per compute unit.
static int joint_bwd_chunk(const JointTile &t, int64_t batches, int64_t tokens) {
  return joint_chunk(batches, tokens, t.nw / t.wpr, kJointWavesBwd / t.nw);
}

// Checks shared by both directions; fills everything but the outputs and the split of the rows.
static int joint_args(JointArgs &a, const void *x, int x_dtype, int64_t x_sb, int64_t x_st, const void *y, int y_dtype,
                      int64_t y_sb, int64_t y_st, const void *gate, int gate_dtype, int64_t gate_sb, const void *scale,
                      const void *shift, int affine_dtype, int64_t scale_sb, int64_t shift_sb, int unit_offset,
                      const void *post_w, int post_dtype, int norm, int post, float alpha, float eps, int64_t batches,
                      int64_t tokens, int64_t width) {
  if (batches < 0 || tokens < 0 || width < 0) return MLORA_ERR_INVALID;
  for (int d : {x_dtype, y_dtype, gate_dtype, affine_dtype, post_dtype})
    if (d != MLORA_BF16 && d != MLORA_F32) return MLORA_ERR_UNSUPPORTED;
  if (x_dtype == MLORA_BF16 && y_dtype == MLORA_F32) return MLORA_ERR_UNSUPPORTED;  // the stream is the wider one
  if (norm != kNormLayer && norm != kNormRms) return MLORA_ERR_INVALID;
  if (post != -1 && post != kNormLayer && post != kNormRms) return MLORA_ERR_INVALID;
  if ((scale == nullptr) != (shift == nullptr) && scale == nullptr) return MLORA_ERR_INVALID;  // a shift needs a scale
  if (post_w != nullptr && post == -1) return MLORA_ERR_INVALID;
  if (!(eps > 0.f && eps < INFINITY) || !(alpha > -INFINITY && alpha < INFINITY)) return MLORA_ERR_INVALID;
  if (width > 0 && (width % 8 != 0 || width > kJointMaxWidth)) return MLORA_ERR_UNSUPPORTED;
  if (batches > 0 && tokens > (INT32_MAX - 8192) / batches) return MLORA_ERR_LIMIT;
  if (batches == 0 || tokens == 0 || width == 0) return MLORA_OK;
  if (x == nullptr || y == nullptr) return MLORA_ERR_INVALID;
  if (!rows_aligned(x, x_sb, x_st) || !rows_aligned(y, y_sb, y_st) || !rows_aligned(gate, gate_sb, 0) ||
      !rows_aligned(scale, scale_sb, 0) || !rows_aligned(shift, shift_sb, 0) || !aligned16(post_w))
    return MLORA_ERR_UNSUPPORTED;
  a = JointArgs{x, y, nullptr, nullptr, gate, scale, shift, post_w, x_sb, x_st, y_sb, y_st, gate_sb, scale_sb, shift_sb,
                (int32_t)tokens, (int32_t)width, 0, 0,
                gate_dtype == MLORA_F32, affine_dtype == MLORA_F32, affine_dtype == MLORA_F32, post_dtype == MLORA_F32,
                norm, post, unit_offset != 0, alpha, eps};
  return MLORA_OK;
}

// The float types of x and y as constants: both bf16, float32 stream over bf16, both float32.
template <class F>
static void with_types(bool xf, bool yf, F &&f) {
  using std::integral_constant;
  if (!xf) f(integral_constant<bool, false>{}, integral_constant<bool, false>{});
  else if (!yf) f(integral_constant<bool, true>{}, integral_constant<bool, false>{});
  else f(integral_constant<bool, true>{}, integral_constant<bool, true>{});
}

}  // namespace mlora

using namespace mlora;

extern "C" int mlora_joint(const void *x, int x_dtype, int64_t x_sb, int64_t x_st, const void *y, int y_dtype,
                           int64_t y_sb, int64_t y_st, const void *gate, int gate_dtype, int64_t gate_sb,
                           const void *scale, const void *shift, int affine_dtype, int64_t scale_sb, int64_t shift_sb,
                           int unit_offset, const void *post_w, int post_dtype, int norm, int post, float alpha,
                           float eps, void *x1, void *out, int64_t batches, int64_t tokens, int64_t width,
                           void *stream) {
  JointArgs a;
  int st = joint_args(a, x, x_dtype, x_sb, x_st, y, y_dtype, y_sb, y_st, gate, gate_dtype, gate_sb, scale, shift,
                      affine_dtype, scale_sb, shift_sb, unit_offset, post_w, post_dtype, norm, post, alpha, eps,
                      batches, tokens, width);
  if (st || batches == 0 || tokens == 0 || width == 0) return st;
  if (x1 == nullptr || out == nullptr) return MLORA_ERR_INVALID;
  if (!aligned16(x1) || !aligned16(out)) return MLORA_ERR_UNSUPPORTED;
  const JointTile tile = joint_tile(width);
  a.x1 = x1, a.out = out;
  a.chunk = joint_chunk(batches, tokens, tile.nw / tile.wpr, kJointMostFwd);
  a.n_chunks = (int32_t)((tokens + a.chunk - 1) / a.chunk);
  const unsigned lds = tile.wpr == 1 ? (unsigned)(kVecs * width * sizeof(float)) : 0;
  with_tile(tile, [&](auto nch, auto wpr, auto nw) {
    with_types(x_dtype == MLORA_F32, y_dtype == MLORA_F32, [&](auto xf, auto yf) {
      auto kernel = joint_kernel<decltype(nch)::value, decltype(wpr)::value, decltype(nw)::value, decltype(xf)::value,
                                 decltype(yf)::value>;
      hipLaunchKernelGGL(kernel, dim3((unsigned)(batches * a.n_chunks)), dim3(64 * decltype(nw)::value), lds,
                         static_cast<hipStream_t>(stream), a);
    });
  });
  return launch_status();
}

extern "C" int64_t mlora_joint_backward_workspace_bytes(int64_t batches, int64_t tokens, int64_t width) {
  if (batches < 0 || tokens < 0 || width < 0) return MLORA_ERR_INVALID;
  if (batches == 0 || tokens == 0 || width == 0) return 0;
  if (width > kJointMaxWidth) return MLORA_ERR_UNSUPPORTED;
  if (tokens > (INT32_MAX - 8192) / batches) return MLORA_ERR_LIMIT;
  const int64_t chunk = joint_bwd_chunk(joint_tile(width), batches, tokens);
  return batches * ((tokens + chunk - 1) / chunk) * kVecs * width * (int64_t)sizeof(float);
}

extern "C" int mlora_joint_backward(const void *x, int x_dtype, int64_t x_sb, int64_t x_st, const void *y, int y_dtype,
                                    int64_t y_sb, int64_t y_st, const void *gx, int64_t gx_sb, int64_t gx_st,
                                    const void *go, int64_t go_sb, int64_t go_st, const void *gate, int gate_dtype,
                                    int64_t gate_sb, const void *scale, const void *shift, int affine_dtype,
                                    int64_t scale_sb, int64_t shift_sb, int unit_offset, const void *post_w,
                                    int post_dtype, int norm, int post, float alpha, float eps, void *dx, void *dy,
                                    void *dgate, void *dscale, void *dshift, void *dpost, int gate_shared,
                                    int scale_shared, int shift_shared, void *workspace, int64_t workspace_bytes,
                                    int64_t batches, int64_t tokens, int64_t width, void *stream) {
  JointBwdArgs ba;
  int st = joint_args(ba.f, x, x_dtype, x_sb, x_st, y, y_dtype, y_sb, y_st, gate, gate_dtype, gate_sb, scale, shift,
                      affine_dtype, scale_sb, shift_sb, unit_offset, post_w, post_dtype, norm, post, alpha, eps,
                      batches, tokens, width);
  if (st) return st;
  if ((dgate != nullptr && gate == nullptr) || (dscale != nullptr && scale == nullptr) ||
      (dshift != nullptr && shift == nullptr) || (dpost != nullptr && post_w == nullptr))
    return MLORA_ERR_INVALID;
  if (width == 0) return MLORA_OK;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool sums = dgate != nullptr || dscale != nullptr || dshift != nullptr || dpost != nullptr;
  for (void *p : {dx, dy, dgate, dscale, dshift, dpost})
    if (!aligned16(p)) return MLORA_ERR_UNSUPPORTED;
  int64_t n_chunks = 0;
  if (batches > 0 && tokens > 0) {
    JointArgs &a = ba.f;
    if (!rows_aligned(gx, gx_sb, gx_st) || !rows_aligned(go, go_sb, go_st)) return MLORA_ERR_UNSUPPORTED;
    if (sums) {
      if (workspace == nullptr || workspace_bytes < mlora_joint_backward_workspace_bytes(batches, tokens, width))
        return MLORA_ERR_WORKSPACE;
      if (!aligned16(workspace)) return MLORA_ERR_UNSUPPORTED;
    }
    const JointTile tile = joint_tile(width);
    a.chunk = joint_bwd_chunk(tile, batches, tokens);
    a.n_chunks = (int32_t)((tokens + a.chunk - 1) / a.chunk);
    n_chunks = a.n_chunks;
    ba.gx = gx, ba.go = go, ba.gx_sb = gx_sb, ba.gx_st = gx_st, ba.go_sb = go_sb, ba.go_st = go_st;
    ba.dx = dx, ba.dy = dy, ba.partial = static_cast<float *>(workspace);
    const unsigned lds = tile.wpr == 1 ? (unsigned)(kVecs * width * sizeof(float)) : 0;
    with_tile(tile, [&](auto nch, auto wpr, auto nw) {
      with_types(x_dtype == MLORA_F32, y_dtype == MLORA_F32, [&](auto xf, auto yf) {
        constexpr int NCH = decltype(nch)::value, WPR = decltype(wpr)::value, NW = decltype(nw)::value;
        constexpr bool XF = decltype(xf)::value, YF = decltype(yf)::value;
        const dim3 grid((unsigned)(batches * a.n_chunks)), block(64 * NW);
        if (sums && post >= 0) hipLaunchKernelGGL((joint_backward_kernel<NCH, WPR, NW, XF, YF, true, true>), grid, block, lds, s, ba);
        else if (sums) hipLaunchKernelGGL((joint_backward_kernel<NCH, WPR, NW, XF, YF, true, false>), grid, block, lds, s, ba);
        else if (post >= 0) hipLaunchKernelGGL((joint_backward_kernel<NCH, WPR, NW, XF, YF, false, true>), grid, block, lds, s, ba);
        else hipLaunchKernelGGL((joint_backward_kernel<NCH, WPR, NW, XF, YF, false, false>), grid, block, lds, s, ba);
      });
    });
    st = launch_status();
    if (st || !sums) return st;
  }
  // the vectors' gradients: per sample, or over all rows (zeros where there is no row)
  ColSums cs;
  const int64_t row = kVecs * width;
  auto job = [&](void *out, int v, int dtype, bool shared) {
    if (out == nullptr) return;
    cs.add({static_cast<const float *>(workspace) + v * width, out, shared ? 0 : n_chunks * row, row,
            (int32_t)(shared ? batches * n_chunks : n_chunks), shared ? 1 : (int32_t)batches, (int32_t)width,
            dtype == MLORA_F32});
  };
  job(dgate, kVecGate, gate_dtype, gate_shared != 0);
  job(dscale, kVecMult, affine_dtype, scale_shared != 0);
  job(dshift, kVecShift, affine_dtype, shift_shared != 0);
  job(dpost, kVecPost, post_dtype, true);
  return launch_col_sums(cs, s);
}
