// Softmax attention with a learned bias by buckets of the relative position, on the FP32 pipes.
//
//   seen(i, j)  = i < q_length and j < kv_length and (not causal or j <= i + start)
//   S(i, j)     = scale q_i . k_j + bias[bucket_of(j - i - start)]           P(i, .) = softmax of S over what i sees
//   o_i = sum_j P(i, j) v_j                                                  (0 where i sees nothing)
//   dV = P^T dO,  dP = dO V^T,  delta_i = dO_i . o_i,  dS = P (dP - delta)
//   dQ = scale dS K,  dK = scale dS^T Q,  dbias[n] = sum of dS over the pairs of bucket n
//
// The scores are kept in units of ln 2 (scale and bias times log2 e), so that the exponential is a power of two.  No score
// leaves the chip: the forward pass walks over the keys with a running maximum m and sum l per row, and keeps m and 1 / l of
// each row; the backward pass computes S again and has P = 2^(S - m) / l.  (m + log2 l as one number would lose l where a
// bias of the type's lowest value makes m huge, and costs P a relative 2^-24 |m| elsewhere.)  A value at a position that no query of a tile sees
// is not read, whatever it holds.
//
// The kernels here take tiles of 64 queries x 64 keys, 16 x 16 threads with 4 x 4 scores each.  They are written for the host
// emulation as well, and on the GPU serve the problems that are too small for the tensor-core kernels.  Bound by the FP32 pipes and
// shared memory: 2 x 4096 positions, 16 heads of 128, forward and backward, 36 ms against 7.6 on the tensor cores (float32).
#pragma once

#include <cfloat>

#include "seq_common.h"

namespace s2c {

struct AttnParams {
  const void *q, *k, *v, *bias, *o, *dout;
  void *out, *dq, *dk, *dv;
  void* out_lo;                   // bfloat16, with stats: what out's rounding left, for delta (see attn_saved_bytes)
  float2* stats;                  // [batch][heads][lq]: m, 1 / l (+inf, 0 where a row sees nothing); forward: null where nobody needs it
  float* delta;                   // [batch][heads][lq]
  float* dbias_part;              // [batch][q tiles][heads][n_buckets], null where not asked for
  float* part;                    // split keys: see AttnFew
  const int *bucket_of, *start, *q_len, *kv_len;
  long qs[3], ks[3], vs[3];       // elements from one batch entry, position, head to the next
  int batch, lq, lk, heads, kv_heads, dim, group;
  int causal, start_all, reach, n_buckets, bias_grad;
  float scale;
  int tiles, splits, chunk;       // tiles of the blocked axis; splits of the keys, of `chunk` keys each
};

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNoScore = -INFINITY;

// lengths and first position of one batch entry, brought into range
struct AttnSeq {
  int qlen, klen, start;
};
S2C_D int attn_clamp(int v, int lo, int hi) { return v < lo ? lo : v > hi ? hi : v; }
S2C_D AttnSeq attn_seq(const AttnParams& p, int b) {
  AttnSeq s;
  s.qlen = p.q_len ? attn_clamp(p.q_len[b], 0, p.lq) : p.lq;
  s.klen = p.kv_len ? attn_clamp(p.kv_len[b], 0, p.lk) : p.lk;
  s.start = attn_clamp(p.start ? p.start[b] : p.start_all, -(1 << 30), 1 << 30);
  return s;
}
// first key beyond all that the queries before `i_end` see
S2C_D int attn_keys(const AttnParams& p, const AttnSeq& s, int i_end) {
  return p.causal ? attn_clamp(i_end + s.start, 0, s.klen) : s.klen;
}
// first query that sees key j (in the order of queries; at most qlen)
S2C_D int attn_first_query(const AttnParams& p, const AttnSeq& s, int j) {
  return p.causal ? attn_clamp(j - s.start, 0, s.qlen) : 0;
}

S2C_D float2 attn_stats(float m, float l) { return l == 0.f ? make_float2(INFINITY, 0.f) : make_float2(m, 1.f / l); }
// a bias in units of ln 2; one of the type's lowest value, as a mask, stays finite
S2C_D float attn_bias_units(float v) {
  constexpr float kLowest = -2.35e38f;                 // times log2 e still a number
  return (v >= -FLT_MAX && v < kLowest ? kLowest : v) * kLog2e;
}
// bias of relative position d at tab[clamp(d) + reach], in units of ln 2; without a bias a single zero
template <class T>
S2C_D void attn_bias_table(const Ctx& ctx, const AttnParams& p, int head, float* tab) {
  for (int e = ctx.tid; e <= 2 * p.reach; e += ctx.nthr) {
    float v = 0.f;
    if (p.bias) {
      const int n = p.bucket_of[e];
      if (n >= 0 && n < p.n_buckets) v = attn_bias_units(widen(static_cast<const T*>(p.bias)[(long)n * p.heads + head]));
    }
    tab[e] = v;
  }
}

constexpr int kAttnTile = 64, kAttnThreads = 256, kAttnPPitch = kAttnTile + 4;

template <int DP>
struct AttnTile {
  static constexpr int kPitch = DP + 4, kFloats = kAttnTile * kPitch;
  static constexpr int kCols = DP / 16;                             // output columns of a thread
  static constexpr int kV = kCols < 4 ? kCols : 4;                  // of them consecutive
  static S2C_D int col(int tx, int c) { return (c / kV) * 16 * kV + tx * kV + c % kV; }

  // rows [r0, r0 + 64) of one head, zeros from row `end` and column dim on
  template <class T>
  static S2C_D void load(const Ctx& ctx, float* dst, const T* src, long row_stride, int r0, int end, int dim) {
    for (int e = ctx.tid; e < kAttnTile * DP; e += kAttnThreads) {
      const int r = e / DP, d = e % DP;
      dst[r * kPitch + d] = r0 + r < end && d < dim ? widen(src[(long)(r0 + r) * row_stride + d]) : 0.f;
    }
  }
  // acc[r][c] = a[4 ty + r] . b[tx + 16 c]
  static S2C_D void dot(const float* a, const float* b, int ty, int tx, float (&acc)[4][4]) {
    float2 s[4][4];
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int c = 0; c < 4; ++c) s[r][c] = make_float2(0.f, 0.f);
#pragma unroll 4
    for (int d = 0; d < DP; d += 4) {
      float4 x[4], y[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) x[r] = *reinterpret_cast<const float4*>(a + (4 * ty + r) * kPitch + d);
#pragma unroll
      for (int c = 0; c < 4; ++c) y[c] = *reinterpret_cast<const float4*>(b + (tx + 16 * c) * kPitch + d);
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          s[r][c] = fma2(make_float2(x[r].x, x[r].y), make_float2(y[c].x, y[c].y), s[r][c]);
          s[r][c] = fma2(make_float2(x[r].z, x[r].w), make_float2(y[c].z, y[c].w), s[r][c]);
        }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int c = 0; c < 4; ++c) acc[r][c] = s[r][c].x + s[r][c].y;
  }
  // acc[r][c] += sum_j w[4 ty + r][j] m[j][col(tx, c)]
  static S2C_D void add_product(const float* w, const float* m, int ty, int tx, float (&acc)[4][kCols]) {
#pragma unroll 2
    for (int j = 0; j < kAttnTile; j += 4) {
      float4 x[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) x[r] = *reinterpret_cast<const float4*>(w + (4 * ty + r) * kAttnPPitch + j);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        float y[kCols];
        const float* row = m + (j + u) * kPitch;
#pragma unroll
        for (int c = 0; c < kCols; ++c) y[c] = row[col(tx, c)];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float f = u == 0 ? x[r].x : u == 1 ? x[r].y : u == 2 ? x[r].z : x[r].w;
#pragma unroll
          for (int c = 0; c < kCols; ++c) acc[r][c] = fmaf(f, y[c], acc[r][c]);
        }
      }
    }
  }
  static S2C_D void put(float* w, int ty, int tx, const float (&v)[4][4]) {
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int c = 0; c < 4; ++c) w[(4 * ty + r) * kAttnPPitch + tx + 16 * c] = v[r][c];
  }
  template <class T>
  static S2C_D void store(T* out, T* lo, long row_stride, int r0, int end, int dim, int ty, int tx, const float (&v)[4][kCols]) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int row = r0 + 4 * ty + r;
      if (row >= end) continue;
#pragma unroll
      for (int c = 0; c < kCols; ++c)
        if (col(tx, c) < dim) {
          const long at = (long)row * row_stride + col(tx, c);
          narrow_with_rest(out + at, lo ? lo + at : nullptr, v[r][c]);
        }
    }
  }
};

// ---- forward: a block takes 64 queries of one head and walks over the keys ---------------------------------------------
template <class T, int DP>
struct AttnForward {
  using Params = AttnParams;
  using Tile = AttnTile<DP>;
  static constexpr int kThreads = kAttnThreads, kBlocks = DP > 64 ? 1 : 2;
  static size_t smem(const Params& p) { return (3 * Tile::kFloats + kAttnTile * kAttnPPitch + 2 * p.reach + 1) * sizeof(float); }
  static S2C_D void run(const Ctx& ctx, const Params& p, unsigned char* smem) {
    float* qt = reinterpret_cast<float*>(smem);
    float *kt = qt + Tile::kFloats, *vt = kt + Tile::kFloats, *pt = vt + Tile::kFloats, *tab = pt + kAttnTile * kAttnPPitch;
    const int tx = ctx.tid % 16, ty = ctx.tid / 16;
    const int i0 = ctx.bid % p.tiles * kAttnTile, bh = ctx.bid / p.tiles, h = bh % p.heads, b = bh / p.heads;
    const AttnSeq s = attn_seq(p, b);
    const T* q = static_cast<const T*>(p.q) + b * p.qs[0] + h * p.qs[2];
    const T* k = static_cast<const T*>(p.k) + b * p.ks[0] + (h / p.group) * p.ks[2];
    const T* v = static_cast<const T*>(p.v) + b * p.vs[0] + (h / p.group) * p.vs[2];
    attn_bias_table<T>(ctx, p, h, tab);
    Tile::load(ctx, qt, q, p.qs[1], i0, s.qlen, p.dim);
    const int keys = i0 < s.qlen ? attn_keys(p, s, i0 + kAttnTile < s.qlen ? i0 + kAttnTile : s.qlen) : 0;
    const float scale = p.scale * kLog2e;
    float m[4], l[4], acc[4][Tile::kCols];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      m[r] = kNoScore;
      l[r] = 0.f;
#pragma unroll
      for (int c = 0; c < Tile::kCols; ++c) acc[r][c] = 0.f;
    }
    for (int j0 = 0; j0 < keys; j0 += kAttnTile) {
      ctx.sync();                                          // the tiles of the turn before have been read
      Tile::load(ctx, kt, k, p.ks[1], j0, keys, p.dim);
      Tile::load(ctx, vt, v, p.vs[1], j0, keys, p.dim);
      ctx.sync();
      float w[4][4];
      Tile::dot(qt, kt, ty, tx, w);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = i0 + 4 * ty + r;
        float top = kNoScore;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int j = j0 + tx + 16 * c, d = j - i - s.start;
          const bool seen = j < keys && i < s.qlen && (!p.causal || d <= 0);
          w[r][c] = seen ? w[r][c] * scale + tab[attn_clamp(d, -p.reach, p.reach) + p.reach] : kNoScore;
          top = w[r][c] > top ? w[r][c] : top;
        }
        top = lanes_max<16>(ctx, top);
        top = top > m[r] ? top : m[r];
        const float base = top == kNoScore ? 0.f : top;      // nothing seen yet: all weights 2^-inf = 0
        const float old = exp2_fast(m[r] - base);
        float sum = 0.f;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          w[r][c] = exp2_fast(w[r][c] - base);
          sum += w[r][c];
        }
        m[r] = top;
        l[r] = l[r] * old + sum;                             // (this lane's share of the sum)
#pragma unroll
        for (int c = 0; c < Tile::kCols; ++c) acc[r][c] *= old;
      }
      Tile::put(pt, ty, tx, w);
      ctx.sync();
      Tile::add_product(pt, vt, ty, tx, acc);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float sum = lanes_sum<16>(ctx, l[r]);
      const float inv = attn_stats(m[r], sum).y;
#pragma unroll
      for (int c = 0; c < Tile::kCols; ++c) acc[r][c] = inv == 0.f ? 0.f : acc[r][c] * inv;      // (0 times a NaN that others see)
      const int i = i0 + 4 * ty + r;
      if (p.stats && tx == 0 && i < p.lq) p.stats[(long)bh * p.lq + i] = attn_stats(m[r], sum);
    }
    const long out = ((long)b * p.lq * p.heads + h) * p.dim;
    Tile::store(static_cast<T*>(p.out) + out, p.out_lo ? static_cast<T*>(p.out_lo) + out : nullptr, (long)p.heads * p.dim, i0, p.lq, p.dim, ty, tx, acc);
  }
};

// ---- gradient of the queries and of the bias: a block takes 64 queries of one head --------------------------------------
// The bias gradient sums dS along the diagonals of the tiles: a diagonal has one relative position.  Thread t of the first
// 127 adds diagonal t of each tile to the slot of its position (one thread per slot and tile), beyond the reach to a
// register; what the buckets of the block get is added from the slots in order.
template <class T, int DP>
struct AttnGradQ {
  using Params = AttnParams;
  using Tile = AttnTile<DP>;
  static constexpr int kThreads = kAttnThreads, kBlocks = DP > 32 ? 1 : 2;
  static size_t smem(const Params& p) {
    return (4 * Tile::kFloats + kAttnTile * kAttnPPitch + 3 * kAttnTile + 2 * (2 * p.reach + 1) + 256) * sizeof(float);
  }
  static S2C_D void run(const Ctx& ctx, const Params& p, unsigned char* smem) {
    float* qt = reinterpret_cast<float*>(smem);
    float *gt = qt + Tile::kFloats, *kt = gt + Tile::kFloats, *vt = kt + Tile::kFloats, *pt = vt + Tile::kFloats;
    float *top = pt + kAttnTile * kAttnPPitch, *inv = top + kAttnTile, *delta = inv + kAttnTile, *far = delta + kAttnTile, *tab = far + 256, *slot = tab + 2 * p.reach + 1;
    const int tx = ctx.tid % 16, ty = ctx.tid / 16;
    const int i0 = ctx.bid % p.tiles * kAttnTile, bh = ctx.bid / p.tiles, h = bh % p.heads, b = bh / p.heads;
    const AttnSeq s = attn_seq(p, b);
    const T* q = static_cast<const T*>(p.q) + b * p.qs[0] + h * p.qs[2];
    const T* k = static_cast<const T*>(p.k) + b * p.ks[0] + (h / p.group) * p.ks[2];
    const T* v = static_cast<const T*>(p.v) + b * p.vs[0] + (h / p.group) * p.vs[2];
    const long row0 = ((long)b * p.lq * p.heads + h) * p.dim, row_stride = (long)p.heads * p.dim;
    attn_bias_table<T>(ctx, p, h, tab);
    for (int e = ctx.tid; e <= 2 * p.reach; e += ctx.nthr) slot[e] = 0.f;
    Tile::load(ctx, qt, q, p.qs[1], i0, s.qlen, p.dim);
    Tile::load(ctx, gt, static_cast<const T*>(p.dout) + row0, row_stride, i0, s.qlen, p.dim);
    Tile::load(ctx, kt, static_cast<const T*>(p.o) + row0, row_stride, i0, s.qlen, p.dim);
    if (p.out_lo) Tile::load(ctx, vt, static_cast<const T*>(p.out_lo) + row0, row_stride, i0, s.qlen, p.dim);
    ctx.sync();
    if (ctx.tid < kAttnTile) {
      float d = 0.f;
      for (int c = 0; c < DP; ++c) {
        const int at = ctx.tid * Tile::kPitch + c;
        d = fmaf(gt[at], p.out_lo ? kt[at] + vt[at] : kt[at], d);
      }
      const int i = i0 + ctx.tid;
      const float2 st = i < s.qlen ? p.stats[(long)bh * p.lq + i] : make_float2(INFINITY, 0.f);
      top[ctx.tid] = st.x;
      inv[ctx.tid] = st.y;
      delta[ctx.tid] = d;
      if (i < p.lq) p.delta[(long)bh * p.lq + i] = d;
    }
    const int keys = i0 < s.qlen ? attn_keys(p, s, i0 + kAttnTile < s.qlen ? i0 + kAttnTile : s.qlen) : 0;
    const float scale = p.scale * kLog2e;
    float acc[4][Tile::kCols], far_before = 0.f, far_behind = 0.f;
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int c = 0; c < Tile::kCols; ++c) acc[r][c] = 0.f;
    for (int j0 = 0; j0 < keys; j0 += kAttnTile) {
      ctx.sync();
      Tile::load(ctx, kt, k, p.ks[1], j0, keys, p.dim);
      Tile::load(ctx, vt, v, p.vs[1], j0, keys, p.dim);
      ctx.sync();
      float w[4][4], g[4][4];
      Tile::dot(qt, kt, ty, tx, w);
      Tile::dot(gt, vt, ty, tx, g);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = i0 + 4 * ty + r;
        const float base = top[4 * ty + r], f = inv[4 * ty + r], dl = delta[4 * ty + r];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int j = j0 + tx + 16 * c, d = j - i - s.start;
          const bool seen = j < keys && i < s.qlen && (!p.causal || d <= 0);
          const float x = w[r][c] * scale + tab[attn_clamp(d, -p.reach, p.reach) + p.reach];
          w[r][c] = seen ? exp2_fast(x - base) * f * (g[r][c] - dl) : 0.f;
        }
      }
      Tile::put(pt, ty, tx, w);
      ctx.sync();
      Tile::add_product(pt, kt, ty, tx, acc);
      if (p.dbias_part && ctx.tid < 2 * kAttnTile - 1) {
        const int off = ctx.tid - (kAttnTile - 1), d = j0 - i0 - s.start + off;     // column minus row, relative position
        float sum = 0.f;
        for (int r = off < 0 ? -off : 0; r < kAttnTile && r + off < kAttnTile; ++r) sum += pt[r * kAttnPPitch + r + off];
        if (d <= -p.reach) far_before += sum;
        else if (d >= p.reach) far_behind += sum;
        else slot[d + p.reach] += sum;
      }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int c = 0; c < Tile::kCols; ++c) acc[r][c] = inv[4 * ty + r] == 0.f ? 0.f : acc[r][c] * p.scale;
    Tile::store(static_cast<T*>(p.dq) + row0, (T*)nullptr, row_stride, i0, p.lq, p.dim, ty, tx, acc);
    if (!p.dbias_part) return;
    ctx.sync();
    if (ctx.tid < 128) { far[ctx.tid] = far_before; far[128 + ctx.tid] = far_behind; }
    ctx.sync();
    if (ctx.tid < 2) {
      float sum = 0.f;
      for (int e = 0; e < 127; ++e) sum += far[128 * ctx.tid + e];
      if (p.reach > 0 || ctx.tid == 0) slot[ctx.tid * 2 * p.reach] = sum;
    }
    ctx.sync();
    if (p.reach == 0 && ctx.tid == 0)                     // one slot for everything: d <= 0 and d > 0
      for (int e = 0; e < 127; ++e) slot[0] += far[128 + e];
    ctx.sync();
    float* part = p.dbias_part + (((long)b * p.tiles + ctx.bid % p.tiles) * p.heads + h) * p.n_buckets;
    for (int n = ctx.tid; n < p.n_buckets; n += ctx.nthr) {
      float sum = 0.f;
      for (int e = 0; e <= 2 * p.reach; ++e)
        if (p.bucket_of[e] == n) sum += slot[e];
      part[n] = sum;
    }
  }
};

// dbias[n][h]: the sum over batch entries and tiles, 8 values to a block, every 32nd part to a thread, in a fixed order
struct AttnBiasSumParams {
  const float* part;    // [parts][heads][n_buckets]
  void* out;            // [n_buckets][heads]
  int parts, heads, n_buckets;
};
template <class T>
struct AttnBiasSum {
  using Params = AttnBiasSumParams;
  static constexpr int kThreads = 256, kBlocks = 4;
  static S2C_D void run(const Ctx& ctx, const Params& p, unsigned char* smem) {
    float* red = reinterpret_cast<float*>(smem);           // [32][8]
    const int values = p.heads * p.n_buckets, v = ctx.bid * 8 + ctx.tid % 8, lane = ctx.tid / 8;
    float s = 0.f;
    if (v < values) {
#pragma unroll 8
      for (int k = lane; k < p.parts; k += 32) s += p.part[(long)k * values + v];
    }
    red[ctx.tid] = s;
    ctx.sync();
    if (lane != 0 || v >= values) return;
    for (int k = 1; k < 32; ++k) s += red[8 * k + ctx.tid];
    narrow(static_cast<T*>(p.out) + (long)(v % p.n_buckets) * p.heads + v / p.n_buckets, s);
  }
};

// ---- gradients of keys and values: a block takes 64 keys of one of their heads and walks over the queries of all heads that
// share it, so that the sum over the shared heads stays in registers ------------------------------------------------------
template <class T, int DP>
struct AttnGradKV {
  using Params = AttnParams;
  using Tile = AttnTile<DP>;
  static constexpr int kThreads = kAttnThreads, kBlocks = DP > 32 ? 1 : 2;
  static size_t smem(const Params& p) {
    return (4 * Tile::kFloats + 2 * kAttnTile * kAttnPPitch + 3 * kAttnTile + 2 * p.reach + 1) * sizeof(float);
  }
  static S2C_D void run(const Ctx& ctx, const Params& p, unsigned char* smem) {
    float* kt = reinterpret_cast<float*>(smem);
    float *vt = kt + Tile::kFloats, *qt = vt + Tile::kFloats, *gt = qt + Tile::kFloats, *pt = gt + Tile::kFloats;
    float *st = pt + kAttnTile * kAttnPPitch, *top = st + kAttnTile * kAttnPPitch, *inv = top + kAttnTile, *delta = inv + kAttnTile, *tab = delta + kAttnTile;
    const int tx = ctx.tid % 16, ty = ctx.tid / 16;
    const int j0 = ctx.bid % p.tiles * kAttnTile, bh = ctx.bid / p.tiles, hk = bh % p.kv_heads, b = bh / p.kv_heads;
    const AttnSeq s = attn_seq(p, b);
    const int keys = attn_keys(p, s, s.qlen);
    Tile::load(ctx, kt, static_cast<const T*>(p.k) + b * p.ks[0] + hk * p.ks[2], p.ks[1], j0, keys, p.dim);
    Tile::load(ctx, vt, static_cast<const T*>(p.v) + b * p.vs[0] + hk * p.vs[2], p.vs[1], j0, keys, p.dim);
    const float scale = p.scale * kLog2e;
    float dk[4][Tile::kCols], dv[4][Tile::kCols];
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int c = 0; c < Tile::kCols; ++c) dk[r][c] = dv[r][c] = 0.f;
    const int first = j0 < keys ? attn_first_query(p, s, j0) / kAttnTile * kAttnTile : s.qlen;
    for (int h = hk * p.group; h < (hk + 1) * p.group; ++h) {
      const T* q = static_cast<const T*>(p.q) + b * p.qs[0] + h * p.qs[2];
      const T* g = static_cast<const T*>(p.dout) + ((long)b * p.lq * p.heads + h) * p.dim;
      const long stat = ((long)b * p.heads + h) * p.lq;
      ctx.sync();
      attn_bias_table<T>(ctx, p, h, tab);
      for (int i0 = first; i0 < s.qlen; i0 += kAttnTile) {
        ctx.sync();
        Tile::load(ctx, qt, q, p.qs[1], i0, s.qlen, p.dim);
        Tile::load(ctx, gt, g, (long)p.heads * p.dim, i0, s.qlen, p.dim);
        if (ctx.tid < kAttnTile) {
          const float2 rs = i0 + ctx.tid < s.qlen ? p.stats[stat + i0 + ctx.tid] : make_float2(INFINITY, 0.f);
          top[ctx.tid] = rs.x;
          inv[ctx.tid] = rs.y;
          delta[ctx.tid] = i0 + ctx.tid < s.qlen ? p.delta[stat + i0 + ctx.tid] : 0.f;
        }
        ctx.sync();
        float w[4][4], x[4][4];                            // rows: keys, columns: queries
        Tile::dot(kt, qt, ty, tx, w);
        Tile::dot(vt, gt, ty, tx, x);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int j = j0 + 4 * ty + r;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int i = i0 + tx + 16 * c, d = j - i - s.start;
            const bool seen = j < keys && i < s.qlen && (!p.causal || d <= 0);
            const float y = w[r][c] * scale + tab[attn_clamp(d, -p.reach, p.reach) + p.reach];
            w[r][c] = seen ? exp2_fast(y - top[tx + 16 * c]) * inv[tx + 16 * c] : 0.f;
            x[r][c] = seen ? w[r][c] * (x[r][c] - delta[tx + 16 * c]) : 0.f;
          }
        }
        Tile::put(pt, ty, tx, w);
        Tile::put(st, ty, tx, x);
        ctx.sync();
        Tile::add_product(pt, gt, ty, tx, dv);
        Tile::add_product(st, qt, ty, tx, dk);
      }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int c = 0; c < Tile::kCols; ++c) dk[r][c] *= p.scale;
    const long out = ((long)b * p.lk * p.kv_heads + hk) * p.dim, row = (long)p.kv_heads * p.dim;
    Tile::store(static_cast<T*>(p.dk) + out, (T*)nullptr, row, j0, p.lk, p.dim, ty, tx, dk);
    Tile::store(static_cast<T*>(p.dv) + out, (T*)nullptr, row, j0, p.lk, p.dim, ty, tx, dv);
  }
};

}  // namespace s2c
