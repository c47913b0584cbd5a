// Attention of few queries (one new position of each recording, say): the queries of all heads that share a key head make up to
// 16 rows, and the time is that of reading the keys and values once, 4 lq dim heads / kv_heads flops for every 2 dim values.
//
// A block of four warps (eight for float32) takes `chunk` keys.  A warp has tiles of 16 keys (8) to itself: it copies them into shared memory, two
// tiles ahead (the copies in flight are what the memory's rate asks for: 100 KB per SM at 128 values), and never waits for
// another warp.  Scores and outputs are products of 16 rows on the warp-level matrix instructions, which are far from their
// limit here; the large tiles of tcgen05 would be one eighth full.  To keep float32 exact to a few units, an operand v is split
// as hi + lo (hi: v rounded to TF32) and lo lo is dropped; bfloat16 weights are split the same way, so that only the output is
// rounded.  The warps' results, and those of the blocks of a split (AttnJoin), are joined in a fixed order.
//
// 16 x 16384 keys, 16 heads of 128 on 4: bfloat16 105 us (5.1 TB/s), lengths 1024 to 16384 73 us (3.9), float32 266 us (4.0).
// Three blocks per SM with two tiles ahead, or a share of the same size for every block whatever the lengths: the same.
#pragma once

#include "attention_kernels.h"

#ifndef S2C_EMUL

namespace s2c {

constexpr int kFewRows = 16;

__device__ __forceinline__ void few_mma(float (&d)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void few_mma_tf32(float (&d)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
  asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ unsigned few_tf32(float v) {
  unsigned r;
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(v));
  return r;
}
struct FewSplit {
  unsigned hi, lo;
};
__device__ __forceinline__ FewSplit few_split(float v) {
  const unsigned h = few_tf32(v);
  return {h, as_bits(v - as_float(h))};
}
template <bool TRANS>
__device__ __forceinline__ void few_ldmatrix(unsigned (&r)[4], unsigned addr) {
  if constexpr (TRANS)
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
  else
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

// Rows in shared memory, in bytes: padded so that the matrix loads (bfloat16) and the fragments of keys and values (float32) of
// a warp come from different banks.
template <class T, int DP>
struct FewLayout {
  static constexpr int kKeyPitch = sizeof(T) == 2 ? (DP + 8) * 2 : (DP + 4) * 4;
  static constexpr int kValuePitch = sizeof(T) == 2 ? (DP + 8) * 2 : (DP + 8) * 4;
  // float32 tiles of 8 keys, so that twice as many warps share the memory: its products take three times the instructions
  static constexpr int kKeys = sizeof(T) == 2 ? 16 : 8, kWarps = sizeof(T) == 2 ? 4 : 8;
  static constexpr int kStage = kKeys * (kKeyPitch + kValuePitch);
  static constexpr int kStages = 3;
  static constexpr int kWarp = kStage * kStages;
};

// PIECE: bytes of one copy, 16 or 4, as alignment and strides allow; 2: by plain loads
template <class T, int DP, int PIECE>
struct AttnFew {
  using Params = AttnParams;
  using L = FewLayout<T, DP>;
  static constexpr int kFewKeys = L::kKeys, kFewWarps = L::kWarps;
  static constexpr int kThreads = 32 * kFewWarps, kBlocks = DP > 64 && sizeof(T) == 4 ? 1 : 2;
  static constexpr int kHalves = kFewKeys / 8;                       // tiles of 8 keys
  static constexpr int kNt = DP / 8;                                 // output tiles of 8 columns
  static constexpr int kKs = sizeof(T) == 2 ? DP / 16 : DP / 8;      // steps of the scores' products
  static size_t smem(const Params& p) {
    const size_t tiles = (size_t)kFewWarps * L::kWarp, join = (size_t)kFewWarps * kFewRows * (DP + 2) * sizeof(float);
    return std::max(tiles, join) + (size_t)p.group * (2 * p.reach + 1) * sizeof(float);
  }
  // `left` rows that hold values (16: a whole tile), zeros behind them.  Where 32 lanes take whole rows a lane's copies are at
  // constant distances.
  static __device__ __forceinline__ void copy_rows(unsigned char* dst, int pitch, const T* src, long stride, int left, int dim, int lane) {
    constexpr int kPer = DP * (int)sizeof(T) / PIECE, kElems = PIECE / (int)sizeof(T);     // pieces of a row, values of a piece
    auto piece = [&](unsigned char* to, const T* from, bool on) {
      if constexpr (PIECE == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((unsigned)__cvta_generic_to_shared(to)), "l"(on ? from : src), "r"(on ? 16 : 0) : "memory");
      else if constexpr (PIECE == 4)
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"((unsigned)__cvta_generic_to_shared(to)), "l"(on ? from : src), "r"(on ? 4 : 0) : "memory");
      else
        *reinterpret_cast<unsigned short*>(to) = on ? reinterpret_cast<const unsigned short*>(from)[0] : (unsigned short)0;
    };
    if constexpr (kPer <= 32) {
      constexpr int kRowsAtOnce = 32 / kPer;
      const int r = lane / kPer, c = lane % kPer;
      const T* from = src + r * stride + c * kElems;
      unsigned char* to = dst + r * pitch + c * PIECE;
      const bool in = c * kElems < dim;
#pragma unroll
      for (int it = 0; it < kFewKeys / kRowsAtOnce; ++it) {
        piece(to + it * kRowsAtOnce * pitch, from, in && it * kRowsAtOnce + r < left);
        from += kRowsAtOnce * stride;
      }
    } else {
#pragma unroll 4
      for (int r = 0; r < kFewKeys; ++r)
#pragma unroll
        for (int c = lane; c < kPer; c += 32) piece(dst + r * pitch + c * PIECE, src + r * stride + c * kElems, r < left && c * kElems < dim);
    }
  }
  static __device__ __forceinline__ void run(const Ctx& ctx, const Params& p, unsigned char* smem) {
    const int lane = ctx.tid % 32, warp = ctx.tid / 32, rows = p.lq * p.group;
    const int split = ctx.bid % p.splits, bh = ctx.bid / p.splits, hk = bh % p.kv_heads, b = bh / p.kv_heads;
    constexpr size_t kTiles = (size_t)kFewWarps * L::kWarp, kJoin = (size_t)kFewWarps * kFewRows * (DP + 2) * sizeof(float);
    float* const tab = reinterpret_cast<float*>(smem + (kTiles > kJoin ? kTiles : kJoin));
    const AttnSeq s = attn_seq(p, b);
    const int keys = attn_keys(p, s, s.qlen), j_lo = split * p.chunk, j_end = min(keys, j_lo + p.chunk);
    const T* k = static_cast<const T*>(p.k) + b * p.ks[0] + hk * p.ks[2];
    const T* v = static_cast<const T*>(p.v) + b * p.vs[0] + hk * p.vs[2];
    unsigned char* const mine = smem + warp * L::kWarp;
    const int n = j_lo < j_end ? (j_end - j_lo + kFewKeys - 1) / kFewKeys : 0;         // tiles of the block; this warp: every kFewWarps-th
    auto fetch = [&](int t, int stage) {
      if (t < n) {
        const int j0 = j_lo + t * kFewKeys;
        copy_rows(mine + stage * L::kStage, L::kKeyPitch, k + j0 * p.ks[1], p.ks[1], j_end - j0, p.dim, lane);
        copy_rows(mine + stage * L::kStage + kFewKeys * L::kKeyPitch, L::kValuePitch, v + j0 * p.vs[1], p.vs[1], j_end - j0, p.dim, lane);
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int i = 0; i < L::kStages - 1; ++i) fetch(warp + i * kFewWarps, i);
    // a chunk that lies before the reach of every query has one bias per head, and needs no table
    const bool far = n && j_end - 1 - s.start <= -p.reach;
    if (n && !far)
      for (int g = 0; g < p.group; ++g) attn_bias_table<T>(ctx, p, hk * p.group + g, tab + g * (2 * p.reach + 1));
    // fragments of the queries: rows lane / 4 and that + 8
    unsigned q_hi[kKs][4], q_lo[sizeof(T) == 2 ? 1 : kKs][4];
    int pos[2], of_tab[2];
    bool in_row[2];
    float flat[2] = {0.f, 0.f};
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = lane / 4 + 8 * e, i = r / p.group;
      in_row[e] = r < rows && i < s.qlen;
      pos[e] = i + s.start;
      of_tab[e] = (r < rows ? r % p.group : 0) * (2 * p.reach + 1) + p.reach;
      const T* q = static_cast<const T*>(p.q) + b * p.qs[0] + (in_row[e] ? i * p.qs[1] + (hk * p.group + r % p.group) * p.qs[2] : 0);
      if (far && p.bias && r < rows) {
        const int which = p.bucket_of[0];
        if (which >= 0 && which < p.n_buckets) flat[e] = attn_bias_units(widen(static_cast<const T*>(p.bias)[(long)which * p.heads + hk * p.group + r % p.group]));
      }
      auto at = [&](int c) { return in_row[e] && n && c < p.dim ? widen(q[c]) : 0.f; };
#pragma unroll
      for (int ks = 0; ks < kKs; ++ks) {
        if constexpr (sizeof(T) == 2) {
          const int c = 16 * ks + 2 * (lane % 4);
          q_hi[ks][e] = pack_bf16(at(c), at(c + 1));
          q_hi[ks][2 + e] = pack_bf16(at(c + 8), at(c + 9));
        } else {
          const int c = 8 * ks + lane % 4;
          const FewSplit x = few_split(at(c)), y = few_split(at(c + 4));
          q_hi[ks][e] = x.hi;
          q_lo[ks][e] = x.lo;
          q_hi[ks][2 + e] = y.hi;
          q_lo[ks][2 + e] = y.lo;
        }
      }
    }
    ctx.sync();                                                       // the table
    const float scale = p.scale * kLog2e;
    float acc[kNt][4], m[2] = {kNoScore, kNoScore}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int t = 0; t < kNt; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[t][e] = 0.f;
    int stage = 0;
    for (int t = warp; t < n; t += kFewWarps) {
      fetch(t + (L::kStages - 1) * kFewWarps, stage == 0 ? L::kStages - 1 : stage - 1);
      asm volatile("cp.async.wait_group %0;" ::"n"(L::kStages - 1) : "memory");
      __syncwarp();
      const unsigned char *kt = mine + stage * L::kStage, *vt = kt + kFewKeys * L::kKeyPitch;
      // ---- scores: two tiles of 8 keys
      float x[kHalves][4] = {};
      if constexpr (sizeof(T) == 2) {
        const unsigned addr = (unsigned)__cvta_generic_to_shared(kt) + (lane % 8 + (lane / 16) * 8) * L::kKeyPitch + ((lane / 8) % 2) * 16;
#pragma unroll
        for (int ks = 0; ks < kKs; ++ks) {
          unsigned r[4];
          few_ldmatrix<false>(r, addr + 32 * ks);
          few_mma(x[0], q_hi[ks], r[0], r[1]);
          few_mma(x[1], q_hi[ks], r[2], r[3]);
        }
      } else {
        float y[2][kHalves][4] = {};
#pragma unroll
        for (int ks = 0; ks < kKs; ++ks)
#pragma unroll
          for (int h = 0; h < kHalves; ++h) {
            const float* row = reinterpret_cast<const float*>(kt + (8 * h + lane / 4) * L::kKeyPitch) + 8 * ks + lane % 4;
            const FewSplit b0 = few_split(row[0]), b1 = few_split(row[4]);
            few_mma_tf32(y[0][h], q_lo[ks], b0.hi, b1.hi);            // three chains side by side, each a third as long
            few_mma_tf32(y[1][h], q_hi[ks], b0.lo, b1.lo);
            few_mma_tf32(x[h], q_hi[ks], b0.hi, b1.hi);
          }
#pragma unroll
        for (int h = 0; h < kHalves; ++h)
#pragma unroll
          for (int e = 0; e < 4; ++e) x[h][e] += y[0][h][e] + y[1][h][e];
      }
      // ---- weights
      float top[2] = {kNoScore, kNoScore};
#pragma unroll
      for (int h = 0; h < kHalves; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int j = j_lo + t * kFewKeys + 8 * h + 2 * (lane % 4) + e % 2, d = j - pos[e / 2];
          const bool seen = j < j_end && in_row[e / 2] && (!p.causal || d <= 0);
          const float bias = far ? flat[e / 2] : tab[of_tab[e / 2] + attn_clamp(d, -p.reach, p.reach)];
          x[h][e] = seen ? fmaf(x[h][e], scale, bias) : kNoScore;
          top[e / 2] = fmaxf(top[e / 2], x[h][e]);
        }
      float f[2], base[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 1));
        top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 2));
        top[e] = fmaxf(top[e], m[e]);
        base[e] = top[e] == kNoScore ? 0.f : top[e];
        f[e] = exp2_fast(m[e] - base[e]);
      }
      if (__any_sync(0xffffffffu, top[0] != m[0] || top[1] != m[1])) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          l[e] *= f[e];
          m[e] = top[e];
        }
#pragma unroll
        for (int c = 0; c < kNt; ++c) {
          acc[c][0] *= f[0];
          acc[c][1] *= f[0];
          acc[c][2] *= f[1];
          acc[c][3] *= f[1];
        }
      }
#pragma unroll
      for (int h = 0; h < kHalves; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[h][e] = exp2_fast(x[h][e] - base[e / 2]);
          l[e / 2] += x[h][e];
        }
      // ---- outputs
      if constexpr (sizeof(T) == 2) {
        unsigned hi[4], lo[4];
#pragma unroll
        for (int h = 0; h < kHalves; ++h)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float u = x[h][2 * e], w = x[h][2 * e + 1];
            const unsigned r = pack_bf16(u, w);
            hi[2 * h + e] = r;
            lo[2 * h + e] = pack_bf16(u - as_float(r << 16), w - as_float(r & 0xffff0000u));
          }
        const unsigned addr = (unsigned)__cvta_generic_to_shared(vt) + (lane % 16) * L::kValuePitch + (lane / 16) * 16;
#pragma unroll
        for (int c = 0; c < kNt; c += 2) {
          unsigned r[4];
          few_ldmatrix<true>(r, addr + 16 * c);
          few_mma(acc[c], lo, r[0], r[1]);
          few_mma(acc[c], hi, r[0], r[1]);
          few_mma(acc[c + 1], lo, r[2], r[3]);
          few_mma(acc[c + 1], hi, r[2], r[3]);
        }
      } else {
        // a step of 8 keys; its columns lane % 4 and that + 4 are keys 2 (lane % 4) and that + 1, as the scores lie
#pragma unroll
        for (int h = 0; h < kHalves; ++h) {
          unsigned hi[4], lo[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const FewSplit w = few_split(x[h][2 * (e % 2) + e / 2]);
            hi[e] = w.hi;
            lo[e] = w.lo;
          }
          const float* row = reinterpret_cast<const float*>(vt + (8 * h + 2 * (lane % 4)) * L::kValuePitch) + lane / 4;
#pragma unroll
          for (int c = 0; c < kNt; ++c) {
            const FewSplit b0 = few_split(row[8 * c]), b1 = few_split(row[8 * c + L::kValuePitch / 4]);
            few_mma_tf32(acc[c], lo, b0.hi, b1.hi);
            few_mma_tf32(acc[c], hi, b0.lo, b1.lo);
            few_mma_tf32(acc[c], hi, b0.hi, b1.hi);
          }
        }
      }
      __syncwarp();                                                   // the stage may be written again
      stage = stage + 1 == L::kStages ? 0 : stage + 1;
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    ctx.sync();
    // ---- the warps' results: [warp][row][DP values, maximum, sum]
    float* const join = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
      l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
      float* to = join + (warp * kFewRows + lane / 4 + 8 * e) * (DP + 2);
#pragma unroll
      for (int c = 0; c < kNt; ++c) {
        to[8 * c + 2 * (lane % 4)] = acc[c][2 * e];
        to[8 * c + 2 * (lane % 4) + 1] = acc[c][2 * e + 1];
      }
      if (lane % 4 == 0) {
        to[DP] = m[e];
        to[DP + 1] = l[e];
      }
    }
    ctx.sync();
    for (int e = ctx.tid; e < rows * DP; e += kThreads) {
      const int r = e / DP, c = e % DP;
      float top = kNoScore;
#pragma unroll
      for (int w = 0; w < kFewWarps; ++w) top = fmaxf(top, join[(w * kFewRows + r) * (DP + 2) + DP]);
      const float base = top == kNoScore ? 0.f : top;
      float o = 0.f, sum = 0.f;
#pragma unroll
      for (int w = 0; w < kFewWarps; ++w) {
        const float* from = join + (w * kFewRows + r) * (DP + 2);
        const float g = exp2_fast(from[DP] - base);
        o = fmaf(from[c], g, o);
        sum = fmaf(from[DP + 1], g, sum);
      }
      const int i = r / p.group, h = hk * p.group + r % p.group;
      if (p.splits == 1) {
        const float2 st = attn_stats(top, sum);
        const long to = (((long)b * p.lq + i) * p.heads + h) * p.dim + c;
        if (c < p.dim) narrow_with_rest(static_cast<T*>(p.out) + to, p.out_lo ? static_cast<T*>(p.out_lo) + to : nullptr, st.y == 0.f ? 0.f : o * st.y);
        if (p.stats && c == 0) p.stats[((long)b * p.heads + h) * p.lq + i] = st;
      } else {
        float* part = p.part + ((long)ctx.bid * rows + r) * (DP + 2);
        part[c] = o;
        if (c == 0) { part[DP] = top; part[DP + 1] = sum; }
      }
    }
  }
};

// Joins the splits: a block per row.  The splits' maxima and sums come in one load per thread and turn, the outputs in loads
// that do not wait for one another: thread t has column t % DP of every kThreads / DP-th split.
template <class T, int DP>
struct AttnJoin {
  using Params = AttnParams;
  static constexpr int kThreads = 128, kBlocks = 8, kSlices = kThreads / DP;
  static size_t smem(const Params& p) { return (p.splits + kThreads + 8) * sizeof(float); }
  static __device__ __forceinline__ void run(const Ctx& ctx, const Params& p, unsigned char* smem) {
    const int rows = p.lq * p.group, t = ctx.tid, lane = t % 32, warp = t / 32;
    float *red = reinterpret_cast<float*>(smem), *outs = red + 8, *weight = outs + kThreads;
    const int r = ctx.bid % rows, bh = ctx.bid / rows, hk = bh % p.kv_heads, b = bh / p.kv_heads;
    const AttnSeq s = attn_seq(p, b);                                  // splits beyond the keys have nothing
    const int keys = attn_keys(p, s, s.qlen), n = (keys + p.chunk - 1) / p.chunk;
    const float* part = p.part + ((long)bh * p.splits * rows + r) * (DP + 2);
    const long step = (long)rows * (DP + 2);
    float m = kNoScore;
    for (int e = t; e < n; e += kThreads) m = fmaxf(m, part[e * step + DP]);
    m = lanes_max<32>(ctx, m);
    if (lane == 0) red[warp] = m;
    ctx.sync();
    m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    const float base = m == kNoScore ? 0.f : m;
    float l = 0.f;
    for (int e = t; e < n; e += kThreads) {
      const float f = exp2_fast(part[e * step + DP] - base);
      weight[e] = f;
      l = fmaf(part[e * step + DP + 1], f, l);
    }
    l = lanes_sum<32>(ctx, l);
    if (lane == 0) red[4 + warp] = l;
    ctx.sync();
    l = (red[4] + red[5]) + (red[6] + red[7]);
    const int c = t % DP;
    float o = 0.f;
#pragma unroll 8
    for (int e = t / DP; e < n; e += kSlices) o = fmaf(part[e * step + c], weight[e], o);
    outs[t] = o;
    ctx.sync();
    if (t >= DP) return;
    for (int e = 1; e < kSlices; ++e) o += outs[e * DP + t];
    const int i = r / p.group, h = hk * p.group + r % p.group;
    const float2 st = attn_stats(m, l);
    if (t < p.dim) {
      const long to = (((long)b * p.lq + i) * p.heads + h) * p.dim + t;
      narrow_with_rest(static_cast<T*>(p.out) + to, p.out_lo ? static_cast<T*>(p.out_lo) + to : nullptr, st.y == 0.f ? 0.f : o * st.y);
    }
    if (p.stats && t == 0) p.stats[((long)b * p.heads + h) * p.lq + i] = st;
  }
};

}  // namespace s2c
#endif  // S2C_EMUL
