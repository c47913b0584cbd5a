// Attention, forward, bfloat16, on the tensor cores.
//
// A block takes one or two tiles of 128 queries that read the same keys: neighbouring tiles of a head, or the same tile of
// heads that share a key head.  Roles (12 warps):
//   * warps 0 - 3 and 4 - 7, one group per query tile: thread = row = tensor-memory lane.  A group takes the finished scores of
//     64 keys from tensor memory, adds the bias, finds the running maximum, writes the weights 2^(x - m), rounded to
//     bfloat16, over the scores (half of their columns) and keeps the sum of the unrounded ones;
//   * warps 8 and 11 issue the products of a group each: scores of a tile, and weights times values into the output in tensor memory;
//   * warps 9 and 10 load keys and values, four tiles ahead of each.
// A group has two buffers of scores: the next tile's are there while it is at the exponentials of this one.  (With one buffer for
// tiles of 128 keys and one issuing thread: 2 x 4096 positions, 16 heads of 128, 287 us, now 269; of 64, in training, 253 / 229.  The
// tiles of 64 with one issuing thread: 278 and 256.)
// Its registers come from the third warpgroup (launched with 168 each: 8 x 208 + 4 x 88 = 12 x 168).
// The output is rescaled only where the maximum of a row has grown by more than 8 (in units of ln 2) since it was last fixed:
// weights then reach 2^8 at most, which costs no precision, and after the first tiles rescaling all but ends.
// 2 x 4096 positions, 16 heads of 128: 257 us, 1071 TFLOP/s (the last wave halved); with a bias 264, and 340 where its gradient is
// asked for.  Bound by the exponentials (16 a clock and SM: 60 % of the time) and the tensor pipe (66 % of the measured peak), which
// overlap but in part.  A quarter of the exponentials as polynomials on the FP32 pipes gave nothing (260 us).
// Weights in bfloat16: a relative 2^-9 on each of the many terms of an output that is itself rounded to bfloat16.
#pragma once

#include "attention_tc.h"

#ifndef S2C_EMUL

namespace s2c {

constexpr int kTcfThreads = 12 * 32;
constexpr float kTcfGrow = 8.f;

// pv_done: products with the values of even and odd tiles.  (The scores of tile j tell a group that the product of j - 2 is done: on one
// barrier for all, whose waits tell two neighbouring phases apart and no more, the one of j - 2 could pass for that of j.)
struct TcfBars {
  uint64_t q_full[2], s_full[2][2], p_full[2][2], pv_done[2][2], k_full[4], k_empty[4], v_full[4], v_empty[4], drained[2];
  uint32_t tmem;
};

inline size_t tcf_smem(int blocks, int per_block, int reach) {       // blocks of 64 columns
  return 1024 + (size_t)(per_block + 4) * blocks * kTcxTile + (size_t)per_block * (2 * reach + 2 * kTcxMargin + 1) * sizeof(float) + sizeof(TcfBars) + 16;
}

// FINE, where a bias gradient will be asked for: the weights' rounding goes into a second product, in the other half of the
// scores' columns.  That gradient sums dS = P (dP - delta) over all rows, delta = dO . O is one number for a whole row, and an output whose weights were rounded
// gives it an error that does not average out (relative error of the bias gradient, 2 x 4096 positions, 16 heads of 128:
// 2.4e-3 without, against 1.7e-3 of its own rounding).
template <int NC, bool FINE>
struct AttnTcForward {
static constexpr int kThreads = kTcfThreads;
static __device__ __forceinline__ void run(const AttnTcParams& pp, float4* s2c_dyn_smem) {
  const AttnParams& p = pp.a;
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  constexpr uint32_t kQ = NC * kTcxTile, kRows = kQ / 2;             // bytes of a tile of 128 queries, of 64 keys
  const uint32_t base = (tcx_addr(s2c_dyn_smem) + 1023u) & ~1023u;
  unsigned char* const smem = reinterpret_cast<unsigned char*>(s2c_dyn_smem) + (base - tcx_addr(s2c_dyn_smem));
    float* const tab = reinterpret_cast<float*>(smem + (size_t)(pp.per_block + 4) * kQ);
  TcfBars* const bars = reinterpret_cast<TcfBars*>((reinterpret_cast<uintptr_t>(tab + pp.per_block * tcx_tab_floats(p.reach)) + 15) & ~(uintptr_t)15);
  const uint32_t q_at = base, k_at = base + pp.per_block * kQ, v_at = k_at + 4 * kRows;

  // the longest rows (the last queries under `causal`) first
  const int heads_all = p.batch * p.kv_heads;
  const int cut = max(0, (int)blockIdx.x - pp.whole), at = (int)blockIdx.x - (cut + 1) / 2;
  const bool single = (int)blockIdx.x >= pp.whole;
  const int pair = pp.pairs - 1 - at / heads_all, bh = at % heads_all, hk = bh % p.kv_heads, b = bh / p.kv_heads;

  const AttnSeq s = attn_seq(p, b);
  // unit = tile * group + (head within its group): first row, head and key tiles of this block's query tiles
  int i0[2], head[2], keys[2], n[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int unit = pair * pp.per_block + u + (single ? cut & 1 : 0);
    const bool on = u < (single ? 1 : pp.per_block) && unit < pp.units;
    i0[u] = on ? unit / p.group * 128 : p.lq;
    head[u] = hk * p.group + (on ? unit % p.group : 0);
    keys[u] = i0[u] < s.qlen ? attn_keys(p, s, min(i0[u] + 128, s.qlen)) : 0;
    n[u] = (keys[u] + 63) / 64;
  }
  const int n_all = max(n[0], n[1]), keys_all = max(keys[0], keys[1]);
  const int users = max(1, (n[0] > 0) + (n[1] > 0));                 // issuing threads that read a tile of keys
  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      tcx_init(&bars->q_full[i], 128);
      for (int e = 0; e < 2; ++e) {
        tcx_init(&bars->s_full[i][e], 1);
        tcx_init(&bars->p_full[i][e], 4);
        tcx_init(&bars->pv_done[i][e], 1);
      }
      tcx_init(&bars->drained[i], 1);
    }
    for (int i = 0; i < 4; ++i) {
      tcx_init(&bars->k_full[i], 32);
      tcx_init(&bars->k_empty[i], users);
      tcx_init(&bars->v_full[i], 32);
      tcx_init(&bars->v_empty[i], users);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 8) {
    __syncwarp();
    tcx_alloc<512>(&bars->tmem);
  }
  for (int u = 0; u < pp.per_block; ++u) tcx_bias_table(p, head[u], tab + u * tcx_tab_floats(p.reach), tid, kTcfThreads, false);
  tcx_before_sync();
  __syncthreads();
  tcx_after_sync();
  const uint32_t tmem = __shfl_sync(0xffffffffu, bars->tmem, 0);
  stream_order_next();
  // tensor memory: scores (and weights) of either tile, then their outputs
  const uint32_t t_scores = tmem, t_out = tmem + 256;
  bool ok = true;

  if (warp >= 8) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
  if (warp == 8 || warp == 11) {
    const int u = warp == 11;
    if (n[u] && tcx_elect()) {               // one thread issues all of a group: a warp's votes cost it 100 clocks a wait
      const int steps = (pp.chunks + 1) / 2;
      const uint32_t is = tcx_idesc(64, false), io = tcx_idesc(16 * steps, true);
      const uint32_t q = q_at + u * kQ, scores = t_scores + 128 * u, out = t_out + 128 * u;
      ok = tcx_wait(&bars->q_full[u], 0);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if (!ok || j >= n_all) break;
        ok = tcx_wait(&bars->k_full[j], 0);
        tcx_seen();
        if (!ok) break;
        if (j < n[u]) {
          tcx_scores<NC, 128, 64>(scores + 64 * j, q, k_at + j * kRows, is);
          tcx_commit(&bars->s_full[u][j]);
        }
        tcx_commit(&bars->k_empty[j]);
      }
      // (a group that is done early still waits for the tiles that the other one needs, so that their slots are given back in turn)
      for (int j = 0; j < n_all && ok; ++j) {
        const int sv = j & 3, sk = (j + 2) & 3, turn = j & 1;
        const uint32_t w = scores + 64 * turn;
        ok = tcx_wait(&bars->v_full[sv], (j >> 2) & 1);
        tcx_seen();
        if (ok && j < n[u]) {
          ok = tcx_wait(&bars->p_full[u][turn], (j >> 1) & 1);
          if (!ok) break;
          tcx_after_sync();
          const uint32_t v = v_at + sv * kRows;
          if (FINE) tcx_combine<64, 64>(out, w + 32, v, io, j > 0);
          tcx_combine<64, 64>(out, w, v, io, FINE || j > 0);
          tcx_commit(&bars->pv_done[u][turn]);
        }
        if (!ok) break;
        tcx_commit(&bars->v_empty[sv]);
        if (j + 2 < n_all) {
          ok = tcx_wait(&bars->k_full[sk], ((j + 2) >> 2) & 1);
          tcx_seen();
          if (!ok) break;
          if (j + 2 < n[u]) {                // in order behind the product that reads the weights from the same columns
            tcx_scores<NC, 128, 64>(w, q, k_at + sk * kRows, is);
            tcx_commit(&bars->s_full[u][turn]);
          }
          tcx_commit(&bars->k_empty[sk]);
        }
      }
      tcx_commit(&bars->drained[u]);         // nothing may be in flight when tensor memory is given back
      tcx_wait(&bars->drained[u], 0);
    }
    __syncwarp();
  } else if (warp == 9 || warp == 10) {
    const bool is_k = warp == 9;
    const bf16* src = static_cast<const bf16*>(is_k ? p.k : p.v) + b * (is_k ? p.ks[0] : p.vs[0]) + hk * (is_k ? p.ks[2] : p.vs[2]);
    const long stride = is_k ? p.ks[1] : p.vs[1];
    uint64_t *full = is_k ? bars->k_full : bars->v_full, *empty = is_k ? bars->k_empty : bars->v_empty;
    const uint32_t at = is_k ? k_at : v_at;
    for (int j = 0; j < n_all && ok; ++j) {
      const int slot = j & 3;
      if (j >= 4) ok = tcx_wait_warp(&empty[slot], (j / 4 - 1) & 1);
      if (!ok) break;
      tcx_load_rows<NC, 32, 64>(at + slot * kRows, src, stride, 64 * j, keys_all, pp.chunks, lane);
      tcx_arrive_copies(&full[slot]);
    }
    tcx_copies_done();
  }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    const int u = warp >> 2, row = 32 * (warp & 3) + lane;
    if (u < pp.per_block && i0[u] < p.lq) {
      const int i = i0[u] + row, h = head[u];
      if (n[u]) {
        tcx_load_rows<NC, 128>(q_at + u * kQ, static_cast<const bf16*>(p.q) + b * p.qs[0] + h * p.qs[2], p.qs[1], i0[u], s.qlen, pp.chunks, tid & 127);
        tcx_loaded();
        tcx_arrive(&bars->q_full[u]);
      }
      const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
      const uint32_t to = t_out + 128 * u + lanes;
      const float* tb = tab + u * tcx_tab_floats(p.reach);
      const float scale = p.scale * kLog2e, far_before = tb[0], far_behind = tb[2 * p.reach + 2 * kTcxMargin];
      float m = kNoScore, l = 0.f;
      for (int j = 0; j < n[u]; ++j) {
        const int j0 = 64 * j, d0 = j0 - i0[u] - s.start;             // relative position of the tile's first key to its first query
        const uint32_t ts = t_scores + 128 * u + 64 * (j & 1) + lanes;
        if (!(ok = tcx_wait_warp(&bars->s_full[u][j & 1], (j >> 1) & 1))) break;
        tcx_after_sync();
        uint32_t raw[64];
        tcx_ld32(ts, raw);
        tcx_ld32(ts + 32, raw + 32);
        tcx_ld_wait(raw);
        tcx_ld_wait(raw + 32);
        float* x = reinterpret_cast<float*>(raw);
        const bool close = d0 + 63 > -p.reach && d0 - 127 < p.reach && p.reach > 0;
        const bool edge = j0 + 64 > keys[u] || (p.causal && d0 + 63 > 0);            // some pairs of the tile are not seen
        const float far = d0 > 0 ? far_behind : far_before;
        // A tile of one bias, all seen: the maximum of the raw scores tells that of the others, and scale, bias and maximum are one
        // multiply-add.  (Not for a bias so large that the scores vanish beside it, see AttnParams::stats.)
        const bool plain = !close && !edge && scale > 0.f && fabsf(far) < 1e30f;
        if (!plain) {
          if (close) {
            const float* near = tb + (d0 - row + p.reach + kTcxMargin);
#pragma unroll
            for (int c = 0; c < 64; ++c) x[c] = fmaf(x[c], scale, near[c]);
          } else {
#pragma unroll
            for (int c = 0; c < 64; ++c) x[c] = fmaf(x[c], scale, far);
          }
          if (edge) {
            const int lim = p.causal ? min(keys[u] - j0, row - d0 + 1) : keys[u] - j0;
#pragma unroll
            for (int c = 0; c < 64; ++c) x[c] = c < lim ? x[c] : kNoScore;
          }
        }
        float top[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
        for (int c = 4; c < 60; c += 8)
#pragma unroll
          for (int e = 0; e < 4; ++e) top[e] = tcx_max3(top[e], x[c + e], x[c + 4 + e]);
        float now = fmaxf(tcx_max3(top[0], top[1], top[2]), tcx_max3(top[3], x[60], x[61]));
        now = tcx_max3(now, x[62], x[63]);
        if (plain) now = fmaf(now, scale, far);
        if (__any_sync(0xffffffffu, now > m + kTcfGrow)) {
          const float fresh = now > m + kTcfGrow ? now : m;
          if (j > 0) {
            const float f = fresh == m ? 1.f : exp2_fast(m - fresh);
            if (!(ok = tcx_wait_warp(&bars->pv_done[u][(j - 1) & 1], ((j - 1) >> 1) & 1))) break;
            tcx_after_sync();
            l *= f;
#pragma unroll
            for (int c = 0; c < 64 * NC; c += 32) {
              uint32_t o[32];
              tcx_ld32(to + c, o);
              tcx_ld_wait(o);
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = as_bits(as_float(o[e]) * f);
              tcx_st32(to + c, o);
            }
          }
          m = fresh;
        }
        const float base = m == kNoScore ? 0.f : -m, mul = plain ? scale : 1.f, add = plain ? far + base : base;
        float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        uint32_t w[32], rest[FINE ? 32 : 1];
#pragma unroll
        for (int c = 0; c < 64; c += 2) {
          float2 y = fma2(make_float2(x[c], x[c + 1]), make_float2(mul, mul), make_float2(add, add));
          y.x = exp2_fast(y.x);
          y.y = exp2_fast(y.y);
          sum[(c / 2) & 1] = tcx_add2(sum[(c / 2) & 1], y);
          w[c / 2] = pack_bf16(y.x, y.y);
          if constexpr (FINE) rest[c / 2] = pack_bf16(y.x - as_float(w[c / 2] << 16), y.y - as_float(w[c / 2] & 0xffff0000u));
        }
        tcx_st32(ts, w);
        if constexpr (FINE) tcx_st32(ts + 32, rest);
        tcx_st_wait();
        tcx_before_sync();
        __syncwarp();
        if (lane == 0) tcx_arrive(&bars->p_full[u][j & 1]);
        l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
      }
      // ---- the output row
      if (i >= s.qlen) l = 0.f;
      const float2 st = attn_stats(m, l);
      if (ok && n[u]) ok = tcx_wait_warp(&bars->pv_done[u][(n[u] - 1) & 1], ((n[u] - 1) >> 1) & 1);
      tcx_after_sync();
      const long at = (((long)b * p.lq + i) * p.heads + h) * p.dim;
      bf16* out = static_cast<bf16*>(p.out) + at;
      bf16* lo = p.out_lo ? static_cast<bf16*>(p.out_lo) + at : nullptr;
      const bool wide = p.dim % 8 == 0 && reinterpret_cast<uintptr_t>(p.out) % 16 == 0;
#pragma unroll
      for (int c = 0; c < 64 * NC; c += 32) {
        uint32_t o[32];
        if (n[u]) {
          tcx_ld32(to + c, o);
          tcx_ld_wait(o);
        }
        float v[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) v[e] = !ok ? bulk_nan() : l == 0.f ? 0.f : as_float(o[e]) * st.y;
        if (i < p.lq) tcx_put_row(out, lo, v, 32, p.dim, c, wide);
      }
      if (p.stats && i < p.lq) p.stats[((long)b * p.heads + h) * p.lq + i] = st;
    }
  }
  tcx_before_sync();
  __syncthreads();
  if (warp == 8) tcx_free<512>(tmem);
}
};

}  // namespace s2c
#endif  // S2C_EMUL
