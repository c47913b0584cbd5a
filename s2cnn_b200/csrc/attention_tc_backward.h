// Attention, backward, bfloat16, on the tensor cores: two kernels, one for the gradient of the queries (and of the bias), one for
// those of keys and values.  Both compute the scores again; a single kernel would save two of seven products but leave the
// sums of the query gradients to atomics, whose order changes results.
//
// Weights and score gradients enter their products in bfloat16: a relative 2^-9 on each of the many terms of a sum that is
// itself rounded to bfloat16.  The bias gradient sums the unrounded ones.
#pragma once

#include "attention_tc.h"

#ifndef S2C_EMUL

namespace s2c {

constexpr int kTcbThreads = 12 * 32;

// Barrier of the 256 threads at the scores.  (A wait that gives up does not take a warp out of their loops: all pass the same
// barriers, and the block writes NaN in the end.)
__device__ __forceinline__ void tcb_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

// ---- gradient of the queries -----------------------------------------------------------------------------------------------
// A block has 128 queries of one head and walks over the keys.  Scores S = Q K^T and dP = dO V^T arrive in tensor memory; warps
// 0 - 3 take the first 64 keys of a tile, warps 4 - 7 the others (thread = query): dS = P (dP - delta) goes back over the scores as
// the left operand of dQ += dS K.  Two score tiles in turn, so that the next scores are there when the threads get to them;
// products are issued by warp 8, keys (three tiles in turn: one is wanted twice, for the scores and for dQ) and values are
// loaded by warps 9 and 10.
// The bias gradient: a tile that lies beyond the reach adds to one bucket, a sum per thread.  In the others each warp adds its 32 x 64
// values along the diagonals: a running sum moves one lane up with every column, so that it follows its diagonal; four runs
// of 16 columns side by side cover the latency of the exchange.  The sums of the eight warps meet in shared memory, where one
// thread per diagonal of the tile adds them in a fixed order to the slot of its relative position.
constexpr int kTcbDiag = 4 * 48;              // floats of a warp: four runs of 47 diagonals
struct TcbQBars {
  uint64_t in_full, s_full[2], dp_full, ds_full, k_full[3], k_empty[3], v_full, v_empty, drained;
  uint32_t tmem;
};
inline size_t tcb_q_smem(int blocks, int reach, bool bias_grad) {
  const size_t tab = 2 * reach + 2 * kTcxMargin + 1;
  return 1024 + (size_t)6 * blocks * kTcxTile + (tab + (bias_grad ? 2 * 8 * kTcbDiag + 2 * reach + 1 : 0) + 512) * sizeof(float) + sizeof(TcbQBars) + 16;
}

template <int NC>
struct AttnTcGradQ {
static constexpr int kThreads = kTcbThreads;
static __device__ __forceinline__ void run(const AttnTcParams& pp, float4* dyn) {
  const AttnParams& p = pp.a;
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  constexpr uint32_t kRows = NC * kTcxTile;
  const uint32_t base = (tcx_addr(dyn) + 1023u) & ~1023u;
  unsigned char* const smem = reinterpret_cast<unsigned char*>(dyn) + (base - tcx_addr(dyn));
  float* const tab = reinterpret_cast<float*>(smem + 6 * (size_t)kRows);
  float* const red = tab + tcx_tab_floats(p.reach);                   // [512]
  float* const diag = red + 512;                                      // [2][8][kTcbDiag], then a slot per relative position
  float* const slot = diag + (p.dbias_part ? 2 * 8 * kTcbDiag : 0);
  TcbQBars* const bars = reinterpret_cast<TcbQBars*>((reinterpret_cast<uintptr_t>(slot + (p.dbias_part ? 2 * p.reach + 1 : 0)) + 15) & ~(uintptr_t)15);
  const uint32_t q_at = base, g_at = base + kRows, k_at = base + 2 * kRows, v_at = base + 5 * kRows;

  const int heads_all = p.batch * p.heads;                            // the longest rows first
  const int tile = p.tiles - 1 - (int)blockIdx.x / heads_all, bh = (int)blockIdx.x % heads_all, h = bh % p.heads, b = bh / p.heads, hk = h / p.group;
  if (tid == 0) {
    tcx_init(&bars->in_full, 256);
    for (int i = 0; i < 2; ++i) tcx_init(&bars->s_full[i], 1);
    tcx_init(&bars->dp_full, 1);
    tcx_init(&bars->ds_full, 8);
    for (int i = 0; i < 3; ++i) {
      tcx_init(&bars->k_full[i], 1);
      tcx_init(&bars->k_empty[i], 1);
    }
    tcx_init(&bars->v_full, 1);
    tcx_init(&bars->v_empty, 1);
    tcx_init(&bars->drained, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  const AttnSeq s = attn_seq(p, b);
  const int i0 = 128 * tile;
  const int keys = i0 < s.qlen ? attn_keys(p, s, min(i0 + 128, s.qlen)) : 0, n = (keys + 127) / 128;
  if (warp == 8) {
    __syncwarp();
    tcx_alloc<512>(&bars->tmem);
  }
  tcx_bias_table(p, h, tab, tid, kTcbThreads, false);
  if (p.dbias_part)
    for (int e = tid; e <= 2 * p.reach; e += kTcbThreads) slot[e] = 0.f;
  tcx_before_sync();
  __syncthreads();
  tcx_after_sync();
  const uint32_t tmem = __shfl_sync(0xffffffffu, bars->tmem, 0);
  stream_order_next();
  const uint32_t t_s = tmem, t_dp = tmem + 256, t_dq = tmem + 384;
  bool ok = true;

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (warp == 8 && n) {
      const int steps = (pp.chunks + 1) / 2;
      const uint32_t is = tcx_idesc(128, false), io = tcx_idesc(16 * steps, true);
      auto scores = [&](int j) {
        if (!(ok = tcx_wait_warp(&bars->k_full[j % 3], (j / 3) & 1))) return;
        if (tcx_elect()) {
          tcx_scores(t_s + 128 * (j & 1), q_at, k_at + (j % 3) * kRows, is, steps);
          tcx_commit(&bars->s_full[j & 1]);
        }
        __syncwarp();
      };
      auto products = [&](int j) {                                     // dP
        if (!(ok = tcx_wait_warp(&bars->v_full, j & 1))) return;
        if (tcx_elect()) {
          tcx_scores(t_dp, g_at, v_at, is, steps);
          tcx_commit(&bars->dp_full);
          tcx_commit(&bars->v_empty);
        }
        __syncwarp();
      };
      ok = tcx_wait_warp(&bars->in_full, 0);
      if (ok) scores(0);
      if (ok) products(0);
      if (ok && n > 1) scores(1);
      for (int j = 0; j < n && ok; ++j) {
        if (!(ok = tcx_wait_warp(&bars->ds_full, j & 1))) break;
        tcx_after_sync();
        if (j + 1 < n) products(j + 1);
        if (!ok) break;
        if (tcx_elect()) {
          tcx_combine(t_dq, t_s + 128 * (j & 1), k_at + (j % 3) * kRows, io, j > 0, 64);
          tcx_commit(&bars->k_empty[j % 3]);
        }
        __syncwarp();
        if (j + 2 < n) scores(j + 2);                                  // in order behind the product that reads these columns
      }
      if (tcx_elect()) tcx_commit(&bars->drained);
      __syncwarp();
      ok = tcx_wait_warp(&bars->drained, 0) && ok;
    } else if (warp == 9) {
      const bf16* src = static_cast<const bf16*>(p.k) + b * p.ks[0] + hk * p.ks[2];
      for (int j = 0; j < n && ok; ++j) {
        if (j >= 3) ok = tcx_wait_warp(&bars->k_empty[j % 3], (j / 3 - 1) & 1);
        if (!ok) break;
        tcx_load_rows<NC, 32>(k_at + (j % 3) * kRows, src, p.ks[1], 128 * j, keys, pp.chunks, lane);
        tcx_loaded();
        __syncwarp();
        if (lane == 0) tcx_arrive(&bars->k_full[j % 3]);
      }
    } else if (warp == 10) {
      const bf16* src = static_cast<const bf16*>(p.v) + b * p.vs[0] + hk * p.vs[2];
      for (int j = 0; j < n && ok; ++j) {
        if (j >= 1) ok = tcx_wait_warp(&bars->v_empty, (j - 1) & 1);
        if (!ok) break;
        tcx_load_rows<NC, 32>(v_at, src, p.vs[1], 128 * j, keys, pp.chunks, lane);
        tcx_loaded();
        __syncwarp();
        if (lane == 0) tcx_arrive(&bars->v_full);
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    const int half = warp >> 2, row = 32 * (warp & 3) + lane, i = i0 + row;
    const long at = (((long)b * p.lq + i) * p.heads + h) * p.dim;
    if (n) {
      tcx_load_rows<NC, 256>(q_at, static_cast<const bf16*>(p.q) + b * p.qs[0] + h * p.qs[2], p.qs[1], i0, s.qlen, pp.chunks, tid);
      tcx_load_rows<NC, 256>(g_at, static_cast<const bf16*>(p.dout) + b * pp.gs[0] + h * pp.gs[2], pp.gs[1], i0, s.qlen, pp.chunks, tid);
      tcx_loaded();
      tcx_arrive(&bars->in_full);
    }
    // delta = dO . O, half of the columns per thread
    float delta = 0.f;
    if (i < s.qlen) {
      const bf16* g = static_cast<const bf16*>(p.dout) + b * pp.gs[0] + (long)i * pp.gs[1] + h * pp.gs[2];
      const bf16 *o = static_cast<const bf16*>(p.o) + at, *lo = static_cast<const bf16*>(p.out_lo) + at;
      if (p.dim % 8 == 0) {
        for (int c = 8 * half; c < p.dim; c += 16) {
          float x[8], y[8], z[8];
          load_vec(g + c, x);
          load_vec(o + c, y);
          load_vec(lo + c, z);
#pragma unroll
          for (int e = 0; e < 8; ++e) delta = fmaf(x[e], y[e] + z[e], delta);
        }
      } else {
        for (int c = half; c < p.dim; c += 2) delta = fmaf(widen(g[c]), widen(o[c]) + widen(lo[c]), delta);
      }
    }
    red[tid] = delta;
    tcb_sync();
    delta = red[row] + red[128 + row];
    const float2 st = i < s.qlen ? p.stats[((long)b * p.heads + h) * p.lq + i] : make_float2(INFINITY, 0.f);
    if (half == 0 && i < p.lq) p.delta[((long)b * p.heads + h) * p.lq + i] = delta;
    const float base_m = -st.x, inv = st.y, shift = -st.y * delta;
    const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
    const float scale = p.scale * kLog2e, tab_before = tab[0], tab_behind = tab[2 * p.reach + 2 * kTcxMargin];
    float far_before = 0.f, far_behind = 0.f;
    int turn = 0;
    for (int j = 0; j < n; ++j) {
      const int j0 = 128 * j, d0 = j0 - i0 - s.start;
      const bool close = d0 + 127 > -p.reach && d0 - 127 < p.reach && p.reach > 0;
      if (ok) ok = tcx_wait_warp(&bars->s_full[j & 1], (j >> 1) & 1);
      tcx_after_sync();
      const uint32_t ts = t_s + 128 * (j & 1) + 64 * half + lanes;
      uint32_t raw[64], grad[64];
      tcx_ld32(ts, raw);
      tcx_ld32(ts + 32, raw + 32);
      tcx_ld_wait(raw);
      tcx_ld_wait(raw + 32);
      float* x = reinterpret_cast<float*>(raw);
      if (close) {
        const float* near = tab + (d0 + 64 * half - row + p.reach + kTcxMargin);
#pragma unroll
        for (int c = 0; c < 64; ++c) x[c] = fmaf(x[c], scale, near[c]) + base_m;      // (as the forward pass rounds it)
      } else {
        const float far = d0 > 0 ? tab_behind : tab_before;
#pragma unroll
        for (int c = 0; c < 64; c += 2) {
          const float2 y = tcx_add2(fma2(make_float2(x[c], x[c + 1]), make_float2(scale, scale), make_float2(far, far)), make_float2(base_m, base_m));
          x[c] = y.x;
          x[c + 1] = y.y;
        }
      }
      const bool edge = j0 + 128 > keys || (p.causal && d0 + 127 > 0);
      const int lim = (p.causal ? min(keys - j0, row - d0 + 1) : keys - j0) - 64 * half;
      if (edge) {
#pragma unroll
        for (int c = 0; c < 64; ++c) x[c] = c < lim ? x[c] : kNoScore;
      }
#pragma unroll
      for (int c = 0; c < 64; ++c) x[c] = exp2_fast(x[c]);
      if (ok) ok = tcx_wait_warp(&bars->dp_full, j & 1);
      tcx_after_sync();
      tcx_ld32(t_dp + 64 * half + lanes, grad);
      tcx_ld32(t_dp + 64 * half + 32 + lanes, grad + 32);
      tcx_ld_wait(grad);
      tcx_ld_wait(grad + 32);
#pragma unroll
      for (int c = 0; c < 64; c += 2) {
        const float2 y = fma2(make_float2(as_float(grad[c]), as_float(grad[c + 1])), make_float2(inv, inv), make_float2(shift, shift));
        x[c] *= y.x;
        x[c + 1] *= y.y;
      }
      if (edge) {
#pragma unroll
        for (int c = 0; c < 64; ++c) x[c] = c < lim ? x[c] : 0.f;
      }
      uint32_t w[32];
#pragma unroll
      for (int c = 0; c < 64; c += 2) w[c / 2] = pack_bf16(x[c], x[c + 1]);
      tcx_st32(ts, w);
      tcx_st_wait();
      tcx_before_sync();
      __syncwarp();
      if (lane == 0) tcx_arrive(&bars->ds_full);
      if (!p.dbias_part) continue;
      if (close) {
        float* mine = diag + (8 * turn + warp) * kTcbDiag;
        float run[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < 16; ++c) {
#pragma unroll
          for (int k = 0; k < 4; ++k) run[k] += x[16 * k + c];
          if (c == 15) break;
          if (lane == 31) {                                            // the diagonal 16 k + c - 31 is complete
#pragma unroll
            for (int k = 0; k < 4; ++k) mine[48 * k + c] = run[k];
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            run[k] = __shfl_up_sync(0xffffffffu, run[k], 1);
            run[k] = lane == 0 ? 0.f : run[k];
          }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) mine[48 * k + 15 + 31 - lane] = run[k];   // diagonals 16 k + 15 - lane
        tcb_sync();
        if (tid < 255) {
          const int off = tid - 127, d = d0 + off;                     // column minus row within the tile, relative position
          float sum = 0.f;
#pragma unroll
          for (int wv = 0; wv < 8; ++wv)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int e = off + 32 * (wv & 3) - 64 * (wv >> 2) - 16 * k + 31;
              if (e >= 0 && e < 47) sum += diag[(8 * turn + wv) * kTcbDiag + 48 * k + e];
            }
          if (d <= -p.reach) far_before += sum;
          else if (d >= p.reach) far_behind += sum;
          else slot[d + p.reach] += sum;
        }
        turn ^= 1;
      } else {
        float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
        for (int c = 0; c < 64; c += 2) sum[(c / 2) & 1] = tcx_add2(sum[(c / 2) & 1], make_float2(x[c], x[c + 1]));
        const float all = (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
        if (d0 > 0) far_behind += all;
        else far_before += all;
      }
    }
    // ---- the gradient of this row: half of the columns per thread
    // (dP's barrier has been followed in every phase, ds_full by the products; the last of them:)
    if (ok && n) ok = tcx_wait_warp(&bars->drained, 0);
    tcx_after_sync();
    const bool wide = p.dim % 8 == 0 && reinterpret_cast<uintptr_t>(p.dq) % 16 == 0;
#pragma unroll
    for (int c = 0; c < 64 * NC; c += 32) {
      if (NC == 1 ? c != 32 * half : c / 64 != half) continue;
      uint32_t o[32];
      if (n) {
        tcx_ld32(t_dq + c + lanes, o);
        tcx_ld_wait(o);
      }
      float v[32];
#pragma unroll
      for (int e = 0; e < 32; ++e) v[e] = !ok ? bulk_nan() : n ? as_float(o[e]) * p.scale : 0.f;
      if (i < p.lq) tcx_put_row(static_cast<bf16*>(p.dq) + at, nullptr, v, 32, p.dim, c, wide);
    }
    if (p.dbias_part) {
      tcb_sync();
      red[tid] = far_before;
      red[256 + tid] = far_behind;
      tcb_sync();
      if (warp < 2) {                                                  // warp 0: before, warp 1: behind
        float sum = 0.f;
        for (int e = lane; e < 256; e += 32) sum += red[256 * warp + e];
#pragma unroll
        for (int m = 16; m >= 1; m /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, m);
        if (lane == 0) red[256 * warp] = sum;
      }
      tcb_sync();
      if (tid == 0) {
        slot[0] = red[0];
        if (p.reach > 0) slot[2 * p.reach] = red[256];
        else slot[0] += red[256];
      }
      tcb_sync();
      float* part = p.dbias_part + (((long)b * p.tiles + tile) * p.heads + h) * p.n_buckets;
      for (int which = tid; which < p.n_buckets; which += 256) {
        float sum = 0.f;
        for (int e = 0; e <= 2 * p.reach; ++e)
          if (p.bucket_of[e] == which) sum += slot[e];
        part[which] = ok ? sum : bulk_nan();
      }
    }
  }
  tcx_before_sync();
  __syncthreads();
  if (warp == 8) tcx_free<512>(tmem);
}
};

// ---- gradients of keys and values -------------------------------------------------------------------------------------------
// A block has 128 keys of one of their heads and walks over the queries of all heads that share it.  The scores are computed
// transposed (thread = key), so that weights and score gradients are left operands again: dV += P^T dO, dK += dS^T Q.  Warps 0 - 3
// take the first 64 queries of a tile, warps 4 - 7 the others; P^T goes over the scores, dS^T over dP^T.  While the threads work on
// dS^T the tensor core has dV and the next scores to do, while they work on the next P^T it has dK and the next dP^T.
// Warps 9 and 10 load queries and dO, warp 11 the rows' statistics.
struct TcbKvBars {
  uint64_t in_full, s_full, dp_full, p_full, ds_full, q_full[2], q_empty[2], g_full[2], g_empty[2], r_full[2], r_empty[2], drained;
  uint32_t tmem;
};
inline size_t tcb_kv_smem(int blocks, int reach) {
  return 1024 + (size_t)6 * blocks * kTcxTile + (2 * 3 * 128 + 2 * reach + 2 * kTcxMargin + 1) * sizeof(float) + sizeof(TcbKvBars) + 16;
}

template <int NC>
struct AttnTcGradKV {
static constexpr int kThreads = kTcbThreads;
static __device__ __forceinline__ void run(const AttnTcParams& pp, float4* dyn) {
  const AttnParams& p = pp.a;
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  constexpr uint32_t kRows = NC * kTcxTile;
  const uint32_t base = (tcx_addr(dyn) + 1023u) & ~1023u;
  unsigned char* const smem = reinterpret_cast<unsigned char*>(dyn) + (base - tcx_addr(dyn));
  float* const stat = reinterpret_cast<float*>(smem + 6 * (size_t)kRows);        // [2][3][128]: -m, 1 / l, -delta
  float* const tab = stat + 2 * 3 * 128;
  TcbKvBars* const bars = reinterpret_cast<TcbKvBars*>((reinterpret_cast<uintptr_t>(tab + tcx_tab_floats(p.reach)) + 15) & ~(uintptr_t)15);
  const uint32_t k_at = base, v_at = base + kRows, q_at = base + 2 * kRows, g_at = base + 4 * kRows;

  const int heads_all = p.batch * p.kv_heads;                         // under `causal` the first keys have the most queries
  const int tile = (int)blockIdx.x / heads_all, bh = (int)blockIdx.x % heads_all, hk = bh % p.kv_heads, b = bh / p.kv_heads;
  if (tid == 0) {
    tcx_init(&bars->in_full, 256);
    tcx_init(&bars->s_full, 1);
    tcx_init(&bars->dp_full, 1);
    tcx_init(&bars->p_full, 8);
    tcx_init(&bars->ds_full, 8);
    for (int i = 0; i < 2; ++i) {
      tcx_init(&bars->q_full[i], 1);
      tcx_init(&bars->q_empty[i], 1);
      tcx_init(&bars->g_full[i], 1);
      tcx_init(&bars->g_empty[i], 1);
      tcx_init(&bars->r_full[i], 1);
      tcx_init(&bars->r_empty[i], 8);
    }
    tcx_init(&bars->drained, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  const AttnSeq s = attn_seq(p, b);
  const int j0 = 128 * tile, keys = attn_keys(p, s, s.qlen);
  const int first = j0 < keys ? attn_first_query(p, s, j0) / 128 : 0;
  const int per_head = j0 < keys ? (s.qlen + 127) / 128 - first : 0, n = per_head > 0 ? per_head * p.group : 0;
  if (warp == 8) {
    __syncwarp();
    tcx_alloc<512>(&bars->tmem);
  }
  tcx_before_sync();
  __syncthreads();
  tcx_after_sync();
  const uint32_t tmem = __shfl_sync(0xffffffffu, bars->tmem, 0);
  stream_order_next();
  const uint32_t t_s = tmem, t_dp = tmem + 128, t_dv = tmem + 256, t_dk = tmem + 384;
  bool ok = true;

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (warp == 8 && n) {
      const int steps = (pp.chunks + 1) / 2;
      const uint32_t is = tcx_idesc(128, false), io = tcx_idesc(16 * steps, true);
      auto scores = [&](int t) {
        if (!(ok = tcx_wait_warp(&bars->q_full[t & 1], (t >> 1) & 1))) return;
        if (tcx_elect()) {
          tcx_scores(t_s, k_at, q_at + (t & 1) * kRows, is, steps);
          tcx_commit(&bars->s_full);
        }
        __syncwarp();
      };
      auto products = [&](int t) {
        if (!(ok = tcx_wait_warp(&bars->g_full[t & 1], (t >> 1) & 1))) return;
        if (tcx_elect()) {
          tcx_scores(t_dp, v_at, g_at + (t & 1) * kRows, is, steps);
          tcx_commit(&bars->dp_full);
        }
        __syncwarp();
      };
      ok = tcx_wait_warp(&bars->in_full, 0);
      if (ok) scores(0);
      if (ok) products(0);
      for (int t = 0; t < n && ok; ++t) {
        if (!(ok = tcx_wait_warp(&bars->p_full, t & 1))) break;
        tcx_after_sync();
        if (tcx_elect()) {
          tcx_combine(t_dv, t_s, g_at + (t & 1) * kRows, io, t > 0, 64);
          tcx_commit(&bars->g_empty[t & 1]);                           // (dP^T of this tile is older)
        }
        __syncwarp();
        if (t + 1 < n) scores(t + 1);
        if (!ok || !(ok = tcx_wait_warp(&bars->ds_full, t & 1))) break;
        tcx_after_sync();
        if (tcx_elect()) {
          tcx_combine(t_dk, t_dp, q_at + (t & 1) * kRows, io, t > 0, 64);
          tcx_commit(&bars->q_empty[t & 1]);
        }
        __syncwarp();
        if (t + 1 < n) products(t + 1);
      }
      if (tcx_elect()) tcx_commit(&bars->drained);
      __syncwarp();
      ok = tcx_wait_warp(&bars->drained, 0) && ok;
    } else if (warp == 9 || warp == 10) {
      const bool is_q = warp == 9;
      uint64_t *full = is_q ? bars->q_full : bars->g_full, *empty = is_q ? bars->q_empty : bars->g_empty;
      const uint32_t to = is_q ? q_at : g_at;
      const long by_head = is_q ? p.qs[2] : pp.gs[2], stride = is_q ? p.qs[1] : pp.gs[1];
      const bf16* src = static_cast<const bf16*>(is_q ? p.q : p.dout) + b * (is_q ? p.qs[0] : pp.gs[0]) + hk * p.group * by_head;
      int g = 0, it = first;
      for (int t = 0; t < n && ok; ++t) {
        if (t >= 2) ok = tcx_wait_warp(&empty[t & 1], (t / 2 - 1) & 1);
        if (!ok) break;
        tcx_load_rows<NC, 32>(to + (t & 1) * kRows, src + g * by_head, stride, 128 * it, s.qlen, pp.chunks, lane);
        tcx_loaded();
        __syncwarp();
        if (lane == 0) tcx_arrive(&full[t & 1]);
        if (++it == first + per_head) { it = first; ++g; }
      }
    } else if (warp == 11) {
      int g = 0, it = first;
      for (int t = 0; t < n && ok; ++t) {
        if (t >= 2) ok = tcx_wait_warp(&bars->r_empty[t & 1], (t / 2 - 1) & 1);
        if (!ok) break;
        const long row0 = ((long)b * p.heads + hk * p.group + g) * p.lq;
        float* to = stat + (t & 1) * 3 * 128;
#pragma unroll
        for (int e = lane; e < 128; e += 32) {
          const int i = 128 * it + e;
          const float2 st = i < s.qlen ? p.stats[row0 + i] : make_float2(INFINITY, 0.f);
          to[e] = -st.x;
          to[128 + e] = st.y;
          to[256 + e] = i < s.qlen ? -p.delta[row0 + i] : 0.f;
        }
        __syncwarp();
        if (lane == 0) tcx_arrive(&bars->r_full[t & 1]);
        if (++it == first + per_head) { it = first; ++g; }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    const int half = warp >> 2, row = 32 * (warp & 3) + lane, j = j0 + row;
    if (n) {
      tcx_load_rows<NC, 256>(k_at, static_cast<const bf16*>(p.k) + b * p.ks[0] + hk * p.ks[2], p.ks[1], j0, keys, pp.chunks, tid);
      tcx_load_rows<NC, 256>(v_at, static_cast<const bf16*>(p.v) + b * p.vs[0] + hk * p.vs[2], p.vs[1], j0, keys, pp.chunks, tid);
      tcx_loaded();
      tcx_arrive(&bars->in_full);
    }
    const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
    const uint32_t ts = t_s + 64 * half + lanes, tp = t_dp + 64 * half + lanes;
    const float scale = p.scale * kLog2e;
    int g = -1, it = first + per_head;
    for (int t = 0; t < n; ++t) {
      if (it == first + per_head) {                                    // the next head: its bias
        it = first;
        ++g;
        tcb_sync();
        tcx_bias_table(p, hk * p.group + g, tab, tid, 256, false);
        tcb_sync();
      }
      const int i0 = 128 * it, d0 = j0 - i0 - s.start;
      const float* sm = stat + (t & 1) * 3 * 128 + 64 * half;          // -m, 1 / l, -delta of this thread's queries
      if (ok) ok = tcx_wait_warp(&bars->r_full[t & 1], (t >> 1) & 1);
      if (ok) ok = tcx_wait_warp(&bars->s_full, t & 1);
      tcx_after_sync();
      uint32_t raw[64], grad[64];
      tcx_ld32(ts, raw);
      tcx_ld32(ts + 32, raw + 32);
      tcx_ld_wait(raw);
      tcx_ld_wait(raw + 32);
      float* x = reinterpret_cast<float*>(raw);
      if (d0 + 127 > -p.reach && d0 - 127 < p.reach && p.reach > 0) {
        const float* near = tab + (d0 + row - 64 * half + p.reach + kTcxMargin);
#pragma unroll
        for (int c = 0; c < 64; c += 4) {
          const float4 m = *reinterpret_cast<const float4*>(sm + c);
          x[c] = fmaf(x[c], scale, near[-c]) + m.x;
          x[c + 1] = fmaf(x[c + 1], scale, near[-c - 1]) + m.y;
          x[c + 2] = fmaf(x[c + 2], scale, near[-c - 2]) + m.z;
          x[c + 3] = fmaf(x[c + 3], scale, near[-c - 3]) + m.w;
        }
      } else {
        const float far = d0 > 0 ? tab[2 * p.reach + 2 * kTcxMargin] : tab[0];
        const float2 f2 = make_float2(far, far), s2 = make_float2(scale, scale);
#pragma unroll
        for (int c = 0; c < 64; c += 4) {
          const float4 m = *reinterpret_cast<const float4*>(sm + c);
          const float2 y = tcx_add2(fma2(make_float2(x[c], x[c + 1]), s2, f2), make_float2(m.x, m.y));
          const float2 z = tcx_add2(fma2(make_float2(x[c + 2], x[c + 3]), s2, f2), make_float2(m.z, m.w));
          x[c] = y.x; x[c + 1] = y.y; x[c + 2] = z.x; x[c + 3] = z.y;
        }
      }
      const bool edge = j0 + 128 > keys || (p.causal && d0 + 127 > 0);
      const int low = j >= keys ? 128 : (p.causal ? d0 + row : 0) - 64 * half;    // first query of this half that sees the key
      if (edge) {
#pragma unroll
        for (int c = 0; c < 64; ++c) x[c] = c >= low ? x[c] : kNoScore;
      }
      uint32_t w[32];
#pragma unroll
      for (int c = 0; c < 64; c += 4) {
        const float4 f = *reinterpret_cast<const float4*>(sm + 128 + c);
        x[c] = exp2_fast(x[c]) * f.x;
        x[c + 1] = exp2_fast(x[c + 1]) * f.y;
        x[c + 2] = exp2_fast(x[c + 2]) * f.z;
        x[c + 3] = exp2_fast(x[c + 3]) * f.w;
        w[c / 2] = pack_bf16(x[c], x[c + 1]);
        w[c / 2 + 1] = pack_bf16(x[c + 2], x[c + 3]);
      }
      tcx_st32(ts, w);
      tcx_st_wait();
      tcx_before_sync();
      __syncwarp();
      if (lane == 0) tcx_arrive(&bars->p_full);
      if (ok) ok = tcx_wait_warp(&bars->dp_full, t & 1);
      tcx_after_sync();
      tcx_ld32(tp, grad);
      tcx_ld32(tp + 32, grad + 32);
      tcx_ld_wait(grad);
      tcx_ld_wait(grad + 32);
#pragma unroll
      for (int c = 0; c < 64; c += 4) {
        const float4 f = *reinterpret_cast<const float4*>(sm + 256 + c);
        x[c] *= as_float(grad[c]) + f.x;
        x[c + 1] *= as_float(grad[c + 1]) + f.y;
        x[c + 2] *= as_float(grad[c + 2]) + f.z;
        x[c + 3] *= as_float(grad[c + 3]) + f.w;
      }
      if (edge) {
#pragma unroll
        for (int c = 0; c < 64; ++c) x[c] = c >= low ? x[c] : 0.f;
      }
#pragma unroll
      for (int c = 0; c < 64; c += 2) w[c / 2] = pack_bf16(x[c], x[c + 1]);
      tcx_st32(tp, w);
      tcx_st_wait();
      tcx_before_sync();
      __syncwarp();
      if (lane == 0) {
        tcx_arrive(&bars->ds_full);
        tcx_arrive(&bars->r_empty[t & 1]);
      }
      ++it;
    }
    // ---- rows of dV (warps 0 - 3) and dK (warps 4 - 7)
    if (ok && n) ok = tcx_wait_warp(&bars->drained, 0);
    tcx_after_sync();
    bf16* out = static_cast<bf16*>(half ? p.dk : p.dv) + (((long)b * p.lk + j) * p.kv_heads + hk) * p.dim;
    const float f = half ? p.scale : 1.f;
    const bool wide = p.dim % 8 == 0 && reinterpret_cast<uintptr_t>(half ? p.dk : p.dv) % 16 == 0;
#pragma unroll
    for (int c = 0; c < 64 * NC; c += 32) {
      uint32_t o[32];
      if (n) {
        tcx_ld32((half ? t_dk : t_dv) + c + lanes, o);
        tcx_ld_wait(o);
      }
      float v[32];
#pragma unroll
      for (int e = 0; e < 32; ++e) v[e] = !ok ? bulk_nan() : n ? as_float(o[e]) * f : 0.f;
      if (j < p.lk) tcx_put_row(out, nullptr, v, 32, p.dim, c, wide);
    }
  }
  tcx_before_sync();
  __syncthreads();
  if (warp == 8) tcx_free<512>(tmem);
}
};

}  // namespace s2c
#endif  // S2C_EMUL
