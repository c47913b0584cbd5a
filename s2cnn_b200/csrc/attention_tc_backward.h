// Attention, backward, bfloat16, on the tensor cores: two kernels, one for the gradient of the queries (and of the bias), one for
// those of keys and values.  Both compute the scores again; a single kernel would save two of seven products but leave the
// sums of the query gradients to atomics, whose order changes results.
//
// Weights and score gradients enter their products in bfloat16: a relative 2^-9 on each of the many terms of a sum that is
// itself rounded to bfloat16.  The bias gradient sums the unrounded ones.
//
// Either kernel walks in tiles of 64 (keys, queries), which its two groups of four warps take in turn, each with score and
// product buffers of its own in tensor memory: while one group is at its exponentials the other one is at its multiplications,
// and the tensor core has the next tile of both to do.  (With tiles of 128, half of the columns to a group, both groups were
// in the same phase and each kernel took the sum of the two.)
//
// 2 x 4096 positions, 16 heads of 128: gradient of the queries 401 us (1027 TFLOP/s), 457 with that of the bias, keys and values 480 us
// (1145 TFLOP/s); 16 of 64: 310, 380 and 427 us.  Tensor pipe active 54 and 61 % of the time, the rest waits between the steps.
#pragma once

#include "attention_tc.h"

#ifndef S2C_EMUL

namespace s2c {

constexpr int kTcbThreads = 12 * 32, kTcbTile = 64;

// Barrier of the 256 threads at the scores, and of one group's 128.  (A wait that gives up does not take a warp out of their loops:
// all pass the same barriers, and the block writes NaN in the end.)
__device__ __forceinline__ void tcb_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }
__device__ __forceinline__ void tcb_sync_group(int group) { asm volatile("bar.sync %0, 128;" ::"r"(2 + group) : "memory"); }

// ---- gradient of the queries -----------------------------------------------------------------------------------------------
// A block has 128 queries of one head (thread = query = tensor-memory lane) and walks over the keys.  Queries and dO lie in
// tensor memory as left operands for the whole time: S = Q K^T, dP = dO V^T, dQ += dS K with dS = P (dP - delta) written over dP.
// The next scores of a group are computed as soon as it has read the last ones.  Warp 8 issues the scores, warp 11 dP and dQ
// (issuing one step with its waits takes a thread some 1500 clocks, as long as two groups take for two tiles), warps 9 and 10 load
// keys and values.
// The bias gradient: a tile that lies beyond the reach adds to one bucket, a sum per thread.  In the others each warp adds its 32 x 64
// values along the diagonals: a running sum moves one lane up with every column, so that it follows its diagonal; four runs
// of 16 columns side by side cover the latency of the exchange.  The sums of a group's four warps meet in shared memory, where
// one thread per diagonal of the tile adds them in a fixed order to the group's slot of the relative position.
constexpr int kTcbDiag = 4 * 48;              // floats of a warp: four runs of 47 diagonals
struct TcbQBars {
  uint64_t in_full, s_full[2], s_read[2], dp_full[2], ds_full[2], k_full[5], k_empty[5], v_full[3], v_empty[3], drained;
  uint32_t tmem;
};

template <int NC>
struct AttnTcGradQ {
  static constexpr int kThreads = kTcbThreads, KS = 5, VS = 3;               // tiles of keys and values in turn
  static constexpr uint32_t kRows = NC * kTcbTile * 128;                     // bytes of a tile
  static size_t smem(int reach, bool bias_grad) {
    const size_t tab = 2 * reach + 2 * kTcxMargin + 1;
    return 1024 + (size_t)(KS + VS) * kRows + (tab + (bias_grad ? 2 * 2 * 4 * kTcbDiag + 2 * (2 * reach + 1) : 0) + 512) * sizeof(float) + sizeof(TcbQBars) + 16;
  }
  static __device__ __forceinline__ void run(const AttnTcParams& pp, float4* dyn) {
    const AttnParams& p = pp.a;
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const uint32_t base = (tcx_addr(dyn) + 1023u) & ~1023u;
    unsigned char* const smem = reinterpret_cast<unsigned char*>(dyn) + (base - tcx_addr(dyn));
    float* const red = reinterpret_cast<float*>(smem + (KS + VS) * (size_t)kRows);     // [512]
    float* const tab = red + 512;
    float* const diag = tab + tcx_tab_floats(p.reach);                       // [group][turn][warp][kTcbDiag], then slots
    float* const slots = diag + (p.dbias_part ? 2 * 2 * 4 * kTcbDiag : 0);   // [group][2 reach + 1]
    TcbQBars* const bars = reinterpret_cast<TcbQBars*>((reinterpret_cast<uintptr_t>(slots + (p.dbias_part ? 2 * (2 * p.reach + 1) : 0)) + 15) & ~(uintptr_t)15);
    const uint32_t k_at = base, v_at = base + KS * kRows;
    const int heads_all = p.batch * p.heads;                                 // the longest rows first
    const int tile = p.tiles - 1 - (int)blockIdx.x / heads_all, bh = (int)blockIdx.x % heads_all, h = bh % p.heads, b = bh / p.heads, hk = h / p.group;
    if (tid == 0) {
      tcx_init(&bars->in_full, 8);
      for (int i = 0; i < 2; ++i) {
        tcx_init(&bars->s_full[i], 1);
        tcx_init(&bars->s_read[i], 4);
        tcx_init(&bars->dp_full[i], 1);
        tcx_init(&bars->ds_full[i], 4);
      }
      for (int i = 0; i < KS; ++i) {
        tcx_init(&bars->k_full[i], 32);
        tcx_init(&bars->k_empty[i], 1);
      }
      for (int i = 0; i < VS; ++i) {
        tcx_init(&bars->v_full[i], 32);
        tcx_init(&bars->v_empty[i], 1);
      }
      tcx_init(&bars->drained, 2);
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    const AttnSeq s = attn_seq(p, b);
    const int i0 = 128 * tile;
    const int keys = i0 < s.qlen ? attn_keys(p, s, min(i0 + 128, s.qlen)) : 0, n = (keys + kTcbTile - 1) / kTcbTile;
    if (warp == 8) {
      __syncwarp();
      tcx_alloc<512>(&bars->tmem);
    }
    tcx_bias_table(p, h, tab, tid, kTcbThreads, false);
    if (p.dbias_part)
      for (int e = tid; e < 2 * (2 * p.reach + 1); e += kTcbThreads) slots[e] = 0.f;
    tcx_before_sync();
    __syncthreads();
    tcx_after_sync();
    const uint32_t tmem = __shfl_sync(0xffffffffu, bars->tmem, 0);
    stream_order_next();
    // scores and products of either group, the gradient, queries and dO as left operands
    const uint32_t t_s = tmem, t_dp = tmem + 128, t_dq = tmem + 256, t_q = t_dq + 64 * NC, t_g = t_q + 32 * NC;
    static_assert(256 + 64 * NC + 2 * 32 * NC <= 512, "tensor memory");
    bool ok = true;

    if (warp >= 8) {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
      if (warp == 8 || warp == 11) {
        if (n && tcx_elect()) {
          const int steps = (pp.chunks + 1) / 2;
          const uint32_t is = tcx_idesc(kTcbTile, false), io = tcx_idesc(16 * steps, true);
          ok = tcx_wait(&bars->in_full, 0);
          tcx_after_sync();
          if (warp == 8) {                                                   // the scores
            TcxRing<KS> k;
            for (int j = 0; j < n && ok; ++j, k.next()) {
              if (j >= 2 && !(ok = tcx_wait(&bars->s_read[j & 1], ((j >> 1) - 1) & 1))) break;
              if (!(ok = tcx_wait(&bars->k_full[k.at], k.parity))) break;
              tcx_after_sync();
              tcx_seen();
              tcx_scores_t<NC, kTcbTile>(t_s + kTcbTile * (j & 1), t_q, k_at + k.at * kRows, is);
              tcx_commit(&bars->s_full[j & 1]);
            }
          } else {                                                           // dP, and the gradient
            TcxRing<KS> k;
            TcxRing<VS> v;
            for (int j = -2; j < n && ok; ++j) {
              if (j >= 0) {
                if (!(ok = tcx_wait(&bars->ds_full[j & 1], (j >> 1) & 1))) break;
                tcx_after_sync();
                tcx_combine<kTcbTile, kTcbTile>(t_dq, t_dp + kTcbTile * (j & 1), k_at + k.at * kRows, io, j > 0);
                tcx_commit(&bars->k_empty[k.at]);
                k.next();
              }
              if (j + 2 < n) {                                               // in order behind the product that reads these columns
                if (!(ok = tcx_wait(&bars->v_full[v.at], v.parity))) break;
                tcx_seen();
                tcx_scores_t<NC, kTcbTile>(t_dp + kTcbTile * (j & 1), t_g, v_at + v.at * kRows, is);
                tcx_commit(&bars->dp_full[j & 1]);
                tcx_commit(&bars->v_empty[v.at]);
                v.next();
              }
            }
          }
          tcx_commit(&bars->drained);
          tcx_wait(&bars->drained, 0);
        }
        __syncwarp();
      } else if (warp == 9) {
        const bf16* src = static_cast<const bf16*>(p.k) + b * p.ks[0] + hk * p.ks[2];
        for (int j = 0; j < n && ok; ++j) {
          if (j >= KS) ok = tcx_wait_warp(&bars->k_empty[j % KS], (j / KS - 1) & 1);
          if (!ok) break;
          tcx_load_rows<NC, 32, kTcbTile>(k_at + (j % KS) * kRows, src, p.ks[1], kTcbTile * j, keys, pp.chunks, lane);
          tcx_arrive_copies(&bars->k_full[j % KS]);
        }
        tcx_copies_done();
      } else if (warp == 10) {
        const bf16* src = static_cast<const bf16*>(p.v) + b * p.vs[0] + hk * p.vs[2];
        for (int j = 0; j < n && ok; ++j) {
          if (j >= VS) ok = tcx_wait_warp(&bars->v_empty[j % VS], (j / VS - 1) & 1);
          if (!ok) break;
          tcx_load_rows<NC, 32, kTcbTile>(v_at + (j % VS) * kRows, src, p.vs[1], kTcbTile * j, keys, pp.chunks, lane);
          tcx_arrive_copies(&bars->v_full[j % VS]);
        }
        tcx_copies_done();
      }
    } else {
      asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
      const int group = warp >> 2, row = 32 * (warp & 3) + lane, i = i0 + row;
      const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
      const long at = (((long)b * p.lq + i) * p.heads + h) * p.dim;
      const bool in = i < s.qlen;
      const bf16* const g_row = static_cast<const bf16*>(p.dout) + b * pp.gs[0] + (long)(in ? i : 0) * pp.gs[1] + h * pp.gs[2];
      if (n) {                                                               // half of the columns of the row per group
        const bf16* const q_row = static_cast<const bf16*>(p.q) + b * p.qs[0] + (long)(in ? i : 0) * p.qs[1] + h * p.qs[2];
#pragma unroll
        for (int c = 0; c < 32 * NC; c += 32) {
          tcx_put_operand(t_q + lanes, q_row, 32 * NC * group + c, pp.chunks, in);
          tcx_put_operand(t_g + lanes, g_row, 32 * NC * group + c, pp.chunks, in);
        }
        tcx_st_wait();
        tcx_before_sync();
        __syncwarp();
        if (lane == 0) tcx_arrive(&bars->in_full);
      }
      // delta = dO . O, half of the columns per thread
      float delta = 0.f;
      if (in) {
        const bf16 *o = static_cast<const bf16*>(p.o) + at, *lo = static_cast<const bf16*>(p.out_lo) + at;
        if (p.dim % 8 == 0 && reinterpret_cast<uintptr_t>(p.o) % 16 == 0) {     // (rows of dO and of the rest are fetched in pieces anyway)
          for (int c = 8 * group; c < p.dim; c += 16) {
            float x[8], y[8], z[8];
            load_vec(g_row + c, x);
            load_vec(o + c, y);
            load_vec(lo + c, z);
#pragma unroll
            for (int e = 0; e < 8; ++e) delta = fmaf(x[e], y[e] + z[e], delta);
          }
        } else {
          for (int c = group; c < p.dim; c += 2) delta = fmaf(widen(g_row[c]), widen(o[c]) + widen(lo[c]), delta);
        }
      }
      red[tid] = delta;
      tcb_sync();
      delta = red[row] + red[128 + row];
      const float2 st = in ? p.stats[((long)b * p.heads + h) * p.lq + i] : make_float2(INFINITY, 0.f);
      if (group == 0 && i < p.lq) p.delta[((long)b * p.heads + h) * p.lq + i] = delta;
      const float base_m = -st.x, inv = st.y, shift = -st.y * delta;
      const float scale = p.scale * kLog2e, tab_before = tab[0], tab_behind = tab[2 * p.reach + 2 * kTcxMargin];
      const uint32_t ts = t_s + kTcbTile * group + lanes, tp = t_dp + kTcbTile * group + lanes;
      float* const slot = slots + (p.dbias_part ? group * (2 * p.reach + 1) : 0);
      float far_before = 0.f, far_behind = 0.f;
      int turn = 0;
      for (int j = group; j < n; j += 2) {
        const uint32_t par = (j >> 1) & 1;
        const int j0 = kTcbTile * j, d0 = j0 - i0 - s.start;
        const bool close = d0 + kTcbTile - 1 > -p.reach && d0 - 127 < p.reach && p.reach > 0;
        if (ok) ok = tcx_wait_warp(&bars->s_full[group], par);
        tcx_after_sync();
        uint32_t raw[64];
        tcx_ld32(ts, raw);
        tcx_ld32(ts + 32, raw + 32);
        tcx_ld_wait(raw);
        tcx_ld_wait(raw + 32);
        tcx_before_sync();
        __syncwarp();
        if (lane == 0) tcx_arrive(&bars->s_read[group]);
        float* x = reinterpret_cast<float*>(raw);
        // (two roundings, as in the forward pass)
        if (close) {
          const float* near = tab + (d0 - row + p.reach + kTcxMargin);
#pragma unroll
          for (int c = 0; c < 64; ++c) x[c] = fmaf(x[c], scale, near[c]) + base_m;
        } else {
          const float far = d0 > 0 ? tab_behind : tab_before;
          if (fabsf(far) < 1e30f) {
            const float sum = far + base_m;
#pragma unroll
            for (int c = 0; c < 64; c += 2) {
              const float2 y = fma2(make_float2(x[c], x[c + 1]), make_float2(scale, scale), make_float2(sum, sum));
              x[c] = y.x;
              x[c + 1] = y.y;
            }
          } else {
#pragma unroll
            for (int c = 0; c < 64; ++c) x[c] = fmaf(x[c], scale, far) + base_m;
          }
        }
        const bool edge = j0 + kTcbTile > keys || (p.causal && d0 + kTcbTile - 1 > 0);
        const int lim = p.causal ? min(keys - j0, row - d0 + 1) : keys - j0;
        if (edge) {
#pragma unroll
          for (int c = 0; c < 64; ++c) x[c] = c < lim ? x[c] : kNoScore;
        }
#pragma unroll
        for (int c = 0; c < 64; ++c) x[c] = exp2_fast(x[c]);
        if (ok) ok = tcx_wait_warp(&bars->dp_full[group], par);
        tcx_after_sync();
#pragma unroll
        for (int k = 0; k < 64; k += 32) {
          uint32_t grad[32], w[16];
          tcx_ld32(tp + k, grad);
          tcx_ld_wait(grad);
#pragma unroll
          for (int c = 0; c < 32; c += 2) {
            const float2 y = fma2(make_float2(as_float(grad[c]), as_float(grad[c + 1])), make_float2(inv, inv), make_float2(shift, shift));
            x[k + c] *= y.x;
            x[k + c + 1] *= y.y;
          }
          if (edge) {
#pragma unroll
            for (int c = 0; c < 32; ++c) x[k + c] = k + c < lim ? x[k + c] : 0.f;
          }
#pragma unroll
          for (int c = 0; c < 32; c += 2) w[c / 2] = pack_bf16(x[k + c], x[k + c + 1]);
          tcx_st16(tp + k / 2, w);                                           // (over products that have been read)
        }
        tcx_st_wait();
        tcx_before_sync();
        __syncwarp();
        if (lane == 0) tcx_arrive(&bars->ds_full[group]);
        if (!p.dbias_part) continue;
        if (close) {
          float* const all = diag + (2 * group + turn) * 4 * kTcbDiag;
          float* const mine = all + (warp & 3) * kTcbDiag;
          float run[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int c = 0; c < 16; ++c) {
#pragma unroll
            for (int k = 0; k < 4; ++k) run[k] += x[16 * k + c];
            if (c == 15) break;
            if (lane == 31) {                                                // the diagonal 16 k + c - 31 is complete
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
          tcb_sync_group(group);
          for (int t = tid & 127; t < 127 + kTcbTile; t += 128) {
            const int off = t - 127, d = d0 + off;                           // column minus row within the tile, relative position
            float sum = 0.f;
#pragma unroll
            for (int wv = 0; wv < 4; ++wv)
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const int e = off + 32 * wv - 16 * k + 31;
                if (e >= 0 && e < 47) sum += all[wv * kTcbDiag + 48 * k + e];
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
      if (ok && n) ok = tcx_wait_warp(&bars->drained, 0);
      tcx_after_sync();
      const bool wide = p.dim % 8 == 0 && reinterpret_cast<uintptr_t>(p.dq) % 16 == 0;
      // (1 / l read again: kept for this it costs the loop 4 %, 8 x 1000 positions, causal, 73 us for 70)
      const bool sees = n && in && p.stats[((long)b * p.heads + h) * p.lq + i].y != 0.f;
#pragma unroll
      for (int k = 0; k < NC; ++k) {
        const int c = 32 * NC * group + 32 * k;
        uint32_t o[32];
        if (n) {
          tcx_ld32(t_dq + c + lanes, o);
          tcx_ld_wait(o);
        }
        float v[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) v[e] = !ok ? bulk_nan() : sees ? as_float(o[e]) * p.scale : 0.f;
        if (i < p.lq) tcx_put_row(static_cast<bf16*>(p.dq) + at, nullptr, v, 32, p.dim, c, wide);
      }
      if (p.dbias_part) {
        tcb_sync();
        red[tid] = far_before;
        red[256 + tid] = far_behind;
        tcb_sync();
        if (warp < 2) {                                                      // warp 0: before, warp 1: behind
          float sum = 0.f;
          for (int e = lane; e < 256; e += 32) sum += red[256 * warp + e];
#pragma unroll
          for (int m = 16; m >= 1; m /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, m);
          if (lane == 0) red[256 * warp] = sum;
        }
        tcb_sync();
        if (tid == 0) {                                                      // (the ends of the slots have taken nothing so far)
          slots[0] = red[0];
          if (p.reach > 0) slots[2 * p.reach] = red[256];
          else slots[0] += red[256];
        }
        tcb_sync();
        float* part = p.dbias_part + (((long)b * p.tiles + tile) * p.heads + h) * p.n_buckets;
        for (int which = tid; which < p.n_buckets; which += 256) {
          float sum = 0.f;
          for (int e = 0; e <= 2 * p.reach; ++e)
            if (p.bucket_of[e] == which) sum += slots[e] + slots[2 * p.reach + 1 + e];
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
// transposed (thread = key), so that weights and score gradients are left operands again: dV += P^T dO, dK += dS^T Q.  P^T goes
// over the scores, dS^T over dP^T; the next scores of a group are computed while it works on dS^T, the next dP^T while it works on
// P^T.  Warp 8 issues scores and dV, warp 11 dP^T and dK, warps 9 and 10 load queries and dO.
struct TcbKvBars {
  uint64_t in_full, s_full[2], dp_full[2], p_full[2], ds_full[2], q_full[4], q_empty[4], g_full[4], g_empty[4], drained;
  uint32_t tmem;
};

template <int NC>
struct AttnTcGradKV {
  static constexpr int kThreads = kTcbThreads, QS = 4;                       // tiles of queries and of dO in turn
  static constexpr uint32_t kKeys = NC * kTcxTile, kRows = NC * kTcbTile * 128;
  static size_t smem(int reach) {
    return 1024 + 2 * (size_t)kKeys + 2 * QS * (size_t)kRows + (2 * 2 * 3 * kTcbTile + 2 * (2 * reach + 2 * kTcxMargin + 1)) * sizeof(float) + sizeof(TcbKvBars) + 16;
  }
  static __device__ __forceinline__ void run(const AttnTcParams& pp, float4* dyn) {
    const AttnParams& p = pp.a;
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const uint32_t base = (tcx_addr(dyn) + 1023u) & ~1023u;
    unsigned char* const smem = reinterpret_cast<unsigned char*>(dyn) + (base - tcx_addr(dyn));
    float* const stat = reinterpret_cast<float*>(smem + 2 * (size_t)kKeys + 2 * QS * (size_t)kRows);      // [group][turn][3][64]: -m, 1 / l, -delta
    float* const tabs = stat + 2 * 2 * 3 * kTcbTile;                            // the bias of its head, for either group
    TcbKvBars* const bars = reinterpret_cast<TcbKvBars*>((reinterpret_cast<uintptr_t>(tabs + 2 * tcx_tab_floats(p.reach)) + 15) & ~(uintptr_t)15);
    const uint32_t k_at = base, v_at = base + kKeys, q_at = base + 2 * kKeys, g_at = q_at + QS * kRows;
    const int heads_all = p.batch * p.kv_heads;                              // under `causal` the first keys have the most queries
    const int tile = (int)blockIdx.x / heads_all, bh = (int)blockIdx.x % heads_all, hk = bh % p.kv_heads, b = bh / p.kv_heads;
    if (tid == 0) {
      tcx_init(&bars->in_full, 256);
      for (int i = 0; i < 2; ++i) {
        tcx_init(&bars->s_full[i], 1);
        tcx_init(&bars->dp_full[i], 1);
        tcx_init(&bars->p_full[i], 4);
        tcx_init(&bars->ds_full[i], 4);
      }
      for (int i = 0; i < QS; ++i) {
        tcx_init(&bars->q_full[i], 32);
        tcx_init(&bars->q_empty[i], 1);
        tcx_init(&bars->g_full[i], 32);
        tcx_init(&bars->g_empty[i], 2);
      }
      tcx_init(&bars->drained, 2);
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    const AttnSeq s = attn_seq(p, b);
    const int j0 = 128 * tile, keys = attn_keys(p, s, s.qlen);
    const int first = j0 < keys ? attn_first_query(p, s, j0) / kTcbTile : 0;
    const int per_head = j0 < keys ? (s.qlen + kTcbTile - 1) / kTcbTile - first : 0, n = per_head > 0 ? per_head * p.group : 0;
    if (warp == 8) {
      __syncwarp();
      tcx_alloc<512>(&bars->tmem);
    }
    tcx_before_sync();
    __syncthreads();
    tcx_after_sync();
    const uint32_t tmem = __shfl_sync(0xffffffffu, bars->tmem, 0);
    stream_order_next();
    const uint32_t t_s = tmem, t_dp = tmem + 128, t_dv = tmem + 256, t_dk = t_dv + 64 * NC;
    bool ok = true;

    if (warp >= 8) {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
      if (warp == 8 || warp == 11) {
        if (n && tcx_elect()) {
          const int steps = (pp.chunks + 1) / 2;
          const uint32_t is = tcx_idesc(kTcbTile, false), io = tcx_idesc(16 * steps, true);
          ok = tcx_wait(&bars->in_full, 0);
          TcxRing<QS> in, out;
          if (warp == 8) {                                                   // the scores, and the gradient of the values
            for (int t = -2; t < n && ok; ++t) {
              if (t >= 0) {
                if (!(ok = tcx_wait(&bars->p_full[t & 1], (t >> 1) & 1))) break;
                if (!(ok = tcx_wait(&bars->g_full[out.at], out.parity))) break;
                tcx_after_sync();
                tcx_seen();
                tcx_combine<kTcbTile, kTcbTile>(t_dv, t_s + kTcbTile * (t & 1), g_at + out.at * kRows, io, t > 0);
                tcx_commit(&bars->g_empty[out.at]);
                out.next();
              }
              if (t + 2 < n) {
                if (!(ok = tcx_wait(&bars->q_full[in.at], in.parity))) break;
                tcx_seen();
                tcx_scores<NC, 128, kTcbTile>(t_s + kTcbTile * (t & 1), k_at, q_at + in.at * kRows, is);
                tcx_commit(&bars->s_full[t & 1]);
                in.next();
              }
            }
          } else {                                                           // dP^T, and the gradient of the keys
            for (int t = -2; t < n && ok; ++t) {
              if (t >= 0) {
                if (!(ok = tcx_wait(&bars->ds_full[t & 1], (t >> 1) & 1))) break;
                if (!(ok = tcx_wait(&bars->q_full[out.at], out.parity))) break;
                tcx_after_sync();
                tcx_seen();
                tcx_combine<kTcbTile, kTcbTile>(t_dk, t_dp + kTcbTile * (t & 1), q_at + out.at * kRows, io, t > 0);
                tcx_commit(&bars->q_empty[out.at]);                          // (the scores of this tile are older)
                out.next();
              }
              if (t + 2 < n) {
                if (!(ok = tcx_wait(&bars->g_full[in.at], in.parity))) break;
                tcx_seen();
                tcx_scores<NC, 128, kTcbTile>(t_dp + kTcbTile * (t & 1), v_at, g_at + in.at * kRows, is);
                tcx_commit(&bars->dp_full[t & 1]);
                tcx_commit(&bars->g_empty[in.at]);
                in.next();
              }
            }
          }
          tcx_commit(&bars->drained);
          tcx_wait(&bars->drained, 0);
        }
        __syncwarp();
      } else if (warp == 9 || warp == 10) {
        const bool is_q = warp == 9;
        uint64_t *full = is_q ? bars->q_full : bars->g_full, *empty = is_q ? bars->q_empty : bars->g_empty;
        const uint32_t to = is_q ? q_at : g_at;
        const long by_head = is_q ? p.qs[2] : pp.gs[2], stride = is_q ? p.qs[1] : pp.gs[1];
        const bf16* src = static_cast<const bf16*>(is_q ? p.q : p.dout) + b * (is_q ? p.qs[0] : pp.gs[0]) + hk * p.group * by_head;
        int g = 0, it = first;
        for (int t = 0; t < n && ok; ++t) {
          if (t >= QS) ok = tcx_wait_warp(&empty[t % QS], (t / QS - 1) & 1);
          if (!ok) break;
          tcx_load_rows<NC, 32, kTcbTile>(to + (t % QS) * kRows, src + g * by_head, stride, kTcbTile * it, s.qlen, pp.chunks, lane);
          tcx_arrive_copies(&full[t % QS]);
          if (++it == first + per_head) { it = first; ++g; }
        }
        tcx_copies_done();
      }
    } else {
      asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
      const int group = warp >> 2, row = 32 * (warp & 3) + lane, j = j0 + row;
      if (n) {
        tcx_load_rows<NC, 256>(k_at, static_cast<const bf16*>(p.k) + b * p.ks[0] + hk * p.ks[2], p.ks[1], j0, keys, pp.chunks, tid);
        tcx_load_rows<NC, 256>(v_at, static_cast<const bf16*>(p.v) + b * p.vs[0] + hk * p.vs[2], p.vs[1], j0, keys, pp.chunks, tid);
        tcx_loaded();
        tcx_arrive(&bars->in_full);
      }
      const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
      const uint32_t ts = t_s + kTcbTile * group + lanes, tp = t_dp + kTcbTile * group + lanes;
      const float scale = p.scale * kLog2e;
      float* const tab = tabs + group * tcx_tab_floats(p.reach);
      int head = -1;
      float2 ahead = make_float2(INFINITY, 0.f);
      float ahead_delta = 0.f;
      auto fetch = [&](int t) {
        if ((tid & 127) >= kTcbTile || t >= n) return;
        const int g = t / per_head, i = kTcbTile * (first + t - g * per_head) + (tid & 63);
        const long at = ((long)b * p.heads + hk * p.group + g) * p.lq + i;
        ahead = i < s.qlen ? p.stats[at] : make_float2(INFINITY, 0.f);
        ahead_delta = i < s.qlen ? p.delta[at] : 0.f;
      };
      fetch(group);
      for (int t = group; t < n; t += 2) {
        const uint32_t par = (t >> 1) & 1;
        const int g = t / per_head, it = first + t - g * per_head;
        if (g != head) {                                                     // the next head: its bias
          head = g;
          tcb_sync_group(group);
          tcx_bias_table(p, hk * p.group + g, tab, tid & 127, 128, false);
          tcb_sync_group(group);
        }
        const int i0 = kTcbTile * it, d0 = j0 - i0 - s.start;
        // -m, 1 / l, -delta of the tile's queries, fetched a tile ahead, by one thread each
        float* const sm = stat + (2 * group + (int)par) * 3 * kTcbTile;
        if ((tid & 127) < kTcbTile) {
          sm[tid & 63] = -ahead.x;
          sm[kTcbTile + (tid & 63)] = ahead.y;
          sm[2 * kTcbTile + (tid & 63)] = -ahead_delta;
        }
        fetch(t + 2);
        tcb_sync_group(group);
        if (ok) ok = tcx_wait_warp(&bars->s_full[group], par);
        tcx_after_sync();
        uint32_t raw[64];
        tcx_ld32(ts, raw);
        tcx_ld32(ts + 32, raw + 32);
        tcx_ld_wait(raw);
        tcx_ld_wait(raw + 32);
        float* x = reinterpret_cast<float*>(raw);
        if (d0 + 127 > -p.reach && d0 - (kTcbTile - 1) < p.reach && p.reach > 0) {
          const float* near = tab + (d0 + row + p.reach + kTcxMargin);
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
        const int low = j >= keys ? 128 : p.causal ? d0 + row : 0;           // first query of the tile that sees the key
        if (edge) {
#pragma unroll
          for (int c = 0; c < 64; ++c) x[c] = c >= low ? x[c] : kNoScore;
        }
#pragma unroll
        for (int k = 0; k < 64; k += 32) {
          uint32_t w[16];
#pragma unroll
          for (int c = 0; c < 32; c += 4) {
            const float4 f = *reinterpret_cast<const float4*>(sm + kTcbTile + k + c);
            float* y = x + k + c;
            y[0] = exp2_fast(y[0]) * f.x;
            y[1] = exp2_fast(y[1]) * f.y;
            y[2] = exp2_fast(y[2]) * f.z;
            y[3] = exp2_fast(y[3]) * f.w;
            w[c / 2] = pack_bf16(y[0], y[1]);
            w[c / 2 + 1] = pack_bf16(y[2], y[3]);
          }
          tcx_st16(ts + k / 2, w);
        }
        tcx_st_wait();
        tcx_before_sync();
        __syncwarp();
        if (lane == 0) tcx_arrive(&bars->p_full[group]);
        if (ok) ok = tcx_wait_warp(&bars->dp_full[group], par);
        tcx_after_sync();
#pragma unroll
        for (int k = 0; k < 64; k += 32) {
          uint32_t grad[32], w[16];
          tcx_ld32(tp + k, grad);
          tcx_ld_wait(grad);
#pragma unroll
          for (int c = 0; c < 32; c += 4) {
            const float4 f = *reinterpret_cast<const float4*>(sm + 2 * kTcbTile + k + c);
            float* y = x + k + c;
            y[0] *= as_float(grad[c]) + f.x;
            y[1] *= as_float(grad[c + 1]) + f.y;
            y[2] *= as_float(grad[c + 2]) + f.z;
            y[3] *= as_float(grad[c + 3]) + f.w;
          }
          if (edge) {
#pragma unroll
            for (int c = 0; c < 32; ++c) x[k + c] = k + c >= low ? x[k + c] : 0.f;
          }
#pragma unroll
          for (int c = 0; c < 32; c += 2) w[c / 2] = pack_bf16(x[k + c], x[k + c + 1]);
          tcx_st16(tp + k / 2, w);                                           // (over products that have been read)
        }
        tcx_st_wait();
        tcx_before_sync();
        __syncwarp();
        if (lane == 0) tcx_arrive(&bars->ds_full[group]);
      }
      // ---- rows of dV (warps 0 - 3) and dK (warps 4 - 7)
      if (ok && n) ok = tcx_wait_warp(&bars->drained, 0);
      tcx_after_sync();
      bf16* out = static_cast<bf16*>(group ? p.dk : p.dv) + (((long)b * p.lk + j) * p.kv_heads + hk) * p.dim;
      const float f = group ? p.scale : 1.f;
      const bool wide = p.dim % 8 == 0 && reinterpret_cast<uintptr_t>(group ? p.dk : p.dv) % 16 == 0;
#pragma unroll
      for (int c = 0; c < 64 * NC; c += 32) {
        uint32_t o[32];
        if (n) {
          tcx_ld32((group ? t_dk : t_dv) + c + lanes, o);
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
