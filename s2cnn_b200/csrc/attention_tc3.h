// Attention, float32, on the tensor cores: every operand in three bfloat16 parts, v = v0 + v1 + v2 with v0 = v rounded, v1 = v - v0
// rounded, v2 the rest rounded (8 bits each, 24 in all), and a product as the six of its nine partial products that are not
// below 2^-27 of the whole.  That is the rate of three TF32 products, with operand tiles that are K- and MN-major alike.
//
// The tensor core's accumulation truncates, a bias of up to one unit in the last place per instruction that adds up along a chain.
// So every chain is short: the small partial products come first, while the accumulator is small, a tile's product starts a
// new accumulator, and the threads add it to sums in their registers, rounded properly.
//
// Operands are split once, by AttnPack, into packed rows; that kernel also brings bfloat16 rows that 16-byte copies cannot
// fetch into aligned ones.
#pragma once

#include "attention_tc.h"

#ifndef S2C_EMUL

namespace s2c {

// ---- rows of a tensor of any strides, packed: [part][batch][head][position][8 chunks], zeros behind the values -----------------
struct AttnPackParams {
  const void* src[4];
  bf16* dst[4];
  long stride[4][3];       // batch entry, position, head
  long part[4];            // elements from one part to the next
  int len[4], heads[4], tensors;
  int batch, dim, chunks;
};
template <class T>
struct AttnPack {
  using Params = AttnPackParams;
  static constexpr int kThreads = 256, kBlocks = 4;
  static __device__ __forceinline__ void run(const Ctx& ctx, const Params& p, unsigned char*) {
    for (int t = 0; t < p.tensors; ++t) {
      const long pieces = (long)p.batch * p.len[t] * p.heads[t] * p.chunks;
      for (long e = (long)ctx.bid * kThreads + ctx.tid; e < pieces; e += (long)ctx.nblk * kThreads) {
        // in the order of memory of the usual [batch][position][head] input
        const int c = (int)(e % p.chunks);
        long r = e / p.chunks;
        const int h = (int)(r % p.heads[t]);
        r /= p.heads[t];
        const int i = (int)(r % p.len[t]), b = (int)(r / p.len[t]);
        const T* from = static_cast<const T*>(p.src[t]) + b * p.stride[t][0] + i * p.stride[t][1] + h * p.stride[t][2] + 8 * c;
        bf16* to = p.dst[t] + (((long)b * p.heads[t] + h) * p.len[t] + i) * 8 * p.chunks + 8 * c;
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = 8 * c + k < p.dim ? widen(from[k]) : 0.f;
#pragma unroll
        for (int part = 0; part < (sizeof(T) == 4 ? 3 : 1); ++part) {
          store_vec(to + part * p.part[t], v);
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            bf16 w;
            narrow(&w, v[k]);
            v[k] -= widen(w);
          }
        }
      }
    }
  }
};

// the six partial products, smallest first
__device__ __forceinline__ int tc3_left(int k) { return k == 0 ? 0 : k == 1 ? 2 : k == 2 ? 1 : k == 3 ? 0 : k == 4 ? 1 : 0; }
__device__ __forceinline__ int tc3_right(int k) { return k == 0 ? 2 : k == 1 ? 0 : k == 2 ? 1 : k == 3 ? 1 : k == 4 ? 0 : 0; }
// D = A B^T over 16 `steps` columns: tiles of A_ROWS and B_ROWS rows, NC blocks of 64 columns, three parts of each
template <int NC, int A_ROWS, int B_ROWS>
__device__ __forceinline__ void tc3_scores(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, int steps) {
#pragma unroll
  for (int k = 0; k < 6; ++k) {
    const uint64_t da = tcx_desc(a + tc3_left(k) * NC * A_ROWS * 128, 0), db = tcx_desc(b + tc3_right(k) * NC * B_ROWS * 128, 0);
#pragma unroll
    for (int s = 0; s < 4 * NC; ++s) {
      if (s >= steps) break;
      tcx_mma(d, da + (uint64_t)(((s / 4) * (A_ROWS * 128) + (s % 4) * 32) >> 4), db + (uint64_t)(((s / 4) * (B_ROWS * 128) + (s % 4) * 32) >> 4), idesc,
              k > 0 || s > 0);
    }
  }
}
// D = A B: A in tensor memory, 128 x K, its parts K / 2 columns apart; B: K rows (from `b` on) of a tile of B_ROWS rows, MN-major
template <int NC, int K, int B_ROWS>
__device__ __forceinline__ void tc3_combine(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc) {
#pragma unroll
  for (int k = 0; k < 6; ++k) {
    const uint64_t db = tcx_desc(b + tc3_right(k) * NC * B_ROWS * 128, B_ROWS * 128);
#pragma unroll
    for (int s = 0; s < K / 16; ++s) tcx_mma_t(d, a + tc3_left(k) * (K / 2) + 8 * s, db + (uint64_t)(s * 2048 >> 4), idesc, k > 0 || s > 0);
  }
}
template <int NC, int N, int ROWS>
__device__ __forceinline__ void tc3_load(uint32_t dst, const bf16* src, long part, long row_stride, int r0, int end, int chunks, int t) {
#pragma unroll
  for (int k = 0; k < 3; ++k) tcx_load_rows<NC, N, ROWS>(dst + k * NC * ROWS * 128, src + k * part, row_stride, r0, end, chunks, t);
}
// N values (32 or 16) of a row in three parts into tensor memory, parts `apart` columns from each other
template <int N>
__device__ __forceinline__ void tc3_put(uint32_t to, int apart, const float* v) {
  float r[N];
#pragma unroll
  for (int c = 0; c < N; ++c) r[c] = v[c];
#pragma unroll
  for (int part = 0; part < 3; ++part) {
    uint32_t w[N / 2];
#pragma unroll
    for (int c = 0; c < N; c += 2) {
      w[c / 2] = pack_bf16(r[c], r[c + 1]);
      r[c] -= as_float(w[c / 2] << 16);
      r[c + 1] -= as_float(w[c / 2] & 0xffff0000u);
    }
    static_assert(N == 32, "16 columns at a time");
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(to + part * apart),
                 "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]), "r"(w[8]), "r"(w[9]), "r"(w[10]), "r"(w[11]),
                 "r"(w[12]), "r"(w[13]), "r"(w[14]), "r"(w[15])
                 : "memory");
  }
}
// `n` values of a float32 row from column c0 on
__device__ __forceinline__ void tc3_store_row(float* out, const float* v, int n, int dim, int c0, bool wide) {
  if (wide) {
#pragma unroll
    for (int c = 0; c < n; c += 4)
      if (c0 + c < dim) *reinterpret_cast<float4*>(out + c0 + c) = make_float4(v[c], v[c + 1], v[c + 2], v[c + 3]);
  } else {
#pragma unroll
    for (int c = 0; c < n; ++c)
      if (c0 + c < dim) out[c0 + c] = v[c];
  }
}

constexpr int kTc3Threads = 12 * 32;
// barrier of the 256 threads at the scores
__device__ __forceinline__ void tc3_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

// ---- forward -----------------------------------------------------------------------------------------------------------------
// A block has 128 queries of one head; key tiles have KT keys.  Warps 0 - 3 take the first half of a tile's keys, warps 4 - 7 the
// other half, as if the keys were split: each half has its own maximum, sum, weights and output, and they meet at the end.
// The next scores are computed while the threads are at the exponentials of the last ones.
struct Tc3FwdBars {
  uint64_t q_full, s_full, s_read, p_full[2], pv_done[2], k_full[2], k_empty[2], v_full, v_empty, drained;
  uint32_t tmem;
};
template <int NC>
struct AttnTc3Forward {
  static constexpr int kThreads = kTc3Threads, KT = NC == 1 ? 128 : 64, HALF = KT / 2, KS = NC == 1 ? 2 : 1;      // KS: key tiles in turn
  static constexpr uint32_t kQ = 3 * NC * 128 * 128, kK = 3 * NC * KT * 128;
  static size_t smem(int reach) {
    return 1024 + kQ + (KS + 1) * (size_t)kK + (2 * reach + 2 * kTcxMargin + 1 + 256) * sizeof(float) + sizeof(Tc3FwdBars) + 16;
  }
  static __device__ __forceinline__ void run(const AttnTcParams& pp, float4* dyn) {
    const AttnParams& p = pp.a;
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const uint32_t base = (tcx_addr(dyn) + 1023u) & ~1023u;
    unsigned char* const smem = reinterpret_cast<unsigned char*>(dyn) + (base - tcx_addr(dyn));
    float* const red = reinterpret_cast<float*>(smem + kQ + (KS + 1) * kK);       // [256]
    float* const tab = red + 256;
    Tc3FwdBars* const bars = reinterpret_cast<Tc3FwdBars*>((reinterpret_cast<uintptr_t>(tab + tcx_tab_floats(p.reach)) + 15) & ~(uintptr_t)15);
    const uint32_t q_at = base, k_at = base + kQ, v_at = k_at + KS * kK;
    const int heads_all = p.batch * p.heads;                              // the longest rows first
    const int tile = p.tiles - 1 - (int)blockIdx.x / heads_all, bh = (int)blockIdx.x % heads_all, h = bh % p.heads, b = bh / p.heads, hk = h / p.group;
    if (tid == 0) {
      tcx_init(&bars->q_full, 256);
      tcx_init(&bars->s_full, 1);
      tcx_init(&bars->s_read, 8);
      for (int i = 0; i < 2; ++i) {
        tcx_init(&bars->p_full[i], 4);
        tcx_init(&bars->pv_done[i], 1);
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
    const int keys = i0 < s.qlen ? attn_keys(p, s, min(i0 + 128, s.qlen)) : 0, n = (keys + KT - 1) / KT;
    if (warp == 8) {
      __syncwarp();
      tcx_alloc<512>(&bars->tmem);
    }
    tcx_bias_table(p, h, tab, tid, kTc3Threads, true);
    tcx_before_sync();
    __syncthreads();
    tcx_after_sync();
    const uint32_t tmem = __shfl_sync(0xffffffffu, bars->tmem, 0);
    stream_order_next();
    // scores (KT columns), three parts of the weights of each half, output of each half
    constexpr uint32_t kW = 3 * HALF / 2, kO = 64 * NC;
    static_assert(KT + 2 * kW + 2 * kO <= 512, "tensor memory");
    const uint32_t t_s = tmem, t_w = tmem + KT, t_o = t_w + 2 * kW;
    bool ok = true;

    if (warp >= 8) {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
      if (warp == 8 && n) {
        const int steps = (pp.chunks + 1) / 2;
        const uint32_t is = tcx_idesc(KT, false), io = tcx_idesc(16 * steps, true);
        auto scores = [&](int j) {
          if (!(ok = tcx_wait_warp(&bars->k_full[j % KS], (j / KS) & 1))) return;
          if (tcx_elect()) {
            tc3_scores<NC, 128, KT>(t_s, q_at, k_at + (j % KS) * kK, is, steps);
            tcx_commit(&bars->s_full);
            tcx_commit(&bars->k_empty[j % KS]);
          }
          __syncwarp();
        };
        ok = tcx_wait_warp(&bars->q_full, 0);
        if (ok) scores(0);
        for (int j = 0; j < n && ok; ++j) {
          if (j + 1 < n) {
            if (!(ok = tcx_wait_warp(&bars->s_read, j & 1))) break;
            tcx_after_sync();
            scores(j + 1);
          }
          if (!ok || !(ok = tcx_wait_warp(&bars->v_full, j & 1))) break;
          for (int w = 0; w < 2 && ok; ++w) {
            if (!(ok = tcx_wait_warp(&bars->p_full[w], j & 1))) break;
            tcx_after_sync();
            if (tcx_elect()) {
              tc3_combine<NC, HALF, KT>(t_o + w * kO, t_w + w * kW, v_at + w * HALF * 128, io);
              tcx_commit(&bars->pv_done[w]);
              if (w == 1) tcx_commit(&bars->v_empty);
            }
            __syncwarp();
          }
        }
        if (tcx_elect()) tcx_commit(&bars->drained);
        __syncwarp();
        ok = tcx_wait_warp(&bars->drained, 0) && ok;
      } else if (warp == 9) {
        const bf16* src = static_cast<const bf16*>(p.k) + b * p.ks[0] + hk * p.ks[2];
        for (int j = 0; j < n && ok; ++j) {
          if (j >= KS) ok = tcx_wait_warp(&bars->k_empty[j % KS], (j / KS - 1) & 1);
          if (!ok) break;
          tc3_load<NC, 32, KT>(k_at + (j % KS) * kK, src, pp.k_split, p.ks[1], KT * j, keys, pp.chunks, lane);
          tcx_loaded();
          __syncwarp();
          if (lane == 0) tcx_arrive(&bars->k_full[j % KS]);
        }
      } else if (warp == 10) {
        const bf16* src = static_cast<const bf16*>(p.v) + b * p.vs[0] + hk * p.vs[2];
        for (int j = 0; j < n && ok; ++j) {
          if (j >= 1) ok = tcx_wait_warp(&bars->v_empty, (j - 1) & 1);
          if (!ok) break;
          tc3_load<NC, 32, KT>(v_at, src, pp.v_split, p.vs[1], KT * j, keys, pp.chunks, lane);
          tcx_loaded();
          __syncwarp();
          if (lane == 0) tcx_arrive(&bars->v_full);
        }
      }
    } else {
      asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
      const int half = warp >> 2, row = 32 * (warp & 3) + lane, i = i0 + row;
      if (n) {
        tc3_load<NC, 256, 128>(q_at, static_cast<const bf16*>(p.q) + b * p.qs[0] + h * p.qs[2], pp.q_split, p.qs[1], i0, s.qlen, pp.chunks, tid);
        tcx_loaded();
        tcx_arrive(&bars->q_full);
      }
      const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
      const float scale = p.scale * kLog2e, tab_before = tab[0], tab_behind = tab[2 * p.reach + 2 * kTcxMargin];
      float acc[kO], m = kNoScore, l = 0.f, f = 1.f;
#pragma unroll
      for (int c = 0; c < (int)kO; ++c) acc[c] = 0.f;
      // adds the output of the last tile, with the weights' unit of that time
      auto drain = [&](int j) {
        if (ok) ok = tcx_wait_warp(&bars->pv_done[half], j & 1);
        tcx_after_sync();
#pragma unroll
        for (int c = 0; c < (int)kO; c += 32) {
          uint32_t o[32];
          tcx_ld32(t_o + half * kO + c + lanes, o);
          tcx_ld_wait(o);
#pragma unroll
          for (int e = 0; e < 32; ++e) acc[c + e] += as_float(o[e]);
        }
      };
      for (int j = 0; j < n; ++j) {
        const int j0 = KT * j, d0 = j0 - i0 - s.start;
        if (ok) ok = tcx_wait_warp(&bars->s_full, j & 1);
        tcx_after_sync();
        uint32_t raw[HALF];
#pragma unroll
        for (int c = 0; c < HALF; c += 32) tcx_ld32(t_s + HALF * half + c + lanes, raw + c);
#pragma unroll
        for (int c = 0; c < HALF; c += 32) tcx_ld_wait(raw + c);
        tcx_before_sync();
        __syncwarp();
        if (lane == 0) tcx_arrive(&bars->s_read);
        float* x = reinterpret_cast<float*>(raw);
        if (d0 + KT - 1 > -p.reach && d0 - 127 < p.reach && p.reach > 0) {
          const float* near = tab + (d0 + HALF * half - row + p.reach + kTcxMargin);
#pragma unroll
          for (int c = 0; c < HALF; ++c) x[c] = fmaf(x[c], scale, near[c]);
        } else {
          const float far = d0 > 0 ? tab_behind : tab_before;
#pragma unroll
          for (int c = 0; c < HALF; ++c) x[c] = fmaf(x[c], scale, far);
        }
        if (j0 + KT > keys || (p.causal && d0 + KT - 1 > 0)) {
          const int lim = (p.causal ? min(keys - j0, row - d0 + 1) : keys - j0) - HALF * half;
#pragma unroll
          for (int c = 0; c < HALF; ++c) x[c] = c < lim ? x[c] : kNoScore;
        }
        float now = x[0];
#pragma unroll
        for (int c = 1; c < HALF; ++c) now = fmaxf(now, x[c]);
        const bool grown = __any_sync(0xffffffffu, now > m + 8.f) != 0;  // (as in the bfloat16 kernel: else the unit stays)
        if (grown) {
          const float fresh = now > m + 8.f ? now : m;
          f = fresh == m ? 1.f : exp2_fast(m - fresh);
          m = fresh;
          l *= f;
        }
        const float off = m == kNoScore ? 0.f : -m;
        float sum[2] = {0.f, 0.f};
#pragma unroll
        for (int c = 0; c < HALF; ++c) {
          x[c] = exp2_fast(x[c] + off);
          sum[c & 1] += x[c];
        }
        l += sum[0] + sum[1];
        if (j > 0) {
          drain(j - 1);
          if (grown) {
#pragma unroll
            for (int c = 0; c < (int)kO; ++c) acc[c] *= f;
          }
        }
#pragma unroll
        for (int c = 0; c < HALF; c += 32) tc3_put<32>(t_w + half * kW + c / 2 + lanes, HALF / 2, x + c);
        tcx_st_wait();
        tcx_before_sync();
        __syncwarp();
        if (lane == 0) tcx_arrive(&bars->p_full[half]);
      }
      if (n) drain(n - 1);
      if (ok && n) ok = tcx_wait_warp(&bars->drained, 0);                // the operand tiles may be overwritten
      // ---- the halves meet: 32 columns at a time through shared memory
      if (i >= s.qlen) l = 0.f;
      red[tid] = m;
      tc3_sync();
      const float top = fmaxf(red[row], red[128 + row]), unit = top == kNoScore ? 0.f : top;
      const float mine = exp2_fast(m - unit);
      tc3_sync();
      red[tid] = l * mine;
      tc3_sync();
      const float2 st = attn_stats(top, red[row] + red[128 + row]);
      const float mul = st.y == 0.f ? 0.f : mine * st.y;
      float* const meet = reinterpret_cast<float*>(smem);                // [kO / 2][128] of either half
      // a half writes out its own columns: kO / 2 of them, and gives the others away
#pragma unroll
      for (int c = 0; c < (int)kO; ++c) acc[c] = st.y == 0.f ? 0.f : acc[c] * mul;
#pragma unroll
      for (int c = 0; c < (int)kO / 2; ++c) meet[(half * (kO / 2) + c) * 128 + row] = half ? acc[c] : acc[kO / 2 + c];
      tc3_sync();
      float v[kO / 2];
#pragma unroll
      for (int c = 0; c < (int)kO / 2; ++c) {
        v[c] = (half ? acc[kO / 2 + c] : acc[c]) + meet[((1 - half) * (kO / 2) + c) * 128 + row];
        if (!ok) v[c] = bulk_nan();
      }
      const bool wide = p.dim % 4 == 0 && reinterpret_cast<uintptr_t>(p.out) % 16 == 0;
      if (i < p.lq) {
        tc3_store_row(static_cast<float*>(p.out) + (((long)b * p.lq + i) * p.heads + h) * p.dim, v, kO / 2, p.dim, half * (kO / 2), wide);
        if (p.stats && half == 0) p.stats[((long)b * p.heads + h) * p.lq + i] = st;
      }
    }
    tcx_before_sync();
    __syncthreads();
    if (warp == 8) tcx_free<512>(tmem);
  }
};

}  // namespace s2c
#endif  // S2C_EMUL
