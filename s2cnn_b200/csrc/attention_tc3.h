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
//
// Bound by the tensor pipe.  2 x 4096 positions, 16 heads of 64 / 128, in us and TFLOP/s of bfloat16 products: forward 692 (1191) /
// 1661 (993), queries 1149 (1076) / 2799 (884), keys and values 1745 (945) / 3121 (1057), copies 57 / 106.
#pragma once

#include "attention_tc.h"

#ifndef S2C_EMUL

namespace s2c {

// ---- rows of a tensor of any strides, packed: [part][batch][head][position][8 chunks], zeros behind the values -----------------
// Only rows that some query sees, and queries that are filled: nothing reads the places of the others.
struct AttnPackParams {
  AttnParams a;            // lengths and positions
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
    const int t = ctx.bid % p.tensors;                                     // a block has one of the tensors
    const long per_entry = (long)p.len[t] * p.heads[t] * p.chunks, pieces = p.batch * per_entry, step = (long)(ctx.nblk / p.tensors) * kThreads;
    for (long e = (long)(ctx.bid / p.tensors) * kThreads + ctx.tid; e < pieces; e += step) {
      // in the order of memory of the usual [batch][position][head] input
      const int c = (int)(e % p.chunks);
      long r = e / p.chunks;
      const int h = (int)(r % p.heads[t]);
      r /= p.heads[t];
      const int i = (int)(r % p.len[t]), b = (int)(r / p.len[t]);
      const AttnSeq s = attn_seq(p.a, b);
      if (i >= (t == 0 || t == 3 ? s.qlen : attn_keys(p.a, s, s.qlen))) {   // nor is what follows of this batch entry: its last turn
        e += ((b + 1) * per_entry - 1 - e) / step * step;
        continue;
      }
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
};

// the six partial products, smallest first
__device__ __forceinline__ int tc3_left(int k) { return k == 0 ? 0 : k == 1 ? 2 : k == 2 ? 1 : k == 3 ? 0 : k == 4 ? 1 : 0; }
__device__ __forceinline__ int tc3_right(int k) { return k == 0 ? 2 : k == 1 ? 0 : k == 2 ? 1 : k == 3 ? 1 : k == 4 ? 0 : 0; }
// D = A B^T: tiles of A_ROWS and B_ROWS rows, NC blocks of 64 columns, three parts of each
template <int NC, int A_ROWS, int B_ROWS>
__device__ __forceinline__ void tc3_scores(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc) {
#pragma unroll
  for (int k = 0; k < 6; ++k)
    tcx_scores<NC, A_ROWS, B_ROWS>(d, a + tc3_left(k) * NC * A_ROWS * 128, b + tc3_right(k) * NC * B_ROWS * 128, idesc, k > 0);
}
// the same with the parts of A side by side in tensor memory
template <int NC, int B_ROWS>
__device__ __forceinline__ void tc3_scores_t(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc) {
#pragma unroll
  for (int k = 0; k < 6; ++k) tcx_scores_t<NC, B_ROWS>(d, a + tc3_left(k) * 32 * NC, b + tc3_right(k) * NC * B_ROWS * 128, idesc, k > 0);
}
// D = A B: A in tensor memory, 128 x K, its parts K / 2 columns apart; B: K rows (from `b` on) of a tile of B_ROWS rows, MN-major
template <int NC, int K, int B_ROWS>
__device__ __forceinline__ void tc3_combine(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc) {
#pragma unroll
  for (int k = 0; k < 6; ++k) tcx_combine<K, B_ROWS>(d, a + tc3_left(k) * (K / 2), b + tc3_right(k) * NC * B_ROWS * 128, idesc, k > 0);
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
        tcx_init(&bars->k_full[i], 32);
        tcx_init(&bars->k_empty[i], 1);
      }
      tcx_init(&bars->v_full, 32);
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
      if (warp == 8) {
        if (n && tcx_elect()) {
          const int steps = (pp.chunks + 1) / 2;
          const uint32_t is = tcx_idesc(KT, false), io = tcx_idesc(16 * steps, true);
          auto scores = [&](int j) {
            if (!(ok = tcx_wait(&bars->k_full[j % KS], (j / KS) & 1))) return;
            tcx_seen();
            tc3_scores<NC, 128, KT>(t_s, q_at, k_at + (j % KS) * kK, is);
            tcx_commit(&bars->s_full);
            tcx_commit(&bars->k_empty[j % KS]);
          };
          ok = tcx_wait(&bars->q_full, 0);
          if (ok) scores(0);
          for (int j = 0; j < n && ok; ++j) {
            if (j + 1 < n) {
              if (!(ok = tcx_wait(&bars->s_read, j & 1))) break;
              tcx_after_sync();
              scores(j + 1);
            }
            if (!ok || !(ok = tcx_wait(&bars->v_full, j & 1))) break;
            tcx_seen();
            for (int w = 0; w < 2 && ok; ++w) {
              if (!(ok = tcx_wait(&bars->p_full[w], j & 1))) break;
              tcx_after_sync();
              tc3_combine<NC, HALF, KT>(t_o + w * kO, t_w + w * kW, v_at + w * HALF * 128, io);
              tcx_commit(&bars->pv_done[w]);
              if (w == 1) tcx_commit(&bars->v_empty);
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
          tc3_load<NC, 32, KT>(k_at + (j % KS) * kK, src, pp.k_split, p.ks[1], KT * j, keys, pp.chunks, lane);
          tcx_arrive_copies(&bars->k_full[j % KS]);
        }
        tcx_copies_done();
      } else if (warp == 10) {
        const bf16* src = static_cast<const bf16*>(p.v) + b * p.vs[0] + hk * p.vs[2];
        for (int j = 0; j < n && ok; ++j) {
          if (j >= 1) ok = tcx_wait_warp(&bars->v_empty, (j - 1) & 1);
          if (!ok) break;
          tc3_load<NC, 32, KT>(v_at, src, pp.v_split, p.vs[1], KT * j, keys, pp.chunks, lane);
          tcx_arrive_copies(&bars->v_full);
        }
        tcx_copies_done();
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

// ---- gradient of the queries -----------------------------------------------------------------------------------------------------
// As AttnTcGradQ, with key tiles of 64: warps 0 - 3 take the first 32 keys of a tile, warps 4 - 7 the others; the gradient of a
// tile's keys is added to registers, half of its columns per group.
// Heads of more than 64 values (NC = 2): the parts of queries and dO do not fit in shared memory beside those of keys and values.
// The queries lie in tensor memory, dS goes over the scores, and there is one tile each of keys and values: a tile is then
// finished before the next one's scores begin.
constexpr int kTc3Diag = 2 * 48;
struct Tc3QBars {
  uint64_t in_full, s_full[2], dp_full, ds_full, dq_done, k_full[3], k_empty[3], v_full, v_empty, drained;
  uint32_t tmem;
};
template <int NC>
struct AttnTc3GradQ {
  static constexpr int kThreads = kTc3Threads, KT = 64, HALF = 32, KS = NC == 1 ? 3 : 1;
  static constexpr uint32_t kQ = 3 * NC * 128 * 128, kK = 3 * NC * KT * 128, kTiles = (NC == 1 ? 2 : 1) * kQ + (KS + 1) * kK;
  static size_t smem(int reach, bool bias_grad) {
    return 1024 + (size_t)kTiles + (2 * reach + 2 * kTcxMargin + 1 + 512 + (bias_grad ? 2 * 8 * kTc3Diag + 2 * reach + 1 : 0)) * sizeof(float) +
           sizeof(Tc3QBars) + 16;
  }
  static __device__ __forceinline__ void run(const AttnTcParams& pp, float4* dyn) {
    const AttnParams& p = pp.a;
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const uint32_t base = (tcx_addr(dyn) + 1023u) & ~1023u;
    unsigned char* const smem = reinterpret_cast<unsigned char*>(dyn) + (base - tcx_addr(dyn));
    float* const red = reinterpret_cast<float*>(smem + kTiles);   // [512]
    float* const tab = red + 512;
    float* const diag = tab + tcx_tab_floats(p.reach);                     // [2][8][kTc3Diag], then a slot per relative position
    float* const slot = diag + (p.dbias_part ? 2 * 8 * kTc3Diag : 0);
    Tc3QBars* const bars = reinterpret_cast<Tc3QBars*>((reinterpret_cast<uintptr_t>(slot + (p.dbias_part ? 2 * p.reach + 1 : 0)) + 15) & ~(uintptr_t)15);
    const uint32_t g_at = base, k_at = base + kQ, v_at = k_at + KS * kK, q_at = v_at + kK;           // (q: NC = 1)
    const int heads_all = p.batch * p.heads;
    const int tile = p.tiles - 1 - (int)blockIdx.x / heads_all, bh = (int)blockIdx.x % heads_all, h = bh % p.heads, b = bh / p.heads, hk = h / p.group;
    if (tid == 0) {
      tcx_init(&bars->in_full, 256);
      for (int i = 0; i < 2; ++i) tcx_init(&bars->s_full[i], 1);
      tcx_init(&bars->dp_full, 1);
      tcx_init(&bars->ds_full, 8);
      tcx_init(&bars->dq_done, 1);
      for (int i = 0; i < KS; ++i) {
        tcx_init(&bars->k_full[i], 32);
        tcx_init(&bars->k_empty[i], 1);
      }
      tcx_init(&bars->v_full, 32);
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
    if (p.dbias_part)
      for (int e = tid; e <= 2 * p.reach; e += kTc3Threads) slot[e] = 0.f;
    tcx_before_sync();
    __syncthreads();
    tcx_after_sync();
    const uint32_t tmem = __shfl_sync(0xffffffffu, bars->tmem, 0);
    stream_order_next();
    // NC = 1: two tiles of scores, products, three parts of dS, the gradient; NC = 2: three parts of the queries, scores and dS in
    // one place, products, the gradient
    const uint32_t t_q = tmem, t_s = NC == 1 ? tmem : tmem + 192, t_dp = NC == 1 ? tmem + 128 : tmem + 288, t_ds = NC == 1 ? tmem + 192 : t_s,
                   t_dq = NC == 1 ? tmem + 288 : tmem + 352;
    bool ok = true;

    if (warp >= 8) {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
      if (warp == 8) {
        if (n && tcx_elect()) {
          const int steps = (pp.chunks + 1) / 2;
          const uint32_t is = tcx_idesc(KT, false), io = tcx_idesc(16 * steps, true);
          auto scores = [&](int j) {
            if (!(ok = tcx_wait(&bars->k_full[j % KS], (j / KS) & 1))) return;
            tcx_seen();
            if constexpr (NC == 1) tc3_scores<1, 128, KT>(t_s + KT * (j & 1), q_at, k_at + (j % KS) * kK, is);
            else tc3_scores_t<NC, KT>(t_s, t_q, k_at, is);
            tcx_commit(&bars->s_full[j & 1]);
          };
          auto products = [&](int j) {
            if (!(ok = tcx_wait(&bars->v_full, j & 1))) return;
            tcx_seen();
            tc3_scores<NC, 128, KT>(t_dp, g_at, v_at, is);
            tcx_commit(&bars->dp_full);
            tcx_commit(&bars->v_empty);
          };
          ok = tcx_wait(&bars->in_full, 0);
          tcx_after_sync();
          if (ok) scores(0);
          if (ok) products(0);
          if (NC == 1 && ok && n > 1) scores(1);
          for (int j = 0; j < n && ok; ++j) {
            if (!(ok = tcx_wait(&bars->ds_full, j & 1))) break;
            tcx_after_sync();
            if (NC == 1 && j + 1 < n) products(j + 1);
            if (!ok) break;
            tc3_combine<NC, KT, KT>(t_dq, t_ds, k_at + (j % KS) * kK, io);
            tcx_commit(&bars->dq_done);
            tcx_commit(&bars->k_empty[j % KS]);
            if (NC == 1 && j + 2 < n) scores(j + 2);
            if (NC == 2 && j + 1 < n) {
              scores(j + 1);
              if (ok) products(j + 1);
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
          tc3_load<NC, 32, KT>(k_at + (j % KS) * kK, src, pp.k_split, p.ks[1], KT * j, keys, pp.chunks, lane);
          tcx_arrive_copies(&bars->k_full[j % KS]);
        }
        tcx_copies_done();
      } else if (warp == 10) {
        const bf16* src = static_cast<const bf16*>(p.v) + b * p.vs[0] + hk * p.vs[2];
        for (int j = 0; j < n && ok; ++j) {
          if (j >= 1) ok = tcx_wait_warp(&bars->v_empty, (j - 1) & 1);
          if (!ok) break;
          tc3_load<NC, 32, KT>(v_at, src, pp.v_split, p.vs[1], KT * j, keys, pp.chunks, lane);
          tcx_arrive_copies(&bars->v_full);
        }
        tcx_copies_done();
      }
    } else {
      asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
      const int half = warp >> 2, row = 32 * (warp & 3) + lane, i = i0 + row;
      const long at = (((long)b * p.lq + i) * p.heads + h) * p.dim;
      if (n) {
        const bf16* const q0 = static_cast<const bf16*>(p.q) + b * p.qs[0] + h * p.qs[2];
        if constexpr (NC == 1) {
          tc3_load<1, 256, 128>(q_at, q0, pp.q_split, p.qs[1], i0, s.qlen, pp.chunks, tid);
        } else {
          const bf16* const row_at = q0 + (long)(i < s.qlen ? i : 0) * p.qs[1];
#pragma unroll
          for (int part = 0; part < 3; ++part)
#pragma unroll
            for (int c = 0; c < 64; c += 32)
              tcx_put_operand(t_q + 64 * part + ((uint32_t)(32 * (warp & 3)) << 16), row_at + part * pp.q_split, 64 * half + c, pp.chunks, i < s.qlen);
          tcx_st_wait();
          tcx_before_sync();
        }
        tc3_load<NC, 256, 128>(g_at, static_cast<const bf16*>(p.dout) + b * pp.gs[0] + h * pp.gs[2], pp.g_split, pp.gs[1], i0, s.qlen, pp.chunks, tid);
        tcx_loaded();
        tcx_arrive(&bars->in_full);
      }
      float delta = 0.f;                                                   // dO . O, every second value per thread
      if (i < s.qlen) {
        const float *g = static_cast<const float*>(pp.grad) + at, *o = static_cast<const float*>(p.o) + at;
        for (int c = half; c < p.dim; c += 2) delta = fmaf(g[c], o[c], delta);
      }
      red[tid] = delta;
      tc3_sync();
      delta = red[row] + red[128 + row];
      const float2 st = i < s.qlen ? p.stats[((long)b * p.heads + h) * p.lq + i] : make_float2(INFINITY, 0.f);
      if (half == 0 && i < p.lq) p.delta[((long)b * p.heads + h) * p.lq + i] = delta;
      const float inv = st.y;
      const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
      const float scale = p.scale * kLog2e, tab_before = tab[0], tab_behind = tab[2 * p.reach + 2 * kTcxMargin];
      float far_before = 0.f, far_behind = 0.f, acc[32 * NC];
#pragma unroll
      for (int c = 0; c < 32 * NC; ++c) acc[c] = 0.f;
      auto drain = [&](int j) {
        if (ok) ok = tcx_wait_warp(&bars->dq_done, j & 1);
        tcx_after_sync();
#pragma unroll
        for (int c = 0; c < 32 * NC; c += 32) {
          uint32_t o[32];
          tcx_ld32(t_dq + 32 * NC * half + c + lanes, o);
          tcx_ld_wait(o);
#pragma unroll
          for (int e = 0; e < 32; ++e) acc[c + e] += as_float(o[e]);
        }
      };
      int turn = 0;
      for (int j = 0; j < n; ++j) {
        const int j0 = KT * j, d0 = j0 - i0 - s.start;
        const bool close = d0 + KT - 1 > -p.reach && d0 - 127 < p.reach && p.reach > 0;
        if (ok) ok = tcx_wait_warp(&bars->s_full[j & 1], (j >> 1) & 1);
        tcx_after_sync();
        uint32_t raw[32], grad[32];
        tcx_ld32(t_s + (NC == 1 ? KT * (j & 1) : 0) + HALF * half + lanes, raw);
        tcx_ld_wait(raw);
        float* x = reinterpret_cast<float*>(raw);
        if (close) {
          const float* near = tab + (d0 + HALF * half - row + p.reach + kTcxMargin);
#pragma unroll
          for (int c = 0; c < 32; ++c) x[c] = fmaf(x[c], scale, near[c]) - st.x;
        } else {
          const float far = d0 > 0 ? tab_behind : tab_before;
#pragma unroll
          for (int c = 0; c < 32; ++c) x[c] = fmaf(x[c], scale, far) - st.x;
        }
        const bool edge = j0 + KT > keys || (p.causal && d0 + KT - 1 > 0);
        const int lim = (p.causal ? min(keys - j0, row - d0 + 1) : keys - j0) - HALF * half;
        if (edge) {
#pragma unroll
          for (int c = 0; c < 32; ++c) x[c] = c < lim ? x[c] : kNoScore;
        }
#pragma unroll
        for (int c = 0; c < 32; ++c) x[c] = exp2_fast(x[c]) * inv;
        if (ok) ok = tcx_wait_warp(&bars->dp_full, j & 1);
        tcx_after_sync();
        tcx_ld32(t_dp + HALF * half + lanes, grad);
        tcx_ld_wait(grad);
#pragma unroll
        for (int c = 0; c < 32; ++c) x[c] *= as_float(grad[c]) - delta;
        if (edge) {
#pragma unroll
          for (int c = 0; c < 32; ++c) x[c] = c < lim ? x[c] : 0.f;
        }
        if (j > 0) drain(j - 1);                                           // (the columns of dS have been read, too)
        if (NC == 2) {                                                     // both groups have read the scores
          tcx_before_sync();
          tc3_sync();
          tcx_after_sync();
        }
        tc3_put<32>(t_ds + 16 * half + lanes, 32, x);
        tcx_st_wait();
        tcx_before_sync();
        __syncwarp();
        if (lane == 0) tcx_arrive(&bars->ds_full);
        if (!p.dbias_part) continue;
        if (close) {
          float* mine = diag + (8 * turn + warp) * kTc3Diag;
          float run[2] = {0.f, 0.f};
#pragma unroll
          for (int c = 0; c < 16; ++c) {
#pragma unroll
            for (int k = 0; k < 2; ++k) run[k] += x[16 * k + c];
            if (c == 15) break;
            if (lane == 31) {
#pragma unroll
              for (int k = 0; k < 2; ++k) mine[48 * k + c] = run[k];
            }
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              run[k] = __shfl_up_sync(0xffffffffu, run[k], 1);
              run[k] = lane == 0 ? 0.f : run[k];
            }
          }
#pragma unroll
          for (int k = 0; k < 2; ++k) mine[48 * k + 46 - lane] = run[k];
          tc3_sync();
          if (tid < 127 + KT) {
            const int off = tid - 127, d = d0 + off;
            float sum = 0.f;
#pragma unroll
            for (int wv = 0; wv < 8; ++wv)
#pragma unroll
              for (int k = 0; k < 2; ++k) {
                const int e = off + 32 * (wv & 3) - HALF * (wv >> 2) - 16 * k + 31;
                if (e >= 0 && e < 47) sum += diag[(8 * turn + wv) * kTc3Diag + 48 * k + e];
              }
            if (d <= -p.reach) far_before += sum;
            else if (d >= p.reach) far_behind += sum;
            else slot[d + p.reach] += sum;
          }
          turn ^= 1;
        } else {
          float sum[2] = {0.f, 0.f};
#pragma unroll
          for (int c = 0; c < 32; ++c) sum[c & 1] += x[c];
          if (d0 > 0) far_behind += sum[0] + sum[1];
          else far_before += sum[0] + sum[1];
        }
      }
      if (n) drain(n - 1);
      if (ok && n) ok = tcx_wait_warp(&bars->drained, 0);
      const bool wide = p.dim % 4 == 0 && reinterpret_cast<uintptr_t>(p.dq) % 16 == 0;
      const bool sees = i < s.qlen && p.stats[((long)b * p.heads + h) * p.lq + i].y != 0.f;      // (read again, see AttnTcGradQ)
#pragma unroll
      for (int c = 0; c < 32 * NC; ++c) acc[c] = !ok ? bulk_nan() : sees ? acc[c] * p.scale : 0.f;
      if (i < p.lq) tc3_store_row(static_cast<float*>(p.dq) + at, acc, 32 * NC, p.dim, 32 * NC * half, wide);
      if (p.dbias_part) {
        tc3_sync();
        red[tid] = far_before;
        red[256 + tid] = far_behind;
        tc3_sync();
        if (warp < 2) {
          float sum = 0.f;
          for (int e = lane; e < 256; e += 32) sum += red[256 * warp + e];
#pragma unroll
          for (int m = 16; m >= 1; m /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, m);
          if (lane == 0) red[256 * warp] = sum;
        }
        tc3_sync();
        if (tid == 0) {
          slot[0] = red[0];
          if (p.reach > 0) slot[2 * p.reach] = red[256];
          else slot[0] += red[256];
        }
        tc3_sync();
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

// ---- gradients of keys and values ------------------------------------------------------------------------------------------------
// As AttnTcGradKV, with query tiles of 64; the products of a tile are added to registers, half of the columns of either gradient
// per group.
// NC = 2: the keys lie in tensor memory, P^T and dS^T go over scores and products, both gradients pass through the same columns one
// after the other, and there is one tile each of queries and dO.
struct Tc3KvBars {
  uint64_t in_full, s_full, s_read, dp_full, dp_read, p_full, ds_full, dv_done, dk_done, q_full[2], q_empty[2], g_full[2], g_empty[2], r_full[2],
      r_empty[2], drained;
  uint32_t tmem;
};
template <int NC>
struct AttnTc3GradKV {
  static constexpr int kThreads = kTc3Threads, QT = 64, HALF = 32, QS = NC == 1 ? 2 : 1;
  static constexpr uint32_t kK = 3 * NC * 128 * 128, kQ = 3 * NC * QT * 128, kTiles = (NC == 1 ? 2 : 1) * kK + 2 * QS * kQ;
  static size_t smem(int reach) {
    return 1024 + (size_t)kTiles + (2 * 3 * QT + 2 * reach + 2 * kTcxMargin + 1) * sizeof(float) + sizeof(Tc3KvBars) + 16;
  }
  static __device__ __forceinline__ void run(const AttnTcParams& pp, float4* dyn) {
    const AttnParams& p = pp.a;
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const uint32_t base = (tcx_addr(dyn) + 1023u) & ~1023u;
    unsigned char* const smem = reinterpret_cast<unsigned char*>(dyn) + (base - tcx_addr(dyn));
    float* const stat = reinterpret_cast<float*>(smem + kTiles);             // [2][3][QT]: m, 1 / l, delta
    float* const tab = stat + 2 * 3 * QT;
    Tc3KvBars* const bars = reinterpret_cast<Tc3KvBars*>((reinterpret_cast<uintptr_t>(tab + tcx_tab_floats(p.reach)) + 15) & ~(uintptr_t)15);
    const uint32_t v_at = base, q_at = base + kK, g_at = q_at + QS * kQ, k_at = g_at + QS * kQ;      // (k: NC = 1)
    const int heads_all = p.batch * p.kv_heads;
    const int tile = (int)blockIdx.x / heads_all, bh = (int)blockIdx.x % heads_all, hk = bh % p.kv_heads, b = bh / p.kv_heads;
    if (tid == 0) {
      tcx_init(&bars->in_full, 256);
      tcx_init(&bars->s_full, 1);
      tcx_init(&bars->s_read, 8);
      tcx_init(&bars->dp_full, 1);
      tcx_init(&bars->dp_read, 8);
      tcx_init(&bars->p_full, 8);
      tcx_init(&bars->ds_full, 8);
      tcx_init(&bars->dv_done, 1);
      tcx_init(&bars->dk_done, 1);
      for (int i = 0; i < 2; ++i) {
        tcx_init(&bars->q_full[i], 32);
        tcx_init(&bars->q_empty[i], 1);
        tcx_init(&bars->g_full[i], 32);
        tcx_init(&bars->g_empty[i], 1);
        tcx_init(&bars->r_full[i], 1);
        tcx_init(&bars->r_empty[i], 8);
      }
      tcx_init(&bars->drained, 1);
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    const AttnSeq s = attn_seq(p, b);
    const int j0 = 128 * tile, keys = attn_keys(p, s, s.qlen);
    const int first = j0 < keys ? attn_first_query(p, s, j0) / QT : 0;
    const int per_head = j0 < keys ? (s.qlen + QT - 1) / QT - first : 0, n = per_head > 0 ? per_head * p.group : 0;
    if (warp == 8) {
      __syncwarp();
      tcx_alloc<512>(&bars->tmem);
    }
    tcx_before_sync();
    __syncthreads();
    tcx_after_sync();
    const uint32_t tmem = __shfl_sync(0xffffffffu, bars->tmem, 0);
    stream_order_next();
    const uint32_t t_k = tmem, t_s = NC == 1 ? tmem : tmem + 192, t_dp = NC == 1 ? tmem + 64 : tmem + 288, t_p = NC == 1 ? tmem + 128 : t_s,
                   t_ds = NC == 1 ? tmem + 224 : t_dp, t_dv = NC == 1 ? tmem + 320 : tmem + 384, t_dk = tmem + 384;
    bool ok = true;

    if (warp >= 8) {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
      if (warp == 8) {
        if (n && tcx_elect()) {
          const int steps = (pp.chunks + 1) / 2;
          const uint32_t is = tcx_idesc(QT, false), io = tcx_idesc(16 * steps, true);
          auto scores = [&](int t) {
            if (!(ok = tcx_wait(&bars->q_full[t % QS], (t / QS) & 1))) return;
            tcx_seen();
            if constexpr (NC == 1) tc3_scores<1, 128, QT>(t_s, k_at, q_at + (t % QS) * kQ, is);
            else tc3_scores_t<NC, QT>(t_s, t_k, q_at, is);
            tcx_commit(&bars->s_full);
          };
          auto products = [&](int t) {
            if (!(ok = tcx_wait(&bars->g_full[t % QS], (t / QS) & 1))) return;
            tcx_seen();
            tc3_scores<NC, 128, QT>(t_dp, v_at, g_at + (t % QS) * kQ, is);
            tcx_commit(&bars->dp_full);
          };
          ok = tcx_wait(&bars->in_full, 0);
          tcx_after_sync();
          if (ok) scores(0);
          if (ok) products(0);
          for (int t = 0; t < n && ok; ++t) {
            if (NC == 1 && t + 1 < n) {
              if (!(ok = tcx_wait(&bars->s_read, t & 1))) break;
              tcx_after_sync();
              scores(t + 1);
            }
            if (!ok || !(ok = tcx_wait(&bars->p_full, t & 1))) break;
            tcx_after_sync();
            tc3_combine<NC, QT, QT>(t_dv, t_p, g_at + (t % QS) * kQ, io);
            tcx_commit(&bars->dv_done);
            tcx_commit(&bars->g_empty[t % QS]);
            if (NC == 1 && t + 1 < n) {
              if (!(ok = tcx_wait(&bars->dp_read, t & 1))) break;
              tcx_after_sync();
              products(t + 1);
            }
            if (!ok || !(ok = tcx_wait(&bars->ds_full, t & 1))) break;
            tcx_after_sync();
            tc3_combine<NC, QT, QT>(t_dk, t_ds, q_at + (t % QS) * kQ, io);
            tcx_commit(&bars->dk_done);
            tcx_commit(&bars->q_empty[t % QS]);
            if (NC == 2 && t + 1 < n) {
              scores(t + 1);
              if (ok) products(t + 1);
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
        const long by_head = is_q ? p.qs[2] : pp.gs[2], stride = is_q ? p.qs[1] : pp.gs[1], part = is_q ? pp.q_split : pp.g_split;
        const bf16* src = static_cast<const bf16*>(is_q ? p.q : p.dout) + b * (is_q ? p.qs[0] : pp.gs[0]) + hk * p.group * by_head;
        int g = 0, it = first;
        for (int t = 0; t < n && ok; ++t) {
          if (t >= QS) ok = tcx_wait_warp(&empty[t % QS], (t / QS - 1) & 1);
          if (!ok) break;
          tc3_load<NC, 32, QT>(to + (t % QS) * kQ, src + g * by_head, part, stride, QT * it, s.qlen, pp.chunks, lane);
          tcx_arrive_copies(&full[t % QS]);
          if (++it == first + per_head) { it = first; ++g; }
        }
        tcx_copies_done();
      } else if (warp == 11) {
        int g = 0, it = first;
        for (int t = 0; t < n && ok; ++t) {
          if (t >= 2) ok = tcx_wait_warp(&bars->r_empty[t & 1], (t / 2 - 1) & 1);
          if (!ok) break;
          const long row0 = ((long)b * p.heads + hk * p.group + g) * p.lq;
          float* to = stat + (t & 1) * 3 * QT;
#pragma unroll
          for (int e = lane; e < QT; e += 32) {
            const int i = QT * it + e;
            const float2 st = i < s.qlen ? p.stats[row0 + i] : make_float2(INFINITY, 0.f);
            to[e] = st.x;
            to[QT + e] = st.y;
            to[2 * QT + e] = i < s.qlen ? p.delta[row0 + i] : 0.f;
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
        const bf16* const k0 = static_cast<const bf16*>(p.k) + b * p.ks[0] + hk * p.ks[2];
        if constexpr (NC == 1) {
          tc3_load<1, 256, 128>(k_at, k0, pp.k_split, p.ks[1], j0, keys, pp.chunks, tid);
        } else {
          const bf16* const row_at = k0 + (long)(j < keys ? j : 0) * p.ks[1];
#pragma unroll
          for (int part = 0; part < 3; ++part)
#pragma unroll
            for (int c = 0; c < 64; c += 32)
              tcx_put_operand(t_k + 64 * part + ((uint32_t)(32 * (warp & 3)) << 16), row_at + part * pp.k_split, 64 * half + c, pp.chunks, j < keys);
          tcx_st_wait();
          tcx_before_sync();
        }
        tc3_load<NC, 256, 128>(v_at, static_cast<const bf16*>(p.v) + b * p.vs[0] + hk * p.vs[2], pp.v_split, p.vs[1], j0, keys, pp.chunks, tid);
        tcx_loaded();
        tcx_arrive(&bars->in_full);
      }
      const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
      const float scale = p.scale * kLog2e;
      float dv[32 * NC], dk[32 * NC];
#pragma unroll
      for (int c = 0; c < 32 * NC; ++c) dv[c] = dk[c] = 0.f;
      auto drain = [&](uint64_t* bar, uint32_t from, int t, float (&acc)[32 * NC]) {
        if (ok) ok = tcx_wait_warp(bar, t & 1);
        tcx_after_sync();
#pragma unroll
        for (int c = 0; c < 32 * NC; c += 32) {
          uint32_t o[32];
          tcx_ld32(from + 32 * NC * half + c + lanes, o);
          tcx_ld_wait(o);
#pragma unroll
          for (int e = 0; e < 32; ++e) acc[c + e] += as_float(o[e]);
        }
      };
      int g = -1, it = first + per_head;
      for (int t = 0; t < n; ++t) {
        if (it == first + per_head) {
          it = first;
          ++g;
          tc3_sync();
          tcx_bias_table(p, hk * p.group + g, tab, tid, 256, true);
          tc3_sync();
        }
        const int i0 = QT * it, d0 = j0 - i0 - s.start;                    // relative position of row 0 to query 0
        const float* sm = stat + (t & 1) * 3 * QT + HALF * half;
        if (ok) ok = tcx_wait_warp(&bars->r_full[t & 1], (t >> 1) & 1);
        if (ok) ok = tcx_wait_warp(&bars->s_full, t & 1);
        tcx_after_sync();
        uint32_t raw[32], grad[32];
        tcx_ld32(t_s + HALF * half + lanes, raw);
        tcx_ld_wait(raw);
        tcx_before_sync();
        __syncwarp();
        if (lane == 0) tcx_arrive(&bars->s_read);
        float* x = reinterpret_cast<float*>(raw);
        if (d0 + 127 > -p.reach && d0 - (QT - 1) < p.reach && p.reach > 0) {
          const float* near = tab + (d0 + row - HALF * half + p.reach + kTcxMargin);
#pragma unroll
          for (int c = 0; c < 32; ++c) x[c] = fmaf(x[c], scale, near[-c]);
        } else {
          const float far = d0 > 0 ? tab[2 * p.reach + 2 * kTcxMargin] : tab[0];
#pragma unroll
          for (int c = 0; c < 32; ++c) x[c] = fmaf(x[c], scale, far);
        }
        const bool edge = j0 + 128 > keys || (p.causal && d0 + 127 > 0);
        const int low = j >= keys ? 128 : (p.causal ? d0 + row : 0) - HALF * half;
        if (edge) {
#pragma unroll
          for (int c = 0; c < 32; ++c) x[c] = c >= low ? x[c] : kNoScore;
        }
#pragma unroll
        for (int c = 0; c < 32; c += 4) {
          const float4 m = *reinterpret_cast<const float4*>(sm + c), f = *reinterpret_cast<const float4*>(sm + QT + c);
          x[c] = exp2_fast(x[c] - m.x) * f.x;
          x[c + 1] = exp2_fast(x[c + 1] - m.y) * f.y;
          x[c + 2] = exp2_fast(x[c + 2] - m.z) * f.z;
          x[c + 3] = exp2_fast(x[c + 3] - m.w) * f.w;
        }
        if (NC == 1) {
          if (t > 0) drain(&bars->dv_done, t_dv, t - 1, dv);
        } else {
          if (t > 0) drain(&bars->dk_done, t_dk, t - 1, dk);
          tcx_before_sync();
          tc3_sync();                                                      // both groups have read the scores
          tcx_after_sync();
        }
        tc3_put<32>(t_p + 16 * half + lanes, 32, x);
        tcx_st_wait();
        tcx_before_sync();
        __syncwarp();
        if (lane == 0) tcx_arrive(&bars->p_full);
        if (ok) ok = tcx_wait_warp(&bars->dp_full, t & 1);
        tcx_after_sync();
        tcx_ld32(t_dp + HALF * half + lanes, grad);
        tcx_ld_wait(grad);
        tcx_before_sync();
        __syncwarp();
        if (lane == 0) tcx_arrive(&bars->dp_read);
#pragma unroll
        for (int c = 0; c < 32; c += 4) {
          const float4 f = *reinterpret_cast<const float4*>(sm + 2 * QT + c);
          x[c] *= as_float(grad[c]) - f.x;
          x[c + 1] *= as_float(grad[c + 1]) - f.y;
          x[c + 2] *= as_float(grad[c + 2]) - f.z;
          x[c + 3] *= as_float(grad[c + 3]) - f.w;
        }
        if (edge) {
#pragma unroll
          for (int c = 0; c < 32; ++c) x[c] = c >= low ? x[c] : 0.f;
        }
        if (NC == 1) {
          if (t > 0) drain(&bars->dk_done, t_dk, t - 1, dk);
        } else {
          drain(&bars->dv_done, t_dv, t, dv);
          tcx_before_sync();
          tc3_sync();                                                      // both have read the products
          tcx_after_sync();
        }
        tc3_put<32>(t_ds + 16 * half + lanes, 32, x);
        tcx_st_wait();
        tcx_before_sync();
        __syncwarp();
        if (lane == 0) {
          tcx_arrive(&bars->ds_full);
          tcx_arrive(&bars->r_empty[t & 1]);
        }
        ++it;
      }
      if (n) {
        if (NC == 1) drain(&bars->dv_done, t_dv, n - 1, dv);
        drain(&bars->dk_done, t_dk, n - 1, dk);
        if (ok) ok = tcx_wait_warp(&bars->drained, 0);
      }
#pragma unroll
      for (int c = 0; c < 32 * NC; ++c) {
        dv[c] = ok ? dv[c] : bulk_nan();
        dk[c] = ok ? dk[c] * p.scale : bulk_nan();
      }
      const long at = (((long)b * p.lk + j) * p.kv_heads + hk) * p.dim;
      if (j < p.lk) {
        tc3_store_row(static_cast<float*>(p.dv) + at, dv, 32 * NC, p.dim, 32 * NC * half, p.dim % 4 == 0 && reinterpret_cast<uintptr_t>(p.dv) % 16 == 0);
        tc3_store_row(static_cast<float*>(p.dk) + at, dk, 32 * NC, p.dim, 32 * NC * half, p.dim % 4 == 0 && reinterpret_cast<uintptr_t>(p.dk) % 16 == 0);
      }
    }
    tcx_before_sync();
    __syncthreads();
    if (warp == 8) tcx_free<512>(tmem);
  }
};

}  // namespace s2c
#endif  // S2C_EMUL
