// Attention of few queries over keys and values in pages: the queries of all heads that share a key head make up to 8 or 16 rows of a
// block (more: several row blocks), and the time is that of reading the keys and values once.
//
// Keys and values never pass through shared memory.  Products are transposed, S^T = K Q^T and O^T = V^T P^T, on the warp-level matrix
// instructions, with keys and values as left operands of 16 rows straight from the registers that they were loaded into.  A sum
// over the values of a head may run in any order that both operands share, and rows of O^T may be any values of a head: so a lane
// loads 16 consecutive bytes of a row and takes them as the operand's elements that it is to hold, and rows 8 positions apart as
// its other half.  For V^T the halves of two words are exchanged (neighbouring positions have to share a register); the weights
// change from rows to columns by one movement within the warp.  The eight columns are the queries: with at most eight no row is wasted.
//
// Keys of the next tile are asked for as soon as the scores of this one are done, its values as soon as the outputs are: a warp has
// up to 8 KB (float32 16) on its way and waits for nobody.  The page of every eighth position comes a tile earlier, by one load per warp.
// A tile that goes past the last position reads that one again there, with a weight of 0, and where the table names no page, page 0: no
// load is guarded.  (Guarded ones, whose registers keep what they held, cost 64 x 16384 positions 579 us.)
//
// Work is dealt in steps of (4 warps x tile) positions of one item (sequence, key head, row block), an equal share to each block as
// the lengths on the device give it: a block finds where its share begins by adding up the sequences' steps.  Items that lie in
// several blocks leave partial results, joined by a second kernel in the order of the blocks.
//
// bfloat16 queries and keys are multiplied as they are; the weights enter the second product as two bfloat16 parts, float32 operands
// as two TF32 parts of which the product of the smaller ones is left out, so that a result's rounding is its own.
//
// Bound by memory where sequences are long: 64 x 16384 positions, 16 heads of 128 on 4, 2.1 GB: 315 us (6.8 TB/s; the measured copy
// rate is 6.56); 16 ragged ones of up to 16384, 285 MB, 49 us (5.9).  Short ones by the chain of a block's loads, lengths, pages, keys, and
// the second launch: one step 5 us, 1 x 16384 positions 15 us (2.3 TB/s).  The steps of a sequence are those of its last query for all of
// its row blocks: rows that see less, or none, take as long.
#pragma once

#include "attention_few.h"
#include "kept_pages.h"

#ifndef S2C_EMUL

namespace s2c {

struct PagedParams {
  AttnParams a;              // k, v are not used
  PageTable pages;
  long ks[3], vs[3];         // page, position, head
  int row_blocks;
  Divisor by_group, by_row_blocks, by_buckets;     // of the rows, the items of a sequence, and n_buckets + 1
  int wide_out;              // out in pieces of four values
  float* part;               // [2 blocks][rows][DP + 4]: slot 2 c: an item that began before block c; 2 c + 1: one that goes on behind it
  int4* split;               // [min(items, blocks)]: item, first block, blocks of an item that is joined; 0 blocks: none
};

__device__ __forceinline__ unsigned paged_movmatrix(unsigned v) {
  unsigned r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ void paged_mma(float (&d)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void paged_mma_tf32(float (&d)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// How rows are read: value by value; in whole pieces of 16 bytes, on whose boundaries they lie, of which the last ones may hold
// less or nothing of a head; or such that a head fills all pieces.
enum PagedRows : int { kRowsByValue, kRowsInPieces, kRowsFull };
// N consecutive values of a row from value c on, as an operand's registers hold them.  Where a head has ended: zeros by value; in
// pieces what lies behind it in the piece that its last value lies in, and in place of pieces beyond that one, the row's first.
template <class T, int N, int ROWS>
__device__ __forceinline__ void paged_load(unsigned (&w)[N * sizeof(T) / 4], const T* row, int c, int dim) {
  if constexpr (ROWS != kRowsByValue) {
    const T* from = row + (ROWS == kRowsFull || c < dim ? c : 0);
    if constexpr (N * sizeof(T) == 16)
      asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "l"(from) : "memory");
    else
      asm volatile("ld.global.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "l"(from) : "memory");
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      if constexpr (sizeof(T) == 4) {
        w[e] = c + e < dim ? reinterpret_cast<const unsigned*>(row)[c + e] : 0u;
      } else if (e % 2 == 0) {
        const unsigned short* at = reinterpret_cast<const unsigned short*>(row) + c + e;
        w[e / 2] = (c + e < dim ? at[0] : 0u) | (c + e + 1 < dim ? (unsigned)at[1] << 16 : 0u);
      }
    }
  }
}

// DP: values of a head, rounded up to 32, 64 or 128; NT: row blocks of 8 NT rows
template <class T, int DP, int NT>
struct PagedShape {
  static constexpr bool kHalf = sizeof(T) == 2;
  static constexpr int kWarps = 4, kThreads = 32 * kWarps, kRows = 8 * NT;
  static constexpr int kTiles = kHalf ? 128 / DP : DP == 128 ? 1 : 64 / DP;     // of 16 positions, for a warp's step
  static constexpr int kKeys = 16 * kTiles, kStep = kWarps * kKeys;
  static constexpr int kQk = kHalf ? DP / 32 : DP / 16;                       // a row's chunks of four 16-byte pieces
  static constexpr int kVd = kHalf && DP > 32 ? 8 : 4, kVc = DP / (8 * kVd);   // a lane's consecutive values of a row of V, chunks
  static constexpr int kOut = DP / 16;                                        // tiles of 16 rows of O^T
  static constexpr size_t kQuery = (size_t)kQk * NT * 32 * 16 * (kHalf ? 1 : 2), kJoin = (size_t)kWarps * kRows * (DP + 4) * 4 + kRows * 5 * 4;
  // where value `m` (0: of the upper eight rows) of tile t of a lane lies in a head
  static __device__ __forceinline__ int value(int t, int lane) { return t / (kVd / 2) * 8 * kVd + lane / 4 * kVd + 2 * (t % (kVd / 2)); }
};

// keys of a sequence that some query sees, and the steps of its items: at least one, which writes the zeros of a sequence without keys
__device__ __forceinline__ int paged_steps(const AttnParams& a, int b, int step) {
  const AttnSeq s = attn_seq(a, b);
  const int n = (attn_keys(a, s, s.qlen) + step - 1) / step;
  return n > 0 ? n : 1;
}

template <class T, int DP, int NT, int ROWS>
struct PagedAttention {
  using Params = PagedParams;
  using H = PagedShape<T, DP, NT>;
  static constexpr int kThreads = H::kThreads;
  // Blocks an SM, and with them 168 or 255 registers a thread.  Those hold a step's keys and values in <bf16, 128, 1> and <float, 64, 1> on
  // whole rows; other instances keep a part in local memory: 4 to 102 bytes a thread with one row group, with two 78 to 298 at 168
  // registers, and at 255 4 to 22 (bfloat16) or 334 to 410 (float32).
  static constexpr int kBlocks = (H::kHalf ? DP <= 64 || NT == 1 : DP <= 64) ? 3 : 2;
  // queries, results, the search for the share; the biases of each row by bucket, 0 behind them, and the bucket of each position
  static size_t smem(const AttnParams& a) {
    return H::kQuery + H::kJoin + 128 + (a.bias ? (size_t)H::kRows * (a.n_buckets + 1) * 4 + (size_t)(2 * a.reach + 1) * 2 : 0);
  }
  // (64 bits only where they are needed: a division of them is a hundred instructions)
  static __device__ __forceinline__ long quotient(long x, long y) {
    return (x | y) >> 32 ? x / y : (long)((unsigned)x / (unsigned)y);
  }

  struct Tile {
    unsigned k[H::kTiles][2][H::kQk][4];
    unsigned v[H::kTiles][4][H::kVc][H::kVd * sizeof(T) / 4];
  };

  static __device__ __forceinline__ void run(const Ctx& ctx, const Params& p, unsigned char* smem) {
    const AttnParams& a = p.a;
    const int lane = ctx.tid % 32, warp = ctx.tid / 32;
    uint4* const query = reinterpret_cast<uint4*>(smem);
    float* const join = reinterpret_cast<float*>(smem + H::kQuery);
    long* const find = reinterpret_cast<long*>(smem + H::kQuery + H::kJoin);      // the warps' sums, twice; [4], [5] where the share begins
    float* const biases = reinterpret_cast<float*>(smem + H::kQuery + H::kJoin + 128);
    unsigned short* const bucket = reinterpret_cast<unsigned short*>(biases + H::kRows * (a.n_buckets + 1));
    const int per_batch = a.kv_heads * p.row_blocks;                              // items of a sequence

    // ---- this block's share
    const int mine = (a.batch + kThreads - 1) / kThreads;                         // sequences of a thread
    // the sum of `of` over the sequences before this thread's, over this thread's, and over all
    const int n_first = ctx.tid * mine < a.batch ? paged_steps(a, ctx.tid * mine, H::kStep) : 0;
    auto add_up = [&](auto of, long* warps, long& sum, long& all) {
      sum = n_first ? of(n_first) : 0;
      for (int i = 1; i < mine; ++i)
        if (ctx.tid * mine + i < a.batch) sum += of(paged_steps(a, ctx.tid * mine + i, H::kStep));
      long before = sum;
#pragma unroll
      for (int m = 1; m < 32; m *= 2) {
        const long o = __shfl_up_sync(0xffffffffu, before, m);
        if (lane >= m) before += o;
      }
      if (lane == 31) warps[warp] = before;
      ctx.sync();
      all = 0;
      for (int w = 0; w < H::kWarps; ++w) {
        if (w == warp) before += all;
        all += warps[w];
      }
      return before - sum;
    };
    long sum, all;
    long before = add_up([](int n) { return n; }, find, sum, all);
    const bool by_item = (long)a.batch * per_batch <= ctx.nblk;                   // as the host counts the splits
    // Steps [lo, hi) of all, an equal share, in which an item counts kOpening steps more than it has, in front: beginning one costs about
    // that (32 x 4000 positions of different lengths, 128 items: 22.4 us, 28.9 without; 1 and 4 steps 24.6 and 23.5).
    constexpr int kOpening = 2;
    int opening = kOpening;
    const long steps = all * per_batch, total = steps + (long)a.batch * per_batch * kOpening, blocks = min((long)ctx.nblk, steps);
    const long each = quotient(total, blocks), rest = total - each * blocks;       // the first `rest` blocks have one more
    long lo = ctx.bid * each + min((long)ctx.bid, rest), used = blocks;
    const long hi = lo + each + (ctx.bid < rest);
    before += (long)min(ctx.tid * mine, a.batch) * kOpening;
    sum += (long)max(min(mine, a.batch - ctx.tid * mine), 0) * kOpening;
    // With few steps a block: pieces of `per` steps of one item each, where the blocks hold them (32 x 1000 positions, 128 items: 16.8 us
    // instead of 18.2; one step a block: the same without a second sum).
    const int per = (int)min(quotient(steps + blocks - 1, blocks), 5L);
    bool pieces = per == 1;
    if (per <= 4) {
      long of_thread = sum, of_all = all, first = before;
      if (per > 1) {
        first = add_up([&](int n) { return (int)((unsigned)(n + per - 1) / (unsigned)per); }, find + 8, of_thread, of_all);
        pieces = of_all * per_batch <= ctx.nblk;
      } else {
        of_thread -= (long)max(min(mine, a.batch - ctx.tid * mine), 0) * kOpening;
        first -= (long)min(ctx.tid * mine, a.batch) * kOpening;
      }
      if (pieces) {
        sum = of_thread;
        before = first;
        used = of_all * per_batch;
        lo = ctx.bid;
        opening = 0;
      }
    }
    if (ctx.bid >= used) {
      if (!by_item && ctx.tid == 0) p.split[ctx.bid] = make_int4(0, 0, 0, 0);
      return;
    }
    auto parts_of = [&](int n) { return pieces ? (int)((unsigned)(n + per - 1) / (unsigned)per) : n + opening; };
    if (a.bias)
      for (int e = ctx.tid; e <= 2 * a.reach; e += 4 * kThreads) {               // (four loads on their way)
        int which[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) which[k] = a.bucket_of[min(e + k * kThreads, 2 * a.reach)];
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (e + k * kThreads <= 2 * a.reach) bucket[e + k * kThreads] = (unsigned short)(which[k] >= 0 && which[k] < a.n_buckets ? which[k] : a.n_buckets);
      }
    if (before * per_batch <= lo && lo < (before + sum) * per_batch) {
      int b = ctx.tid * mine;
      for (;; ++b) {
        const int n = parts_of(paged_steps(a, b, H::kStep));
        if (lo < (before + n) * per_batch) break;
        before += n;
      }
      find[4] = b;
      find[5] = lo - before * per_batch;
    }
    ctx.sync();
    int b = (int)find[4];
    int n = paged_steps(a, b, H::kStep);
    const int of_item = parts_of(n);
    int within = (int)quotient(find[5], of_item), v0 = (int)(find[5] - (long)within * of_item) * (pieces ? per : 1);     // in the item, its opening counted
    bool joined = false;
    for (long at = lo, left = pieces ? min(per, n - v0) : hi - lo; left > 0;) {
      const int v1 = (int)min((long)n + opening, v0 + left), s0 = max(v0 - opening, 0), s1 = max(v1 - opening, 0);
      if (s0 < s1) {
        const int hk = p.by_row_blocks.quotient(within), rb = within - hk * p.row_blocks, item = b * per_batch + within;
        const bool whole = s0 == 0 && s1 == n;
        float* part = whole ? nullptr : p.part + (2L * ctx.bid + (s0 == 0 ? 1 : 0)) * H::kRows * (DP + 4);
        piece(ctx, p, query, join, biases, bucket, b, hk, rb, s0, s1, part);
        if (ctx.tid == 0) {
          if (by_item && whole) p.split[item] = make_int4(0, 0, 0, 0);
          if (!whole && s0 == 0) {
            const long end = at - v0 + opening + n - 1, more = rest * (each + 1), last = end < more ? quotient(end, each + 1) : rest + quotient(end - more, each);
            p.split[by_item ? item : ctx.bid] = make_int4(item, ctx.bid, pieces ? of_item : (int)(last - ctx.bid) + 1, 0);
            joined = true;
          }
        }
      }
      at += v1 - v0;
      left -= v1 - v0;
      v0 = 0;
      if (left > 0 && ++within == per_batch) {
        within = 0;
        n = paged_steps(a, ++b, H::kStep);
      }
    }
    if (!by_item && !joined && ctx.tid == 0) p.split[ctx.bid] = make_int4(0, 0, 0, 0);
  }

  // S^T: 16 positions x 8 rows a tile
  static __device__ __forceinline__ void scores(const uint4* query, int lane, int dim, Tile& t, float (&x)[H::kTiles][NT][4]) {
    // a piece that the head ends in holds what lies behind it, pieces beyond it the row's first values
    if (ROWS == kRowsInPieces)
#pragma unroll
      for (int c = 0; c < H::kQk; ++c)
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const int left = dim - (4 * c + lane % 4) * (16 / (int)sizeof(T)) - w * (4 / (int)sizeof(T));      // values of the word
          const unsigned keep = left >= 4 / (int)sizeof(T) ? 0xffffffffu : left == 1 ? 0xffffu : 0u;
#pragma unroll
          for (int m = 0; m < 2 * H::kTiles; ++m) t.k[m / 2][m % 2][c][w] &= keep;
        }
#pragma unroll
    for (int k = 0; k < H::kTiles; ++k)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) x[k][nt][e] = 0.f;
    if constexpr (H::kHalf) {
#pragma unroll
      for (int c = 0; c < H::kQk; ++c)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const uint4 y = query[(c * NT + nt) * 32 + lane];
#pragma unroll
          for (int k = 0; k < H::kTiles; ++k) {
            paged_mma(x[k][nt], t.k[k][0][c][0], t.k[k][1][c][0], t.k[k][0][c][1], t.k[k][1][c][1], y.x, y.y);
            paged_mma(x[k][nt], t.k[k][0][c][2], t.k[k][1][c][2], t.k[k][0][c][3], t.k[k][1][c][3], y.z, y.w);
          }
        }
    } else {
      float z[H::kTiles][NT][4] = {};                  // the small products
#pragma unroll
      for (int c = 0; c < H::kQk; ++c)
#pragma unroll
        for (int k = 0; k < H::kTiles; ++k) {
          FewSplit u[2][4];
#pragma unroll
          for (int e = 0; e < 8; ++e) u[e / 4][e % 4] = few_split(as_float(t.k[k][e / 4][c][e % 4]));
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const uint4 hi = query[2 * ((c * NT + nt) * 32 + lane)], lo = query[2 * ((c * NT + nt) * 32 + lane) + 1];
            paged_mma_tf32(z[k][nt], u[0][0].lo, u[1][0].lo, u[0][1].lo, u[1][1].lo, hi.x, hi.y);
            paged_mma_tf32(z[k][nt], u[0][0].hi, u[1][0].hi, u[0][1].hi, u[1][1].hi, lo.x, lo.y);
            paged_mma_tf32(x[k][nt], u[0][0].hi, u[1][0].hi, u[0][1].hi, u[1][1].hi, hi.x, hi.y);
            paged_mma_tf32(z[k][nt], u[0][2].lo, u[1][2].lo, u[0][3].lo, u[1][3].lo, hi.z, hi.w);
            paged_mma_tf32(z[k][nt], u[0][2].hi, u[1][2].hi, u[0][3].hi, u[1][3].hi, lo.z, lo.w);
            paged_mma_tf32(x[k][nt], u[0][2].hi, u[1][2].hi, u[0][3].hi, u[1][3].hi, hi.z, hi.w);
          }
        }
#pragma unroll
      for (int k = 0; k < H::kTiles; ++k)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) x[k][nt][e] += z[k][nt][e];
    }
  }

  // steps [s0, s1) of one item; to `part`, or to the output where that is null
  static __device__ __forceinline__ void piece(const Ctx& ctx, const Params& p, uint4* query, float* join, float* biases, const unsigned short* bucket, int b, int hk,
                                               int rb, int s0, int s1, float* part) {
    const AttnParams& a = p.a;
    const int lane = ctx.tid % 32, warp = ctx.tid / 32, g = lane / 4, q4 = lane % 4;
    const int rows = a.lq * a.group, r0 = rb * H::kRows, left = min(H::kRows, rows - r0);
    const AttnSeq s = attn_seq(a, b);
    const int i0 = p.by_group.quotient(r0), i1 = min((int)p.by_group.quotient(r0 + left - 1) + 1, s.qlen);      // queries of the block
    const int keys = i0 < s.qlen ? attn_keys(a, s, i1) : 0;
    const T* const kbase = static_cast<const T*>(p.pages.array[0]) + hk * p.ks[2];
    const T* const vbase = static_cast<const T*>(p.pages.array[1]) + hk * p.vs[2];
    const int* const table = p.pages.table + (long)b * p.pages.columns;
    const int page = p.pages.page, log_page = p.pages.log_page;

    Tile t = {};
    // the page of every eighth position of a step, one to a lane; -1: none
    auto pages_of = [&](int step) {
      const int j = step < s1 ? min((step * H::kWarps + warp) * H::kKeys + 8 * lane, keys - 1) : keys - 1;
      const int id = lane < 2 * H::kTiles && j >= 0 ? table[j >> log_page] : -1;
      return id < p.pages.count ? id : -1;
    };
    constexpr int kPiece = 16 / (int)sizeof(T);
    auto load_keys = [&](int step, int ids) {
      const int j0 = step < s1 ? (step * H::kWarps + warp) * H::kKeys : keys;      // (behind the last step: the last position)
#pragma unroll
      for (int m = 0; m < 2 * H::kTiles; ++m) {
        const int id = max(__shfl_sync(0xffffffffu, ids, m), 0), j = max(min(j0 + 8 * m + g, keys - 1), 0);
        const T* row = kbase + (id * p.ks[0] + (j & (page - 1)) * p.ks[1]);
#pragma unroll
        for (int c = 0; c < H::kQk; ++c) paged_load<T, kPiece, ROWS>(t.k[m / 2][m % 2][c], row, (4 * c + q4) * kPiece, a.dim);
      }
    };
    auto load_values = [&](int step, int ids) {
      const int j0 = step < s1 ? (step * H::kWarps + warp) * H::kKeys : keys;      // (behind the last step: the last position)
#pragma unroll
      for (int m = 0; m < 2 * H::kTiles; ++m) {
        const int id = max(__shfl_sync(0xffffffffu, ids, m), 0);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int j = max(min(j0 + 8 * m + (H::kHalf ? 2 * q4 + e : q4 + 4 * e), keys - 1), 0);
          const T* row = vbase + (id * p.vs[0] + (j & (page - 1)) * p.vs[1]);
#pragma unroll
          for (int c = 0; c < H::kVc; ++c) paged_load<T, H::kVd, ROWS>(t.v[m / 2][2 * (m % 2) + e][c], row, (8 * c + g) * H::kVd, a.dim);
        }
      }
    };
    int now = pages_of(s0), ids = pages_of(s0 + 1);
    load_keys(s0, now);
    load_values(s0, now);

    // ---- queries as the right operands of the scores, and what each row sees
    for (int e = ctx.tid; e < H::kQk * NT * 32; e += kThreads) {
      const int c = e / 32 / NT, nt = e / 32 % NT, l = e % 32, r = r0 + 8 * nt + l / 4, i = p.by_group.quotient(r);
      unsigned w[4];
      paged_load<T, kPiece, kRowsByValue>(w, static_cast<const T*>(a.q) + b * a.qs[0] + i * a.qs[1] + (hk * a.group + r - i * a.group) * a.qs[2],
                                          (4 * c + l % 4) * kPiece, r < rows && i < s.qlen && keys > 0 ? a.dim : 0);
      if constexpr (H::kHalf) {
        query[e] = make_uint4(w[0], w[1], w[2], w[3]);
      } else {
        FewSplit x[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) x[u] = few_split(as_float(w[u]));
        query[2 * e] = make_uint4(x[0].hi, x[1].hi, x[2].hi, x[3].hi);
        query[2 * e + 1] = make_uint4(x[0].lo, x[1].lo, x[2].lo, x[3].lo);
      }
    }
    if (a.bias) {
      const int all = H::kRows * (a.n_buckets + 1);
      for (int e = ctx.tid; e < all; e += 8 * kThreads) {                         // (eight loads on their way)
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int at = min(e + k * kThreads, all - 1), row = p.by_buckets.quotient(at), r = min(r0 + row, rows - 1);
          const int which = min(at - row * (a.n_buckets + 1), a.n_buckets - 1);
          v[k] = widen(static_cast<const T*>(a.bias)[(long)which * a.heads + hk * a.group + p.by_group.rest(r)]);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int at = e + k * kThreads;
          if (at < all) biases[at] = p.by_buckets.rest(at) < a.n_buckets ? attn_bias_units(v[k]) : 0.f;
        }
      }
    }
    int lim[NT][2];                                      // a row sees the positions before lim
    int all_see = keys;                                  // that every row sees
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = r0 + 8 * nt + 2 * q4 + e, i = p.by_group.quotient(r);
        lim[nt][e] = r >= rows ? keys : i < s.qlen ? attn_keys(a, s, i + 1) : 0;
        all_see = min(all_see, lim[nt][e]);
      }
    all_see = min(all_see, __shfl_xor_sync(0xffffffffu, all_see, 1));
    all_see = min(all_see, __shfl_xor_sync(0xffffffffu, all_see, 2));
    ctx.sync();                                          // queries and biases
    float flat[NT][2];                                   // the bias of what lies beyond the reach
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) flat[nt][e] = a.bias ? biases[(8 * nt + 2 * q4 + e) * (a.n_buckets + 1) + bucket[0]] : 0.f;

    const float scale = a.scale * kLog2e;
    float acc[H::kOut][NT][4], m[NT][2], l[NT][2];
#pragma unroll
    for (int c = 0; c < H::kOut; ++c)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[c][nt][e] = 0.f;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) { m[nt][e] = kNoScore; l[nt][e] = 0.f; }

    for (int step = s0; step < s1; ++step) {
      const int j0 = (step * H::kWarps + warp) * H::kKeys, next = pages_of(step + 2);
      const bool there = __all_sync(0xffffffffu, now >= 0 || lane >= 2 * H::kTiles);
      float x[H::kTiles][NT][4];
      scores(query, lane, a.dim, t, x);
      load_keys(step + 1, ids);
      // ---- weights
      const bool far = !a.bias || j0 + H::kKeys - 1 - (i0 + s.start) <= -a.reach;    // one bias per head
      const bool plain = j0 + H::kKeys <= all_see && there;
      float top[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) top[nt][e] = kNoScore;
      if (plain && far) {
#pragma unroll
        for (int k = 0; k < H::kTiles; ++k)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              x[k][nt][e] = fmaf(x[k][nt][e], scale, flat[nt][e % 2]);
              top[nt][e % 2] = fmaxf(top[nt][e % 2], x[k][nt][e]);
            }
      } else {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int row = 8 * nt + 2 * q4 + e, position = (int)p.by_group.quotient(r0 + row) + s.start;
            const float* const of_row = biases + row * (a.n_buckets + 1);
            const int away = j0 + g - position + a.reach, sees = lim[nt][e] - j0 - g;      // of position j0 + g
#pragma unroll
            for (int k = 0; k < 2 * H::kTiles; ++k) {
              float& y = x[k / 2][nt][2 * (k % 2) + e];
              y = fmaf(y, scale, far ? flat[nt][e] : of_row[bucket[attn_clamp(away + 8 * k, 0, 2 * a.reach)]]);
              if (!there && __shfl_sync(0xffffffffu, now, k) < 0) y = as_float(0x7fffffffu);    // a page that is none
              if (8 * k >= sees) y = kNoScore;
              top[nt][e] = fmaxf(top[nt][e], y);
            }
          }
      }
      // The maximum is raised only where a score passes it by 8 (weights up to 2^8), so that hardly any step after a warp's first
      // exchanges maxima or scales its sums.
      bool more = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) more = more || top[nt][e] > m[nt][e] + 8.f;
      if (__any_sync(0xffffffffu, more)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float f[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float& y = top[nt][e];
            y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 4));
            y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 8));
            y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 16));
            y = fmaxf(y, m[nt][e]);
            f[e] = exp2_fast(m[nt][e] - (y == kNoScore ? 0.f : y));
            l[nt][e] *= f[e];
            m[nt][e] = y;
          }
#pragma unroll
          for (int c = 0; c < H::kOut; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[c][nt][e] *= f[e % 2];
        }
      }
      float base[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) base[nt][e] = m[nt][e] == kNoScore ? 0.f : m[nt][e];
#pragma unroll
      for (int k = 0; k < H::kTiles; ++k)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            x[k][nt][e] = exp2_fast(x[k][nt][e] - base[nt][e % 2]);
            l[nt][e % 2] += x[k][nt][e];
          }
      // ---- outputs
#pragma unroll
      for (int k = 0; k < H::kTiles; ++k) {
        if constexpr (H::kHalf) {
          unsigned hi[NT][2], lo[NT][2];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float u = x[k][nt][2 * e], w = x[k][nt][2 * e + 1];
              const unsigned r = pack_bf16(u, w);
              hi[nt][e] = paged_movmatrix(r);
              lo[nt][e] = paged_movmatrix(pack_bf16(u - as_float(r << 16), w - as_float(r & 0xffff0000u)));
            }
#pragma unroll
          for (int c = 0; c < H::kOut; ++c) {
            const int vc = c / (H::kVd / 2), w = c % (H::kVd / 2);
            const unsigned a0 = __byte_perm(t.v[k][0][vc][w], t.v[k][1][vc][w], 0x5410), a1 = __byte_perm(t.v[k][0][vc][w], t.v[k][1][vc][w], 0x7632);
            const unsigned a2 = __byte_perm(t.v[k][2][vc][w], t.v[k][3][vc][w], 0x5410), a3 = __byte_perm(t.v[k][2][vc][w], t.v[k][3][vc][w], 0x7632);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              paged_mma(acc[c][nt], a0, a1, a2, a3, lo[nt][0], lo[nt][1]);
              paged_mma(acc[c][nt], a0, a1, a2, a3, hi[nt][0], hi[nt][1]);
            }
          }
        } else {
          // a step of 8 positions; row g's weight of position q4 (+ 4) lies in lane 4 q4 (+ 16) + g / 2
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            FewSplit w[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const int from = 4 * q4 + 16 * e + g / 2;
                const float even = __shfl_sync(0xffffffffu, x[k][nt][2 * h], from), odd = __shfl_sync(0xffffffffu, x[k][nt][2 * h + 1], from);
                w[nt][e] = few_split(g % 2 ? odd : even);
              }
#pragma unroll
            for (int c = 0; c < H::kOut; ++c) {
              const int vc = c / 2, d = 2 * (c % 2);
              const FewSplit v0 = few_split(as_float(t.v[k][2 * h][vc][d])), v1 = few_split(as_float(t.v[k][2 * h][vc][d + 1]));
              const FewSplit v2 = few_split(as_float(t.v[k][2 * h + 1][vc][d])), v3 = few_split(as_float(t.v[k][2 * h + 1][vc][d + 1]));
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                paged_mma_tf32(acc[c][nt], v0.lo, v1.lo, v2.lo, v3.lo, w[nt][0].hi, w[nt][1].hi);
                paged_mma_tf32(acc[c][nt], v0.hi, v1.hi, v2.hi, v3.hi, w[nt][0].lo, w[nt][1].lo);
                paged_mma_tf32(acc[c][nt], v0.hi, v1.hi, v2.hi, v3.hi, w[nt][0].hi, w[nt][1].hi);
              }
            }
          }
        }
      }
      load_values(step + 1, ids);
      now = ids;
      ids = next;
    }
    // ---- the warps' results: [warp][row][DP values, maximum, sum]
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float& y = l[nt][e];
        y += __shfl_xor_sync(0xffffffffu, y, 4);
        y += __shfl_xor_sync(0xffffffffu, y, 8);
        y += __shfl_xor_sync(0xffffffffu, y, 16);
        float* to = join + (warp * H::kRows + 8 * nt + 2 * q4 + e) * (DP + 4);
#pragma unroll
        for (int c = 0; c < H::kOut; ++c) *reinterpret_cast<float2*>(to + H::value(c, lane)) = make_float2(acc[c][nt][e], acc[c][nt][2 + e]);
        if (g == 0) {
          to[DP] = m[nt][e];
          to[DP + 1] = y;
        }
      }
    ctx.sync();
    float* const factor = join + H::kWarps * H::kRows * (DP + 4);                       // [row][5]: of the warps, 1 / sum
    if (ctx.tid < H::kRows) {
      const float* from = join + ctx.tid * (DP + 4);
      constexpr int kNext = H::kRows * (DP + 4);
      float top = kNoScore, sum = 0.f;
#pragma unroll
      for (int w = 0; w < H::kWarps; ++w) top = fmaxf(top, from[w * kNext + DP]);
      const float base = top == kNoScore ? 0.f : top;
#pragma unroll
      for (int w = 0; w < H::kWarps; ++w) {
        const float f = exp2_fast(from[w * kNext + DP] - base);
        factor[5 * ctx.tid + w] = f;
        sum = fmaf(from[w * kNext + DP + 1], f, sum);
      }
      factor[5 * ctx.tid + 4] = sum == 0.f ? 0.f : 1.f / sum;
      if (part) *reinterpret_cast<float2*>(part + ctx.tid * (DP + 4) + DP) = make_float2(top, sum);
    }
    ctx.sync();
    for (int e = ctx.tid; e < left * (DP / 4); e += kThreads) {
      const int r = e / (DP / 4), c = e % (DP / 4) * 4;
      float o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < H::kWarps; ++w) {
        const float4 x = *reinterpret_cast<const float4*>(join + (w * H::kRows + r) * (DP + 4) + c);
        const float f = factor[5 * r + w];
        o[0] = fmaf(x.x, f, o[0]);
        o[1] = fmaf(x.y, f, o[1]);
        o[2] = fmaf(x.z, f, o[2]);
        o[3] = fmaf(x.w, f, o[3]);
      }
      if (part) store_four(part + r * (DP + 4) + c, o);
      else write<4>(p, b, hk, r0 + r, c, o, factor[5 * r + 4]);
    }
    ctx.sync();                                          // queries and results are written again
  }
  // N values of a row of the output from value c on
  template <int N>
  static __device__ __forceinline__ void write(const Params& p, int b, int hk, int r, int c, float (&o)[N], float over_sum) {
    const AttnParams& a = p.a;
    const int i = p.by_group.quotient(r), h = hk * a.group + r - i * a.group;
    T* out = static_cast<T*>(a.out) + (((long)b * a.lq + i) * a.heads + h) * a.dim;
#pragma unroll
    for (int e = 0; e < N; ++e) o[e] = over_sum == 0.f ? 0.f : o[e] * over_sum;
    if constexpr (N == 4) {
      if (p.wide_out) {
        if (c < a.dim) store_four(out + c, o);
        return;
      }
    }
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (c + e < a.dim) narrow(out + c + e, o[e]);
  }
};

// Joins the blocks' results of an item, ROWS rows of it to a block: thread t of a row with four columns of every kSlices-th block's part,
// the first loads on their way together.  One row to a block where there may be many parts (1 x 16384 positions, of 111 parts: 14.7 us in
// all, with one column a thread 19.8), four where there are few (32 x 1000 positions of 48 rows, of at most 8: 18.2 us and 21.6).
template <class T, int DP, int NT, int ROWS>
struct PagedJoin {
  using Params = PagedParams;
  using H = PagedShape<T, DP, NT>;
  static constexpr int kThreads = 256, kBlocks = 4, kRowThreads = kThreads / ROWS, kCols = DP / 4, kSlices = kRowThreads / kCols, kWarps = kRowThreads / 32;
  static size_t smem(long parts) { return (16 + 4 * kThreads + ROWS * (size_t)parts) * sizeof(float); }      // (most parts of an item)
  static __device__ __forceinline__ void run(const Ctx& ctx, const Params& p, unsigned char* smem) {
    const AttnParams& a = p.a;
    const int4 what = p.split[ctx.bid / (H::kRows / ROWS)];
    const int n = what.z, per_batch = a.kv_heads * p.row_blocks, b = what.x / per_batch, within = what.x - b * per_batch;
    const int hk = p.by_row_blocks.quotient(within), which = ctx.tid / kRowThreads;
    const int r = ctx.bid % (H::kRows / ROWS) * ROWS + which, r0 = (within - hk * p.row_blocks) * H::kRows, row = r0 + r, rows = a.lq * a.group;
    if (n == 0 || row - which >= rows) return;           // (a whole block)
    const int t = ctx.tid % kRowThreads, lane = t % 32, warp = t / 32;
    float *red = reinterpret_cast<float*>(smem) + 2 * kWarps * which, *outs = reinterpret_cast<float*>(smem) + 16 + 4 * kRowThreads * which;
    float* const weight = reinterpret_cast<float*>(smem) + 16 + 4 * kThreads + n * which;
    // block k's part of it: the first one's lies where what goes on is kept
    auto part = [&](int k) { return p.part + ((2L * (what.y + k) + (k == 0)) * H::kRows + r) * (DP + 4); };
    // the first columns come while the maxima do
    const int c = t % kCols * 4, slice = t / kCols;
    constexpr int kAhead = 4;
    float4 x[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (slice + k * kSlices < n) x[k] = *reinterpret_cast<const float4*>(part(slice + k * kSlices) + c);
    float m = kNoScore;
    for (int e = t; e < n; e += kRowThreads) {
      const float top = part(e)[DP];
      weight[e] = top;
      m = fmaxf(m, top);
    }
    m = lanes_max<32>(ctx, m);
    if (lane == 0) red[warp] = m;
    ctx.sync();
#pragma unroll
    for (int w = 0; w < kWarps; ++w) m = fmaxf(m, red[w]);
    const float base = m == kNoScore ? 0.f : m;
    float l = 0.f;
    for (int e = t; e < n; e += kRowThreads) {
      const float f = exp2_fast(weight[e] - base);
      weight[e] = f;
      l = fmaf(part(e)[DP + 1], f, l);
    }
    l = lanes_sum<32>(ctx, l);
    if (lane == 0) red[kWarps + warp] = l;
    ctx.sync();
    float o[4] = {0.f, 0.f, 0.f, 0.f};
    auto add = [&](const float4& y, float f) {
      o[0] = fmaf(y.x, f, o[0]);
      o[1] = fmaf(y.y, f, o[1]);
      o[2] = fmaf(y.z, f, o[2]);
      o[3] = fmaf(y.w, f, o[3]);
    };
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (slice + k * kSlices < n) add(x[k], weight[slice + k * kSlices]);
#pragma unroll 4
    for (int e = slice + kAhead * kSlices; e < n; e += kSlices) add(*reinterpret_cast<const float4*>(part(e) + c), weight[e]);
    store_vec(outs + 4 * t, o);
    ctx.sync();
    if (slice != 0 || row >= rows) return;
    l = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) l += red[kWarps + w];
    for (int e = 1; e < min(n, kSlices); ++e) add(*reinterpret_cast<const float4*>(outs + 4 * (e * kCols + t)), 1.f);
    PagedAttention<T, DP, NT, kRowsFull>::template write<4>(p, b, hk, row, c, o, l == 0.f ? 0.f : 1.f / l);
  }
};

}  // namespace s2c
#endif  // S2C_EMUL
