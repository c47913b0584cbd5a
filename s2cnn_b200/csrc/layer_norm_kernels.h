// Layer norm over the last axis, forward and backward:
//   y = (x - mean) rstd w + b,  rstd = 1 / sqrt(mean((x - mean)^2) + eps)
//   dx = rstd (g - mean(g) - x^ mean(g x^)),  g = dy w,  x^ = (x - mean) rstd;   dw = sum_rows dy x^,  db = sum_rows dy
// A row is held in the registers of a team of T threads: it is read once, the mean is taken before the squared deviations
// (no cancellation), and in the backward pass a thread owns the same columns of every row of its team, so that the weight
// sums of a team stay in its registers.  The teams of a block add theirs in a fixed order, the block's sums go to a row of
// the workspace, and a second kernel adds those rows, again in a fixed order: gradients are the same to the last bit in
// every call.
#pragma once

#include <cstring>
#include <type_traits>

#include "seq_common.h"

namespace s2c {

struct LayerNormParams {
  const void *x, *w, *b, *dy;   // w, b null: ones, zeros
  void *y, *dx;
  float* stats;                 // [rows][2]: mean, rstd (forward: null where nobody needs them)
  float* part;                  // backward: [blocks][2][cols], null where no weight gradient is asked for
  long rows;
  int cols;
  float eps;
  int wide;                     // rows of whole 16-byte pieces, all arrays aligned to them
};

// Pieces of 16 bytes where the columns are whole pieces, single elements otherwise; an unaligned array is read element by
// element into the same pieces, so that alignment changes no sum.
// T threads per row (4 ... 32 neighbouring lanes, or the whole block), each with EPT elements in pieces of VEC consecutive ones.
// A row's raw pieces are loaded one turn ahead where they fit in 16 registers (and the team is not a block of 512), and weight
// and bias are kept from turn to turn: what a warp has on its way is then two rows of 2 KB.  Bound by memory: 16384 x 1024
// bfloat16, forward and backward, 34 and 54 us without, 14 and 23 with (4.9 and 4.5 TB/s; 5 more for the sums of the blocks);
// float32, a block of 128 per row whose sums are barriers, 39 and some 53 us (3.5 and 3.8 TB/s).
template <class T_, int T, int EPT, int VEC>
struct LayerNormTeam {
  static constexpr int kThreads = T <= 32 ? 256 : T, kTeams = kThreads / T;
  static constexpr int kPieces = EPT / VEC;
  static constexpr bool kAhead = EPT * sizeof(T_) <= 64 && T < 512;
  struct Raw {                    // a thread's part of a row as it lies in memory
    typename std::conditional<(VEC > 1), Vec16, T_>::type piece[kPieces];
  };
  static S2C_D int col(int t, int v) { return (v * T + t) * VEC; }
  static S2C_D void fetch(const T_* row, int t, int cols, int wide, Raw& r) {
#pragma unroll
    for (int k = 0; k < kPieces; ++k) {
      const int c = col(t, k);
      if constexpr (VEC > 1) {
        Vec16 u = {{0u, 0u, 0u, 0u}};
        if (c < cols) {                              // cols is a multiple of VEC
          if (wide) {
            u = *reinterpret_cast<const Vec16*>(row + c);
          } else {
            T_ e[VEC];
#pragma unroll
            for (int i = 0; i < VEC; ++i) e[i] = row[c + i];
            std::memcpy(&u, e, 16);
          }
        }
        r.piece[k] = u;
      } else {
        T_ zero = {};
        r.piece[k] = c < cols ? row[c] : zero;
      }
    }
  }
  static S2C_D void open(const Raw& r, float (&v)[EPT]) {
#pragma unroll
    for (int k = 0; k < kPieces; ++k) {
      if constexpr (VEC > 1) {
        float e[VEC];
        load_vec(reinterpret_cast<const T_*>(&r.piece[k]), e);
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[k * VEC + i] = e[i];
      } else {
        v[k] = widen(r.piece[k]);
      }
    }
  }
  static S2C_D void store(T_* row, int t, int cols, int wide, const float (&v)[EPT]) {
#pragma unroll
    for (int k = 0; k < kPieces; ++k) {
      const int c = col(t, k);
      if (c >= cols) continue;
      if constexpr (VEC > 1) {
        float e[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) e[i] = v[k * VEC + i];
        if (wide) {
          store_vec(row + c, e);
        } else {
#pragma unroll
          for (int i = 0; i < VEC; ++i) narrow(row + c + i, e[i]);
        }
      } else {
        narrow(row + c, v[k]);
      }
    }
  }
  // sum over the team; `red` holds one float per warp (two buffers in turn, so that one barrier a sum is enough)
  static S2C_D float sum(const Ctx& ctx, float v, float* red) {
    v = lanes_sum<(T < 32 ? T : 32)>(ctx, v);
    if constexpr (T <= 32) return v;
    if (ctx.tid % 32 == 0) red[ctx.tid / 32] = v;
    ctx.sync();
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < T / 32; ++i) s += red[i];
    return s;
  }
};

template <class T_, int T, int EPT, int VEC>
struct LayerNormFwd : LayerNormTeam<T_, T, EPT, VEC> {
  using Team = LayerNormTeam<T_, T, EPT, VEC>;
  using Raw = typename Team::Raw;
  using Params = LayerNormParams;
  static constexpr int kBlocks = 1024 / Team::kThreads / (EPT > 16 ? 2 : 1);
  static size_t smem() { return T <= 32 ? 0 : 2 * (T / 32) * sizeof(float); }
  static S2C_D void run(const Ctx& ctx, const Params& p, unsigned char* smem) {
    const int team = ctx.tid / T, t = ctx.tid % T;
    float* red = reinterpret_cast<float*>(smem);
    const long per = (long)ctx.nblk * Team::kTeams;
    auto fetch_row = [&](long r, Raw& raw) { Team::fetch(static_cast<const T_*>(p.x) + (r < p.rows ? r : 0) * p.cols, t, p.cols, p.wide, raw); };
    Raw now, next, w, b;
    fetch_row((long)ctx.bid * Team::kTeams + team, now);
    if (Team::kAhead && p.w) Team::fetch(static_cast<const T_*>(p.w), t, p.cols, p.wide, w);
    if (Team::kAhead && p.b) Team::fetch(static_cast<const T_*>(p.b), t, p.cols, p.wide, b);
    // (every team takes the same number of turns: lanes meet in shuffles, and in the emulation in block barriers)
    for (long r0 = (long)ctx.bid * Team::kTeams; r0 < p.rows; r0 += per) {
      const long r = r0 + team;
      const bool on = r < p.rows, more = r0 + per < p.rows;
      if (Team::kAhead && more) fetch_row(r + per, next);
      float x[EPT];
      Team::open(now, x);
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < EPT; ++i) s += x[i];
      const float mean = Team::sum(ctx, s, red) / (float)p.cols;
      s = 0.f;
#pragma unroll
      for (int i = 0; i < EPT; ++i) {
        const float d = Team::col(t, i / VEC) < p.cols ? x[i] - mean : 0.f;
        s += d * d;
      }
      const float rstd = inv_sqrt(Team::sum(ctx, s, red + T / 32) / (float)p.cols + p.eps);
      float v[EPT];
      if (p.w) {
        if (!Team::kAhead) Team::fetch(static_cast<const T_*>(p.w), t, p.cols, p.wide, w);
        Team::open(w, v);
#pragma unroll
        for (int i = 0; i < EPT; ++i) x[i] = (x[i] - mean) * rstd * v[i];
      } else {
#pragma unroll
        for (int i = 0; i < EPT; ++i) x[i] = (x[i] - mean) * rstd;
      }
      if (p.b) {
        if (!Team::kAhead) Team::fetch(static_cast<const T_*>(p.b), t, p.cols, p.wide, b);
        Team::open(b, v);
#pragma unroll
        for (int i = 0; i < EPT; ++i) x[i] += v[i];
      }
      if (on) {
        Team::store(static_cast<T_*>(p.y) + r * p.cols, t, p.cols, p.wide, x);
        if (p.stats && t == 0) {
          p.stats[2 * r] = mean;
          p.stats[2 * r + 1] = rstd;
        }
      }
      if (!Team::kAhead && more) fetch_row(r + per, next);
      now = next;
    }
  }
};

template <class T_, int T, int EPT, int VEC>
struct LayerNormBwd : LayerNormTeam<T_, T, EPT, VEC> {
  using Team = LayerNormTeam<T_, T, EPT, VEC>;
  using Raw = typename Team::Raw;
  using Params = LayerNormParams;
  static constexpr int kBlocks = EPT * sizeof(T_) <= 32 ? 512 / Team::kThreads : Team::kThreads == 128 ? 2 : 1;   // (255 registers for the larger)
  static size_t smem() { return T <= 32 ? (size_t)EPT * T * 2 * sizeof(float) : 4 * (T / 32) * sizeof(float); }
  static S2C_D void run(const Ctx& ctx, const Params& p, unsigned char* smem) {
    const int team = ctx.tid / T, t = ctx.tid % T;
    float* red = reinterpret_cast<float*>(smem);
    float dw[EPT], db[EPT];
#pragma unroll
    for (int i = 0; i < EPT; ++i) { dw[i] = 0.f; db[i] = 0.f; }
    const long per = (long)ctx.nblk * Team::kTeams;
    Raw now_x, now_g, next_x, next_g, w;
    float2 stat, next_stat;
    auto fetch_row = [&](long r, Raw& x, Raw& g, float2& st) {
      const long row = r < p.rows ? r : 0;
      Team::fetch(static_cast<const T_*>(p.x) + row * p.cols, t, p.cols, p.wide, x);
      Team::fetch(static_cast<const T_*>(p.dy) + row * p.cols, t, p.cols, p.wide, g);
      st = make_float2(p.stats[2 * row], r < p.rows ? p.stats[2 * row + 1] : 0.f);
    };
    if ((long)ctx.bid * Team::kTeams < p.rows) fetch_row((long)ctx.bid * Team::kTeams + team, now_x, now_g, stat);
    if (p.w) Team::fetch(static_cast<const T_*>(p.w), t, p.cols, p.wide, w);
    int turn = 0;
    for (long r0 = (long)ctx.bid * Team::kTeams; r0 < p.rows; r0 += per, turn ^= 1) {
      const long r = r0 + team;
      const bool on = r < p.rows, more = r0 + per < p.rows;
      if (Team::kAhead && more) fetch_row(r + per, next_x, next_g, next_stat);
      float x[EPT], g[EPT], v[EPT];
      Team::open(now_x, x);
      Team::open(now_g, g);
      if (p.w) Team::open(w, v);
      const float mean = stat.x, rstd = stat.y;
      float s0 = 0.f, s1 = 0.f;
#pragma unroll
      for (int i = 0; i < EPT; ++i) {
        x[i] = (x[i] - mean) * rstd;
        if (!on) g[i] = 0.f;
        dw[i] += g[i] * x[i];
        db[i] += g[i];
        if (p.w) g[i] *= v[i];        // (beyond the row's end g is 0)
        s0 += g[i];
        s1 += g[i] * x[i];
      }
      if (p.dx) {
        s0 = Team::sum(ctx, s0, red + (2 * turn) * (T / 32)) / (float)p.cols;
        s1 = Team::sum(ctx, s1, red + (2 * turn + 1) * (T / 32)) / (float)p.cols;
#pragma unroll
        for (int i = 0; i < EPT; ++i) x[i] = rstd * (g[i] - s0 - x[i] * s1);
        if (on) Team::store(static_cast<T_*>(p.dx) + r * p.cols, t, p.cols, p.wide, x);
      }
      if (!Team::kAhead && more) fetch_row(r + per, next_x, next_g, next_stat);
      now_x = next_x;
      now_g = next_g;
      stat = next_stat;
    }
    if (!p.part) return;
    if constexpr (T <= 32) {          // the teams of a warp, then the warps one after another in shared memory
#pragma unroll
      for (int m = T; m < 32; m *= 2)
#pragma unroll
        for (int i = 0; i < EPT; ++i) {
          dw[i] += ctx.shfl_xor(dw[i], m);
          db[i] += ctx.shfl_xor(db[i], m);
        }
      ctx.sync();
      for (int k = 0; k < 8; ++k) {
        if (ctx.tid / 32 == k && ctx.tid % 32 < T) {
#pragma unroll
          for (int i = 0; i < EPT; ++i) {
            float* at = red + 2 * (i * T + t);
            at[0] = (k ? at[0] : 0.f) + dw[i];
            at[1] = (k ? at[1] : 0.f) + db[i];
          }
        }
        ctx.sync();
      }
      if (team != 0) return;
#pragma unroll
      for (int i = 0; i < EPT; ++i) {
        dw[i] = red[2 * (i * T + t)];
        db[i] = red[2 * (i * T + t) + 1];
      }
    }
    float* out = p.part + (long)ctx.bid * 2 * p.cols;
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
      const int c = Team::col(t, i / VEC) + i % VEC;
      if (Team::col(t, i / VEC) < p.cols) {
        out[c] = dw[i];
        out[p.cols + c] = db[i];
      }
    }
  }
};

// dw and db: the sums of the blocks' rows.  A block takes 32 of the 2 cols columns; its 8 warps take every eighth row, and
// their sums are added in order.
struct LayerNormSumParams {
  const float* part;
  void *dw, *db;          // null: not asked for
  int blocks, cols;
};
template <class T_>
struct LayerNormSum {
  using Params = LayerNormSumParams;
  static constexpr int kThreads = 256, kBlocks = 4;
  static S2C_D void run(const Ctx& ctx, const Params& p, unsigned char* smem) {
    float* red = reinterpret_cast<float*>(smem);      // [8][32]
    const int lane = ctx.tid % 32, warp = ctx.tid / 32, c = ctx.bid * 32 + lane;
    float s = 0.f;
    if (c < 2 * p.cols) {
      float part[4] = {0.f, 0.f, 0.f, 0.f};           // four loads on the way
      int k = warp;
      for (; k + 24 < p.blocks; k += 32)
#pragma unroll
        for (int u = 0; u < 4; ++u) part[u] += p.part[(long)(k + 8 * u) * 2 * p.cols + c];
      for (; k < p.blocks; k += 8) part[0] += p.part[(long)k * 2 * p.cols + c];
      s = (part[0] + part[1]) + (part[2] + part[3]);
    }
    red[warp * 32 + lane] = s;
    ctx.sync();
    if (warp != 0 || c >= 2 * p.cols) return;
    for (int k = 1; k < 8; ++k) s += red[k * 32 + lane];
    T_* out = static_cast<T_*>(c < p.cols ? p.dw : p.db);
    if (out) narrow(out + (c < p.cols ? c : c - p.cols), s);
  }
};

}  // namespace s2c
