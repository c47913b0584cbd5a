// Heads of queries and keys: norm and rotation by position in one pass, forward and backward, and the same with the keys, and values
// beside them, written to pages of a cache (kept_pages.h).
//
//   x^ = x rstd, rstd = 1 / sqrt(mean(x^2) + eps) over a head's values;  z = x^ w            (without a norm: z = x)
//   y_a = mu (z_a cos t - z_b sin t),  y_b = mu (z_a sin t + z_b cos t),  t = position f      (pairs (a, b), mu the magnitude)
//   backward: g the gradient of z (the rotation by -t of that of y, times mu), h = g w:
//   dx = rstd (h - x^ mean(h x^)),  dw = sum over all heads g x^;  rstd is computed again from x: nothing is stored
//
// Angles.  t of a position in the hundred thousands loses its digits in float32.  The frequency of each pair is kept as a fraction
// of a turn in 64 bits of fixed point, F = round(2^64 f / 2 pi mod 2^64); position F modulo 2^64 is then the angle modulo whole
// turns by one integer product, whatever the position (also a negative one).  What is lost is f / 2 pi's own rounding, a relative
// 2^-52, times the position.  The nearest quarter turn is taken off in integers, the rest (an eighth at most) goes through
// the Taylor series of sine and cosine to x^9 and x^10, whose first terms left out are below 2e-9 and 2e-10 there.
//
// A team of 4, 8 or 16 neighbouring lanes holds a head of up to 32, 64 or 128 values, four pairs to a lane, and takes several heads of
// one position, which share the four sines and cosines and, times the weights, the pairs' factors.  Blocks are dealt to queries, keys and
// values, so that a lane has one weight.
//
// Bound by instructions and their latencies with 16 warps an SM, half of what memory would take: 4 x 4096 positions, 20 heads of 128
// bfloat16 values, forward 36 us (4.7 TB/s), without a norm 31 (5.4); backward 53 us (4.8), and 4 for the sums of the blocks; a first pass
// of 4 x 2049 ragged positions, 20 heads of 64, into pages 12.6.  Two blocks an SM with four heads of a turn loaded ahead (two in float32
// and backward).  Others, when this was chosen: three blocks with two heads 36.6 us where this had 37, but 14.0 for the first pass, where
// this had 12.3; backward with one head a turn 111 where this had 94 for both passes, with one and three blocks 97.  Instances of single
// values with four heads ahead keep up to 274 bytes a thread of them in local memory (bfloat16, heads of 65 to 128 values).
#pragma once

#include <cstring>
#include <type_traits>

#include "kept_pages.h"
#include "seq_common.h"

namespace s2c {

struct HeadKind {                // queries, keys or values
  const void* x;                 // [batch][length][heads][dim]
  const void* w;                 // norm weight, null: ones
  const void* dy;                // backward: gradient of out, contiguous
  void* out;                     // contiguous; the gradient of x in the backward pass; null: pages
  long stride[3], pstride[3];    // of x; of the pages (page, position, head)
  int heads, blocks;             // blocks of this kind
  int span;                      // heads of a unit
  Divisor spans;                 // units of a position
  int turn;                      // norm and rotation (queries, keys)
};
struct HeadParams {
  HeadKind kind[3];
  const double* frequencies;     // radians per position
  const int *positions, *lengths;
  float* part;                   // backward: [blocks][dim], sums of the weight gradients
  PageTable pages;
  Divisor by_length;
  int batch, length, dim, pairs, interleaved, norm;
  int each, first;               // positions: one per position of a sequence, or its first; null: `first` for all
  float eps, magnitude, over_dim;
};

// f in radians per position as a fraction of a turn, in units of 2^-64
S2C_D unsigned long long turn_units(double f) {
  double t = f * 0.15915494309189533577;
  t -= floor(t);                                             // [0, 1), or 1 by rounding; NaN and infinities: the magnitude tells
  return t >= 0. && t < 1. ? (unsigned long long)(t * 18446744073709551616.) : 0ull;
}
// cosine and sine of `turns`, in units of 2^-64
S2C_D void turn_cos_sin(unsigned long long turns, float& c, float& s) {
  const unsigned high = (unsigned)(turns >> 32), quarter = (high + 0x20000000u) >> 30;
  const float x = (float)(int)(high - (quarter << 30)) * 1.4629180792671596e-9f;      // 2 pi 2^-32
  const float y = x * x;
  float a = fmaf(y, 2.7557319223985893e-6f, -1.9841269841269841e-4f);
  a = fmaf(y, a, 8.3333333333333333e-3f);
  a = fmaf(y, a, -1.6666666666666667e-1f);
  a = fmaf(y * x, a, x);
  float b = fmaf(y, -2.7557319223985888e-7f, 2.4801587301587302e-5f);
  b = fmaf(y, b, -1.3888888888888889e-3f);
  b = fmaf(y, b, 4.1666666666666664e-2f);
  b = fmaf(y, b, -0.5f);
  b = fmaf(y, b, 1.f);
  const bool swap = quarter & 1;
  const float c0 = swap ? a : b, s0 = swap ? b : a;
  c = (quarter + 1) & 2 ? -c0 : c0;
  s = quarter & 2 ? -s0 : s0;
}

S2C_D int min_of(int a, int b) { return a < b ? a : b; }

// How the values of a head lie to a lane: one by one, or in two pieces of four, the first values of four pairs
// and their second ones (halves) or eight consecutive values (neighbours).  Pieces off their boundaries (apart) are read and
// written value by value, so that alignment changes no sum.
enum HeadRows : int { kHeadByValue, kHeadHalves, kHeadNeighbours, kHeadHalvesApart, kHeadNeighboursApart };

// NP: two pairs of a lane each.  Pieces: NP = 2, pairs 4 t ... 4 t + 3; by value: pairs t, t + LANES, ..., so that what a team reads or writes
// at a time lies together (3601 positions, 16 heads of 25 float32 values: 6.6 us; in the order of pieces, whose stores are single
// values 32 bytes apart, 11.0).
template <class T, int LANES, int ROWS, int NP>
struct HeadTeam {
  static constexpr int kThreads = 256, kTeams = kThreads / LANES, kPairs = 2 * NP;
  static constexpr bool kPieces = ROWS != kHeadByValue, kWide = ROWS == kHeadHalves || ROWS == kHeadNeighbours;
  static constexpr bool kNext = ROWS == kHeadNeighbours || ROWS == kHeadNeighboursApart;
  using Four = typename std::conditional<sizeof(T) == 2, Vec8, Vec16>::type;
  struct Wide {
    Four piece[2];
  };
  struct Narrow {
    float v[2][kPairs];
  };
  using Raw = typename std::conditional<kPieces, Wide, Narrow>::type;      // a lane's values as they were loaded

  int t;                          // lane of the team
  int at[2][kPieces ? 1 : kPairs];   // where the first and second values of its pairs lie, or its pieces; -1: none
  unsigned turned;                // bit e: pair e is turned

  static S2C_D int pair(int t, int e) { return kPieces ? 4 * t + e : t + LANES * e; }
  // where value k of pair i lies: what is not turned pairs up as what is
  static S2C_D int place(const HeadParams& p, int i, int k) {
    if (p.interleaved) return 2 * i + k < p.dim ? 2 * i + k : -1;
    const int rest = p.dim - 2 * p.pairs, low = (rest + 1) / 2, r = i - p.pairs;
    return r < 0 ? i + k * p.pairs : r < (k ? rest - low : low) ? 2 * p.pairs + k * low + r : -1;
  }
  S2C_D HeadTeam(const HeadParams& p, int lane) : t(lane), turned(0) {
#pragma unroll
    for (int e = 0; e < kPairs; ++e)
      if (pair(t, e) < p.pairs) turned |= 1u << e;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if constexpr (kPieces) {
        at[k][0] = kNext ? place(p, pair(t, 2 * k), 0) : place(p, pair(t, 0), k);
      } else {
#pragma unroll
        for (int e = 0; e < kPairs; ++e) at[k][e] = place(p, pair(t, e), k);
      }
    }
  }
  // (a lane's piece behind the head: the head's first one, which counts in no sum and is stored nowhere)
  S2C_D void fetch(const T* x, Raw& r) const {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if constexpr (kPieces) {
        const T* from = x + (at[k][0] >= 0 ? at[k][0] : 0);
        if constexpr (kWide) {
          r.piece[k] = *reinterpret_cast<const Four*>(from);
        } else {
          const T v[4] = {from[0], from[1], from[2], from[3]};
          std::memcpy(&r.piece[k], v, sizeof(v));
        }
      } else {
#pragma unroll
        for (int e = 0; e < kPairs; ++e) r.v[k][e] = at[k][e] >= 0 ? widen(x[at[k][e]]) : 0.f;
      }
    }
  }
  // as pairs (a[e], b[e])
  S2C_D void open(const Raw& r, float2 (&a)[NP], float2 (&b)[NP]) const {
    if constexpr (kPieces) {
      float v[2][4];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        load_four(reinterpret_cast<const T*>(&r.piece[k]), v[k]);
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        a[e] = kNext ? make_float2(v[e][0], v[e][2]) : make_float2(v[0][2 * e], v[0][2 * e + 1]);
        b[e] = kNext ? make_float2(v[e][1], v[e][3]) : make_float2(v[1][2 * e], v[1][2 * e + 1]);
      }
    } else {
#pragma unroll
      for (int e = 0; e < NP; ++e) {
        a[e] = make_float2(r.v[0][2 * e], r.v[0][2 * e + 1]);
        b[e] = make_float2(r.v[1][2 * e], r.v[1][2 * e + 1]);
      }
    }
  }
  S2C_D void store(T* y, const float2 (&a)[NP], const float2 (&b)[NP]) const {
    if constexpr (kPieces) {
      float v[2][4];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        v[0][2 * e] = kNext ? (e ? a[0].y : a[0].x) : a[e].x;
        v[0][2 * e + 1] = kNext ? (e ? b[0].y : b[0].x) : a[e].y;
        v[1][2 * e] = kNext ? (e ? a[1].y : a[1].x) : b[e].x;
        v[1][2 * e + 1] = kNext ? (e ? b[1].y : b[1].x) : b[e].y;
      }
#pragma unroll
      for (int k = 0; k < 2; ++k)
        if (at[k][0] >= 0) {
          if constexpr (kWide) {
            store_four(y + at[k][0], v[k]);
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) narrow(y + at[k][0] + e, v[k][e]);
          }
        }
    } else {
#pragma unroll
      for (int e = 0; e < kPairs; ++e) {
        if (at[0][e] >= 0) narrow(y + at[0][e], e % 2 ? a[e / 2].y : a[e / 2].x);
        if (at[1][e] >= 0) narrow(y + at[1][e], e % 2 ? b[e / 2].y : b[e / 2].x);
      }
    }
  }
  // What is the same for all teams of a block, in shared memory: a unit's sines and cosines are made from it, and a lane's registers
  // are for heads (with it in registers, and the kind of heads, 110 were taken before the first head).
  struct alignas(16) Shared {
    float w[2][kPairs][LANES];    // weights of the first and second values of a lane's pairs (as long as a head, or longer)
    HeadKind kind;
    float mu[kPairs][LANES];      // magnitudes: 1 where nothing is turned, NaN where the frequency is no number
    unsigned long long f[kPairs][LANES];      // frequencies
  };
  // FORWARD: the magnitude goes with the weights; otherwise with sines and cosines
  template <bool FORWARD>
  static S2C_D void share(const Ctx& ctx, const HeadParams& p, const HeadKind& kind, Shared* to) {
    if (ctx.tid < LANES * kPairs) {
      const int lane = ctx.tid % LANES, e = ctx.tid / LANES, i = pair(lane, e);
      const double f = kind.turn && i < p.pairs ? p.frequencies[i] : 0.;
      const float mu = f - f != 0. ? as_float(0x7fffffffu) : i < p.pairs ? p.magnitude : 1.f;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int c = place(p, i, k);
        to->w[k][e][lane] = (kind.w && c >= 0 ? widen(static_cast<const T*>(kind.w)[c]) : 1.f) * (FORWARD ? mu : 1.f);
      }
      to->mu[e][lane] = mu;
      to->f[e][lane] = turn_units(f);
    }
    if (ctx.tid == ctx.nthr - 1) to->kind = kind;
    ctx.sync();
  }
  // cosines and sines of the pairs; of what is not turned 1 and 0
  template <bool FORWARD>
  S2C_D void angles(const Shared* s, long position, float2 (&c)[NP], float2 (&si)[NP]) const {
#pragma unroll
    for (int e = 0; e < NP; ++e) {
      turn_cos_sin(s->f[2 * e][t] * (unsigned long long)position, c[e].x, si[e].x);
      turn_cos_sin(s->f[2 * e + 1][t] * (unsigned long long)position, c[e].y, si[e].y);
      if (!FORWARD) {
        const float2 mu = make_float2(s->mu[2 * e][t], s->mu[2 * e + 1][t]);
        c[e] = mul2(c[e], mu);
        si[e] = mul2(si[e], mu);
      }
    }
  }
  S2C_D float2 weights(const Shared* s, int k, int e) const { return make_float2(s->w[k][2 * e][t], s->w[k][2 * e + 1][t]); }
  // sum over a head of a x + b y, in every lane
  S2C_D float product(const Ctx& ctx, const float2 (&a)[NP], const float2 (&b)[NP], const float2 (&x)[NP], const float2 (&y)[NP]) const {
    float2 sum[NP];
#pragma unroll
    for (int e = 0; e < NP; ++e) sum[e] = fma2(b[e], y[e], mul2(a[e], x[e]));
    if constexpr (kPieces) {      // without the pieces behind the head (by selection: a factor of 0 would make NaN of what overflows there)
      const bool in = at[0][0] >= 0;
      const float first = sum[0].x + sum[0].y, second = sum[1].x + sum[1].y;
      return lanes_sum<LANES>(ctx, (in ? first : 0.f) + ((kNext ? at[1][0] >= 0 : in) ? second : 0.f));
    } else {
      float s = sum[0].x + sum[0].y;
#pragma unroll
      for (int e = 1; e < NP; ++e) s += sum[e].x + sum[e].y;
      return lanes_sum<LANES>(ctx, s);
    }
  }
  // A unit: `span` neighbouring heads of one position.
  struct Unit {
    const T* x;                   // its first head
    long to, at;                  // where that lies among contiguous heads; position
    int left, b, i;               // heads of the kind from the first one on; sequence and row of it
    bool on;
  };
  static S2C_D Unit unit(const HeadParams& p, const HeadKind& kind, long u, long units) {
    Unit n;
    n.on = u < units;
    const unsigned v = n.on ? (unsigned)u : 0u, row = kind.spans.quotient(v);
    const int h = (int)(v - row * kind.spans.d) * kind.span;
    n.b = (int)p.by_length.quotient(row);
    n.i = (int)row - n.b * p.length;
    n.left = kind.heads - h;
    n.x = static_cast<const T*>(kind.x) + n.b * kind.stride[0] + n.i * kind.stride[1] + h * kind.stride[2];
    n.to = ((long)row * kind.heads + h) * p.dim;
    n.at = !p.positions ? (long)p.first + n.i : p.each ? p.positions[row] : (long)p.positions[n.b] + n.i;
    return n;
  }
};

// Per lane: GROUP heads loaded while the GROUP before them are worked on, four sines and cosines for all heads of a unit.
template <class T, int LANES, int ROWS, int NP, int GROUP>
struct HeadForward {
  using Team = HeadTeam<T, LANES, ROWS, NP>;
  using Unit = typename Team::Unit;
  using Raw = typename Team::Raw;
  using Params = HeadParams;
  static constexpr int kThreads = Team::kThreads, kBlocks = 2;
  static constexpr size_t kSmem = sizeof(typename Team::Shared);
  static S2C_D void run(const Ctx& ctx, const Params& p, unsigned char* smem) {
    int which = 0, bid = ctx.bid;
    while (which < 2 && bid >= p.kind[which].blocks) bid -= p.kind[which++].blocks;
    typename Team::Shared* const shared = reinterpret_cast<typename Team::Shared*>(smem);
    const HeadKind& kind = shared->kind;
    Team::template share<true>(ctx, p, p.kind[which], shared);
    const Team team(p, ctx.tid % LANES);
    const long units = (long)p.batch * p.length * kind.spans.d, per = (long)kind.blocks * Team::kTeams, mine = ctx.tid / LANES;
    // values that are not turned: an infinity times a sine of 0 would be none (in a norm's head nothing is left of it)
    const bool rest = 2 * p.pairs < p.dim && !p.norm, turn = kind.turn;
    const int span = kind.span;
    long step = kind.stride[2];
    Raw raw[GROUP];
    auto fetch = [&](const T* x, int left) {            // (beyond the last head: the first of the group again)
#pragma unroll
      for (int g = 0; g < GROUP; ++g) team.fetch(x + (g < left ? g * step : 0), raw[g]);
    };
    long u0 = (long)bid * Team::kTeams;
    // the next unit, its heads, and in a store its page, while the heads before are worked on
    Unit now;
    bool next_filled = true, next_work = true;          // (rows that are not filled: a warp of them alone has nothing to do)
    int next_page = 0;
    auto open_unit = [&](long u) {
      now = Team::unit(p, kind, u, units);
      if (p.pages.table) {
        next_filled = !p.lengths || now.i < p.lengths[now.b];
        next_work = ctx.warp_any(next_filled && now.on);
        if (next_work) next_page = p.pages.of(now.b, now.at);
        // A row that is not filled need not be there: what is read in its place lies in shared memory.
        step = next_filled && now.on ? kind.stride[2] : 0;
        if (!(next_filled && now.on)) now.x = reinterpret_cast<const T*>(shared->w);
      }
      if (next_work) fetch(now.x, now.left);
    };
    open_unit(u0 + mine);
    for (; u0 < units; u0 += per) {                     // (every team takes the same number of turns)
      // where the unit's heads go (null: nowhere), and what is said of a row that has no value
      const bool filled = next_filled, work = next_work;
      const int page = next_page;
      T* y = nullptr;
      long y_step = p.dim;
      if (now.on && kind.out) {
        y = static_cast<T*>(kind.out) + now.to;
      } else if (now.on && filled && page >= 0) {
        y_step = kind.pstride[2];
        y = static_cast<T*>(p.pages.array[which - 1]) + page * kind.pstride[0] + (now.at & (p.pages.page - 1)) * kind.pstride[1] + (kind.heads - now.left) * y_step;
      }
      // y_a = x_a k0 + x_b k1, y_b = x_a k2 + x_b k3
      float2 k0[NP], k1[NP], k2[NP], k3[NP];
      if (turn && work) {
        float2 c[NP], s[NP];
        team.template angles<true>(shared, now.at, c, s);
#pragma unroll
        for (int e = 0; e < NP; ++e) {
          const float2 x = team.weights(shared, 0, e), z = team.weights(shared, 1, e);
          k0[e] = mul2(x, c[e]);
          k1[e] = mul2(z, make_float2(-s[e].x, -s[e].y));
          k2[e] = mul2(x, s[e]);
          k3[e] = mul2(z, c[e]);
        }
      }
      int left = now.left;
      const T* x = now.x;
      for (int n = 0; n < span; n += GROUP, left -= GROUP) {
        Raw old[GROUP];
#pragma unroll
        for (int g = 0; g < GROUP; ++g) old[g] = raw[g];
        if (n + GROUP < span) {
          if (left > GROUP && work) fetch(x += GROUP * step, left - GROUP);
        } else {
          open_unit(u0 + per + mine);
        }
#pragma unroll
        for (int g = 0; g < GROUP; ++g) {
          float2 a[NP], b[NP];
          team.open(old[g], a, b);
          if (turn && work) {
            if (p.norm) {
              const float rstd = inv_sqrt(fmaf(team.product(ctx, a, b, a, b), p.over_dim, p.eps));
              const float2 r2 = make_float2(rstd, rstd);
#pragma unroll
              for (int e = 0; e < NP; ++e) {
                a[e] = mul2(a[e], r2);
                b[e] = mul2(b[e], r2);
              }
            }
#pragma unroll
            for (int e = 0; e < NP; ++e) {
              const float2 u = a[e], v = b[e];
              a[e] = fma2(u, k0[e], mul2(v, k1[e]));
              b[e] = fma2(u, k2[e], mul2(v, k3[e]));
              if (rest) {
                if (!(team.turned >> 2 * e & 1)) a[e].x = u.x * k0[e].x, b[e].x = v.x * k3[e].x;
                if (!(team.turned >> 2 * e & 2)) a[e].y = u.y * k0[e].y, b[e].y = v.y * k3[e].y;
              }
            }
          }
          if (!filled || page < 0) {                    // a row that is not filled, and a query whose key has no place
            const float none = filled ? as_float(0x7fffffffu) : 0.f;
#pragma unroll
            for (int e = 0; e < NP; ++e) a[e] = b[e] = make_float2(none, none);
          }
          if (y && g < left && n + g < span) team.store(y + g * y_step, a, b);
        }
        if (y) y += GROUP * y_step;
      }
    }
  }
};

template <class T, int LANES, int ROWS, int NP, int GROUP>
struct HeadBackward {
  using Team = HeadTeam<T, LANES, ROWS, NP>;
  using Unit = typename Team::Unit;
  using Raw = typename Team::Raw;
  using Params = HeadParams;
  static constexpr int kThreads = Team::kThreads, kBlocks = 2;
  static constexpr size_t kSmem = sizeof(typename Team::Shared) + 8 * LANES * sizeof(float);
  static S2C_D void run(const Ctx& ctx, const Params& p, unsigned char* smem) {
    const int which = ctx.bid >= p.kind[0].blocks ? 1 : 0;
    const int bid = ctx.bid - (which ? p.kind[0].blocks : 0);
    typename Team::Shared* const shared = reinterpret_cast<typename Team::Shared*>(smem);
    const HeadKind& kind = shared->kind;
    Team::template share<false>(ctx, p, p.kind[which], shared);
    const Team team(p, ctx.tid % LANES);
    const long units = (long)p.batch * p.length * kind.spans.d, per = (long)kind.blocks * Team::kTeams, mine = ctx.tid / LANES;
    const bool rest = 2 * p.pairs < p.dim;
    const int span = kind.span;
    const long step = kind.stride[2];
    Raw raw_x[GROUP], raw_d[GROUP];
    auto fetch = [&](const T* x, long to, int left) {
      const T* dy = static_cast<const T*>(kind.dy) + to;
#pragma unroll
      for (int g = 0; g < GROUP; ++g) {
        team.fetch(dy + (g < left ? g * p.dim : 0), raw_d[g]);
        if (p.norm) team.fetch(x + (g < left ? g * step : 0), raw_x[g]);
      }
    };
    long u0 = (long)bid * Team::kTeams;
    Unit now = Team::unit(p, kind, u0 + mine, units);
    fetch(now.x, now.to, now.left);
    float2 da[NP], db[NP];
#pragma unroll
    for (int e = 0; e < NP; ++e) da[e] = db[e] = make_float2(0.f, 0.f);
    for (; u0 < units; u0 += per) {
      float2 c[NP], s[NP], w[2][NP];
      team.template angles<false>(shared, now.at, c, s);
#pragma unroll
      for (int e = 0; e < NP; ++e) {
        w[0][e] = team.weights(shared, 0, e);
        w[1][e] = team.weights(shared, 1, e);
      }
      const bool on = now.on;
      const T* x = now.x;
      long to = now.to;
      int left = now.left;
      for (int n = 0; n < span; n += GROUP, left -= GROUP, to += GROUP * p.dim) {
        Raw old_x[GROUP], old_d[GROUP];
#pragma unroll
        for (int g = 0; g < GROUP; ++g) {
          old_x[g] = raw_x[g];
          old_d[g] = raw_d[g];
        }
        if (n + GROUP < span) {
          if (left > GROUP) fetch(x += GROUP * step, to + GROUP * p.dim, left - GROUP);
        } else {
          now = Team::unit(p, kind, u0 + per + mine, units);
          fetch(now.x, now.to, now.left);
        }
#pragma unroll
        for (int g = 0; g < GROUP; ++g) {
          const bool in = on && g < left && n + g < span;
          float2 ga[NP], gb[NP];
          team.open(old_d[g], ga, gb);
#pragma unroll
          for (int e = 0; e < NP; ++e) {
            const float2 u = ga[e], v = gb[e];
            ga[e] = fma2(u, c[e], mul2(v, s[e]));
            gb[e] = fma2(v, c[e], mul2(u, make_float2(-s[e].x, -s[e].y)));
            if (rest) {
              if (!(team.turned >> 2 * e & 1)) ga[e].x = u.x, gb[e].x = v.x;
              if (!(team.turned >> 2 * e & 2)) ga[e].y = u.y, gb[e].y = v.y;
            }
          }
          if (p.norm) {
            float2 xa[NP], xb[NP];
            team.open(old_x[g], xa, xb);
            const float rstd = inv_sqrt(fmaf(team.product(ctx, xa, xb, xa, xb), p.over_dim, p.eps));
            const float2 r2 = make_float2(rstd, rstd);
#pragma unroll
            for (int e = 0; e < NP; ++e) {
              xa[e] = mul2(xa[e], r2);
              xb[e] = mul2(xb[e], r2);
              if (in) {
                da[e] = fma2(ga[e], xa[e], da[e]);
                db[e] = fma2(gb[e], xb[e], db[e]);
              }
              ga[e] = mul2(ga[e], w[0][e]);
              gb[e] = mul2(gb[e], w[1][e]);
            }
            const float dot = -team.product(ctx, ga, gb, xa, xb) * p.over_dim;
            const float2 dot2 = make_float2(dot, dot);
#pragma unroll
            for (int e = 0; e < NP; ++e) {
              ga[e] = mul2(r2, fma2(xa[e], dot2, ga[e]));
              gb[e] = mul2(r2, fma2(xb[e], dot2, gb[e]));
            }
          }
          if (in && kind.out) team.store(static_cast<T*>(kind.out) + to + g * p.dim, ga, gb);
        }
      }
    }
    if (!p.part || !kind.w) return;                 // (a whole block)
    // the teams of a warp, then the warps in their order: [value of a pair][pair][lane]
    float* red = reinterpret_cast<float*>(smem + sizeof(typename Team::Shared));
    constexpr int kPairs = Team::kPairs;
    float sums[2][kPairs];
#pragma unroll
    for (int e = 0; e < kPairs; ++e) {
      sums[0][e] = e % 2 ? da[e / 2].y : da[e / 2].x;
      sums[1][e] = e % 2 ? db[e / 2].y : db[e / 2].x;
#pragma unroll
      for (int m = LANES; m < 32; m *= 2)
#pragma unroll
        for (int k = 0; k < 2; ++k) sums[k][e] += ctx.shfl_xor(sums[k][e], m);
    }
    for (int w = 0; w < 8; ++w) {
      if (ctx.tid / 32 == w && ctx.tid % 32 < LANES)
#pragma unroll
        for (int e = 0; e < 2 * kPairs; ++e) {
          float* to = red + e * LANES + team.t;
          *to = (w ? *to : 0.f) + sums[e / kPairs][e % kPairs];
        }
      ctx.sync();
    }
    for (int e = ctx.tid; e < 2 * kPairs * LANES; e += ctx.nthr) {
      const int c = Team::place(p, Team::pair(e % LANES, e / LANES % kPairs), e / LANES / kPairs);
      if (c >= 0) p.part[(long)ctx.bid * p.dim + c] = red[e];
    }
  }
};

// Weight gradients: the blocks' rows added in their order, 32 columns to a block, by eight warps that take every eighth row.
struct HeadSumParams {
  const float* part;
  void* dw[2];
  int first[2], blocks[2], dim;
};
template <class T>
struct HeadWeightSum {
  using Params = HeadSumParams;
  static constexpr int kThreads = 256, kBlocks = 4;
  static S2C_D void run(const Ctx& ctx, const Params& p, unsigned char* smem) {
    float* red = reinterpret_cast<float*>(smem);      // [8][32]
    const int per = (p.dim + 31) / 32, which = ctx.bid / per, lane = ctx.tid % 32, warp = ctx.tid / 32, c = ctx.bid % per * 32 + lane;
    if (!p.dw[which]) return;
    float s = 0.f;
    if (c < p.dim) {
      const float* from = p.part + (long)p.first[which] * p.dim + c;
      float part[4] = {0.f, 0.f, 0.f, 0.f};           // four loads on the way
      int k = warp;
      for (; k + 24 < p.blocks[which]; k += 32)
#pragma unroll
        for (int u = 0; u < 4; ++u) part[u] += from[(long)(k + 8 * u) * p.dim];
      for (; k < p.blocks[which]; k += 8) part[0] += from[(long)k * p.dim];
      s = (part[0] + part[1]) + (part[2] + part[3]);
    }
    red[warp * 32 + lane] = s;
    ctx.sync();
    if (warp != 0 || c >= p.dim) return;
    for (int k = 1; k < 8; ++k) s += red[k * 32 + lane];
    narrow(static_cast<T*>(p.dw[which]) + c, s);
  }
};

}  // namespace s2c
