// Heads of queries and keys: norm and rotation by position in one pass, forward and backward, and the same with the keys, and values
// beside them, written to pages of a cache (kept_pages.h).
//
//   x^ = x rstd, rstd = 1 / sqrt(mean(x^2) + eps) over a head's values;  z = x^ w            (without a norm: z = x)
//   y_a = mu (z_a cos t - z_b sin t),  y_b = mu (z_a sin t + z_b cos t),  t = position f      (pairs (a, b), mu the magnitude)
//   backward: g the gradient of z (the rotation by -t of that of y, times mu), h = g w:
//   dx = rstd (h - x^ mean(h x^)),  dw = sum over all heads g x^;  rstd is computed again from x: nothing is stored
//
// Angles.  t of a position in the hundred thousands loses its digits in float32.  A lane keeps the frequency of each of its pairs as a
// fraction of a turn in 64 bits of fixed point, F = round(2^64 f / 2 pi mod 2^64); position F modulo 2^64 is then the angle modulo whole
// turns by one integer product, whatever the position (also a negative one).  What is lost is f / 2 pi's own rounding, a relative
// 2^-52, times the position.  The nearest quarter turn is taken off in integers, the rest (an eighth at most) goes through
// the Taylor series of sine and cosine to x^9 and x^10, whose first terms left out are below 2e-9 and 2e-10 there.
//
// A team of 4, 8 or 16 neighbouring lanes holds a head of up to 32, 64 or 128 values, four pairs to a lane, and takes GROUP heads of
// one position at once: their loads are on the way together, and they share the four sines and cosines.  Blocks are dealt to queries,
// keys and values, so that a lane has one weight.
#pragma once

#include "kept_pages.h"
#include "seq_common.h"

namespace s2c {

struct HeadKind {                // queries, keys or values
  const void* x;                 // [batch][length][heads][dim]
  const void* w;                 // norm weight, null: ones
  const void* dy;                // backward: gradient of out, contiguous; null: none arrived (zeros)
  void* out;                     // contiguous; the gradient of x in the backward pass; null: pages
  long stride[3], pstride[3];    // of x; of the pages (page, position, head)
  int heads, blocks;             // blocks of this kind
  int wide;                      // all arrays of this kind in pieces of four values on their boundaries
  int turn;                      // norm and rotation (queries, keys)
};
struct HeadParams {
  HeadKind kind[3];
  const double* frequencies;     // radians per position
  const int *positions, *lengths;
  float* part;                   // backward: [blocks][dim], sums of the weight gradients
  PageTable pages;
  int batch, length, dim, pairs, interleaved, norm;
  int each, first;               // positions: one per position of a sequence, or its first; null: `first` for all
  float eps, magnitude;
};

// f in radians per position as a fraction of a turn, in units of 2^-64
S2C_D unsigned long long turn_units(double f) {
  double t = f * 0.15915494309189533577;
  t -= floor(t);                                             // [0, 1); NaN and infinities: a frequency of 0
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

template <class T, int LANES>
struct HeadTeam {
  static constexpr int kThreads = 256, kTeams = kThreads / LANES;
  // A lane's two pieces of four values, by value e: pairs 4 t ... 4 t + 3.  Halves: the pair's first values and its second ones;
  // neighbours: eight consecutive values.  What is not turned pairs up in the same way.  -1: no value.
  static S2C_D int index(const HeadParams& p, int t, int piece, int e) {
    if (p.interleaved) {
      const int c = 8 * t + 4 * piece + e;
      return c < p.dim ? c : -1;
    }
    const int i = 4 * t + e, rest = p.dim - 2 * p.pairs, low = (rest + 1) / 2;
    if (i < p.pairs) return i + piece * p.pairs;
    const int r = i - p.pairs;
    return piece == 0 ? (r < low ? 2 * p.pairs + r : -1) : r < rest - low ? 2 * p.pairs + low + r : -1;
  }
  static S2C_D void load(const HeadParams& p, int wide, const T* x, int t, float (&v)[2][4]) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int c = index(p, t, k, 0);
      if (wide) {
        if (c >= 0) load_four(x + c, v[k]);
        else
#pragma unroll
          for (int e = 0; e < 4; ++e) v[k][e] = 0.f;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int i = index(p, t, k, e);
          v[k][e] = i >= 0 ? widen(x[i]) : 0.f;
        }
      }
    }
  }
  static S2C_D void store(const HeadParams& p, int wide, T* y, int t, const float (&v)[2][4]) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int c = index(p, t, k, 0);
      if (wide) {
        if (c >= 0) store_four(y + c, v[k]);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int i = index(p, t, k, e);
          if (i >= 0) narrow(y + i, v[k][e]);
        }
      }
    }
  }
  // the pairs' frequencies; what is not turned has 0
  static S2C_D void frequencies(const HeadParams& p, int t, unsigned long long (&f)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = 4 * t + e < p.pairs ? turn_units(p.frequencies[4 * t + e]) : 0ull;
  }
  // the pairs of two pieces, turned (sign 1) or turned back (-1)
  static S2C_D void turn(const HeadParams& p, int t, const float (&c)[4], const float (&s)[4], float sign, float (&v)[2][4]) {
    float a[4], b[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      a[e] = p.interleaved ? v[e / 2][2 * (e % 2)] : v[0][e];
      b[e] = p.interleaved ? v[e / 2][2 * (e % 2) + 1] : v[1][e];
      if (4 * t + e < p.pairs) {                        // (others stay as they are: an infinity times 0 would be none)
        const float x = a[e], y = b[e], si = sign * s[e];
        a[e] = x * c[e] - y * si;
        b[e] = x * si + y * c[e];
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[0][e] = p.interleaved ? (e % 2 ? b[e / 2] : a[e / 2]) : a[e];
      v[1][e] = p.interleaved ? (e % 2 ? b[2 + e / 2] : a[2 + e / 2]) : b[e];
    }
  }
  static S2C_D long position(const HeadParams& p, int b, int i) {
    if (!p.positions) return (long)p.first + i;
    return p.each ? p.positions[(long)b * p.length + i] : (long)p.positions[b] + i;
  }
  static S2C_D void angles(const HeadParams& p, const unsigned long long (&f)[4], long at, float (&c)[4], float (&s)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      turn_cos_sin(f[e] * (unsigned long long)at, c[e], s[e]);
      c[e] *= p.magnitude;
      s[e] *= p.magnitude;
    }
  }
};

// A unit is GROUP neighbouring heads of one position.
template <class T, int LANES, int GROUP>
struct HeadForward : HeadTeam<T, LANES> {
  using Team = HeadTeam<T, LANES>;
  using Params = HeadParams;
  static constexpr int kBlocks = 3;
  static S2C_D void run(const Ctx& ctx, const Params& p, unsigned char*) {
    int which = 0, bid = ctx.bid;
    while (which < 2 && bid >= p.kind[which].blocks) bid -= p.kind[which++].blocks;
    const HeadKind& kind = p.kind[which];
    const int team = ctx.tid / LANES, t = ctx.tid % LANES;
    const int groups = (kind.heads + GROUP - 1) / GROUP;
    const long units = (long)p.batch * p.length * groups, per = (long)kind.blocks * Team::kTeams;
    unsigned long long f[4];
    float w[2][4];
    if (kind.turn) {
      Team::frequencies(p, t, f);
      if (kind.w) Team::load(p, 0, static_cast<const T*>(kind.w), t, w);
    }
    for (long u0 = (long)bid * Team::kTeams; u0 < units; u0 += per) {     // (every team takes the same number of turns)
      const bool on = u0 + team < units;
      const long u = on ? u0 + team : 0, row = u / groups;
      const int h0 = (int)(u % groups) * GROUP, b = (int)(row / p.length), i = (int)(row % p.length);
      const bool filled = !p.lengths || i < p.lengths[b];
      const long at = Team::position(p, b, i);
      const T* x = static_cast<const T*>(kind.x) + b * kind.stride[0] + i * kind.stride[1];
      float v[GROUP][2][4];
#pragma unroll
      for (int g = 0; g < GROUP; ++g)
        if (on && filled && h0 + g < kind.heads) Team::load(p, kind.wide, x + (h0 + g) * kind.stride[2], t, v[g]);
        else
#pragma unroll
          for (int e = 0; e < 8; ++e) v[g][e / 4][e % 4] = 0.f;
      long slot = 0;
      const bool stored = p.pages.table && p.pages.at(b, at, slot);
      if (kind.turn) {
        float c[4], s[4];
        Team::angles(p, f, at, c, s);
#pragma unroll
        for (int g = 0; g < GROUP; ++g) {
          if (p.norm) {
            float sum = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) sum += v[g][e / 4][e % 4] * v[g][e / 4][e % 4];
            const float rstd = inv_sqrt(lanes_sum<LANES>(ctx, sum) / (float)p.dim + p.eps);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              v[g][e / 4][e % 4] *= rstd;
              if (kind.w) v[g][e / 4][e % 4] *= w[e / 4][e % 4];
            }
          }
          Team::turn(p, t, c, s, 1.f, v[g]);
        }
      }
      if (!on) continue;
      if (kind.out) {
        T* y = static_cast<T*>(kind.out) + (row * kind.heads + h0) * p.dim;
        const bool lost = p.pages.table && filled && !stored;              // a query whose key has no place
#pragma unroll
        for (int g = 0; g < GROUP; ++g) {
          if (h0 + g >= kind.heads) break;
          if (!filled || lost)
#pragma unroll
            for (int e = 0; e < 8; ++e) v[g][e / 4][e % 4] = lost ? as_float(0x7fffffffu) : 0.f;
          Team::store(p, kind.wide, y + g * p.dim, t, v[g]);
        }
      } else if (filled && stored) {
        T* y = static_cast<T*>(p.pages.array[which - 1]) + slot / p.pages.page * kind.pstride[0] + slot % p.pages.page * kind.pstride[1] + h0 * kind.pstride[2];
#pragma unroll
        for (int g = 0; g < GROUP; ++g)
          if (h0 + g < kind.heads) Team::store(p, kind.wide, y + g * kind.pstride[2], t, v[g]);
      }
    }
  }
};

template <class T, int LANES, int GROUP>
struct HeadBackward : HeadTeam<T, LANES> {
  using Team = HeadTeam<T, LANES>;
  using Params = HeadParams;
  static constexpr int kBlocks = 2;
  static size_t smem() { return 8 * LANES * sizeof(float); }
  static S2C_D void run(const Ctx& ctx, const Params& p, unsigned char* smem) {
    const int which = ctx.bid >= p.kind[0].blocks ? 1 : 0;
    const HeadKind& kind = p.kind[which];
    const int bid = ctx.bid - (which ? p.kind[0].blocks : 0), team = ctx.tid / LANES, t = ctx.tid % LANES;
    const int groups = (kind.heads + GROUP - 1) / GROUP;
    const long units = (long)p.batch * p.length * groups, per = (long)kind.blocks * Team::kTeams;
    unsigned long long f[4];
    Team::frequencies(p, t, f);
    float w[2][4], dw[2][4];
    if (kind.w) Team::load(p, 0, static_cast<const T*>(kind.w), t, w);
#pragma unroll
    for (int e = 0; e < 8; ++e) dw[e / 4][e % 4] = 0.f;
    for (long u0 = (long)bid * Team::kTeams; u0 < units; u0 += per) {
      const bool on = u0 + team < units;
      const long u = on ? u0 + team : 0, row = u / groups;
      const int h0 = (int)(u % groups) * GROUP, b = (int)(row / p.length), i = (int)(row % p.length);
      const T* x = static_cast<const T*>(kind.x) + b * kind.stride[0] + i * kind.stride[1];
      const T* dy = static_cast<const T*>(kind.dy) + (row * kind.heads + h0) * p.dim;
      float v[GROUP][2][4], d[GROUP][2][4];
#pragma unroll
      for (int g = 0; g < GROUP; ++g) {
        const bool in = on && h0 + g < kind.heads;
        if (in) Team::load(p, kind.wide, dy + g * p.dim, t, d[g]);
        else
#pragma unroll
          for (int e = 0; e < 8; ++e) d[g][e / 4][e % 4] = 0.f;
        if (in && p.norm) Team::load(p, kind.wide, x + (h0 + g) * kind.stride[2], t, v[g]);
        else
#pragma unroll
          for (int e = 0; e < 8; ++e) v[g][e / 4][e % 4] = 0.f;
      }
      float c[4], s[4];
      Team::angles(p, f, Team::position(p, b, i), c, s);
#pragma unroll
      for (int g = 0; g < GROUP; ++g) {
        Team::turn(p, t, c, s, -1.f, d[g]);
        if (p.norm) {
          float sum = 0.f, dot = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) sum += v[g][e / 4][e % 4] * v[g][e / 4][e % 4];
          const float rstd = inv_sqrt(lanes_sum<LANES>(ctx, sum) / (float)p.dim + p.eps);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            float &xh = v[g][e / 4][e % 4], &gr = d[g][e / 4][e % 4];
            xh *= rstd;
            dw[e / 4][e % 4] += gr * xh;
            if (kind.w) gr *= w[e / 4][e % 4];
            dot += gr * xh;
          }
          dot = lanes_sum<LANES>(ctx, dot) / (float)p.dim;
#pragma unroll
          for (int e = 0; e < 8; ++e) d[g][e / 4][e % 4] = rstd * (d[g][e / 4][e % 4] - v[g][e / 4][e % 4] * dot);
        }
        if (on && h0 + g < kind.heads && kind.out) Team::store(p, kind.wide, static_cast<T*>(kind.out) + (row * kind.heads + h0 + g) * p.dim, t, d[g]);
      }
    }
    if (!p.part || !kind.w) return;                 // (a whole block)
    // the teams of a warp, then the warps in their order
    float* red = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int m = LANES; m < 32; m *= 2)
#pragma unroll
      for (int e = 0; e < 8; ++e) dw[e / 4][e % 4] += ctx.shfl_xor(dw[e / 4][e % 4], m);
    for (int k = 0; k < 8; ++k) {
      if (ctx.tid / 32 == k && ctx.tid % 32 < LANES)
#pragma unroll
        for (int e = 0; e < 8; ++e) red[e * LANES + t] = (k ? red[e * LANES + t] : 0.f) + dw[e / 4][e % 4];
      ctx.sync();
    }
    if (team != 0) return;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int c = Team::index(p, t, e / 4, e % 4);
      if (c >= 0) p.part[(long)ctx.bid * p.dim + c] = red[e * LANES + t];
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
