// Dropout whose mask is computed where it is needed and never stored:
//   y[i] = residual[i] + (word[i] >= p 2^32 ? x[i] / (1 - p) : 0)
// word[i] is word i % 4 of block i / 4 of a counter-based generator, Philox-4x32 (J. Salmon, M. Moraes, R. Dror, D. Shaw:
// "Parallel random numbers: as easy as 1, 2, 3", 2011) with key = seed and counter = (block, step), low words first.  Each
// round takes the four words (a, b, c, d) to (hi(M1 c) ^ b ^ k0, lo(M1 c), hi(M0 a) ^ d ^ k1, lo(M0 a)) and adds a Weyl
// constant to either half of the key.  Seven rounds are the fewest that the paper found to pass all of BigCrush.
// The gradient is the same kernel on the gradient of y, without a residual: the mask follows from the index alone, whatever
// the shape of the launch.  Bound by the loads on their way, not by their bytes: a thread has one 16-byte piece of each input in
// flight, and the generator (some 60 instructions for 4 elements) between one piece and the next.  16384 x 1024 with a residual and
// without, in calls among others: bfloat16 22 and 17 us (4.5 and 3.9 TB/s), float32 36 and 30 us (5.6 and 4.5).
#pragma once

#include "seq_common.h"

namespace s2c {

struct DropoutParams {
  const void* x;
  const void* residual;   // null: none
  void* out;
  long n;
  unsigned threshold;     // floor(p 2^32): a word below it drops its element
  float scale;            // 1 / (1 - p)
  unsigned key[2], step[2];
  const unsigned long long* numbers;   // seed and step in memory, null: those above
};

S2C_D void philox7(unsigned long long block, const unsigned (&key)[2], const unsigned (&step)[2], unsigned (&w)[4]) {
  unsigned a = (unsigned)block, b = (unsigned)(block >> 32), c = step[0], d = step[1], k0 = key[0], k1 = key[1];
#pragma unroll
  for (int r = 0; r < 7; ++r) {
    const unsigned long long x = 0xD2511F53ull * a, y = 0xCD9E8D57ull * c;
    a = (unsigned)(y >> 32) ^ b ^ k0;
    b = (unsigned)y;
    c = (unsigned)(x >> 32) ^ d ^ k1;
    d = (unsigned)x;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  w[0] = a; w[1] = b; w[2] = c; w[3] = d;
}

// VEC: x, residual and out 16-byte aligned; a thread takes the elements of one 16-byte access at a time.
template <class T, bool VEC>
struct Dropout {
  using Params = DropoutParams;
  static constexpr int kThreads = 256, kBlocks = 4;
  static constexpr int kStep = VEC ? kVec<T> : 4;     // consecutive elements of a thread: whole blocks of words
  static S2C_D void run(const Ctx& ctx, const Params& p, unsigned char*) {
    const T* x = static_cast<const T*>(p.x);
    const T* res = static_cast<const T*>(p.residual);
    T* out = static_cast<T*>(p.out);
    const long stride = (long)ctx.nblk * ctx.nthr * kStep;
    unsigned key[2] = {p.key[0], p.key[1]}, step[2] = {p.step[0], p.step[1]};
    if (p.numbers) {
      key[0] = (unsigned)p.numbers[0];
      key[1] = (unsigned)(p.numbers[0] >> 32);
      step[0] = (unsigned)p.numbers[1];
      step[1] = (unsigned)(p.numbers[1] >> 32);
    }
    for (long i = ((long)ctx.bid * ctx.nthr + ctx.tid) * kStep; i < p.n; i += stride) {
      unsigned w[kStep];
#pragma unroll
      for (int b = 0; b < kStep / 4; ++b) {
        unsigned four[4];
        philox7((unsigned long long)(i / 4 + b), key, step, four);
#pragma unroll
        for (int e = 0; e < 4; ++e) w[4 * b + e] = four[e];
      }
      float v[kStep], r[kStep];
#pragma unroll
      for (int e = 0; e < kStep; ++e) r[e] = 0.f;
      if (VEC && i + kStep <= p.n) {
        if constexpr (VEC) {
          load_vec(x + i, v);
          if (res) load_vec(res + i, r);
        }
      } else {
#pragma unroll
        for (int e = 0; e < kStep; ++e) {
          v[e] = i + e < p.n ? widen(x[i + e]) : 0.f;
          if (res && i + e < p.n) r[e] = widen(res[i + e]);
        }
      }
#pragma unroll
      for (int e = 0; e < kStep; ++e) v[e] = r[e] + (w[e] >= p.threshold ? v[e] * p.scale : 0.f);
      if (VEC && i + kStep <= p.n) {
        if constexpr (VEC) store_vec(out + i, v);
      } else {
#pragma unroll
        for (int e = 0; e < kStep; ++e)
          if (i + e < p.n) narrow(out + i + e, v[e]);
      }
    }
  }
};

}  // namespace s2c
