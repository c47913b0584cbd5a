// Keys and values in pages: where a position lies, pages copied within their pool, and keys and values brought from their pages into one
// array for the kernels of whole tiles.
#pragma once

#include <type_traits>

#include "../../include/s2cnn_b200.h"
#include "seq_common.h"

namespace s2c {

constexpr int kPageLeast = 8;
struct PageTable {
  const int* table = nullptr;     // [batch][columns]: the page of positions [c page, (c + 1) page)
  void* array[2] = {};            // keys, values
  int columns = 0, count = 0, page = 1, log_page = 0;     // pages of the pool; positions of a page, a power of two
  // the page of position `at` of sequence b; -1: it has none
  S2C_D int of(int b, long at) const {
    if (at < 0 || at >= (long)columns * page) return -1;
    const int which = table[(long)b * columns + (at >> log_page)];
    return which < count ? which : -1;
  }
};

// what every call on pages has to fulfil
inline int page_check(const char* who, const s2c_page_desc* d) {
  const std::string w = std::string(who) + ": ";
  if (!d || !d->table) return fail(S2C_ERR_BAD_ARG, w + "no pages");
  if (d->columns < 0 || d->count < 0) return fail(S2C_ERR_BAD_ARG, w + "bad sizes");
  if (d->page < kPageLeast || (d->page & (d->page - 1))) return fail(S2C_ERR_UNSUPPORTED, w + "the positions of a page are a power of two, at least 8");
  if ((long)d->columns * d->page > (1L << 28) || (long)d->count * d->page > 0x7fffffffL) return fail(S2C_ERR_UNSUPPORTED, w + "at most 2^28 positions in a sequence and 2^31 in a pool");
  return S2C_OK;
}
inline PageTable page_table(const s2c_page_desc* d, const void* keys, const void* values) {
  PageTable t;
  t.table = d->table; t.columns = d->columns; t.count = d->count; t.page = d->page;
  while ((1 << t.log_page) < d->page) ++t.log_page;
  t.array[0] = const_cast<void*>(keys); t.array[1] = const_cast<void*>(values);
  return t;
}
// ---- pages copied within their pool -----------------------------------------------------------------------------------
struct PageCopyParams {
  char* base;
  long stride, bytes;             // from one page to the next; of a page
  const int *source, *target;
  long n, chunks;                 // copies; pieces of kChunk bytes of each
  int count;
};
// P: bytes of one access.  A block copies a chunk, all of its loads before its stores.  Bound by memory: 1024 pages of 256 KB 82 us, 6.5 TB/s
// read and written, the measured copy rate; with four loads ahead 122.
template <int P>
struct PageCopy {
  using Params = PageCopyParams;
  using Piece = typename std::conditional<P == 16, Vec16, typename std::conditional<P == 4, unsigned, unsigned char>::type>::type;
  static constexpr int kThreads = 256, kBlocks = 4, kAhead = 8;
  static constexpr long kChunk = (long)kThreads * kAhead * P;
  static S2C_D void run(const Ctx& ctx, const Params& p, unsigned char*) {
    for (long u = ctx.bid; u < p.n * p.chunks; u += ctx.nblk) {
      const long i = u / p.chunks, at = (u - i * p.chunks) * kChunk + (long)ctx.tid * P;
      const int from = p.source[i], to = p.target[i];
      if (from < 0 || from >= p.count || to < 0 || to >= p.count) continue;
      const Piece* x = reinterpret_cast<const Piece*>(p.base + from * p.stride + at);
      Piece* y = reinterpret_cast<Piece*>(p.base + to * p.stride + at);
      const long left = p.bytes - at;                    // of the chunk, from this thread's first piece on
      Piece v[kAhead];
      if (left > (long)(kAhead - 1) * kThreads * P) {
#pragma unroll
        for (int k = 0; k < kAhead; ++k) v[k] = x[k * kThreads];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) y[k * kThreads] = v[k];
      } else {
#pragma unroll
        for (int k = 0; k < kAhead; ++k)
          if (left > (long)k * kThreads * P) v[k] = x[k * kThreads];
#pragma unroll
        for (int k = 0; k < kAhead; ++k)
          if (left > (long)k * kThreads * P) y[k * kThreads] = v[k];
      }
    }
  }
};

// ---- keys and values of every sequence, one after another --------------------------------------------------------------
struct PageGatherParams {
  PageTable pages;
  void* out[2];                   // [batch][length][heads][dim]
  long stride[2][3];              // page, position, head
  const int *q_len, *kv_len, *start;
  Divisor by_head, by_length;     // of a position's pieces, of the rows
  int batch, length, heads, dim, lq, causal, start_all;
};
// A warp takes a position, in pieces of N values; NaN where its page is none.  Rows that no query sees are left as they are.
template <class T, int N>
struct PageGather {
  using Params = PageGatherParams;
  using Piece = typename std::conditional<N == 1, T, Vec16>::type;
  static constexpr int kThreads = 256, kBlocks = 4;
  static S2C_D void run(const Ctx& ctx, const Params& p, unsigned char*) {
    const long warps = (long)ctx.nblk * (kThreads / 32), rows = (long)p.batch * p.length;
    const int lane = ctx.tid % 32, pieces = p.heads * p.dim / N;
    Piece none;
    T nan[N];
#pragma unroll
    for (int e = 0; e < N; ++e) narrow(nan + e, as_float(0x7fffffffu));
    std::memcpy(&none, nan, sizeof(none));
    for (long r = (long)ctx.bid * (kThreads / 32) + ctx.tid / 32; r < rows; r += warps) {
      const int b = (int)p.by_length.quotient((unsigned)r), j = (int)(r - (long)b * p.length);
      if ((p.kv_len && j >= p.kv_len[b]) || (p.causal && j > (long)(p.start ? p.start[b] : p.start_all) + (p.q_len ? p.q_len[b] : p.lq) - 1)) {
        r += (unsigned)(p.length - 1 - j) / (unsigned)warps * warps;       // nor is what follows of this sequence: its last turn
        continue;
      }
      const int page = p.pages.of(b, j), at = j & (p.pages.page - 1);
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        const T* from = static_cast<const T*>(p.pages.array[which]) + (page >= 0 ? page * p.stride[which][0] + at * p.stride[which][1] : 0);
        Piece* to = static_cast<Piece*>(p.out[which]) + r * pieces;
        for (int e = lane; e < pieces; e += 32) {
          const int h = (int)p.by_head.quotient(e);
          to[e] = page >= 0 ? *reinterpret_cast<const Piece*>(from + h * p.stride[which][2] + (e - h * (p.dim / N)) * N) : none;
        }
      }
    }
  }
};

}  // namespace s2c
