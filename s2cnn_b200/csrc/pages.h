// C-ABI entry points of attention over pages and of copying them (the end of the section on sequences in include/s2cnn_b200.h):
// checks and the choice of kernels.  Compiled from pages.cu beside lib.cu; part of lib.cu's translation unit in the host-emulation build.
#pragma once

#include "../../include/s2cnn_b200.h"

#include <algorithm>
#include <cfloat>
#include <cmath>

#include "attention_kernels.h"
#include "kept_pages.h"
#include "paged_attention_kernels.h"

namespace s2c {

// ---- pages ---------------------------------------------------------------------------------------------------------------
inline size_t page_align(size_t n) { return (n + 255) / 256 * 256; }
// the call on gathered keys and values
inline s2c_attention_desc gathered(const s2c_attention_desc* d, const s2c_page_desc* pages) {
  s2c_attention_desc g = *d;
  g.lk = pages->columns * pages->page;
  const long row = (long)d->kv_heads * d->dim, stride[3] = {row * g.lk, row, d->dim};
  for (int i = 0; i < 3; ++i) g.k_stride[i] = g.v_stride[i] = stride[i];
  g.bias_grad = 0;
  return g;
}
inline size_t gathered_bytes(const s2c_attention_desc& g) {
  return page_align((size_t)g.batch * g.lk * g.kv_heads * g.dim * (g.dtype == kSeqF32 ? 4 : 2));
}
// How many sequences are brought into one array at a time: all, or equal groups whose keys and values take at most 1 GB; 0: one takes more.
constexpr size_t kGatherMost = 1ul << 30;
inline long gathered_at_once(const s2c_attention_desc* d, const s2c_page_desc* pages) {
  s2c_attention_desc g = gathered(d, pages);
  g.batch = 1;
  const size_t one = 2 * gathered_bytes(g);
  if (one > kGatherMost) return 0;
  const long batch = std::max(1, d->batch), n = one ? std::min(batch, (long)(kGatherMost / one)) : batch, groups = (batch + n - 1) / n;
  return (batch + groups - 1) / groups;
}
// their workspace: gathered keys and values, and what the call on them wants
inline size_t gathered_need(const s2c_attention_desc* d, const s2c_page_desc* pages, long n) {
  s2c_attention_desc g = gathered(d, pages);
  g.batch = (int)n;
  return 2 * gathered_bytes(g) + s2c_attention_workspace(&g);
}
template <class T>
int page_gather(const s2c_attention_desc* d, const s2c_page_desc* pages, const void* keys, const void* values, int length, void* k, void* v, stream_t st) {
  PageGatherParams p = {};
  p.pages = page_table(pages, keys, values);
  p.out[0] = k; p.out[1] = v;
  bool wide = d->dim % kVec<T> == 0 && aligned16(keys) && aligned16(values);
  for (int i = 0; i < 3; ++i) {
    p.stride[0][i] = pages->key_stride[i];
    p.stride[1][i] = pages->value_stride[i];
    wide = wide && pages->key_stride[i] % kVec<T> == 0 && pages->value_stride[i] % kVec<T> == 0;
  }
  p.q_len = d->q_lengths; p.kv_len = d->kv_lengths; p.start = d->q_starts;
  p.batch = d->batch; p.length = length; p.heads = d->kv_heads; p.dim = d->dim; p.lq = d->lq; p.causal = d->causal; p.start_all = d->q_start;
  p.by_length = Divisor(std::max(1, length));
  p.by_head = Divisor(wide ? d->dim / kVec<T> : d->dim);
  const long rows = (long)d->batch * length;
  if (rows > 0x7fffffffL || (long)d->kv_heads * d->dim > 0x7fffffffL) return fail(S2C_ERR_UNSUPPORTED, "s2c_paged_attention: too many positions");
  const long blocks = std::min<long>((rows + 7) / 8, 16L * dev_sm_count());
  return wide ? seq_launch<PageGather<T, kVec<T>>>("page_gather", blocks, 0, st, p) : seq_launch<PageGather<T, 1>>("page_gather", blocks, 0, st, p);
}

#ifndef S2C_EMUL
inline AttnParams paged_params(const s2c_attention_desc* d, const s2c_page_desc* pages, const void* q, const void* bias, void* out) {
  AttnParams p = {};
  p.q = q; p.bias = d->bucket_of ? bias : nullptr; p.out = out;
  p.bucket_of = d->bucket_of; p.start = d->q_starts; p.q_len = d->q_lengths; p.kv_len = d->kv_lengths;
  for (int i = 0; i < 3; ++i) p.qs[i] = d->q_stride[i];
  p.batch = d->batch; p.lq = d->lq; p.lk = pages->columns * pages->page; p.heads = d->heads; p.kv_heads = d->kv_heads; p.dim = d->dim;
  p.group = d->heads / d->kv_heads;
  p.causal = d->causal != 0; p.scale = d->scale; p.start_all = d->q_start;
  p.reach = p.bias ? d->reach : 0; p.n_buckets = p.bias ? d->n_buckets : 0;
  return p;
}
// Many queries: keys and values are brought into one array for the kernels of whole tiles, instead of being read again by every 16 rows.
// 4 x 4096 positions, 4 key heads of 128, 32, 128, 256 and 512 rows for each: in pages 23, 56, 95 and 174 us (float32 45, 127, 224 and
// 427), in one array 48 to 49 (253 to 259) and some 11 (17) to bring them there.  Not where that takes more than 1 GB for one sequence (by its
// columns, since what is kept of them only the device knows; packed copies come on top, in float32 1.5 times as much).  In groups of
// sequences only where their tiles fill half of the SMs: float32, tables of 65536 positions, 16 heads of 128 on 4, groups of 32, 48, 64 and 96
// tiles 1194, 2375, 373 and 397 us, in pages 916, 1641, 385 and 916 (16 x 1000 kept and 256 queries, 64 x 300 and 300, 9 x 400 and 400, and the
// first again with three sequences to a group; bfloat16 99 us and 366, 288 and 751, 55 and 174).
inline bool paged_gathers(const s2c_attention_desc* d, const s2c_page_desc* pages) {
  const long rows = (long)d->lq * (d->heads / d->kv_heads), n = gathered_at_once(d, pages);
  if (rows <= (d->dtype == kSeqF32 ? 256 : 128) || n == 0) return false;
  return n >= d->batch || n * d->heads * ((d->lq + 127) / 128) >= dev_sm_count() / 2;
}
// rows of 16-byte pieces (of four values at least): keys and values as they lie
template <class T>
bool paged_wide(const s2c_page_desc* d, const void* keys, const void* values) {
  bool ok = on_boundary(keys, 16) && on_boundary(values, 16);
  for (int i = 0; i < 3; ++i) ok = ok && d->key_stride[i] % kVec<T> == 0 && d->value_stride[i] % kVec<T> == 0;
  return ok;
}
struct PagedPlan {
  long items = 0, blocks = 0;
  int row_blocks = 0, nt = 1;
  long parts = 1;              // of an item at most
  size_t part = 0, bytes = 0;
};
template <class T, class F>
int paged_by_shape(int dim, int nt, F f) {
#define S2C_PAGED(DP) return nt == 1 ? f(std::integral_constant<int, DP>(), std::integral_constant<int, 1>()) : f(std::integral_constant<int, DP>(), std::integral_constant<int, 2>())
  if (dim <= 32) S2C_PAGED(32);
  if (dim <= 64) S2C_PAGED(64);
  S2C_PAGED(128);
#undef S2C_PAGED
}
// How many blocks share the work: as many as run at once, or fewer where the columns hold fewer steps.
template <class T>
PagedPlan paged_plan(const AttnParams& a) {
  PagedPlan plan;
  const long rows = (long)a.lq * a.group;
  plan.nt = rows <= 8 ? 1 : 2;
  plan.row_blocks = (int)((rows + 8 * plan.nt - 1) / (8 * plan.nt));
  plan.items = (long)a.batch * a.kv_heads * plan.row_blocks;
  paged_by_shape<T>(a.dim, plan.nt, [&](auto dp, auto nt) {
    using K = PagedAttention<T, decltype(dp)::value, decltype(nt)::value, kRowsFull>;
    const long steps = std::max(1, (a.lk + K::H::kStep - 1) / K::H::kStep);
    plan.blocks = std::min((long)K::kBlocks * dev_sm_count(), plan.items * steps);
    plan.parts = std::min(steps, plan.blocks);
    plan.part = page_align(2 * (size_t)plan.blocks * K::H::kRows * (decltype(dp)::value + 4) * sizeof(float));
    return (int)S2C_OK;
  });
  plan.bytes = plan.part + (size_t)std::min(plan.items, plan.blocks) * sizeof(int4);
  return plan;
}
template <class T>
int paged_launch(const AttnParams& a, const s2c_page_desc* pages, const void* keys, const void* values, void* ws, stream_t st) {
  const PagedPlan plan = paged_plan<T>(a);
  if (plan.items == 0) return S2C_OK;
  if (plan.items > 0x7fffffffL || (long)a.lq * a.group > 0x7fffff00L) return fail(S2C_ERR_UNSUPPORTED, "s2c_paged_attention: too many heads and queries");
  PagedParams p = {};
  p.a = a;
  p.pages = page_table(pages, keys, values);
  for (int i = 0; i < 3; ++i) { p.ks[i] = pages->key_stride[i]; p.vs[i] = pages->value_stride[i]; }
  if (pages->count == 0) {                     // what is read in the place of a page that is none, with a score of NaN
    for (int i = 0; i < 3; ++i) p.ks[i] = p.vs[i] = 0;
    p.pages.array[0] = p.pages.array[1] = ws;
  }
  p.row_blocks = plan.row_blocks;
  p.by_group = Divisor(a.group);
  p.by_row_blocks = Divisor(plan.row_blocks);
  p.by_buckets = Divisor(a.n_buckets + 1);
  p.wide_out = a.dim % 4 == 0 && on_boundary(a.out, 4 * sizeof(T));
  p.part = static_cast<float*>(ws);
  p.split = reinterpret_cast<int4*>(static_cast<char*>(ws) + plan.part);
  const bool wide = paged_wide<T>(pages, p.pages.array[0], p.pages.array[1]);
  return paged_by_shape<T>(a.dim, plan.nt, [&](auto dp, auto nt) {
    constexpr int DP = decltype(dp)::value, NT = decltype(nt)::value;
    using F = PagedAttention<T, DP, NT, kRowsFull>;
    using W = PagedAttention<T, DP, NT, kRowsInPieces>;
    using N = PagedAttention<T, DP, NT, kRowsByValue>;
    S2C_SEQ_TRY(!wide ? seq_launch<N>("paged_attention", plan.blocks, N::smem(a), st, p)
                : a.dim < DP ? seq_launch<W>("paged_attention", plan.blocks, W::smem(a), st, p)
                             : seq_launch<F>("paged_attention", plan.blocks, F::smem(a), st, p));
    if (plan.parts == 1) return (int)S2C_OK;
    using Few = PagedJoin<T, DP, NT, 4>;
    using Many = PagedJoin<T, DP, NT, 1>;
    const long rows = std::min(plan.items, plan.blocks) * F::H::kRows;
    return plan.blocks <= 16 * plan.items ? seq_launch<Few>("paged_join", rows / 4, Few::smem(plan.parts), st, p)
                                          : seq_launch<Many>("paged_join", rows, Many::smem(plan.parts), st, p);
  });
}
#endif

}  // namespace s2c

using namespace s2c;

extern "C" {

size_t s2c_paged_attention_workspace(const s2c_attention_desc* d, const s2c_page_desc* pages) {
  if (page_check("s2c_paged_attention_workspace", pages) != S2C_OK || attn_check("s2c_paged_attention_workspace", d) != S2C_OK) return 0;
#ifndef S2C_EMUL
  if (!paged_gathers(d, pages)) {
    const AttnParams a = paged_params(d, pages, nullptr, nullptr, nullptr);
    return d->dtype == kSeqF32 ? paged_plan<float>(a).bytes : paged_plan<bf16>(a).bytes;
  }
#endif
  const long n = std::max(1L, gathered_at_once(d, pages)), rest = d->batch % n;
  return std::max(gathered_need(d, pages, n), rest ? gathered_need(d, pages, rest) : 0);
}

int s2c_paged_attention(const s2c_attention_desc* d, const s2c_page_desc* pages, const void* q, const void* keys, const void* values, const void* bias,
                        void* out, void* workspace, size_t workspace_bytes, void* stream) {
  S2C_SEQ_TRY(page_check("s2c_paged_attention", pages));
  S2C_SEQ_TRY(attn_check("s2c_paged_attention", d));
  if (d->batch == 0 || d->lq == 0) return S2C_OK;
  if (!q || !out || (pages->count > 0 && (!keys || !values))) return fail(S2C_ERR_BAD_ARG, "s2c_paged_attention: a pointer is missing");
  if ((bias != nullptr) != (d->bucket_of != nullptr)) return fail(S2C_ERR_BAD_ARG, "s2c_paged_attention: a bias needs its buckets, and buckets a bias");
  if (!aligned16(workspace)) return fail(S2C_ERR_BAD_ARG, "s2c_paged_attention: the workspace starts on a 16-byte boundary");
  const size_t need = s2c_paged_attention_workspace(d, pages);
  if (need > workspace_bytes || (need && !workspace)) return fail(S2C_ERR_WORKSPACE, "s2c_paged_attention: workspace too small");
#ifndef S2C_EMUL
  if (!paged_gathers(d, pages)) {
    const AttnParams a = paged_params(d, pages, q, bias, out);
    return d->dtype == kSeqF32 ? paged_launch<float>(a, pages, keys, values, workspace, (stream_t)stream)
                               : paged_launch<bf16>(a, pages, keys, values, workspace, (stream_t)stream);
  }
#endif
  const long at_once = std::max(1L, gathered_at_once(d, pages)), size = d->dtype == kSeqF32 ? 4 : 2;
  for (long b = 0; b < d->batch; b += at_once) {
    s2c_attention_desc g = gathered(d, pages);
    s2c_page_desc some = *pages;
    g.batch = (int)std::min(at_once, d->batch - b);
    some.table += b * pages->columns;
    for (const int** of : {&g.q_starts, &g.q_lengths, &g.kv_lengths})
      if (*of) *of += b;
    const size_t part = gathered_bytes(g);
    char* at = static_cast<char*>(workspace);
    S2C_SEQ_TRY(d->dtype == kSeqF32 ? page_gather<float>(&g, &some, keys, values, g.lk, at, at + part, (stream_t)stream)
                                    : page_gather<bf16>(&g, &some, keys, values, g.lk, at, at + part, (stream_t)stream));
    S2C_SEQ_TRY(s2c_attention(&g, static_cast<const char*>(q) + b * d->q_stride[0] * size, at, at + part, bias,
                              static_cast<char*>(out) + b * d->lq * d->heads * d->dim * size, nullptr, at + 2 * part, workspace_bytes - 2 * part, stream));
  }
  return S2C_OK;
}

int s2c_copy_pages(void* storage, long page_stride, long page_bytes, int count, const int* source, const int* target, long n, void* stream) {
  if (count < 0 || n < 0 || page_bytes < 0 || (n > 0 && count > 0 && page_bytes > 0 && (!storage || !source || !target)) || (count > 1 && page_stride < page_bytes))
    return fail(S2C_ERR_BAD_ARG, "s2c_copy_pages: bad argument");
  if (page_bytes == 0 || count == 0) return S2C_OK;
  PageCopyParams p = {};
  p.base = static_cast<char*>(storage); p.stride = page_stride; p.bytes = page_bytes; p.source = source; p.target = target; p.n = n; p.count = count;
  auto go = [&](auto k) {
    using K = typename decltype(k)::type;
    p.chunks = (page_bytes + K::kChunk - 1) / K::kChunk;
    return seq_launch<K>("copy_pages", std::min<long>(n * p.chunks, 0x7fffffffL), 0, (stream_t)stream, p);
  };
  struct A { using type = PageCopy<16>; };
  struct B { using type = PageCopy<4>; };
  struct C { using type = PageCopy<1>; };
  auto fits = [&](long b) { return on_boundary(storage, b) && page_stride % b == 0 && page_bytes % b == 0; };
  return fits(16) ? go(A()) : fits(4) ? go(B()) : go(C());
}

}  // extern "C"
