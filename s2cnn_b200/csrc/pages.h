// C-ABI entry points of the rotation of heads by position and of kept keys in pages (the end of the section on sequences in
// include/s2cnn_b200.h): checks and the choice of kernels.  Compiled from pages.cu beside lib.cu; part of lib.cu's translation unit in
// the host-emulation build.
#pragma once

#include "../../include/s2cnn_b200.h"

#include <algorithm>
#include <cfloat>
#include <cmath>

#include "attention_kernels.h"
#include "head_rotation_kernels.h"
#include "kept_pages.h"
#include "paged_attention_kernels.h"

namespace s2c {

inline bool on_boundary(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// ---- heads ---------------------------------------------------------------------------------------------------------------
constexpr int kHeadMaxDim = 128;
inline int head_check(const char* who, const s2c_head_desc* d) {
  const std::string w = std::string(who) + ": ";
  if (!d) return fail(S2C_ERR_BAD_ARG, w + "no description");
  S2C_SEQ_TRY(seq_check_type(who, d->dtype));
  if (d->batch < 0 || d->length < 0 || d->heads < 0 || d->kv_heads < 0 || d->dim < 1) return fail(S2C_ERR_BAD_ARG, w + "bad sizes");
  if (d->dim > kHeadMaxDim) return fail(S2C_ERR_UNSUPPORTED, w + "at most 128 values per head");
  if (d->pairs < 0 || 2 * d->pairs > d->dim || (d->pairs > 0 && !d->frequencies)) return fail(S2C_ERR_BAD_ARG, w + "more frequencies than pairs of values, or none");
  if (!(std::fabs(d->magnitude) <= FLT_MAX) || (d->norm && !(d->eps >= 0.f))) return fail(S2C_ERR_BAD_ARG, w + "magnitude or eps is no number, or eps negative");
  return S2C_OK;
}
inline HeadParams head_params(const s2c_head_desc* d) {
  HeadParams p = {};
  p.frequencies = d->frequencies; p.positions = d->positions; p.lengths = d->lengths;
  p.batch = d->batch; p.length = d->length; p.dim = d->dim; p.pairs = d->pairs; p.interleaved = d->interleaved != 0; p.norm = d->norm != 0;
  p.each = d->each != 0; p.first = d->start;
  p.eps = d->eps; p.magnitude = d->magnitude;
  return p;
}
inline void head_kind(HeadKind& k, const void* x, const void* w, void* out, const long (&stride)[3], int heads, int turn) {
  k.x = x; k.w = w; k.out = out; k.heads = x ? heads : 0; k.turn = turn;
  for (int i = 0; i < 3; ++i) k.stride[i] = stride[i];
}
// Pieces of four values: those of a lane have to lie together (halves: whole pieces of pairs, and of what is not turned), and rows
// on their boundaries.  (The weights are read value by value, once per block.)
inline bool head_wide(const HeadParams& p, const HeadKind& k, int size) {
  bool ok = p.interleaved ? p.dim % 4 == 0 : p.pairs % 4 == 0 && (p.dim - 2 * p.pairs) % 8 == 0;
  ok = ok && on_boundary(k.x, 4 * size) && on_boundary(k.dy, 4 * size) && on_boundary(k.out, 4 * size);
  for (int i = 0; i < 3; ++i) ok = ok && k.stride[i] % 4 == 0;
  return ok;
}
// Blocks of each kind: one turn for every team where `most` blocks hold them, and the kinds' share of `most` otherwise.
inline long head_blocks(HeadParams& p, int kinds, int group, int teams, long most) {
  long want[3] = {}, all = 0;
  for (int k = 0; k < kinds; ++k) {
    want[k] = ((long)p.batch * p.length * ((p.kind[k].heads + group - 1) / group) + teams - 1) / teams;
    all += want[k];
  }
  long sum = 0;
  for (int k = 0; k < kinds; ++k) {
    const long n = all <= most ? want[k] : want[k] ? std::max(1L, (long)((double)want[k] / (double)all * (double)most)) : 0;
    p.kind[k].blocks = (int)n;
    sum += n;
  }
  return sum;
}
template <class T, class F>
int head_by_dim(int dim, F f) {
  if (dim <= 32) return f(std::integral_constant<int, 4>());
  if (dim <= 64) return f(std::integral_constant<int, 8>());
  return f(std::integral_constant<int, 16>());
}
template <class T>
int head_forward(HeadParams p, int kinds, const char* name, stream_t st) {
  for (int k = 0; k < kinds; ++k) p.kind[k].wide = p.kind[k].wide && head_wide(p, p.kind[k], sizeof(T));
  return head_by_dim<T>(p.dim, [&](auto lanes) {
    constexpr int L = decltype(lanes)::value;
    using Four = HeadForward<T, L, 4>;
    using One = HeadForward<T, L, 1>;
    const long most = 2L * Four::kBlocks * dev_sm_count();
    // four heads to a team where that leaves two blocks for every SM
    long blocks = head_blocks(p, kinds, 4, Four::kTeams, most);
    if (blocks >= 2L * dev_sm_count()) return seq_launch<Four>(name, blocks, 0, st, p);
    blocks = head_blocks(p, kinds, 1, One::kTeams, most);
    return seq_launch<One>(name, blocks, 0, st, p);
  });
}
// blocks of the backward pass; the same for a workspace query, which knows the sizes alone
template <class T>
long head_backward_blocks(HeadParams& p) {
  long n = 0;
  head_by_dim<T>(p.dim, [&](auto lanes) {
    constexpr int L = decltype(lanes)::value;
    n = head_blocks(p, 2, 2, HeadBackward<T, L, 2>::kTeams, 2L * HeadBackward<T, L, 2>::kBlocks * dev_sm_count());
    return (int)S2C_OK;
  });
  return n;
}
template <class T>
int head_backward(HeadParams p, void* dqw, void* dkw, stream_t st) {
  const long blocks = head_backward_blocks<T>(p);
  for (int k = 0; k < 2; ++k) p.kind[k].wide = head_wide(p, p.kind[k], sizeof(T));
  S2C_SEQ_TRY(head_by_dim<T>(p.dim, [&](auto lanes) {
    using K = HeadBackward<T, decltype(lanes)::value, 2>;
    return seq_launch<K>("norm_rotate_backward", blocks, K::smem(), st, p);
  }));
  if (!p.part) return S2C_OK;
  HeadSumParams s = {};
  s.part = p.part; s.dw[0] = dqw; s.dw[1] = dkw; s.dim = p.dim;
  s.blocks[0] = p.kind[0].blocks; s.first[1] = p.kind[0].blocks; s.blocks[1] = p.kind[1].blocks;
  return seq_launch<HeadWeightSum<T>>("norm_rotate_sums", 2L * ((p.dim + 31) / 32), 256 * sizeof(float), st, s);
}

// ---- pages ---------------------------------------------------------------------------------------------------------------
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
  t.array[0] = const_cast<void*>(keys); t.array[1] = const_cast<void*>(values);
  return t;
}
template <class T>
int page_gather(const PageGatherParams& p, stream_t st) {
  const long rows = (long)p.batch * p.length;
  return seq_launch<PageGather<T>>("page_gather", std::min<long>((rows + 7) / 8, 16L * dev_sm_count()), 0, st, p);
}
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
  bool joined = false;
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
    plan.joined = steps > 1;
    plan.part = page_align(2 * (size_t)plan.blocks * K::H::kRows * (decltype(dp)::value + 4) * sizeof(float));
    return (int)S2C_OK;
  });
  plan.bytes = plan.part + (size_t)std::min(plan.items, plan.blocks) * sizeof(int4);
  return plan;
}
template <class T>
int paged_launch(const AttnParams& a, const s2c_page_desc* pages, const void* keys, const void* values, void* ws, size_t ws_bytes, stream_t st) {
  const PagedPlan plan = paged_plan<T>(a);
  if (plan.items == 0) return S2C_OK;
  if (plan.items > 0x7fffffffL || (long)a.lq * a.group > 0x7fffff00L) return fail(S2C_ERR_UNSUPPORTED, "s2c_paged_attention: too many heads and queries");
  if (plan.bytes > ws_bytes || !ws) return fail(S2C_ERR_WORKSPACE, "s2c_paged_attention: workspace too small");
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
    if (!plan.joined) return (int)S2C_OK;
    using J = PagedJoin<T, DP, NT>;
    return seq_launch<J>("paged_join", std::min(plan.items, plan.blocks) * F::H::kRows, J::smem(plan.blocks), st, p);
  });
}
#endif

}  // namespace s2c

using namespace s2c;

extern "C" {

int s2c_norm_rotate(const s2c_head_desc* d, const void* q, const void* k, const void* q_weight, const void* k_weight, void* q_out, void* k_out, void* stream) {
  S2C_SEQ_TRY(head_check("s2c_norm_rotate", d));
  if ((q && !q_out) || (k && !k_out)) return fail(S2C_ERR_BAD_ARG, "s2c_norm_rotate: a pointer is missing");
  HeadParams p = head_params(d);
  p.lengths = nullptr;
  head_kind(p.kind[0], q, p.norm ? q_weight : nullptr, q_out, d->q_stride, d->heads, 1);
  head_kind(p.kind[1], k, p.norm ? k_weight : nullptr, k_out, d->k_stride, d->kv_heads, 1);
  p.kind[0].wide = p.kind[1].wide = 1;
  return d->dtype == kSeqF32 ? head_forward<float>(p, 2, "norm_rotate", (stream_t)stream) : head_forward<bf16>(p, 2, "norm_rotate", (stream_t)stream);
}

size_t s2c_norm_rotate_backward_workspace(const s2c_head_desc* d) {
  if (head_check("s2c_norm_rotate_backward_workspace", d) != S2C_OK || !d->norm) return 0;
  HeadParams p = head_params(d);
  p.kind[0].heads = d->heads;
  p.kind[1].heads = d->kv_heads;
  return (size_t)(d->dtype == kSeqF32 ? head_backward_blocks<float>(p) : head_backward_blocks<bf16>(p)) * d->dim * sizeof(float);
}

int s2c_norm_rotate_backward(const s2c_head_desc* d, const void* q, const void* k, const void* q_weight, const void* k_weight, const void* dq_out,
                             const void* dk_out, void* dq, void* dk, void* dq_weight, void* dk_weight, void* workspace, size_t workspace_bytes,
                             void* stream) {
  S2C_SEQ_TRY(head_check("s2c_norm_rotate_backward", d));
  const bool some = d->batch > 0 && d->length > 0;
  if (some && ((d->heads > 0 && (!q || !dq_out)) || (d->kv_heads > 0 && (!k || !dk_out)))) return fail(S2C_ERR_BAD_ARG, "s2c_norm_rotate_backward: a pointer is missing");
  if ((dq_weight || dk_weight) && !d->norm) return fail(S2C_ERR_BAD_ARG, "s2c_norm_rotate_backward: a weight needs a norm");
  if ((dq_weight && !q_weight) || (dk_weight && !k_weight)) return fail(S2C_ERR_BAD_ARG, "s2c_norm_rotate_backward: the gradient of a weight that is not given");
  const bool sums = dq_weight || dk_weight;
  const size_t need = sums ? s2c_norm_rotate_backward_workspace(d) : 0;
  if (need && (!workspace || workspace_bytes < need)) return fail(S2C_ERR_WORKSPACE, "s2c_norm_rotate_backward: workspace too small");
  if (!on_boundary(workspace, 4)) return fail(S2C_ERR_BAD_ARG, "s2c_norm_rotate_backward: the workspace starts on a 4-byte boundary");
  HeadParams p = head_params(d);
  p.lengths = nullptr;
  static const float none = 0.f;               // (no rows: the sums are written as zeros, nothing is read)
  head_kind(p.kind[0], d->heads ? (q ? q : &none) : nullptr, p.norm ? q_weight : nullptr, dq, d->q_stride, d->heads, 1);
  head_kind(p.kind[1], d->kv_heads ? (k ? k : &none) : nullptr, p.norm ? k_weight : nullptr, dk, d->k_stride, d->kv_heads, 1);
  p.kind[0].dy = dq_out;
  p.kind[1].dy = dk_out;
  p.part = !sums ? nullptr : need ? static_cast<float*>(workspace) : const_cast<float*>(&none);
  return d->dtype == kSeqF32 ? head_backward<float>(p, dq_weight, dk_weight, (stream_t)stream) : head_backward<bf16>(p, dq_weight, dk_weight, (stream_t)stream);
}

int s2c_norm_rotate_store(const s2c_head_desc* d, const s2c_page_desc* pages, const void* q, const void* k, const void* v, const void* q_weight,
                          const void* k_weight, void* q_out, void* keys, void* values, void* stream) {
  S2C_SEQ_TRY(head_check("s2c_norm_rotate_store", d));
  S2C_SEQ_TRY(page_check("s2c_norm_rotate_store", pages));
  if (q && !q_out) return fail(S2C_ERR_BAD_ARG, "s2c_norm_rotate_store: a pointer is missing");
  if (d->batch > 0 && d->length > 0 && d->kv_heads > 0 && (!k || !v || (pages->count > 0 && (!keys || !values))))
    return fail(S2C_ERR_BAD_ARG, "s2c_norm_rotate_store: a pointer is missing");
  HeadParams p = head_params(d);
  p.pages = page_table(pages, keys, values);
  head_kind(p.kind[0], q, p.norm ? q_weight : nullptr, q_out, d->q_stride, d->heads, 1);
  head_kind(p.kind[1], k, p.norm ? k_weight : nullptr, nullptr, d->k_stride, d->kv_heads, 1);
  head_kind(p.kind[2], v, nullptr, nullptr, d->v_stride, d->kv_heads, 0);
  for (int i = 0; i < 3; ++i) {
    p.kind[1].pstride[i] = pages->key_stride[i];
    p.kind[2].pstride[i] = pages->value_stride[i];
  }
  const int size = d->dtype == kSeqF32 ? 4 : 2;
  p.kind[0].wide = 1;
  for (int which = 1; which < 3; ++which) {
    const HeadKind& kind = p.kind[which];
    p.kind[which].wide = on_boundary(p.pages.array[which - 1], 4 * size) && kind.pstride[0] % 4 == 0 && kind.pstride[1] % 4 == 0 && kind.pstride[2] % 4 == 0;
  }
  return d->dtype == kSeqF32 ? head_forward<float>(p, 3, "norm_rotate_store", (stream_t)stream) : head_forward<bf16>(p, 3, "norm_rotate_store", (stream_t)stream);
}

size_t s2c_paged_attention_workspace(const s2c_attention_desc* d, const s2c_page_desc* pages) {
  if (page_check("s2c_paged_attention_workspace", pages) != S2C_OK || attn_check("s2c_paged_attention_workspace", d) != S2C_OK) return 0;
#ifndef S2C_EMUL
  const AttnParams a = paged_params(d, pages, nullptr, nullptr, nullptr);
  return d->dtype == kSeqF32 ? paged_plan<float>(a).bytes : paged_plan<bf16>(a).bytes;
#else
  const s2c_attention_desc g = gathered(d, pages);
  return 2 * gathered_bytes(g) + s2c_attention_workspace(&g);
#endif
}

int s2c_paged_attention(const s2c_attention_desc* d, const s2c_page_desc* pages, const void* q, const void* keys, const void* values, const void* bias,
                        void* out, void* workspace, size_t workspace_bytes, void* stream) {
  S2C_SEQ_TRY(page_check("s2c_paged_attention", pages));
  S2C_SEQ_TRY(attn_check("s2c_paged_attention", d));
  if (d->batch > 0 && d->lq > 0 && (!q || !out || (pages->count > 0 && (!keys || !values)))) return fail(S2C_ERR_BAD_ARG, "s2c_paged_attention: a pointer is missing");
  if ((bias != nullptr) != (d->bucket_of != nullptr)) return fail(S2C_ERR_BAD_ARG, "s2c_paged_attention: a bias needs its buckets, and buckets a bias");
  if (!aligned16(workspace)) return fail(S2C_ERR_BAD_ARG, "s2c_paged_attention: the workspace starts on a 16-byte boundary");
#ifndef S2C_EMUL
  const AttnParams a = paged_params(d, pages, q, bias, out);
  return d->dtype == kSeqF32 ? paged_launch<float>(a, pages, keys, values, workspace, workspace_bytes, (stream_t)stream)
                             : paged_launch<bf16>(a, pages, keys, values, workspace, workspace_bytes, (stream_t)stream);
#else
  const s2c_attention_desc g = gathered(d, pages);
  const size_t need = s2c_paged_attention_workspace(d, pages), part = gathered_bytes(g);
  if (need > workspace_bytes || (need && !workspace)) return fail(S2C_ERR_WORKSPACE, "s2c_paged_attention: workspace too small");
  PageGatherParams p = {};
  p.pages = page_table(pages, keys, values);
  char* at = static_cast<char*>(workspace);
  for (int i = 0; i < 2; ++i) p.out[i] = at + i * part;
  for (int i = 0; i < 3; ++i) { p.stride[0][i] = pages->key_stride[i]; p.stride[1][i] = pages->value_stride[i]; }
  p.q_len = d->q_lengths; p.kv_len = d->kv_lengths; p.start = d->q_starts;
  p.batch = d->batch; p.length = g.lk; p.heads = d->kv_heads; p.dim = d->dim; p.lq = d->lq; p.causal = d->causal; p.start_all = d->q_start;
  if (d->batch > 0 && d->lq > 0) S2C_SEQ_TRY(d->dtype == kSeqF32 ? page_gather<float>(p, (stream_t)stream) : page_gather<bf16>(p, (stream_t)stream));
  return s2c_attention(&g, q, p.out[0], p.out[1], bias, out, nullptr, at + 2 * part, workspace_bytes - 2 * part, stream);
#endif
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
