// C-ABI entry points of the rotation of heads by position (include/s2cnn_b200.h, end of the section on sequences): checks and the
// choice of kernels.  Compiled from heads.cu beside lib.cu; part of lib.cu's translation unit in the host-emulation build.
#pragma once

#include "../../include/s2cnn_b200.h"

#include <algorithm>
#include <cfloat>
#include <cmath>

#include "head_rotation_kernels.h"
#include "kept_pages.h"

namespace s2c {

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
  p.by_length = Divisor(std::max(1, d->length));
  p.each = d->each != 0; p.first = d->start;
  p.eps = d->eps; p.magnitude = d->magnitude; p.over_dim = 1.f / (float)d->dim;
  return p;
}
inline void head_kind(HeadKind& k, const void* x, const void* w, void* out, const long (&stride)[3], int heads, int turn) {
  k.x = x; k.w = w; k.out = out; k.heads = x ? heads : 0; k.turn = turn;
  for (int i = 0; i < 3; ++i) k.stride[i] = stride[i];
}
// Whether a lane's values lie together in pieces of four (halves: whole pieces of pairs, and of what is not turned), and whether those
// lie on their boundaries.  (The weights are read value by value, once per block.)
inline bool head_pieces(const HeadParams& p) { return p.interleaved ? p.dim % 4 == 0 : p.pairs % 4 == 0 && (p.dim - 2 * p.pairs) % 8 == 0; }
inline bool head_wide(const HeadParams& p, int kinds, int size) {
  bool ok = p.dim % 4 == 0 && on_boundary(p.pages.array[0], 4 * size) && on_boundary(p.pages.array[1], 4 * size);
  for (int n = 0; n < kinds; ++n) {
    const HeadKind& k = p.kind[n];
    if (k.heads == 0) continue;
    ok = ok && on_boundary(k.x, 4 * size) && on_boundary(k.dy, 4 * size) && on_boundary(k.out, 4 * size);
    for (int i = 0; i < 3; ++i) ok = ok && k.stride[i] % 4 == 0 && k.pstride[i] % 4 == 0;
  }
  return ok;
}
// Blocks of each kind: one unit for every team where `most` blocks hold them, and the kinds' share of `most` otherwise.
inline long head_blocks(HeadParams& p, int kinds, int group, int span, int teams, long most) {
  long want[3] = {}, all = 0;
  for (int k = 0; k < kinds; ++k) {
    // (a kind's heads in equal units, of whole groups)
    const long spans = (p.kind[k].heads + span - 1) / span;
    const int own = spans ? (int)((p.kind[k].heads + spans * group - 1) / (spans * group)) * group : group;
    p.kind[k].span = own;
    p.kind[k].spans = Divisor(std::max(1L, spans));
    want[k] = ((long)p.batch * p.length * spans + teams - 1) / teams;
    all += want[k];
  }
  long sum = 0, work = 0;
  for (int k = 0; k < kinds; ++k) work += want[k] * p.kind[k].span;
  for (int k = 0; k < kinds; ++k) {
    const long n = all <= most ? want[k] : want[k] ? std::max(1L, (long)((double)want[k] * p.kind[k].span / (double)work * (double)most)) : 0;
    p.kind[k].blocks = (int)n;
    sum += n;
  }
  return sum;
}
// Heads of a unit: the more, the fewer sines and cosines; as many as leave every team that runs at once three units or more (16384
// positions, 20 heads of 128 bfloat16 values: forward 37 us, with the fewest 39; both passes 94 and 107).
inline int head_span(const HeadParams& p, int kinds, int group, long teams) {
  long heads = 0;
  int widest = 0;
  for (int k = 0; k < kinds; ++k) {
    heads += p.kind[k].heads;
    widest = std::max(widest, p.kind[k].heads);
  }
  int span = group;
  while (span < widest && (long)p.batch * p.length * heads / (2 * span) >= 3 * teams) span *= 2;
  return span;
}
// Lanes of a team, how rows lie, pairs of a lane in twos: f(lanes, rows, twos)
template <class F>
int head_by_shape(const HeadParams& p, bool wide, F f) {
  using std::integral_constant;
  if (!head_pieces(p)) {
    integral_constant<int, kHeadByValue> rows;
    if (p.dim <= 32) return f(integral_constant<int, 8>(), rows, integral_constant<int, 1>());
    if (p.dim <= 64) return f(integral_constant<int, 16>(), rows, integral_constant<int, 1>());
    return f(integral_constant<int, 16>(), rows, integral_constant<int, 2>());
  }
  auto lanes = [&](auto rows) {
    if (p.dim <= 32) return f(integral_constant<int, 4>(), rows, integral_constant<int, 2>());
    if (p.dim <= 64) return f(integral_constant<int, 8>(), rows, integral_constant<int, 2>());
    return f(integral_constant<int, 16>(), rows, integral_constant<int, 2>());
  };
  if (p.interleaved) return wide ? lanes(integral_constant<int, kHeadNeighbours>()) : lanes(integral_constant<int, kHeadNeighboursApart>());
  return wide ? lanes(integral_constant<int, kHeadHalves>()) : lanes(integral_constant<int, kHeadHalvesApart>());
}
template <class T>
int head_forward(HeadParams p, int kinds, const char* name, stream_t st) {
  for (int k = 0; k < kinds; ++k)
    if ((long)p.batch * p.length * p.kind[k].heads > 0x7fffffffL) return fail(S2C_ERR_UNSUPPORTED, std::string(name) + ": at most 2^31 heads of all positions");
  return head_by_shape(p, head_wide(p, kinds, sizeof(T)), [&](auto lanes, auto rows, auto twos) {
    constexpr int L = decltype(lanes)::value, R = decltype(rows)::value, P = decltype(twos)::value, G = sizeof(T) == 2 ? 4 : 2;
    using One = HeadForward<T, L, R, P, 1>;
    // As many blocks as run at once, or, with rows that are not filled, twice as many: those of few filled rows make room for others (a
    // first pass of 4 x 2049 positions into pages, ragged 12.4 / 11.4 us, full 13.8 either way; 4 x 4096 without lengths 37 / 39).
    const long at_once = (long)One::kBlocks * dev_sm_count(), teams = at_once * (One::kThreads / L), most = p.lengths ? 2 * at_once : at_once;
    long heads = 0;
    for (int k = 0; k < kinds; ++k) heads += p.kind[k].heads;
    // Single heads where every team has one at most, several of a turn on their way otherwise (single / several: 64 positions, 20 heads of
    // 128 bfloat16 values, 2.7 / 3.5 us; 256, 3.8 / 3.5; 1024, 7.1 / 5.8; 16384, 75 / 37).
    if constexpr (R != kHeadHalvesApart && R != kHeadNeighboursApart) {
      using Many = HeadForward<T, L, R, P, G>;
      if ((long)p.batch * p.length * heads > teams)
        return seq_launch<Many>(name, head_blocks(p, kinds, G, head_span(p, kinds, G, teams), Many::kThreads / L, most), Many::kSmem, st, p);
    }
    return seq_launch<One>(name, head_blocks(p, kinds, 1, 1, One::kThreads / L, most), One::kSmem, st, p);
  });
}
constexpr int kHeadBackwardGroup = 2;
// Most blocks of the backward pass, for a workspace query, which knows the sizes alone: those of the smallest teams' kernels, or of as many
// as run at once.
inline long head_backward_most(const HeadParams& p) {
  return std::min(2L * dev_sm_count(), (long)p.batch * p.length * (p.kind[0].heads + p.kind[1].heads) / 16) + 2;
}
template <class T>
int head_backward(HeadParams p, void* dqw, void* dkw, stream_t st) {
  for (int k = 0; k < 2; ++k)
    if ((long)p.batch * p.length * p.kind[k].heads > 0x7fffffffL) return fail(S2C_ERR_UNSUPPORTED, "norm_rotate: at most 2^31 heads of all positions");
  S2C_SEQ_TRY(head_by_shape(p, head_wide(p, 2, sizeof(T)), [&](auto lanes, auto rows, auto twos) {
    constexpr int G = kHeadBackwardGroup;
    using K = HeadBackward<T, decltype(lanes)::value, decltype(rows)::value, decltype(twos)::value, G>;
    const long most = (long)K::kBlocks * dev_sm_count(), teams = K::kThreads / decltype(lanes)::value;
    return seq_launch<K>("norm_rotate_backward", head_blocks(p, 2, G, head_span(p, 2, G, most * teams), (int)teams, most), K::kSmem, st, p);
  }));
  if (!p.part) return S2C_OK;
  HeadSumParams s = {};
  s.part = p.part; s.dw[0] = dqw; s.dw[1] = dkw; s.dim = p.dim;
  s.blocks[0] = p.kind[0].blocks; s.first[1] = p.kind[0].blocks; s.blocks[1] = p.kind[1].blocks;
  return seq_launch<HeadWeightSum<T>>("norm_rotate_sums", 2L * ((p.dim + 31) / 32), 256 * sizeof(float), st, s);
}

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
  return d->dtype == kSeqF32 ? head_forward<float>(p, 2, "norm_rotate", (stream_t)stream) : head_forward<bf16>(p, 2, "norm_rotate", (stream_t)stream);
}

size_t s2c_norm_rotate_backward_workspace(const s2c_head_desc* d) {
  if (head_check("s2c_norm_rotate_backward_workspace", d) != S2C_OK || !d->norm) return 0;
  HeadParams p = head_params(d);
  p.kind[0].heads = d->heads;
  p.kind[1].heads = d->kv_heads;
  return (size_t)head_backward_most(p) * d->dim * sizeof(float);
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
  return d->dtype == kSeqF32 ? head_forward<float>(p, 3, "norm_rotate_store", (stream_t)stream) : head_forward<bf16>(p, 3, "norm_rotate_store", (stream_t)stream);
}

}  // extern "C"
