// C-ABI entry points of the operators for sequences of signals (the last section of include/s2cnn_b200.h): checks and the
// choice of kernels.  Compiled from sequence.cu beside lib.cu; part of lib.cu's translation unit in the host-emulation build.
#pragma once

#include "../../include/s2cnn_b200.h"

#include <algorithm>
#include <atomic>
#include <cmath>

#include "attention_few.h"
#include "attention_kernels.h"
#include "attention_tc_backward.h"
#include "attention_tc3.h"
#include "attention_tc_forward.h"
#include "dropout_kernels.h"
#include "layer_norm_kernels.h"

namespace s2c {

// ---- layer norm --------------------------------------------------------------------------------------------------------
// A row takes the fewest threads that hold it, and the next one as it lies in memory, in their registers: neighbouring lanes up
// to 1024 columns (512 of float32), a block of 128 up to 4096 (2048), of 512 beyond.
constexpr int kNormMaxCols = 16384;
template <class F>
int norm_by_cols(int cols, int size, F f) {
#define S2C_NORM(T, EPT) return f(std::integral_constant<int, T>(), std::integral_constant<int, EPT>())
  if (cols <= 32) S2C_NORM(4, 8);
  if (cols <= 128) S2C_NORM(16, 8);
  if (cols <= 256) S2C_NORM(32, 8);
  if (cols <= 512) S2C_NORM(32, 16);
  if (cols <= 1024 && size == 2) S2C_NORM(32, 32);
  if (cols <= 2048) S2C_NORM(128, 16);
  if (cols <= 4096 && size == 2) S2C_NORM(128, 32);
  if (cols <= 8192) S2C_NORM(512, 16);
  S2C_NORM(512, 32);
#undef S2C_NORM
}
inline int norm_bwd_blocks(long rows, int cols, int size) {
  return norm_by_cols(cols, size, [&](auto t, auto ept) {
    using K = LayerNormBwd<float, decltype(t)::value, decltype(ept)::value, 1>;
    return (int)std::min<long>((rows + K::kTeams - 1) / K::kTeams, (long)dev_sm_count() * K::kBlocks);
  });
}
template <class T>
int norm_forward(LayerNormParams p, stream_t st) {
  const bool vec = p.cols % kVec<T> == 0;
  p.wide = vec && aligned16(p.x) && aligned16(p.y) && aligned16(p.w) && aligned16(p.b);
  return norm_by_cols(p.cols, sizeof(T), [&](auto t, auto ept) {
    constexpr int TT = decltype(t)::value, E = decltype(ept)::value;
    using V = LayerNormFwd<T, TT, E, kVec<T>>;
    using S = LayerNormFwd<T, TT, E, 1>;
    const long blocks = std::min<long>((p.rows + V::kTeams - 1) / V::kTeams, (long)dev_sm_count() * V::kBlocks);
    return vec ? seq_launch<V>("layer_norm", blocks, V::smem(), st, p) : seq_launch<S>("layer_norm", blocks, S::smem(), st, p);
  });
}
template <class T>
int norm_backward(LayerNormParams p, void* dw, void* db, stream_t st) {
  const int blocks = norm_bwd_blocks(p.rows, p.cols, sizeof(T));
  const bool vec = p.cols % kVec<T> == 0;
  p.wide = vec && aligned16(p.x) && aligned16(p.dy) && aligned16(p.dx) && aligned16(p.w);
  S2C_SEQ_TRY(norm_by_cols(p.cols, sizeof(T), [&](auto t, auto ept) {
    constexpr int TT = decltype(t)::value, E = decltype(ept)::value;
    using V = LayerNormBwd<T, TT, E, kVec<T>>;
    using S = LayerNormBwd<T, TT, E, 1>;
    return vec ? seq_launch<V>("layer_norm_backward", blocks, V::smem(), st, p)
               : seq_launch<S>("layer_norm_backward", blocks, S::smem(), st, p);
  }));
  if (!p.part) return S2C_OK;
  LayerNormSumParams s;
  s.part = p.part; s.dw = dw; s.db = db; s.blocks = blocks; s.cols = p.cols;
  return seq_launch<LayerNormSum<T>>("layer_norm_sums", (2L * p.cols + 31) / 32, 256 * sizeof(float), st, s);
}

// ---- dropout -----------------------------------------------------------------------------------------------------------
inline int dropout(const char* who, int dtype, DropoutParams p, const void* x, const void* residual, void* out, long n, double probability, stream_t st) {
  S2C_SEQ_TRY(seq_check_type(who, dtype));
  if (n < 0 || (n > 0 && (!x || !out)) || !(probability >= 0. && probability < 1.)) return fail(S2C_ERR_BAD_ARG, std::string(who) + ": bad argument");
  p.x = x; p.residual = residual; p.out = out; p.n = n;
  p.threshold = (unsigned)std::floor(probability * 4294967296.);
  p.scale = (float)(1. / (1. - probability));
  const bool vec = aligned16(x) && aligned16(residual) && aligned16(out);
  auto go = [&](auto k) {
    using K = typename decltype(k)::type;
    const long blocks = (n + (long)K::kThreads * K::kStep - 1) / ((long)K::kThreads * K::kStep);
    return seq_launch<K>("dropout", std::min<long>(blocks, 32L * dev_sm_count()), 0, st, p);
  };
  struct A { using type = Dropout<float, true>; };
  struct B { using type = Dropout<float, false>; };
  struct C { using type = Dropout<bf16, true>; };
  struct D { using type = Dropout<bf16, false>; };
  return dtype == kSeqF32 ? (vec ? go(A()) : go(B())) : (vec ? go(C()) : go(D()));
}

// ---- attention ---------------------------------------------------------------------------------------------------------
// what the library lays out itself; the caller's arrays need no more alignment than their type
inline int attn_check_own(const char* who, const void* saved, const void* workspace) {
  return aligned16(saved) && aligned16(workspace) ? S2C_OK : fail(S2C_ERR_BAD_ARG, std::string(who) + ": saved and workspace start on 16-byte boundaries");
}
inline AttnParams attn_params(const s2c_attention_desc* d, const void* q, const void* k, const void* v, const void* bias) {
  AttnParams p = {};
  p.q = q; p.k = k; p.v = v; p.bias = d->bucket_of ? bias : nullptr;
  p.bucket_of = d->bucket_of; p.start = d->q_starts; p.q_len = d->q_lengths; p.kv_len = d->kv_lengths;
  for (int i = 0; i < 3; ++i) { p.qs[i] = d->q_stride[i]; p.ks[i] = d->k_stride[i]; p.vs[i] = d->v_stride[i]; }
  p.batch = d->batch; p.lq = d->lq; p.lk = d->lk; p.heads = d->heads; p.kv_heads = d->kv_heads; p.dim = d->dim;
  p.group = d->heads / d->kv_heads;
  p.causal = d->causal != 0; p.scale = d->scale; p.start_all = d->q_start;
  p.reach = p.bias ? d->reach : 0; p.n_buckets = p.bias ? d->n_buckets : 0; p.bias_grad = p.bias && d->bias_grad;
  p.splits = 1;
  return p;
}
template <class T, class F>
int attn_by_dim(int dim, F f) {
  if (dim <= 16) return f(std::integral_constant<int, 16>());
  if (dim <= 32) return f(std::integral_constant<int, 32>());
  if (dim <= 64) return f(std::integral_constant<int, 64>());
  return f(std::integral_constant<int, 128>());
}
inline int attn_padded(int dim) { return dim <= 16 ? 16 : dim <= 32 ? 32 : dim <= 64 ? 64 : 128; }

inline size_t attn_align(size_t n) { return (n + 255) / 256 * 256; }
// What the backward pass needs beside the output: the statistics of the rows, and in bfloat16 what the rounding of the output
// left.  delta = dO . O is one error for a whole row of dS, which the bias gradient sums over all rows: with the rounded output
// its relative error is 3.1e-3 (8 x 1000 positions, 8 heads of 64), with the rest 1.9e-3, which is its own rounding.
inline size_t attn_stats_bytes(const AttnParams& p) { return attn_align((size_t)p.batch * p.heads * p.lq * sizeof(float2)); }
inline size_t attn_saved_bytes(const AttnParams& p, int dtype) {
  return attn_stats_bytes(p) + (dtype == kSeqBf16 ? (size_t)p.batch * p.lq * p.heads * p.dim * 2 : 0);
}
inline void attn_set_saved(AttnParams& p, int dtype, void* saved) {
  if (!saved) return;
  p.stats = static_cast<float2*>(saved);
  if (dtype == kSeqBf16) p.out_lo = static_cast<char*>(saved) + attn_stats_bytes(p);
}

#ifndef S2C_EMUL
// Few rows per key head: chunks of keys, six blocks per SM of them where there are as many keys (lengths differ: what is short
// ends early), at least 256 keys each.
inline bool attn_few_rows(const AttnParams& p) { return (long)p.lq * p.group <= kFewRows; }
inline void attn_split(AttnParams& p) {
  const long blocks = std::max(1L, (long)p.batch * p.kv_heads), pieces = std::max(1, (p.lk + 255) / 256);
  const long want = std::min(pieces, std::max(1L, 6L * dev_sm_count() / blocks)), per = (pieces + want - 1) / want;
  p.chunk = (int)per * 256;
  p.splits = (int)((pieces + per - 1) / per);
}
inline size_t attn_split_bytes(const AttnParams& p) {
  return p.splits > 1 ? (size_t)p.batch * p.kv_heads * p.splits * p.lq * p.group * (attn_padded(p.dim) + 2) * sizeof(float) : 0;
}
// the largest pieces that rows of k and v can be copied in
template <class T>
int attn_few_piece(const AttnParams& p) {
  auto fits = [&](int bytes) {
    const long n = bytes / (long)sizeof(T);
    bool ok = reinterpret_cast<uintptr_t>(p.k) % bytes == 0 && reinterpret_cast<uintptr_t>(p.v) % bytes == 0 && p.dim % n == 0;
    for (int i = 0; i < 3; ++i) ok = ok && p.ks[i] % n == 0 && p.vs[i] % n == 0;
    return ok;
  };
  return fits(16) ? 16 : fits(4) ? 4 : 2;
}
// The bias tables of all heads of a group have to lie beside the tiles.  Heads of more than 64 values, float32: not from a reach of 208
// on with 16 heads per key head, 416 with 8, 832 with 4, 1664 with 2; bfloat16 and smaller heads have more room (bfloat16, 128 values, 16
// heads: up to 999).  Such calls take the tiles of 64 or 128 queries.
template <class T>
bool attn_few_fits(const AttnParams& p) {
  return attn_few_rows(p) && attn_by_dim<T>(p.dim, [&](auto d) {
    return (int)(AttnFew<T, decltype(d)::value, 4>::smem(p) <= (size_t)dev_smem_limit());
  });
}
template <class T>
int attn_few(AttnParams p, void* ws, size_t ws_bytes, stream_t st) {
  attn_split(p);
  if (attn_split_bytes(p) > ws_bytes || (p.splits > 1 && !ws)) return fail(S2C_ERR_WORKSPACE, "s2c_attention: workspace too small");
  p.part = static_cast<float*>(ws);
  const int piece = attn_few_piece<T>(p);
  return attn_by_dim<T>(p.dim, [&](auto d) {
    constexpr int DP = decltype(d)::value;
    const long grid = (long)p.batch * p.kv_heads * p.splits;
    auto go = [&](auto k) {
      using K = typename decltype(k)::type;
      return seq_launch<K>("attention_few", grid, K::smem(p), st, p);
    };
    struct A { using type = AttnFew<T, DP, 16>; };
    struct B { using type = AttnFew<T, DP, 4>; };
    struct C { using type = AttnFew<T, DP, sizeof(T) == 2 ? 2 : 4>; };
    S2C_SEQ_TRY(piece == 16 ? go(A()) : piece == 4 ? go(B()) : go(C()));
    if (p.splits == 1) return (int)S2C_OK;
    using J = AttnJoin<T, DP>;
    return seq_launch<J>("attention_join", (long)p.batch * p.kv_heads * p.lq * p.group, J::smem(p), st, p);
  });
}
#endif
#ifndef S2C_EMUL
// ---- tensor-core kernels: which calls they take, and the packed copies they need
// Rows that they can fetch in 16-byte pieces, as far as sizes and strides tell: others are packed first, as float32 always is.
// (Bases that are not aligned to 16 bytes, with rows that would be: not on the tensor cores.  A workspace query does not see
// them; the Python functions copy such a tensor.)
inline bool attn_pieces(const long (&stride)[3], int dim) { return dim % 8 == 0 && stride[0] % 8 == 0 && stride[1] % 8 == 0 && stride[2] % 8 == 0; }
inline bool attn_packs(const AttnParams& p, int size) {
  return size == 4 || !(attn_pieces(p.qs, p.dim) && attn_pieces(p.ks, p.dim) && attn_pieces(p.vs, p.dim));
}
static std::atomic<int> g_attention{0};      // test switch: 0 by size, 1 never the tensor-core kernels, 2 always

// Packed copies of q, k, v (and dout) in a workspace: three parts of float32, one of bfloat16.
struct AttnPacked {
  int tensors = 0, chunks = 0;
  size_t at[4], bytes = 0;
  long part[4];
};
inline AttnPacked attn_packed(const AttnParams& p, int size, int tensors) {
  AttnPacked k;
  k.tensors = tensors;
  k.chunks = (p.dim + 7) / 8;
  for (int t = 0; t < tensors; ++t) {
    const bool of_q = t == 0 || t == 3;
    k.part[t] = (long)p.batch * (of_q ? p.lq : p.lk) * (of_q ? p.heads : p.kv_heads) * 8 * k.chunks;
    k.at[t] = k.bytes;
    k.bytes += attn_align((size_t)k.part[t] * sizeof(bf16) * (size == 4 ? 3 : 1));
  }
  return k;
}
// launches the copies into `ws` and turns t's operands to them
template <class T>
int attn_pack(AttnTcParams& t, const AttnPacked& k, char* ws, stream_t st) {
  AttnParams& p = t.a;
  AttnPackParams c = {};
  const void* src[4] = {p.q, p.k, p.v, p.dout};
  const long* stride[4] = {p.qs, p.ks, p.vs, t.gs};
  long most = 0;
  c.a = p;
  c.tensors = k.tensors; c.batch = p.batch; c.dim = p.dim; c.chunks = k.chunks;
  for (int i = 0; i < k.tensors; ++i) {
    const bool of_q = i == 0 || i == 3;
    c.src[i] = src[i];
    c.dst[i] = reinterpret_cast<bf16*>(ws + k.at[i]);
    for (int e = 0; e < 3; ++e) c.stride[i][e] = stride[i][e];
    c.part[i] = k.part[i];
    c.len[i] = of_q ? p.lq : p.lk;
    c.heads[i] = of_q ? p.heads : p.kv_heads;
    most = std::max(most, k.part[i] / 8);
  }
  S2C_SEQ_TRY(seq_launch<AttnPack<T>>("attention_pack", k.tensors * std::min<long>((most + 255) / 256, 4L * dev_sm_count()), 0, st, c));
  const long row = 8L * k.chunks;
  auto turn = [&](const void*& x, long* s, long& part, int i) {
    x = c.dst[i];
    s[0] = row * c.len[i] * c.heads[i];
    s[1] = row;
    s[2] = row * c.len[i];
    part = k.part[i];
  };
  turn(p.q, p.qs, t.q_split, 0);
  turn(p.k, p.ks, t.k_split, 1);
  turn(p.v, p.vs, t.v_split, 2);
  if (k.tensors > 3) turn(p.dout, t.gs, t.g_split, 3);
  t.chunks = k.chunks;
  return S2C_OK;
}
// Whether a call is worth the tensor cores.  Rows they can fetch: always (tiles of 64 on the FP32 pipes / tensor cores, forward and
// backward: 32 x 17 positions, 4 heads of 64, 66 / 49 us; 32 x 60, 82 / 48).  Rows to be packed: from 96 x 96 scores per head on
// (float32, 4 x 100, 4 heads of 64, packing included: 98 / 76 us; 32 x 60, 4 heads of 10: 49 / 67; 128 x 60, 8 of 32: 195 / 260).
inline bool attn_tc_worth(const AttnParams& p, bool packed) {
  const int mode = g_attention.load(std::memory_order_relaxed);
  if (p.batch < 1 || p.lq < 1 || p.lk < 1 || mode == 1) return false;
  if (mode == 2) return true;
  return !packed || (long)p.lq * p.lk >= 96 * 96;
}
template <class T>
bool attn_forward_tc(const AttnParams& p) {
  const bool packed = attn_packs(p, sizeof(T));
  if (!packed && !(aligned16(p.q) && aligned16(p.k) && aligned16(p.v))) return false;
  const size_t smem = sizeof(T) == 4 ? (p.dim > 64 ? AttnTc3Forward<2>::smem(p.reach) : AttnTc3Forward<1>::smem(p.reach)) : tcf_smem(p.dim > 64 ? 2 : 1, 1, p.reach);
  return attn_tc_worth(p, packed) && smem <= (size_t)dev_smem_limit();
}
template <class T>
int attn_tc_forward_launch(const AttnParams& p, char* ws, size_t ws_bytes, stream_t st) {
  AttnTcParams t = {};
  t.a = p;
  t.chunks = p.dim / 8;
  if (attn_packs(p, sizeof(T))) {
    const AttnPacked k = attn_packed(p, sizeof(T), 3);
    if (k.bytes > ws_bytes || !ws) return fail(S2C_ERR_WORKSPACE, "s2c_attention: workspace too small");
    S2C_SEQ_TRY(attn_pack<T>(t, k, ws, st));
  }
  const int nc = p.dim > 64 ? 2 : 1;
  if constexpr (sizeof(T) == 4) {
    t.a.tiles = (p.lq + 127) / 128;
    const long blocks = (long)p.batch * p.heads * t.a.tiles;
    return nc == 1 ? attn_tc_launch<AttnTc3Forward<1>>("attention_tc3", blocks, AttnTc3Forward<1>::smem(p.reach), st, t)
                   : attn_tc_launch<AttnTc3Forward<2>>("attention_tc3", blocks, AttnTc3Forward<2>::smem(p.reach), st, t);
  } else {
    t.units = (p.lq + 127) / 128 * p.group;
    const long heads = (long)p.batch * p.kv_heads;
    t.per_block = heads * ((t.units + 1) / 2) >= dev_sm_count() && tcf_smem(nc, 2, p.reach) <= (size_t)dev_smem_limit() ? 2 : 1;
    t.pairs = (t.units + t.per_block - 1) / t.per_block;
    // The last wave of blocks, where it fills half of the SMs at most: one tile per block, in two thirds of a pair's time (2 x 4096
    // positions, 16 heads, 512 pairs on 148 SMs: of 128 values 269 us without, 257 with; of 64, in training, 229 / 221).
    const long blocks = heads * t.pairs, rest = blocks % dev_sm_count();
    const bool halve = t.per_block == 2 && rest > 0 && rest <= dev_sm_count() / 2;
    t.whole = (int)(halve ? blocks - rest : blocks);
    const long grid = blocks + (halve ? rest : 0);
    const size_t smem = tcf_smem(nc, t.per_block, p.reach);
    if (p.bias_grad)
      return nc == 1 ? attn_tc_launch<AttnTcForward<1, true>>("attention_tc", grid, smem, st, t)
                     : attn_tc_launch<AttnTcForward<2, true>>("attention_tc", grid, smem, st, t);
    return nc == 1 ? attn_tc_launch<AttnTcForward<1, false>>("attention_tc", grid, smem, st, t)
                   : attn_tc_launch<AttnTcForward<2, false>>("attention_tc", grid, smem, st, t);
  }
}
#endif
template <class T>
size_t attn_forward_bytes(AttnParams p) {
#ifndef S2C_EMUL
  if (attn_few_rows(p)) {
    attn_split(p);
    if (attn_few_fits<T>(p)) return attn_split_bytes(p);
  }
  if (attn_packs(p, sizeof(T)) && attn_forward_tc<T>(p)) return attn_packed(p, sizeof(T), 3).bytes;
#endif
  return 0;
}
template <class T>
int attn_forward(AttnParams p, void* ws, size_t ws_bytes, stream_t st) {
  if (p.batch == 0 || p.lq == 0) return S2C_OK;
#ifndef S2C_EMUL
  if (attn_few_fits<T>(p)) return attn_few<T>(p, ws, ws_bytes, st);
  if (attn_forward_tc<T>(p)) return attn_tc_forward_launch<T>(p, static_cast<char*>(ws), ws_bytes, st);
#endif
  p.tiles = (p.lq + kAttnTile - 1) / kAttnTile;
  return attn_by_dim<T>(p.dim, [&](auto d) {
    using K = AttnForward<T, decltype(d)::value>;
    return seq_launch<K>("attention", (long)p.batch * p.heads * p.tiles, K::smem(p), st, p);
  });
}

inline size_t attn_delta_bytes(const AttnParams& p) { return attn_align((size_t)p.batch * p.heads * p.lq * sizeof(float)); }
inline size_t attn_parts_bytes(const AttnParams& p, bool with_bias) {
  const size_t tiles = (p.lq + kAttnTile - 1) / kAttnTile;
  return with_bias ? attn_align((size_t)p.batch * tiles * p.heads * p.n_buckets * sizeof(float)) : 0;
}
#ifndef S2C_EMUL
template <class T>
bool attn_backward_tc(const AttnParams& p, bool with_bias) {
  const bool packed = attn_packs(p, sizeof(T));
  if (!packed && !(aligned16(p.q) && aligned16(p.k) && aligned16(p.v) && aligned16(p.dout))) return false;
  const int nc = p.dim > 64 ? 2 : 1;
  const size_t q = sizeof(T) == 4 ? (nc == 1 ? AttnTc3GradQ<1>::smem(p.reach, with_bias) : AttnTc3GradQ<2>::smem(p.reach, with_bias)) : nc == 1 ? AttnTcGradQ<1>::smem(p.reach, with_bias) : AttnTcGradQ<2>::smem(p.reach, with_bias);
  const size_t kv = sizeof(T) == 4 ? (nc == 1 ? AttnTc3GradKV<1>::smem(p.reach) : AttnTc3GradKV<2>::smem(p.reach)) : nc == 1 ? AttnTcGradKV<1>::smem(p.reach) : AttnTcGradKV<2>::smem(p.reach);
  return attn_tc_worth(p, packed) && std::max(q, kv) <= (size_t)dev_smem_limit();
}
template <class T>
int attn_tc_backward_launch(AttnParams& p, char* packs, stream_t st) {
  AttnTcParams t = {};
  t.gs[0] = (long)p.lq * p.heads * p.dim;
  t.gs[1] = (long)p.heads * p.dim;
  t.gs[2] = p.dim;
  t.grad = p.dout;
  t.chunks = p.dim / 8;
  p.tiles = (p.lq + 127) / 128;
  t.a = p;
  if (attn_packs(p, sizeof(T))) S2C_SEQ_TRY(attn_pack<T>(t, attn_packed(p, sizeof(T), 4), packs, st));
  const int nc = p.dim > 64 ? 2 : 1;
  const bool bias_grad = p.dbias_part != nullptr;
  const long q_blocks = (long)p.batch * p.heads * p.tiles, kv_tiles = (p.lk + 127) / 128, kv_blocks = (long)p.batch * p.kv_heads * kv_tiles;
  if constexpr (sizeof(T) == 4) {
    S2C_SEQ_TRY(nc == 1 ? attn_tc_launch<AttnTc3GradQ<1>>("attention_tc3_grad_q", q_blocks, AttnTc3GradQ<1>::smem(p.reach, bias_grad), st, t)
                        : attn_tc_launch<AttnTc3GradQ<2>>("attention_tc3_grad_q", q_blocks, AttnTc3GradQ<2>::smem(p.reach, bias_grad), st, t));
    t.a.tiles = (int)kv_tiles;
    return nc == 1 ? attn_tc_launch<AttnTc3GradKV<1>>("attention_tc3_grad_kv", kv_blocks, AttnTc3GradKV<1>::smem(p.reach), st, t)
                   : attn_tc_launch<AttnTc3GradKV<2>>("attention_tc3_grad_kv", kv_blocks, AttnTc3GradKV<2>::smem(p.reach), st, t);
  } else {
    S2C_SEQ_TRY(nc == 1 ? attn_tc_launch<AttnTcGradQ<1>>("attention_tc_grad_q", q_blocks, AttnTcGradQ<1>::smem(p.reach, bias_grad), st, t)
                        : attn_tc_launch<AttnTcGradQ<2>>("attention_tc_grad_q", q_blocks, AttnTcGradQ<2>::smem(p.reach, bias_grad), st, t));
    t.a.tiles = (int)kv_tiles;
    return nc == 1 ? attn_tc_launch<AttnTcGradKV<1>>("attention_tc_grad_kv", kv_blocks, AttnTcGradKV<1>::smem(p.reach), st, t)
                   : attn_tc_launch<AttnTcGradKV<2>>("attention_tc_grad_kv", kv_blocks, AttnTcGradKV<2>::smem(p.reach), st, t);
  }
}
#endif
// (asked without pointers: then as if all were aligned)
template <class T>
size_t attn_backward_bytes(const AttnParams& p, bool with_bias) {
  size_t n = attn_delta_bytes(p) + attn_parts_bytes(p, with_bias);
#ifndef S2C_EMUL
  if (attn_packs(p, sizeof(T)) && attn_backward_tc<T>(p, with_bias)) n += attn_packed(p, sizeof(T), 4).bytes;
#endif
  return n;
}
template <class T>
int attn_backward(AttnParams p, void* dbias, void* ws, size_t ws_bytes, stream_t st) {
  const size_t need = attn_backward_bytes<T>(p, dbias != nullptr);
  if (need > ws_bytes || (need && !ws)) return fail(S2C_ERR_WORKSPACE, "s2c_attention_backward: workspace too small");
  char* const at = static_cast<char*>(ws);
  p.delta = reinterpret_cast<float*>(at);
  p.dbias_part = dbias ? reinterpret_cast<float*>(at + attn_delta_bytes(p)) : nullptr;
  bool done = false;
#ifndef S2C_EMUL
  done = attn_backward_tc<T>(p, dbias != nullptr);
  if (done) S2C_SEQ_TRY(attn_tc_backward_launch<T>(p, at + attn_delta_bytes(p) + attn_parts_bytes(p, dbias != nullptr), st));
#endif
  if (!done) S2C_SEQ_TRY(attn_by_dim<T>(p.dim, [&](auto d) {
    constexpr int DP = decltype(d)::value;
    using Q = AttnGradQ<T, DP>;
    using KV = AttnGradKV<T, DP>;
    p.tiles = (p.lq + kAttnTile - 1) / kAttnTile;
    S2C_SEQ_TRY(seq_launch<Q>("attention_grad_q", (long)p.batch * p.heads * p.tiles, Q::smem(p), st, p));
    AttnParams kv = p;
    kv.tiles = (p.lk + kAttnTile - 1) / kAttnTile;
    return seq_launch<KV>("attention_grad_kv", (long)p.batch * p.kv_heads * kv.tiles, KV::smem(kv), st, kv);
  }));
  if (!dbias) return S2C_OK;
  AttnBiasSumParams s;
  s.part = p.dbias_part; s.out = dbias; s.parts = p.batch * p.tiles; s.heads = p.heads; s.n_buckets = p.n_buckets;
  return seq_launch<AttnBiasSum<T>>("attention_bias_sums", ((long)p.heads * p.n_buckets + 7) / 8, 256 * sizeof(float), st, s);
}

}  // namespace s2c

using namespace s2c;

extern "C" {

int s2c_layer_norm(int dtype, const void* x, const void* weight, const void* bias, void* y, float* stats, long rows, int cols,
                   float eps, void* stream) {
  S2C_SEQ_TRY(seq_check_type("s2c_layer_norm", dtype));
  if (rows < 0 || cols < 1 || (rows > 0 && (!x || !y)) || !(eps >= 0.f)) return fail(S2C_ERR_BAD_ARG, "s2c_layer_norm: bad argument");
  if (cols > kNormMaxCols) return fail(S2C_ERR_UNSUPPORTED, "s2c_layer_norm: at most 16384 columns");
  LayerNormParams p = {};
  p.x = x; p.w = weight; p.b = bias; p.y = y; p.stats = stats; p.rows = rows; p.cols = cols; p.eps = eps;
  return dtype == kSeqF32 ? norm_forward<float>(p, (stream_t)stream) : norm_forward<bf16>(p, (stream_t)stream);
}

size_t s2c_layer_norm_backward_workspace(long rows, int cols) {
  if (rows < 1 || cols < 1 || cols > kNormMaxCols) return 0;
  return (size_t)std::max(norm_bwd_blocks(rows, cols, 2), norm_bwd_blocks(rows, cols, 4)) * 2 * cols * sizeof(float);
}

int s2c_layer_norm_backward(int dtype, const void* x, const void* weight, const float* stats, const void* dy, void* dx, void* dweight,
                            void* dbias, long rows, int cols, void* workspace, size_t workspace_bytes, void* stream) {
  S2C_SEQ_TRY(seq_check_type("s2c_layer_norm_backward", dtype));
  if (rows < 0 || cols < 1 || (rows > 0 && (!x || !dy || !stats))) return fail(S2C_ERR_BAD_ARG, "s2c_layer_norm_backward: bad argument");
  if (cols > kNormMaxCols) return fail(S2C_ERR_UNSUPPORTED, "s2c_layer_norm_backward: at most 16384 columns");
  const bool sums = dweight || dbias;
  const size_t need = sums ? s2c_layer_norm_backward_workspace(rows, cols) : 0;
  if (need && (!workspace || workspace_bytes < need)) return fail(S2C_ERR_WORKSPACE, "s2c_layer_norm_backward: workspace too small");
  LayerNormParams p = {};
  static float none;           // (no rows: the sums are written as zeros, nothing is read)
  p.x = x; p.w = weight; p.dy = dy; p.dx = dx; p.stats = const_cast<float*>(stats); p.rows = rows; p.cols = cols;
  p.part = !sums ? nullptr : need ? static_cast<float*>(workspace) : &none;
  return dtype == kSeqF32 ? norm_backward<float>(p, dweight, dbias, (stream_t)stream) : norm_backward<bf16>(p, dweight, dbias, (stream_t)stream);
}

int s2c_dropout(int dtype, const void* x, const void* residual, void* out, long n, double probability, unsigned long long seed,
                unsigned long long step, void* stream) {
  DropoutParams p = {};
  for (int i = 0; i < 2; ++i) {
    p.key[i] = (unsigned)(seed >> (32 * i));
    p.step[i] = (unsigned)(step >> (32 * i));
  }
  return dropout("s2c_dropout", dtype, p, x, residual, out, n, probability, (stream_t)stream);
}

int s2c_dropout_numbers(int dtype, const void* x, const void* residual, void* out, long n, double probability,
                        const unsigned long long* numbers, void* stream) {
  if (!numbers || reinterpret_cast<uintptr_t>(numbers) % 8) return fail(S2C_ERR_BAD_ARG, "s2c_dropout_numbers: no seed and step, or not aligned to their type");
  DropoutParams p = {};
  p.numbers = numbers;
  return dropout("s2c_dropout_numbers", dtype, p, x, residual, out, n, probability, (stream_t)stream);
}

size_t s2c_attention_workspace(const s2c_attention_desc* d) {
  if (attn_check("s2c_attention_workspace", d) != S2C_OK) return 0;
  const AttnParams p = attn_params(d, nullptr, nullptr, nullptr, d->bucket_of);
  return d->dtype == kSeqF32 ? attn_forward_bytes<float>(p) : attn_forward_bytes<bf16>(p);
}

size_t s2c_attention_saved_bytes(const s2c_attention_desc* d) {
  if (attn_check("s2c_attention_saved_bytes", d) != S2C_OK) return 0;
  return attn_saved_bytes(attn_params(d, nullptr, nullptr, nullptr, nullptr), d->dtype);
}

int s2c_attention(const s2c_attention_desc* d, const void* q, const void* k, const void* v, const void* bias, void* out, void* saved,
                  void* workspace, size_t workspace_bytes, void* stream) {
  S2C_SEQ_TRY(attn_check("s2c_attention", d));
  const bool some = d->batch > 0 && d->lq > 0;
  if (some && (!q || !out || (d->lk > 0 && (!k || !v)))) return fail(S2C_ERR_BAD_ARG, "s2c_attention: a pointer is missing");
  if ((bias != nullptr) != (d->bucket_of != nullptr)) return fail(S2C_ERR_BAD_ARG, "s2c_attention: a bias needs its buckets, and buckets a bias");
  AttnParams p = attn_params(d, q, k, v, bias);
  S2C_SEQ_TRY(attn_check_own("s2c_attention", saved, workspace));
  p.out = out;
  attn_set_saved(p, d->dtype, saved);
  return d->dtype == kSeqF32 ? attn_forward<float>(p, workspace, workspace_bytes, (stream_t)stream)
                             : attn_forward<bf16>(p, workspace, workspace_bytes, (stream_t)stream);
}

size_t s2c_attention_backward_workspace(const s2c_attention_desc* d) {
  if (attn_check("s2c_attention_backward_workspace", d) != S2C_OK) return 0;
  AttnParams p = attn_params(d, nullptr, nullptr, nullptr, d->bucket_of);
  // (whether the gradient of a bias is wanted is not known here)
  auto bytes = [&](bool with_bias) { return d->dtype == kSeqF32 ? attn_backward_bytes<float>(p, with_bias) : attn_backward_bytes<bf16>(p, with_bias); };
  return std::max(bytes(d->bucket_of != nullptr), bytes(false));
}

int s2c_attention_backward(const s2c_attention_desc* d, const void* q, const void* k, const void* v, const void* bias, const void* out,
                           const void* saved, const void* dout, void* dq, void* dk, void* dv, void* dbias, void* workspace,
                           size_t workspace_bytes, void* stream) {
  S2C_SEQ_TRY(attn_check("s2c_attention_backward", d));
  if (d->batch > 0 && d->lq > 0 && (!q || !out || !saved || !dout || !dq)) return fail(S2C_ERR_BAD_ARG, "s2c_attention_backward: a pointer is missing");
  if (d->batch > 0 && d->lk > 0 && (!k || !v || !dk || !dv)) return fail(S2C_ERR_BAD_ARG, "s2c_attention_backward: a pointer is missing");
  if ((bias != nullptr) != (d->bucket_of != nullptr) || (dbias && !bias))
    return fail(S2C_ERR_BAD_ARG, "s2c_attention_backward: a bias needs its buckets, and buckets a bias");
  AttnParams p = attn_params(d, q, k, v, bias);
  S2C_SEQ_TRY(attn_check_own("s2c_attention_backward", saved, workspace));
  p.o = out; p.dout = dout; p.dq = dq; p.dk = dk; p.dv = dv;
  attn_set_saved(p, d->dtype, const_cast<void*>(saved));
  return d->dtype == kSeqF32 ? attn_backward<float>(p, dbias, workspace, workspace_bytes, (stream_t)stream)
                             : attn_backward<bf16>(p, dbias, workspace, workspace_bytes, (stream_t)stream);
}

// test hook, see the header
void s2c_debug_attention(int mode) {
#ifndef S2C_EMUL
  g_attention = mode;
#else
  (void)mode;
#endif
}

}  // extern "C"
