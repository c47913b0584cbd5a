// What the kernels for sequences of signals (attention, layer norm, dropout) share: the two element types, wide accesses,
// base-2 exponentials and the launcher of a kernel written as a struct.
//
// Sums and what is computed element by element are float32; a bfloat16 input is widened exactly when it is read and a result
// rounded once, to nearest even, when it is written.  (The bfloat16 attention kernels on the tensor cores also round the left operands of
// their second products, weights and score gradients: see there.)
#pragma once

#include "backend.h"

namespace s2c {

enum SeqType : int { kSeqF32 = 0, kSeqBf16 = 1 };

struct bf16 {
  unsigned short bits;
};

#ifndef S2C_EMUL
S2C_D float as_float(unsigned u) { return __uint_as_float(u); }
S2C_D unsigned as_bits(float f) { return __float_as_uint(f); }
// two floats as bfloat16, `lo` in the lower half
S2C_D unsigned pack_bf16(float lo, float hi) {
  unsigned r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// 2^x as the special-function unit gives it (relative error of 2^x: 2^-22); 2^-inf = 0
S2C_D float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
S2C_D float inv_sqrt(float x) { return rsqrtf(x); }
#else
inline float as_float(unsigned u) {
  float f;
  std::memcpy(&f, &u, 4);
  return f;
}
inline unsigned as_bits(float f) {
  unsigned u;
  std::memcpy(&u, &f, 4);
  return u;
}
inline unsigned emu_bf16(float f) {
  const unsigned u = as_bits(f);
  if (f != f) return 0x7fff;
  return (u + 0x7fffu + ((u >> 16) & 1u)) >> 16;
}
inline unsigned pack_bf16(float lo, float hi) { return (emu_bf16(lo) & 0xffffu) | (emu_bf16(hi) << 16); }
inline float exp2_fast(float x) { return std::exp2(x); }
inline float inv_sqrt(float x) { return 1.f / std::sqrt(x); }
#endif

S2C_D float widen(float v) { return v; }
S2C_D float widen(bf16 v) { return as_float((unsigned)v.bits << 16); }
S2C_D void narrow(float* p, float v) { *p = v; }
S2C_D void narrow(bf16* p, float v) { p->bits = (unsigned short)pack_bf16(v, 0.f); }
// v as T, and what is left of it (bfloat16 only; lo null: not wanted)
S2C_D void narrow_with_rest(float* p, float*, float v) { *p = v; }
S2C_D void narrow_with_rest(bf16* p, bf16* lo, float v) {
  narrow(p, v);
  if (lo) narrow(lo, v - widen(*p));
}

// `n` consecutive values (a power of two, 16 bytes at most), aligned to their size
struct alignas(16) Vec16 {
  unsigned w[4];
};
template <class T>
constexpr int kVec = 16 / (int)sizeof(T);
S2C_D void load_vec(const float* p, float (&v)[4]) {
  const Vec16 u = *reinterpret_cast<const Vec16*>(p);
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = as_float(u.w[i]);
}
S2C_D void load_vec(const bf16* p, float (&v)[8]) {
  const Vec16 u = *reinterpret_cast<const Vec16*>(p);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = as_float(u.w[i] << 16);
    v[2 * i + 1] = as_float(u.w[i] & 0xffff0000u);
  }
}
S2C_D void store_vec(float* p, const float (&v)[4]) {
  Vec16 u;
#pragma unroll
  for (int i = 0; i < 4; ++i) u.w[i] = as_bits(v[i]);
  *reinterpret_cast<Vec16*>(p) = u;
}
S2C_D void store_vec(bf16* p, const float (&v)[8]) {
  Vec16 u;
#pragma unroll
  for (int i = 0; i < 4; ++i) u.w[i] = pack_bf16(v[2 * i], v[2 * i + 1]);
  *reinterpret_cast<Vec16*>(p) = u;
}

// A kernel as a struct: Params, kThreads, kBlocks (per SM, for the register budget) and a static run(ctx, p, smem).
#ifndef S2C_EMUL
template <class Impl>
__global__ void __launch_bounds__(Impl::kThreads, Impl::kBlocks) seq_kernel(const typename Impl::Params p) {
  extern __shared__ float4 s2c_dyn_smem[];
  const Ctx ctx{(int)threadIdx.x, (int)blockDim.x, (int)blockIdx.x, (int)gridDim.x};
  stream_order_wait();
  Impl::run(ctx, p, reinterpret_cast<unsigned char*>(s2c_dyn_smem));
  stream_order_next();
}
template <class Impl>
inline int seq_launch(const char* name, long grid, size_t smem, stream_t st, const typename Impl::Params& p) {
  return launch_impl<seq_kernel<Impl>>(name, grid, Impl::kThreads, smem, st, p);
}
#else
template <class Impl>
inline int seq_launch(const char* name, long grid, size_t smem, stream_t, const typename Impl::Params& p) {
  return emu_launch<Impl>(name, grid, Impl::kThreads, smem, p);
}
#endif

// Sum and maximum over `W` neighbouring lanes (a power of two, 32 at most), in every one of them.
template <int W>
S2C_D float lanes_sum(const Ctx& ctx, float v) {
#pragma unroll
  for (int m = W / 2; m >= 1; m /= 2) v += ctx.shfl_xor(v, m);
  return v;
}
template <int W>
S2C_D float lanes_max(const Ctx& ctx, float v) {
#pragma unroll
  for (int m = W / 2; m >= 1; m /= 2) {
    const float o = ctx.shfl_xor(v, m);
    v = o > v ? o : v;
  }
  return v;
}

}  // namespace s2c
