// What the attention kernels on the 5th-generation tensor cores (tcgen05.mma, accumulators in TMEM) share.
//
// Operand tiles lie in shared memory as rows of 64 bfloat16 (128 bytes), in blocks of 64 columns, the 16-byte pieces of row r
// exchanged by r % 8 (the 128-byte swizzle): for a product along the columns such a tile is a "K-major" operand, for a product
// along the rows an "MN-major" one, so that keys serve both for the scores and for the gradient of the queries from one copy.
// They are filled with 16-byte cp.async, which writes zeros in place of rows beyond the lengths: what lies there is never read.
// Weights and score gradients pass from the threads to the tensor core through tensor memory, as its left operand.
#pragma once

#include "attention_kernels.h"

#ifndef S2C_EMUL

#include <stdint.h>

namespace s2c {

struct AttnTcParams {
  AttnParams a;        // q, k, v (and dout): 16-byte aligned, strides multiples of 8 elements
  long gs[3];          // strides of dout
  const void* grad;    // dout as the caller gave it, laid out as the output
  int chunks;          // 16-byte pieces of a row that hold values
  int units, pairs;    // query tiles of 128 per (batch entry, key head), and blocks of one or two of them
  int per_block;       // query tiles of a block: 1 or 2
  int whole;           // forward: blocks from this one on take one tile of a pair each
  long q_split, k_split, v_split, g_split;     // float32: elements from one part of an operand to the next (attention_tc3.h)
};

// A tensor-core kernel as a struct: kThreads and run(p, smem), which lets the next kernel's blocks in itself.
template <class Impl>
__global__ void __launch_bounds__(Impl::kThreads, 1) attn_tc_kernel(const AttnTcParams p) {
  extern __shared__ float4 s2c_dyn_smem[];
  stream_order_wait();
  Impl::run(p, s2c_dyn_smem);
}
template <class Impl>
inline int attn_tc_launch(const char* name, long grid, size_t smem, stream_t st, const AttnTcParams& p) {
  return launch_impl<attn_tc_kernel<Impl>>(name, grid, Impl::kThreads, smem, st, p);
}

__device__ __forceinline__ uint32_t tcx_addr(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

__device__ __forceinline__ void tcx_init(uint64_t* bar, int count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(tcx_addr(bar)), "r"(count));
}
__device__ __forceinline__ void tcx_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(tcx_addr(bar)) : "memory");
}
__device__ __forceinline__ bool tcx_try(uint32_t addr, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done)
      : "r"(addr), "r"(parity)
      : "memory");
  return done != 0;
}
// Bounded: false where the phase is not over after some tenths of a second.  (The first try stands in line with the code around
// it: a role that issues products runs through cold instructions, which come quickly only where nothing branches.)
__device__ __forceinline__ bool tcx_wait(uint64_t* bar, uint32_t parity) {
  const uint32_t addr = tcx_addr(bar);
  if (__builtin_expect(tcx_try(addr, parity), 1)) return true;
#pragma unroll 1
  for (int spin = 0; spin < (1 << 22); ++spin) {
    if (tcx_try(addr, parity)) return true;
    if (spin > 256) __nanosleep(40);
  }
  return false;
}
// a place in a ring of N barriers and the parity of its phase
template <int N>
struct TcxRing {
  int at = 0;
  uint32_t parity = 0;
  __device__ __forceinline__ void next() {
    if (++at == N) {
      at = 0;
      parity ^= 1;
    }
  }
};
// the same by a whole warp, which goes on together
__device__ __forceinline__ bool tcx_wait_warp(uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, tcx_wait(bar, parity)) != 0; }

__device__ __forceinline__ bool tcx_elect() {
  uint32_t pred;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(pred));
  return pred != 0;
}
__device__ __forceinline__ void tcx_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(tcx_addr(bar)) : "memory");
}
__device__ __forceinline__ void tcx_before_sync() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tcx_after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

template <int COLS>
__device__ __forceinline__ void tcx_alloc(uint32_t* slot) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tcx_addr(slot)), "r"(COLS) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
template <int COLS>
__device__ __forceinline__ void tcx_free(uint32_t base) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(COLS) : "memory");
}

// Shared-memory descriptor of a swizzled tile: 8 rows of 128 bytes are 1024 bytes from the next 8.  `block`: bytes from one
// block of 64 columns to the next (an MN-major operand wider than 64; a K-major one steps through its blocks by address).
__device__ __forceinline__ uint64_t tcx_desc(uint32_t addr, uint32_t block) {
  return (uint64_t)((addr & 0x3FFFF) >> 4) | (uint64_t)(block >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// Instruction descriptor: D float32, A and B bfloat16, 128 rows, n columns; `b_mn`: B is MN-major.
__device__ __forceinline__ uint32_t tcx_idesc(int n, bool b_mn) {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}
// one step of 16 columns, left operand in tensor memory
__device__ __forceinline__ void tcx_mma_t(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// four steps, each step's operands A_STEP and B_STEP (in descriptor units) behind the last ones', as straight-line code: the loops
// at the scores push the issuing thread's code out of the instruction caches, and what has no branches is fetched ahead (with a number
// of steps at run time the gradient of the queries of 2 x 4096 positions, 16 heads of 128, took 517 us, now 401)
template <int A_STEP, int B_STEP>
__device__ __forceinline__ void tcx_mma4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 x, y;\n\tsetp.ne.b32 q, %4, 0;\n\tsetp.eq.b32 p, 0, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, q;\n\t"
      "add.s64 x, %1, %5;\n\tadd.s64 y, %2, %6;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n\t"
      "add.s64 x, %1, %7;\n\tadd.s64 y, %2, %8;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n\t"
      "add.s64 x, %1, %9;\n\tadd.s64 y, %2, %10;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "n"(A_STEP), "n"(B_STEP), "n"(2 * A_STEP), "n"(2 * B_STEP), "n"(3 * A_STEP), "n"(3 * B_STEP)
      : "memory");
}
template <int B_STEP>
__device__ __forceinline__ void tcx_mma4_t(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b32 x;\n\t.reg .b64 y;\n\tsetp.ne.b32 q, %4, 0;\n\tsetp.eq.b32 p, 0, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, q;\n\t"
      "add.s32 x, %1, 8;\n\tadd.s64 y, %2, %5;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [x], y, %3, p;\n\t"
      "add.s32 x, %1, 16;\n\tadd.s64 y, %2, %6;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [x], y, %3, p;\n\t"
      "add.s32 x, %1, 24;\n\tadd.s64 y, %2, %7;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [x], y, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate), "n"(B_STEP), "n"(2 * B_STEP), "n"(3 * B_STEP)
      : "memory");
}
constexpr uint32_t kTcxTile = 128 * 128;      // bytes of 128 rows of 64 columns
// D (128 x ROWS) (+)= A B^T over NC blocks of 64 columns, both operands K-major tiles: A of A_ROWS rows, B of ROWS.  (Zeros behind
// the values: straight-line code for every width.)
template <int NC, int A_ROWS, int ROWS>
__device__ __forceinline__ void tcx_scores(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate = 0) {
#pragma unroll
  for (int k = 0; k < NC; ++k)
    tcx_mma4<2, 2>(d, tcx_desc(a, 0) + (uint64_t)(k * A_ROWS * 128 >> 4), tcx_desc(b, 0) + (uint64_t)(k * ROWS * 128 >> 4), idesc, accumulate | (uint32_t)k);
}
// the same with A in tensor memory
template <int NC, int ROWS>
__device__ __forceinline__ void tcx_scores_t(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate = 0) {
#pragma unroll
  for (int k = 0; k < NC; ++k) tcx_mma4_t<2>(d, a + 32 * k, tcx_desc(b, 0) + (uint64_t)(k * ROWS * 128 >> 4), idesc, accumulate | (uint32_t)k);
}
// D (128 x n) (+)= A B over K rows of B: A 128 x K in tensor memory, B K rows (from `b` on) of a tile of ROWS rows, MN-major
template <int K, int ROWS>
__device__ __forceinline__ void tcx_combine(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool accumulate) {
  const uint64_t db = tcx_desc(b, ROWS * 128);
#pragma unroll
  for (int s = 0; s < K / 16; s += 4) {
    if constexpr (K % 64 == 0) {
      tcx_mma4_t<(2048 >> 4)>(d, a + 8 * s, db + (uint64_t)(s * 2048 >> 4), idesc, accumulate || s > 0);
    } else {
#pragma unroll
      for (int e = 0; e < K / 16; ++e) tcx_mma_t(d, a + 8 * e, db + (uint64_t)(e * 2048 >> 4), idesc, accumulate || e > 0);
    }
  }
}

// 32 columns of a lane's row; the values are there after tcx_ld_wait
__device__ __forceinline__ void tcx_ld32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
        "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
        "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
// (the registers pass through, so that nothing reads them earlier)
__device__ __forceinline__ void tcx_ld_wait(uint32_t* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]),
                 "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]),
                 "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
}
__device__ __forceinline__ void tcx_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
      "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]),
      "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tcx_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
               "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
               "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
               : "memory");
}
// 32 values of a bfloat16 row (columns c0 ... c0 + 31; zeros from `chunks` pieces on, or all of them) as a left operand
__device__ __forceinline__ void tcx_put_operand(uint32_t taddr, const bf16* row, int c0, int chunks, bool on) {
  uint32_t r[16];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    uint4 u = make_uint4(0u, 0u, 0u, 0u);
    if (on && c0 / 8 + k < chunks) u = *reinterpret_cast<const uint4*>(row + c0 + 8 * k);
    r[4 * k] = u.x; r[4 * k + 1] = u.y; r[4 * k + 2] = u.z; r[4 * k + 3] = u.w;
  }
  tcx_st16(taddr + c0 / 2, r);
}
__device__ __forceinline__ void tcx_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// rows [r0, r0 + ROWS) of one head into a swizzled tile, by N threads of which this is number t: `chunks` pieces of a row of
// values, zeros beyond them and in rows from `end` on.  A thread has the same piece of every
// N / 8-th row, so that a copy costs it an addition and a comparison: one warp keeps up with the tensor core.
template <int NC, int N, int ROWS = 128>
__device__ __forceinline__ void tcx_load_rows(uint32_t dst, const bf16* src, long row_stride, int r0, int end, int chunks, int t) {
  const int c = t % 8, r = t / 8, left = end - r0 - r;               // rows of this thread that hold values: it * N / 8 < left
  const long step = (long)(N / 8) * row_stride;
#pragma unroll
  for (int b = 0; b < NC; ++b) {
    const int cc = 8 * b + c;
    const bool in = cc < chunks;
    const bf16* from = src + (long)(r0 + r) * row_stride + 8 * cc;
    const uint32_t to = dst + b * (ROWS * 128) + r * 128;
    // (N = 32: rows r and r + 4 in turn, more threads: r % 8 stays)
    const uint32_t even = (uint32_t)((c ^ (r % 8)) << 4), odd = (uint32_t)((c ^ ((r + N / 8) % 8)) << 4);
#pragma unroll 8
    for (int it = 0; it < ROWS * 8 / N; ++it) {
      const bool on = in && it * (N / 8) < left;
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + it * (16 * N) + (it % 2 ? odd : even)), "l"(on ? from : src),
                   "r"(on ? 16 : 0)
                   : "memory");
      from += step;
    }
  }
}
// Arrives at the barrier (whose count has this thread in it) once this thread's copies so far have landed; the thread goes on.
// Who waits for that and then issues products has tcx_seen in between.
__device__ __forceinline__ void tcx_arrive_copies(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(tcx_addr(bar)) : "memory");
}
__device__ __forceinline__ void tcx_copies_done() { asm volatile("cp.async.wait_all;" ::: "memory"); }
__device__ __forceinline__ void tcx_seen() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// all of this thread's copies have landed and are seen by the tensor core
__device__ __forceinline__ void tcx_loaded() {
  asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 0;\n\tfence.proxy.async.shared::cta;" ::: "memory");
}

// The bias by relative position, in units of ln 2, with its last values repeated 256 positions beyond the reach on either side:
// a tile that lies partly within the reach reads it without clamping.  At tab[d + reach + 256].
constexpr int kTcxMargin = 256;
__device__ __forceinline__ int tcx_tab_floats(int reach) { return 2 * reach + 2 * kTcxMargin + 1; }
__device__ __forceinline__ void tcx_bias_table(const AttnParams& p, int head, float* tab, int t, int n, bool wide) {
  for (int e = t; e < tcx_tab_floats(p.reach); e += n) {
    const int at = attn_clamp(e - kTcxMargin, 0, 2 * p.reach);
    float v = 0.f;
    if (p.bias) {
      const int which = p.bucket_of[at];
      if (which >= 0 && which < p.n_buckets) {
        const long i = (long)which * p.heads + head;
        v = attn_bias_units(wide ? static_cast<const float*>(p.bias)[i] : widen(static_cast<const bf16*>(p.bias)[i]));
      }
    }
    tab[e] = v;
  }
}
__device__ __forceinline__ float tcx_max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float2 tcx_add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tadd.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

// `n` values of a row (a multiple of 8), as bfloat16 and, for `lo`, what the rounding left
__device__ __forceinline__ void tcx_put_row(bf16* out, bf16* lo, const float* v, int n, int dim, int c0, bool wide) {
  if (wide) {                                // rows of whole 16-byte pieces
#pragma unroll
    for (int c = 0; c < n; c += 8) {
      if (c0 + c >= dim) break;
      uint4 u;
      u.x = pack_bf16(v[c], v[c + 1]);
      u.y = pack_bf16(v[c + 2], v[c + 3]);
      u.z = pack_bf16(v[c + 4], v[c + 5]);
      u.w = pack_bf16(v[c + 6], v[c + 7]);
      *reinterpret_cast<uint4*>(out + c0 + c) = u;
      if (lo) {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
        uint32_t r[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          r[i] = pack_bf16(v[c + 2 * i] - as_float(w[i] << 16), v[c + 2 * i + 1] - as_float(w[i] & 0xffff0000u));
        *reinterpret_cast<uint4*>(lo + c0 + c) = make_uint4(r[0], r[1], r[2], r[3]);
      }
    }
  } else {
#pragma unroll
    for (int c = 0; c < n; ++c)
      if (c0 + c < dim) narrow_with_rest(out + c0 + c, lo ? lo + c0 + c : nullptr, v[c]);
  }
}

}  // namespace s2c
#endif  // S2C_EMUL
