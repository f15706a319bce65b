// Device helpers shared by the kernels of libb2attn.so: bf16 packing, mbarriers
// with bounded waits, TMA loads, the q/k norm + RoPE of one head vector, warp-level
// tensor-core products (mma.sync) and tcgen05 / tensor-memory access.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace {

constexpr int kDim = 64;  // head_dim

__device__ __forceinline__ void unpack8(const uint4 &w, float f[8]) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = __uint_as_float(u[i] << 16);
    f[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
  }
}

// round-to-nearest-even fp32 -> bf16 bits (the rounding torch uses on CPU)
__device__ __forceinline__ uint32_t bf16_bits(float x) {
  return static_cast<uint32_t>(__bfloat16_as_ushort(__float2bfloat16_rn(x)));
}

__device__ __forceinline__ float bf16_round(float x) {
  return __uint_as_float(bf16_bits(x) << 16);
}

// two fp32 -> one bf16x2 word (lo in the low half), round-to-nearest-even,
// in one paired conversion instruction
__device__ __forceinline__ uint32_t pack_bf16x2_rn(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&h);
}

__device__ __forceinline__ uint4 pack8(const float f[8]) {
  uint4 w;
  w.x = pack_bf16x2_rn(f[0], f[1]);
  w.y = pack_bf16x2_rn(f[2], f[3]);
  w.z = pack_bf16x2_rn(f[4], f[5]);
  w.w = pack_bf16x2_rn(f[6], f[7]);
  return w;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint64_t global_ns() {
  uint64_t t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}

__device__ __forceinline__ uint32_t smem_u32(const void *p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}

__device__ __forceinline__ void mbar_fence_init() {
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
}

__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done)
      : "r"(bar), "r"(parity)
      : "memory");
  return done != 0;
}

// Wait for the phase with the given parity to complete; false after
// limit_ns (the caller reports B2_DEV_TIMEOUT and unwinds).
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, uint64_t limit_ns) {
  if (mbar_try(bar, parity)) return true;
  const uint64_t t0 = global_ns();
  for (;;) {
#pragma unroll 1
    for (int i = 0; i < 32; ++i)
      if (mbar_try(bar, parity)) return true;
    if (global_ns() - t0 > limit_ns) return false;
  }
}

__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}

// Expect `bytes` more of the current phase's transfer without arriving: the
// phase completes once the bytes have landed and the arrival comes later.
__device__ __forceinline__ void mbar_expect_tx_only(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}

__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes)
               : "memory");
}

// 2-D tiled TMA load into this CTA alone, completing on an mbarrier; KV tiles are
// read once per step, so they are marked evict-first in L2.
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap *map, int x, int y,
                                            uint32_t bar, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      ".L2::cache_hint [%0], [%1, {%2, %3}], [%4], %5;" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar), "l"(policy)
      : "memory");
}

__device__ __forceinline__ uint64_t evict_first_policy() {
  uint64_t p;
  asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
  return p;
}

// Per-head RMSNorm (optional) and rotate-half RoPE (optional) of one 64-wide
// head vector spread over an aligned group of 8 lanes: chunk j = lane % 8
// holds x[8] = elements 8j..8j+7.  Every lane of the warp must call this
// (it shuffles with the full mask); `norm` / `rope` may differ per group.
//  * Lfm2RMSNorm: gamma * bf16(x * 1/sqrt(mean(x^2) + eps)) with fp32 math and
//    IEEE-rounded sqrt and divide, as torch's CPU rsqrt computes 1/sqrt.
//  * RoPE: bf16(bf16(x*cos) + bf16(rotate_half(x)*sin)), rotate_half(x) =
//    [-x[32:], x[:32]]; the partner chunk j^4 sits on lane^4.
//
// mean(x^2) is bit-identical to torch's CPU x.pow(2).mean(-1) of a contiguous
// 64-float row: rounded squares, summed in the order of ATen's vectorised
// inner-dimension sum, whose vectors are 8 floats wide on every CPU build
// (the reduction is not dispatched to 16-wide vectors), then divided by 64
// (exact).  With v_k = squares 8k..8k+7 (chunk k, held by lane k of the group):
//   a_k = v_k + v_{k+4}              k = 0..3, lane-wise
//   p   = ((a_0 + a_1) + a_2) + a_3   lane-wise
//   sum = (((p[0] + p[1]) + p[2]) + ...) + p[7]
// No fused multiply-add anywhere in the chain.
__device__ __forceinline__ float sum_squares64(const float x[8]) {
  const int base = (threadIdx.x & 31) & ~7;
  float a[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float sq = __fmul_rn(x[e], x[e]);
    a[e] = __fadd_rn(sq, __shfl_xor_sync(0xffffffffu, sq, 4));  // a_k on lanes k = 0..3
  }
  float s = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float a0 = __shfl_sync(0xffffffffu, a[e], base);
    const float a1 = __shfl_sync(0xffffffffu, a[e], base + 1);
    const float a2 = __shfl_sync(0xffffffffu, a[e], base + 2);
    const float a3 = __shfl_sync(0xffffffffu, a[e], base + 3);
    const float p = __fadd_rn(__fadd_rn(__fadd_rn(a0, a1), a2), a3);
    s = e == 0 ? p : __fadd_rn(s, p);
  }
  return s;
}

__device__ __forceinline__ void norm_rope8_v(float x[8], int j, bool norm, bool rope, const uint4 gam,
                                             float eps, const uint4 cos8, const uint4 sin8) {
  const float ss = sum_squares64(x);
  if (norm) {
    const float inv = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(ss * (1.0f / kDim), eps)));
    float g[8];
    unpack8(gam, g);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = bf16_round(__fmul_rn(g[e], bf16_round(__fmul_rn(x[e], inv))));
  }
  float p[8];
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    const uint32_t w = bf16_bits(x[e]) | (bf16_bits(x[e + 1]) << 16);
    const uint32_t o = __shfl_xor_sync(0xffffffffu, w, 4);
    p[e] = __uint_as_float(o << 16);
    p[e + 1] = __uint_as_float(o & 0xffff0000u);
  }
  if (rope) {
    float c[8], s[8];
    unpack8(cos8, c);
    unpack8(sin8, s);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float rot = j < 4 ? -p[e] : p[e];
      const float part1 = bf16_round(__fmul_rn(x[e], c[e]));
      const float part2 = bf16_round(__fmul_rn(rot, s[e]));
      x[e] = bf16_round(__fadd_rn(part1, part2));
    }
  }
}

// The same with gamma (the 8 values at j * 8) and the RoPE rows read here.
__device__ __forceinline__ void norm_rope8(float x[8], int j, bool norm, bool rope,
                                           const uint16_t *gamma, float eps,
                                           const uint16_t *cos_row, const uint16_t *sin_row) {
  const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
  norm_rope8_v(x, j, norm, rope, norm ? *reinterpret_cast<const uint4 *>(gamma + j * 8) : zero, eps,
               rope ? *reinterpret_cast<const uint4 *>(cos_row + j * 8) : zero,
               rope ? *reinterpret_cast<const uint4 *>(sin_row + j * 8) : zero);
}

// ---- warp-level tensor-core helpers (mma.sync m16n8k16 bf16 -> fp32)

__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t &r0, uint32_t &r1, uint32_t &r2, uint32_t &r3) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3)
               : "r"(addr));
}

__device__ __forceinline__ void ldsm_x4_t(uint32_t addr, uint32_t &r0, uint32_t &r1, uint32_t &r2, uint32_t &r3) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3)
               : "r"(addr));
}

__device__ __forceinline__ void mma_bf16(float c[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Shared-memory matrix descriptor for tcgen05.mma: 128-byte swizzle, rows of
// 128 bytes, 8-row groups 1024 bytes apart (SBO); LBO as given (unused for a
// single swizzle atom along the contiguous dimension); version 1 (sm_100).
__device__ __forceinline__ uint64_t umma_desc(uint32_t smem_addr, uint32_t lbo_bytes) {
  return (uint64_t)((smem_addr >> 4) & 0x3FFFu) | ((uint64_t)((lbo_bytes >> 4) & 0x3FFFu) << 16) |
         ((uint64_t)(1024u >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}

__device__ __forceinline__ void umma_f16(uint32_t d_tmem, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a), "l"(b), "r"(idesc), "r"(acc));
}

// The same with A from tensor memory: M rows = TMEM lanes, K along the
// columns (two bf16 per 32-bit column).
__device__ __forceinline__ void umma_f16_ta(uint32_t d_tmem, uint32_t a_tmem, uint64_t b, uint32_t idesc,
                                            uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b), "r"(idesc), "r"(acc));
}

__device__ __forceinline__ void umma_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

// Packed fp32 pairs (sm_100 f32x2 arithmetic): one instruction for two lanes'
// worth of FMA / add, halving the softmax's FMA-pipe instructions.
__device__ __forceinline__ void ffma2(float &d0, float &d1, float a0, float a1, float b0, float b1, float c0,
                                      float c1) {
  asm("{\n\t.reg .b64 ra, rb, rc, rd;\n\t"
      "mov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\tmov.b64 rc, {%6, %7};\n\t"
      "fma.rn.f32x2 rd, ra, rb, rc;\n\t"
      "mov.b64 {%0, %1}, rd;\n\t}"
      : "=f"(d0), "=f"(d1)
      : "f"(a0), "f"(a1), "f"(b0), "f"(b1), "f"(c0), "f"(c1));
}

__device__ __forceinline__ void fadd2(float &d0, float &d1, float a0, float a1, float b0, float b1) {
  asm("{\n\t.reg .b64 ra, rb, rd;\n\t"
      "mov.b64 ra, {%2, %3};\n\tmov.b64 rb, {%4, %5};\n\t"
      "add.rn.f32x2 rd, ra, rb;\n\t"
      "mov.b64 {%0, %1}, rd;\n\t}"
      : "=f"(d0), "=f"(d1)
      : "f"(a0), "f"(a1), "f"(b0), "f"(b1));
}

__device__ __forceinline__ void tmem_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// 16 consecutive fp32 columns of this thread's TMEM lane, without waiting
// (several loads in flight; tmem_wait_ld() before using any of them).
__device__ __forceinline__ void tmem_ld16_nowait(uint32_t taddr, uint32_t r[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}

__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// 16 consecutive fp32 columns into this thread's TMEM lane.
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const float v[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
          taddr),
      "r"(__float_as_uint(v[0])), "r"(__float_as_uint(v[1])), "r"(__float_as_uint(v[2])), "r"(__float_as_uint(v[3])),
      "r"(__float_as_uint(v[4])), "r"(__float_as_uint(v[5])), "r"(__float_as_uint(v[6])), "r"(__float_as_uint(v[7])),
      "r"(__float_as_uint(v[8])), "r"(__float_as_uint(v[9])), "r"(__float_as_uint(v[10])),
      "r"(__float_as_uint(v[11])), "r"(__float_as_uint(v[12])), "r"(__float_as_uint(v[13])),
      "r"(__float_as_uint(v[14])), "r"(__float_as_uint(v[15]))
      : "memory");
}

// 32 consecutive 32-bit columns into this thread's TMEM lane.
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t v[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]),
      "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]),
      "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]),
      "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
      : "memory");
}

__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 64 consecutive fp32 columns of this thread's TMEM lane (4 loads, one wait).
__device__ __forceinline__ void tmem_ld64(uint32_t taddr, float v[64]) {
  uint32_t r[64];
#pragma unroll
  for (int c = 0; c < 64; c += 16) tmem_ld16_nowait(taddr + c, r + c);
  tmem_wait_ld();
#pragma unroll
  for (int i = 0; i < 64; ++i) v[i] = __uint_as_float(r[i]);
}

}  // namespace
