// Pieces shared by the block-scaled e4m3 GEMM kernels (gemm_block.cu, gemm_block_wide.cu).
#pragma once
#include "../../include/fastworld_b200.h"
#include "fw_block8.cuh"
#include "fw_internal.h"

namespace fw {

enum : int { ACT_NONE = 0, ACT_TANH = 1, ACT_ERF = 2 };

struct BlockGemmArgs {
  int M, N, K;                 // K as padded to 128
  const uint32_t *sa, *sb;     // exponent words [groups, M], [groups, N]
  const __nv_bfloat16* bias;   // [N] or null
  int act, out_dtype;
  int splits;                  // CTAs that share a tile's k-blocks (gemm_block.cu)
  void* out;                   // bf16 / fp32 [M, N], or codes [M, Np]
  uint8_t* out_s;              // exponents of codes
  int* status;                 // a wait that runs out records its code here, or null
};

// Instruction descriptor of kind::mxf8f6f4: e4m3 operands, both K-major, UE8M0 scales (bit 23).
__host__ __device__ constexpr uint32_t idesc_mx8(int M, int N) {
  return ((uint32_t)(N >> 3) << 17) | (1u << 23) | ((uint32_t)(M >> 4) << 24);
}
// ... with byte `id` of the scale words of both operands
__device__ __forceinline__ uint32_t with_scale_byte(uint32_t idesc, uint32_t id) {
  return idesc | (id << 4) | (id << 29);
}

// The four MMAs of a k-block (128 of K, 32 each), issued by the lane with `one` != 0 while the whole warp
// runs the loop around them: control flow and operands then stay uniform, where a branch on the lane
// would cost a move to a uniform register for every operand of every instruction.  adesc / bdesc are the low
// words of the operands' 128-byte-swizzled descriptors (32 bytes of K further is + 2); `accumulate` 0 overwrites.
template <int CG>
__device__ __forceinline__ void umma_mx8_block(uint32_t one, uint32_t d, uint32_t adesc, uint32_t bdesc, uint32_t idesc,
                                               uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
  // high word: 1024 bytes between 8-row groups, descriptor version 1, 128-byte swizzle
  constexpr uint32_t HI = (1024u >> 4) | (1u << 14) | (2u << 29);
#define FW_MX8(CGN)                                                                                                    \
  asm volatile(                                                                                                        \
      "{\n\t.reg .pred p, q, e;\n\t.reg .b64 a, b;\n\t.reg .b32 x, y;\n\t"                                           \
      "setp.ne.b32 p, %6, 0;\n\tsetp.eq.b32 q, %6, %6;\n\tsetp.ne.b32 e, %8, 0;\n\t"                               \
      "mov.b64 a, {%1, %7};\n\tmov.b64 b, {%2, %7};\n\t"                                                             \
      "@e tcgen05.mma.cta_group::" CGN ".kind::mxf8f6f4.block_scale.scale_vec::1X [%0], a, b, %3, [%4], [%5], p;\n\t"  \
      "add.u32 x, %1, 2;\n\tadd.u32 y, %2, 2;\n\tmov.b64 a, {x, %7};\n\tmov.b64 b, {y, %7};\n\t"                   \
      "@e tcgen05.mma.cta_group::" CGN ".kind::mxf8f6f4.block_scale.scale_vec::1X [%0], a, b, %3, [%4], [%5], q;\n\t"  \
      "add.u32 x, %1, 4;\n\tadd.u32 y, %2, 4;\n\tmov.b64 a, {x, %7};\n\tmov.b64 b, {y, %7};\n\t"                   \
      "@e tcgen05.mma.cta_group::" CGN ".kind::mxf8f6f4.block_scale.scale_vec::1X [%0], a, b, %3, [%4], [%5], q;\n\t"  \
      "add.u32 x, %1, 6;\n\tadd.u32 y, %2, 6;\n\tmov.b64 a, {x, %7};\n\tmov.b64 b, {y, %7};\n\t"                   \
      "@e tcgen05.mma.cta_group::" CGN ".kind::mxf8f6f4.block_scale.scale_vec::1X [%0], a, b, %3, [%4], [%5], q;\n\t}" \
      ::"r"(d), "r"(adesc), "r"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate), "r"(HI), "r"(one)             \
      : "memory")
  if constexpr (CG == 2)
    FW_MX8("2");
  else
    FW_MX8("1");
#undef FW_MX8
}
// In both CTAs of a pair, 32 rows of 16 bytes (512 contiguous bytes of its shared memory) to four columns of its
// Tensor Memory, the same in every lane quarter: lane l of column c gets word c of row l.  Issued by another warp than
// the MMAs that use the words: a commit behind the copies tells that they are there, one behind the MMAs that they are
// used.
__device__ __forceinline__ void tmem_copy_pair_if(uint32_t one, uint32_t taddr, uint32_t saddr) {
  // descriptor: 128 bytes between 8-row groups, version 1, no swizzle
  const uint64_t desc = (uint64_t)((saddr >> 4) & 0x3fffu) | ((uint64_t)(128 >> 4) << 32) | ((uint64_t)1 << 46);
  asm volatile(
      "{\n\t.reg .pred e;\n\tsetp.ne.b32 e, %2, 0;\n\t"
      "@e tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;\n\t}" ::"r"(taddr), "l"(desc), "r"(one)
      : "memory");
}

// Low word of a tile's descriptor: address and (unused with this swizzle) leading offset.
__device__ __forceinline__ uint32_t desc_lo(uint32_t saddr) { return ((saddr >> 4) & 0x3fffu) | (1u << 16); }

// Arrive once on `bar` when all MMAs issued so far by the lane with `one` != 0 complete; for a pair, on the
// barrier at this offset in both CTAs, by one commit (two, one for each CTA, cost 8 % of the kernel).
template <int CG>
__device__ __forceinline__ void umma_commit_if(uint32_t one, uint64_t* bar) {
  if constexpr (CG == 2)
    asm volatile(
        "{\n\t.reg .pred e;\n\tsetp.ne.b32 e, %2, 0;\n\t"
        "@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n\t}" ::"r"(
            smem_u32(bar)),
        "h"((uint16_t)3), "r"(one)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred e;\n\tsetp.ne.b32 e, %1, 0;\n\t"
        "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar)), "r"(one)
        : "memory");
}

// ... a pair's MMAs, on this CTA's barrier alone.
__device__ __forceinline__ void umma_commit_local_if(uint32_t one, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred e;\n\tsetp.ne.b32 e, %1, 0;\n\t"
      "@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar)), "r"(one)
      : "memory");
}

// One 32-bit column per register, this warp's lane quarter.
template <int N>
__device__ __forceinline__ void tmem_st(uint32_t taddr, const uint32_t (&r)[N]);
template <>
__device__ __forceinline__ void tmem_st<1>(uint32_t taddr, const uint32_t (&r)[1]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x1.b32 [%0], {%1};" ::"r"(taddr), "r"(r[0]) : "memory");
}
template <>
__device__ __forceinline__ void tmem_st<2>(uint32_t taddr, const uint32_t (&r)[2]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x2.b32 [%0], {%1, %2};" ::"r"(taddr), "r"(r[0]), "r"(r[1]) : "memory");
}
template <>
__device__ __forceinline__ void tmem_st<4>(uint32_t taddr, const uint32_t (&r)[4]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};" ::"r"(taddr), "r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3])
               : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}

// GELU of two values.  tanh form: 0.5 v (1 + tanh u) = v / (1 + 2^(-2 u log2 e)), within a few fp32 roundings
// (the hardware's tanh.approx, relative error 2^-11, would show in an fp32 result, and 1 + tanh cancels
// for negative v); where the power overflows the reciprocal is 0, as it should be.  erf form by erfc,
// which keeps its relative precision where 1 + erf cancels: a block of small negative results is scaled by
// them.  It is called, not inlined: its code, once per value, would not fit the epilogue loops.  2640 x 8960 x 1536
// takes 38.0 us with the first form and 111 with the second.
__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
static __device__ __noinline__ float gelu_erf1(float v) { return 0.5f * v * erfcf(v * -0.70710678118654752f); }
template <int ACT>
__device__ __forceinline__ float2 activate2(float2 v) {
  if constexpr (ACT == ACT_TANH) {
    constexpr float C0 = -2.302208198f, C1 = C0 * 0.044715f;   // -2 log2(e) sqrt(2 / pi)
    const float2 p = __ffma2_rn(__fmul2_rn(v, v), make_float2(C1, C1), make_float2(C0, C0));
    const float2 w = __fmul2_rn(v, p);
    const float2 d = __fadd2_rn(make_float2(ex2(w.x), ex2(w.y)), make_float2(1.f, 1.f));
    return __fmul2_rn(v, make_float2(rcp_approx(d.x), rcp_approx(d.y)));
  }
  if constexpr (ACT == ACT_ERF) return make_float2(gelu_erf1(v.x), gelu_erf1(v.y));
  return v;
}

// Abort flag of CTA `lane` of a cluster of `ranks`, 0 for lanes without one.  Behind a cluster barrier that follows all
// of the ranks' waits, a vote over it tells every warp of every rank the same: whether all of them staged their part.
__device__ __forceinline__ int cluster_abort_flag(const volatile int* flag, int ranks) {
  const int lane = threadIdx.x & 31;
  int v = 0;
  if (lane < ranks)
    asm volatile("ld.shared::cluster.b32 %0, [%1];"
                 : "=r"(v)
                 : "r"(mapa_cluster(const_cast<const int*>(flag), (uint32_t)lane))
                 : "memory");
  return v;
}

// gemm_block_wide.cu: persistent kernel for large problems.
int gemm_block_wide_launch(const void* A8, const void* B8, const BlockGemmArgs& a, cudaStream_t s);

}  // namespace fw
