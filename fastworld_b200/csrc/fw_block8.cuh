// Block-scaled e4m3: the operand format of gemm_block.cu and the row encoder that quant, norm and
// GEMM epilogues share.
//
// x [R, K] is held as codes q [R, Kp] (e4m3 bytes; Kp = K rounded up to 128, zeros behind K) and
// exponents s [ceil(Kp / 512), R, 4] (bytes): s[g, r, j] - 127 is the power of two that scales row
// r's columns [128 (4 g + j), + 128); places behind the last block hold 127.  A block's exponent is the
// smallest e >= -127 with max|x| <= 448 * 2^e over its finite elements, found from the bits of the
// maximum, so the same input always gives the same code.  Powers of two are what the tensor core
// multiplies in by itself (UE8M0 scales); they cost no precision, since an e4m3 code is
// as precise in every binade (only the range at the bottom of a block shrinks, by less than one of
// e4m3's 17 binades).  Four exponents of a row are one 32-bit word, and neighbouring rows' words are
// adjacent: a warp fetches the words of 32 rows with one 128-byte load, for a tile at any row.
#pragma once
#include <cuda_fp16.h>
#include <stdint.h>

#include "fw_ptx.cuh"

namespace fw {

// Bounded wait for a phase, for loops whose issue rate counts: one try that lets the hardware hold
// the thread until the phase completes (up to a millisecond), and everything else out of line, so
// that little code sits between two MMAs.  CLUSTER: the phase may be completed from the other CTA of a
// pair, whose work is observed only by an acquire at cluster scope.
template <bool CLUSTER>
__device__ __forceinline__ bool mbar_try_held(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
#define FW_TRY(SCOPE)                                                           \
  asm volatile(                                                                 \
      "{\n\t.reg .pred p;\n\t"                                                  \
      "mbarrier.try_wait.parity.acquire." SCOPE ".shared::cta.b64 p, [%1], %2, %3;\n\t" \
      "selp.u32 %0, 1, 0, p;\n\t}\n"                                           \
      : "=r"(ok)                                                                \
      : "r"(smem_u32(bar)), "r"(parity), "r"(1000000u)                          \
      : "memory")
  if constexpr (CLUSTER)
    FW_TRY("cluster");
  else
    FW_TRY("cta");
#undef FW_TRY
  return ok != 0;
}
template <bool CLUSTER>
static __device__ __noinline__ bool wait_again(uint64_t* bar, uint32_t parity, volatile int* abort, int* status,
                                               int code, uint64_t limit_ns) {
  const uint64_t t0 = globaltimer();
  for (;;) {
    if (mbar_try_held<CLUSTER>(bar, parity)) return true;
    if (*abort) return false;
    if (globaltimer() - t0 > limit_ns) {
      *abort = 1;
      record_status(status, code);
      return false;
    }
  }
}
template <bool CLUSTER = false>
__device__ __forceinline__ bool wait_on(uint64_t* bar, uint32_t parity, volatile int* abort, int* status, int code,
                                        uint64_t limit_ns = FW_WAIT_LIMIT_NS) {
  return mbar_try_held<CLUSTER>(bar, parity) || wait_again<CLUSTER>(bar, parity, abort, status, code, limit_ns);
}

namespace b8 {

constexpr int BLK = 128;            // columns that share a scale
constexpr int GRP = 4;              // blocks of one 32-bit word of exponents
constexpr uint32_t ONES = 0x7f7f7f7fu;   // four times 2^0: rows and blocks that do not exist

__host__ __device__ constexpr int blocks(int K) { return (K + BLK - 1) / BLK; }
__host__ __device__ constexpr int groups(int K) { return (blocks(K) + GRP - 1) / GRP; }
__host__ __device__ constexpr int padded(int K) { return blocks(K) * BLK; }

// |x| as ordered bits, 0 for what is not finite (such elements have no say in the scale).
__device__ __forceinline__ uint32_t abs_bits(float x) {
  const uint32_t b = __float_as_uint(x) & 0x7fffffffu;
  return b < 0x7f800000u ? b : 0u;
}
// Biased exponent byte (e + 127) of a block whose largest finite magnitude has the bits `amax`.
// 448 = 1.75 * 2^8: e = floor(log2 amax) - 8, one more where the mantissa is above 1.75.
__device__ __forceinline__ uint32_t block_exp(uint32_t amax) {
  const int e = (int)(amax >> 23) - 8 + ((amax & 0x7fffffu) > 0x600000u ? 1 : 0);   // biased
  return (uint32_t)max(e, 0);
}
// 2^-e of a biased exponent byte (at most 247, the byte of the largest fp32 value).
__device__ __forceinline__ float inv_scale(uint32_t eb) { return __uint_as_float((254u - eb) << 23); }

// Four codes of x * inv where no x is infinite (a NaN becomes the NaN code by itself).
__device__ __forceinline__ uint32_t encode4_finite(float a, float b, float c, float d, float inv) {
  const float2 lo2 = __fmul2_rn(make_float2(a, b), make_float2(inv, inv));
  const float2 hi2 = __fmul2_rn(make_float2(c, d), make_float2(inv, inv));
  uint32_t r;
  asm("{\n\t.reg .b16 l, h;\n\t"
      "cvt.rn.satfinite.e4m3x2.f32 l, %2, %1;\n\tcvt.rn.satfinite.e4m3x2.f32 h, %4, %3;\n\tmov.b32 %0, {l, h};\n\t}"
      : "=r"(r)
      : "f"(lo2.x), "f"(lo2.y), "f"(hi2.x), "f"(hi2.y));
  return r;
}
// Four codes of x * inv (round to nearest even; NaN and infinities become the NaN code).
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d, float inv) {
  auto in = [&](float v) {
    return (__float_as_uint(v) & 0x7fffffffu) < 0x7f800000u ? v * inv : __uint_as_float(0x7fffffffu);
  };
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(in(b)), "f"(in(a)));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(in(d)), "f"(in(c)));
  return (uint32_t)lo | ((uint32_t)hi << 16);
}
// One block across a warp, four consecutive columns per lane: codes of this lane, exponent byte.
__device__ __forceinline__ uint32_t encode_block(const float2 (&v)[2], uint32_t& eb) {
  // the largest magnitude, passing over NaN; only an infinity needs the look at every element
  const float top = fmaxf(fmaxf(fabsf(v[0].x), fabsf(v[0].y)), fmaxf(fabsf(v[1].x), fabsf(v[1].y)));
  const uint32_t m = __reduce_max_sync(0xffffffffu, __float_as_uint(top));
  if (m < 0x7f800000u) {
    eb = block_exp(m);
    return encode4_finite(v[0].x, v[0].y, v[1].x, v[1].y, inv_scale(eb));
  }
  const uint32_t f = max(max(abs_bits(v[0].x), abs_bits(v[0].y)), max(abs_bits(v[1].x), abs_bits(v[1].y)));
  eb = block_exp(__reduce_max_sync(0xffffffffu, f));
  return encode4(v[0].x, v[0].y, v[1].x, v[1].y, inv_scale(eb));
}

}  // namespace b8
}  // namespace fw
