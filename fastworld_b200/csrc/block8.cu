// Row kernels of the block-scaled e4m3 linears (format: fw_block8.cuh): the quantiser, and the norms
// around a block fused with its gate and residual update.  Both move each byte once; HBM bounds them.
#include "../../include/fastworld_b200.h"
#include "fw_block8.cuh"
#include "fw_internal.h"

namespace fw {

namespace {

// A lane's four columns of a block of 128.  VEC: adjacent ones, one access, where rows start at addresses aligned
// to it.  Else every STEP-th one by scalar accesses.
template <typename T, bool VEC, int STEP>
struct Four {
  float v[4];
  __device__ __forceinline__ void load(const T* row, int c, int K) {   // zeros behind K
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = c + i * STEP < K ? static_cast<float>(row[c + i * STEP]) : 0.f;
  }
  __device__ __forceinline__ void get(float2 (&o)[2]) const {
    o[0] = make_float2(v[0], v[1]);
    o[1] = make_float2(v[2], v[3]);
  }
};
template <int STEP>
struct Four<float, true, STEP> {
  float4 u;
  __device__ __forceinline__ void load(const float* row, int c, int K) {
    u = c < K ? *reinterpret_cast<const float4*>(row + c) : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  __device__ __forceinline__ void get(float2 (&o)[2]) const {
    o[0] = make_float2(u.x, u.y);
    o[1] = make_float2(u.z, u.w);
  }
};
template <int STEP>
struct Four<__nv_bfloat16, true, STEP> {
  uint2 u;
  __device__ __forceinline__ void load(const __nv_bfloat16* row, int c, int K) {
    u = c < K ? *reinterpret_cast<const uint2*>(row + c) : make_uint2(0u, 0u);
  }
  __device__ __forceinline__ void get(float2 (&o)[2]) const {
    o[0] = unpack_bf16(u.x);
    o[1] = unpack_bf16(u.y);
  }
};
template <int STEP>
struct Four<__half, true, STEP> {
  uint2 u;
  __device__ __forceinline__ void load(const __half* row, int c, int K) {
    u = c < K ? *reinterpret_cast<const uint2*>(row + c) : make_uint2(0u, 0u);
  }
  __device__ __forceinline__ void get(float2 (&o)[2]) const {
    o[0] = __half22float2(*reinterpret_cast<const __half2*>(&u.x));
    o[1] = __half22float2(*reinterpret_cast<const __half2*>(&u.y));
  }
};

// ---------------------------------------------------------------- quantiser
// A warp takes one row's group of 512 columns: four blocks, four columns per lane and block, so
// each load and each store of codes is contiguous over the warp and a block's maximum is one warp
// reduction.  The eight warps of a CTA take eight neighbouring rows, whose words of exponents are one 32-byte
// sector.  Many short CTAs keep HBM busiest: 2640 x 8960 bf16 in 13.5 us (5.3 TB/s), fp32 in 18.5 us
// (6.4 TB/s); warps that took two, three or six groups of bf16 with the next one's loads in flight took 16.0, 16.2 and
// 17.3 us.
constexpr int QROWS = 8;

template <typename T, bool VEC>
__global__ void __launch_bounds__(QROWS * 32) quant_block_kernel(const T* __restrict__ x, int M, int K,
                                                                 uint8_t* __restrict__ q, uint32_t* __restrict__ s) {
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31, g = blockIdx.y;
  const long long row = (long long)blockIdx.x * QROWS + (threadIdx.x >> 5);
  if (row >= M) return;
  const int Kp = b8::padded(K), c0 = g * b8::GRP * b8::BLK + lane * 4;
  Four<T, VEC, 1> in[b8::GRP];
#pragma unroll
  for (int b = 0; b < b8::GRP; ++b) in[b].load(x + (size_t)row * K, c0 + b * b8::BLK, K);
  uint32_t word = b8::ONES;
#pragma unroll
  for (int b = 0; b < b8::GRP; ++b) {
    const int c = c0 + b * b8::BLK;
    if (c < Kp) {   // the same for the whole warp: Kp is a multiple of 128
      float2 v[2];
      in[b].get(v);
      uint32_t eb;
      *reinterpret_cast<uint32_t*>(q + (size_t)row * Kp + c) = b8::encode_block(v, eb);
      word = (word & ~(0xffu << (8 * b))) | (eb << (8 * b));
    }
  }
  if (lane == 0) s[(size_t)g * M + row] = word;
}

template <typename T>
int quant_launch(const void* x, int M, int K, void* q, void* s, cudaStream_t st) {
  const dim3 grid((M + QROWS - 1) / QROWS, b8::groups(K));
  const bool vec = K % 4 == 0 && reinterpret_cast<uintptr_t>(x) % (4 * sizeof(T)) == 0;
  const cudaError_t e =
      vec ? launch_k(quant_block_kernel<T, true>, grid, QROWS * 32, 0, st, static_cast<const T*>(x), M, K,
                     static_cast<uint8_t*>(q), static_cast<uint32_t*>(s))
          : launch_k(quant_block_kernel<T, false>, grid, QROWS * 32, 0, st, static_cast<const T*>(x), M, K,
                     static_cast<uint8_t*>(q), static_cast<uint32_t*>(s));
  return e == cudaSuccess ? FW_OK : FW_ECUDA;
}

// ---------------------------------------------------------------- norms around a block
struct NormArgs {
  float* resid;
  const void* y;                                  // the block's output, null: no residual update
  const __nv_bfloat16 *post_w, *post_b, *pre_w, *pre_b;
  const float *gate, *shift, *scale;              // [frames, D]
  float resid_scale, branch_scale, eps;
  int post, pre;                                  // FW_NORM_*
  int M, D, rows_per_frame;
  void* out;                                      // bf16 [M, D] or codes [M, Dp]; null: no second norm
  uint8_t* out_s;                                 // exponents of codes, null: bf16
};

// One row per CTA of W warps; warp w holds blocks [w NB, w NB + NB) of 128 columns in
// registers, four columns per lane and block.  HBM bounds it (12 bytes per element in bf16), but a row's bytes wait
// behind up to four sums over the row, so many rows have to be in flight: 2640 x 1536 in 11.1 us (4.4 TB/s),
// 6032 x 1536 in 21.5 us (5.2 TB/s), 4680 x 5120 in 54.0 us (5.3 TB/s), to e4m3 58.0.  Slower: CTAs that take several
// rows, the next one's loads in flight (16.8 us at 2640 x 1536), and rows brought to a ring in shared memory by bulk copies
// with a warp or four per row (27 us): fewer warps per SM are left to work through the sums; mean and square in one
// sum of three numbers, joined pairwise (13.4 us); and asking for later rows in L2 ahead of their CTAs (2640 rows
// 11.7 -> 11.8, 4680 rows 56.3 -> 54.4 in bf16 but 59.5 -> 60.2 in e4m3).
template <int W>
__device__ __forceinline__ float row_sum(float v, float* slot, int warp, int lane) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (lane == 0) slot[warp] = v;
  __syncthreads();
  float t = 0.f;
#pragma unroll
  for (int i = 0; i < W; ++i) t += slot[i];
  return t;
}

// From one of a lane's four columns of a block to the next: where a row's addresses are not aligned to
// four elements, a lane takes every 32nd column, so that each of the warp's scalar accesses is contiguous
// (2640 x 1535 14.0 us; scalar accesses of four adjacent columns 27.0).
template <bool VEC>
constexpr int column_step = VEC ? 1 : 32;

// Normalises x in place: fp32 mean and, about it, fp32 mean square (two sums, no cancellation).  Pairs of
// columns on the packed fp32 pipe: with few rows per SM in flight, instructions count as much as bytes.
template <bool VEC, int W, int NB>
__device__ __forceinline__ void norm_row(float2 (&x)[NB][2], int kind, float eps, int D, int c0, float* slots, int warp,
                                         int lane) {
  const float inv_d = 1.f / (float)D;
  if (kind == FW_NORM_LAYER) {
    float2 t = make_float2(0.f, 0.f);
#pragma unroll
    for (int b = 0; b < NB; ++b) t = __fadd2_rn(t, __fadd2_rn(x[b][0], x[b][1]));   // zeros behind D
    const float mu = row_sum<W>(t.x + t.y, slots, warp, lane) * inv_d;
    const float2 m2 = make_float2(-mu, -mu);
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      x[b][0] = __fadd2_rn(x[b][0], m2);
      x[b][1] = __fadd2_rn(x[b][1], m2);
    }
    if (D % (W * NB * b8::BLK) != 0) {   // zeros behind D again
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        const int c = c0 + b * b8::BLK;
        if (c >= D) x[b][0].x = 0.f;
        if (c + column_step<VEC> >= D) x[b][0].y = 0.f;
        if (c + 2 * column_step<VEC> >= D) x[b][1].x = 0.f;
        if (c + 3 * column_step<VEC> >= D) x[b][1].y = 0.f;
      }
    }
  }
  float2 t = make_float2(0.f, 0.f);
#pragma unroll
  for (int b = 0; b < NB; ++b) t = __ffma2_rn(x[b][1], x[b][1], __ffma2_rn(x[b][0], x[b][0], t));
  const float r = rsqrtf(row_sum<W>(t.x + t.y, slots + W, warp, lane) * inv_d + eps);
  const float2 r2 = make_float2(r, r);
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    x[b][0] = __fmul2_rn(x[b][0], r2);
    x[b][1] = __fmul2_rn(x[b][1], r2);
  }
}

// Warps that an SM has to hold, which sets the registers: 48 of them (about 40 registers) measured 15.7 us at
// 2640 x 1536, 40 11.7, 32 11.5 (but 23.7 against 22.4 at 6032 rows), as many as the compiler's 67 registers allow
// 12.0; at 4680 x 5120 30 warps 56.3 us, 20 (69 registers) 63.7, 40 97.  Scalar accesses take more registers: 2640 x
// 1535 40 warps 18.8 us, 32 14.0, 24 15.0; 4680 x 4799 30 warps 97, 20 75.6.
constexpr int norm_warps(bool VEC, int NB) {
  return VEC ? (NB <= 3 ? 40 : NB == 4 ? 32 : 16) : (NB <= 3 ? 32 : NB == 4 ? 20 : 16);
}

template <typename Y, bool VEC, int W, int NB>
__global__ void __launch_bounds__(W * 32, norm_warps(VEC, NB) / W) norm_gate_resid_kernel(const NormArgs a) {
  pdl_trigger();
  pdl_wait();
  __shared__ float slots[4 * W];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row = blockIdx.x, D = a.D;
  const int b0 = warp * NB, c0 = b0 * b8::BLK + (VEC ? lane * 4 : lane);
  constexpr int STEP = column_step<VEC>;
  const size_t frame = (size_t)(row / a.rows_per_frame) * D;
  float* xr = a.resid + (size_t)row * D;
  // A parameter's loads for all blocks are issued together, several parameters' before one is used: with
  // one block after the other, each waited for its own.  The branch's parameters are asked for before the first
  // sum, the output's after the last one (earlier, their registers would cost rows in flight).
  Four<__nv_bfloat16, VEC, STEP> w[NB];
  Four<float, VEC, STEP> f[NB], f2[NB];
  auto fetch = [&](auto& v, const auto* base) {
#pragma unroll
    for (int b = 0; b < NB; ++b) v[b].load(base, c0 + b * b8::BLK, D);
  };
  auto mul = [&](float2 (&v)[NB][2], auto& by) {
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      float2 p[2];
      by[b].get(p);
      v[b][0] = __fmul2_rn(v[b][0], p[0]);
      v[b][1] = __fmul2_rn(v[b][1], p[1]);
    }
  };
  auto add = [&](float2 (&v)[NB][2], auto& by) {
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      float2 p[2];
      by[b].get(p);
      v[b][0] = __fadd2_rn(v[b][0], p[0]);
      v[b][1] = __fadd2_rn(v[b][1], p[1]);
    }
  };
  Four<float, VEC, STEP> xin[NB];
  fetch(xin, xr);
  float2 x[NB][2];
  if (a.y) {
    Four<Y, VEC, STEP> yin[NB];
    fetch(yin, static_cast<const Y*>(a.y) + (size_t)row * D);
    if (a.post_w) fetch(w, a.post_w);
    if (a.gate) fetch(f, a.gate + frame);
    float2 y[NB][2];
#pragma unroll
    for (int b = 0; b < NB; ++b) yin[b].get(y[b]);
    if (a.post != FW_NORM_NONE) norm_row<VEC, W, NB>(y, a.post, a.eps, D, c0, slots, warp, lane);
    if (a.post_w) mul(y, w);
    if (a.post_b) {
      fetch(w, a.post_b);
      add(y, w);
    }
    if (a.gate) mul(y, f);
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const int c = c0 + b * b8::BLK;
      xin[b].get(x[b]);
      const float2 rs = make_float2(a.resid_scale, a.resid_scale), bs = make_float2(a.branch_scale, a.branch_scale);
      x[b][0] = __ffma2_rn(bs, y[b][0], __fmul2_rn(rs, x[b][0]));
      x[b][1] = __ffma2_rn(bs, y[b][1], __fmul2_rn(rs, x[b][1]));
      if (VEC) {
        if (c < D) *reinterpret_cast<float4*>(xr + c) = make_float4(x[b][0].x, x[b][0].y, x[b][1].x, x[b][1].y);
      } else {
        if (c < D) xr[c] = x[b][0].x;
        if (c + STEP < D) xr[c + STEP] = x[b][0].y;
        if (c + 2 * STEP < D) xr[c + 2 * STEP] = x[b][1].x;
        if (c + 3 * STEP < D) xr[c + 3 * STEP] = x[b][1].y;
      }
    }
  } else {
#pragma unroll
    for (int b = 0; b < NB; ++b) xin[b].get(x[b]);
  }
  if (!a.out) return;
  if (a.pre != FW_NORM_NONE) norm_row<VEC, W, NB>(x, a.pre, a.eps, D, c0, slots + 2 * W, warp, lane);
  if (a.pre_w) fetch(w, a.pre_w);
  if (a.scale) {
    fetch(f, a.scale + frame);
    fetch(f2, a.shift + frame);
  }
  if (a.pre_w) mul(x, w);
  if (a.pre_b) {
    fetch(w, a.pre_b);
    add(x, w);
  }
  if (a.scale) {
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      float2 p[2], t[2];
      f[b].get(p);
      f2[b].get(t);
#pragma unroll
      for (int i = 0; i < 2; ++i) x[b][i] = __ffma2_rn(x[b][i], p[i], __fadd2_rn(x[b][i], t[i]));   // x (1 + p) + t
    }
  }
  const int Dp = b8::padded(D);
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    const int c = c0 + b * b8::BLK;
    if (a.out_s) {
      const int blk = b0 + b;
      if (blk * b8::BLK < Dp) {
        // Behind D every parameter reads as zero and so is the value, or it is NaN where the row's norm is; neither has
        // a say in the exponent, and the codes there are zero.
        uint32_t eb;
        const uint32_t code = b8::encode_block(x[b], eb);
        uint8_t* o = static_cast<uint8_t*>(a.out) + (size_t)row * Dp + c;
        if (VEC) {
          *reinterpret_cast<uint32_t*>(o) = c < D ? code : 0u;   // D % 4 == 0
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) o[i * STEP] = c + i * STEP < D ? (uint8_t)(code >> (8 * i)) : 0;
        }
        if (lane == 0) a.out_s[((size_t)(blk / b8::GRP) * a.M + row) * b8::GRP + blk % b8::GRP] = (uint8_t)eb;
      }
    } else if (VEC) {
      if (c < D)
        *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(a.out) + (size_t)row * D + c) =
            make_uint2(pack_bf16(x[b][0].x, x[b][0].y), pack_bf16(x[b][1].x, x[b][1].y));
    } else {
      __nv_bfloat16* o = static_cast<__nv_bfloat16*>(a.out) + (size_t)row * D;
      if (c < D) o[c] = __float2bfloat16_rn(x[b][0].x);
      if (c + STEP < D) o[c + STEP] = __float2bfloat16_rn(x[b][0].y);
      if (c + 2 * STEP < D) o[c + 2 * STEP] = __float2bfloat16_rn(x[b][1].x);
      if (c + 3 * STEP < D) o[c + 3 * STEP] = __float2bfloat16_rn(x[b][1].y);
    }
  }
  if (a.out_s && threadIdx.x == 0)   // places behind the last block
    for (int blk = b8::blocks(D); blk < b8::groups(D) * b8::GRP; ++blk)
      a.out_s[((size_t)(blk / b8::GRP) * a.M + row) * b8::GRP + blk % b8::GRP] = 127;
}

// Warps per row and blocks per warp (W x NB) by the row's width, as close a fit as there is: blocks that a warp
// holds behind the row cost registers and idle lanes.  Measured for 6032 rows: 384 columns 2 x 2 9.4 us, 4 x 1 10.6;
// 768 columns 3 x 2 13.1, 4 x 2 14.6, 4 x 3 17.4; 1152 columns 3 x 3 18.4, 4 x 3 19.9; for 4680 rows: 2560 columns
// 7 x 3 31.2, 8 x 3 34.1; 4096 columns 8 x 4 45.4, 11 x 3 49.9, 10 x 4 52.2; 6144 columns 16 x 3 72.8, 12 x 4 72.8 (but 24.9
// and 30.8 for 1000 rows of 6143), 16 x 4 83.2.  Fewer blocks per warp make more warps wait for a row's sums: 1536
// columns 4 x 3 11.2 for 2640 rows, 6 x 2 11.5, 12 x 1 17.1; 5120 columns 10 x 4 57.2 for 4680 rows, 14 x 3 63.5, 20 x 2
// 65.2; rows that are not aligned: 1535 columns 13.1, 13.8 and 18.0; 4799 columns 74, 76 and 112.
template <typename Y, bool VEC>
int norm_launch(const NormArgs& a, cudaStream_t s) {
  const int nb = b8::blocks(a.D);
  auto go = [&](auto kern, int warps) {
    return launch_k(kern, dim3(a.M), dim3(warps * 32), 0, s, a) == cudaSuccess ? FW_OK : FW_ECUDA;
  };
  if (nb <= 2) return go(norm_gate_resid_kernel<Y, VEC, 2, 1>, 2);
  if (nb <= 4) return go(norm_gate_resid_kernel<Y, VEC, 2, 2>, 2);
  if (nb <= 6) return go(norm_gate_resid_kernel<Y, VEC, 3, 2>, 3);
  if (nb <= 8) return go(norm_gate_resid_kernel<Y, VEC, 4, 2>, 4);
  if (nb <= 9) return go(norm_gate_resid_kernel<Y, VEC, 3, 3>, 3);
  if (nb <= 12) return go(norm_gate_resid_kernel<Y, VEC, 4, 3>, 4);
  if (nb <= 15) return go(norm_gate_resid_kernel<Y, VEC, 5, 3>, 5);
  if (nb <= 18) return go(norm_gate_resid_kernel<Y, VEC, 6, 3>, 6);
  if (nb <= 21) return go(norm_gate_resid_kernel<Y, VEC, 7, 3>, 7);
  if (nb <= 24) return go(norm_gate_resid_kernel<Y, VEC, 8, 3>, 8);
  if (nb <= 32) return go(norm_gate_resid_kernel<Y, VEC, 8, 4>, 8);
  if (nb <= 40) return go(norm_gate_resid_kernel<Y, VEC, 10, 4>, 10);
  if (nb <= 48) return go(norm_gate_resid_kernel<Y, VEC, 16, 3>, 16);
  if (nb <= 64) return go(norm_gate_resid_kernel<Y, VEC, 16, 4>, 16);
  return go(norm_gate_resid_kernel<Y, VEC, 16, 8>, 16);
}

}  // namespace
}  // namespace fw

extern "C" {

int fw_quant_e4m3_block(const void* x, int dtype, int M, int K, void* q, void* s, void* stream) {
  using namespace fw;
  if (M < 0 || K <= 0 || K > FW_BLOCK_MAX_COLS) return FW_ESHAPE;
  if (M == 0) return FW_OK;
  if (!x || !q || !s) return FW_EINVAL;
  if (dtype != FW_BF16 && dtype != FW_F16 && dtype != FW_F32) return FW_EINVAL;
  if (reinterpret_cast<uintptr_t>(q) % 16 || reinterpret_cast<uintptr_t>(s) % 4 ||
      reinterpret_cast<uintptr_t>(x) % (dtype == FW_F32 ? 4 : 2))
    return FW_EALIGN;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (dtype) {
    case FW_BF16: return quant_launch<__nv_bfloat16>(x, M, K, q, s, st);
    case FW_F16: return quant_launch<__half>(x, M, K, q, s, st);
    default: return quant_launch<float>(x, M, K, q, s, st);
  }
}

int fw_norm_gate_resid(const fw_norm_args* n, void* stream) {
  using namespace fw;
  if (!n) return FW_EINVAL;
  if (n->M < 0 || n->D <= 0 || n->D > FW_NORM_MAX_COLS || n->rows_per_frame <= 0) return FW_ESHAPE;
  if (n->post < FW_NORM_NONE || n->post > FW_NORM_RMS || n->pre < FW_NORM_NONE || n->pre > FW_NORM_RMS) return FW_EINVAL;
  if (n->y_dtype != FW_BF16 && n->y_dtype != FW_F32) return FW_EINVAL;
  if (n->M == 0) return FW_OK;
  if (!n->resid || (!n->scale) != (!n->shift) || (n->out_s && !n->out) || (!n->y && !n->out)) return FW_EINVAL;
  if (n->out_s && reinterpret_cast<uintptr_t>(n->out) % 16) return FW_EALIGN;
  NormArgs a;
  a.resid = n->resid;
  a.y = n->y;
  a.post_w = static_cast<const __nv_bfloat16*>(n->post_w);
  a.post_b = static_cast<const __nv_bfloat16*>(n->post_b);
  a.pre_w = static_cast<const __nv_bfloat16*>(n->pre_w);
  a.pre_b = static_cast<const __nv_bfloat16*>(n->pre_b);
  a.gate = n->gate;
  a.shift = n->shift;
  a.scale = n->scale;
  a.resid_scale = n->resid_scale;
  a.branch_scale = n->branch_scale;
  a.eps = n->eps;
  a.post = n->post;
  a.pre = n->pre;
  a.M = n->M;
  a.D = n->D;
  a.rows_per_frame = n->rows_per_frame;
  a.out = n->out;
  a.out_s = static_cast<uint8_t*>(n->out_s);
  // four columns at a time where every row of every tensor starts at a multiple of four elements
  uintptr_t f32 = 0, b16 = 0;
  for (const void* p : {(const void*)n->resid, (const void*)n->gate, (const void*)n->shift, (const void*)n->scale,
                        n->y_dtype == FW_F32 ? n->y : nullptr})
    f32 |= reinterpret_cast<uintptr_t>(p);
  for (const void* p : {n->post_w, n->post_b, n->pre_w, n->pre_b, n->y_dtype == FW_BF16 ? n->y : nullptr,
                        n->out_s ? nullptr : (const void*)n->out})
    b16 |= reinterpret_cast<uintptr_t>(p);
  if (f32 % 4 || b16 % 2) return FW_EALIGN;
  const bool vec = n->D % 4 == 0 && f32 % 16 == 0 && b16 % 8 == 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (n->y_dtype == FW_F32) return vec ? norm_launch<float, true>(a, s) : norm_launch<float, false>(a, s);
  return vec ? norm_launch<__nv_bfloat16, true>(a, s) : norm_launch<__nv_bfloat16, false>(a, s);
}

}  // extern "C"
