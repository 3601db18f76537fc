// Matrix product of block-scaled e4m3 operands (format: fw_block8.cuh) on tcgen05 for sm_100a:
//   C[m, n] = act(sum over blocks b of 2^(ea[m,b] + eb[n,b]) * sum over k in b of a[m,k] b[n,k] + bias[n])
// with C in bf16, fp32, or e4m3 with block scales again.
//
// The scales are powers of two held as UE8M0 bytes, so tcgen05.mma kind::mxf8f6f4 multiplies them
// in at full e4m3 rate: its scale factors live in Tensor Memory, one 32-bit word per row (row r of an
// operand: lane r % 32 of every lane quarter, column r / 32), of which an instruction picks one byte for its 32 of
// K.  A word here holds the exponents of four blocks of 128, so a word loaded once serves
// 512 of K: the four instructions of a block name the same byte.
#include "fw_gemm_block.cuh"

#include <cmath>
#include <type_traits>

namespace fw {

namespace {

// ---------------------------------------------------------------- one CTA, 128 columns of C x BN rows
// The weights' 128 rows are the instruction's M side and BN rows of A its N side, so a few rows
// cost a small tile (BN = 16) instead of an idle 128-row one, and a tile's 128 columns of C
// are one block of an e4m3 result.  Warp 0 loads tiles, warp 1 issues the MMAs, warps 2-5
// carry the exponent words to Tensor Memory, then transpose the accumulator through the
// (then idle) tile memory; all warps write C a row at a time.
//
// Few tiles would leave most SMs idle and stream the weights through few of them, so the k-blocks of a tile are
// split over a cluster of CTAs.  Each stages its partial accumulator in its own shared memory; then each takes
// every splits-th row, adds the partials of all ranks in rank order (the same sum on every run) and writes it.
//
// What bounds it: with a few rows the weights' bytes behind about 4 us of launch, first loads and result
// (1 x 1536 x 1536 4.4 us; 1 x 5120 x 13824, 71 MB, 16.0 us or 4.4 TB/s); with a few hundred rows the chain of
// k-blocks of a CTA, 0.5 us each, which the split shortens for a join of 2.7 us (of 11.4 us at 512 x 1536 x 4096).
namespace nk {
constexpr int THREADS = 192, MAX_SPLITS = 8;
template <int BN>
struct Cfg {
  static constexpr int P_BYTES = 128 * 128, Q_BYTES = BN * 128, STAGE = P_BYTES + Q_BYTES;
  static constexpr int STAGES = BN >= 128 ? 3 : 4;
  static constexpr int BAR_OFF = STAGES * STAGE;
  static constexpr int SMEM = BAR_OFF + 256 + 1024;
  static constexpr int QCOLS = BN >= 32 ? BN / 32 : 1;                // scale columns of the BN rows
  static constexpr int SF_COL = BN >= 32 ? BN : 32;                   // two buffers of 4 + QCOLS columns, 8 apart
  static constexpr uint32_t TMEM_COLS = SF_COL + 16 <= 64 ? 64 : SF_COL + 16 <= 128 ? 128 : 256;
  static_assert(4 + QCOLS <= 8 && SF_COL + 16 <= 256, "scale columns");
  static_assert(BN * 128 * 4 <= BAR_OFF, "accumulator staging");
};
}  // namespace nk

__device__ __forceinline__ float4 ld_cluster4(uint32_t addr) {   // shared memory of a CTA of the cluster
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

// v: columns [n, n + 4) of row m of C before the bias; columns that do not exist hold anything.
template <int ACT, int OUT>
__device__ __forceinline__ void write_row4(const BlockGemmArgs& a, int m, int n, const float4& u,
                                           const float (&bias)[4], bool vec) {
  const int N = a.N;
  const float2 x = activate2<ACT>(make_float2(u.x + bias[0], u.y + bias[1]));
  const float2 y = activate2<ACT>(make_float2(u.z + bias[2], u.w + bias[3]));
  if constexpr (OUT == FW_U8) {
    const float2 v[2] = {make_float2(n < N ? x.x : 0.f, n + 1 < N ? x.y : 0.f),
                         make_float2(n + 2 < N ? y.x : 0.f, n + 3 < N ? y.y : 0.f)};
    uint32_t eb;
    const uint32_t code = b8::encode_block(v, eb);
    const int blk = n / b8::BLK;
    *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(a.out) + (size_t)m * b8::padded(N) + n) = code;
    if ((threadIdx.x & 31) == 0) {
      uint8_t* s = a.out_s + ((size_t)(blk / b8::GRP) * a.M + m) * b8::GRP;
      s[blk % b8::GRP] = (uint8_t)eb;
      if (blk == b8::blocks(N) - 1)   // places behind the last block
        for (int j = blk % b8::GRP + 1; j < b8::GRP; ++j) s[j] = 127;
    }
  } else {
    const size_t at = (size_t)m * N + n;
    if constexpr (OUT == FW_F32) {
      float* o = static_cast<float*>(a.out) + at;
      if (vec) {
        *reinterpret_cast<float4*>(o) = make_float4(x.x, x.y, y.x, y.y);
      } else {
        if (n < N) o[0] = x.x;
        if (n + 1 < N) o[1] = x.y;
        if (n + 2 < N) o[2] = y.x;
        if (n + 3 < N) o[3] = y.y;
      }
    } else {
      __nv_bfloat16* o = static_cast<__nv_bfloat16*>(a.out) + at;
      if (vec) {
        *reinterpret_cast<uint2*>(o) = make_uint2(pack_bf16(x.x, x.y), pack_bf16(y.x, y.y));
      } else {
        if (n < N) o[0] = __float2bfloat16_rn(x.x);
        if (n + 1 < N) o[1] = __float2bfloat16_rn(x.y);
        if (n + 2 < N) o[2] = __float2bfloat16_rn(y.x);
        if (n + 3 < N) o[3] = __float2bfloat16_rn(y.y);
      }
    }
  }
}

template <int BN, int ACT, int OUT>
__global__ void __launch_bounds__(nk::THREADS)
    gemm_block_kernel(const __grid_constant__ CUtensorMap tmP, const __grid_constant__ CUtensorMap tmQ,
                      const BlockGemmArgs a) {
  using C = nk::Cfg<BN>;
  pdl_trigger();
  extern __shared__ uint8_t smem_raw[];
  const uint32_t pad = (1024u - (smem_u32(smem_raw) & 1023u)) & 1023u;
  uint8_t* smem = smem_raw + pad;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::BAR_OFF);
  uint64_t* empty = full + C::STAGES;
  uint64_t* sf_full = empty + C::STAGES;   // [2]
  uint64_t* sf_free = sf_full + 2;         // [2]
  uint64_t* done = sf_free + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int splits = a.splits, rank = splits > 1 ? (int)cluster_ctarank() : 0;
  const int n0 = (int)(blockIdx.x / splits) * 128, m0 = blockIdx.y * BN;
  const int num_kb = a.K / b8::BLK, kb0 = num_kb * rank / splits, kb1 = num_kb * (rank + 1) / splits;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(full + s, 1);
      mbar_init(empty + s, 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(sf_full + b, 128);
      mbar_init(sf_free + b, 1);
    }
    mbar_init(done, 1);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, C::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();
  if (warp == 0) {
    if (lane == 0) {
      uint32_t used = 0, last_par = 0;
      for (int kb = kb0, i = 0; kb < kb1; ++kb, ++i) {
        const int s = i % C::STAGES;
        const uint32_t par = (uint32_t)(i / C::STAGES) & 1u;
        if (!wait_on(empty + s, par ^ 1u, abort_flag, a.status, DEV_TIMEOUT_PRODUCER)) break;
        mbar_arrive_expect_tx(full + s, C::STAGE);
        tma_load_2d(smem + s * C::STAGE, &tmP, full + s, kb * b8::BLK, n0);
        tma_load_2d(smem + s * C::STAGE + C::P_BYTES, &tmQ, full + s, kb * b8::BLK, m0);
        used |= 1u << s;
        last_par = (last_par & ~(1u << s)) | (par << s);
      }
      volatile int no_abort = 0;   // no copy into this CTA's memory is in flight at exit
      for (int s = 0; s < C::STAGES; ++s)
        if (used >> s & 1u) mbar_wait(full + s, last_par >> s & 1u, &no_abort, a.status, DEV_TIMEOUT_DRAIN);
    }
  } else if (warp == 1) {
    const uint32_t one = lane == 0;
    constexpr uint32_t idesc = idesc_mx8(128, BN);
    bool ok = true;
    for (int kb = kb0, i = 0; kb < kb1; ++kb, ++i) {
      const int s = i % C::STAGES, grp = kb / b8::GRP - kb0 / b8::GRP, buf = grp & 1;
      if (i == 0 || kb % b8::GRP == 0)
        ok = wait_on(sf_full + buf, (uint32_t)(grp >> 1) & 1u, abort_flag, a.status, DEV_TIMEOUT_MMA);
      if (ok) ok = wait_on(full + s, (uint32_t)(i / C::STAGES) & 1u, abort_flag, a.status, DEV_TIMEOUT_MMA);
      if (!ok) break;
      tc_fence_after();
      const uint32_t desc = desc_lo(smem_u32(smem + s * C::STAGE));
      const uint32_t sf = tmem + (uint32_t)(C::SF_COL + buf * 8);
      umma_mx8_block<1>(one, tmem, desc, desc + (C::P_BYTES >> 4), with_scale_byte(idesc, (uint32_t)(kb % b8::GRP)), sf,
                        sf + 4, i != 0);
      umma_commit_if<1>(one, empty + s);
      if (kb % b8::GRP == b8::GRP - 1) umma_commit_if<1>(one, sf_free + buf);
    }
    umma_commit_if<1>(one, done);
    volatile int no_abort = 0;
    mbar_wait(done, 0, &no_abort, a.status, DEV_TIMEOUT_DRAIN);
  } else if (warp < 6) {
    const int q = warp & 3;   // lane quarter of Tensor Memory
    const uint32_t quarter = tmem + ((uint32_t)(q * 32) << 16);
    bool ok = true;
    for (int g = kb0 / b8::GRP, i = 0; g * b8::GRP < kb1; ++g, ++i) {
      uint32_t wp[4], wq[C::QCOLS];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int r = n0 + c * 32 + lane;
        wp[c] = r < a.N ? __ldg(a.sb + (size_t)g * a.N + r) : b8::ONES;
      }
#pragma unroll
      for (int c = 0; c < C::QCOLS; ++c) {
        const int r = m0 + c * 32 + lane;
        wq[c] = r < a.M && c * 32 + lane < BN ? __ldg(a.sa + (size_t)g * a.M + r) : b8::ONES;
      }
      const int buf = i & 1;
      if (i >= 2) {
        ok = __all_sync(0xffffffffu, wait_on(sf_free + buf, (uint32_t)((i - 2) >> 1) & 1u, abort_flag, a.status,
                                             DEV_TIMEOUT_EPILOGUE));
        if (!ok) break;
        tc_fence_after();
      }
      tmem_st(quarter + (uint32_t)(C::SF_COL + buf * 8), wp);
      tmem_st(quarter + (uint32_t)(C::SF_COL + buf * 8 + 4), wq);
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(sf_full + buf);
    }
    if (ok) ok = __all_sync(0xffffffffu, wait_on(done, 0, abort_flag, a.status, DEV_TIMEOUT_EPILOGUE));
    if (ok) {
      // accumulator lane = column of C, column = row of C; staged as [row][128 columns]
      tc_fence_after();
      float* st = reinterpret_cast<float*>(smem);
      const int col = q * 32 + lane;
      if constexpr (BN == 16) {
        uint32_t r[16];
        tmem_ld16(quarter, r);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 16; ++i) st[i * 128 + col] = __uint_as_float(r[i]);
      } else {
#pragma unroll 1
        for (int c = 0; c < BN / 32; ++c) {
          uint32_t r[32];
          tmem_ld32(quarter + (uint32_t)(c * 32), r);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; ++i) st[(c * 32 + i) * 128 + col] = __uint_as_float(r[i]);
        }
      }
      tc_fence_before();
    }
    if (!ok) *abort_flag = 1;
  }
  tc_fence_before();
  const int n = n0 + lane * 4;   // this lane's columns of C; their bias arrives during the barrier
  unsigned short bias_bits[4] = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (a.bias && n + i < a.N) bias_bits[i] = __ldg(reinterpret_cast<const unsigned short*>(a.bias) + n + i);
  if (splits > 1)
    cluster_sync();   // every rank's partial is staged
  else
    __syncthreads();
  // Nothing is written where a wait ran out, nor, in a split, where another rank's did: its part is not staged.
  const int gave_up = splits > 1 ? cluster_abort_flag(abort_flag, splits) : *abort_flag;
  if (splits > 1 || __all_sync(0xffffffffu, !gave_up)) {
    float bias[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) bias[i] = __uint_as_float((uint32_t)bias_bits[i] << 16);
    const bool vec = a.N % 4 == 0 && n < a.N;   // four columns at an address aligned to them
    const float* st = reinterpret_cast<const float*>(smem) + lane * 4;
    const int rows = min(BN, a.M - m0);
    constexpr int WARPS = nk::THREADS / 32;
    if (splits == 1) {
      for (int r = warp; r < rows; r += 4 * WARPS) {   // four rows at a time, for as many loads in flight
        float4 u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) u[i] = *reinterpret_cast<const float4*>(st + min(r + i * WARPS, BN - 1) * 128);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (r + i * WARPS < rows) write_row4<ACT, OUT>(a, m0 + r + i * WARPS, n, u[i], bias, vec);
      }
    } else {
      for (int r = warp * splits + rank; r < rows; r += WARPS * splits) {
        float4 u[nk::MAX_SPLITS];
#pragma unroll
        for (int k = 0; k < nk::MAX_SPLITS; ++k)
          if (k < splits) u[k] = ld_cluster4(mapa_cluster(st + r * 128, (uint32_t)k));
        if (__any_sync(0xffffffffu, gave_up)) break;   // looked at here, the flags' way is hidden behind the partials'
#pragma unroll
        for (int k = 1; k < nk::MAX_SPLITS; ++k)
          if (k < splits) u[0].x += u[k].x, u[0].y += u[k].y, u[0].z += u[k].z, u[0].w += u[k].w;
        write_row4<ACT, OUT>(a, m0 + r, n, u[0], bias, vec);
      }
    }
  }
  if (splits > 1) cluster_sync();   // no CTA leaves while another reads its partial
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, C::TMEM_COLS);
  }
}

template <int BN>
int launch_nk(const void* A8, const void* B8, const BlockGemmArgs& a, cudaStream_t s) {
  using C = nk::Cfg<BN>;
  CUtensorMap tp, tq;
  int rc = make_tmap_2d(&tp, B8, 1, a.N, a.K, a.K, 128, 128, true);
  if (!rc) rc = make_tmap_2d(&tq, A8, 1, a.M, a.K, a.K, BN, 128, true);
  if (rc) return rc;
  const dim3 grid((a.N + 127) / 128 * a.splits, (a.M + BN - 1) / BN);
  if (grid.y > 65535) return FW_ESHAPE;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = nk::THREADS;
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  cfg.attrs = attr;
  if (a.splits > 1) {
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = a.splits;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.numAttrs = 1;
  }
  if (pdl_enabled()) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
    ++cfg.numAttrs;
  }
  auto go = [&](auto kern) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM) != cudaSuccess)
      return FW_ECUDA;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, tp, tq, a);
    note_launch();
    return e == cudaSuccess ? FW_OK : FW_ECUDA;
  };
  auto by_act = [&](auto out) {
    constexpr int O = decltype(out)::value;
    switch (a.act) {
      case ACT_TANH: return go(gemm_block_kernel<BN, ACT_TANH, O>);
      case ACT_ERF: return go(gemm_block_kernel<BN, ACT_ERF, O>);
      default: return go(gemm_block_kernel<BN, ACT_NONE, O>);
    }
  };
  switch (a.out_dtype) {
    case FW_U8: return by_act(std::integral_constant<int, FW_U8>{});
    case FW_F32: return by_act(std::integral_constant<int, FW_F32>{});
    default: return by_act(std::integral_constant<int, FW_BF16>{});
  }
}

// Which kernel, tile and split: the least of a time model (us) whose constants were fitted to measured times (small
// tiles: 70 sizes of 1 to 4000 rows, 30 to 13824 columns, 60 to 8960 of K; between the two kernels: 37 sizes).  Of 52
// sizes near the border measured since, nine went to the slower kernel by more than 2 %, most of them to small tiles
// with a short K and an e4m3 or fp32 result (3250 x 1742 x 489 to e4m3 18.1 us, 9.9 wide). Small tiles: launch, then
// the busiest SM's operand bytes, or the latency of a CTA's chain of k-blocks, or HBM, then the exposed epilogue and
// the join of a split; wide kernel: waves of 256 x 256 tiles, more for rows that no TMA store can address.
// Both sides, measured (us):
//   small tiles   880 x 1536 x 8960   18.7 (split 3 ways; 30.9 unsplit)   27.7 wide
//                 512 x 1536 x 13824  18.5                                38.2 wide
//                 1001 x 777 x 1283    7.6                                11.6 wide
//                 512 x 1536 x 4096   11.4 (split 5 ways; 16.2 unsplit)   15.5 wide
//   wide         2640 x 1536 x 1536   10.2 small tiles                    10.6 wide (the border)
//                 512 x 13824 x 5120  45.6                                35.6
//                6032 x 1536 x 1536   20.1                                15.8
//   a split         1 x 1536 x 1536    4.4 split 6 ways, 6.2 unsplit; 1 x 9216 x 1536 7.0 split 4 ways, 6.8 unsplit
// A split's CTAs fill at most 9/10 of two per SM: clusters do not fit every SM of a GPC, and what is left over
// waits for whole tiles to end (512 x 1536 x 4096 on 64-row tiles split 3 ways, 288 CTAs: 18.6 us).
struct Plan {
  int bn, splits;   // bn 0: the wide kernel
};
Plan make_plan(int M, int N, int num_kb, int out_dtype) {
  const int sms = num_sms();
  auto up = [](long long x, long long y) { return (x + y - 1) / y; };
  const double hbm = (((double)M + N) * num_kb * b8::BLK + 2.0 * M * N) / 5.2e6;
  const long long wide = up(M, 256) * up(N, 256), waves = up(wide, sms / 2);
  const bool tma_out = out_dtype == FW_U8 || N % (out_dtype == FW_F32 ? 4 : 8) == 0;
  Plan best = {0, 1};
  const double kb_us = 0.27 + 0.08 * fmin(1.0, wide / (sms * 0.5));   // of a k-block, on one pair and on all
  double least = 4.9 + waves * (num_kb * kb_us + (tma_out ? 0.4 : 1.9));
  for (int bn = 16; bn <= 128; bn *= 2) {
    if (up(M, bn) > 65535) continue;
    const long long tiles = up(N, 128) * up(M, bn);
    for (int sp = 1; sp <= nk::MAX_SPLITS && sp <= num_kb; ++sp) {
      if (sp > 1 && tiles * sp > sms * 9 / 5) break;
      const double per_sm = (double)up(tiles * sp, sms), kbs = (double)up(num_kb, sp);
      const double load = per_sm * kbs * (128 + bn) * b8::BLK / 1.8e5;
      const double chain = up(tiles * sp, 2 * sms) * kbs * 0.5;
      const double join = sp == 1 ? 0.0 : bn == 128 ? 4.6 : 3.4;
      const double t = 1.7 + fmax(fmax(load, chain), hbm) + 0.9 * bn / 128 * per_sm + join;
      if (t < least) {
        least = t;
        best = {bn, sp};
      }
    }
    if (bn >= M) break;   // one tile of rows
  }
  return best;
}

}  // namespace
}  // namespace fw

extern "C" int fw_gemm_e4m3_block(const void* A8, const void* sa, const void* B8, const void* sb, const void* bias,
                                  void* out, void* out_s, int M, int N, int K, int epilogue, int out_dtype,
                                  void* stream) {
  return fw_gemm_e4m3_block_status(A8, sa, B8, sb, bias, out, out_s, M, N, K, epilogue, out_dtype, nullptr, stream);
}

extern "C" int fw_gemm_e4m3_block_status(const void* A8, const void* sa, const void* B8, const void* sb,
                                         const void* bias, void* out, void* out_s, int M, int N, int K, int epilogue,
                                         int out_dtype, int* status, void* stream) {
  using namespace fw;
  if (M < 0 || N < 0 || K <= 0 || K > FW_BLOCK_MAX_COLS || N > FW_BLOCK_MAX_COLS) return FW_ESHAPE;
  BlockGemmArgs a;
  switch (epilogue) {
    case EPI_BF16: a.act = ACT_NONE; break;
    case EPI_GELU_BF16: a.act = ACT_TANH; break;
    case EPI_GELU_ERF_BF16: a.act = ACT_ERF; break;
    default: return FW_EINVAL;
  }
  if (out_dtype != FW_BF16 && out_dtype != FW_F32 && out_dtype != FW_U8) return FW_EINVAL;
  if (M == 0 || N == 0) return FW_OK;
  if (!A8 || !sa || !B8 || !sb || !out || (out_dtype == FW_U8) != (out_s != nullptr)) return FW_EINVAL;
  for (const void* p : {A8, B8, (const void*)out})
    if (reinterpret_cast<uintptr_t>(p) % 16) return FW_EALIGN;
  for (const void* p : {sa, sb, (const void*)out_s})
    if (reinterpret_cast<uintptr_t>(p) % 4) return FW_EALIGN;
  if (reinterpret_cast<uintptr_t>(bias) % 2 || reinterpret_cast<uintptr_t>(status) % 4) return FW_EALIGN;
  a.M = M;
  a.N = N;
  a.K = b8::padded(K);
  a.sa = static_cast<const uint32_t*>(sa);
  a.sb = static_cast<const uint32_t*>(sb);
  a.bias = static_cast<const __nv_bfloat16*>(bias);
  a.out_dtype = out_dtype;
  a.out = out;
  a.out_s = static_cast<uint8_t*>(out_s);
  a.status = status;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const Plan p = make_plan(M, N, a.K / b8::BLK, out_dtype);
  a.splits = p.splits;
  switch (p.bn) {
    case 16: return launch_nk<16>(A8, B8, a, s);
    case 32: return launch_nk<32>(A8, B8, a, s);
    case 64: return launch_nk<64>(A8, B8, a, s);
    case 128: return launch_nk<128>(A8, B8, a, s);
    default: return gemm_block_wide_launch(A8, B8, a, s);
  }
}
