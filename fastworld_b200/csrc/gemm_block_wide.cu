// Block-scaled e4m3 GEMM for large problems: 256 x 256 tiles of C on CTA pairs (tcgen05 cta_group::2).
//
// The two CTAs of a cluster each hold 128 rows of A and 128 rows of B of a k-block (32 KB instead of
// the 48 KB of a 128 x 256 tile on one CTA), and each one's Tensor Memory gets its 128 rows of the
// accumulator, all 256 columns.  Persistent over tiles; 12 warps per CTA:
//   warp 0      TMA producer of this CTA's halves (loads complete on the even CTA's `full`);
//   warp 1      even CTA: the one MMA issuer of the pair; both: Tensor Memory of the pair;
//   warp 2      exponent words of A's 128 rows and of all 256 rows of B to this CTA's shared memory, a group of
//               512 of K at a time, in the order that the copy reads;
//   warp 3      even CTA: copies them to the Tensor Memory of both (tcgen05.cp), two buffers of a group each;
//               odd CTA: tells the even one that its group is there;
//   warps 4-11  epilogue: lane quarter w % 4, column half (w - 4) / 4.
// Tensor Memory has 512 columns; two accumulators of 256 and the 24 of the scales do not
// fit side by side, so the accumulators overlap by 32 columns: even tiles at [0, 256), odd ones at [224, 480),
// scales from 480.  An epilogue reads the shared 32 columns first (an even tile's last, an
// odd tile's first) and the next tile's MMAs start once it has, so they still run under the rest of the epilogue.
// Every wait is bounded; a wait that runs out makes both CTAs unwind.
//
// What bounds it: the tensor core needs 2048 cycles for four k-blocks of 256 x 256 x 128, and their issue takes
// 2240 (270 cycles for a block's four MMAs, 100 for its wait, 60 for its commit), 0.30 us a block; with all pairs
// loading 0.36 us, 13 TB/s out of L2.  A call adds 4 us (first tile, last epilogue), a tile change 0.4 us.  2640 rows,
// bf16 result and bias, bursts of a millisecond at 1965 MHz: 4608 x 1536 19.7 us (1.9 PFLOP/s), 8960 x 1536 36.4 (2.0),
// 1536 x 8960 31.8 (2.3); 4680 x 13824 x 5120 242 us (2.7), and 279 us when it repeats for seconds at the power limit
// (1.30 GHz).  GELU in the tanh form hides behind the MMAs (8960 x 1536 38.0 us), in the erf form it does not (111 us:
// an erfcf call for each value, where a tile's 12 k-blocks take 4 us).
// Tried (before the exponents of the odd CTA were announced by a warp of their own with a release at cluster scope):
// tiles of 240 columns whose accumulators do not overlap (18.5 -> 20.7 us, 237 -> 260), four stages (240 -> 245), a
// store wait and an exit barrier without release (18.5 -> 18.2; but then arrivals at a CTA that has left are excluded
// by timing only); halves of 128 columns for a last wave that leaves pairs idle (issue takes as long for a half: 880 x
// 1536 x 8960 26.6 -> 27.4); the next wait tried before a block's MMAs (30.1 -> 31.0).
#include "fw_gemm_block.cuh"

namespace fw {

namespace {
namespace wide {
constexpr int BM = 256, BN = 256, HALF = 128;
constexpr int OP_BYTES = HALF * b8::BLK;          // 128 rows x 128 codes
constexpr int STAGE = 2 * OP_BYTES, STAGES = 5;   // 32 KB per CTA
constexpr int SF_RING = 4, SF_BYTES = 12 * 128;   // words of 128 rows of A and 256 of B, a group of 512 of K
constexpr int EPI_WARPS = 8, BOX = 4096, BIAS = 512;
constexpr int BOX_OFF = STAGES * STAGE;
constexpr int BIAS_OFF = BOX_OFF + EPI_WARPS * BOX;
constexpr int SF_OFF = BIAS_OFF + EPI_WARPS * BIAS;
constexpr int BAR_OFF = SF_OFF + SF_RING * SF_BYTES;
constexpr int SMEM = BAR_OFF + 256;
constexpr int THREADS = 384, EPI0 = 4;        // first epilogue warp
constexpr uint32_t SHIFT = 224;              // first column of the odd tiles' accumulator
constexpr uint32_t SF_COL = 480, SF_STRIDE = 16;
static_assert(SMEM <= 232448, "shared memory of a CTA");
}  // namespace wide

// Arrive on an mbarrier of either CTA, given by its shared::cluster address, after reads of Tensor Memory: the
// reads are complete (tcgen05.wait::ld) and ordered before what the waiting thread issues by the tcgen05 fences on
// both sides (before_thread_sync here, after_thread_sync behind its wait); an arrival between them need not
// order anything else, and one that does (release) waits for all that the thread has in flight, 0.6-1 us at
// every tile change.
__device__ __forceinline__ void mbar_arrive_tmem_read(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}

// Rows of C leave through a warp's 4 KB box: 32 rows of 128 bytes, 128-byte swizzle, one TMA store
// (the tensor map clips rows and columns that do not exist).
__device__ __forceinline__ void box_put(uint8_t* box, int row, int chunk, uint4 v) {
  *reinterpret_cast<uint4*>(box + row * 128 + ((chunk ^ (row & 7)) << 4)) = v;
}
__device__ __forceinline__ void box_free(int lane) {   // the last store has read the box
  if (lane == 0) bulk_wait_read0();
  __syncwarp();
}
__device__ __forceinline__ void box_store(const CUtensorMap* m, const uint8_t* box, int x, int y, int lane) {
  fence_proxy_async_smem();
  __syncwarp();
  if (lane == 0) {
    tma_store_2d(m, box, x, y);
    bulk_commit();
  }
}

// 32 accumulator columns of one row: bias (fp32, this warp's shared memory) and activation.
template <int ACT>
__device__ __forceinline__ void finish(float2 (&v)[16], const uint32_t (&r)[32], const float* bias) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float4 b = *reinterpret_cast<const float4*>(bias + 4 * i);
    const float2 x = make_float2(__uint_as_float(r[4 * i]), __uint_as_float(r[4 * i + 1]));
    const float2 y = make_float2(__uint_as_float(r[4 * i + 2]), __uint_as_float(r[4 * i + 3]));
    v[2 * i] = activate2<ACT>(__fadd2_rn(x, make_float2(b.x, b.y)));
    v[2 * i + 1] = activate2<ACT>(__fadd2_rn(y, make_float2(b.z, b.w)));
  }
}

template <int OUT, int ACT, bool TMA_OUT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(wide::THREADS, 1)
    gemm_block_wide_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                           const __grid_constant__ CUtensorMap tmO, const BlockGemmArgs a) {
  using namespace wide;
  pdl_trigger();
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + BAR_OFF);
  uint64_t* empty = full + STAGES;
  uint64_t* sf_full = empty + STAGES;    // [SF_RING] a group's exponents are in shared memory: the odd CTA's in
                                         // its own; the even CTA's: in both
  uint64_t* sf_free = sf_full + SF_RING; // [SF_RING] ... are copied to Tensor Memory
  uint64_t* tfull = sf_free + SF_RING;   // [2] accumulator of an even / odd tile complete
  uint64_t* tfree = tfull + 2;           // [1] the shared columns of the last tile are read, even CTA's
  uint64_t* sf_used = tfree + 1;         // [2] MMAs have read a buffer of scales in Tensor Memory, even CTA's
  uint64_t* drain = sf_used + 2;         // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int pair = blockIdx.x >> 1, npairs = gridDim.x >> 1;
  const int num_m = (a.M + BM - 1) / BM, num_n = (a.N + BN - 1) / BN, num_tiles = num_m * num_n;
  const int num_kb = a.K / b8::BLK, num_g = (num_kb + b8::GRP - 1) / b8::GRP;
  const uint32_t groups = pair < num_tiles ? (uint32_t)((num_tiles - 1 - pair) / npairs + 1) * (uint32_t)num_g : 0;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full + s, 1);
      mbar_init(empty + s, 1);
    }
    for (int b = 0; b < SF_RING; ++b) {
      mbar_init(sf_free + b, 1);
      mbar_init(sf_full + b, rank == 0 ? 2 : 1);   // one arrival per warp: those of all lanes queue up on the barrier
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(tfull + b, 1);
      mbar_init(sf_used + b, 1);
      mbar_init(drain + b, 1);
    }
    mbar_init(tfree, 2 * EPI_WARPS);
    *abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch(&tmA);
    tma_prefetch(&tmB);
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, 512);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  cluster_sync();   // both CTAs' barriers initialised and the pair's Tensor Memory allocated
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();

  if (warp == 0) {
    if (lane == 0) {
      const uint32_t full0 = mapa_cluster(full, 0);
      uint32_t cnt = 0;   // stages filled so far
      bool ok = true;
      for (int t = pair; t < num_tiles && ok; t += npairs) {
        const int m = (t % num_m) * BM + (int)rank * HALF, n = (t / num_m) * BN + (int)rank * HALF;
        for (int kb = 0; kb < num_kb; ++kb, ++cnt) {
          const uint32_t stage = cnt % STAGES;
          ok = wait_on<true>(empty + stage, ((cnt / STAGES) & 1u) ^ 1u, abort_flag, a.status, DEV_TIMEOUT_PRODUCER);
          if (!ok) break;
          if (rank == 0) mbar_arrive_expect_tx(full + stage, 2 * STAGE);
          uint8_t* dst = smem + stage * STAGE;
          tma_load_2d_pair(dst, &tmA, full0 + 8u * stage, kb * b8::BLK, m);
          tma_load_2d_pair(dst + OP_BYTES, &tmB, full0 + 8u * stage, kb * b8::BLK, n);
        }
      }
      // the MMAs consumed every stage this thread filled: no copy into this CTA is in flight at exit
      volatile int no_abort = 0;
      for (uint32_t c = cnt < STAGES ? 0 : cnt - STAGES; c < cnt; ++c)
        mbar_wait(empty + c % STAGES, (c / STAGES) & 1u, &no_abort, a.status, DEV_TIMEOUT_DRAIN);
    }
  } else if (warp == 1) {
    if (rank == 0) {
      const uint32_t one = lane == 0;
      // This loop issues four MMAs per k-block and must keep ahead of them: as little as possible is
      // computed in it.
      constexpr uint32_t SCALE_BYTE = (1u << 4) | (1u << 29);   // next byte of both operands' scale words
      const uint32_t desc0 = desc_lo(smem_u32(smem));
      uint32_t stage = 0, phase = 0, desc = desc0, slot = 0, slot_phase = 0, buf = 0, it = 0;
      bool ok = true;
      for (int t = pair; t < num_tiles && ok; t += npairs, ++it) {
        const uint32_t d = tmem + (it & 1u) * SHIFT;
        uint32_t accumulate = 0;
        for (int left = num_kb; left > 0;) {
          ok = wait_on(sf_free + slot, slot_phase, abort_flag, a.status, DEV_TIMEOUT_MMA);   // copied
          const uint32_t sf = tmem + SF_COL + buf * SF_STRIDE;
          uint32_t id = idesc_mx8(BM, BN);
          // a tile's first MMA: tile it - 1's shared columns have been read, and all of tile it - 2
          if (ok && !accumulate && it > 0)
            ok = wait_on<true>(tfree, (it - 1) & 1u, abort_flag, a.status, DEV_TIMEOUT_MMA);
          if (!ok) break;
          const int n = min(left, b8::GRP);
          for (int k = 0; k < n; ++k) {
            ok = wait_on<true>(full + stage, phase, abort_flag, a.status, DEV_TIMEOUT_MMA);
            if (!ok) break;
            tc_fence_after();
            umma_mx8_block<2>(one, d, desc, desc + (OP_BYTES >> 4), id, sf, sf + 4, accumulate);
            umma_commit_if<2>(one, empty + stage);
            accumulate = 1;
            id += SCALE_BYTE;
            desc += STAGE >> 4;
            if (++stage == STAGES) {
              stage = 0;
              phase ^= 1u;
              desc = desc0;
            }
          }
          if (!ok) break;
          umma_commit_local_if(one, sf_used + buf);
          left -= n;
          buf ^= 1u;
          if (++slot == SF_RING) {
            slot = 0;
            slot_phase ^= 1u;
          }
        }
        if (!ok) break;
        umma_commit_if<2>(one, tfull + (it & 1u));
      }
      if (one) umma_commit_pair(smem_u32(drain));   // this CTA's only: nothing arrives at a CTA that has left
      volatile int no_abort = 0;
      mbar_wait(drain, 0, &no_abort, a.status, DEV_TIMEOUT_DRAIN);
    }
  } else if (warp == 3) {
    if (rank == 0) {
      // not by the MMA issuer: the three copies cost it 0.2 us per group (4680 x 7680 x 5120 134 us, 130 this way)
      const uint32_t one = lane == 0;
      const uint32_t sf_smem = smem_u32(smem + SF_OFF);
      for (uint32_t grp = 0; grp < groups; ++grp) {
        const uint32_t slot = grp % SF_RING, buf = grp & 1u;
        if (!wait_on<true>(sf_full + slot, (grp / SF_RING) & 1u, abort_flag, a.status, DEV_TIMEOUT_MMA)) break;
        if (!wait_on(sf_used + buf, ((grp >> 1) & 1u) ^ 1u, abort_flag, a.status, DEV_TIMEOUT_MMA)) break;
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < 3; ++c)
          tmem_copy_pair_if(one, tmem + SF_COL + buf * SF_STRIDE + 4 * c, sf_smem + slot * SF_BYTES + 512 * c);
        umma_commit_if<2>(one, sf_free + slot);
      }
      if (one) umma_commit_pair(smem_u32(drain + 1));
      volatile int no_abort = 0;
      mbar_wait(drain + 1, 0, &no_abort, a.status, DEV_TIMEOUT_DRAIN);
    } else if (lane == 0) {
      // This CTA's groups announced to the even CTA's copier.  The release at cluster scope that its scales need
      // waits for all that the thread has in flight: by warp 2 itself, with the next group's loads, 1536 x 8960 took
      // 33.4 us instead of 31.6 (two such warps, a group each in turn: no difference).
      const uint32_t sf_full0 = mapa_cluster(sf_full, 0);
      for (uint32_t grp = 0; grp < groups; ++grp) {
        const uint32_t slot = grp % SF_RING;
        if (!wait_on(sf_full + slot, (grp / SF_RING) & 1u, abort_flag, a.status, DEV_TIMEOUT_MMA)) break;
        mbar_arrive_cluster(sf_full0 + 8u * slot);
      }
    }
  } else if (warp == 2) {
    // A group is fetched before the last one is stored: the loads queue behind the tiles' traffic (fetched two
    // groups ahead, 2640 x 4608 x 1536 takes 18.9 us instead of 18.6).
    uint32_t w[12], next[12];
    int lt = pair, lg = 0;   // next group to fetch
    auto fetch = [&](uint32_t(&v)[12]) {
      if (lt < num_tiles) {
        const int m0 = (lt % num_m) * BM + (int)rank * HALF + lane, n0 = (lt / num_m) * BN + lane;
        const uint32_t* pa = a.sa + (size_t)lg * a.M;
        const uint32_t* pb = a.sb + (size_t)lg * a.N;
#pragma unroll
        for (int c = 0; c < 4; ++c) v[c] = m0 + c * 32 < a.M ? __ldg(pa + m0 + c * 32) : b8::ONES;
#pragma unroll
        for (int c = 0; c < 8; ++c) v[4 + c] = n0 + c * 32 < a.N ? __ldg(pb + n0 + c * 32) : b8::ONES;
        if (++lg == num_g) {
          lg = 0;
          lt += npairs;
        }
      }
    };
    fetch(w);
    bool ok = true;
    for (uint32_t grp = 0; grp < groups; ++grp) {
      fetch(next);
      const uint32_t slot = grp % SF_RING;
      ok = __all_sync(0xffffffffu, wait_on<true>(sf_free + slot, ((grp / SF_RING) & 1u) ^ 1u, abort_flag, a.status,
                                                 DEV_TIMEOUT_PRODUCER));
      if (!ok) break;
      uint4* dst = reinterpret_cast<uint4*>(smem + SF_OFF + slot * SF_BYTES);
#pragma unroll
      for (int c = 0; c < 3; ++c) dst[32 * c + lane] = make_uint4(w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(sf_full + slot);
#pragma unroll
      for (int c = 0; c < 12; ++c) w[c] = next[c];
    }
    // the last copies' arrivals from the even CTA have come: none is under way to this CTA at exit
    for (uint32_t grp = groups < SF_RING ? 0 : groups - SF_RING; grp < groups && ok; ++grp)
      ok = wait_on<true>(sf_free + grp % SF_RING, (grp / SF_RING) & 1u, abort_flag, a.status, DEV_TIMEOUT_PRODUCER);
  } else if (warp >= EPI0) {
    const int q = warp & 3, h = (warp - EPI0) >> 2;
    const uint32_t tfree0 = mapa_cluster(tfree, 0);
    uint8_t* box = smem + BOX_OFF + (warp - EPI0) * BOX;
    float* bias = reinterpret_cast<float*>(smem + BIAS_OFF + (warp - EPI0) * BIAS);
    uint32_t it = 0;
    for (int t = pair; t < num_tiles; t += npairs, ++it) {
      const int row0 = (t % num_m) * BM + (int)rank * HALF + q * 32, row = row0 + lane;
      const int col0 = (t / num_m) * BN + h * 128;
      __syncwarp();
      {
        float4 u = make_float4(0.f, 0.f, 0.f, 0.f);
        const int c = col0 + lane * 4;
        if (a.bias) {
          if (c + 0 < a.N) u.x = __bfloat162float(a.bias[c]);
          if (c + 1 < a.N) u.y = __bfloat162float(a.bias[c + 1]);
          if (c + 2 < a.N) u.z = __bfloat162float(a.bias[c + 2]);
          if (c + 3 < a.N) u.w = __bfloat162float(a.bias[c + 3]);
        }
        *reinterpret_cast<float4*>(bias + lane * 4) = u;
      }
      __syncwarp();
      bool ok = __all_sync(0xffffffffu, wait_on<true>(tfull + (it & 1u), (it >> 1) & 1u, abort_flag, a.status,
                                                      DEV_TIMEOUT_EPILOGUE));
      if (!ok) break;
      tc_fence_after();
      const uint32_t acc = tmem + ((uint32_t)(q * 32) << 16) + (it & 1u) * SHIFT + (uint32_t)(h * 128);
      // chunks of 32 columns, the one shared with the next tile first
      const int first = (it & 1u) ? 0 : 3, dir = (it & 1u) ? 1 : -1;
      if constexpr (OUT == FW_U8) {
        // 128 columns are one block.  First pass: activate, find the maximum, write back to Tensor Memory (the
        // shared columns stay in registers: the next tile starts over them); second pass: encode.
        uint32_t keep[32], r[32];
        float top = 0.f;
        auto scan = [&](uint32_t(&x)[32], int c) {
          float2 v[16];
          finish<ACT>(v, x, bias + c);
          if (col0 + c + 32 > a.N) {   // columns that do not exist
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              if (col0 + c + 2 * k >= a.N) v[k].x = 0.f;
              if (col0 + c + 2 * k + 1 >= a.N) v[k].y = 0.f;
            }
          }
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            top = fmaxf(top, fmaxf(fabsf(v[k].x), fabsf(v[k].y)));   // passes over NaN
            x[2 * k] = __float_as_uint(v[k].x);
            x[2 * k + 1] = __float_as_uint(v[k].y);
          }
        };
        tmem_ld32(acc + (uint32_t)(first * 32), keep);
        tmem_ld_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_tmem_read(tfree0);
        scan(keep, first * 32);
#pragma unroll 1
        for (int j = 1; j < 4; ++j) {
          const int c = (first + dir * j) * 32;
          tmem_ld32(acc + (uint32_t)c, r);
          tmem_ld_wait();
          scan(r, c);
          tmem_st32(acc + (uint32_t)c, r);
        }
        tmem_st_wait();
        // an infinity in some row of the warp (its loads are collective): the finite values scale the row
        const bool finite = __all_sync(0xffffffffu, top < INFINITY);
        uint32_t m = __float_as_uint(top);
        if (!finite) {
          m = 0;
#pragma unroll
          for (int k = 0; k < 32; ++k) m = max(m, b8::abs_bits(__uint_as_float(keep[k])));
#pragma unroll 1
          for (int j = 1; j < 4; ++j) {
            tmem_ld32(acc + (uint32_t)((first + dir * j) * 32), r);
            tmem_ld_wait();
#pragma unroll
            for (int k = 0; k < 32; ++k) m = max(m, b8::abs_bits(__uint_as_float(r[k])));
          }
        }
        const uint32_t eb = b8::block_exp(m);
        const float inv = b8::inv_scale(eb);
        auto put = [&](const uint32_t(&x)[32], int c) {
#pragma unroll
          for (int h16 = 0; h16 < 2; ++h16) {
            uint32_t w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const uint32_t* y = x + 16 * h16 + 4 * k;
              const float e0 = __uint_as_float(y[0]), e1 = __uint_as_float(y[1]);
              const float e2 = __uint_as_float(y[2]), e3 = __uint_as_float(y[3]);
              w[k] = finite ? b8::encode4_finite(e0, e1, e2, e3, inv) : b8::encode4(e0, e1, e2, e3, inv);
            }
            box_put(box, lane, 2 * c + h16, make_uint4(w[0], w[1], w[2], w[3]));
          }
        };
        box_free(lane);
        put(keep, first);
#pragma unroll 1
        for (int j = 1; j < 4; ++j) {
          const int c = first + dir * j;
          tmem_ld32(acc + (uint32_t)(c * 32), r);
          tmem_ld_wait();
          put(r, c);
        }
        tc_fence_before();
        if (col0 < a.N) {
          box_store(&tmO, box, col0, row0, lane);
          if (row < a.M) {
            const int blk = col0 / b8::BLK;
            uint8_t* s = a.out_s + ((size_t)(blk / b8::GRP) * a.M + row) * b8::GRP;
            s[blk % b8::GRP] = (uint8_t)eb;
            if (blk == b8::blocks(a.N) - 1)   // places behind the last block
              for (int j = blk % b8::GRP + 1; j < b8::GRP; ++j) s[j] = 127;
          }
        }
      } else {
        uint32_t r[32], next[32];
        tmem_ld32(acc + (uint32_t)(first * 32), r);
        tmem_ld_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_tmem_read(tfree0);
#pragma unroll 1
        for (int j = 0; j < 4; ++j) {
          const int c = first + dir * j;
          if (j < 3) tmem_ld32(acc + (uint32_t)((c + dir) * 32), next);
          float2 v[16];
          finish<ACT>(v, r, bias + c * 32);
          if constexpr (!TMA_OUT) {
            // rows that no TMA store can address (stride not a multiple of 16 bytes): across the box,
            // then 32 columns of a row per warp store
            float* f = reinterpret_cast<float*>(box);
            __syncwarp();
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              f[lane * 32 + ((2 * k) ^ lane)] = v[k].x;
              f[lane * 32 + ((2 * k + 1) ^ lane)] = v[k].y;
            }
            __syncwarp();
            const int col = col0 + c * 32 + lane;
            if (col < a.N)
#pragma unroll 4
              for (int k = 0; k < 32 && row0 + k < a.M; ++k) {
                const float x = f[k * 32 + (lane ^ k)];
                const size_t at = (size_t)(row0 + k) * a.N + col;
                if (OUT == FW_F32)
                  static_cast<float*>(a.out)[at] = x;
                else
                  static_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16_rn(x);
              }
          } else if constexpr (OUT == FW_F32) {   // a box holds 32 columns
            box_free(lane);
#pragma unroll
            for (int k = 0; k < 8; ++k)
              box_put(box, lane, k, make_uint4(__float_as_uint(v[2 * k].x), __float_as_uint(v[2 * k].y),
                                               __float_as_uint(v[2 * k + 1].x), __float_as_uint(v[2 * k + 1].y)));
            if (col0 + c * 32 < a.N) box_store(&tmO, box, col0 + c * 32, row0, lane);
          } else {                                // ... 64 columns, two of these chunks
            if ((j & 1) == 0) box_free(lane);
#pragma unroll
            for (int k = 0; k < 4; ++k)
              box_put(box, lane, (c & 1) * 4 + k,
                      make_uint4(pack_bf16(v[4 * k].x, v[4 * k].y), pack_bf16(v[4 * k + 1].x, v[4 * k + 1].y),
                                 pack_bf16(v[4 * k + 2].x, v[4 * k + 2].y), pack_bf16(v[4 * k + 3].x, v[4 * k + 3].y)));
            const int col = col0 + (c >> 1) * 64;
            if ((j & 1) == 1 && col < a.N) box_store(&tmO, box, col, row0, lane);
          }
          tmem_ld_wait();
#pragma unroll
          for (int k = 0; k < 32; ++k) r[k] = next[k];
        }
        tc_fence_before();
      }
    }
    if (lane == 0) bulk_wait0();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();   // neither CTA releases the pair's Tensor Memory or exits while the other uses it
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc_pair(tmem, 512);
  }
}


}  // namespace

int gemm_block_wide_launch(const void* A8, const void* B8, const BlockGemmArgs& a, cudaStream_t s) {
  using namespace wide;
  CUtensorMap ta, tb, to;
  int rc = make_tmap_2d(&ta, A8, 1, a.M, a.K, a.K, HALF, b8::BLK, true);
  if (!rc) rc = make_tmap_2d(&tb, B8, 1, a.N, a.K, a.K, HALF, b8::BLK, true);
  const bool tma_out = a.out_dtype == FW_U8 || (a.out_dtype == FW_F32 ? a.N % 4 == 0 : a.N % 8 == 0);
  if (!rc && a.out_dtype == FW_U8) {
    rc = make_tmap_2d(&to, a.out, 1, a.M, b8::padded(a.N), b8::padded(a.N), 32, 128, true);
  } else if (!rc && tma_out) {
    const int eb = a.out_dtype == FW_F32 ? 4 : 2;
    rc = make_tmap_2d(&to, a.out, eb, a.M, a.N, a.N, 32, 128 / eb, true);
  }
  if (rc) return rc;
  if (!tma_out) to = ta;   // not read
  const long long tiles = (long long)((a.M + BM - 1) / BM) * ((a.N + BN - 1) / BN);
  if (tiles > (1 << 30)) return FW_ESHAPE;
  const int pairs = (int)(tiles < num_sms() / 2 ? tiles : num_sms() / 2);
  auto go = [&](auto kern) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM) != cudaSuccess) return FW_ECUDA;
    return launch_k(kern, dim3(2 * pairs), dim3(THREADS), SMEM, s, ta, tb, to, a) == cudaSuccess ? FW_OK : FW_ECUDA;
  };
  auto by_act = [&](auto out, auto tma) {
    constexpr int O = decltype(out)::value;
    constexpr bool T = decltype(tma)::value;
    switch (a.act) {
      case ACT_TANH: return go(gemm_block_wide_kernel<O, ACT_TANH, T>);
      case ACT_ERF: return go(gemm_block_wide_kernel<O, ACT_ERF, T>);
      default: return go(gemm_block_wide_kernel<O, ACT_NONE, T>);
    }
  };
  using Yes = std::integral_constant<bool, true>;
  using No = std::integral_constant<bool, false>;
  const std::integral_constant<int, FW_F32> f32;
  const std::integral_constant<int, FW_BF16> b16;
  if (a.out_dtype == FW_U8) return by_act(std::integral_constant<int, FW_U8>{}, Yes{});
  if (a.out_dtype == FW_F32) return tma_out ? by_act(f32, Yes{}) : by_act(f32, No{});
  return tma_out ? by_act(b16, Yes{}) : by_act(b16, No{});
}

}  // namespace fw
