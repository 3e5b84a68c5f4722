// Block-scaled product of two matrices in microscaled 4-bit floats: out[M][N] = x[M][K] w[N][K]^T, on tcgen05.
//
// 256 values of K are 128 bytes of a row, one swizzle atom: a K step of 256 moves and multiplies the same bytes as one of 64 values of bf16,
// four MMAs of 64 values each.  Its scales (1 KB per 128 rows) travel into the same stage and are copied to tensor memory by the thread that
// issues the MMAs, a row's scales in the lane of its number modulo 32.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/bshmem/mxfp4.h"
#include "../../include/bshmem/tcgen05.cuh"

namespace bshmem {
namespace mx {
using namespace sm100;

constexpr int BLOCK = 32;              // values per scale
constexpr int SCALE_BLOCK = 512;       // bytes: 128 rows x 4 scales

__host__ __device__ __forceinline__ int64_t k_blocks(int64_t K) { return (K + 255) / 256 * 2; }      // of 128 values, even
__host__ __device__ __forceinline__ int64_t row_blocks(int64_t R) { return (R + 127) / 128; }

// ------------------------------------------------------------------ CTA pairs
// Pairs of CTAs walk tiles of 256 rows of x by COLS rows of w (persistent).  Each CTA loads its own 128 rows of x and half the rows of w, the
// even one issues the MMAs for both, and each CTA's tensor memory gets its own 128 x COLS accumulator: 70 bytes
// a clock and SM at the full rate of the tensor cores, instead of a single CTA's 102.  Some 50 arrive (12 TB/s over all SMs), which is what
// bounds it: 8192 x 8192 x 3584 in 82 us (5.9 PFLOP/s), 8192^3 in 165 (6.7), tensor cores busy 0.72 of the time.  One CTA per 128 x 256 tile
// without overlapped epilogue took 131 us.
// Tensor memory (COLS = 256): two accumulators, which overlap by the 48 columns that two steps' scales take:
//   [0, 256) accumulator 0    [208, 464) accumulator 1    [464, 512) scales
// The epilogue drains the shared columns of a tile first; from then on the other accumulator may be written.
// The scales of a step replace those of two steps before; the MMAs that read them are known to be complete (their stage's barrier).
//   warp 0  TMA producer   warp 1  MMA issuer (even CTA)   warp 2  tensor memory   warps 4 to 7  epilogue
constexpr int P_THREADS = 256, P_EPI_WARP0 = 4, P_EPI_THREADS = 128, P_CHUNK = 64;
constexpr int P_STAGE_A = 128 * 128, P_OUT = 128 * P_CHUNK * 2;
template <int COLS>
struct PairTile {
  static constexpr int B_ROWS = COLS / 2, B_BYTES = B_ROWS * 128, S_BLOCKS = COLS / 128, S_BYTES = 1024 * (1 + S_BLOCKS);
  static constexpr int STAGE = P_STAGE_A + B_BYTES + S_BYTES, STAGES = COLS == 256 ? 5 : 7;
  static constexpr int S_COLS = 8 + 8 * S_BLOCKS, S_FIRST = 512 - 2 * S_COLS, ACC1 = COLS < S_FIRST - COLS ? COLS : S_FIRST - COLS;
  static constexpr int TILES = STAGES * STAGE + 2 * P_OUT, SMEM = TILES + 1024 /*alignment slack*/ + 256 /*barriers*/;
  static_assert(COLS - ACC1 <= P_CHUNK, "the first chunk that the epilogue drains holds all shared columns");
  static_assert(SMEM <= 227 * 1024, "shared memory");
};

struct alignas(64) PairParams {
  CUtensorMap tmA, tmB, tmSA, tmSB, tmOut;
  int* error_flag;
  uint64_t wait_limit_ns;
  int M, N, K;
  int tiles_m, tiles_n, tiles;
  __nv_bfloat16* direct;  // not null: rows of the output are no whole 16-byte units, and are stored value by value
};

// The shorter side of the tiles runs fastest, in bands of up to 32: the pairs that run at a time share rows of both operands.  Rows of x fastest
// and without bands: 16384 x 2048 x 7168 86 us (79 so), 32768 x 8192 x 2048 219 (194), 8192 x 4096 x 14336 151 (144), 16384 x 16384 x 4096 370
// (356); bands of 16 take 202 for the second and 87 instead of 85 for 8192 x 8192 x 3584.
constexpr int P_BAND = 32;
struct TilePlace {
  int m, n;
};
__device__ __forceinline__ TilePlace place_of(const PairParams& p, int t) {
  const bool rows_fast = p.tiles_m <= p.tiles_n;
  const int fast = rows_fast ? p.tiles_m : p.tiles_n, slow = rows_fast ? p.tiles_n : p.tiles_m, band = min(P_BAND, fast);
  const int first = t / (band * slow) * band, width = min(band, fast - first), at = t - first * slow;
  return rows_fast ? TilePlace{first + at % width, at / width} : TilePlace{at / width, first + at % width};
}

template <int COLS>
__global__ void __launch_bounds__(P_THREADS, 1) gemm_pair_kernel(const __grid_constant__ PairParams p) {
  using Tile = PairTile<COLS>;
  constexpr int STAGES = Tile::STAGES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t* sA = smem;
  uint8_t* sB = sA + STAGES * P_STAGE_A;
  uint8_t* sE = sB + STAGES * Tile::B_BYTES;     // two output chunks
  uint8_t* sS = sE + 2 * P_OUT;                  // per stage: 1 KB of A's scales, then B's
  uint64_t* full = (uint64_t*)(smem + Tile::TILES);
  uint64_t* empty = full + STAGES;
  uint64_t* acc_full = empty + STAGES;           // [2]
  uint64_t* acc_free = acc_full + 2;             // a tile's shared columns have been drained
  uint32_t* tmem_slot = (uint32_t*)(acc_free + 1);
  volatile int* abort_flag = (volatile int*)(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rank = (int)cluster_ctarank();
  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&full[i], 2);   // one arrival, with its byte count, from each CTA's producer
      mbar_init(&empty[i], 1);
    }
    mbar_init(&acc_full[0], 1);
    mbar_init(&acc_full[1], 1);
    mbar_init(acc_free, 2 * P_EPI_THREADS / 32);
    mbar_fence_init();
    fence_proxy_async_smem();
  }
  if (warp == 2) {
    tmem_alloc<2>(tmem_slot, 512);
    tmem_relinquish<2>();
  }
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_all();  // the other CTA's barriers are initialised before anything arrives on them
  tc_fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  asm volatile("griddepcontrol.wait;" ::: "memory");  // the launch may overlap the end of the kernel before it
  const int steps = (p.K + 255) / 256, first = (int)blockIdx.x >> 1, walkers = (int)gridDim.x >> 1;

  if (warp == 0) {
    if (elect_one()) {
      tma_prefetch_desc(&p.tmA);
      tma_prefetch_desc(&p.tmB);
      int stage = 0;
      uint32_t phase = 0;
      for (int t = first; t < p.tiles && !*abort_flag; t += walkers) {
        const TilePlace at = place_of(p, t);
        const int tm = at.m, tn = at.n;
        for (int k = 0; k < steps; ++k) {
          if (!mbar_wait(&empty[stage], phase ^ 1, p.wait_limit_ns, abort_flag)) break;
          const uint32_t lead = mapa_u32(smem_u32(&full[stage]), 0);
          mbar_expect_tx_cluster(lead, Tile::STAGE);
          tma_load_2d_pair(sA + stage * P_STAGE_A, &p.tmA, lead, k * 64, tm * 256 + rank * 128);
          tma_load_2d_pair(sB + stage * Tile::B_BYTES, &p.tmB, lead, k * 64, tn * COLS + rank * Tile::B_ROWS);
          tma_load_2d_pair(sS + stage * Tile::S_BYTES, &p.tmSA, lead, k * 256, tm * 2 + rank);
          tma_load_2d_pair(sS + stage * Tile::S_BYTES + 1024, &p.tmSB, lead, k * 256, tn * Tile::S_BLOCKS);
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
      }
      // The last fills' stages are still handed back by the even CTA: this CTA stays until they are.
      for (int i = 0; i < STAGES && !*abort_flag; ++i) {
        if (!mbar_wait(&empty[stage], phase ^ 1, p.wait_limit_ns, abort_flag)) break;
        if (++stage == STAGES) { stage = 0; phase ^= 1; }
      }
    }
  } else if (warp == 1) {
    if (rank == 0 && elect_one()) {
      constexpr uint32_t idesc[2] = {umma_idesc_mxf4(256, COLS, 0), umma_idesc_mxf4(256, COLS, 2)};
      int stage = 0, acc = 0, n = 0;
      uint32_t phase = 0, step = 0;
      for (int t = first; t < p.tiles && !*abort_flag; t += walkers, ++n) {
        if (n && !mbar_wait(acc_free, (n - 1) & 1, p.wait_limit_ns, abort_flag)) break;
        tc_fence_after_sync();
        const uint32_t d = tmem + (acc ? Tile::ACC1 : 0);
        bool ok = true;
        for (int k = 0; k < steps; ++k, ++step) {
          if (step >= 2) {  // the MMAs of two steps before are complete: their scales may be replaced
            const uint32_t s2 = step - 2;
            if (!mbar_wait(&empty[s2 % STAGES], s2 / STAGES & 1, p.wait_limit_ns, abort_flag)) { ok = false; break; }
          }
          if (!mbar_wait(&full[stage], phase, p.wait_limit_ns, abort_flag)) { ok = false; break; }
          tc_fence_after_sync();
          const uint32_t sf = tmem + Tile::S_FIRST + (step & 1) * Tile::S_COLS;  // A: 4 columns per 128 values of K; B: 4 per 128 values and 128 rows
          const uint32_t s = smem_u32(sS + stage * Tile::S_BYTES);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            umma_copy_scales_pair(sf + h * 4, umma_desc_scales(s + h * SCALE_BLOCK));
#pragma unroll
            for (int b = 0; b < Tile::S_BLOCKS; ++b)
              umma_copy_scales_pair(sf + 8 + (h * Tile::S_BLOCKS + b) * 4, umma_desc_scales(s + 1024 + b * 1024 + h * SCALE_BLOCK));
          }
          const uint64_t da = umma_desc_k_sw128(smem_u32(sA + stage * P_STAGE_A)), db = umma_desc_k_sw128(smem_u32(sB + stage * Tile::B_BYTES));
#pragma unroll
          for (int i = 0; i < 4; ++i)  // 64 values of K are 32 bytes
            umma_mxf4_pair(d, da + i * 2, db + i * 2, idesc[i & 1], sf + (i >> 1) * 4, sf + 8 + (i >> 1) * Tile::S_BLOCKS * 4, (k | i) != 0);
          umma_commit_pair(&empty[stage]);
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
        if (!ok) break;
        umma_commit_pair(&acc_full[acc]);
        acc ^= 1;
      }
    }
  } else if (warp >= P_EPI_WARP0) {
    const int ew = warp - P_EPI_WARP0, row = ew * 32 + lane;
    const bool issuer = threadIdx.x == P_EPI_WARP0 * 32;
    int acc = 0, buf = 0;
    uint32_t phase[2] = {0, 0};
    for (int t = first; t < p.tiles; t += walkers) {
      const TilePlace at = place_of(p, t);
      const int row0 = at.m * 256 + rank * 128, col0 = at.n * COLS;
      const uint32_t ok = mbar_wait(&acc_full[acc], phase[acc], p.wait_limit_ns, abort_flag) ? 1u : 0u;
      phase[acc] ^= 1;
      if (!named_bar_and(1, P_EPI_THREADS, ok)) break;  // either all epilogue threads go on or all leave
      tc_fence_after_sync();
      const uint32_t src = tmem + ((uint32_t)(ew * 32) << 16) + (uint32_t)(acc ? Tile::ACC1 : 0);
#pragma unroll 1
      for (int i = 0; i < COLS / P_CHUNK; ++i) {
        const int c = (acc ? i : (i + COLS / P_CHUNK - 1) % (COLS / P_CHUNK)) * P_CHUNK;  // shared columns first
        float f[P_CHUNK];
        tmem_ld_32x32(src + c, (uint32_t*)f);
        tmem_ld_32x32(src + c + 32, (uint32_t*)f + 32);
        tmem_ld_wait();
        if (i == 0) {
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(mapa_u32(smem_u32(acc_free), 0));
        }
        if (issuer) bulk_wait_read<1>();  // the store that read this buffer last
        named_bar_sync(1, P_EPI_THREADS);
        uint8_t* dst = sE + buf * P_OUT + row * 128;
#pragma unroll
        for (int j = 0; j < P_CHUNK / 8; ++j) {
          uint4 v;
          __nv_bfloat162* h = (__nv_bfloat162*)&v;
#pragma unroll
          for (int e = 0; e < 4; ++e) h[e] = __floats2bfloat162_rn(f[j * 8 + 2 * e], f[j * 8 + 2 * e + 1]);
          *(uint4*)(dst + ((j ^ (row & 7)) << 4)) = v;
        }
        if (!p.direct) fence_proxy_async_smem();
        named_bar_sync(1, P_EPI_THREADS);
        if (p.direct) {
          const uint8_t* rows = sE + buf * P_OUT;
          for (int r = ew * 32; r < ew * 32 + 32 && row0 + r < p.M; ++r) {   // a warp takes a row: two values a lane
            const int at = col0 + c + lane * 2;
            const __nv_bfloat162 v = *(const __nv_bfloat162*)(rows + r * 128 + ((lane >> 2 ^ (r & 7)) << 4) + (lane & 3) * 4);
            __nv_bfloat16* to = p.direct + (int64_t)(row0 + r) * p.N + at;
            if (at < p.N) to[0] = v.x;
            if (at + 1 < p.N) to[1] = v.y;
          }
        } else if (issuer) {
          if (row0 < p.M && col0 + c < p.N) tma_store_2d(&p.tmOut, sE + buf * P_OUT, col0 + c, row0);  // clipped to the matrix
          bulk_commit();
        }
        buf ^= 1;
      }
      acc ^= 1;
    }
    if (issuer) bulk_wait<0>();
  }
  if (*abort_flag) {  // copies still in flight land before the shared memory goes away
    const uint64_t t0 = timer_ns();
    while (timer_ns() - t0 < 200000) __nanosleep(1000);
  }
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_all();  // neither CTA frees tensor memory that the other's MMAs write
  if (warp == 2) tmem_dealloc<2>(tmem, 512);
  if (threadIdx.x == 0 && *abort_flag) atomicOr(p.error_flag, 1);
}

// ------------------------------------------------------------------ few rows of x
// One tile of 128 rows of w by COLS rows of x per CTA, in steps of 256 values of K: the weights are the tensor core's first operand.  Here
// reading the weights is what takes the time beside a fixed part, so as many SMs as possible have to read, and a cluster of CTAs
// divides K.  Each sends its sums to the shared memory of the CTA that owns the row of x (its number modulo the cluster's size), which
// adds them in order.  (Owners that fetch the sums instead wait for a round trip per value: 64 x 1024 x 8192 took 19 us that way, 7.5 now.)
// 16 x 8192 x 8192: 11.7 us with cold weights, 8.9 to 9.2 with warm ones, of which 5.3 are what the smallest product takes (launch, tensor memory, the
// first loads, the exchange, the stores): the other 6.4 read 36 MB at 5.6 TB/s, from L2 3.7 at 9.7.
//   warp 0  TMA producer   warp 1  MMA issuer   warp 2  tensor memory   then all eight warps store
constexpr int F_THREADS = 256, F_STAGE_W = 128 * 128;
template <int COLS>
struct FewTile {
  static constexpr int X_BYTES = COLS * 128, STAGE = F_STAGE_W + X_BYTES + 2048, OUT = 128 * COLS * 4;  // OUT: the finished tile, [split][COLS / split][128]
  static constexpr int FIT = (225 * 1024 - OUT) / STAGE, STAGES = FIT < 8 ? FIT : 8;
  static constexpr int RING = STAGES * STAGE, SMEM = RING + OUT + 1024 /*alignment slack*/ + 256 /*barriers*/;
  static_assert(SMEM <= 227 * 1024, "shared memory");
};

struct alignas(64) FewParams {
  CUtensorMap tmW, tmX, tmSW, tmSX;
  __nv_bfloat16* out;
  int* error_flag;
  uint64_t wait_limit_ns;
  int64_t M, N;
  int K, tiles_w;
  int split;                // CTAs that divide K (a cluster)
  int early;                // the weights are complete before the kernel ahead of this one on the stream began
};

template <int COLS>
__global__ void __launch_bounds__(F_THREADS, 1) gemm_few_kernel(const __grid_constant__ FewParams p) {
  using Tile = FewTile<COLS>;
  constexpr int STAGES = Tile::STAGES, S_COLS = 16;   // S_COLS: columns of tensor memory for a stage's scales
  constexpr int TMEM = 256;
  static_assert(COLS + STAGES * S_COLS <= TMEM, "tensor memory");
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t* sW = smem;
  uint8_t* sX = smem + STAGES * F_STAGE_W;
  uint8_t* sS = sX + STAGES * Tile::X_BYTES;         // per stage: 1 KB of the weights' scales, 1 KB of x's
  float* sums = (float*)(smem + Tile::RING);
  uint64_t* full = (uint64_t*)(smem + Tile::RING + Tile::OUT);
  uint64_t* empty = full + STAGES;
  uint64_t* acc_full = empty + STAGES;
  uint32_t* tmem_slot = (uint32_t*)(acc_full + 1);
  volatile int* abort_flag = (volatile int*)(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = p.split, rank = split > 1 ? (int)cluster_ctarank() : 0;
  const int tile_number = (int)blockIdx.x / split;
  const int64_t row_w = (int64_t)(tile_number % p.tiles_w) * 128, row_x = (int64_t)(tile_number / p.tiles_w) * COLS;
  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    mbar_init(acc_full, 1);
    mbar_fence_init();
    fence_proxy_async_smem();
  }
  if (warp == 2) {
    tmem_alloc(tmem_slot, TMEM);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  if (split > 1) cluster_arrive();
  const uint32_t tmem = *tmem_slot;
  const int all_steps = (p.K + 255) / 256, k0 = (int)((int64_t)all_steps * rank / split), k1 = (int)((int64_t)all_steps * (rank + 1) / split);
  // The launch may overlap the end of the kernel before it.  Where that kernel made x only, the first stages of the weights are
  // fetched before waiting for it.
  if (!p.early) asm volatile("griddepcontrol.wait;" ::: "memory");

  if (warp == 0) {
    if (elect_one()) {
      tma_prefetch_desc(&p.tmW);
      tma_prefetch_desc(&p.tmX);
      tma_prefetch_desc(&p.tmSW);
      tma_prefetch_desc(&p.tmSX);
      int stage = 0;
      uint32_t phase = 0;
      auto load_w = [&](int k, int to) {
        mbar_expect_tx(&full[to], Tile::STAGE);
        tma_load_2d(sW + to * F_STAGE_W, &p.tmW, &full[to], k * 64, (int)row_w);
        tma_load_2d(sS + to * 2048, &p.tmSW, &full[to], k * 256, (int)(row_w / 128));
      };
      const int ahead = p.early ? (k1 - k0 < STAGES ? k1 - k0 : STAGES) : 0;
      for (int k = 0; k < ahead; ++k) load_w(k0 + k, k);
      if (p.early) asm volatile("griddepcontrol.wait;" ::: "memory");
      for (int k = k0; k < k1; ++k) {
        if (!mbar_wait(&empty[stage], phase ^ 1, p.wait_limit_ns, abort_flag)) break;
        if (k - k0 >= ahead) load_w(k, stage);
        tma_load_2d(sX + stage * Tile::X_BYTES, &p.tmX, &full[stage], k * 64, (int)row_x);
        tma_load_2d(sS + stage * 2048 + 1024, &p.tmSX, &full[stage], k * 256, (int)(row_x / 128));
        if (++stage == STAGES) { stage = 0; phase ^= 1; }
      }
    }
  } else if (warp == 1) {
    if (elect_one()) {
      constexpr uint32_t idesc[2] = {umma_idesc_mxf4(128, COLS, 0), umma_idesc_mxf4(128, COLS, 2)};
      const uint32_t sfx_first = (uint32_t)(row_x % 128 / 32);  // a tile of 64 rows may start in the middle of a row block
      int stage = 0;
      uint32_t phase = 0;
      for (int k = k0; k < k1; ++k) {
        if (!mbar_wait(&full[stage], phase, p.wait_limit_ns, abort_flag)) break;
        tc_fence_after_sync();
        // Four columns per 128 values of K for each operand.  Written again only after the stage's MMAs are done.
        const uint32_t sf = tmem + COLS + stage * S_COLS;
        const uint32_t s = smem_u32(sS + stage * 2048);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          umma_copy_scales(sf + h * 4, umma_desc_scales(s + h * SCALE_BLOCK));
          umma_copy_scales(sf + 8 + h * 4, umma_desc_scales(s + 1024 + h * SCALE_BLOCK));
        }
        const uint64_t da = umma_desc_k_sw128(smem_u32(sW + stage * F_STAGE_W)), db = umma_desc_k_sw128(smem_u32(sX + stage * Tile::X_BYTES));
#pragma unroll
        for (int i = 0; i < 4; ++i)  // 64 values of K are 32 bytes
          umma_mxf4(tmem, da + i * 2, db + i * 2, idesc[i & 1], sf + (i >> 1) * 4, sf + 8 + (i >> 1) * 4 + sfx_first, k > k0 || i > 0);
        umma_commit(&empty[stage]);
        if (++stage == STAGES) { stage = 0; phase ^= 1; }
      }
      umma_commit(acc_full);
    }
  }
  __syncwarp();
  // Every MMA of this CTA is complete, so every load has been consumed and the ring is free for the finished tile.
  const bool ok = mbar_wait(acc_full, 0, p.wait_limit_ns, abort_flag) && !*abort_flag;
  if (!ok) {
    const uint64_t t0 = timer_ns();  // copies still in flight land before the shared memory is reused or goes away
    while (timer_ns() - t0 < 200000) __nanosleep(1000);
  }
  tc_fence_after_sync();
  const int quarter = (warp & 3) * 32;
  constexpr int HALF = COLS / 2 < 32 ? 32 : COLS / 2;
  const int c0 = (warp >> 2) * HALF;   // this warp's rows are quarter + lane, its columns [c0, c0 + HALF)
  // row r of the tile is output column row_w + r, column c output row row_x + c
  if (split > 1) cluster_wait();     // the others run: their shared memory may be written
  const int share = COLS / split;
  if (c0 < COLS) {
#pragma unroll
    for (int c = c0; c < c0 + HALF; c += 32) {
      float f[32];
      tmem_ld_32x32(tmem + ((uint32_t)quarter << 16) + (uint32_t)c, (uint32_t*)f);
      tmem_ld_wait();
#pragma unroll
      for (int j = 0; j < 32; ++j) {
        float* at = sums + ((rank * share + (c + j) / split) * 128 + quarter + lane);
        if (split == 1) *at = f[j];
        else asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(mapa_u32(smem_u32(at), (uint32_t)((c + j) & (split - 1)))), "f"(f[j]) : "memory");
      }
    }
  }
  tc_fence_before_sync();
  if (split > 1) cluster_sync_all();
  else __syncthreads();
  if (warp == 2) tmem_dealloc(tmem, TMEM);
  const int cols = p.M - row_x < COLS ? (int)(p.M - row_x) : COLS, r = lane * 4;
  const bool vec = p.N % 4 == 0 && ((uintptr_t)p.out & 7) == 0;
  for (int i = warp; i * split + rank < cols; i += F_THREADS / 32) {   // a warp takes a column: 128 values of an output row
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (int q = 0; q < split; ++q) {
      const float4 s = *(const float4*)(sums + (q * share + i) * 128 + r);
      v.x += s.x, v.y += s.y, v.z += s.z, v.w += s.w;
    }
    __nv_bfloat16* dst = p.out + (row_x + i * split + rank) * p.N + row_w + r;
    alignas(8) __nv_bfloat162 o[2] = {__floats2bfloat162_rn(v.x, v.y), __floats2bfloat162_rn(v.z, v.w)};
    if (vec && row_w + r + 4 <= p.N) {
      *(uint2*)dst = *(uint2*)o;
    } else {
      for (int j = 0; j < 4; ++j)
        if (row_w + r + j < p.N) dst[j] = ((__nv_bfloat16*)o)[j];
    }
  }
  if (threadIdx.x == 0 && *abort_flag) atomicOr(p.error_flag, 1);
}

}  // namespace mx
}  // namespace bshmem
