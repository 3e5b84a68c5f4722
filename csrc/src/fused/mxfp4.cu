// Microscaled 4-bit floating point: quantisation, reading back, and the block-scaled product on tcgen05.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <stdio.h>
#include <string.h>

#include <atomic>
#include <type_traits>

#include "../../include/bshmem/mxfp4.h"
#include "../../include/bshmem/tcgen05.cuh"
#include "gemm_mxfp4.cuh"
#include "launch.cuh"
#include "tensor_map.cuh"

namespace bshmem {
namespace mx {
using namespace sm100;

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float from_f(float, float v) { return v; }
__device__ __forceinline__ __nv_bfloat16 from_f(__nv_bfloat16, float v) { return __float2bfloat16_rn(v); }
__device__ __forceinline__ __half from_f(__half, float v) { return __float2half_rn(v); }

// ------------------------------------------------------------------ quantisation
// Bound by memory: 2 or 4 bytes read and 17/32 written per value, and the reverse.  A warp takes 1024 or 2048 values of a row, all its loads on
// their way before the first is used, marked as read once; so are the values that are read back (8192 x 8192 to fp32 51.5 -> 44.5 us).  The eight rows of a CTA are those whose scales share a 32-byte sector: r, r + 1 and the same
// 32, 64 and 96 rows on.
constexpr int Q_THREADS = 256, Q_CHUNK = 2048;

struct RowSlot {
  int64_t row;
  int64_t scale;   // offset of the row's scales inside a block of 128 rows
};
__device__ __forceinline__ RowSlot row_slot() {
  const int warp = threadIdx.x >> 5, in32 = (blockIdx.x & 15) * 2 + (warp & 1), quarter = warp >> 1;
  return {(int64_t)(blockIdx.x >> 4) * 128 + quarter * 32 + in32, in32 * 16 + quarter * 4};
}
constexpr int MAX_GRID_Y = 65535;
static int64_t chunks_of(int64_t K, int chunk) { return (k_blocks(K) * 128 + chunk - 1) / chunk; }
static dim3 row_grid(int64_t R, int64_t chunks) { return dim3((unsigned)(row_blocks(R) * 16), (unsigned)chunks); }

// A lane takes a block of 32 values, so that their largest exponent needs no exchange (8192 x 8192 bf16 34.0 -> 29.9 us against eight values a
// lane), and four lanes' scales go out as a word.  A scale is a power of two, so x / scale is exact and the only rounding is the one to E2M1.
__device__ __forceinline__ uint32_t pack_e2m1(const float* f) {  // eight values, the first in the low four bits; nearest even, saturating
  uint32_t out;
  asm("{\n .reg .b8 a, b, c, d;\n cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n"
      " cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n mov.b32 %0, {a, b, c, d};\n}\n"
      : "=r"(out)
      : "f"(f[0]), "f"(f[1]), "f"(f[2]), "f"(f[3]), "f"(f[4]), "f"(f[5]), "f"(f[6]), "f"(f[7]));
  return out;
}
// Largest magnitude of eight values, as the bits of a float (up to the lowest bits of 16-bit types, which do not reach the exponent).
template <typename T>
__device__ __forceinline__ uint32_t exponent_bits(const uint4* raw, const float* f) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {  // the upper half of a float: the largest of each pair at once
    const uint32_t m = __vmaxu2(__vmaxu2(raw->x & 0x7fff7fffu, raw->y & 0x7fff7fffu), __vmaxu2(raw->z & 0x7fff7fffu, raw->w & 0x7fff7fffu));
    return max(m & 0xffff0000u, m << 16);
  } else {
    uint32_t m = 0;  // bits order like the magnitudes; a NaN is above infinity
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(f[i]) & 0x7fffffffu);
    return m;
  }
}

// Values of a row that a warp takes, all its loads at once: one block a lane of fp32, two of 16-bit types (1001 x 1184 fp32 3.1 us; with
// 2048 values in two steps 3.9).
template <typename T>
__host__ __device__ constexpr int quantize_chunk() { return sizeof(T) == 4 ? 1024 : 2048; }

template <typename T, bool VEC>
__global__ void __launch_bounds__(Q_THREADS) quantize_kernel(const T* __restrict__ x, int64_t R, int K, int64_t stride, uint8_t* __restrict__ data,
                                                             uint8_t* __restrict__ scales, int first_chunk) {
  constexpr int UNROLL = quantize_chunk<T>() / 1024, WORDS = sizeof(T) * 32 / 16;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // a product may set up, and fetch its weights, beside this kernel
  const RowSlot slot = row_slot();
  const int lane = threadIdx.x & 31;
  const int KB = (int)k_blocks(K), base = (first_chunk + (int)blockIdx.y) * quantize_chunk<T>() + lane * 32;
  const bool row_live = slot.row < R;
  const T* src = x + slot.row * stride;
  uint8_t* dst = data + slot.row * (K / 2);
  uint8_t* sdst = scales + (slot.row / 128) * KB * SCALE_BLOCK + slot.scale;
  uint4 raw[UNROLL][WORDS];
#pragma unroll
  for (int u = 0; u < UNROLL; ++u) {
    const bool live = row_live && base + u * 1024 < K;
    if constexpr (VEC) {
#pragma unroll
      for (int i = 0; i < WORDS; ++i) raw[u][i] = live ? __ldcs((const uint4*)(src + base + u * 1024) + i) : make_uint4(0u, 0u, 0u, 0u);
    } else {
      T* v = (T*)raw[u];
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = live ? src[base + u * 1024 + i] : T(0.f);
    }
  }
#pragma unroll
  for (int u = 0; u < UNROLL; ++u) {
    const int at = base + u * 1024;
    uint32_t amax = 0;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      float f[8];
      const T* v = (const T*)raw[u] + 8 * g;
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = to_f(v[i]);
      amax = max(amax, exponent_bits<T>(raw[u] + g * (WORDS / 4), f));
    }
    const uint32_t biased = amax >> 23;  // floor(log2 amax) + 127; 0 for subnormals
    const uint32_t code = biased == 255 ? 255 : max(biased, 2u) - 2;
    const float inv = __uint_as_float((254u - min(code, 254u)) << 23);  // 2^(127 - code)
    uint32_t packed[4];
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      float f[8];
      const T* v = (const T*)raw[u] + 8 * g;
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = to_f(v[i]) * inv;
      packed[g] = pack_e2m1(f);
    }
    uint32_t word = code << (8 * (lane & 3));  // four lanes' scales as one word
    word |= __shfl_xor_sync(0xffffffffu, word, 1);
    word |= __shfl_xor_sync(0xffffffffu, word, 2);
    if (row_live && at < K) *(uint4*)(dst + at / 2) = make_uint4(packed[0], packed[1], packed[2], packed[3]);
    if ((lane & 3) == 0 && at < KB * 128) *(uint32_t*)(sdst + at / 128 * SCALE_BLOCK) = word;  // of rows and K past the end too: zeros
  }
}

static_assert((1 << 26) / Q_CHUNK <= MAX_GRID_Y, "the longest row in one launch");
// The reverse; a lane's values fill one 16-byte store: four fp32 or eight 16-bit ones.
template <typename T>
__global__ void __launch_bounds__(Q_THREADS) dequantize_kernel(const uint8_t* __restrict__ data, const uint8_t* __restrict__ scales, int64_t R, int K, T* __restrict__ out) {
  constexpr int PER_LANE = 16 / sizeof(T), STEP = 32 * PER_LANE, UNROLL = Q_CHUNK / STEP < 8 ? Q_CHUNK / STEP : 8;
  typedef typename std::conditional<PER_LANE == 8, uint32_t, uint16_t>::type Packed;
  const RowSlot slot = row_slot();
  if (slot.row >= R) return;
  const int lane = threadIdx.x & 31;
  const uint8_t* ssrc = scales + (slot.row / 128) * k_blocks(K) * SCALE_BLOCK + slot.scale;
  const uint8_t* src = data + slot.row * (K / 2);
  T* dst = out + slot.row * K;
  const int first = (int)blockIdx.y * Q_CHUNK, last = first + Q_CHUNK < K ? first + Q_CHUNK : K;
#pragma unroll 1
  for (int base = first + lane * PER_LANE; base < last; base += UNROLL * STEP) {
    uint32_t packed[UNROLL], code[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int col = base + u * STEP;
      if (col >= last) continue;
      packed[u] = *(const Packed*)(src + col / 2);
      code[u] = ssrc[col / 128 * SCALE_BLOCK + col % 128 / BLOCK];
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int col = base + u * STEP;
      if (col >= last) continue;
      const float scale = __uint_as_float(code[u] == 255 ? 0x7fffffffu : code[u] ? code[u] << 23 : 0x00400000u);
      alignas(16) T raw[PER_LANE];
#pragma unroll
      for (int j = 0; j < PER_LANE; ++j) {
        // E2M1's exponent and mantissa in a float's places stand for the value times 2^-126, its 0.5 included (a subnormal)
        const uint32_t q = packed[u] << (28 - 4 * j);
        const float v = __uint_as_float((q & 0x80000000u) | (q >> 28 & 7) << 22) * 0x1p126f;
        raw[j] = from_f(T(), v * scale);
      }
      __stcs((uint4*)(dst + col), *(uint4*)raw);
    }
  }
}

static int launched(const char* what, cudaError_t e) {
  if (e == cudaSuccess) return BSHMEM_MX_OK;
  fprintf(stderr, "%s: launch failed: %s\n", what, cudaGetErrorString(e));
  return BSHMEM_MX_ERR_DRIVER;
}

template <typename T>
static int launch_quantize(const void* x, int64_t R, int64_t K, int64_t stride, void* data, void* scales, cudaStream_t stream) {
  const bool vec = ((uintptr_t)x & 15) == 0 && (stride * (int64_t)sizeof(T)) % 16 == 0;
  // The longest rows of fp32 have one chunk more than a grid's second dimension takes.
  const int64_t chunks = chunks_of(K, quantize_chunk<T>());
  for (int64_t first = 0; first < chunks; first += MAX_GRID_Y) {
    const int64_t n = chunks - first < MAX_GRID_Y ? chunks - first : MAX_GRID_Y;
    const int st = launched("bshmem_mxfp4_quantize", launch_kernel(vec ? quantize_kernel<T, true> : quantize_kernel<T, false>, row_grid(R, n), Q_THREADS, stream, (const T*)x, R,
                                                                   (int)K, stride, (uint8_t*)data, (uint8_t*)scales, (int)first));
    if (st) return st;
  }
  return BSHMEM_MX_OK;
}
template <typename T>
static int launch_dequantize(const void* data, const void* scales, int64_t R, int64_t K, void* out, cudaStream_t stream) {
  return launched("bshmem_mxfp4_dequantize",
                  launch_kernel(dequantize_kernel<T>, row_grid(R, chunks_of(K, Q_CHUNK)), Q_THREADS, stream, (const uint8_t*)data, (const uint8_t*)scales, R, (int)K, (T*)out));
}

// Tensor map of scales: rows are row blocks, elements words; a box is 1 KB (256 values of K) of `blocks` row blocks.
static int make_scale_map(CUtensorMap* out, const void* base, int64_t rows, int64_t K, uint32_t blocks) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return BSHMEM_FUSED_ERR_DRIVER;
  cuuint64_t dims[2] = {(cuuint64_t)k_blocks(K) * (SCALE_BLOCK / 4), (cuuint64_t)row_blocks(rows)};
  cuuint64_t strides[1] = {dims[0] * 4};
  cuuint32_t box[2] = {256, blocks}, estr[2] = {1, 1};
  const CUresult r = fn(out, CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, (void*)base, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : BSHMEM_FUSED_ERR_DRIVER;
}
static int map_status(int st) { return st == 0 ? BSHMEM_MX_OK : st == BSHMEM_FUSED_ERR_ALIGNMENT ? BSHMEM_MX_ERR_ALIGNMENT : BSHMEM_MX_ERR_DRIVER; }
// Raises a kernel's shared-memory limit, once per GPU (`ready`: the GPUs done, bit = ordinal).
static bool reserve_smem(const void* kernel, int bytes, std::atomic<uint64_t>& ready) {
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess) return false;
  if (device < 64 && (ready.load(std::memory_order_acquire) >> device & 1)) return true;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return false;
  if (device < 64) ready.fetch_or(1ull << device, std::memory_order_release);
  return true;
}
static int sm_count() {
  int device = 0, sms = 0;
  cudaGetDevice(&device);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
  return sms > 1 ? sms : 2;
}

// A launch that may begin before the kernel ahead of it on the stream has ended (the kernels wait themselves).
template <typename P>
static int launch_clusters(void (*kernel)(P), const P& p, int grid, int threads, int smem, int cluster, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
  if (e == cudaSuccess) return BSHMEM_MX_OK;
  fprintf(stderr, "bshmem_mxfp4_gemm: launch failed: %s\n", cudaGetErrorString(e));
  return BSHMEM_MX_ERR_DRIVER;
}

template <int COLS>
static int launch_pair(const bshmem_mxfp4_gemm_args_t* a, uint64_t wait_limit_ns, cudaStream_t stream) {
  PairParams p;
  memset(&p, 0, sizeof(p));
  int st = make_map(&p.tmA, a->x, (uint64_t)a->M, (uint64_t)a->K / 4, 128);  // bytes, in pairs: the box is 128 rows by 128 bytes
  if (!st) st = make_map(&p.tmB, a->w, (uint64_t)a->N, (uint64_t)a->K / 4, COLS / 2);
  if (a->N % 8 == 0 && ((uintptr_t)a->out & 15) == 0) {
    if (!st) st = make_map(&p.tmOut, a->out, (uint64_t)a->M, (uint64_t)a->N, 128);
  } else {
    p.direct = (__nv_bfloat16*)a->out;
  }
  if (!st) st = make_scale_map(&p.tmSA, a->x_scales, a->M, a->K, 1);
  if (!st) st = make_scale_map(&p.tmSB, a->w_scales, a->N, a->K, COLS / 128);
  if (st) return map_status(st);
  p.error_flag = a->error_flag;
  p.wait_limit_ns = wait_limit_ns;
  p.M = (int)a->M; p.N = (int)a->N; p.K = (int)a->K;
  p.tiles_m = (int)((a->M + 255) / 256);
  p.tiles_n = (int)((a->N + COLS - 1) / COLS);
  const int64_t tiles = (int64_t)p.tiles_m * p.tiles_n;
  if (tiles > 0x3fffffff) return BSHMEM_MX_ERR_SHAPE;
  p.tiles = (int)tiles;
  static std::atomic<uint64_t> ready;
  if (!reserve_smem((const void*)gemm_pair_kernel<COLS>, PairTile<COLS>::SMEM, ready)) return BSHMEM_MX_ERR_DRIVER;
  const int most = sm_count() / 2;
  return launch_clusters(gemm_pair_kernel<COLS>, p, 2 * (p.tiles < most ? p.tiles : most), P_THREADS, PairTile<COLS>::SMEM, 2, stream);
}

template <int COLS>
static int launch_few(const bshmem_mxfp4_gemm_args_t* g, int split, uint64_t wait_limit_ns, cudaStream_t stream) {
  FewParams p;
  memset(&p, 0, sizeof(p));
  int st = make_map(&p.tmW, g->w, (uint64_t)g->N, (uint64_t)g->K / 4, 128);
  if (!st) st = make_map(&p.tmX, g->x, (uint64_t)g->M, (uint64_t)g->K / 4, COLS);
  if (!st) st = make_scale_map(&p.tmSW, g->w_scales, g->N, g->K, 1);
  if (!st) st = make_scale_map(&p.tmSX, g->x_scales, g->M, g->K, 1);
  if (st) return map_status(st);
  p.out = (__nv_bfloat16*)g->out;
  p.error_flag = g->error_flag;
  p.wait_limit_ns = wait_limit_ns;
  p.M = g->M;
  p.N = g->N;
  p.K = (int)g->K;
  p.tiles_w = (int)((g->N + 127) / 128);
  p.split = split;
  p.early = g->raw_x != nullptr;  // the kernel ahead quantised x, and began after everything before it was complete
  const int64_t ctas = (int64_t)p.tiles_w * ((g->M + COLS - 1) / COLS) * split;
  if (ctas > 0x7fffffff) return BSHMEM_MX_ERR_SHAPE;
  static std::atomic<uint64_t> ready;
  if (!reserve_smem((const void*)gemm_few_kernel<COLS>, FewTile<COLS>::SMEM, ready)) return BSHMEM_MX_ERR_DRIVER;
  return launch_clusters(gemm_few_kernel<COLS>, p, (int)ctas, F_THREADS, FewTile<COLS>::SMEM, split, stream);
}

// Which kernel takes a product, by a model of measured times (us, operands in memory): a fixed part and, per step of 256 values of K and
// wave of tiles, what an SM takes to load its share.  Measured (few rows with 64 columns, pairs of 128 and 256 columns):
//     64 x 8192 x 8192   12.6 / 12.8 / 16.2      512 x 2048 x 2048    7.5 /  6.4 /  7.8
//    100 x 8192 x 8192   14.2 / 13.0 / 16.5      512 x 4096 x 7168   22.9 / 12.1 / 15.2
//    129 x 2048 x 8192    9.9 / 11.5 / 14.7      512 x 8192 x 8192   47.3 / 21.2 / 18.1
//    300 x  512 x 8192    7.9 / 11.2 / 14.2     1024 x 8192 x 3584   59.5 / 20.4 / 17.4
struct Plan {
  int cols;    // 32, 64: few rows; 128, 256: pairs
  int split;   // CTAs that divide K
};
static Plan plan_product(int64_t M, int64_t N, int64_t K, int sms) {
  const int64_t steps = (K + 255) / 256;
  Plan best = {0, 1};
  double best_us = 0.0;
  auto offer = [&](int cols, int split, double us) {
    if (best.cols && us >= best_us) return;
    best = {cols, split};
    best_us = us;
  };
  for (int cols = 32; cols <= 64; cols *= 2) {
    if (cols == 32 && M > 32) continue;   // scales of a tile start at a multiple of 64 rows
    const int64_t tiles = (N + 127) / 128 * ((M + cols - 1) / cols);
    // K is divided as long as that brings in SMs that would be idle, and leaves a CTA two steps at least.
    int split = 1;
    while (split < 8 && tiles * split * 2 <= sms && steps >= split * 4) split *= 2;
    const double waves = (double)((tiles * split + sms - 1) / sms), per_cta = (double)((steps + split - 1) / split);
    offer(cols, split, 5.0 + (split > 1 ? 1.0 : 0.0) + waves * per_cta * (cols == 32 ? 0.22 : 0.29));
  }
  for (int cols = 128; cols <= 256; cols *= 2) {
    const int64_t tiles = (M + 255) / 256 * ((N + cols - 1) / cols), pairs = sms / 2;
    offer(cols, 1, 5.2 + (double)((tiles + pairs - 1) / pairs) * (double)steps * (cols == 128 ? 0.22 : 0.37));
  }
  return best;
}

}  // namespace mx
}  // namespace bshmem

using namespace bshmem;
using namespace bshmem::mx;

extern "C" size_t bshmem_mxfp4_scale_bytes(int64_t R, int64_t K) { return R > 0 && K > 0 ? (size_t)(row_blocks(R) * k_blocks(K)) * SCALE_BLOCK : 0; }

static int check_matrix(int64_t R, int64_t K) { return R < 0 || K < BLOCK || K % BLOCK || R > 0x7fffff00ll || K >= 1 << 26 ? BSHMEM_MX_ERR_SHAPE : BSHMEM_MX_OK; }

extern "C" int bshmem_mxfp4_quantize(const void* x, int type, int64_t R, int64_t K, int64_t stride, void* data, void* scales, cudaStream_t stream) {
  const int st = check_matrix(R, K);
  if (st || R == 0) return st;
  if (!x || !data || !scales) return BSHMEM_MX_ERR_ARGS;
  if (((uintptr_t)data | (uintptr_t)scales) & 15) return BSHMEM_MX_ERR_ALIGNMENT;
  if (type == BSHMEM_MX_BF16) return launch_quantize<__nv_bfloat16>(x, R, K, stride, data, scales, stream);
  if (type == BSHMEM_MX_F16) return launch_quantize<__half>(x, R, K, stride, data, scales, stream);
  if (type == BSHMEM_MX_F32) return launch_quantize<float>(x, R, K, stride, data, scales, stream);
  return BSHMEM_MX_ERR_ARGS;
}

extern "C" int bshmem_mxfp4_dequantize(const void* data, const void* scales, int64_t R, int64_t K, int type, void* out, cudaStream_t stream) {
  const int st = check_matrix(R, K);
  if (st || R == 0) return st;
  if (!data || !scales || !out) return BSHMEM_MX_ERR_ARGS;
  if (((uintptr_t)data | (uintptr_t)scales | (uintptr_t)out) & 15) return BSHMEM_MX_ERR_ALIGNMENT;
  if (type == BSHMEM_MX_BF16) return launch_dequantize<__nv_bfloat16>(data, scales, R, K, out, stream);
  if (type == BSHMEM_MX_F16) return launch_dequantize<__half>(data, scales, R, K, out, stream);
  if (type == BSHMEM_MX_F32) return launch_dequantize<float>(data, scales, R, K, out, stream);
  return BSHMEM_MX_ERR_ARGS;
}

extern "C" int bshmem_mxfp4_gemm(const bshmem_mxfp4_gemm_args_t* a, cudaStream_t stream) {
  if (!a) return BSHMEM_MX_ERR_ARGS;
  const int st = check_matrix(a->M, a->K) | check_matrix(a->N, a->K);
  if (st || a->M == 0 || a->N == 0) return st ? BSHMEM_MX_ERR_SHAPE : BSHMEM_MX_OK;
  if (!a->x || !a->x_scales || !a->w || !a->w_scales || !a->out || !a->error_flag) return BSHMEM_MX_ERR_ARGS;
  if (((uintptr_t)a->x_scales | (uintptr_t)a->w_scales) & 15) return BSHMEM_MX_ERR_ALIGNMENT;
  if (a->raw_x) {
    const int q = bshmem_mxfp4_quantize(a->raw_x, a->raw_type, a->M, a->K, a->raw_stride, (void*)a->x, (void*)a->x_scales, stream);
    if (q) return q;
  }
  const uint64_t limit = a->wait_limit_ms ? (uint64_t)a->wait_limit_ms * 1000000ull : 10000000000ull;
  const Plan plan = plan_product(a->M, a->N, a->K, sm_count());
  if (plan.cols == 32) return launch_few<32>(a, plan.split, limit, stream);
  if (plan.cols == 64) return launch_few<64>(a, plan.split, limit, stream);
  return plan.cols == 128 ? launch_pair<128>(a, limit, stream) : launch_pair<256>(a, limit, stream);
}

// Test hook (host only): the tile width and the division of K that plan_product chooses.
extern "C" void bshmem_mxfp4_test_plan(int64_t M, int64_t N, int64_t K, int sms, int* out) {
  const Plan plan = plan_product(M, N, K, sms);
  out[0] = plan.cols;
  out[1] = plan.split;
}
