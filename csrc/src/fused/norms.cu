// Norms before and after a block, fused with the block's gate and the scaled residual, forward and backward.
//
// A row of H values belongs to a group of threads (a warp up to a whole CTA), eight neighbouring values per thread and chunk.
// Everything a row needs stays in registers between its loads and its stores, so each input is read once and each output
// written once.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <stdio.h>

#include "../../include/bshmem/norms.h"

namespace bshmem {
namespace norms {

constexpr int CHUNK = 8;          // values per thread and chunk: 16 bytes of a 16-bit type
constexpr int MAX_THREADS = 1024;

template <typename T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }

// Values [col, col + 8) of a row of H; zero past the end.  VEC: H, the row's start and col allow 16-byte accesses.
template <bool VEC, typename T>
__device__ __forceinline__ void load8(float* f, const T* row, int col, int H) {
  if constexpr (VEC) {
    alignas(16) T raw[CHUNK];
    const uint4* src = (const uint4*)(row + col);
    constexpr int N = sizeof(raw) / 16;
#pragma unroll
    for (int i = 0; i < N; ++i) ((uint4*)raw)[i] = col < H ? src[i] : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
    for (int i = 0; i < CHUNK; ++i) f[i] = to_f<T>(raw[i]);
  } else {
#pragma unroll
    for (int i = 0; i < CHUNK; ++i) f[i] = col + i < H ? to_f<T>(row[col + i]) : 0.f;
  }
}
template <bool VEC, typename T>
__device__ __forceinline__ void store8(T* row, int col, int H, const float* f) {
  if constexpr (VEC) {
    if (col >= H) return;
    alignas(16) T raw[CHUNK];
#pragma unroll
    for (int i = 0; i < CHUNK; ++i) raw[i] = from_f<T>(f[i]);
    uint4* dst = (uint4*)(row + col);
    constexpr int N = sizeof(raw) / 16;
#pragma unroll
    for (int i = 0; i < N; ++i) dst[i] = ((uint4*)raw)[i];
  } else {
#pragma unroll
    for (int i = 0; i < CHUNK; ++i)
      if (col + i < H) row[col + i] = from_f<T>(f[i]);
  }
}
// The parameters are of the rows' type or fp32: one flag for all, the same for every thread.
template <bool VEC, typename T>
__device__ __forceinline__ void load8_wt(float* f, const void* row, bool wide, int col, int H) {
  if (wide) load8<VEC, float>(f, (const float*)row, col, H);
  else load8<VEC, T>(f, (const T*)row, col, H);
}
template <typename T>
__device__ __forceinline__ float load1_wt(const void* p, bool wide, size_t i) {
  return wide ? ((const float*)p)[i] : to_f<T>(((const T*)p)[i]);
}
template <typename T>
__device__ __forceinline__ void store1_wt(void* p, bool wide, size_t i, float v) {
  if (wide) ((float*)p)[i] = v;
  else ((T*)p)[i] = from_f<T>(v);
}

// Sum over the threads of a row's group (a power of two of at least 32 threads that starts at a multiple of itself), the same
// value in every thread.  All threads of the CTA call it.
template <int N>
__device__ __forceinline__ void group_sum(float (&v)[N], int group, float (*s)[N]) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  if (group == 32) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = group >> 5, first = warp & ~(warps - 1);
  __syncthreads();  // the sums of the call before have been read
  if (lane == 0)
#pragma unroll
    for (int i = 0; i < N; ++i) s[warp][i] = v[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = lane < warps ? s[first + lane][i] : 0.f;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
}

struct Params {
  bshmem_norm_args_t a;
  int group;  // threads per row
};

template <typename T, typename R, int CH, bool VEC>
__global__ void __launch_bounds__(MAX_THREADS) forward_kernel(const __grid_constant__ Params p) {
  const bshmem_norm_args_t& a = p.a;
  __shared__ float sums[MAX_THREADS / 32][1];
  const int H = a.H, group = p.group, g = threadIdx.x & (group - 1);
  const size_t row = (size_t)blockIdx.x * (blockDim.x / group) + threadIdx.x / group;
  const bool live = row < (size_t)a.T, wide = a.wt_type == BSHMEM_NORM_F32 && sizeof(T) < 4;
  const int h_end = live ? H : 0;  // a group without a row loads and stores nothing
  float r[CH][CHUNK];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    load8<VEC, R>(r[c], (const R*)a.residual + row * a.res_stride, (c * group + g) * CHUNK, h_end);
#pragma unroll
    for (int i = 0; i < CHUNK; ++i) r[c][i] *= a.residual_scale;
  }
  if (a.h) {
    float z[CH][CHUNK], ss[1] = {0.f};
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      load8<VEC, T>(z[c], (const T*)a.h + row * a.h_stride, (c * group + g) * CHUNK, h_end);
#pragma unroll
      for (int i = 0; i < CHUNK; ++i) ss[0] += z[c][i] * z[c][i];
    }
    float scale = a.branch_scale;
    if (a.post) {
      group_sum<1>(ss, group, sums);
      const float inv = rsqrtf(ss[0] / (float)H + a.eps);
      if (live && g == 0 && a.stat) a.stat[row] = inv;
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        float w[CHUNK];
        load8_wt<VEC, T>(w, a.post, wide, (c * group + g) * CHUNK, h_end);
#pragma unroll
        for (int i = 0; i < CHUNK; ++i) z[c][i] *= inv * (w[i] + a.weight_offset);
      }
    }
    if (a.gate_mode == BSHMEM_NORM_GATE_TOKEN && live) scale *= load1_wt<T>(a.gate, wide, row);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      if (a.gate_mode == BSHMEM_NORM_GATE_CHANNEL || a.gate_mode == BSHMEM_NORM_GATE_FULL) {
        float w[CHUNK];
        const size_t at = a.gate_mode == BSHMEM_NORM_GATE_FULL ? row * a.gate_stride : 0;
        load8_wt<VEC, T>(w, wide ? (const void*)((const float*)a.gate + at) : (const void*)((const T*)a.gate + at), wide, (c * group + g) * CHUNK, h_end);
#pragma unroll
        for (int i = 0; i < CHUNK; ++i) z[c][i] *= w[i];
      }
#pragma unroll
      for (int i = 0; i < CHUNK; ++i) r[c][i] += scale * z[c][i];
    }
  }
  if (a.r) {
#pragma unroll
    for (int c = 0; c < CH; ++c) store8<VEC, R>((R*)a.r + row * H, (c * group + g) * CHUNK, h_end, r[c]);
  }
  if (a.y) {
    float ss[1] = {0.f};
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int i = 0; i < CHUNK; ++i) ss[0] += r[c][i] * r[c][i];
    group_sum<1>(ss, group, sums);
    const float inv = rsqrtf(ss[0] / (float)H + a.eps);
    if (live && g == 0 && a.stat) a.stat[a.T + row] = inv;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      float w[CHUNK];
      load8_wt<VEC, T>(w, a.pre, wide, (c * group + g) * CHUNK, h_end);
#pragma unroll
      for (int i = 0; i < CHUNK; ++i) w[i] = r[c][i] * inv * (w[i] + a.weight_offset);
      store8<VEC, T>((T*)a.y + row * H, (c * group + g) * CHUNK, h_end, w);
    }
  }
}

// Backward.  With hhat = h s1, rhat = r s2 (s1, s2 from forward), q = branch_scale gate z:
//   c1 = mean(dy pre rhat)     G = dr + s2 (dy pre - rhat c1)          gradient of r
//   dresidual = residual_scale G    dgate = branch_scale G z
//   dh = s1 (branch_scale gate G post - hhat c2),  c2 = mean(q G) = mean(q (dr + s2 dy pre)) - c1 mean(q s2 rhat)
//   dpost = sum over rows of branch_scale gate G hhat     dpre = sum of dy rhat
// c2 is linear in G, so one reduction of three sums serves a row.  (For a gate per token the sums are taken without the gate:
// they are its gradient.)  A CTA walks rows with a stride of the grid and keeps its part of the sums over rows in shared
// memory; a second kernel adds the CTAs' parts in order.
template <typename T, typename R, int CH, bool VEC>
__global__ void __launch_bounds__(MAX_THREADS) backward_kernel(const __grid_constant__ Params p) {
  const bshmem_norm_args_t& a = p.a;
  extern __shared__ float acc[];  // [groups of the CTA][3][H]
  __shared__ float sums[MAX_THREADS / 32][3];
  const int H = a.H, group = p.group, g = threadIdx.x & (group - 1), groups = blockDim.x / group, mine = threadIdx.x / group;
  const bool wide = a.wt_type == BSHMEM_NORM_F32 && sizeof(T) < 4;
  const bool token = a.gate_mode == BSHMEM_NORM_GATE_TOKEN, elementwise = a.gate_mode == BSHMEM_NORM_GATE_CHANNEL || a.gate_mode == BSHMEM_NORM_GATE_FULL;
  float* my_acc = acc + (size_t)mine * 3 * H;
  if (a.partials)
    for (int i = threadIdx.x; i < groups * 3 * H; i += blockDim.x) acc[i] = 0.f;
  __syncthreads();
  for (size_t base = (size_t)blockIdx.x * groups; base < (size_t)a.T; base += (size_t)gridDim.x * groups) {
    const size_t row = base + mine;
    const bool live = row < (size_t)a.T;
    const int h_end = live ? H : 0;
    const float s1 = live && a.h && a.post ? a.stat[row] : 1.f, s2 = live && a.dy ? a.stat[a.T + row] : 0.f;
    const float tgate = token && live ? load1_wt<T>(a.gate, wide, row) : 1.f;
    float hv[CH][CHUNK], rh[CH][CHUNK], gr[CH][CHUNK], v[3] = {0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int col = (c * group + g) * CHUNK;
      float gate[CHUNK], post[CHUNK];
      load8<VEC, R>(rh[c], (const R*)a.residual + row * a.res_stride, col, h_end);
      if (a.h) load8<VEC, T>(hv[c], (const T*)a.h + row * a.h_stride, col, h_end);
      if (a.dr) load8<VEC, R>(gr[c], (const R*)a.dr + row * a.dr_stride, col, h_end);
      if (elementwise) {
        const size_t at = a.gate_mode == BSHMEM_NORM_GATE_FULL ? row * a.gate_stride : 0;
        load8_wt<VEC, T>(gate, wide ? (const void*)((const float*)a.gate + at) : (const void*)((const T*)a.gate + at), wide, col, h_end);
      }
      if (a.post) load8_wt<VEC, T>(post, a.post, wide, col, h_end);
      float dyw[CHUNK];
      if (a.dy) {
        float pre[CHUNK];
        load8<VEC, T>(dyw, (const T*)a.dy + row * a.dy_stride, col, h_end);
        load8_wt<VEC, T>(pre, a.pre, wide, col, h_end);
#pragma unroll
        for (int i = 0; i < CHUNK; ++i) pre[i] += a.weight_offset;
        float z[CHUNK];
#pragma unroll
        for (int i = 0; i < CHUNK; ++i) {
          z[i] = a.h ? hv[c][i] * s1 * (a.post ? post[i] + a.weight_offset : 1.f) : 0.f;
          const float q = z[i] * (elementwise ? gate[i] : tgate);
          rh[c][i] = s2 * (a.residual_scale * rh[c][i] + a.branch_scale * q);
        }
        if (a.partials && a.dpre) {
#pragma unroll
          for (int i = 0; i < CHUNK; ++i)
            if (col + i < h_end) my_acc[H + col + i] += dyw[i] * rh[c][i];
        }
#pragma unroll
        for (int i = 0; i < CHUNK; ++i) {
          dyw[i] *= pre[i];
          v[0] += dyw[i] * rh[c][i];
        }
      }
#pragma unroll
      for (int i = 0; i < CHUNK; ++i) {
        gr[c][i] = (a.dr ? gr[c][i] : 0.f) + (a.dy ? s2 * dyw[i] : 0.f);
        if (a.h) {
          const float z = hv[c][i] * s1 * (a.post ? post[i] + a.weight_offset : 1.f);
          const float q = a.branch_scale * z * (elementwise ? gate[i] : 1.f);
          v[1] += q * gr[c][i];
          if (a.dy) v[2] += q * s2 * rh[c][i];
        }
      }
    }
    group_sum<3>(v, group, sums);
    const float c1 = v[0] / (float)H, qg = v[1] - c1 * v[2];
    const float c2 = qg * tgate / (float)H;
    if (token && a.dgate && live && g == 0) store1_wt<T>(a.dgate, wide, row, qg);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int col = (c * group + g) * CHUNK;
      if (a.dy) {
#pragma unroll
        for (int i = 0; i < CHUNK; ++i) gr[c][i] -= s2 * rh[c][i] * c1;
      }
      if (a.dresidual) {
        float o[CHUNK];
#pragma unroll
        for (int i = 0; i < CHUNK; ++i) o[i] = a.residual_scale * gr[c][i];
        store8<VEC, R>((R*)a.dresidual + row * H, col, h_end, o);
      }
      if (!a.h) continue;
      float gate[CHUNK], post[CHUNK];
      if (elementwise) {
        const size_t at = a.gate_mode == BSHMEM_NORM_GATE_FULL ? row * a.gate_stride : 0;
        load8_wt<VEC, T>(gate, wide ? (const void*)((const float*)a.gate + at) : (const void*)((const T*)a.gate + at), wide, col, h_end);
      }
      if (a.post) load8_wt<VEC, T>(post, a.post, wide, col, h_end);
      float o[CHUNK];
#pragma unroll
      for (int i = 0; i < CHUNK; ++i) {
        const float hhat = hv[c][i] * s1, w = a.post ? post[i] + a.weight_offset : 1.f;
        const float bg = a.branch_scale * gr[c][i], dz = bg * (elementwise ? gate[i] : tgate);
        o[i] = a.post ? s1 * (dz * w - hhat * c2) : dz;
        if (a.partials && col + i < h_end) {
          if (a.dpost) my_acc[col + i] += dz * hhat;
          if (a.gate_mode == BSHMEM_NORM_GATE_CHANNEL && a.dgate) my_acc[2 * H + col + i] += bg * hhat * w;
        }
        post[i] = bg * hhat * w;
      }
      if (a.dh) store8<VEC, T>((T*)a.dh + row * H, col, h_end, o);
      if (a.gate_mode == BSHMEM_NORM_GATE_FULL && a.dgate) {
        if (wide) store8<VEC, float>((float*)a.dgate + row * H, col, h_end, post);
        else store8<VEC, T>((T*)a.dgate + row * H, col, h_end, post);
      }
    }
  }
  if (!a.partials) return;
  __syncthreads();
  for (int i = threadIdx.x; i < 3 * H; i += blockDim.x) {
    float s = 0.f;
    for (int k = 0; k < groups; ++k) s += acc[(size_t)k * 3 * H + i];
    a.partials[(size_t)blockIdx.x * 3 * H + i] = s;
  }
}

// Sums of the CTAs' parts, in order: dpost, dpre and the channel gate's gradient.
template <typename T>
__global__ void column_sum_kernel(const __grid_constant__ Params p, int parts) {
  const bshmem_norm_args_t& a = p.a;
  const int i = blockIdx.x * 32 + threadIdx.x, which = blockIdx.y;
  void* dst = which == 0 ? a.dpost : which == 1 ? a.dpre : a.gate_mode == BSHMEM_NORM_GATE_CHANNEL ? a.dgate : nullptr;
  if (!dst) return;
  __shared__ float s[8][32];
  float v = 0.f;
  if (i < a.H)
    for (int k = threadIdx.y; k < parts; k += 8) v += a.partials[((size_t)k * 3 + which) * a.H + i];
  s[threadIdx.y][threadIdx.x] = v;
  __syncthreads();
  if (threadIdx.y == 0 && i < a.H) {
#pragma unroll
    for (int k = 1; k < 8; ++k) v += s[k][threadIdx.x];
    store1_wt<T>(dst, a.wt_type == BSHMEM_NORM_F32 && sizeof(T) < 4, i, v);
  }
}

static bool aligned(const void* p) { return ((uintptr_t)p & 15) == 0; }

// Rows and parameters may be read and written 16 bytes at a time.
static bool vectors(const bshmem_norm_args_t* a) {
  if (a->H % CHUNK) return false;
  const void* ptrs[] = {a->h, a->residual, a->post, a->pre, a->gate, a->r, a->y, a->dr, a->dy, a->dh, a->dresidual, a->dgate};
  for (const void* q : ptrs)
    if (!aligned(q)) {
      if (q == a->gate || q == a->dgate) {
        if (a->gate_mode == BSHMEM_NORM_GATE_TOKEN) continue;
      }
      return false;
    }
  return !((a->h_stride | a->res_stride | a->dr_stride | a->dy_stride) & 7) && (a->gate_mode != BSHMEM_NORM_GATE_FULL || !(a->gate_stride & 7));
}

static int check(const bshmem_norm_args_t* a) {
  if (!a || a->T < 0 || a->H < 1 || a->H > BSHMEM_NORM_MAX_H) return BSHMEM_NORM_ERR_SHAPE;
  if (a->type < 0 || a->type > 2 || (a->res_type != a->type && a->res_type != BSHMEM_NORM_F32) || (a->wt_type != a->type && a->wt_type != BSHMEM_NORM_F32)) return BSHMEM_NORM_ERR_ARGS;
  if (a->gate_mode < 0 || a->gate_mode > 3 || (a->gate_mode && (!a->gate || !a->h)) || !a->residual || (a->post && !a->h)) return BSHMEM_NORM_ERR_ARGS;
  if ((a->y || a->dy) && !a->pre) return BSHMEM_NORM_ERR_ARGS;
  return BSHMEM_NORM_OK;
}

static int group_threads(int H, int chunks) {
  int g = 32;
  while (g * CHUNK * chunks < H && g < MAX_THREADS) g *= 2;
  return g;
}

static int sm_count() {
  int device = 0, sms = 0;
  cudaGetDevice(&device);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
  return sms > 0 ? sms : 1;
}

static int backward_ctas(int T, int H) {
  const int group = group_threads(H, 1), groups = group < 128 ? 128 / group : 1;
  const int want = (T + groups - 1) / groups, most = sm_count() * (H <= 4096 ? 4 : 1);
  return want < most ? want : most;
}

template <typename T, typename R>
static int launch_forward(const Params& p, int chunks, bool vec, cudaStream_t stream) {
  const int threads = p.group < 128 ? 128 : p.group, rows = threads / p.group;
  const unsigned grid = (unsigned)(((size_t)p.a.T + rows - 1) / rows);
  if (chunks == 1 && vec) forward_kernel<T, R, 1, true><<<grid, threads, 0, stream>>>(p);
  else if (chunks == 1) forward_kernel<T, R, 1, false><<<grid, threads, 0, stream>>>(p);
  else if (vec) forward_kernel<T, R, 2, true><<<grid, threads, 0, stream>>>(p);
  else forward_kernel<T, R, 2, false><<<grid, threads, 0, stream>>>(p);
  return cudaGetLastError() == cudaSuccess ? BSHMEM_NORM_OK : BSHMEM_NORM_ERR_DRIVER;
}

template <typename T, typename R>
static int launch_backward(const Params& p, int chunks, bool vec, cudaStream_t stream) {
  const int threads = p.group < 128 ? 128 : p.group, groups = threads / p.group;
  const int smem = p.a.partials ? groups * 3 * p.a.H * 4 : 0, grid = backward_ctas(p.a.T, p.a.H);
  void (*const kernel)(Params) = chunks == 1 ? (vec ? backward_kernel<T, R, 1, true> : backward_kernel<T, R, 1, false>)
                                             : (vec ? backward_kernel<T, R, 2, true> : backward_kernel<T, R, 2, false>);
  if (smem > 48 * 1024 && cudaFuncSetAttribute((const void*)kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return BSHMEM_NORM_ERR_DRIVER;
  kernel<<<grid, threads, smem, stream>>>(p);
  if (p.a.partials) column_sum_kernel<T><<<dim3((p.a.H + 31) / 32, 3), dim3(32, 8), 0, stream>>>(p, grid);
  return cudaGetLastError() == cudaSuccess ? BSHMEM_NORM_OK : BSHMEM_NORM_ERR_DRIVER;
}

template <typename F>
static int by_type(const bshmem_norm_args_t* a, F&& f) {
  const bool same = a->res_type == a->type;
  if (a->type == BSHMEM_NORM_F32) return f((float*)nullptr, (float*)nullptr);
  if (a->type == BSHMEM_NORM_BF16) return same ? f((__nv_bfloat16*)nullptr, (__nv_bfloat16*)nullptr) : f((__nv_bfloat16*)nullptr, (float*)nullptr);
  return same ? f((__half*)nullptr, (__half*)nullptr) : f((__half*)nullptr, (float*)nullptr);
}

}  // namespace norms
}  // namespace bshmem

using namespace bshmem::norms;

extern "C" size_t bshmem_block_norms_partials(int T, int H) { return T > 0 && H > 0 ? (size_t)backward_ctas(T, H) * 3 * H : 0; }

extern "C" int bshmem_block_norms(const bshmem_norm_args_t* a, cudaStream_t stream) {
  if (a && a->T == 0) return BSHMEM_NORM_OK;
  const int st = check(a);
  if (st) return st;
  if (!a->r && !a->y) return BSHMEM_NORM_ERR_ARGS;
  const int group = group_threads(a->H, 1), chunks = a->H > group * CHUNK ? 2 : 1;
  const Params p = {*a, group};
  const bool vec = vectors(a);
  return by_type(a, [&](auto* t, auto* r) {
    return launch_forward<std::remove_pointer_t<decltype(t)>, std::remove_pointer_t<decltype(r)>>(p, chunks, vec, stream);
  });
}

extern "C" int bshmem_block_norms_backward(const bshmem_norm_args_t* a, cudaStream_t stream) {
  if (a && a->T == 0) return BSHMEM_NORM_OK;
  const int st = check(a);
  if (st) return st;
  const bool sums = a->dpost || a->dpre || (a->dgate && a->gate_mode == BSHMEM_NORM_GATE_CHANNEL);
  if ((!a->dr && !a->dy) || (a->dpre && !a->dy) || (a->dpost && !a->post) || ((a->dh || a->dgate) && !a->h) || (a->dgate && !a->gate_mode)) return BSHMEM_NORM_ERR_ARGS;
  if ((sums && !a->partials) || ((a->post || a->dy) && !a->stat)) return BSHMEM_NORM_ERR_ARGS;
  const int group = group_threads(a->H, 1), chunks = a->H > group * CHUNK ? 2 : 1;
  Params p = {*a, group};
  if (!sums) p.a.partials = nullptr;
  const bool vec = vectors(a);
  return by_type(a, [&](auto* t, auto* r) {
    return launch_backward<std::remove_pointer_t<decltype(t)>, std::remove_pointer_t<decltype(r)>>(p, chunks, vec, stream);
  });
}
