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
#include "../../include/bshmem/tcgen05.cuh"

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

// Backward.  With hhat = h s1, rhat = r s2 (s1, s2 from forward), u = branch_scale post, q = gate u hhat:
//   c1 = mean(dy pre rhat)     G = dr + s2 (dy pre - rhat c1)          gradient of r
//   dresidual = residual_scale G      dgate = G u hhat
//   dh = s1 (gate u G - hhat c2),  c2 = mean(q G) = mean(q (dr + s2 dy pre)) - c1 s2 mean(q rhat)
//   dpost = branch_scale sum over rows of gate G hhat     dpre = sum of dy rhat
// c2 is linear in G, so one reduction of three sums serves a row.  (For a gate per token the sums are taken without the gate:
// they are its gradient.)  Where the gate is per channel it is the same for every row, and one sum S = sum of G hhat gives both
// dpost = branch_scale gate S and dgate = u S.  A CTA walks rows with a stride of the grid and keeps its part of the two sums
// over rows; a second kernel adds the CTAs' parts in order.
template <typename T, typename R, int CH, bool VEC>
__global__ void __launch_bounds__(MAX_THREADS) backward_kernel(const __grid_constant__ Params p) {
  const bshmem_norm_args_t& a = p.a;
  extern __shared__ float acc[];  // [groups of the CTA][2][H]: S, dpre
  __shared__ float sums[MAX_THREADS / 32][3];
  const int H = a.H, group = p.group, g = threadIdx.x & (group - 1), groups = blockDim.x / group, mine = threadIdx.x / group;
  const bool wide = a.wt_type == BSHMEM_NORM_F32 && sizeof(T) < 4;
  const bool full = a.gate_mode == BSHMEM_NORM_GATE_FULL;
  const bool token = a.gate_mode == BSHMEM_NORM_GATE_TOKEN, elementwise = a.gate_mode == BSHMEM_NORM_GATE_CHANNEL || a.gate_mode == BSHMEM_NORM_GATE_FULL;
  float* my_acc = acc + (size_t)mine * 2 * H;
  if (a.partials)
    for (int i = threadIdx.x; i < groups * 2 * H; i += blockDim.x) acc[i] = 0.f;
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
        if (a.partials && col + i < h_end) my_acc[col + i] += (full ? gate[i] : tgate) * gr[c][i] * hhat;
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
  for (int i = threadIdx.x; i < 2 * H; i += blockDim.x) {
    float s = 0.f;
    for (int k = 0; k < groups; ++k) s += acc[(size_t)k * 2 * H + i];
    a.partials[(size_t)blockIdx.x * 2 * H + i] = s;
  }
}

// Sums of the CTAs' parts, in order: S (dpost and the channel gate's gradient) and dpre.
template <typename T>
__global__ void __launch_bounds__(256) column_sum_kernel(const __grid_constant__ Params p, int parts) {
  const bshmem_norm_args_t& a = p.a;
  const int i = blockIdx.x * 32 + threadIdx.x;
  const bool pre = blockIdx.y != 0, channel = a.gate_mode == BSHMEM_NORM_GATE_CHANNEL, wide = a.wt_type == BSHMEM_NORM_F32 && sizeof(T) < 4;
  if (pre ? !a.dpre : !a.dpost && !(a.dgate && channel)) return;
  __shared__ float s[8][32];
  float v = 0.f;
  if (i < a.H)
    for (int k = threadIdx.y; k < parts; k += 8) v += a.partials[((size_t)k * 2 + pre) * a.H + i];
  s[threadIdx.y][threadIdx.x] = v;
  __syncthreads();
  if (threadIdx.y || i >= a.H) return;
#pragma unroll
  for (int k = 1; k < 8; ++k) v += s[k][threadIdx.x];
  if (pre) {
    store1_wt<T>(a.dpre, wide, i, v);
    return;
  }
  if (a.dpost) store1_wt<T>(a.dpost, wide, i, a.branch_scale * v * (channel ? load1_wt<T>(a.gate, wide, i) : 1.f));
  if (a.dgate && channel) store1_wt<T>(a.dgate, wide, i, a.branch_scale * v * (a.post ? load1_wt<T>(a.post, wide, i) + a.weight_offset : 1.f));
}

// ------------------------------------------------------------------ many rows
// The kernels above keep only the rows in flight that fit the registers.  With more rows than the SMs take at once, each CTA walks
// rows instead: one warp copies rows (cp.async.bulk, 16-byte aligned) into a ring in shared memory ahead of the other warps, each thread of
// which owns sixteen columns for the whole run, with their parameters and their sums over rows in registers.
constexpr int RING_CH = 4, RING_COLS = 4 * RING_CH, RING_MAX_H = 8192, RING_THREADS = RING_MAX_H / RING_COLS + 32, RING_MAX_STAGES = 8;
constexpr int RING_SMEM = 216 * 1024;  // of an SM, shared by its CTAs

struct RingParams {
  bshmem_norm_args_t a;
  int stages, stage_bytes;
};

// The rows that are copied, in the order of their places in a stage.
struct RingRows {
  int h, residual, dr, dy, gate;  // offsets; -1: absent
  int bytes;
};
__host__ __device__ __forceinline__ int type_bytes(int t) { return t == BSHMEM_NORM_F32 ? 4 : 2; }
__host__ __device__ __forceinline__ RingRows ring_rows(const bshmem_norm_args_t& a, bool backward) {
  RingRows r;
  const int t = a.H * type_bytes(a.type), rt = a.H * type_bytes(a.res_type), wt = a.H * type_bytes(a.wt_type);
  int at = 0;
  auto place = [&](bool present, int bytes) {
    const int here = present ? at : -1;
    if (present) at += bytes;
    return here;
  };
  r.residual = place(true, rt);
  r.h = place(a.h != nullptr, t);
  r.dr = place(backward && a.dr, rt);
  r.dy = place(backward && a.dy, t);
  r.gate = place(a.gate_mode == BSHMEM_NORM_GATE_FULL, wt);
  r.bytes = at;
  return r;
}

struct Ring {
  uint8_t* data;
  uint64_t *full, *empty;
  volatile int* abort_flag;
  int stage;
  uint32_t phase;
};
constexpr uint64_t RING_WAIT_NS = 10000000000ull;  // the waits are for this CTA's own copies and threads

__device__ __forceinline__ Ring ring_setup(const RingParams& p, uint8_t* smem, int consumer_warps) {
  Ring r;
  r.data = smem;
  r.full = (uint64_t*)(smem + (size_t)p.stages * p.stage_bytes);
  r.empty = r.full + RING_MAX_STAGES;
  r.abort_flag = (volatile int*)(r.empty + RING_MAX_STAGES);
  r.stage = 0;
  r.phase = 0;
  if (threadIdx.x == 0) {
    *r.abort_flag = 0;
    for (int i = 0; i < p.stages; ++i) {
      sm100::mbar_init(&r.full[i], 1);
      sm100::mbar_init(&r.empty[i], consumer_warps);
    }
    sm100::mbar_fence_init();
    sm100::fence_proxy_async_smem();
  }
  __syncthreads();
  return r;
}
__device__ __forceinline__ void ring_next(Ring& r, int stages) {
  if (++r.stage == stages) {
    r.stage = 0;
    r.phase ^= 1;
  }
}
// The copying warp: every row of this CTA, as stages become free.
__device__ __forceinline__ void ring_fill(const RingParams& p, Ring& r, bool backward) {
  const bshmem_norm_args_t& a = p.a;
  if (sm100::elect_one()) {
    const RingRows rows = ring_rows(a, backward);
    const size_t ts = type_bytes(a.type), rs = type_bytes(a.res_type), ws = type_bytes(a.wt_type);
    for (size_t row = blockIdx.x; row < (size_t)a.T; row += gridDim.x) {
      if (!sm100::mbar_wait(&r.empty[r.stage], r.phase ^ 1, RING_WAIT_NS, r.abort_flag)) break;
      uint8_t* dst = r.data + (size_t)r.stage * p.stage_bytes;
      uint64_t* bar = &r.full[r.stage];
      sm100::mbar_expect_tx(bar, rows.bytes);
      sm100::bulk_load(dst + rows.residual, (const uint8_t*)a.residual + row * a.res_stride * rs, a.H * rs, bar);
      if (rows.h >= 0) sm100::bulk_load(dst + rows.h, (const uint8_t*)a.h + row * a.h_stride * ts, a.H * ts, bar);
      if (rows.dr >= 0) sm100::bulk_load(dst + rows.dr, (const uint8_t*)a.dr + row * a.dr_stride * rs, a.H * rs, bar);
      if (rows.dy >= 0) sm100::bulk_load(dst + rows.dy, (const uint8_t*)a.dy + row * a.dy_stride * ts, a.H * ts, bar);
      if (rows.gate >= 0) sm100::bulk_load(dst + rows.gate, (const uint8_t*)a.gate + row * a.gate_stride * ws, a.H * ws, bar);
      ring_next(r, p.stages);
    }
  }
  __syncwarp();
}
__device__ __forceinline__ void ring_end(const RingParams& p, const Ring& r) {
  __syncthreads();
  if (!*r.abort_flag) return;
  const uint64_t t0 = sm100::timer_ns();  // copies still in flight land before the shared memory goes away
  while (sm100::timer_ns() - t0 < 200000) __nanosleep(1000);
  if (threadIdx.x == 0) atomicOr(p.a.error_flag, 1);
}

// Sum over the consumer warps (at most 16), the same value in every thread.  `s` alternates between two buffers, so that one
// barrier per sum is enough.
template <int N>
__device__ __forceinline__ void ring_sum(float (&v)[N], float (*s)[N], int warps) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
  if (warps == 1) return;
  if (lane == 0)
#pragma unroll
    for (int i = 0; i < N; ++i) s[warp][i] = v[i];
  sm100::named_bar_sync(1, warps * 32);
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = lane < warps ? s[lane][i] : 0.f;
#pragma unroll
  for (int o = 8; o > 0; o >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = __shfl_sync(0xffffffffu, v[i], 0);
}

// Four neighbouring values: 8 or 16 bytes a thread, so that a warp's accesses to shared memory are free of bank conflicts for
// both sizes of type, and few values are live at a time.
template <typename T>
__device__ __forceinline__ void load4(float* f, const T* row, int col, int H) {
  alignas(16) T raw[4];
  if constexpr (sizeof(T) == 4) *(uint4*)raw = col < H ? *(const uint4*)(row + col) : make_uint4(0u, 0u, 0u, 0u);
  else *(uint2*)raw = col < H ? *(const uint2*)(row + col) : make_uint2(0u, 0u);
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = to_f<T>(raw[i]);
}
template <typename T>
__device__ __forceinline__ void store4(T* row, int col, int H, const float* f) {
  if (col >= H) return;
  alignas(16) T raw[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) raw[i] = from_f<T>(f[i]);
  if constexpr (sizeof(T) == 4) *(uint4*)(row + col) = *(uint4*)raw;
  else *(uint2*)(row + col) = *(uint2*)raw;
}
template <typename T>
__device__ __forceinline__ void load4_wt(float* f, const void* row, bool wide, int col, int H) {
  if (wide) load4<float>(f, (const float*)row, col, H);
  else load4<T>(f, (const T*)row, col, H);
}

// u = branch_scale (post + offset) gate, without the gate where it differs from row to row.
template <typename T>
__device__ __forceinline__ void load_u(float* u, const bshmem_norm_args_t& a, bool wide, int col) {
#pragma unroll
  for (int i = 0; i < 4; ++i) u[i] = 1.f;
  if (a.post) {
    load4_wt<T>(u, a.post, wide, col, a.H);
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] += a.weight_offset;
  }
  if (a.gate_mode == BSHMEM_NORM_GATE_CHANNEL) {
    float g[4];
    load4_wt<T>(g, a.gate, wide, col, a.H);
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] *= g[i];
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) u[i] *= a.branch_scale;
}
__device__ __forceinline__ int ring_col(int c, int threads) { return (c * threads + (int)threadIdx.x) * 4; }

// FULL: the gate is [T][H].
template <typename T, typename R, bool FULL>
__global__ void __launch_bounds__(RING_THREADS, 1) forward_ring_kernel(const __grid_constant__ RingParams p) {
  const bshmem_norm_args_t& a = p.a;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float sums[2][16][1];
  const int threads = blockDim.x - 32, warps = threads >> 5, warp = threadIdx.x >> 5;
  Ring ring = ring_setup(p, smem, warps);
  if (warp == warps) {
    ring_fill(p, ring, false);
  } else {
    const RingRows rows = ring_rows(a, false);
    const bool wide = a.wt_type == BSHMEM_NORM_F32 && sizeof(T) < 4, token = a.gate_mode == BSHMEM_NORM_GATE_TOKEN;
    float u[RING_CH][4], wp[RING_CH][4];
    if (a.h) {
#pragma unroll
      for (int c = 0; c < RING_CH; ++c) load_u<T>(u[c], a, wide, ring_col(c, threads));
    }
    if (a.y) {
#pragma unroll
      for (int c = 0; c < RING_CH; ++c) {
        load4_wt<T>(wp[c], a.pre, wide, ring_col(c, threads), a.H);
#pragma unroll
        for (int i = 0; i < 4; ++i) wp[c][i] += a.weight_offset;
      }
    }
    for (size_t row = blockIdx.x; row < (size_t)a.T; row += gridDim.x) {
      const float tg = token ? load1_wt<T>(a.gate, wide, row) : 1.f;
      sm100::mbar_wait(&ring.full[ring.stage], ring.phase, RING_WAIT_NS, ring.abort_flag);
      const uint8_t* src = ring.data + (size_t)ring.stage * p.stage_bytes;
      float r[RING_CH][4], ss[1];
      if (a.h) {
        float inv = 1.f;
        ss[0] = 0.f;
#pragma unroll
        for (int c = 0; c < RING_CH; ++c) {
          load4<T>(r[c], (const T*)(src + rows.h), ring_col(c, threads), a.H);
#pragma unroll
          for (int i = 0; i < 4; ++i) ss[0] += r[c][i] * r[c][i];
        }
        if (a.post) {
          ring_sum<1>(ss, sums[0], warps);
          inv = rsqrtf(ss[0] / (float)a.H + a.eps);
          if (threadIdx.x == 0 && a.stat) a.stat[row] = inv;
        }
        inv *= tg;
#pragma unroll
        for (int c = 0; c < RING_CH; ++c) {
          float x[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) r[c][i] *= inv * u[c][i];
          if constexpr (FULL) {
            load4_wt<T>(x, src + rows.gate, wide, ring_col(c, threads), a.H);
#pragma unroll
            for (int i = 0; i < 4; ++i) r[c][i] *= x[i];
          }
          load4<R>(x, (const R*)(src + rows.residual), ring_col(c, threads), a.H);
#pragma unroll
          for (int i = 0; i < 4; ++i) r[c][i] += a.residual_scale * x[i];
        }
      } else {
#pragma unroll
        for (int c = 0; c < RING_CH; ++c) {
          load4<R>(r[c], (const R*)(src + rows.residual), ring_col(c, threads), a.H);
#pragma unroll
          for (int i = 0; i < 4; ++i) r[c][i] *= a.residual_scale;
        }
      }
      __syncwarp();
      if ((threadIdx.x & 31) == 0) sm100::mbar_arrive(&ring.empty[ring.stage]);
      ring_next(ring, p.stages);
      if (a.r) {
#pragma unroll
        for (int c = 0; c < RING_CH; ++c) store4<R>((R*)a.r + row * a.H, ring_col(c, threads), a.H, r[c]);
      }
      if (a.y) {
        ss[0] = 0.f;
#pragma unroll
        for (int c = 0; c < RING_CH; ++c)
#pragma unroll
          for (int i = 0; i < 4; ++i) ss[0] += r[c][i] * r[c][i];
        ring_sum<1>(ss, sums[1], warps);
        const float inv = rsqrtf(ss[0] / (float)a.H + a.eps);
        if (threadIdx.x == 0 && a.stat) a.stat[a.T + row] = inv;
#pragma unroll
        for (int c = 0; c < RING_CH; ++c) {
#pragma unroll
          for (int i = 0; i < 4; ++i) r[c][i] *= inv * wp[c][i];
          store4<T>((T*)a.y + row * a.H, ring_col(c, threads), a.H, r[c]);
        }
      }
      // one of the two sums alone would write its buffer again before all have read it
      if (!(a.h && a.post && a.y)) sm100::named_bar_sync(1, threads);
    }
  }
  ring_end(p, ring);
}

// The values are taken from the stage twice, before and after the row's sums, instead of being held in registers.
template <typename T, typename R, bool FULL>
__global__ void __launch_bounds__(RING_THREADS, 1) backward_ring_kernel(const __grid_constant__ RingParams p) {
  const bshmem_norm_args_t& a = p.a;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float sums[2][16][3];
  const int threads = blockDim.x - 32, warps = threads >> 5, warp = threadIdx.x >> 5;
  Ring ring = ring_setup(p, smem, warps);
  if (warp == warps) {
    ring_fill(p, ring, true);
  } else {
    const RingRows rows = ring_rows(a, true);
    const bool wide = a.wt_type == BSHMEM_NORM_F32 && sizeof(T) < 4, token = a.gate_mode == BSHMEM_NORM_GATE_TOKEN;
    float u[RING_CH][4], wp[RING_CH][4], acc_s[RING_CH][4], acc_p[RING_CH][4];
#pragma unroll
    for (int c = 0; c < RING_CH; ++c) {
      if (a.h) load_u<T>(u[c], a, wide, ring_col(c, threads));
      if (a.dy) load4_wt<T>(wp[c], a.pre, wide, ring_col(c, threads), a.H);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        wp[c][i] = a.dy ? wp[c][i] + a.weight_offset : 0.f;
        if (!a.h) u[c][i] = 0.f;
        acc_s[c][i] = acc_p[c][i] = 0.f;
      }
    }
    int buf = 0;
    for (size_t row = blockIdx.x; row < (size_t)a.T; row += gridDim.x) {
      const float tg = token ? load1_wt<T>(a.gate, wide, row) : 1.f;
      const float s1 = a.h && a.post ? a.stat[row] : 1.f, s2 = a.dy ? a.stat[a.T + row] : 0.f;
      sm100::mbar_wait(&ring.full[ring.stage], ring.phase, RING_WAIT_NS, ring.abort_flag);
      const uint8_t* src = ring.data + (size_t)ring.stage * p.stage_bytes;
      // hh = hhat, ge = the row's gate, rh = rhat, dy, g = dr + s2 dy pre of four columns
      auto values = [&](int c, float* hh, float* ge, float* rh, float* dy, float* g) {
        const int col = ring_col(c, threads);
        load4<R>(rh, (const R*)(src + rows.residual), col, a.H);
        if (a.h) load4<T>(hh, (const T*)(src + rows.h), col, a.H);
        if constexpr (FULL) load4_wt<T>(ge, src + rows.gate, wide, col, a.H);
        if (a.dr) load4<R>(g, (const R*)(src + rows.dr), col, a.H);
        if (a.dy) load4<T>(dy, (const T*)(src + rows.dy), col, a.H);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (!FULL) ge[i] = tg;
          hh[i] = a.h ? hh[i] * s1 : 0.f;
          if (!a.dr) g[i] = 0.f;
          if (!a.dy) dy[i] = 0.f;
          rh[i] = s2 * (a.residual_scale * rh[i] + ge[i] * u[c][i] * hh[i]);
          g[i] += s2 * (dy[i] * wp[c][i]);
        }
      };
      float v[3] = {0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < RING_CH; ++c) {
        float hh[4], ge[4], rh[4], dy[4], g[4];
        values(c, hh, ge, rh, dy, g);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float q = u[c][i] * hh[i] * (FULL ? ge[i] : 1.f);   // without a gate per token: see c2
          v[0] += dy[i] * wp[c][i] * rh[i];
          v[1] += q * g[i];
          v[2] += q * rh[i];
        }
      }
      ring_sum<3>(v, sums[buf], warps);
      buf ^= 1;
      const float c1 = s2 * v[0] / (float)a.H, qg = v[1] - c1 * v[2], c2 = a.post ? qg * tg / (float)a.H : 0.f;
      if (token && a.dgate && threadIdx.x == 0) store1_wt<T>(a.dgate, wide, row, qg);
#pragma unroll
      for (int c = 0; c < RING_CH; ++c) {
        const int col = ring_col(c, threads);
        float hh[4], ge[4], rh[4], dy[4], g[4];
        values(c, hh, ge, rh, dy, g);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          g[i] -= c1 * rh[i];
          acc_p[c][i] += dy[i] * rh[i];
          acc_s[c][i] += ge[i] * g[i] * hh[i];
          dy[i] = a.residual_scale * g[i];
        }
        if (a.dresidual) store4<R>((R*)a.dresidual + row * a.H, col, a.H, dy);
        if (a.dh) {
#pragma unroll
          for (int i = 0; i < 4; ++i) dy[i] = s1 * (ge[i] * u[c][i] * g[i] - hh[i] * c2);
          store4<T>((T*)a.dh + row * a.H, col, a.H, dy);
        }
        if (FULL && a.dgate) {
#pragma unroll
          for (int i = 0; i < 4; ++i) dy[i] = g[i] * u[c][i] * hh[i];
          if (wide) store4<float>((float*)a.dgate + row * a.H, col, a.H, dy);
          else store4<T>((T*)a.dgate + row * a.H, col, a.H, dy);
        }
      }
      __syncwarp();
      if ((threadIdx.x & 31) == 0) sm100::mbar_arrive(&ring.empty[ring.stage]);
      ring_next(ring, p.stages);
    }
    if (a.partials) {
#pragma unroll
      for (int c = 0; c < RING_CH; ++c) {
        store4<float>(a.partials + (size_t)blockIdx.x * 2 * a.H, ring_col(c, threads), a.H, acc_s[c]);
        store4<float>(a.partials + ((size_t)blockIdx.x * 2 + 1) * a.H, ring_col(c, threads), a.H, acc_p[c]);
      }
    }
  }
  ring_end(p, ring);
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

// How the ring kernels run a call; `ctas` 0: they do not take it.
struct RingPlan {
  int ctas, threads, stages, stage_bytes, smem;
};
static RingPlan ring_plan(const bshmem_norm_args_t* a, bool backward, bool vec) {
  RingPlan r = {0, 0, 0, 0, 0};
  if (!vec || a->H < 1024 || a->H > RING_MAX_H) return r;
  r.threads = (a->H + RING_COLS * 32 - 1) / (RING_COLS * 32) * 32;
  const int per_sm = r.threads >= 320 ? 1 : 512 / r.threads < 6 ? 512 / r.threads : 6, sms = sm_count();
  r.stage_bytes = ring_rows(*a, backward).bytes;
  const int budget = RING_SMEM / per_sm - 2048;
  r.stages = budget / r.stage_bytes < RING_MAX_STAGES ? budget / r.stage_bytes : RING_MAX_STAGES;
  if (r.stages < 2 || a->T <= 2 * sms) return r;
  r.smem = r.stages * r.stage_bytes + RING_MAX_STAGES * 16 + 16;
  r.threads += 32;
  r.ctas = a->T < sms * per_sm ? a->T : sms * per_sm;
  return r;
}
// Raises a kernel's shared-memory limit to what a ring may take.
static bool reserve_smem(const void* kernel, int bytes) {
  return bytes <= 48 * 1024 || cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) == cudaSuccess;
}

template <typename T, typename R>
static int launch_forward(const Params& p, int chunks, bool vec, cudaStream_t stream) {
  const RingPlan ring = ring_plan(&p.a, false, vec);
  if (ring.ctas) {
    const RingParams rp = {p.a, ring.stages, ring.stage_bytes};
    void (*const kernel)(RingParams) = p.a.gate_mode == BSHMEM_NORM_GATE_FULL ? forward_ring_kernel<T, R, true> : forward_ring_kernel<T, R, false>;
    if (!reserve_smem((const void*)kernel, ring.smem)) return BSHMEM_NORM_ERR_DRIVER;
    kernel<<<ring.ctas, ring.threads, ring.smem, stream>>>(rp);
    return cudaGetLastError() == cudaSuccess ? BSHMEM_NORM_OK : BSHMEM_NORM_ERR_DRIVER;
  }
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
  const RingPlan ring = ring_plan(&p.a, true, vec);
  int grid = ring.ctas;
  if (grid) {
    const RingParams rp = {p.a, ring.stages, ring.stage_bytes};
    void (*const kernel)(RingParams) = p.a.gate_mode == BSHMEM_NORM_GATE_FULL ? backward_ring_kernel<T, R, true> : backward_ring_kernel<T, R, false>;
    if (!reserve_smem((const void*)kernel, ring.smem)) return BSHMEM_NORM_ERR_DRIVER;
    kernel<<<grid, ring.threads, ring.smem, stream>>>(rp);
  } else {
    const int threads = p.group < 128 ? 128 : p.group, groups = threads / p.group, smem = p.a.partials ? groups * 2 * p.a.H * 4 : 0;
    grid = backward_ctas(p.a.T, p.a.H);
    void (*const kernel)(Params) = chunks == 1 ? (vec ? backward_kernel<T, R, 1, true> : backward_kernel<T, R, 1, false>)
                                               : (vec ? backward_kernel<T, R, 2, true> : backward_kernel<T, R, 2, false>);
    if (!reserve_smem((const void*)kernel, smem)) return BSHMEM_NORM_ERR_DRIVER;
    kernel<<<grid, threads, smem, stream>>>(p);
  }
  if (p.a.partials) column_sum_kernel<T><<<dim3((p.a.H + 31) / 32, 2), dim3(32, 8), 0, stream>>>(p, grid);
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

// Parts of at most the CTAs of either backward kernel.
extern "C" size_t bshmem_block_norms_partials(int T, int H) {
  if (T <= 0 || H <= 0) return 0;
  const int most = sm_count() * 6, ctas = backward_ctas(T, H);
  return (size_t)(T < most ? (T > ctas ? T : ctas) : most) * 2 * H;
}

extern "C" int bshmem_block_norms(const bshmem_norm_args_t* a, cudaStream_t stream) {
  if (a && a->T == 0) return BSHMEM_NORM_OK;
  const int st = check(a);
  if (st) return st;
  if ((!a->r && !a->y) || !a->error_flag) return BSHMEM_NORM_ERR_ARGS;
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
  if (!a->error_flag) return BSHMEM_NORM_ERR_ARGS;
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
