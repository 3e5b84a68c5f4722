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
constexpr int SLICES = 32;
template <typename T>
__global__ void __launch_bounds__(32 * SLICES) column_sum_kernel(const __grid_constant__ Params p, int parts) {
  const bshmem_norm_args_t& a = p.a;
  const int i = blockIdx.x * 32 + threadIdx.x;
  const bool pre = blockIdx.y != 0, channel = a.gate_mode == BSHMEM_NORM_GATE_CHANNEL, wide = a.wt_type == BSHMEM_NORM_F32 && sizeof(T) < 4;
  if (pre ? !a.dpre : !a.dpost && !(a.dgate && channel)) return;
  __shared__ float s[SLICES][33];
  float v = 0.f;
  if (i < a.H) {
#pragma unroll 4
    for (int k = threadIdx.y; k < parts; k += SLICES) v += a.partials[((size_t)k * 2 + pre) * a.H + i];
  }
  s[threadIdx.y][threadIdx.x] = v;
  __syncthreads();
  if (threadIdx.y || i >= a.H) return;
#pragma unroll
  for (int k = 1; k < SLICES; ++k) v += s[k][threadIdx.x];
  if (pre) {
    store1_wt<T>(a.dpre, wide, i, v);
    return;
  }
  if (a.dpost) store1_wt<T>(a.dpost, wide, i, a.branch_scale * v * (channel ? load1_wt<T>(a.gate, wide, i) : 1.f));
  if (a.dgate && channel) store1_wt<T>(a.dgate, wide, i, a.branch_scale * v * (a.post ? load1_wt<T>(a.post, wide, i) + a.weight_offset : 1.f));
}

// ------------------------------------------------------------------ rows of up to 8192
// Every thread owns sixteen columns for the whole run, with their parameters and their sums over rows in registers; its CTA (or, up to 512
// columns, its warp) walks rows with the stride of the grid.  512 threads of 128 registers take rows of 8192.
//   STAGED  one thread copies rows (cp.async.bulk, 16-byte aligned) into a ring in shared memory ahead of their use, so that the bytes in
//           flight do not depend on the threads.  (A warp of its own for the copies would leave 96 registers a thread, which spill:
//           backward at 4096 x 8192 took 269 us with it, 128 without.)
//   VECTOR  rows are read where they lie, 8 or 16 bytes at a time: few rows, or rows too large for two stages
//   SCALAR  the same one value at a time, for odd sizes and addresses
enum Mode { STAGED, VECTOR, SCALAR };
constexpr int ROW_CH = 4, ROW_COLS = 4 * ROW_CH, ROW_MAX_H = 8192, ROW_THREADS = ROW_MAX_H / ROW_COLS, MAX_STAGES = 8;
constexpr int WARP_MAX_H = 32 * ROW_COLS, WARP_GROUPS = 8;   // rows of a warp each
constexpr int STAGE_SMEM = 216 * 1024;  // of an SM, shared by its CTAs

struct RowParams {
  bshmem_norm_args_t a;
  int threads;              // per row
  int stages, stage_bytes;  // STAGED
};

// The rows that are copied, in the order of their places in a stage.
struct StageRows {
  int h, residual, dr, dy, gate;  // offsets; -1: absent
  int bytes;
};
__host__ __device__ __forceinline__ int type_bytes(int t) { return t == BSHMEM_NORM_F32 ? 4 : 2; }
__host__ __device__ __forceinline__ StageRows stage_rows(const bshmem_norm_args_t& a, bool backward) {
  StageRows r;
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

// A row's inputs, wherever they are.
struct RowSource {
  const uint8_t *h, *residual, *dr, *dy, *gate;
};

template <Mode MODE>
struct Rows {
  const RowParams& p;
  uint8_t* data = nullptr;
  uint64_t* full = nullptr;
  volatile int* abort_flag = nullptr;
  StageRows at;
  int tid, threads, stage = 0;
  uint32_t phase = 0;
  size_t first, step;

  static constexpr uint64_t WAIT_NS = 10000000000ull;  // the waits are for this CTA's own copies

  // Starts the copy of a row into a stage that nobody reads any more.  One thread.
  __device__ __forceinline__ void load(size_t row, int to) const {
    const RowSource g = global(row);
    const int ts = type_bytes(p.a.type), rs = type_bytes(p.a.res_type), ws = type_bytes(p.a.wt_type), H = p.a.H;
    uint8_t* dst = data + (size_t)to * p.stage_bytes;
    uint64_t* bar = &full[to];
    sm100::mbar_expect_tx(bar, at.bytes);
    sm100::bulk_load(dst + at.residual, g.residual, H * rs, bar);
    if (at.h >= 0) sm100::bulk_load(dst + at.h, g.h, H * ts, bar);
    if (at.dr >= 0) sm100::bulk_load(dst + at.dr, g.dr, H * rs, bar);
    if (at.dy >= 0) sm100::bulk_load(dst + at.dy, g.dy, H * ts, bar);
    if (at.gate >= 0) sm100::bulk_load(dst + at.gate, g.gate, H * ws, bar);
  }
  __device__ __forceinline__ RowSource global(size_t row) const {
    const bshmem_norm_args_t& a = p.a;
    const size_t ts = type_bytes(a.type), rs = type_bytes(a.res_type), ws = type_bytes(a.wt_type);
    RowSource g;
    g.residual = (const uint8_t*)a.residual + row * a.res_stride * rs;
    g.h = (const uint8_t*)a.h + row * a.h_stride * ts;
    g.dr = (const uint8_t*)a.dr + row * a.dr_stride * rs;
    g.dy = (const uint8_t*)a.dy + row * a.dy_stride * ts;
    g.gate = (const uint8_t*)a.gate + row * a.gate_stride * ws;
    return g;
  }
  __device__ __forceinline__ Rows(const RowParams& params, uint8_t* smem, bool backward) : p(params), at(stage_rows(params.a, backward)) {
    threads = p.threads;
    const int groups = blockDim.x / threads;
    tid = threadIdx.x % threads;
    first = (size_t)blockIdx.x * groups + threadIdx.x / threads;
    step = (size_t)gridDim.x * groups;
    if constexpr (MODE == STAGED) {
      data = smem;
      full = (uint64_t*)(smem + (size_t)p.stages * p.stage_bytes);
      abort_flag = (volatile int*)(full + MAX_STAGES);
      if (threadIdx.x == 0) {
        *abort_flag = 0;
        for (int i = 0; i < p.stages; ++i) sm100::mbar_init(&full[i], 1);
        sm100::mbar_fence_init();
        sm100::fence_proxy_async_smem();
        for (int i = 0; i < p.stages; ++i)
          if (first + i * step < (size_t)p.a.T) load(first + i * step, i);
      }
      __syncthreads();
    }
  }
  __device__ __forceinline__ RowSource wait(size_t row) const {
    if constexpr (MODE == STAGED) {
      sm100::mbar_wait(&full[stage], phase, WAIT_NS, abort_flag);
      const uint8_t* s = data + (size_t)stage * p.stage_bytes;
      return {s + at.h, s + at.residual, s + at.dr, s + at.dy, s + at.gate};
    } else {
      return global(row);
    }
  }
  // All threads are past their last look at the stage of `row` (`behind` = 0) or of the row before it (1): it takes the next row that
  // falls to it.
  __device__ __forceinline__ void refill(size_t row, int behind) const {
    if constexpr (MODE == STAGED) {
      const size_t next = row + (size_t)(p.stages - behind) * step;
      if (threadIdx.x == 0 && row >= first + behind * step && next < (size_t)p.a.T) load(next, stage >= behind ? stage - behind : p.stages - 1);
    }
  }
  __device__ __forceinline__ void next() {
    if constexpr (MODE == STAGED) {
      if (++stage == p.stages) {
        stage = 0;
        phase ^= 1;
      }
    }
  }
  __device__ __forceinline__ void end() const {
    if constexpr (MODE == STAGED) {
      __syncthreads();
      if (!*abort_flag) return;
      const uint64_t t0 = sm100::timer_ns();  // copies still in flight land before the shared memory goes away
      while (sm100::timer_ns() - t0 < 200000) __nanosleep(1000);
      if (threadIdx.x == 0) atomicOr(p.a.error_flag, 1);
    }
  }

  // This thread's four columns of chunk c.  With vectors they are neighbours (8 or 16 bytes a thread: a warp's accesses to shared memory
  // are free of bank conflicts for both sizes of type); without, they are a row's threads apart.
  template <typename T>
  __device__ __forceinline__ void load4(float* f, const void* row, int c) const {
    if constexpr (MODE == SCALAR) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int col = (c * 4 + i) * threads + tid;
        f[i] = col < p.a.H ? to_f<T>(((const T*)row)[col]) : 0.f;
      }
    } else {
      const int col = (c * threads + tid) * 4;
      alignas(16) T raw[4];
      if constexpr (sizeof(T) == 4) *(uint4*)raw = col < p.a.H ? *(const uint4*)((const T*)row + col) : make_uint4(0u, 0u, 0u, 0u);
      else *(uint2*)raw = col < p.a.H ? *(const uint2*)((const T*)row + col) : make_uint2(0u, 0u);
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = to_f<T>(raw[i]);
    }
  }
  template <typename T>
  __device__ __forceinline__ void store4(void* row, int c, const float* f) const {
    if constexpr (MODE == SCALAR) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int col = (c * 4 + i) * threads + tid;
        if (col < p.a.H) ((T*)row)[col] = from_f<T>(f[i]);
      }
    } else {
      const int col = (c * threads + tid) * 4;
      if (col >= p.a.H) return;
      alignas(16) T raw[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) raw[i] = from_f<T>(f[i]);
      if constexpr (sizeof(T) == 4) *(uint4*)((T*)row + col) = *(uint4*)raw;
      else *(uint2*)((T*)row + col) = *(uint2*)raw;
    }
  }
  template <typename T>
  __device__ __forceinline__ void load4_wt(float* f, const void* row, bool wide, int c) const {
    if (wide) load4<float>(f, row, c);
    else load4<T>(f, row, c);
  }
  // u = branch_scale (post + offset) gate, without the gate where it differs from row to row.
  template <typename T>
  __device__ __forceinline__ void load_u(float* u, bool wide, int c) const {
    const bshmem_norm_args_t& a = p.a;
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] = 1.f;
    if (a.post) {
      load4_wt<T>(u, a.post, wide, c);
#pragma unroll
      for (int i = 0; i < 4; ++i) u[i] += a.weight_offset;
    }
    if (a.gate_mode == BSHMEM_NORM_GATE_CHANNEL) {
      float g[4];
      load4_wt<T>(g, a.gate, wide, c);
#pragma unroll
      for (int i = 0; i < 4; ++i) u[i] *= g[i];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] *= a.branch_scale;
  }
  // Sum over a row's threads, the same value in every one of them.  One barrier per sum: consecutive sums of a CTA use two
  // buffers in turn.
  template <int N>
  __device__ __forceinline__ void sum(float (&v)[N], float (*s)[N]) const {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
    if (blockDim.x != threads) return;  // a warp's row
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    if (lane == 0)
#pragma unroll
      for (int i = 0; i < N; ++i) s[warp][i] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = lane < warps ? s[lane][i] : 0.f;
#pragma unroll
    for (int o = 8; o > 0; o >>= 1)
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = __shfl_sync(0xffffffffu, v[i], 0);
  }
  __device__ __forceinline__ void barrier() const {
    if (blockDim.x == threads) __syncthreads();
  }
};

// ALL: h, both norms, and a gate per channel or none, as compile-time facts; without it each part is looked up.
template <typename T, typename R, Mode MODE, bool ALL>
__global__ void __launch_bounds__(ROW_THREADS, 1) forward_rows_kernel(const __grid_constant__ RowParams p) {
  const bshmem_norm_args_t& a = p.a;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float sums[2][16][1];
  Rows<MODE> rows(p, smem, false);
  const bool wide = a.wt_type == BSHMEM_NORM_F32 && sizeof(T) < 4;
  const bool token = !ALL && a.gate_mode == BSHMEM_NORM_GATE_TOKEN, full = !ALL && a.gate_mode == BSHMEM_NORM_GATE_FULL;
  const bool has_h = ALL || a.h, has_post = ALL || a.post, has_y = ALL || a.y;
  const float inv_h = 1.f / (float)a.H;
  float u[ROW_CH][4], wp[ROW_CH][4];
#pragma unroll
  for (int c = 0; c < ROW_CH; ++c) {
    if (has_h) rows.template load_u<T>(u[c], wide, c);
    if (has_y) {
      rows.template load4_wt<T>(wp[c], a.pre, wide, c);
#pragma unroll
      for (int i = 0; i < 4; ++i) wp[c][i] += a.weight_offset;
    }
  }
  for (size_t row = rows.first; row < (size_t)a.T; row += rows.step) {
    const float tg = token ? load1_wt<T>(a.gate, wide, row) : 1.f;
    const RowSource src = rows.wait(row);
    float r[ROW_CH][4], ss[1];
    if (has_h) {
      float inv = 1.f;
      ss[0] = 0.f;
#pragma unroll
      for (int c = 0; c < ROW_CH; ++c) {
        rows.template load4<T>(r[c], src.h, c);
#pragma unroll
        for (int i = 0; i < 4; ++i) ss[0] += r[c][i] * r[c][i];
      }
      if (has_post) {
        rows.sum(ss, sums[0]);
        inv = rsqrtf(ss[0] * inv_h + a.eps);
        if (rows.tid == 0 && a.stat) a.stat[row] = inv;
      }
      inv *= tg;
#pragma unroll
      for (int c = 0; c < ROW_CH; ++c) {
        float x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) r[c][i] *= inv * u[c][i];
        if (full) {
          rows.template load4_wt<T>(x, src.gate, wide, c);
#pragma unroll
          for (int i = 0; i < 4; ++i) r[c][i] *= x[i];
        }
        rows.template load4<R>(x, src.residual, c);
#pragma unroll
        for (int i = 0; i < 4; ++i) r[c][i] += a.residual_scale * x[i];
      }
    } else {
#pragma unroll
      for (int c = 0; c < ROW_CH; ++c) {
        rows.template load4<R>(r[c], src.residual, c);
#pragma unroll
        for (int i = 0; i < 4; ++i) r[c][i] *= a.residual_scale;
      }
    }
    if (a.r) {
#pragma unroll
      for (int c = 0; c < ROW_CH; ++c) rows.template store4<R>((R*)a.r + row * a.H, c, r[c]);
    }
    float inv = 0.f;
    if (has_y) {
      ss[0] = 0.f;
#pragma unroll
      for (int c = 0; c < ROW_CH; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) ss[0] += r[c][i] * r[c][i];
      rows.sum(ss, sums[1]);
      inv = rsqrtf(ss[0] * inv_h + a.eps);
      if (rows.tid == 0 && a.stat) a.stat[a.T + row] = inv;
    } else {
      rows.barrier();
    }
    rows.refill(row, 0);  // the barrier of the sum: every thread has taken the row out of its stage
    rows.next();
    if (has_y) {
#pragma unroll
      for (int c = 0; c < ROW_CH; ++c) {
#pragma unroll
        for (int i = 0; i < 4; ++i) r[c][i] *= inv * wp[c][i];
        rows.template store4<T>((T*)a.y + row * a.H, c, r[c]);
      }
      if (!(has_h && has_post)) rows.barrier();  // the one buffer of this sum has been read by all
    }
  }
  rows.end();
}

// The values are taken from the source twice, before and after the row's sums, instead of being held in registers.
// ALL: h, dr, dy, post and a gate per channel or none, as compile-time facts; without it each part is looked up.
template <typename T, typename R, Mode MODE, bool ALL>
__global__ void __launch_bounds__(ROW_THREADS, 1) backward_rows_kernel(const __grid_constant__ RowParams p) {
  const bshmem_norm_args_t& a = p.a;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float sums[2][16][3];
  Rows<MODE> rows(p, smem, true);
  const bool wide = a.wt_type == BSHMEM_NORM_F32 && sizeof(T) < 4;
  const bool token = !ALL && a.gate_mode == BSHMEM_NORM_GATE_TOKEN, full = !ALL && a.gate_mode == BSHMEM_NORM_GATE_FULL;
  const bool has_h = ALL || a.h, has_post = ALL || a.post, has_dr = ALL || a.dr, has_dy = ALL || a.dy;
  const float inv_h = 1.f / (float)a.H;
  float u[ROW_CH][4], wp[ROW_CH][4], acc_s[ROW_CH][4], acc_p[ROW_CH][4];
#pragma unroll
  for (int c = 0; c < ROW_CH; ++c) {
    if (has_h) rows.template load_u<T>(u[c], wide, c);
    if (has_dy) rows.template load4_wt<T>(wp[c], a.pre, wide, c);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      wp[c][i] = has_dy ? wp[c][i] + a.weight_offset : 0.f;
      if (!has_h) u[c][i] = 0.f;
      acc_s[c][i] = acc_p[c][i] = 0.f;
    }
  }
  int buf = 0;
  for (size_t row = rows.first; row < (size_t)a.T; row += rows.step) {
    const float tg = token ? load1_wt<T>(a.gate, wide, row) : 1.f;
    const float s1 = has_h && has_post ? a.stat[row] : 1.f, s2 = has_dy ? a.stat[a.T + row] : 0.f;
    const RowSource src = rows.wait(row);
    // hh = hhat, ge = the row's gate, rh = rhat, dy, g = dr + s2 dy pre of four columns
    auto values = [&](int c, float* hh, float* ge, float* rh, float* dy, float* g) {
      rows.template load4<R>(rh, src.residual, c);
      if (has_h) rows.template load4<T>(hh, src.h, c);
      if (full) rows.template load4_wt<T>(ge, src.gate, wide, c);
      if (has_dr) rows.template load4<R>(g, src.dr, c);
      if (has_dy) rows.template load4<T>(dy, src.dy, c);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (!full) ge[i] = tg;
        hh[i] = has_h ? hh[i] * s1 : 0.f;
        if (!has_dr) g[i] = 0.f;
        if (!has_dy) dy[i] = 0.f;
        rh[i] = s2 * (a.residual_scale * rh[i] + ge[i] * u[c][i] * hh[i]);
        g[i] += s2 * (dy[i] * wp[c][i]);
      }
    };
    float v[3] = {0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < ROW_CH; ++c) {
      float hh[4], ge[4], rh[4], dy[4], g[4];
      values(c, hh, ge, rh, dy, g);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float q = u[c][i] * hh[i] * (full ? ge[i] : 1.f);   // without a gate per token: see c2
        v[0] += dy[i] * wp[c][i] * rh[i];
        v[1] += q * g[i];
        v[2] += q * rh[i];
      }
    }
    rows.sum(v, sums[buf]);
    buf ^= 1;
    rows.refill(row, 1);  // the barrier of the sum: every thread is done with the row before
    const float c1 = s2 * v[0] * inv_h, qg = v[1] - c1 * v[2], c2 = has_post ? qg * tg * inv_h : 0.f;
    if (token && a.dgate && rows.tid == 0) store1_wt<T>(a.dgate, wide, row, qg);
#pragma unroll
    for (int c = 0; c < ROW_CH; ++c) {
      float hh[4], ge[4], rh[4], dy[4], g[4];
      values(c, hh, ge, rh, dy, g);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        g[i] -= c1 * rh[i];
        acc_p[c][i] += dy[i] * rh[i];
        acc_s[c][i] += ge[i] * g[i] * hh[i];
        dy[i] = a.residual_scale * g[i];
      }
      if (a.dresidual) rows.template store4<R>((R*)a.dresidual + row * a.H, c, dy);
      if (a.dh) {
#pragma unroll
        for (int i = 0; i < 4; ++i) dy[i] = s1 * (ge[i] * u[c][i] * g[i] - hh[i] * c2);
        rows.template store4<T>((T*)a.dh + row * a.H, c, dy);
      }
      if (full && a.dgate) {
#pragma unroll
        for (int i = 0; i < 4; ++i) dy[i] = g[i] * u[c][i] * hh[i];
        if (wide) rows.template store4<float>((float*)a.dgate + row * a.H, c, dy);
        else rows.template store4<T>((T*)a.dgate + row * a.H, c, dy);
      }
    }
    rows.next();
  }
  if (a.partials) {
    float* part = a.partials + (size_t)blockIdx.x * 2 * a.H;
    if (MODE == STAGED || blockDim.x == rows.threads) {
#pragma unroll
      for (int c = 0; c < ROW_CH; ++c) {
        rows.template store4<float>(part, c, acc_s[c]);
        rows.template store4<float>(part + a.H, c, acc_p[c]);
      }
    } else {  // the warps' sums, in order
      float* s = (float*)smem;  // [warps][2][H]
      const int warps = blockDim.x >> 5;
#pragma unroll
      for (int c = 0; c < ROW_CH; ++c) {
        rows.template store4<float>(s + (threadIdx.x >> 5) * 2 * a.H, c, acc_s[c]);
        rows.template store4<float>(s + ((threadIdx.x >> 5) * 2 + 1) * a.H, c, acc_p[c]);
      }
      __syncthreads();
      for (int i = threadIdx.x; i < 2 * a.H; i += blockDim.x) {
        float v = 0.f;
        for (int k = 0; k < warps; ++k) v += s[k * 2 * a.H + i];
        part[i] = v;
      }
    }
  }
  rows.end();
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

static int sm_count() {
  int device = 0, sms = 0;
  cudaGetDevice(&device);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
  return sms > 0 ? sms : 1;
}

// How the kernels for rows of up to 8192 run a call; `ctas` 0: they do not take it.
struct RowPlan {
  Mode mode;
  int ctas, block, threads, stages, stage_bytes, smem;
};
static RowPlan row_plan(const bshmem_norm_args_t* a, bool backward, bool vec) {
  RowPlan r = {vec ? VECTOR : SCALAR, 0, 0, 0, 0, 0, 0};
  if (a->H > ROW_MAX_H) return r;
  const int sms = sm_count();
  r.threads = (a->H + ROW_COLS * 32 - 1) / (ROW_COLS * 32) * 32;
  if (a->H <= WARP_MAX_H) {
    r.block = 32 * WARP_GROUPS;
    r.smem = backward && a->partials ? WARP_GROUPS * 2 * a->H * 4 : 0;
  } else {
    r.block = r.threads;
  }
  int per_sm = ROW_THREADS / r.block;
  if (vec && a->H > WARP_MAX_H && a->T > sms * per_sm) {
    // Two stages at least; rather fewer CTAs of an SM than none.
    r.stage_bytes = stage_rows(*a, backward).bytes;
    for (int n = per_sm < 6 ? per_sm : 6; n > 0; --n) {
      const int fit = (STAGE_SMEM / n - 2048) / r.stage_bytes;
      if (fit < 2) continue;
      r.mode = STAGED;
      r.stages = fit < MAX_STAGES ? fit : MAX_STAGES;
      r.smem = r.stages * r.stage_bytes + MAX_STAGES * 8 + 16;
      per_sm = n;
      break;
    }
  }
  const int groups = r.block / r.threads, want = (int)(((int64_t)a->T + groups - 1) / groups);
  r.ctas = want < sms * per_sm ? want : sms * per_sm;
  return r;
}
static bool plain_gate(const bshmem_norm_args_t& a) { return a.gate_mode == BSHMEM_NORM_GATE_NONE || a.gate_mode == BSHMEM_NORM_GATE_CHANNEL; }
// Raises a kernel's shared-memory limit to what it may take.
static bool reserve_smem(const void* kernel, int bytes) {
  return bytes <= 48 * 1024 || cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) == cudaSuccess;
}
static int long_row_ctas(int T) {
  const int sms = sm_count();
  return T < sms ? T : sms;
}

template <typename T, typename R>
static int launch_forward(const bshmem_norm_args_t* a, cudaStream_t stream) {
  const bool vec = vectors(a);
  const RowPlan plan = row_plan(a, false, vec);
  if (plan.ctas) {
    const RowParams p = {*a, plan.threads, plan.stages, plan.stage_bytes};
    const bool all = plan.mode == STAGED && plain_gate(*a) && a->post && a->y;
    void (*const kernel)(RowParams) = all ? forward_rows_kernel<T, R, STAGED, true> : plan.mode == STAGED ? forward_rows_kernel<T, R, STAGED, false>
                                      : plan.mode == VECTOR ? forward_rows_kernel<T, R, VECTOR, false> : forward_rows_kernel<T, R, SCALAR, false>;
    if (!reserve_smem((const void*)kernel, plan.smem)) return BSHMEM_NORM_ERR_DRIVER;
    kernel<<<plan.ctas, plan.block, plan.smem, stream>>>(p);
  } else {
    const Params p = {*a, MAX_THREADS};
    if (vec) forward_kernel<T, R, 2, true><<<a->T, MAX_THREADS, 0, stream>>>(p);
    else forward_kernel<T, R, 2, false><<<a->T, MAX_THREADS, 0, stream>>>(p);
  }
  return cudaGetLastError() == cudaSuccess ? BSHMEM_NORM_OK : BSHMEM_NORM_ERR_DRIVER;
}

template <typename T, typename R>
static int launch_backward(const bshmem_norm_args_t* a, cudaStream_t stream) {
  const bool vec = vectors(a);
  const RowPlan plan = row_plan(a, true, vec);
  const Params long_row = {*a, MAX_THREADS};
  int parts = plan.ctas;
  if (plan.ctas) {
    const RowParams p = {*a, plan.threads, plan.stages, plan.stage_bytes};
    const bool all = plan.mode == STAGED && plain_gate(*a) && a->post && a->dr && a->dy;
    void (*const kernel)(RowParams) = all ? backward_rows_kernel<T, R, STAGED, true> : plan.mode == STAGED ? backward_rows_kernel<T, R, STAGED, false>
                                      : plan.mode == VECTOR ? backward_rows_kernel<T, R, VECTOR, false> : backward_rows_kernel<T, R, SCALAR, false>;
    if (!reserve_smem((const void*)kernel, plan.smem)) return BSHMEM_NORM_ERR_DRIVER;
    kernel<<<plan.ctas, plan.block, plan.smem, stream>>>(p);
  } else {
    parts = long_row_ctas(a->T);
    const int smem = a->partials ? 2 * a->H * 4 : 0;
    void (*const kernel)(Params) = vec ? backward_kernel<T, R, 2, true> : backward_kernel<T, R, 2, false>;
    if (!reserve_smem((const void*)kernel, smem)) return BSHMEM_NORM_ERR_DRIVER;
    kernel<<<parts, MAX_THREADS, smem, stream>>>(long_row);
  }
  if (a->partials) column_sum_kernel<T><<<dim3((a->H + 31) / 32, 2), dim3(32, SLICES), 0, stream>>>(long_row, parts);
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

// One part per CTA, of whichever kernel takes the call.
extern "C" size_t bshmem_block_norms_partials(int T, int H) {
  if (T <= 0 || H <= 0) return 0;
  const int most = sm_count() * (ROW_THREADS / 64);
  return (size_t)(T < most ? T : most) * 2 * H;
}

extern "C" int bshmem_block_norms(const bshmem_norm_args_t* a, cudaStream_t stream) {
  if (a && a->T == 0) return BSHMEM_NORM_OK;
  const int st = check(a);
  if (st) return st;
  if ((!a->r && !a->y) || !a->error_flag) return BSHMEM_NORM_ERR_ARGS;
  return by_type(a, [&](auto* t, auto* r) { return launch_forward<std::remove_pointer_t<decltype(t)>, std::remove_pointer_t<decltype(r)>>(a, stream); });
}

extern "C" int bshmem_block_norms_backward(const bshmem_norm_args_t* a, cudaStream_t stream) {
  if (a && a->T == 0) return BSHMEM_NORM_OK;
  const int st = check(a);
  if (st) return st;
  if (!a->error_flag) return BSHMEM_NORM_ERR_ARGS;
  const bool sums = a->dpost || a->dpre || (a->dgate && a->gate_mode == BSHMEM_NORM_GATE_CHANNEL);
  if ((!a->dr && !a->dy) || (a->dpre && !a->dy) || (a->dpost && !a->post) || ((a->dh || a->dgate) && !a->h) || (a->dgate && !a->gate_mode)) return BSHMEM_NORM_ERR_ARGS;
  if ((sums && !a->partials) || ((a->post || a->dy) && !a->stat)) return BSHMEM_NORM_ERR_ARGS;
  bshmem_norm_args_t args = *a;
  if (!sums) args.partials = nullptr;
  return by_type(a, [&](auto* t, auto* r) { return launch_backward<std::remove_pointer_t<decltype(t)>, std::remove_pointer_t<decltype(r)>>(&args, stream); });
}
