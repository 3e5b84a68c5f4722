// Kernels of the norms around a block; norms_{bf16,f16,f32}.cu instantiate them, norms.cu checks calls and picks a type.
//
// Every thread owns sixteen columns for the whole run, with their parameters and their sums over rows in registers; its CTA (up to 512
// columns its warp, above 8192 its pair of CTAs, half a row each) walks rows with the stride of the grid.  512 threads of 128 registers
// take 8192 columns.  Each input is read once from memory and each output written once.
//   STAGED  threads of the first warps copy rows (cp.async.bulk, 16-byte aligned) into a ring in shared memory ahead of their use, so that
//           the bytes in flight do not depend on the threads.  (A warp of its own for the copies would leave 96 registers a thread, which
//           spill: backward at 4096 x 8192 took 269 us with it, 119 without, before the steps that followed.)
//   EARLY   the same, but a stage is filled again as soon as all warps have left it, not at the barrier of the next row (backward)
//   VECTOR  rows are read where they lie, 8 or 16 bytes at a time: few rows, or rows too large for two stages
//   SCALAR  the same one value at a time, for odd sizes and addresses
//
// Backward.  With hhat = h s1, rhat = r s2 (s1, s2 from forward), u = branch_scale post, q = gate u hhat:
//   c1 = mean(dy pre rhat)     G = dr + s2 (dy pre - rhat c1)          gradient of r
//   dresidual = residual_scale G      dgate = G u hhat
//   dh = s1 (gate u G - hhat c2),  c2 = mean(q G) = mean(q (dr + s2 dy pre)) - c1 s2 mean(q rhat)
//   dpost = branch_scale sum over rows of gate G hhat     dpre = sum of dy rhat
// c2 is linear in G, so one reduction of three sums serves a row.  (For a gate per token the sums are taken without the gate:
// they are its gradient.)  Where the gate is per channel it is the same for every row, and one sum S = sum of G hhat gives both
// dpost = branch_scale gate S and dgate = u S.  A CTA keeps its part of the two sums over rows; a second kernel adds the CTAs' parts
// in order.
//
// Bound by memory, and behind it by the instructions and the one barrier of a row.  4096 x 8192, kernel times (bytes over time): forward bf16 46 us
// (5.8 TB/s), with an fp32 residual 67 (6.0); backward 70 (5.8) and 96 (6.3), the sums over rows 5 more.  Few rows: 8 x 7168 forward 3.2 us,
// 777 x 1001 fp16 4.2 and 8.9 + 6.  Pairs: 2000 x 16384 bf16 63 and 98.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>
#include <type_traits>

#include "../../include/bshmem/norms.h"
#include "../../include/bshmem/tcgen05.cuh"

namespace bshmem {
namespace norms {

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

// Two values of a 16-bit type that share a word.
template <typename T>
__device__ __forceinline__ void pair(float* f, uint32_t word) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    f[0] = __uint_as_float(word << 16);
    f[1] = __uint_as_float(word & 0xffff0000u);
  } else {
    const float2 v = __half22float2(*(const __half2*)&word);
    f[0] = v.x, f[1] = v.y;
  }
}
// Element i of a parameter of type W.
template <typename W>
__device__ __forceinline__ float load1(const void* p, size_t i) {
  return to_f<W>(((const W*)p)[i]);
}
template <typename W>
__device__ __forceinline__ void store1(void* p, size_t i, float v) {
  ((W*)p)[i] = from_f<W>(v);
}

enum Mode { STAGED, EARLY, VECTOR, SCALAR };
__host__ __device__ constexpr bool staged(Mode m) { return m == STAGED || m == EARLY; }
// What a kernel knows of its calls at compile time, besides a multiple of 512 columns (every warp has all of its own):
//   BOTH  h, both norms, a gate per channel or none (backward: both gradients)
//   IN    no h: the norm of a row alone      OUT  h, the norm after it, no norm that follows, any gate but [T][H]
//   ANY   nothing; each part is looked up, and columns are guarded
enum Kind { ANY, BOTH, IN, OUT };
// CTAs of 512 threads an SM: two sums and two parameters a column need 128 registers a thread, one of each 64.
constexpr int ctas_per_sm(Kind kind) { return kind == IN || kind == OUT ? 2 : 1; }
constexpr int ROW_CH = 4, ROW_COLS = 4 * ROW_CH, CTA_COLS = 8192, ROW_THREADS = CTA_COLS / ROW_COLS, MAX_STAGES = 8;
constexpr int MAX_CTAS_PER_SM = 8;
constexpr int WARP_COLS = 32 * ROW_COLS, WARP_GROUPS = 8;   // rows of a warp each
constexpr int STAGE_SMEM = 216 * 1024;  // of an SM, shared by its CTAs
constexpr int SUM_ROWS = 17;            // 16 warps, and the other CTA of a pair
constexpr int OWN_SMEM = 2 * SUM_ROWS * 4 * sizeof(float), DEFAULT_SMEM = 48 * 1024;  // a kernel's arrays for sums at most; what a launch gets of both without asking
static_assert(BSHMEM_NORM_MAX_H == 2 * CTA_COLS, "a pair of CTAs takes the longest row");

struct RowParams {
  bshmem_norm_args_t a;
  int threads;              // per row and CTA
  int half;                 // columns of the first CTA of a pair; 0: no pairs
  int stages, stage_bytes;  // STAGED
};

// The parts of a row that are copied, in the order of their places in a stage.
struct StageRows {
  int h, residual, dr, dy, gate;  // offsets; -1: absent
  int bytes;
};
__host__ __device__ __forceinline__ int type_bytes(int t) { return t == BSHMEM_NORM_F32 ? 4 : 2; }
__host__ __device__ __forceinline__ StageRows stage_rows(const bshmem_norm_args_t& a, int cols, bool backward, Kind kind) {
  StageRows r;
  const int t = cols * type_bytes(a.type), rt = cols * type_bytes(a.res_type), wt = cols * type_bytes(a.wt_type);
  int at = 0;
  auto place = [&](bool present, int bytes) {
    const int here = present ? at : -1;
    if (present) at += bytes;
    return here;
  };
  r.residual = place(!(backward && kind == OUT), rt);  // of no use to it
  r.h = place(a.h != nullptr, t);
  r.dr = place(backward && a.dr, rt);
  r.dy = place(backward && a.dy, t);
  r.gate = place(a.gate_mode == BSHMEM_NORM_GATE_FULL, wt);
  r.bytes = at;
  return r;
}

// This CTA's columns of a row's inputs, wherever they are.  Rows that are absent are read from the residual's place (it is at least as
// long) and their values dropped, which takes no branch.
struct RowSource {
  const uint8_t *h, *residual, *dr, *dy, *gate;
};

template <Mode MODE, Kind KIND>
struct Rows {
  static constexpr bool EVEN = KIND != ANY;  // whole warps of columns: nothing to guard
  const RowParams& p;
  uint8_t* data = nullptr;
  uint64_t *full = nullptr, *empty = nullptr;
  volatile int* abort_flag = nullptr;
  StageRows at;
  int tid, threads, base, cols, stage = 0;  // base, cols: this CTA's columns
  uint32_t phase = 0, copies = 0;  // copies: the parts of a row that this thread copies, by number
  uint32_t first, step;  // rows are below 2^31, and what is added to them far below

  static constexpr uint32_t ARRIVE = 1u << 31;   // of one thread
  static constexpr uint64_t WAIT_NS = 10000000000ull;  // the waits are for this CTA's own copies

  __device__ __forceinline__ RowSource global(uint32_t row) const {
    const bshmem_norm_args_t& a = p.a;
    const size_t ts = type_bytes(a.type), rs = type_bytes(a.res_type), ws = type_bytes(a.wt_type);
    RowSource g;
    g.residual = (const uint8_t*)a.residual + (row * a.res_stride + base) * rs;
    g.h = a.h ? (const uint8_t*)a.h + (row * a.h_stride + base) * ts : g.residual;
    g.dr = a.dr ? (const uint8_t*)a.dr + (row * a.dr_stride + base) * rs : g.residual;
    g.dy = a.dy ? (const uint8_t*)a.dy + (row * a.dy_stride + base) * ts : g.residual;
    g.gate = (const uint8_t*)a.gate + (row * a.gate_stride + base) * ws;
    return g;
  }
  // Starts this thread's share of the copy of a row into a stage that nobody reads any more.  Only the addresses that it needs are formed:
  // its warp issues whatever one of its lanes does.
  __device__ __forceinline__ void load(uint32_t row, int to) const {
    uint8_t* dst = data + (size_t)to * p.stage_bytes;
    uint64_t* bar = &full[to];
    auto copy = [&](int number, int offset, const void* rows, int64_t stride, int bytes) {
      if (copies >> number & 1) sm100::bulk_load(dst + offset, (const uint8_t*)rows + (row * stride + base) * bytes, cols * bytes, bar);
    };
    const bshmem_norm_args_t& a = p.a;
    const int ts = type_bytes(a.type), rs = type_bytes(a.res_type), ws = type_bytes(a.wt_type);
    if (copies & ARRIVE) sm100::mbar_expect_tx(bar, at.bytes);  // the phase ends when this has arrived and the bytes of all copies are in
    copy(0, at.residual, a.residual, a.res_stride, rs);
    copy(1, at.h, a.h, a.h_stride, ts);
    copy(2, at.dr, a.dr, a.dr_stride, rs);
    copy(3, at.dy, a.dy, a.dy_stride, ts);
    copy(4, at.gate, a.gate, a.gate_stride, ws);
  }
  __device__ __forceinline__ Rows(const RowParams& params, uint8_t* smem, bool backward) : p(params) {
    const int pair = p.half ? 2 : 1, rank = p.half ? blockIdx.x & 1 : 0, groups = blockDim.x / p.threads;
    threads = p.threads;
    base = rank ? p.half : 0;
    cols = !p.half ? p.a.H : rank ? p.a.H - p.half : p.half;
    at = stage_rows(p.a, cols, backward, KIND);
    tid = threadIdx.x % threads;
    first = (blockIdx.x / pair) * groups + threadIdx.x / threads;
    step = (gridDim.x / pair) * groups;
    if constexpr (staged(MODE)) {
      data = smem;
      full = (uint64_t*)(smem + (size_t)p.stages * p.stage_bytes);
      empty = full + MAX_STAGES;
      abort_flag = (volatile int*)(empty + MAX_STAGES);
      if (threadIdx.x == 0) {
        *abort_flag = 0;
        for (int i = 0; i < p.stages; ++i) {
          sm100::mbar_init(&full[i], 1);
          sm100::mbar_init(&empty[i], blockDim.x >> 5);
        }
        sm100::mbar_fence_init();
        sm100::fence_proxy_async_smem();
      }
      __syncthreads();
      // One thread of each of the first five warps (of all, if there are fewer), so that no warp is held up by all the copies.
      if ((threadIdx.x & 31) == 0) {
        const int warp = threadIdx.x >> 5, warps = blockDim.x >> 5, offsets[5] = {at.residual, at.h, at.dr, at.dy, at.gate};
#pragma unroll
        for (int i = 0; i < 5; ++i)
          if (offsets[i] >= 0 && i % warps == warp) copies |= 1u << i;
        if (warp == 0) copies |= ARRIVE;
      }
      if (copies)
        for (int i = 0; i < p.stages; ++i)
          if (first + i * step < (uint32_t)p.a.T) load(first + i * step, i);
    }
    if (p.half) sm100::cluster_sync_all();  // the other CTA runs: its shared memory may be written
  }
  __device__ __forceinline__ RowSource wait(uint32_t row) const {
    if constexpr (staged(MODE)) {
      sm100::mbar_wait(&full[stage], phase, WAIT_NS, abort_flag);
      const uint8_t* s = data + (size_t)stage * p.stage_bytes;
      return {s + max(at.h, 0), s + max(at.residual, 0), s + max(at.dr, 0), s + max(at.dy, 0), s + at.gate};
    } else {
      return global(row);
    }
  }
  // All threads are past their last look at `row`, which was in `its_stage`: the stage takes the next row that falls to it.
  __device__ __forceinline__ void refill(uint32_t row, int its_stage) const {
    if constexpr (staged(MODE)) {
      const uint32_t next = row + p.stages * step;
      if (copies && next < (uint32_t)p.a.T) load(next, its_stage);
    }
  }
  // The same without a barrier (EARLY): a warp says that it is past its last look at the current row, and the threads that copy wait
  // for all to have said so of the row before this one a little later, when that is hardly a wait.
  __device__ __forceinline__ void release() const {
    if constexpr (MODE == EARLY) {
      __syncwarp();
      if ((threadIdx.x & 31) == 0) sm100::mbar_arrive(&empty[stage]);
    }
  }
  __device__ __forceinline__ void refill_before(uint32_t row) const {
    if constexpr (MODE == EARLY) {
      const uint32_t next = row + (p.stages - 1) * step;
      if (copies && row != first && next < (uint32_t)p.a.T) {
        const int its_stage = stage ? stage - 1 : p.stages - 1;
        sm100::mbar_wait(&empty[its_stage], stage ? phase : phase ^ 1, WAIT_NS, abort_flag);
        load(next, its_stage);
      }
    }
  }
  __device__ __forceinline__ void next() {
    if constexpr (staged(MODE)) {
      if (++stage == p.stages) {
        stage = 0;
        phase ^= 1;
      }
    }
  }
  __device__ __forceinline__ void end() const {
    if constexpr (staged(MODE)) {
      __syncthreads();
      if (!*abort_flag) return;
      const uint64_t t0 = sm100::timer_ns();  // copies still in flight land before the shared memory goes away
      while (sm100::timer_ns() - t0 < 200000) __nanosleep(1000);
      if (threadIdx.x == 0) atomicOr(p.a.error_flag, 1);
    }
  }

  // This thread's four columns of chunk c, of the 512 neighbouring ones of its warp.  With vectors they are neighbours (8 or 16 bytes a
  // thread: a warp's accesses to shared memory are free of bank conflicts for both sizes of type); without, they are 32 apart.
  __device__ __forceinline__ int col(int c, int i) const {
    const int lane = tid & 31, warp_first = (tid >> 5) * WARP_COLS;
    return MODE == SCALAR ? warp_first + lane + (c * 4 + i) * 32 : warp_first + lane * 4 + c * 128 + i;
  }
  template <typename T>
  __device__ __forceinline__ void load4(float* f, const void* row, int c) const {
    if constexpr (MODE == SCALAR) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        f[i] = EVEN || col(c, i) < cols ? to_f<T>(((const T*)row)[col(c, i)]) : 0.f;
      }
    } else {
      const int at = col(c, 0);
      if constexpr (sizeof(T) == 4) {
        const float4 raw = EVEN || at < cols ? *(const float4*)((const T*)row + at) : make_float4(0.f, 0.f, 0.f, 0.f);
        f[0] = raw.x, f[1] = raw.y, f[2] = raw.z, f[3] = raw.w;
      } else {
        const uint2 raw = EVEN || at < cols ? *(const uint2*)((const T*)row + at) : make_uint2(0u, 0u);
        pair<T>(f, raw.x);
        pair<T>(f + 2, raw.y);
      }
    }
  }
  template <typename T>
  __device__ __forceinline__ void store4(T* row, int c, const float* f) const {
    if constexpr (MODE == SCALAR) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (col(c, i) < cols) row[col(c, i)] = from_f<T>(f[i]);
      }
    } else {
      const int at = col(c, 0);
      if (!EVEN && at >= cols) return;
      alignas(16) T raw[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) raw[i] = from_f<T>(f[i]);
      if constexpr (sizeof(T) == 4) *(uint4*)(row + at) = *(uint4*)raw;
      else *(uint2*)(row + at) = *(uint2*)raw;
    }
  }
  // This CTA's part of a parameter, and of a row of a dense output.
  template <typename W>
  __device__ __forceinline__ const W* mine(const void* parameter) const { return (const W*)parameter + base; }
  template <typename T>
  __device__ __forceinline__ T* out(void* rows, uint32_t row) const { return (T*)rows + (size_t)row * p.a.H + base; }

  // u = branch_scale (post + offset) gate, without the gate where it differs from row to row.  The loads do not hang on one another.
  template <typename W>
  __device__ __forceinline__ void load_u(float* u, int c, bool has_post) const {
    const bshmem_norm_args_t& a = p.a;
    const bool channel = a.gate_mode == BSHMEM_NORM_GATE_CHANNEL;
    float g[4];
    if (has_post) {
      load4<W>(u, mine<W>(a.post), c);
      load4<W>(g, mine<W>(channel ? a.gate : a.post), c);
    } else if (channel) {
      load4<W>(g, mine<W>(a.gate), c);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] = (has_post ? u[i] + a.weight_offset : 1.f) * (channel ? g[i] : 1.f) * a.branch_scale;
  }
  // Sums over a row's threads, the same values in every one of them.  One barrier per sum: consecutive sums use two buffers in turn.
  // Two to four values: a lane gives away half of what it holds at each of the first exchanges, so that 6 shuffles do what 5 a value would; a
  // lane then holds value `lane % PLACES`, its bits the other way round.
  template <int N>
  static constexpr int PLACES = N == 1 ? 1 : N == 2 ? 2 : 4;
  template <int N>
  __device__ __forceinline__ void sum(float (&v)[N], float (*s)[PLACES<N>]) const {
    static_assert(N <= 4, "places");
    constexpr int P = PLACES<N>;
    const int lane = threadIdx.x & 31;
    auto exchange = [&](float keep_low, float keep_high, int bit) {  // the sum of what the lanes with (without) the bit keep
      const bool high = lane & bit;
      return (high ? keep_high : keep_low) + __shfl_xor_sync(0xffffffffu, high ? keep_low : keep_high, bit);
    };
    float x = v[0];
    if constexpr (P == 2) x = exchange(v[0], v[1], 1);
    if constexpr (P == 4) {
      float y[2];
      y[0] = exchange(v[0], v[2], 1);
      y[1] = N == 4 ? exchange(v[1], v[N - 1], 1) : exchange(v[1], 0.f, 1);
      x = exchange(y[0], y[1], 2);
    }
#pragma unroll
    for (int o = P; o < 32; o *= 2) x += __shfl_xor_sync(0xffffffffu, x, o);
    auto lane_of = [](int i) { return P == 4 ? (i >> 1) + (i & 1) * 2 : i; };
    if (blockDim.x != threads) {  // a warp's row
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = __shfl_sync(0xffffffffu, x, lane_of(i));
      return;
    }
    const int warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    if (lane < P) s[warp][lane] = x;
    __syncthreads();
    x = 0.f;
#pragma unroll
    for (int w = 0; w < ROW_THREADS / 32; w += 32 / P) {
      const int from = w + lane / P;
      if (from < warps) x += s[from][lane % P];
    }
#pragma unroll
    for (int o = P; o < 32; o *= 2) x += __shfl_xor_sync(0xffffffffu, x, o);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = __shfl_sync(0xffffffffu, x, lane_of(i));
    if (!p.half) return;
    if (threadIdx.x == 0) {  // to the other CTA
      const uint32_t other = sm100::mapa_u32(sm100::smem_u32(&s[SUM_ROWS - 1][0]), (sm100::cluster_ctarank() ^ 1));
#pragma unroll
      for (int i = 0; i < N; ++i) asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(other + 4 * i), "f"(v[i]) : "memory");
    }
    sm100::cluster_sync_all();
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += s[SUM_ROWS - 1][i];
  }
};

template <typename T, typename R, typename W, Mode MODE, Kind KIND>
__global__ void __launch_bounds__(ROW_THREADS, ctas_per_sm(KIND)) forward_rows_kernel(const __grid_constant__ RowParams p) {
  const bshmem_norm_args_t& a = p.a;
  extern __shared__ __align__(128) uint8_t smem[];
  constexpr int SUMS = staged(MODE) && KIND == BOTH ? 2 : 1;
  __shared__ float sums[2][SUM_ROWS][SUMS];
  static_assert(sizeof(sums) <= OWN_SMEM, "see launch");
  Rows<MODE, KIND> rows(p, smem, false);
  const bool token = (KIND == ANY || KIND == OUT) && a.gate_mode == BSHMEM_NORM_GATE_TOKEN, full = KIND == ANY && a.gate_mode == BSHMEM_NORM_GATE_FULL;
  const bool has_h = KIND == ANY ? a.h != nullptr : KIND != IN, has_post = KIND == ANY ? a.post != nullptr : KIND != IN, has_y = KIND == ANY ? a.y != nullptr : KIND != OUT;
  const float inv_h = 1.f / (float)a.H;
  float u[ROW_CH][4], wp[ROW_CH][4];
#pragma unroll
  for (int c = 0; c < ROW_CH; ++c) {
    if (has_h) rows.template load_u<W>(u[c], c, has_post);
    if (has_y) {
      rows.template load4<W>(wp[c], rows.template mine<W>(a.pre), c);
#pragma unroll
      for (int i = 0; i < 4; ++i) wp[c][i] += a.weight_offset;
    }
  }
  if constexpr (staged(MODE) && KIND == BOTH) {
    // One barrier a row: the sum of squares of the next row's h goes together with the one of this row's r.
    auto squares = [&](const RowSource& src) {
      float sum = 0.f;
#pragma unroll
      for (int c = 0; c < ROW_CH; ++c) {
        float h[4];
        rows.template load4<T>(h, src.h, c);
#pragma unroll
        for (int i = 0; i < 4; ++i) sum += h[i] * h[i];
      }
      return sum;
    };
    int buf = 1;
    RowSource src = rows.wait(rows.first);   // there are more rows than CTAs
    float v[2] = {squares(src), 0.f};
    rows.sum(v, sums[0]);
    for (uint32_t row = rows.first; row < (uint32_t)a.T; row += rows.step) {
      const float inv = rsqrtf(v[0] * inv_h + a.eps);
      float r[ROW_CH][4];
      v[0] = v[1] = 0.f;
#pragma unroll
      for (int c = 0; c < ROW_CH; ++c) {
        float x[4];
        rows.template load4<T>(r[c], src.h, c);
        rows.template load4<R>(x, src.residual, c);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          r[c][i] = r[c][i] * inv * u[c][i] + a.residual_scale * x[i];
          v[1] += r[c][i] * r[c][i];
        }
        rows.store4(rows.template out<R>(a.r, row), c, r[c]);
      }
      const int stage = rows.stage;
      rows.next();
      if (row + rows.step < (uint32_t)a.T) {
        src = rows.wait(row + rows.step);
        v[0] = squares(src);
      }
      rows.sum(v, sums[buf]);
      buf ^= 1;
      rows.refill(row, stage);  // after a barrier: every thread has taken the row out of its stage
      const float inv_r = rsqrtf(v[1] * inv_h + a.eps);
      if (rows.tid == 0 && a.stat) {
        a.stat[row] = inv;
        a.stat[a.T + row] = inv_r;
      }
#pragma unroll
      for (int c = 0; c < ROW_CH; ++c) {
#pragma unroll
        for (int i = 0; i < 4; ++i) r[c][i] *= inv_r * wp[c][i];
        rows.store4(rows.template out<T>(a.y, row), c, r[c]);
      }
    }
    rows.end();
    return;
  }
  int buf = 0;
  for (uint32_t row = rows.first; row < (uint32_t)a.T; row += rows.step) {
    const float tg = token ? load1<W>(a.gate, row) : 1.f;
    const RowSource src = rows.wait(row);
    float r[ROW_CH][4], ss[SUMS] = {};
    if (has_h) {
      float inv = 1.f, res[staged(MODE) ? 1 : ROW_CH][4];
      ss[0] = 0.f;
#pragma unroll
      for (int c = 0; c < ROW_CH; ++c) {
        rows.template load4<T>(r[c], src.h, c);
        if constexpr (!staged(MODE)) rows.template load4<R>(res[c], src.residual, c);  // on the way during the sum
      }
#pragma unroll
      for (int c = 0; c < ROW_CH; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) ss[0] += r[c][i] * r[c][i];
      if (has_post) {
        rows.sum(ss, sums[buf]);
        buf ^= 1;
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
          rows.template load4<W>(x, src.gate, c);
#pragma unroll
          for (int i = 0; i < 4; ++i) r[c][i] *= x[i];
        }
        if constexpr (staged(MODE)) rows.template load4<R>(x, src.residual, c);
#pragma unroll
        for (int i = 0; i < 4; ++i) r[c][i] += a.residual_scale * (staged(MODE) ? x[i] : res[staged(MODE) ? 0 : c][i]);
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
      for (int c = 0; c < ROW_CH; ++c) rows.store4(rows.template out<R>(a.r, row), c, r[c]);
    }
    float inv = 0.f;
    if (has_y) {
      ss[0] = 0.f;
#pragma unroll
      for (int c = 0; c < ROW_CH; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) ss[0] += r[c][i] * r[c][i];
      rows.sum(ss, sums[buf]);
      buf ^= 1;
      inv = rsqrtf(ss[0] * inv_h + a.eps);
      if (rows.tid == 0 && a.stat) a.stat[a.T + row] = inv;
    } else if (staged(MODE)) {
      __syncthreads();
    }
    rows.refill(row, rows.stage);  // after a barrier: every thread has taken the row out of its stage
    rows.next();
    if (has_y) {
#pragma unroll
      for (int c = 0; c < ROW_CH; ++c) {
#pragma unroll
        for (int i = 0; i < 4; ++i) r[c][i] *= inv * wp[c][i];
        rows.store4(rows.template out<T>(a.y, row), c, r[c]);
      }
    }
  }
  rows.end();
}

// The values are taken from the source twice, before and after the row's sums, instead of being held in registers.
template <typename T, typename R, typename W, Mode MODE, Kind KIND>
__global__ void __launch_bounds__(ROW_THREADS, ctas_per_sm(KIND)) backward_rows_kernel(const __grid_constant__ RowParams p) {
  const bshmem_norm_args_t& a = p.a;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float sums[2][SUM_ROWS][4];   // room for three and an empty place
  static_assert(sizeof(sums) <= OWN_SMEM, "see launch");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the kernel that adds the CTAs' sums waits for this one itself
  Rows<MODE, KIND> rows(p, smem, true);
  const bool token = (KIND == ANY || KIND == OUT) && a.gate_mode == BSHMEM_NORM_GATE_TOKEN, full = KIND == ANY && a.gate_mode == BSHMEM_NORM_GATE_FULL;
  const bool has_h = KIND == ANY ? a.h != nullptr : KIND != IN, has_post = KIND == ANY ? a.post != nullptr : KIND != IN;
  const bool has_dr = KIND == ANY ? a.dr != nullptr : KIND != IN, has_dy = KIND == ANY ? a.dy != nullptr : KIND != OUT;
  const float inv_h = 1.f / (float)a.H;
  float u[ROW_CH][4], wp[ROW_CH][4], acc_s[ROW_CH][4], acc_p[ROW_CH][4];
#pragma unroll
  for (int c = 0; c < ROW_CH; ++c) {
    if (has_h) rows.template load_u<W>(u[c], c, has_post);
    if (has_dy) rows.template load4<W>(wp[c], rows.template mine<W>(a.pre), c);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      wp[c][i] = has_dy ? wp[c][i] + a.weight_offset : 0.f;
      if (!has_h) u[c][i] = 0.f;
      acc_s[c][i] = acc_p[c][i] = 0.f;
    }
  }
  // The row's scalars, read one row ahead.
  float tg = 1.f, s1 = 1.f, s2 = 0.f, tg_next = 1.f, s1_next = 1.f, s2_next = 0.f;
  auto scalars = [&](uint32_t row) {
    if (row >= (uint32_t)a.T) return;
    if (token) tg_next = load1<W>(a.gate, row);
    if (has_h && has_post) s1_next = a.stat[row];
    if (has_dy) s2_next = a.stat[a.T + row];
  };
  scalars(rows.first);
  int buf = 0;
  for (uint32_t row = rows.first; row < (uint32_t)a.T; row += rows.step) {
    tg = tg_next, s1 = s1_next, s2 = s2_next;
    scalars(row + rows.step);
    const RowSource src = rows.wait(row);
    // Of four columns: h, ge = the row's gate, uh = u h (with the row's gate), rh = rhat, dy, g = dr + s2 dy pre.  s1 and s2 stay out of what
    // they need not be in: q = s1 uh, and rhat = s2 residual_scale residual + s1 s2 uh.
    // (Products with an absent part are left out where that is known: 0 * x is not 0 for every x.)
    const float s12 = s1 * s2, s2r = s2 * a.residual_scale;
    auto values = [&](int c, float* h, float* ge, float* uh, float* rh, float* dy, float* g) {
      if (KIND != OUT) rows.template load4<R>(rh, src.residual, c);
      if (KIND != IN) rows.template load4<T>(h, src.h, c);
      if (KIND != IN) rows.template load4<R>(g, src.dr, c);
      if (KIND != OUT) rows.template load4<T>(dy, src.dy, c);
      if (full) rows.template load4<W>(ge, src.gate, c);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (!full) ge[i] = tg;
        if (!has_h) h[i] = 0.f;
        if (!has_dr) g[i] = 0.f;
        if (!has_dy) dy[i] = 0.f;
        if constexpr (KIND != IN) {
          uh[i] = u[c][i] * h[i];
          if (full || token) uh[i] *= ge[i];
        }
        if constexpr (KIND == IN) {
          rh[i] *= s2r;
          g[i] = s2 * (dy[i] * wp[c][i]);
        } else if constexpr (KIND != OUT) {
          rh[i] = s2r * rh[i] + s12 * uh[i];
          g[i] += s2 * (dy[i] * wp[c][i]);
          if (!has_dy) rh[i] = 0.f;
        }
      }
    };
    float v[3] = {0.f, 0.f, 0.f};
#pragma unroll
    for (int c = 0; c < ROW_CH; ++c) {
      float h[4], ge[4], uh[4], rh[4], dy[4], g[4];
      values(c, h, ge, uh, rh, dy, g);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (KIND != OUT) v[0] += dy[i] * wp[c][i] * rh[i];
        if constexpr (KIND != IN) {
          if (token) uh[i] = u[c][i] * h[i];   // without the gate: see c2
          v[1] += uh[i] * g[i];
          if constexpr (KIND != OUT) v[2] += uh[i] * rh[i];
        }
      }
      if (c == 0) rows.refill_before(row);
    }
    rows.sum(v, sums[buf]);
    buf ^= 1;
    if (MODE != EARLY && row != rows.first) rows.refill(row - rows.step, rows.stage ? rows.stage - 1 : p.stages - 1);  // the barrier of the sum: all are done with the row before
    const float c1 = v[0] * inv_h * s2, qg = s1 * (v[1] - c1 * v[2]), c2 = qg * tg * inv_h * s1 * s1;   // times s2, a sum, and times s1^2
    if (token && a.dgate && rows.tid == 0) store1<W>(a.dgate, row, qg);
#pragma unroll
    for (int c = 0; c < ROW_CH; ++c) {
      float h[4], ge[4], uh[4], rh[4], dy[4], g[4];
      values(c, h, ge, uh, rh, dy, g);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (KIND != OUT) {
          g[i] -= c1 * rh[i];
          acc_p[c][i] += dy[i] * rh[i];
        }
        dy[i] = a.residual_scale * g[i];
        if constexpr (KIND != IN) {
          g[i] *= s1;
          if (full && a.dgate) uh[i] = u[c][i] * h[i] * g[i];
          if (full || token) g[i] *= ge[i];
          acc_s[c][i] += g[i] * h[i];
          h[i] = has_post ? u[c][i] * g[i] - c2 * h[i] : u[c][i] * g[i];
        }
      }
      if (a.dresidual) rows.store4(rows.template out<R>(a.dresidual, row), c, dy);
      if (KIND != IN && a.dh) rows.store4(rows.template out<T>(a.dh, row), c, h);
      if (full && a.dgate) rows.store4(rows.template out<W>(a.dgate, row), c, uh);
    }
    rows.release();
    rows.next();
  }
  if (a.partials) {
    float* part = a.partials + (size_t)(p.half ? blockIdx.x / 2 : blockIdx.x) * 2 * a.H;
    if (staged(MODE) || blockDim.x == rows.threads) {
#pragma unroll
      for (int c = 0; c < ROW_CH; ++c) {
        rows.store4(part + rows.base, c, acc_s[c]);
        rows.store4(part + a.H + rows.base, c, acc_p[c]);
      }
    } else {  // the warps' sums, in order
      float* s = (float*)smem;  // [warps][2][H]
      const int warps = blockDim.x >> 5;
#pragma unroll
      for (int c = 0; c < ROW_CH; ++c) {
        rows.store4(s + (threadIdx.x >> 5) * 2 * a.H, c, acc_s[c]);
        rows.store4(s + ((threadIdx.x >> 5) * 2 + 1) * a.H, c, acc_p[c]);
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

// Sums of the CTAs' parts, in order: S (dpost and the channel gate's gradient) and dpre.
constexpr int SLICES = 32;
template <typename W>
static __global__ void __launch_bounds__(32 * SLICES) column_sum_kernel(const __grid_constant__ bshmem_norm_args_t a, int parts) {
  const int i = blockIdx.x * 32 + threadIdx.x;
  const bool pre = blockIdx.y != 0, channel = a.gate_mode == BSHMEM_NORM_GATE_CHANNEL;
  if (pre ? !a.dpre : !a.dpost && !(a.dgate && channel)) {
    asm volatile("griddepcontrol.wait;" ::: "memory");  // the end of this kernel is the end of both
    return;
  }
  __shared__ float s[SLICES][33];
  float v = 0.f;
  asm volatile("griddepcontrol.wait;" ::: "memory");
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
    store1<W>(a.dpre, i, v);
    return;
  }
  if (a.dpost) store1<W>(a.dpost, i, a.branch_scale * v * (channel ? load1<W>(a.gate, i) : 1.f));
  if (a.dgate && channel) store1<W>(a.dgate, i, a.branch_scale * v * (a.post ? load1<W>(a.post, i) + a.weight_offset : 1.f));
}

// ------------------------------------------------------------------ host
static inline bool aligned(const void* p) { return ((uintptr_t)p & 15) == 0; }

// Rows and parameters may be read and written 16 bytes at a time.
static inline bool vectors(const bshmem_norm_args_t* a) {
  if (a->H % 8) return false;
  const bool per_token = a->gate_mode == BSHMEM_NORM_GATE_TOKEN;   // read one by one
  const void* ptrs[] = {a->h, a->residual, a->post, a->pre, per_token ? nullptr : a->gate, a->r, a->y, a->dr, a->dy, a->dh, a->dresidual, per_token ? nullptr : a->dgate};
  for (const void* q : ptrs)
    if (!aligned(q)) return false;
  return !((a->h_stride | a->res_stride | a->dr_stride | a->dy_stride) & 7) && (a->gate_mode != BSHMEM_NORM_GATE_FULL || !(a->gate_stride & 7));
}

static inline int sm_count() {
  int device = 0, sms = 0;
  cudaGetDevice(&device);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
  return sms > 0 ? sms : 1;
}

// How a call runs.
struct RowPlan {
  Mode mode;
  Kind kind;
  int ctas, block, threads, half, stages, stage_bytes, smem, parts;
};
static inline RowPlan row_plan(const bshmem_norm_args_t* a, bool backward) {
  const bool vec = vectors(a);
  RowPlan r = {vec ? VECTOR : SCALAR, ANY, 0, 0, 0, 0, 0, 0, 0, 0};
  if (a->H > CTA_COLS) r.half = ((a->H + 1) / 2 + 7) / 8 * 8;
  const int sms = sm_count(), pair = r.half ? 2 : 1;
  const bool after = backward ? a->dr != nullptr : a->r != nullptr, before = backward ? a->dy != nullptr : a->y != nullptr;
  if (vec && a->H % (WARP_COLS * pair) == 0) {
    if (!a->h && before && !(backward && a->dr)) r.kind = IN;
    else if (a->h && a->post && after && !before && a->gate_mode != BSHMEM_NORM_GATE_FULL) r.kind = OUT;
    else if (a->h && a->post && after && before && (a->gate_mode == BSHMEM_NORM_GATE_NONE || a->gate_mode == BSHMEM_NORM_GATE_CHANNEL)) r.kind = BOTH;
  }
  const int cols = r.half ? r.half : a->H;
  r.threads = (cols + ROW_COLS * 32 - 1) / (ROW_COLS * 32) * 32;
  if (a->H <= WARP_COLS) {
    r.block = 32 * WARP_GROUPS;
    r.smem = backward && a->partials ? WARP_GROUPS * 2 * a->H * 4 : 0;
  } else {
    r.block = r.threads;
  }
  int per_sm = ctas_per_sm(r.kind) * ROW_THREADS / r.block;
  if (per_sm > MAX_CTAS_PER_SM) per_sm = MAX_CTAS_PER_SM;
  if (vec && a->H > WARP_COLS && a->T > sms * per_sm / pair) {
    // Two stages at least; rather fewer CTAs of an SM than none.  Forward three at most: more rows on their way favour some SMs over others, and the
    // rows are dealt out beforehand (4096 x 8192 bf16 48.5 us with six, 46.5 with three; 8192 x 4096 48.4 and 45.2; fp32 residual 70 and 68; a
    // norm alone, bf16, 4096 x 8192 25.0 and 24.1, 4096 x 5120 19.2 and 16.4, 8192 x 2048 15.8 and 13.5, fp32 4096 x 8192 49.1 both).
    const int most_stages = backward ? MAX_STAGES : 3;
    r.stage_bytes = stage_rows(*a, cols, backward, r.kind).bytes;
    for (int n = per_sm; n > 0; --n) {
      const int fit = (STAGE_SMEM / n - 2048) / r.stage_bytes;
      if (fit < 2) continue;
      r.mode = STAGED;
      r.stages = fit < most_stages ? fit : most_stages;
      r.smem = r.stages * r.stage_bytes + MAX_STAGES * 16 + 16;
      // With two stages the copies would have half a row's time only (backward, fp32 residual, 4096 x 8192: 116 us, 101 early).  With three, or
      // more CTAs, it costs instructions and gains nothing (bf16 74 us, 76 early; pairs 98 and 109), but for the short rows of a norm alone (4096 x 8192
      // bf16 47.0 us, 45.1 early; 8192 x 4096 48.1 and 46.4; 16384 x 2048 48.6 both).
      if (backward && (r.kind == IN || (r.kind != OUT && r.stages == 2 && n == 1))) r.mode = EARLY;
      per_sm = n;
      break;
    }
  }
  const int groups = r.block / r.threads, want = (int)(((int64_t)a->T + groups - 1) / groups), most = sms * per_sm / pair;
  r.parts = want < most ? want : most;
  r.ctas = r.parts * pair;
  return r;
}
// Launches a kernel; `ready`: the GPUs (bit = ordinal) on which its shared-memory limit has been raised.
template <typename P>
static int launch(void (*kernel)(P), const RowPlan& plan, const P& p, std::atomic<uint64_t>& ready, cudaStream_t stream) {
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess) return BSHMEM_NORM_ERR_DRIVER;
  if (plan.smem + OWN_SMEM > DEFAULT_SMEM && (device >= 64 || !(ready.load(std::memory_order_acquire) >> device & 1))) {
    if (cudaFuncSetAttribute((const void*)kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, STAGE_SMEM) != cudaSuccess) return BSHMEM_NORM_ERR_DRIVER;
    if (device < 64) ready.fetch_or(1ull << device, std::memory_order_release);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(plan.ctas);
  cfg.blockDim = dim3(plan.block);
  cfg.dynamicSmemBytes = plan.smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = 2;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = plan.half ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, p) == cudaSuccess ? BSHMEM_NORM_OK : BSHMEM_NORM_ERR_DRIVER;
}
// The second kernel of a backward pass is set up while the first runs, and waits for it itself.
template <typename W>
static int launch_column_sums(const bshmem_norm_args_t& a, int parts, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((a.H + 31) / 32, 2);
  cfg.blockDim = dim3(32, SLICES);
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, column_sum_kernel<W>, a, parts) == cudaSuccess ? BSHMEM_NORM_OK : BSHMEM_NORM_ERR_DRIVER;
}

// The kernel of a plan.  A row alone (IN) has one type.
template <typename T, typename R, typename W, bool BACKWARD, Mode MODE, Kind KIND>
constexpr auto kernel_of() {
  if constexpr (BACKWARD) return backward_rows_kernel<T, R, W, MODE, KIND>;
  else return forward_rows_kernel<T, R, W, MODE, KIND>;
}
template <typename T, typename R, typename W, bool BACKWARD, Mode MODE>
static void (*by_kind(Kind kind))(RowParams) {
  if constexpr (std::is_same<T, R>::value && !(BACKWARD && MODE == STAGED))   // backward, a row alone is EARLY
    if (kind == IN) return kernel_of<T, R, W, BACKWARD, MODE, IN>();
  return kind == BOTH ? kernel_of<T, R, W, BACKWARD, MODE, BOTH>() : kind == OUT ? kernel_of<T, R, W, BACKWARD, MODE, OUT>() : kernel_of<T, R, W, BACKWARD, MODE, ANY>();
}
template <typename T, typename R, typename W, bool BACKWARD>
static void (*early_kernel(Kind kind))(RowParams) {
  if constexpr (!BACKWARD) return nullptr;   // forward never is
  else if constexpr (std::is_same<T, R>::value) return kind == IN ? kernel_of<T, R, W, true, EARLY, IN>() : kind == BOTH ? kernel_of<T, R, W, true, EARLY, BOTH>() : kernel_of<T, R, W, true, EARLY, ANY>();
  else return kind == BOTH ? kernel_of<T, R, W, true, EARLY, BOTH>() : kernel_of<T, R, W, true, EARLY, ANY>();
}
template <typename T, typename R, typename W, bool BACKWARD>
static int launch_rows(const bshmem_norm_args_t* a, cudaStream_t stream) {
  const RowPlan plan = row_plan(a, BACKWARD);
  const RowParams p = {*a, plan.threads, plan.half, plan.stages, plan.stage_bytes};
  void (*const kernel)(RowParams) = plan.mode == EARLY ? early_kernel<T, R, W, BACKWARD>(plan.kind) : plan.mode == STAGED ? by_kind<T, R, W, BACKWARD, STAGED>(plan.kind) : plan.mode == VECTOR ? by_kind<T, R, W, BACKWARD, VECTOR>(plan.kind)
                                                                                                        : kernel_of<T, R, W, BACKWARD, SCALAR, ANY>();
  static std::atomic<uint64_t> ready[4][4];
  const int st = launch(kernel, plan, p, ready[plan.mode][plan.kind], stream);
  return st || !BACKWARD || !a->partials ? st : launch_column_sums<W>(*a, plan.parts, stream);
}
template <typename T, typename R, typename W>
static int launch_either(const bshmem_norm_args_t* a, bool backward, cudaStream_t stream) {
  return backward ? launch_rows<T, R, W, true>(a, stream) : launch_rows<T, R, W, false>(a, stream);
}

// A call whose rows are of type T: by the types of the residual and of the parameters.
template <typename T>
static int run(const bshmem_norm_args_t* a, bool backward, cudaStream_t stream) {
  const bool r = a->res_type == a->type, w = a->wt_type == a->type;
  if constexpr (sizeof(T) == 4) return launch_either<T, T, T>(a, backward, stream);
  else if (r) return w ? launch_either<T, T, T>(a, backward, stream) : launch_either<T, T, float>(a, backward, stream);
  else return w ? launch_either<T, float, T>(a, backward, stream) : launch_either<T, float, float>(a, backward, stream);
}
int run_bf16(const bshmem_norm_args_t* a, bool backward, cudaStream_t stream);
int run_f16(const bshmem_norm_args_t* a, bool backward, cudaStream_t stream);
int run_f32(const bshmem_norm_args_t* a, bool backward, cudaStream_t stream);

}  // namespace norms
}  // namespace bshmem
