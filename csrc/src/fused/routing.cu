// Expert router (choice and weights of K experts per token) and balance loss, forward and backward.
//
// A warp takes a token: lane l holds the logits of experts l, l + 32, ... in registers, so a row is read once in whole lines and
// everything after that is shuffles.  The choice is K rounds of a maximum over the warp of keys that order like the floats
// (redux.sync), the lowest expert among equal keys, over the few keys that a bound leaves.  Bound by latency: a warp loads its row, then goes through
// a chain of rounds, and at 55 tokens an SM other warps fill a part of the gaps only.  8192 x 256 top-8 issues in 44 slots of a hundred, with 2.5
// warps on average waiting for their row, 2.5 for the instruction before and 1.9 for the integer pipe (40 % busy); DRAM is at 11 %.  It takes 5.2 us with
// one expert a token and 7.1 us with eight (8.9 MB: 1.4 us of memory time).  A decode batch (64 x 256, top-8) takes 3.0 us, most of it the launch
// and the chain of rounds.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <limits.h>
#include <math_constants.h>
#include <stdint.h>

#include "../../include/bshmem/routing.h"
#include "launch.cuh"

namespace bshmem {
namespace routing {

constexpr int THREADS = 256, WARPS = THREADS / 32;

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void put(__half* p, float v) { *p = __float2half_rn(v); }

// Unsigned keys in the order of the floats; 0 for -inf and NaN, which are never chosen.  -0 and 0 are equal.
__device__ __forceinline__ uint32_t key32(float v) {
  if (!(v > -CUDART_INF_F)) return 0u;
  const uint32_t b = __float_as_uint(v + 0.f);
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float value32(uint32_t key) { return __uint_as_float(key ^ ((key >> 31) ? 0x80000000u : 0xffffffffu)); }
__device__ __forceinline__ uint64_t key64(double v) {
  if (!(v > -CUDART_INF)) return 0ull;
  const uint64_t b = (uint64_t)__double_as_longlong(v + 0.0);
  return b ^ ((b >> 63) ? ~0ull : 1ull << 63);
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// Largest value of the warp, NaN ignored; -inf if there is none.
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// Logits of this lane's experts; -inf past the last.
template <typename T, int VPL>
__device__ __forceinline__ void load_row(float (&l)[VPL], const T* row, int E, int lane) {
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    const int e = lane + 32 * i;
    l[i] = e < E ? to_f(row[e]) : -CUDART_INF_F;
  }
}

// The `rounds` largest of the warp's keys, the lowest expert first among equal ones: lane k gets the k-th as (expert, key), (-1, 0) where none
// is left.
template <int VPL>
__device__ __forceinline__ void select(uint32_t (&key)[VPL], int rounds, int lane, int& expert, uint32_t& its_key) {
  expert = -1;
  its_key = 0;
  for (int k = 0; k < rounds; ++k) {
    uint32_t best = 0;
    int e = 0;
#pragma unroll
    for (int i = 0; i < VPL; ++i)
      if (key[i] > best) {
        best = key[i];
        e = lane + 32 * i;
      }
    const uint32_t most = __reduce_max_sync(0xffffffffu, best);
    if (most == 0) break;
    const int chosen = (int)__reduce_min_sync(0xffffffffu, best == most ? (unsigned)e : 0xffffffffu);
    if (lane == k) {
      expert = chosen;
      its_key = most;
    }
#pragma unroll
    for (int i = 0; i < VPL; ++i)
      if (lane + 32 * i == chosen) key[i] = 0;
  }
}

// The same by way of a bound: of the lanes' largest keys the one in place `rounds` is no larger than any key that is chosen, and few
// keys reach it (some 10 to 14 of 256 for eight experts, whatever their scale).  Those are set side by side, in the order of the experts, a
// key a lane.  A round over all keys takes some 50 instructions for 256 experts, and over these seven: 8192 x 256 top-8 9.8 us by select
// alone, 7.1 so; 512 experts 15.6 and 9.1.  One expert takes 5.3 by select and 5.7 so; up to 128 experts there is no difference.
// Should more than 32 reach the bound, as when the largest share a few lanes, the rounds go over all keys.
struct Candidate {
  uint32_t key;
  int expert;
};
template <int VPL>
__device__ __forceinline__ void select_bounded(uint32_t (&key)[VPL], int rounds, int lane, Candidate* room, int& expert, uint32_t& its_key) {
  if (rounds > 1) {
    uint32_t head = 0, bound = 0;
#pragma unroll
    for (int i = 0; i < VPL; ++i) head = max(head, key[i]);
    for (int k = 0; k < rounds; ++k) {
      bound = __reduce_max_sync(0xffffffffu, head);
      if (head == bound) head = 0;   // equal ones at once, which only lowers the bound
    }
    bound = max(bound, 1u);
    int n = 0;
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      const bool in = key[i] >= bound;
      const unsigned mask = __ballot_sync(0xffffffffu, in);
      const int at = n + __popc(mask & ((1u << lane) - 1));
      if (in && at < 32) room[at] = {key[i], lane + 32 * i};
      n += __popc(mask);
    }
    if (n <= 32) {
      __syncwarp();
      uint32_t one[1] = {lane < n ? room[lane].key : 0u};
      select(one, rounds, lane, expert, its_key);
      if (expert >= 0) expert = room[expert].expert;
      return;
    }
  }
  select(key, rounds, lane, expert, its_key);
}

// Numerator of the softmax that the biased choice goes by, as 32 bits take it below: over the logits that are numbers, those of +inf sharing it
// evenly, so that a row has an order whichever of the two decides.
__device__ __forceinline__ double term64(double l, double top) { return l == top ? 1.0 : l > -CUDART_INF ? exp(l - top) : 0.0; }

// Score + bias of one expert in 64 bits; `sum` is the softmax's.
__device__ __forceinline__ uint64_t key_of(const bshmem_route_args_t& a, double l, double top, double sum, int e) {
  const double s = a.score == BSHMEM_ROUTE_SOFTMAX ? term64(l, top) / sum : 1.0 / (1.0 + exp(-l));
  return l > -CUDART_INF ? key64(s + (double)a.bias[e]) : 0ull;
}
template <typename T>
__device__ __forceinline__ double sum_of(const bshmem_route_args_t& a, const T* row, float top, int lane) {
  double sum = 0.0;
#pragma unroll 1
  for (int e = lane; e < a.E; e += 32) sum += term64((double)to_f(row[e]), (double)top);
  return warp_sum(sum);
}

// The experts of lanes 0 to n - 1 (-1: none) in the order of score + bias in 64 bits.
template <typename T>
__device__ __noinline__ int order64(const bshmem_route_args_t& a, const T* row, float top, int lane, int expert, int n) {
  const double sum = a.score == BSHMEM_ROUTE_SOFTMAX ? sum_of(a, row, top, lane) : 1.0;
  const uint64_t key = lane < n && expert >= 0 ? key_of(a, (double)to_f(row[expert]), (double)top, sum, expert) : 0ull;
  int rank = 0, from = lane;
  for (int j = 0; j < n; ++j) {
    const uint64_t other = __shfl_sync(0xffffffffu, key, j);
    const int e = __shfl_sync(0xffffffffu, expert, j);
    rank += other > key || (other == key && (e < expert || (e == expert && j < lane)));
  }
  for (int j = 0; j < n; ++j)
    if (__shfl_sync(0xffffffffu, rank, j) == lane) from = j;
  return __shfl_sync(0xffffffffu, expert, from);
}

// The whole choice in 64 bits, for the odd token whose K-th, next and next but one lie that close: short code, not fast.
template <typename T, int VPL>
__device__ __noinline__ int select64(const bshmem_route_args_t& a, const T* row, float top, int lane) {
  uint64_t key[VPL];
  const double sum = a.score == BSHMEM_ROUTE_SOFTMAX ? sum_of(a, row, top, lane) : 1.0;
  int expert = -1;
#pragma unroll 1
  for (int i = 0; i < VPL; ++i) {
    const int e = lane + 32 * i;
    key[i] = e < a.E ? key_of(a, (double)to_f(row[e]), (double)top, sum, e) : 0ull;
  }
#pragma unroll 1
  for (int k = 0; k < a.K; ++k) {
    uint64_t best = 0;
    int at = 0;
#pragma unroll 1
    for (int i = 0; i < VPL; ++i)
      if (key[i] > best) {
        best = key[i];
        at = i;
      }
    const uint32_t hi = (uint32_t)(best >> 32), lo = (uint32_t)best;
    const uint32_t most = __reduce_max_sync(0xffffffffu, hi);
    if (most == 0) break;  // the high half of a key of a finite number is never 0
    const uint32_t most_lo = __reduce_max_sync(0xffffffffu, hi == most ? lo : 0u);
    const int chosen = (int)__reduce_min_sync(0xffffffffu, hi == most && lo == most_lo ? (unsigned)(lane + 32 * at) : 0xffffffffu);
    if (lane == k) expert = chosen;
    if (lane + 32 * at == chosen) key[at] = 0;
  }
  return expert;
}

// Numerator of a score whose sum over a set of experts is divided out.  `top` is the largest logit of the set:
//   softmax  exp(l - top)
//   sigmoid  1 / (1 + exp(-l)), times exp(-top) where top < 0, so that a set of very negative logits does not underflow
__device__ __forceinline__ float numerator(float l, float top, int score) {
  if (score == BSHMEM_ROUTE_SOFTMAX) return expf(l - top);
  return expf(fminf(l, 0.f) - fminf(top, 0.f)) / (1.f + expf(-fabsf(l)));
}
__device__ __forceinline__ float sigmoid(float l) { return 1.f / (1.f + expf(-l)); }

struct Params {
  bshmem_route_args_t a;
};

template <typename T, int VPL, bool BIAS>
__global__ void __launch_bounds__(THREADS) route_kernel(const __grid_constant__ Params p) {
  const bshmem_route_args_t& a = p.a;
  const int lane = threadIdx.x & 31, K = a.K, E = a.E;
  const long t = (long)blockIdx.x * WARPS + (threadIdx.x >> 5);
  if (t >= a.T) return;
  if (a.valid && !a.valid[t]) {
    if (lane < K) {
      a.idx[t * K + lane] = -1;
      a.weight[t * K + lane] = 0.f;
    }
    return;
  }
  const T* row = (const T*)a.logits + t * a.stride;
  float l[VPL];
  load_row(l, row, E, lane);
  bool nan = false;
  float top = -CUDART_INF_F;
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    nan |= l[i] != l[i];
    top = fmaxf(top, l[i]);
  }
  nan = __any_sync(0xffffffffu, nan);
  top = warp_max(top);
  constexpr bool BOUNDED = VPL >= 8;
  __shared__ Candidate s_room[BOUNDED ? WARPS : 1][32];
  int mine;  // lane k: the k-th chosen expert
  uint32_t key[VPL], mine_key;
  auto choose = [&](int rounds) {
    if constexpr (!BOUNDED) select(key, rounds, lane, mine, mine_key);
    else select_bounded(key, rounds, lane, s_room[threadIdx.x >> 5], mine, mine_key);
  };
  if constexpr (!BIAS) {
#pragma unroll
    for (int i = 0; i < VPL; ++i) key[i] = key32(l[i]);
    choose(K);
  } else {
    // Score + bias in 32 bits with the fast exponential and division first.  An exponential of -x is off by (2 + 1.2 x) ulp and x half steps, the sum of
    // up to 37 terms by as many half steps: together less than 5e-6 of a score down to 2^-10 of the largest, and less than that share of 2^-10 of
    // it below; the sum with the bias is off by half a step.  No expert at or below a value v of score + bias has a score above v less the
    // smallest bias, so that bounds what all of them are off by.  Where two neighbours in the order are closer than twice that for the upper one,
    // the choice is made in 64 bits.  256 experts, top-8: 0.04 tokens in a hundred for a softmax of logits of deviation 1.5, 1 and 4 for 0.1 and
    // 0.02, 6 for 10, 1 for sigmoids; sigmoids that round to 1 side by side need it always.  (A bound of 1e-5 for all sent 2, 83, 100 and 46.)
    // 8192 x 256, top-8, us: 13.1, 14.5, 16.0 and 20.2 for these four, 13.0 for sigmoids, 7.5 to 8.1 without a bias.
    float s[VPL], sum = 0.f;
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      if (a.score == BSHMEM_ROUTE_SOFTMAX) s[i] = l[i] > -CUDART_INF_F ? __expf(l[i] - top) : 0.f;   // 0 for NaN
      else s[i] = __fdividef(1.f, 1.f + __expf(-l[i]));  // 0 from where the divisor passes 2^126 on
      sum += s[i];
    }
    if (a.score == BSHMEM_ROUTE_SOFTMAX && top == CUDART_INF_F) {
      sum = 0.f;
#pragma unroll
      for (int i = 0; i < VPL; ++i) sum += s[i] = l[i] == top ? 1.f : 0.f;
    }
    const float inv = a.score == BSHMEM_ROUTE_SOFTMAX ? 1.f / warp_sum(sum) : 1.f;
    // the largest score; a sigmoid below 2^-10, whose exponential is of a larger x, counts as that
    const float most = a.score == BSHMEM_ROUTE_SOFTMAX ? inv : fmaxf(__fdividef(1.f, 1.f + __expf(-top)), 0x1p-10f);
    float least_bias = CUDART_INF_F;
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      const int e = lane + 32 * i;
      key[i] = 0u;
      if (e < E && l[i] > -CUDART_INF_F) {
        const float b = a.bias[e];
        key[i] = key32(s[i] * inv + b);
        least_bias = fminf(least_bias, b);
      }
    }
    least_bias = -value32(__reduce_max_sync(0xffffffffu, key32(-least_bias)));
    const int rounds = K + 2;
    choose(rounds);
    const uint32_t next = __shfl_down_sync(0xffffffffu, mine_key, 1);
    const float v = value32(mine_key), score = fminf(most, fmaxf(v - least_bias, most * 0x1p-10f));
    const unsigned unclear = __ballot_sync(0xffffffffu, lane <= K && mine_key && next && !(v - value32(next) > 1e-5f * score + 5e-7f * fabsf(v)));
    if ((unclear >> (K - 1) & 3) == 3) mine = select64<T, VPL>(a, row, top, lane);  // what was not picked may belong to the K, too
    else if (unclear & ((1u << K) - 1)) mine = order64(a, row, top, lane, mine, rounds);
    if (lane >= K) mine = -1;
  }
  float w = 0.f;
  if (a.renormalize) {
    // the largest chosen logit is the row's unless a bias chose otherwise
    const float lm = mine >= 0 ? to_f(row[mine]) : -CUDART_INF_F;
    const float set_top = warp_max(lm);
    const float num = mine >= 0 ? numerator(lm, set_top, a.score) : 0.f;
    const float sum = warp_sum(num);
    w = mine >= 0 ? num / sum : 0.f;
  } else if (a.score == BSHMEM_ROUTE_SOFTMAX) {
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < VPL; ++i) sum += l[i] > -CUDART_INF_F ? expf(l[i] - top) : 0.f;
    sum = warp_sum(sum);
    if (mine >= 0) w = expf(to_f(row[mine]) - top) / sum;
  } else if (mine >= 0) {
    w = sigmoid(to_f(row[mine]));
  }
  if (mine >= 0 && (nan || top == CUDART_INF_F) && a.score == BSHMEM_ROUTE_SOFTMAX) w = CUDART_NAN_F;  // the sum over all experts is NaN
  if (lane < K) {
    a.idx[t * K + lane] = mine;
    a.weight[t * K + lane] = w * a.scale;
  }
}

// Gradient of the weights.  With w the weights before `scale`, over the chosen experts k:
//   renormalised    dl_k = scale w_k (dw_k - sum_j dw_j w_j), for sigmoids times (1 - s_k); zero elsewhere
//   softmax         dl_e = scale p_e ([e chosen] dw_e - sum_j dw_j p_j)
//   sigmoid         dl_k = scale dw_k s_k (1 - s_k); zero elsewhere
template <typename T, int VPL>
__global__ void __launch_bounds__(THREADS) route_backward_kernel(const __grid_constant__ Params p) {
  const bshmem_route_args_t& a = p.a;
  const int lane = threadIdx.x & 31, K = a.K, E = a.E;
  const long t = (long)blockIdx.x * WARPS + (threadIdx.x >> 5);
  if (t >= a.T) return;
  T* out = (T*)a.dlogits + t * E;
  const T* row = (const T*)a.logits + t * a.stride;
  const int mine = lane < K ? a.idx[t * K + lane] : -1;
  const float dw = mine >= 0 ? a.dweight[t * K + lane] : 0.f;
  const float lm = mine >= 0 ? to_f(row[mine]) : -CUDART_INF_F;
  const float poison = mine >= 0 ? 0.f * a.weight[t * K + lane] : 0.f;  // NaN where the forward's weight was
  float d = 0.f;
  if (!a.renormalize && a.score == BSHMEM_ROUTE_SOFTMAX) {
    float l[VPL], top = -CUDART_INF_F, sum = 0.f;
    load_row(l, row, E, lane);
#pragma unroll
    for (int i = 0; i < VPL; ++i) top = fmaxf(top, l[i]);
    top = warp_max(top);
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
      l[i] = l[i] > -CUDART_INF_F ? expf(l[i] - top) : 0.f;
      sum += l[i];
    }
    sum = warp_sum(sum);
    const float pm = mine >= 0 ? expf(lm - top) / sum + poison : 0.f;
    const float g = warp_sum(dw * pm);
    const bool any = __any_sync(0xffffffffu, mine >= 0);
#pragma unroll
    for (int i = 0; i < VPL; ++i)
      if (lane + 32 * i < E) put(out + lane + 32 * i, any ? -a.scale * (l[i] / sum) * g : 0.f);
    d = a.scale * pm * (dw - g);
  } else {
#pragma unroll
    for (int i = 0; i < VPL; ++i)
      if (lane + 32 * i < E) put(out + lane + 32 * i, 0.f);
    if (a.renormalize) {
      const float set_top = warp_max(lm);
      const float num = mine >= 0 ? numerator(lm, set_top, a.score) : 0.f;
      const float sum = warp_sum(num);
      const float w = mine >= 0 ? num / sum + poison : 0.f;
      d = a.scale * w * (dw - warp_sum(dw * w));
      if (a.score == BSHMEM_ROUTE_SIGMOID) d *= sigmoid(-lm);
    } else {
      d = a.scale * dw * sigmoid(lm) * sigmoid(-lm);
    }
  }
  __syncwarp();  // the row's other values are written; the chosen ones replace theirs
  if (mine >= 0) put(out + mine, d);
}

// Probabilities of the balance loss for this lane's experts, in place of the logits; all zero for a row of -inf.  s1[i] is the
// derivative's factor 1 - sigmoid(l).
template <int VPL, bool SLOPE>
__device__ __forceinline__ void probabilities(float (&l)[VPL], float (&slope)[SLOPE ? VPL : 1], int score) {
  float top = -CUDART_INF_F, sum = 0.f;
#pragma unroll
  for (int i = 0; i < VPL; ++i) top = fmaxf(top, l[i]);
  top = warp_max(top);
  if (top == -CUDART_INF_F) top = 0.f;
#pragma unroll
  for (int i = 0; i < VPL; ++i) {
    if constexpr (SLOPE) slope[i] = score == BSHMEM_ROUTE_SIGMOID ? sigmoid(-l[i]) : 1.f;
    l[i] = numerator(l[i], top, score);
    sum += l[i];
  }
  sum = warp_sum(sum);
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
  for (int i = 0; i < VPL; ++i) l[i] *= inv;
}

// Each CTA's sums of the probabilities and counts over its tokens: [grid][E] floats, [grid][E] counts, [grid] valid tokens.
struct Workspace {
  float* p;
  int* counts;
  int* n;
};
__host__ __device__ __forceinline__ Workspace workspace(void* base, int grid, int E) {
  Workspace w;
  w.p = (float*)base;
  w.counts = (int*)(w.p + (size_t)grid * E);
  w.n = w.counts + (size_t)grid * E;
  return w;
}

// What an expert of probability sum `p` and count `c` over n tokens adds to the loss; writes its count and dloss / dp, from which the
// mean over the experts is taken off: it drops out of the gradient (the probabilities of a token sum to 1), and its rounding with it.
__device__ __forceinline__ float finish_expert(const bshmem_route_args_t& a, int e, float p, int c, int n, int all) {
  const double nn = n > 0 ? (double)n : 1.0, scale = (double)a.E / (a.K * nn * nn);
  a.counts[e] = c;
  if (a.coef) a.coef[e] = (float)(scale * ((double)c - (double)all / a.E));
  return (float)(scale * c) * p;
}

// 8192 x 256: 9.4 us and the finishing kernel's part, bound by latency: the sums of an SM's tokens lie in the registers of one CTA, whose 16 warps issue in
// 23 slots of a hundred and wait for rows most of the time, though each has its next one on the way.
constexpr int B_THREADS = 512, B_WARPS = B_THREADS / 32;
constexpr int ONE_CTA_TOKENS = 8 * B_WARPS;   // up to here one CTA does all: 61 x 40 in 5.4 us; two kernels took 2.9 + 3.2 us and a second launch

template <typename T, int VPL>
__global__ void __launch_bounds__(B_THREADS) balance_kernel(const __grid_constant__ Params p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // the finishing kernel waits for this one itself
  const bshmem_route_args_t& a = p.a;
  __shared__ int s_count[32 * VPL];
  __shared__ float s_p[B_WARPS][32 * VPL <= 512 ? 32 * VPL : 1];  // up to 512 experts; beyond, warps add up in turn
  __shared__ float s_sum[32 * VPL <= 512 ? 1 : 32 * VPL];
  __shared__ int s_n, s_all;
  __shared__ float s_loss[B_WARPS];
  constexpr bool TURNS = 32 * VPL > 512;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, K = a.K, E = a.E;
  for (int e = threadIdx.x; e < 32 * VPL; e += B_THREADS) {
    s_count[e] = 0;
    if (TURNS) s_sum[e] = 0.f;
  }
  if (threadIdx.x == 0) s_n = s_all = 0;
  __syncthreads();
  float acc[VPL], l[VPL];
#pragma unroll
  for (int i = 0; i < VPL; ++i) acc[i] = 0.f;
  int n = 0, found = 0;
  const long first = (long)blockIdx.x * B_WARPS + warp, step = (long)gridDim.x * B_WARPS;
  auto fetch = [&](long t) {
    if (t < a.T) load_row(l, (const T*)a.logits + t * a.stride, E, lane);
  };
  fetch(first);
  for (long t = first; t < a.T; t += step) {
    float q[VPL], unused[1];
#pragma unroll
    for (int i = 0; i < VPL; ++i) q[i] = l[i];
    fetch(t + step);   // on the way while this token is worked on
    if (a.valid && !a.valid[t]) continue;
    ++n;
    if (lane < K) {
      const int e = a.idx[t * K + lane];
      if (e >= 0 && e < E) {
        atomicAdd(&s_count[e], 1);
        ++found;
      }
    }
    probabilities<VPL, false>(q, unused, a.score);
#pragma unroll
    for (int i = 0; i < VPL; ++i) acc[i] += q[i];
  }
  found = __reduce_add_sync(0xffffffffu, found);
  if (lane == 0 && n) atomicAdd(&s_n, n);
  if (lane == 0 && found) atomicAdd(&s_all, found);
  if constexpr (TURNS) {
    for (int k = 0; k < B_WARPS; ++k) {
      if (k == warp)
#pragma unroll
        for (int i = 0; i < VPL; ++i) s_sum[lane + 32 * i] += acc[i];
      __syncthreads();
    }
  } else {
#pragma unroll
    for (int i = 0; i < VPL; ++i) s_p[warp][lane + 32 * i] = acc[i];
    __syncthreads();
  }
  const Workspace w = workspace(a.workspace, gridDim.x, E);
  float term = 0.f;
  for (int e = threadIdx.x; e < E; e += B_THREADS) {
    float s = 0.f;
    if constexpr (TURNS) {
      s = s_sum[e];
    } else {
#pragma unroll
      for (int k = 0; k < B_WARPS; ++k) s += s_p[k][e];
    }
    if (gridDim.x == 1) {
      term += finish_expert(a, e, s, s_count[e], s_n, s_all);
    } else {
      w.p[(size_t)blockIdx.x * E + e] = s;
      w.counts[(size_t)blockIdx.x * E + e] = s_count[e];
    }
  }
  if (gridDim.x > 1) {
    if (threadIdx.x == 0) w.n[blockIdx.x] = s_n;
    return;
  }
  term = warp_sum(term);
  if (lane == 0) s_loss[warp] = term;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int k = 1; k < B_WARPS; ++k) term += s_loss[k];
    *a.loss = term;
  }
}

// Adds the CTAs' sums in order and forms the loss.  One CTA of 1024 threads; each column's CTAs are divided among 1024 / E of them.
__global__ void __launch_bounds__(1024) balance_finish_kernel(const __grid_constant__ Params p, int parts) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const bshmem_route_args_t& a = p.a;
  __shared__ int s_n, s_all;
  __shared__ float s_loss[32];
  __shared__ float s_p[1024];
  __shared__ int s_c[1024];
  const Workspace w = workspace(a.workspace, parts, a.E);
  if (threadIdx.x == 0) s_n = s_all = 0;
  int cols = 32;
  while (cols < a.E) cols *= 2;
  const int slices = 1024 / cols, e = threadIdx.x % cols, slice = threadIdx.x / cols;
  float ps = 0.f;
  int cs = 0, n = 0;
  if (e < a.E) {
#pragma unroll 8
    for (int k = slice; k < parts; k += slices) {
      ps += w.p[(size_t)k * a.E + e];
      cs += w.counts[(size_t)k * a.E + e];
    }
  }
  for (int k = threadIdx.x; k < parts; k += 1024) n += w.n[k];
  s_p[threadIdx.x] = ps;
  s_c[threadIdx.x] = cs;
  __syncthreads();
  const int all = __reduce_add_sync(0xffffffffu, cs);
  n = __reduce_add_sync(0xffffffffu, n);
  if ((threadIdx.x & 31) == 0) {
    if (all) atomicAdd(&s_all, all);
    if (n) atomicAdd(&s_n, n);
  }
  __syncthreads();
  float term = 0.f;
  if (slice == 0 && e < a.E) {
    for (int k = 1; k < slices; ++k) {
      ps += s_p[k * cols + e];
      cs += s_c[k * cols + e];
    }
    term = finish_expert(a, e, ps, cs, s_n, s_all);
  }
  term = warp_sum(term);
  if ((threadIdx.x & 31) == 0) s_loss[threadIdx.x >> 5] = term;
  __syncthreads();
  if (threadIdx.x < 32) {
    term = warp_sum(s_loss[threadIdx.x]);
    if (threadIdx.x == 0) *a.loss = term;
  }
}

// dl_e = dloss p_e (coef_e - sum_j p_j coef_j), for sigmoids times (1 - s_e); coef up to a constant.
template <typename T, int VPL>
__global__ void __launch_bounds__(THREADS) balance_backward_kernel(const __grid_constant__ Params p) {
  const bshmem_route_args_t& a = p.a;
  const int lane = threadIdx.x & 31, E = a.E;
  const long t = (long)blockIdx.x * WARPS + (threadIdx.x >> 5);
  if (t >= a.T) return;
  T* out = (T*)a.dlogits + t * E;
  if (a.valid && !a.valid[t]) {
#pragma unroll
    for (int i = 0; i < VPL; ++i)
      if (lane + 32 * i < E) put(out + lane + 32 * i, 0.f);
    return;
  }
  float l[VPL], slope[VPL], c[VPL];
  load_row(l, (const T*)a.logits + t * a.stride, E, lane);
#pragma unroll
  for (int i = 0; i < VPL; ++i) c[i] = lane + 32 * i < E ? a.coef[lane + 32 * i] : 0.f;
  const float dloss = *a.dloss;
  probabilities<VPL, true>(l, slope, a.score);
  float mean = 0.f;
#pragma unroll
  for (int i = 0; i < VPL; ++i) mean += l[i] * c[i];
  mean = warp_sum(mean);
#pragma unroll
  for (int i = 0; i < VPL; ++i)
    if (lane + 32 * i < E) put(out + lane + 32 * i, dloss * (l[i] * (c[i] - mean)) * slope[i]);
}

static int check(const bshmem_route_args_t* a) {
  if (!a) return BSHMEM_ROUTE_ERR_ARGS;
  if (a->T < 0 || a->E < 1 || a->E > BSHMEM_ROUTE_MAX_EXPERTS || a->K < 1 || a->K > BSHMEM_ROUTE_MAX_TOPK || a->K > a->E) return BSHMEM_ROUTE_ERR_SHAPE;
  if ((long)a->T * a->K > INT_MAX) return BSHMEM_ROUTE_ERR_SHAPE;
  if (a->type < 0 || a->type > 2 || a->score < 0 || a->score > 1) return BSHMEM_ROUTE_ERR_ARGS;
  return BSHMEM_ROUTE_OK;
}

static int balance_ctas(int T) {
  int device = 0, sms = 0;
  cudaGetDevice(&device);
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
  if (T <= ONE_CTA_TOKENS) return 1;
  const int want = (T + B_WARPS - 1) / B_WARPS, most = sms > 0 ? sms : 1;
  return want < most ? want : most;
}

// Calls f<T, VPL> for the type and the number of experts.
template <typename T, typename F>
static int by_experts(int E, F&& f) {
  if (E <= 32) return f.template operator()<T, 1>();
  if (E <= 64) return f.template operator()<T, 2>();
  if (E <= 128) return f.template operator()<T, 4>();
  if (E <= 256) return f.template operator()<T, 8>();
  if (E <= 512) return f.template operator()<T, 16>();
  return f.template operator()<T, 32>();
}
template <typename F>
static int dispatch(const bshmem_route_args_t* a, F&& f) {
  if (a->type == BSHMEM_ROUTE_F32) return by_experts<float>(a->E, f);
  if (a->type == BSHMEM_ROUTE_BF16) return by_experts<__nv_bfloat16>(a->E, f);
  return by_experts<__half>(a->E, f);
}
static int launched(cudaError_t e) { return e == cudaSuccess ? BSHMEM_ROUTE_OK : BSHMEM_ROUTE_ERR_DRIVER; }

struct Route {
  const Params& p;
  cudaStream_t stream;
  template <typename T, int VPL>
  int operator()() const {
    const unsigned grid = ((unsigned)p.a.T + WARPS - 1) / WARPS;
    return launched(launch_kernel(p.a.bias ? route_kernel<T, VPL, true> : route_kernel<T, VPL, false>, grid, THREADS, stream, p));
  }
};
struct RouteBackward {
  const Params& p;
  cudaStream_t stream;
  template <typename T, int VPL>
  int operator()() const {
    return launched(launch_kernel(route_backward_kernel<T, VPL>, ((unsigned)p.a.T + WARPS - 1) / WARPS, THREADS, stream, p));
  }
};
struct Balance {
  const Params& p;
  cudaStream_t stream;
  template <typename T, int VPL>
  int operator()() const {
    const int grid = balance_ctas(p.a.T);
    const int st = launched(launch_kernel(balance_kernel<T, VPL>, grid, B_THREADS, stream, p));
    if (st || grid == 1) return st;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(1);
    cfg.blockDim = dim3(1024);
    cfg.stream = stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return launched(cudaLaunchKernelEx(&cfg, balance_finish_kernel, p, grid));
  }
};
struct BalanceBackward {
  const Params& p;
  cudaStream_t stream;
  template <typename T, int VPL>
  int operator()() const {
    return launched(launch_kernel(balance_backward_kernel<T, VPL>, ((unsigned)p.a.T + WARPS - 1) / WARPS, THREADS, stream, p));
  }
};

}  // namespace routing
}  // namespace bshmem

using namespace bshmem::routing;

extern "C" size_t bshmem_balance_workspace(int T, int E) {
  const size_t grid = (size_t)balance_ctas(T);
  return (grid * E * 2 + grid) * 4;
}

extern "C" int bshmem_route(const bshmem_route_args_t* a, cudaStream_t stream) {
  const int st = check(a);
  if (st || a->T == 0) return st;
  if (!a->logits || !a->idx || !a->weight) return BSHMEM_ROUTE_ERR_ARGS;
  const Params p = {*a};
  return dispatch(a, Route{p, stream});
}

extern "C" int bshmem_route_backward(const bshmem_route_args_t* a, cudaStream_t stream) {
  const int st = check(a);
  if (st || a->T == 0) return st;
  if (!a->logits || !a->idx || !a->weight || !a->dweight || !a->dlogits) return BSHMEM_ROUTE_ERR_ARGS;
  const Params p = {*a};
  return dispatch(a, RouteBackward{p, stream});
}

extern "C" int bshmem_balance(const bshmem_route_args_t* a, cudaStream_t stream) {
  const int st = check(a);
  if (st) return st;
  if ((a->T && (!a->logits || !a->idx)) || !a->loss || !a->counts || !a->workspace) return BSHMEM_ROUTE_ERR_ARGS;
  const Params p = {*a};
  return dispatch(a, Balance{p, stream});
}

extern "C" int bshmem_balance_backward(const bshmem_route_args_t* a, cudaStream_t stream) {
  const int st = check(a);
  if (st || a->T == 0) return st;
  if (!a->logits || !a->coef || !a->dloss || !a->dlogits) return BSHMEM_ROUTE_ERR_ARGS;
  const Params p = {*a};
  return dispatch(a, BalanceBackward{p, stream});
}
