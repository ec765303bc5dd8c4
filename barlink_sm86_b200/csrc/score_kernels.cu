// SPDX-License-Identifier: MIT
//
// Log probabilities of given tokens, the entropy of the distribution and its most likely tokens, from logits.
//
//   m = max x,  S = sum e^(x - m),  T = sum (x - m) e^(x - m)
//   logprob(id) = x_id - m - log S,  entropy = log S - T / S
//
// One pass: a block goes through its share of a row in laps, a thread with kScoreLap vectors of 16 bytes in registers and those of the next lap on
// their way; it finds their maximum and adds up S and T relative to it.  Sums of laps, threads, warps and the blocks of a cluster, which share a
// row, are joined afterwards.
//
// The `top` greatest: in the first lap 64 groups of four threads each put forward the greatest logit; the top-th greatest of these is one that at least
// `top` logits reach, so whatever is below it is out; that is the border for all laps.  Those that reach it, some 1.4 times `top` a lap on logits, are
// ranked by counting, which gives the order and leaves ties to the lowest index.  Where a block takes many laps for a row they can be more than the list
// holds (20 alternatives of 152064 fp32 logits, 30 laps: some 720 of 1024, 32: 1290); the greatest are then found one by one from memory, a pass each.
//
// Measured, as captured and replayed, 152064 bf16 logits a row, no alternatives: 2000 rows 99 us (6.1 TB/s, 0.94 of the rate of a copy; bound by memory); 64 rows and 5
// alternatives 12.2 us, one row and 20 alternatives 8.3 us (latency: launch, a trip to memory, border, ranking, the cluster's join).  2000 rows with 5, 20 and 32 alternatives
// 143, 235 and 4451 us, fp32 (no alternatives 183) 213, 2953 and 31387: the last ones and that of 20 go by rows whose list overflows.
#include <math.h>
#include <stdio.h>

#include "attn_tc.cuh"
#include "bl_ops.h"
#include "heap.h"
#include "launch.h"
#include "ptx.cuh"

namespace bl {

constexpr int kScoreThreads = 256;
constexpr int kScoreLap = 5;         // vectors of a thread and lap
constexpr int kScoreTop = 32;        // alternatives at most
constexpr int kScoreGroups = 64;
constexpr int kScoreList = 1024;     // tokens that reach the border
static_assert(8 * kScoreTop == kScoreThreads, "a thread for every token that a cluster puts forward");
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct Score {
  const void* logits;
  size_t ld;
  int n;           // columns of the vocabulary, from token `offset` on
  int offset, top, n_ids, raw;
  const int* ids;  // [rows][n_ids]
  float *given, *entropy, *top_val, *parts;
  int* top_ids;
};

// Sums of a set of logits: t in units of log2.  None: m = -inf, s = t = 0.
struct ScoreSum {
  float m, s, t;
};
// (a sum whose m is +inf or that holds NaN has s = NaN: the result is NaN whichever way it is weighed)
__device__ __forceinline__ ScoreSum score_join(ScoreSum a, ScoreSum b) {
  ScoreSum r;
  r.m = fmaxf(a.m, b.m);
  const float ref = r.m == -INFINITY ? 0.f : r.m;
  // a set of nothing has no distance that could be multiplied by zero
  const float da = a.m == -INFINITY ? 0.f : (a.m - ref) * kLog2e, db = b.m == -INFINITY ? 0.f : (b.m - ref) * kLog2e;
  const float ea = ex2_approx(da), eb = ex2_approx(db);
  r.s = a.s * ea + b.s * eb;
  // (a distance of -inf comes with weight 0)
  r.t = ea * (a.t + fmaxf(da, -1e30f) * a.s) + eb * (b.t + fmaxf(db, -1e30f) * b.s);
  return r;
}
__device__ __forceinline__ ScoreSum score_xor(ScoreSum a, int lane_mask) {
  ScoreSum b;
  b.m = __shfl_xor_sync(0xffffffffu, a.m, lane_mask);
  b.s = __shfl_xor_sync(0xffffffffu, a.s, lane_mask);
  b.t = __shfl_xor_sync(0xffffffffu, a.t, lane_mask);
  return score_join(a, b);
}

// Order of tokens: the greater logit, of equals the lower index.  0: none (-inf and NaN among them).
__device__ __forceinline__ uint32_t score_order(float x) {
  if (!(x > -INFINITY)) return 0;
  const uint32_t u = __float_as_uint(x + 0.f);  // (-0 counts as 0)
  return u ^ (u >> 31 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ uint64_t score_key(float x, int idx) {
  const uint32_t u = score_order(x);
  return u ? uint64_t(u) << 32 | uint32_t(~idx) : 0;
}
__device__ __forceinline__ float score_unorder(uint32_t u) { return __uint_as_float(u >> 31 ? u ^ 0x80000000u : ~u); }
__device__ __forceinline__ float score_key_value(uint64_t k) { return k == 0 ? -INFINITY : score_unorder(uint32_t(k >> 32)); }
__device__ __forceinline__ int score_key_index(uint64_t k) { return k == 0 ? -1 : int(~uint32_t(k)); }

template <bool FP32>
struct ScoreVec {
  static constexpr int N = FP32 ? 4 : 8;
  static __device__ __forceinline__ float at(const uint4& v, int e) {
    const uint32_t w = (&v.x)[FP32 ? e : e >> 1];
    return FP32 ? __uint_as_float(w) : __uint_as_float(e & 1 ? w & 0xffff0000u : w << 16);
  }
  static __device__ __forceinline__ uint4 none() {
    return FP32 ? make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u) : make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u);
  }
  static __device__ __forceinline__ float load(const void* row, size_t i) {
    return FP32 ? static_cast<const float*>(row)[i] : __bfloat162float(static_cast<const __nv_bfloat16*>(row)[i]);
  }
  // the greatest element; NaN is passed over
  static __device__ __forceinline__ float most(const uint4& v) {
    if constexpr (FP32) return fmaxf(fmaxf(at(v, 0), at(v, 1)), fmaxf(at(v, 2), at(v, 3)));
    __nv_bfloat162 a = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&v.x), *reinterpret_cast<const __nv_bfloat162*>(&v.y));
    const __nv_bfloat162 b = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&v.z), *reinterpret_cast<const __nv_bfloat162*>(&v.w));
    a = __hmax2(a, b);
    return fmaxf(__low2float(a), __high2float(a));
  }
};

// the place of `key` among keys[0..n) (all different but for 0): how many are greater
__device__ __forceinline__ int score_rank(uint64_t key, const uint64_t* keys, int n) {
  int above = 0;
#pragma unroll 4
  for (int i = 0; i < n; ++i) above += keys[i] > key;
  return above;
}

template <bool FP32, bool TOP>
__global__ void __launch_bounds__(kScoreThreads, 4) k_token_logprobs(const Score a) {
  using V = ScoreVec<FP32>;
  constexpr int kWarps = kScoreThreads / 32;
  __shared__ float s_sum[kWarps][3];
  __shared__ float s_parts[8][3];                          // of the cluster's blocks, in the first one
  __shared__ uint64_t s_best[TOP ? 8 * kScoreTop : 1];     // their most likely tokens
  __shared__ uint32_t s_group[TOP ? kScoreGroups : 1];
  __shared__ uint64_t s_list[TOP ? kScoreList : 1];
  __shared__ uint64_t s_round[TOP ? kWarps : 1];
  __shared__ float s_border;
  __shared__ int s_count;
  pdl_launch_dependents();
  const int share = cluster_nctarank(), rank = cluster_ctarank(), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = blockIdx.x / share;
  if constexpr (TOP) {
    s_best[tid] = 0;  // (as many as threads)
    if (tid == 0) s_count = 0;
  }
  if (share > 1) cluster_arrive();
  pdl_wait();
  const uint8_t* x = static_cast<const uint8_t*>(a.logits) + size_t(row) * a.ld * (FP32 ? 4 : 2);
  // Whole vectors on 16-byte boundaries, and up to N - 1 elements ahead of them and behind, which are the first and the last block's, one to a thread.
  const int shift = int(reinterpret_cast<uintptr_t>(x) & 15) / (FP32 ? 4 : 2), head = min(a.n, (V::N - shift) % V::N);
  const uint4* vecs = reinterpret_cast<const uint4*>(x + size_t(head) * (FP32 ? 4 : 2));
  const int n_vecs = (a.n - head) / V::N, rest = (a.n - head) % V::N;
  const int per = (n_vecs + share - 1) / share, v0 = min(rank * per, n_vecs), v1 = min(v0 + per, n_vecs);
  const int single = rank == 0 && tid < head ? tid : rank == share - 1 && tid >= V::N && tid - V::N < rest ? a.n - rest + tid - V::N : -1;
  // the logits of the given tokens, asked for ahead of everything else
  const bool gives = rank == 0 && tid < a.n_ids;
  auto logit_of = [&](int id) {
    const int64_t c = int64_t(id) - a.offset;
    return id >= 0 && c >= 0 && c < a.n ? V::load(x, size_t(c)) : -INFINITY;
  };
  const float extra = single >= 0 ? V::load(x, size_t(single)) : -INFINITY;
  const float mine = gives ? logit_of(a.ids[size_t(row) * a.n_ids + tid]) : 0.f;
  auto ask = [&](uint4 (&v)[kScoreLap], int lap) {
    const uint4* from = vecs + lap + tid;
    if (lap + kScoreLap * kScoreThreads <= v1) {
#pragma unroll
      for (int j = 0; j < kScoreLap; ++j) v[j] = ld_nc_v4(from + j * kScoreThreads);
    } else {
#pragma unroll
      for (int j = 0; j < kScoreLap; ++j) {
        v[j] = V::none();
        if (lap + tid + j * kScoreThreads < v1) v[j] = ld_nc_v4(from + j * kScoreThreads);
      }
    }
  };

  ScoreSum sum = {-INFINITY, 0.f, 0.f};
  uint4 next[kScoreLap];
  ask(next, v0);
  float border = -INFINITY;
#pragma unroll 1
  for (int lap = v0; lap < v1; lap += kScoreLap * kScoreThreads) {
    uint4 v[kScoreLap];
#pragma unroll
    for (int j = 0; j < kScoreLap; ++j) v[j] = next[j];
    if (lap + kScoreLap * kScoreThreads < v1) ask(next, lap + kScoreLap * kScoreThreads);
    float each[kScoreLap], most = -INFINITY;
#pragma unroll
    for (int j = 0; j < kScoreLap; ++j) most = fmaxf(most, each[j] = V::most(v[j]));
    {
      const float ref = most == -INFINITY ? 0.f : most;
      const float2 neg = make_float2(-ref, -ref), log2e = make_float2(kLog2e, kLog2e);
      float2 ss = make_float2(0.f, 0.f), tt = make_float2(0.f, 0.f);
#pragma unroll
      for (int j = 0; j < kScoreLap; ++j)
#pragma unroll
        for (int e = 0; e < V::N; e += 2) {
          // (the difference first: it is exact or nearly so, where two rounded products would not be)
          const float2 t = mul2(add2(make_float2(V::at(v[j], e), V::at(v[j], e + 1)), neg), log2e);
          const float2 p = make_float2(ex2_approx(t.x), ex2_approx(t.y));
          ss = add2(ss, p);
          // (-inf weighs nothing; NaN is in p)
          tt = fma2(make_float2(fmaxf(t.x, -1e30f), fmaxf(t.y, -1e30f)), p, tt);
        }
      sum = score_join(sum, ScoreSum{most, ss.x + ss.y, tt.x + tt.y});
    }
    if constexpr (TOP) {
      // ---- the border ----
      if (lap == v0) {
        uint32_t key = score_order(most);
        key = max(key, __shfl_xor_sync(0xffffffffu, key, 1));
        key = max(key, __shfl_xor_sync(0xffffffffu, key, 2));
        if ((tid & 3) == 0) s_group[tid >> 2] = key;
        if (tid == 0) s_border = -INFINITY;  // fewer than `top` groups with anything: everything is looked at
        __syncthreads();
        int above = 0;
#pragma unroll
        for (int i = 0; i < kScoreGroups / 4; ++i) {
          const int g = (tid & 3) + 4 * i;
          above += s_group[g] > key || (s_group[g] == key && g < (tid >> 2));
        }
        above += __shfl_xor_sync(0xffffffffu, above, 1);
        above += __shfl_xor_sync(0xffffffffu, above, 2);
        if (key && above == a.top - 1 && (tid & 3) == 0) s_border = score_unorder(key);
        __syncthreads();
        border = s_border;  // (a border for all laps)
      }
      // ---- those that reach it ----
      uint32_t hits = 0;
#pragma unroll
      for (int j = 0; j < kScoreLap; ++j)
        if (each[j] >= border && each[j] > -INFINITY) hits |= 1u << j;
#pragma unroll 1
      for (; hits; hits &= hits - 1) {
        const int jj = __ffs(hits) - 1, at = head + (lap + jj * kScoreThreads + tid) * V::N;
        uint4 w = v[0];
#pragma unroll
        for (int j = 1; j < kScoreLap; ++j)
          if (jj == j) w = v[j];
        uint32_t these = 0;
#pragma unroll
        for (int e = 0; e < V::N; ++e) {
          const float f = V::at(w, e);
          these |= uint32_t((f >= border) & (f > -INFINITY)) << e;
        }
        int to = atomicAdd(&s_count, __popc(these));
#pragma unroll 1
        for (; these; these &= these - 1, ++to) {
          const int e = __ffs(these) - 1, q = FP32 ? e : e >> 1;
          const uint32_t word = q == 0 ? w.x : q == 1 ? w.y : q == 2 ? w.z : w.w;
          const float f = FP32 ? __uint_as_float(word) : __uint_as_float(e & 1 ? word & 0xffff0000u : word << 16);
          if (to < kScoreList) s_list[to] = score_key(f, at + e);
        }
      }
    }
  }

  if (extra > -INFINITY || extra != extra) sum = score_join(sum, ScoreSum{extra, extra - extra + 1.f, 0.f});
  // ---- this block's most likely tokens, in order, into the first block ----
  if constexpr (TOP) {
    if (v0 >= v1) __syncthreads();  // (no lap: the count is zero all the same)
    if (extra >= border && extra > -INFINITY) {
      const int to = atomicAdd(&s_count, 1);
      if (to < kScoreList) s_list[to] = score_key(extra, single);
    }
    __syncthreads();
    int n = s_count;
    if (n > kScoreList) {
      // Too many for the list (more than a thousand at the border or above: equal ones, or the greatest of a few threads): the greatest, the greatest
      // below it, and so on, from memory.
      uint64_t last = ~uint64_t(0);
#pragma unroll 1
      for (n = 0; n < a.top; ++n) {
        uint64_t best = 0;
#pragma unroll 1
        for (int i = head + v0 * V::N + tid; i < head + v1 * V::N; i += kScoreThreads) {
          const uint64_t k = score_key(V::load(x, size_t(i)), i);
          if (k < last && k > best) best = k;
        }
        const uint64_t k = score_key(extra, single);
        if (k < last && k > best) best = k;
#pragma unroll
        for (int o = 16; o; o >>= 1) {
          const uint64_t other = __shfl_xor_sync(0xffffffffu, best, o);
          best = best > other ? best : other;
        }
        if (lane == 0) s_round[warp] = best;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kWarps; ++w) best = best > s_round[w] ? best : s_round[w];
        if (tid == 0) s_list[n] = best;
        last = best;
        __syncthreads();
      }
    }
    if (share > 1) cluster_wait();  // (for the arrivals at the start) the first block runs, and its places are empty
    const uint32_t to = map_to_cta(smem_u32(s_best), 0);
#pragma unroll 1
    for (int i = tid; i < n; i += kScoreThreads) {
      const uint64_t k = s_list[i];
      const int at = k ? score_rank(k, s_list, n) : kScoreTop;
      if (at < a.top) {
        st_cluster_u32(to + 8 * (rank * a.top + at), uint32_t(k));
        st_cluster_u32(to + 8 * (rank * a.top + at) + 4, uint32_t(k >> 32));
      }
    }
  } else if (share > 1) {
    cluster_wait();
  }
  // ---- sums of threads, warps, blocks ----
#pragma unroll
  for (int o = 16; o; o >>= 1) sum = score_xor(sum, o);
  if (lane == 0) {
    s_sum[warp][0] = sum.m;
    s_sum[warp][1] = sum.s;
    s_sum[warp][2] = sum.t;
  }
  __syncthreads();
  if (warp == 0) {
    sum = lane < kWarps ? ScoreSum{s_sum[lane][0], s_sum[lane][1], s_sum[lane][2]} : ScoreSum{-INFINITY, 0.f, 0.f};
#pragma unroll
    for (int o = kWarps / 2; o; o >>= 1) sum = score_xor(sum, o);
    if (lane == 0) {
      const uint32_t to = map_to_cta(smem_u32(&s_parts[rank][0]), 0);
      st_cluster_u32(to, __float_as_uint(sum.m));
      st_cluster_u32(to + 4, __float_as_uint(sum.s));
      st_cluster_u32(to + 8, __float_as_uint(sum.t));
    }
  }
  if (share > 1) {
    cluster_sync_all();
    if (rank != 0) return;
  } else {
    __syncthreads();
  }
  sum = (lane & 7) < share ? ScoreSum{s_parts[lane & 7][0], s_parts[lane & 7][1], s_parts[lane & 7][2]} : ScoreSum{-INFINITY, 0.f, 0.f};
#pragma unroll
  for (int o = 4; o; o >>= 1) sum = score_xor(sum, o);

  // ---- results; a row without anything above -inf: no token has a probability, and nothing is uncertain ----
  const float log_s = logf(sum.s);
  const bool none = sum.m == -INFINITY && sum.s == 0.f;
  auto out = [&](float logit) { return a.raw ? logit : none ? -INFINITY : (logit - sum.m) - log_s; };
  if (gives) a.given[size_t(row) * a.n_ids + tid] = out(mine);
  for (int i = tid + kScoreThreads; i < a.n_ids; i += kScoreThreads)
    a.given[size_t(row) * a.n_ids + i] = out(logit_of(a.ids[size_t(row) * a.n_ids + i]));
  if (tid == 0) {
    if (a.raw) {
      a.parts[3 * size_t(row)] = sum.m;
      a.parts[3 * size_t(row) + 1] = sum.s;
      a.parts[3 * size_t(row) + 2] = sum.t * kLn2;
    } else {
      a.entropy[row] = none ? 0.f : log_s - sum.t * kLn2 / sum.s;
    }
  }
  if constexpr (TOP) {
    const uint64_t k = tid < share * a.top ? s_best[tid] : 0;
    const int there = __syncthreads_count(k != 0);
    const size_t to = size_t(row) * a.top;
    if (k) {
      // every block's are in order: how many are greater is found by halving, in all of them at once
      int lo[8] = {0}, at = 0;
#pragma unroll 1
      for (int step = kScoreTop; step; step >>= 1) {
        if (step > a.top) continue;
        uint64_t other[8];
#pragma unroll
        for (int b = 0; b < 8; ++b) other[b] = s_best[min(b, share - 1) * a.top + min(lo[b] + step, a.top) - 1];
#pragma unroll
        for (int b = 0; b < 8; ++b) lo[b] += (b < share) & (lo[b] + step <= a.top) & (other[b] > k) ? step : 0;
      }
#pragma unroll
      for (int b = 0; b < 8; ++b) at += lo[b];
      if (at < a.top) {
        a.top_ids[to + at] = score_key_index(k) + a.offset;
        a.top_val[to + at] = out(score_key_value(k));
      }
    }
    if (tid >= there && tid < a.top) {
      a.top_ids[to + tid] = -1;
      // (a row with NaN or +inf has no probabilities, also where nothing else is left)
      a.top_val[to + tid] = sum.s != sum.s && !a.raw ? NAN : -INFINITY;
    }
  }
}

}  // namespace bl

using namespace bl;

extern "C" int bl_token_logprobs(const blScoreArgs* s, void* stream, char* err, size_t errlen) {
  auto refuse = [&](const char* why) {
    set_err(err, errlen, "barlink: token_logprobs %s", why);
    return -1;
  };
  if (!s) return refuse("needs arguments");
  if (s->rows < 0 || s->n < 0 || s->vocab < 0 || s->offset < 0 || int64_t(s->offset) + s->n > 0x7fffffffLL - kScoreThreads) return refuse("needs token ids that fit 32 bits");
  if (s->top < 0 || s->top > kScoreTop) return refuse("gives at most 32 alternatives");
  if (s->n_ids < 0 || s->rows > 0x7fffffff / 8) return refuse("has too many rows, or fewer than no tokens");
  if (s->rows == 0) return 0;
  if ((s->n > 0 && !s->logits) || (s->n_ids && (!s->ids || !s->given)) || (s->raw ? !s->parts : !s->entropy) || (s->top && (!s->top_ids || !s->top_val)))
    return refuse("needs logits, tokens and outputs");
  if (reinterpret_cast<uintptr_t>(s->logits) % (s->fp32 ? 4 : 2)) return refuse("needs logits on their own boundaries");
  Score a;
  a.logits = s->logits;
  a.ld = s->ld;
  a.n = s->vocab <= s->offset ? 0 : (s->vocab - s->offset < s->n ? s->vocab - s->offset : s->n);
  a.offset = s->offset;
  a.top = s->top;
  a.n_ids = s->n_ids;
  a.raw = s->raw;
  a.ids = static_cast<const int*>(s->ids);
  a.given = static_cast<float*>(s->given);
  a.entropy = static_cast<float*>(s->entropy);
  a.top_ids = static_cast<int*>(s->top_ids);
  a.top_val = static_cast<float*>(s->top_val);
  a.parts = static_cast<float*>(s->parts);
  // Blocks of a row: as many as it has laps (eight at most) where there are few rows, fewer the more rows there are, so that all blocks are resident together
  // and half the places for them stay free.  152064 bf16 logits, five alternatives, 1 2 4 8 blocks a row: 1 row 20 13.5 9.0 6.8 us, 64 rows 24 18 14.7 12.3, 128 rows
  // 32 24 18.0 22.4, 256 rows 43 29 32 40.
  const int lap = kScoreThreads * kScoreLap * (s->fp32 ? 4 : 8), slots = sm_count() * 4;
  int share = 1;
  while (share < 8 && int64_t(share) * lap < a.n && int64_t(s->rows) * share * 2 <= slots) share *= 2;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto* kernel = s->fp32 ? (s->top ? k_token_logprobs<true, true> : k_token_logprobs<true, false>)
                         : (s->top ? k_token_logprobs<false, true> : k_token_logprobs<false, false>);
  cudaError_t e = launch_cluster(kernel, dim3(unsigned(s->rows) * share), dim3(kScoreThreads), 0, share, st, a);
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) {
    set_err(err, errlen, "barlink: token_logprobs launch failed: %s", cudaGetErrorString(e));
    return -1;
  }
  return 0;
}
