// SPDX-License-Identifier: MIT
//
// Log probabilities of given tokens, the entropy of the distribution and its most likely tokens, from logits.
//
//   m = max x,  S = sum e^(x - m),  T = sum (x - m) e^(x - m)
//   logprob(id) = x_id - m - log S,  entropy = log S - T / S
//
// One pass: a thread takes its share of a row into registers (up to kScoreLap vectors of 16 bytes, all asked for at once), finds their
// maximum, adds up S and T relative to it, and looks through the same registers again for the most likely tokens.  Sums of
// threads, warps and the blocks of a cluster, which share a row, are joined afterwards.
//
// The `top` greatest: 64 groups of four threads each put forward the greatest element (of equals the first); the top-th greatest of these is
// one that at least `top` elements reach, so whatever is below it is out.  Those that reach it, hardly more than `top` on logits, are
// ranked by counting, which gives the order and leaves ties to the lowest index.
#include <math.h>
#include <stdio.h>

#include "bl_ops.h"
#include "heap.h"
#include "launch.h"
#include "ptx.cuh"

namespace bl {

constexpr int kScoreThreads = 256;
constexpr int kScoreLap = 10;        // vectors of a thread in registers: 8 blocks of a row of 152064 bf16 logits need one lap
constexpr int kScoreTop = 32;        // alternatives at most
constexpr int kScoreGroups = 64;
constexpr int kScoreList = 1024;     // tokens that reach the border
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct Score {
  const void* logits;
  size_t ld;
  int rows, n;     // n: columns of the vocabulary, from token `offset` on
  int offset, top, n_ids, raw;
  const int* ids;  // [rows][n_ids]
  float *given, *entropy, *top_val, *parts;
  int* top_ids;
};

// Sums of a set of logits: t in units of log2.  None: m = -inf, s = t = 0.
struct ScoreSum {
  float m, s, t;
};
__device__ __forceinline__ float score_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// (a sum whose m is +inf or that holds NaN has s = NaN: the result is NaN whichever way it is weighed)
__device__ __forceinline__ ScoreSum score_join(ScoreSum a, ScoreSum b) {
  ScoreSum r;
  r.m = fmaxf(a.m, b.m);
  const float ref = r.m == -INFINITY ? 0.f : r.m;
  // a set of nothing has no distance that could be multiplied by zero
  const float da = a.m == -INFINITY ? 0.f : (a.m - ref) * kLog2e, db = b.m == -INFINITY ? 0.f : (b.m - ref) * kLog2e;
  const float ea = score_ex2(da), eb = score_ex2(db);
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
__device__ __forceinline__ uint64_t score_key(float x, int idx) {
  if (!(x > -INFINITY)) return 0;
  const uint32_t u = __float_as_uint(x + 0.f);  // (-0 counts as 0)
  return uint64_t(u ^ (u >> 31 ? 0xffffffffu : 0x80000000u)) << 32 | uint32_t(~idx);
}
__device__ __forceinline__ float score_key_value(uint64_t k) {
  const uint32_t u = uint32_t(k >> 32);
  return k == 0 ? -INFINITY : __uint_as_float(u >> 31 ? u ^ 0x80000000u : ~u);
}
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
  static __device__ __forceinline__ void set(uint4& v, int e, const void* row, size_t i) {
    uint32_t& w = (&v.x)[FP32 ? e : e >> 1];
    if constexpr (FP32)
      w = static_cast<const uint32_t*>(row)[i];
    else
      w = e & 1 ? (w & 0xffffu) | uint32_t(static_cast<const uint16_t*>(row)[i]) << 16 : (w & 0xffff0000u) | static_cast<const uint16_t*>(row)[i];
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
  for (int i = 0; i < n; ++i) above += keys[i] > key;
  return above;
}

template <bool FP32, bool TOP>
__global__ void __launch_bounds__(kScoreThreads) k_token_logprobs(const Score a) {
  using V = ScoreVec<FP32>;
  constexpr int kWarps = kScoreThreads / 32;
  __shared__ float s_sum[kWarps][3];
  __shared__ float s_parts[8][3];                          // of the cluster's blocks, in the first one
  __shared__ uint64_t s_best[TOP ? 8 * kScoreTop : 1];     // their most likely tokens
  __shared__ uint64_t s_group[TOP ? kScoreGroups : 1];
  __shared__ uint64_t s_list[TOP ? kScoreList + kScoreTop : 1];
  __shared__ uint64_t s_kept[TOP ? kScoreTop : 1];         // the greatest of this block so far
  __shared__ uint64_t s_border, s_round[TOP ? kWarps : 1];
  __shared__ int s_count;
  pdl_launch_dependents();
  const int share = cluster_nctarank(), rank = cluster_ctarank(), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = blockIdx.x / share;
  pdl_wait();
  const uint8_t* x = static_cast<const uint8_t*>(a.logits) + size_t(row) * a.ld * (FP32 ? 4 : 2);
  // Vectors on 16-byte boundaries; the row starts `shift` elements into the first one.
  const int shift = int(reinterpret_cast<uintptr_t>(x) & 15) / (FP32 ? 4 : 2);
  const uint4* vecs = reinterpret_cast<const uint4*>(x - (reinterpret_cast<uintptr_t>(x) & 15));
  const int n_vecs = a.n > 0 ? int((int64_t(a.n) + shift + V::N - 1) / V::N) : 0;
  const int per = (n_vecs + share - 1) / share, v0 = min(rank * per, n_vecs), v1 = min(v0 + per, n_vecs);
  // the logits of the given tokens, asked for ahead of everything else
  const bool gives = rank == 0 && tid < a.n_ids;
  auto logit_of = [&](int id) {
    const int64_t c = int64_t(id) - a.offset;
    return id >= 0 && c >= 0 && c < a.n ? V::load(x, size_t(c)) : -INFINITY;
  };
  const float mine = gives ? logit_of(a.ids[size_t(row) * a.n_ids + tid]) : 0.f;
  if constexpr (TOP) {
    if (tid < kScoreTop) s_kept[tid] = 0;
  }

  ScoreSum sum = {-INFINITY, 0.f, 0.f};
  for (int lap = v0; lap < v1 || lap == v0; lap += kScoreLap * kScoreThreads) {
    uint4 v[kScoreLap];
#pragma unroll
    for (int j = 0; j < kScoreLap; ++j) {
      const int i = lap + j * kScoreThreads + tid;
      v[j] = V::none();
      if (i < v1) {
        const int64_t at = int64_t(i) * V::N - shift;
        if (at >= 0 && at + V::N <= a.n) {
          v[j] = ld_nc_v4(vecs + i);
        } else {
#pragma unroll
          for (int e = 0; e < V::N; ++e)
            if (at + e >= 0 && at + e < a.n) V::set(v[j], e, x, size_t(at + e));
        }
      }
    }
    float most = -INFINITY;
#pragma unroll
    for (int j = 0; j < kScoreLap; ++j) most = fmaxf(most, V::most(v[j]));
    {
      ScoreSum s = {most, 0.f, 0.f};
      const float ref = most == -INFINITY ? 0.f : most;
#pragma unroll
      for (int j = 0; j < kScoreLap; ++j)
#pragma unroll
        for (int e = 0; e < V::N; ++e) {
          const float t = (V::at(v[j], e) - ref) * kLog2e, p = score_ex2(t);
          s.s += p;
          s.t += fmaxf(t, -1e30f) * p;  // (-inf weighs nothing; NaN is in p)
        }
      sum = score_join(sum, s);
    }
    if constexpr (TOP) {
      // ---- the border: what the groups put forward ----
      int first = 0x7fffffff;
      if (most > -INFINITY) {
#pragma unroll
        for (int j = kScoreLap - 1; j >= 0; --j)
          if (V::most(v[j]) == most) {
#pragma unroll
            for (int e = V::N - 1; e >= 0; --e)
              if (V::at(v[j], e) == most) first = (lap + j * kScoreThreads + tid) * V::N - shift + e;
          }
      }
      uint64_t key = most > -INFINITY ? score_key(most, first) : 0;
#pragma unroll
      for (int o = 1; o < 4; o <<= 1) {
        const uint64_t other = __shfl_xor_sync(0xffffffffu, key, o);
        key = key > other ? key : other;
      }
      if ((tid & 3) == 0) s_group[tid >> 2] = key;
      if (tid == 0) {
        s_border = 1;  // fewer than `top` groups with anything: everything is looked at
        s_count = 0;
      }
      __syncthreads();
      int above = 0;
#pragma unroll
      for (int i = 0; i < kScoreGroups / 4; ++i) above += s_group[(tid & 3) * (kScoreGroups / 4) + i] > key;
      above += __shfl_xor_sync(0xffffffffu, above, 1);
      above += __shfl_xor_sync(0xffffffffu, above, 2);
      if (key && above == a.top - 1 && (tid & 3) == 0) s_border = key;
      __syncthreads();
      const uint64_t border = s_border;
      const float bv = border == 1 ? -INFINITY : score_key_value(border);
      // ---- those that reach it ----
#pragma unroll
      for (int j = 0; j < kScoreLap; ++j) {
        if (!(V::most(v[j]) >= bv)) continue;
        const int at = (lap + j * kScoreThreads + tid) * V::N - shift;
#pragma unroll
        for (int e = 0; e < V::N; ++e) {
          const float f = V::at(v[j], e);
          if (f >= bv) {
            const uint64_t k = score_key(f, at + e);
            if (k >= border) {
              const int to = atomicAdd(&s_count, 1);
              if (to < kScoreList) s_list[to] = k;
            }
          }
        }
      }
      __syncthreads();
      int n = s_count;
      if (n > kScoreList) {
        // Too many for the list (more than a thousand of a block's logits above the border: none that a model computes): the greatest, the
        // greatest below it, and so on.
        uint64_t last = ~uint64_t(0);
        for (n = 0; n < a.top; ++n) {
          uint64_t best = 0;
#pragma unroll
          for (int j = 0; j < kScoreLap; ++j)
#pragma unroll
            for (int e = 0; e < V::N; ++e) {
              const uint64_t k = score_key(V::at(v[j], e), (lap + j * kScoreThreads + tid) * V::N - shift + e);
              if (k < last && k > best) best = k;
            }
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
      // with what earlier laps left
      if (lap > v0 && tid < a.top) s_list[n + tid] = s_kept[tid];
      if (lap > v0) n += a.top;
      __syncthreads();
      if (lap > v0 && tid < kScoreTop) s_kept[tid] = 0;
      if (lap > v0) __syncthreads();
      for (int i = tid; i < n; i += kScoreThreads) {
        const uint64_t k = s_list[i];
        if (k == 0) continue;
        const int at = score_rank(k, s_list, n);
        if (at < a.top) s_kept[at] = k;
      }
      __syncthreads();
    }
  }

  // ---- threads, warps, blocks of the cluster ----
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
  }
  if (share > 1) {
    cluster_sync_all();  // the first block runs: its shared memory may be written
    if (tid == 0) {
      const uint32_t to = map_to_cta(smem_u32(&s_parts[rank][0]), 0);
      st_cluster_u32(to, __float_as_uint(sum.m));
      st_cluster_u32(to + 4, __float_as_uint(sum.s));
      st_cluster_u32(to + 8, __float_as_uint(sum.t));
    }
    if constexpr (TOP) {
      if (tid < a.top) {
        const uint32_t to = map_to_cta(smem_u32(&s_best[rank * a.top + tid]), 0);
        st_cluster_u32(to, uint32_t(s_kept[tid]));
        st_cluster_u32(to + 4, uint32_t(s_kept[tid] >> 32));
      }
    }
    cluster_sync_all();
    if (rank != 0) return;
    sum = {s_parts[0][0], s_parts[0][1], s_parts[0][2]};
    for (int i = 1; i < share; ++i) sum = score_join(sum, ScoreSum{s_parts[i][0], s_parts[i][1], s_parts[i][2]});
  } else {
    if (tid == 0) {
      s_parts[0][0] = sum.m;
      s_parts[0][1] = sum.s;
      s_parts[0][2] = sum.t;
    }
    __syncthreads();
    sum = {s_parts[0][0], s_parts[0][1], s_parts[0][2]};
  }

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
    const uint64_t* keys = share > 1 ? s_best : s_kept;
    const int n = share > 1 ? share * a.top : a.top;
    if (share > 1) {
      // places that no token takes
      if (tid < kScoreTop) s_kept[tid] = 0;
      __syncthreads();
      for (int i = tid; i < n; i += kScoreThreads) {
        const uint64_t k = keys[i];
        const int at = k ? score_rank(k, keys, n) : kScoreTop;
        if (at < a.top) s_kept[at] = k;
      }
      __syncthreads();
    }
    if (tid < a.top) {
      const uint64_t k = s_kept[tid];
      const int idx = score_key_index(k);
      const size_t to = size_t(row) * a.top + tid;
      a.top_ids[to] = idx < 0 ? -1 : idx + a.offset;
      // (a row with NaN or +inf has no probabilities, also where nothing else is left)
      a.top_val[to] = k || sum.s != sum.s ? out(score_key_value(k)) : -INFINITY;
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
  if (s->rows < 0 || s->n < 0 || s->vocab < 0 || s->offset < 0 || int64_t(s->offset) + s->n > 0x7fffffffLL) return refuse("needs token ids that fit 32 bits");
  if (s->top < 0 || s->top > kScoreTop) return refuse("gives at most 32 alternatives");
  if (s->n_ids < 0 || s->rows > 0x7fffffff / 8) return refuse("has too many rows, or fewer than no tokens");
  if (s->rows == 0) return 0;
  if ((s->n > 0 && !s->logits) || (s->n_ids && (!s->ids || !s->given)) || (s->raw ? !s->parts : !s->entropy) || (s->top && (!s->top_ids || !s->top_val)))
    return refuse("needs logits, tokens and outputs");
  if (reinterpret_cast<uintptr_t>(s->logits) % (s->fp32 ? 4 : 2)) return refuse("needs logits on their own boundaries");
  Score a;
  a.logits = s->logits;
  a.ld = s->ld;
  a.rows = s->rows;
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
  // A lap's worth of a row to a block, eight blocks to a row at most.
  const int lap = kScoreThreads * kScoreLap * (s->fp32 ? 4 : 8);
  int share = 1;
  while (share < 8 && int64_t(share) * lap < a.n) share *= 2;
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
