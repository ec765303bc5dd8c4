// SPDX-License-Identifier: MIT
//
// What a serving step does around the model: request lengths to block tables and slots, token histories to
// count tables, and the rules on the logits (penalties for repeated tokens, biases, grammar masks) with the arg max.
#include <math.h>
#include <stdio.h>

#include "bl_ops.h"
#include "heap.h"
#include "launch.h"
#include "ptx.cuh"

namespace bl {

#define SERVE_LAUNCH_CHECK(what)                                                           \
  do {                                                                                     \
    cudaError_t _e = cudaGetLastError();                                                   \
    if (_e != cudaSuccess) {                                                               \
      set_err(err, errlen, "barlink: %s launch failed: %s", what, cudaGetErrorString(_e)); \
      return -1;                                                                           \
    }                                                                                      \
  } while (0)

// ---------------------------------------------------------------------------
// block tables, row offsets, positions and slots
// ---------------------------------------------------------------------------
constexpr int kLayoutThreads = 1024;
constexpr int kLayoutMaxBatch = 8192;
constexpr int kLayoutAlone = 2048;  // rows up to which the one block writes them itself

struct RequestLayout {
  const int* new_lens;  // tokens that a request gets now; below 0: it has ended
  const int* past_lens;
  int* tables;
  int* ring;  // the free blocks: `free` of them from `head` on, around the end
  const int* range;
  int *cu, *positions, *slots, *ctx_lens, *range_out;
  int batch, width, cap, tokens, block_size;
};

// exclusive block-wide scan of three ints per thread; total in tot
__device__ __forceinline__ void block_scan3(int (&v)[3], int (&tot)[3], int (*s_warp)[3]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int in[3] = {v[0], v[1], v[2]};
#pragma unroll
  for (int o = 1; o < 32; o <<= 1)
#pragma unroll
    for (int c = 0; c < 3; ++c) {
      const int u = __shfl_up_sync(0xffffffffu, v[c], o);
      if (lane >= o) v[c] += u;
    }
  if (lane == 31)
#pragma unroll
    for (int c = 0; c < 3; ++c) s_warp[warp][c] = v[c];
  __syncthreads();
#pragma unroll
  for (int c = 0; c < 3; ++c) {
    int w = lane < kLayoutThreads / 32 ? s_warp[lane][c] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += u;
    }
    tot[c] = __shfl_sync(0xffffffffu, w, 31);
    const int before = __shfl_sync(0xffffffffu, w, warp > 0 ? warp - 1 : 0);
    v[c] += (warp > 0 ? before : 0) - in[c];
  }
  __syncthreads();
}

// last b with first[b] <= x, first[0] = 0 (requests without items are passed over)
__device__ __forceinline__ int owner_of(const int* first, int batch, int x) {
  int lo = 0, hi = batch;  // first[hi] > x
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ int pages_of(int64_t tokens, int block_size, int width) {
  const int64_t n = (tokens + block_size - 1) / block_size;
  return n < width ? int(n) : width;
}

// One block.  Three running sums over the requests (tokens, fresh blocks, blocks given back) stay in shared memory;
// every token and every fresh block then finds its request by bisection.
__global__ void __launch_bounds__(kLayoutThreads) k_paged_layout(const RequestLayout a) {
  pdl_launch_dependents();
  pdl_wait();
  extern __shared__ int s_dyn[];
  __shared__ int s_warp[kLayoutThreads / 32][3];
  __shared__ int s_ended;
  const int B = a.batch, bs = a.block_size, tid = threadIdx.x;
  int* s_cu = s_dyn;               // [B + 1]
  int* s_fresh = s_cu + B + 1;     // [B + 1]
  int* s_had = s_fresh + B + 1;    // [B] blocks in the table before
  int* s_past = s_had + B;         // [B]
  int* s_back = s_past + B;        // [B] blocks given back, then their running sum
  int* s_list = s_back + B;        // [B] requests that have ended
  const int head = a.range[0], free_n = min(max(a.range[1], 0), a.cap);
  if (tid == 0) s_ended = 0;
  __syncthreads();
  for (int b = tid; b < B; b += kLayoutThreads) {
    const int n = a.new_lens[b], past = max(a.past_lens[b], 0);
    const int had = pages_of(past, bs, a.width);
    s_cu[b] = max(n, 0);
    s_fresh[b] = n < 0 ? 0 : pages_of(int64_t(past) + n, bs, a.width) - had;
    s_had[b] = had;
    s_past[b] = past;
    s_back[b] = 0;
    if (n < 0) s_list[atomicAdd(&s_ended, 1)] = b;  // (in any order: what is kept of it is one sum per request)
  }
  __syncthreads();
  const int ended = s_ended, warp = tid >> 5, lane = tid & 31;
  for (int e = warp; e < ended; e += kLayoutThreads / 32) {
    const int b = s_list[e];
    int n = 0;
    for (int p = lane; p < s_had[b]; p += 32) n += a.tables[size_t(b) * a.width + p] >= 0;
    n = __reduce_add_sync(0xffffffffu, n);
    if (lane == 0) s_back[b] = n;
  }
  __syncthreads();
  const int per = (B + kLayoutThreads - 1) / kLayoutThreads, b0 = min(tid * per, B), b1 = min(b0 + per, B);
  int sum[3] = {0, 0, 0}, tot[3];
  for (int b = b0; b < b1; ++b) {
    sum[0] += s_cu[b];
    sum[1] += s_fresh[b];
    sum[2] += s_back[b];
  }
  block_scan3(sum, tot, s_warp);
  for (int b = b0; b < b1; ++b) {
    const int n0 = s_cu[b], n1 = s_fresh[b], n2 = s_back[b];
    a.cu[b] = s_cu[b] = sum[0];
    s_fresh[b] = sum[1];
    s_back[b] = sum[2];
    const bool gone = a.new_lens[b] < 0;  // (read before ctx_lens, which may be past_lens or new_lens)
    a.ctx_lens[b] = gone ? 0 : s_past[b] + n0;
    sum[0] += n0;
    sum[1] += n1;
    sum[2] += n2;
  }
  if (tid == 0) {
    a.cu[B] = s_cu[B] = tot[0];
    s_fresh[B] = tot[1];
    const int taken = min(tot[1], free_n), given = min(tot[2], a.cap - free_n);
    a.range_out[0] = int((int64_t(head) + taken) % a.cap);
    a.range_out[1] = free_n - taken + given;
    a.range_out[2] = max(tot[1] - free_n, 0);
  }
  __syncthreads();
  auto ring_at = [&](int i) { return int((int64_t(head) + i) % a.cap); };
  // blocks that come back go behind the free ones, in the order of requests and pages
  for (int e = warp; e < ended; e += kLayoutThreads / 32) {
    const int b = s_list[e];
    int at = free_n + s_back[b];
    for (int p0 = 0; p0 < s_had[b]; p0 += 32) {
      const int id = p0 + lane < s_had[b] ? a.tables[size_t(b) * a.width + p0 + lane] : -1;
      const uint32_t m = __ballot_sync(0xffffffffu, id >= 0);
      const int mine = at + __popc(m & ((1u << lane) - 1));
      if (id >= 0 && mine < a.cap) a.ring[ring_at(mine)] = id;
      at += __popc(m);
    }
  }
  for (int j = tid; j < tot[1]; j += kLayoutThreads) {
    const int b = owner_of(s_fresh, B, j);
    a.tables[size_t(b) * a.width + s_had[b] + j - s_fresh[b]] = j < free_n ? a.ring[ring_at(j)] : -1;
  }
  if (a.tokens > kLayoutAlone) return;  // k_layout_rows does the rest
  for (int row = tid; row < a.tokens; row += kLayoutThreads) {
    int pos = 0, slot = -1;
    if (row < tot[0]) {
      const int b = owner_of(s_cu, B, row);
      pos = s_past[b] + row - s_cu[b];
      const int page = pos / bs;
      if (pos >= 0 && page < a.width) {
        const int j = s_fresh[b] + page - s_had[b];
        const int id = page < s_had[b] ? a.tables[size_t(b) * a.width + page] : j < free_n ? a.ring[ring_at(j)] : -1;
        if (id >= 0) slot = id * bs + pos % bs;
      }
    }
    a.positions[row] = pos;
    a.slots[row] = slot;
  }
}

// The rows of many tokens, behind k_paged_layout: four rows a thread, the first by bisection, the others by going on.
__global__ void __launch_bounds__(256) k_layout_rows(const RequestLayout a) {
  pdl_launch_dependents();
  pdl_wait();
  const int row0 = (blockIdx.x * 256 + threadIdx.x) * 4, bs = a.block_size;
  if (row0 >= a.tokens) return;
  int pos[4] = {0, 0, 0, 0}, slot[4] = {-1, -1, -1, -1};
  if (row0 < a.cu[a.batch]) {
    int b = owner_of(a.cu, a.batch, row0), next = a.cu[b + 1];
    int base = a.ctx_lens[b] - next;  // position = base + row
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = row0 + i;
      while (row >= next && ++b < a.batch) {
        next = a.cu[b + 1];
        base = a.ctx_lens[b] - next;
      }
      if (b >= a.batch) break;
      pos[i] = base + row;
      const int page = pos[i] / bs;
      if (pos[i] >= 0 && page < a.width) {
        const int id = a.tables[size_t(b) * a.width + page];
        if (id >= 0) slot[i] = id * bs + pos[i] % bs;
      }
    }
  }
  if (row0 + 4 <= a.tokens && ((reinterpret_cast<uintptr_t>(a.positions) | reinterpret_cast<uintptr_t>(a.slots)) & 15) == 0) {
    *reinterpret_cast<int4*>(a.positions + row0) = make_int4(pos[0], pos[1], pos[2], pos[3]);
    *reinterpret_cast<int4*>(a.slots + row0) = make_int4(slot[0], slot[1], slot[2], slot[3]);
  } else {
    for (int i = 0; i < 4 && row0 + i < a.tokens; ++i) {
      a.positions[row0 + i] = pos[i];
      a.slots[row0 + i] = slot[i];
    }
  }
}

// ---------------------------------------------------------------------------
// token histories to count tables
// ---------------------------------------------------------------------------
// A cluster of blocks owns a row: empties its tables, if asked to, and counts its tokens behind the cluster's barrier.
constexpr int kCountThreads = 512;
__device__ __forceinline__ void zero_words(uint32_t* p, size_t n, int who, int of) {
  const size_t skip = min(n, size_t(-(reinterpret_cast<uintptr_t>(p) >> 2) & 3));  // to the next 16 bytes
  if (size_t(who) < skip) p[who] = 0;
  uint4* v = reinterpret_cast<uint4*>(p + skip);
  const size_t nv = (n - skip) / 4;
  for (size_t i = who; i < nv; i += of) v[i] = make_uint4(0, 0, 0, 0);
  const size_t at = skip + nv * 4 + who;
  if (at < n) p[at] = 0;
}
__global__ void __launch_bounds__(kCountThreads) k_count_tokens(const int* __restrict__ ids, const int* __restrict__ cu,
                                                                const int* __restrict__ prompt, int* __restrict__ counts,
                                                                uint32_t* __restrict__ seen, int n_ids, int vocab, int words, int reset) {
  pdl_launch_dependents();
  pdl_wait();
  const int row = blockIdx.x / cluster_nctarank(), who = cluster_ctarank() * kCountThreads + threadIdx.x, of = cluster_nctarank() * kCountThreads;
  counts += size_t(row) * vocab;
  seen += size_t(row) * words;
  if (reset) {
    zero_words(reinterpret_cast<uint32_t*>(counts), vocab, who, of);
    zero_words(seen, words, who, of);
    __threadfence();
    __syncwarp();
    cluster_sync_all();
  }
  const int lo = cu ? max(cu[row], 0) : row, hi = cu ? min(cu[row + 1], n_ids) : row + 1;
  const int p = prompt ? prompt[row] : 0;
  for (int i = lo + who; i < hi; i += of) {
    const int id = ids[i];
    if (id < 0 || id >= vocab) continue;
    atomicOr(seen + (id >> 5), 1u << (id & 31));
    if (i - lo >= p) atomicAdd(counts + id, 1);
  }
}

// ---------------------------------------------------------------------------
// rules on the logits
// ---------------------------------------------------------------------------
struct Rules {
  const void* logits;
  void* out;     // same type, or null
  float2* part;  // [rows] (value, token), or null
  int* idx;      // [rows], with val; or null
  float* val;
  const float* penalties;  // [rows][3]: repetition, presence, frequency; or null
  const int* counts;
  const uint32_t* seen;
  const int* bias_ids;
  const float* bias;
  const uint32_t* mask;
  int rows, n, vocab, offset, n_bias, words;
  size_t ld, ld_out, ld_mask;
};

template <typename T>
__device__ __forceinline__ float to_float(T v) {
  if constexpr (sizeof(T) == 2) return __bfloat162float(v);
  else return v;
}
template <typename T>
__device__ __forceinline__ T from_float(float v) {
  if constexpr (sizeof(T) == 2) return __float2bfloat16(v);
  else return v;
}

// bits [at, at + 8) of a row of `total` bits; those behind it are 0
__device__ __forceinline__ uint32_t bits8(const uint32_t* words, int at, int total) {
  const uint8_t* p = reinterpret_cast<const uint8_t*>(words) + (at >> 3);
  const int left = total - at, sh = at & 7;
  if (left <= 0) return 0;
  uint32_t v = p[0] >> sh;
  if (sh && left > 8 - sh) v |= uint32_t(p[1]) << (8 - sh);
  return left >= 8 ? v & 0xffu : v & ((1u << left) - 1);
}

template <typename T>
__device__ __forceinline__ void load8(const T* p, int m, bool vec, float (&x)[8]) {
  if (vec && m == 8) {
    if constexpr (sizeof(T) == 2) {
      const uint4 v = *reinterpret_cast<const uint4*>(p);
      const float2 a = unpack_bf16x2(v.x), b = unpack_bf16x2(v.y), c = unpack_bf16x2(v.z), d = unpack_bf16x2(v.w);
      x[0] = a.x; x[1] = a.y; x[2] = b.x; x[3] = b.y; x[4] = c.x; x[5] = c.y; x[6] = d.x; x[7] = d.y;
    } else {
      const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
      x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = j < m ? to_float<T>(p[j]) : -INFINITY;
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, int m, bool vec, const float (&x)[8]) {
  if (vec && m == 8) {
    if constexpr (sizeof(T) == 2) {
      *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
    } else {
      *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
      *reinterpret_cast<float4*>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < m) p[j] = from_float<T>(x[j]);
  }
}
__device__ __forceinline__ void better(float& best, int& bi, float v, int i) {
  if (v > best || (v == best && i < bi)) {
    best = v;
    bi = i;
  }
}

// A cluster of blocks shares a row, a thread takes eight neighbouring logits (16 bytes of bf16) with a byte of each bit table; only where a
// byte says so are counts and biases read.  Two such vectors are on their way at a time.  Each operation is rounded by itself
// (no fused multiply-add): the values are the formula's to the bit.  The blocks' maxima meet in the first block's shared memory.
constexpr int kRulesThreads = 512;
constexpr int kRulesShare = 8;  // blocks of a row at most
template <typename T>
__global__ void __launch_bounds__(kRulesThreads) k_logit_rules(const Rules a) {
  extern __shared__ uint32_t s_biased[];  // a bit per logit of this block's slice: some bias entry names it
  __shared__ float s_v[kRulesThreads / 32];
  __shared__ int s_i[kRulesThreads / 32];
  __shared__ uint32_t s_all[kRulesShare][2];
  pdl_launch_dependents();
  const int share = cluster_nctarank(), rank = cluster_ctarank(), row = blockIdx.x / share, tid = threadIdx.x;
  const int per = ((a.n + share - 1) / share + 7) & ~7, lo = min(rank * per, a.n), hi = min(lo + per, a.n);
  const bool pick = a.part || a.idx;
  if (pick) cluster_sync_all();  // the first block runs: its shared memory may be written
  if (a.n_bias) {
    for (int i = tid; i < (per + 31) / 32; i += kRulesThreads) s_biased[i] = 0;
    __syncthreads();
  }
  pdl_wait();
  if (a.n_bias) {
    for (int j = tid; j < a.n_bias; j += kRulesThreads) {
      const int id = a.bias_ids[size_t(row) * a.n_bias + j], at = id - a.offset - lo;
      if (id >= 0 && at >= 0 && at < hi - lo) atomicOr(s_biased + (at >> 5), 1u << (at & 31));
    }
    __syncthreads();
  }
  const T* in = static_cast<const T*>(a.logits) + size_t(row) * a.ld;
  T* out = a.out ? static_cast<T*>(a.out) + size_t(row) * a.ld_out : nullptr;
  const bool vin = (reinterpret_cast<uintptr_t>(in) & 15) == 0, vout = (reinterpret_cast<uintptr_t>(out) & 15) == 0;
  const bool pen = a.penalties != nullptr;
  const float again = pen ? a.penalties[row * 3] : 1.f, presence = pen ? a.penalties[row * 3 + 1] : 0.f,
              frequency = pen ? a.penalties[row * 3 + 2] : 0.f;
  const uint32_t* seen = a.seen + size_t(row) * a.words;
  const uint32_t* mask = a.mask + size_t(row) * a.ld_mask;
  const int* counts = a.counts + size_t(row) * a.vocab + a.offset;
  float best = -INFINITY;
  int bi = 0x7fffffff;
  constexpr int U = 2;
  for (int i0 = lo + tid * 8; i0 < hi; i0 += U * kRulesThreads * 8) {
    float x[U][8];
    uint32_t ok[U], sb[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * kRulesThreads * 8, m = min(8, hi - i);
      ok[u] = sb[u] = 0;
      if (m <= 0) continue;
      load8<T>(in + i, m, vin, x[u]);
      ok[u] = a.mask ? bits8(mask, i + a.offset, a.vocab) : 0xffu;
      if (pen) sb[u] = bits8(seen, i + a.offset, a.vocab);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * kRulesThreads * 8, m = min(8, hi - i);
      if (m <= 0) continue;
      if (sb[u]) {
        int c[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) c[j] = sb[u] >> j & (j < m) ? counts[i + j] : 0;
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (sb[u] >> j & 1) {
            float v = x[u][j];
            v = v > 0.f ? __fdiv_rn(v, again) : __fmul_rn(v, again);
            if (c[j] > 0) v = __fsub_rn(__fsub_rn(v, __fmul_rn(frequency, float(c[j]))), presence);
            x[u][j] = v;
          }
      }
      if (a.n_bias) {
        const uint32_t named = s_biased[(i - lo) >> 5] >> ((i - lo) & 31) & 0xffu;  // (whole bytes: i - lo is a multiple of 8)
        if (named) {
          for (int e = 0; e < a.n_bias; ++e) {
            const int id = a.bias_ids[size_t(row) * a.n_bias + e], at = id - a.offset - i;
            if (id < 0 || at < 0 || at >= 8) continue;
            const float v = a.bias[size_t(row) * a.n_bias + e];
#pragma unroll
            for (int j = 0; j < 8; ++j)
              if (j == at) x[u][j] = __fadd_rn(x[u][j], v);
          }
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (!(ok[u] >> j & 1)) x[u][j] = -INFINITY;
        if (j < m && x[u][j] > best) {  // (ascending: the first of equals)
          best = x[u][j];
          bi = i + j + a.offset;
        }
      }
      if (out) store8<T>(out + i, m, vout, x[u]);
    }
  }
  if (!pick) return;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) better(best, bi, __shfl_xor_sync(0xffffffffu, best, o), __shfl_xor_sync(0xffffffffu, bi, o));
  if ((tid & 31) == 0) {
    s_v[tid >> 5] = best;
    s_i[tid >> 5] = bi;
  }
  __syncthreads();
  if (tid < 32) {
    best = tid < kRulesThreads / 32 ? s_v[tid] : -INFINITY;
    bi = tid < kRulesThreads / 32 ? s_i[tid] : 0x7fffffff;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) better(best, bi, __shfl_xor_sync(0xffffffffu, best, o), __shfl_xor_sync(0xffffffffu, bi, o));
    if (tid == 0) {
      const uint32_t to = map_to_cta(smem_u32(&s_all[rank][0]), 0);
      st_cluster_u32(to, __float_as_uint(best));
      st_cluster_u32(to + 4, uint32_t(bi));
    }
    __syncwarp();
  }
  cluster_sync_all();
  if (rank == 0 && tid == 0) {
    best = -INFINITY;
    bi = 0x7fffffff;
    for (int r = 0; r < share; ++r) better(best, bi, __uint_as_float(s_all[r][0]), int(s_all[r][1]));
    if (a.part) a.part[row] = make_float2(best, __int_as_float(bi));
    if (a.idx) {
      a.idx[row] = bi == 0x7fffffff ? -1 : bi;
      a.val[row] = best;
    }
  }
}

}  // namespace bl

using namespace bl;

extern "C" int bl_paged_layout(const int* new_lens, const int* past_lens, int* block_tables, int* free_list, const int* free_range,
                               int* cu, int* positions, int* slots, int* ctx_lens, int* free_range_out, int batch, int max_blocks,
                               int n_free, int tokens, int block_size, void* stream, char* err, size_t errlen) {
  if (batch < 1 || batch > kLayoutMaxBatch || max_blocks < 1 || n_free < 1 || tokens < 0 || block_size < 1) {
    set_err(err, errlen, "barlink: paged_layout takes 1 to %d requests, a table and a list of free blocks", kLayoutMaxBatch);
    return -1;
  }
  if (int64_t(n_free) * block_size > 0x7fffffffLL || int64_t(batch) * max_blocks > 0x7fffffffLL) {
    set_err(err, errlen, "barlink: paged_layout: the cache's slots and the table's entries must fit 32 bits");
    return -1;
  }
  RequestLayout a;
  a.new_lens = new_lens; a.past_lens = past_lens; a.tables = block_tables; a.ring = free_list; a.range = free_range;
  a.cu = cu; a.positions = positions; a.slots = slots; a.ctx_lens = ctx_lens; a.range_out = free_range_out;
  a.batch = batch; a.width = max_blocks; a.cap = n_free; a.tokens = tokens; a.block_size = block_size;
  const int smem = int((size_t(batch) * 6 + 2) * sizeof(int));
  static bool attr[64] = {};
  const cudaError_t e = allow_smem(reinterpret_cast<const void*>(k_paged_layout), (kLayoutMaxBatch * 6 + 2) * int(sizeof(int)), attr);
  if (e != cudaSuccess) {
    set_err(err, errlen, "barlink: paged_layout shared memory opt-in failed: %s", cudaGetErrorString(e));
    return -1;
  }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  launch_k(k_paged_layout, dim3(1), dim3(kLayoutThreads), smem, st, a);
  SERVE_LAUNCH_CHECK("paged_layout");
  if (tokens > kLayoutAlone) {
    launch_k(k_layout_rows, dim3((tokens + 1023) / 1024), dim3(256), 0, st, a);
    SERVE_LAUNCH_CHECK("layout_rows");
  }
  return 0;
}

extern "C" int bl_count_tokens(const int* ids, const int* cu, const int* prompt_lens, int* counts, void* seen, int rows, int n_ids,
                               int vocab, int reset, void* stream, char* err, size_t errlen) {
  if (rows < 1 || vocab < 1 || (!cu && n_ids != rows)) {
    set_err(err, errlen, "barlink: count_tokens needs one id per row, or row offsets");
    return -1;
  }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int words = (vocab + 31) / 32;
  // Eight blocks a row while the GPU holds them all at once; one where a step adds a token per row.
  const int share = !cu && !reset ? 1 : rows <= 2 * sm_count() / 4 ? 8 : rows <= 2 * sm_count() ? 2 : 1;
  const cudaError_t e = launch_cluster(k_count_tokens, dim3(unsigned(rows) * share), dim3(kCountThreads), 0, share, st, ids, cu, prompt_lens,
                                       counts, static_cast<uint32_t*>(seen), n_ids, vocab, words, reset);
  if (e != cudaSuccess) {
    set_err(err, errlen, "barlink: count_tokens launch failed: %s", cudaGetErrorString(e));
    return -1;
  }
  SERVE_LAUNCH_CHECK("count_tokens");
  return 0;
}

extern "C" int bl_logit_rules(const blRulesArgs* r, void* stream, char* err, size_t errlen) {
  if (r->rows < 1 || r->n < 1 || (!r->out && !r->part && !r->idx) || !r->idx != !r->val || (r->penalties && (!r->counts || !r->seen)) ||
      (r->n_bias > 0 && (!r->bias_ids || !r->bias)) || r->vocab < 0 ||
      (r->mask && int64_t(r->mask_words) * 32 < r->vocab)) {
    set_err(err, errlen, "barlink: logit rules need logits, an output, and the tables of the rules that are set");
    return -1;
  }
  Rules a;
  a.logits = r->logits; a.out = r->out; a.part = static_cast<float2*>(r->part); a.penalties = static_cast<const float*>(r->penalties);
  a.counts = static_cast<const int*>(r->counts); a.seen = static_cast<const uint32_t*>(r->seen);
  a.bias_ids = static_cast<const int*>(r->bias_ids); a.bias = static_cast<const float*>(r->bias);
  a.mask = static_cast<const uint32_t*>(r->mask);
  a.rows = r->rows; a.n = r->n; a.vocab = r->vocab; a.offset = r->offset; a.n_bias = r->n_bias;
  a.words = (r->vocab + 31) / 32;
  a.ld = r->ld; a.ld_out = r->ld_out; a.ld_mask = r->ld_mask;
  a.idx = static_cast<int*>(r->idx); a.val = static_cast<float*>(r->val);
  // Blocks of a row: as many as leave all of them resident at once (four to an SM), none with less than 2048 logits.
  const int slots = 4 * sm_count();
  int share = 1;
  while (share < kRulesShare && r->rows * int64_t(2 * share) <= slots && r->n >= 2048 * 2 * share) share *= 2;
  const int per = (r->n + share - 1) / share + 8, smem = r->n_bias ? (per + 31) / 32 * 4 : 0;
  if (smem > 200 * 1024) {
    set_err(err, errlen, "barlink: logit rules: biases on rows of at most 1600000 logits");
    return -1;
  }
  const auto kernel = r->fp32 ? k_logit_rules<float> : k_logit_rules<__nv_bfloat16>;
  static bool attr[2][64] = {};
  cudaError_t e = smem > 40 * 1024 ? allow_smem(reinterpret_cast<const void*>(kernel), 200 * 1024, attr[r->fp32 ? 1 : 0]) : cudaSuccess;
  if (e == cudaSuccess)
    e = launch_cluster(kernel, dim3(unsigned(r->rows) * share), dim3(kRulesThreads), smem, share, static_cast<cudaStream_t>(stream), a);
  if (e != cudaSuccess) {
    set_err(err, errlen, "barlink: logit_rules launch failed: %s", cudaGetErrorString(e));
    return -1;
  }
  SERVE_LAUNCH_CHECK("logit_rules");
  return 0;
}
