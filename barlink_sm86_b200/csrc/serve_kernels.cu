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
constexpr int kLayoutMaxBatch = 8192;
// Rows up to which the one block writes them itself.  us, alone and with a second kernel: 64 requests with 2048 rows 6.1 and 6.7, with 4096
// 8.8 and 6.8; 256 requests 5.5 and 6.4, 9.6 and 7.2.
constexpr int kLayoutAlone = 2048;

struct RequestLayout {
  const int* new_lens;  // tokens that a request gets now; below 0: it has ended
  const int* past_lens;
  int* tables;
  int* ring;  // the free blocks: `free` of them from `head` on, around the end
  const int* range;
  int *cu, *positions, *slots, *ctx_lens, *range_out;
  int batch, width, cap, tokens, block_size;
  int per;  // rows of a request where every request has as many (those behind its tokens are empty); 0: packed
  int* lost;  // += tokens that have a row and no slot; or null
};

// exclusive block-wide scan of three ints per thread; total in tot
template <int T>
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
    int w = lane < T / 32 ? s_warp[lane][c] : 0;
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
template <int T>
__global__ void __launch_bounds__(T) k_paged_layout(const RequestLayout a) {
  pdl_launch_dependents();
  pdl_wait();
  extern __shared__ int s_dyn[];
  __shared__ int s_warp[T / 32][3];
  __shared__ int s_ended;
  const int B = a.batch, bs = a.block_size, tid = threadIdx.x;
  int* s_cu = s_dyn;               // [B + 1]
  int* s_fresh = s_cu + B + 1;     // [B + 1]
  int* s_had = s_fresh + B + 1;    // [B] blocks in the table before
  int* s_past = s_had + B;         // [B]
  int* s_back = s_past + B;        // [B] blocks given back, then their running sum
  int* s_list = s_back + B;        // [B] requests that have ended
  // (whatever stands there: an entry of the ring, and no more free blocks than it has)
  const int first = a.range[0] % a.cap, head = first < 0 ? first + a.cap : first, free_n = min(max(a.range[1], 0), a.cap);
  if (tid == 0) s_ended = 0;
  __syncthreads();
  for (int b = tid; b < B; b += T) {
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
  for (int e = warp; e < ended; e += T / 32) {
    const int b = s_list[e];
    int n = 0;
    for (int p = lane; p < s_had[b]; p += 32) n += a.tables[size_t(b) * a.width + p] >= 0;
    n = __reduce_add_sync(0xffffffffu, n);
    if (lane == 0) s_back[b] = n;
  }
  __syncthreads();
  const int per = (B + T - 1) / T, b0 = min(tid * per, B), b1 = min(b0 + per, B);
  int sum[3] = {0, 0, 0}, tot[3];
  for (int b = b0; b < b1; ++b) {
    sum[0] += s_cu[b];
    sum[1] += s_fresh[b];
    sum[2] += s_back[b];
  }
  block_scan3<T>(sum, tot, s_warp);
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
  for (int e = warp; e < ended; e += T / 32) {
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
  for (int j = tid; j < tot[1]; j += T) {
    const int b = owner_of(s_fresh, B, j);
    a.tables[size_t(b) * a.width + s_had[b] + j - s_fresh[b]] = j < free_n ? a.ring[ring_at(j)] : -1;
  }
  if (a.tokens > kLayoutAlone) return;  // k_layout_rows does the rest
  int lost = 0;
  for (int row = tid; row < a.tokens; row += T) {
    int pos = 0, slot = -1, b = -1, i = 0;  // the i-th token of request b
    if (a.per > 0) {
      b = row / a.per;
      i = row - b * a.per;
      if (b >= B || i >= s_cu[b + 1] - s_cu[b]) b = -1;
    } else if (row < tot[0]) {
      b = owner_of(s_cu, B, row);
      i = row - s_cu[b];
    }
    if (b >= 0) {
      pos = s_past[b] + i;
      const int page = pos / bs;
      if (pos >= 0 && page < a.width) {
        const int j = s_fresh[b] + page - s_had[b];
        const int id = page < s_had[b] ? a.tables[size_t(b) * a.width + page] : j < free_n ? a.ring[ring_at(j)] : -1;
        if (id >= 0) slot = id * bs + pos % bs;
      }
      lost += slot < 0;
    }
    a.positions[row] = pos;
    a.slots[row] = slot;
  }
  if (lost > 0 && a.lost) atomicAdd(a.lost, lost);
}

// The rows of many tokens, behind k_paged_layout: four rows a thread, the first by bisection of the offsets in shared memory, the others by
// going on.
__global__ void __launch_bounds__(256) k_layout_rows(const RequestLayout a) {
  extern __shared__ int s_dyn[];  // [batch + 1] row offsets, where the rows are packed
  pdl_launch_dependents();
  pdl_wait();
  const int row0 = (blockIdx.x * 256 + threadIdx.x) * 4, bs = a.block_size;
  if (a.per == 0) {
    for (int b = threadIdx.x; b <= a.batch; b += 256) s_dyn[b] = a.cu[b];
    __syncthreads();
  }
  if (row0 >= a.tokens) return;
  int pos[4] = {0, 0, 0, 0}, slot[4] = {-1, -1, -1, -1};
  int b = a.per > 0 ? row0 / a.per : row0 < s_dyn[a.batch] ? owner_of(s_dyn, a.batch, row0) : a.batch;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int row = row0 + k;
    if (a.per > 0) b = row / a.per;
    else
      while (b < a.batch && row >= s_dyn[b + 1]) ++b;
    if (b >= a.batch) break;
    const int first = a.per > 0 ? a.cu[b] : s_dyn[b], n = (a.per > 0 ? a.cu[b + 1] : s_dyn[b + 1]) - first, i = row - (a.per > 0 ? b * a.per : first);
    if (i >= n) continue;
    pos[k] = a.ctx_lens[b] - n + i;
    const int page = pos[k] / bs;
    if (pos[k] >= 0 && page < a.width) {
      const int id = a.tables[size_t(b) * a.width + page];
      if (id >= 0) slot[k] = id * bs + pos[k] % bs;
    }
    if (slot[k] < 0 && a.lost) atomicAdd(a.lost, 1);
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
// Tokens added to tables that stand.
constexpr int kCountThreads = 512;
__global__ void __launch_bounds__(kCountThreads) k_count_tokens(const int* __restrict__ ids, const int* __restrict__ cu,
                                                                const int* __restrict__ prompt, int* __restrict__ counts,
                                                                uint32_t* __restrict__ seen, int n_ids, int vocab, int words) {
  pdl_launch_dependents();
  pdl_wait();
  const int row = blockIdx.y;
  const int lo = cu ? max(cu[row], 0) : row, hi = cu ? min(cu[row + 1], n_ids) : row + 1;
  const int p = prompt ? prompt[row] : 0;
  for (int64_t i = int64_t(lo) + blockIdx.x * kCountThreads + threadIdx.x; i < hi; i += gridDim.x * kCountThreads) {
    const int id = ids[i];
    if (id < 0 || id >= vocab) continue;
    atomicOr(seen + size_t(row) * words + (id >> 5), 1u << (id & 31));
    if (i - lo >= p) atomicAdd(counts + size_t(row) * vocab + id, 1);
  }
}
// Tables made anew: block (slice, row) counts the row's tokens of its slice of the vocabulary in shared memory and writes the slice, so
// that the tables are written once and nobody waits for zeros.  64 x 152064: 9.8 us; zeros, a fence, then counting in global memory
// 11; a fill of the 40 MB alone 6.1.
constexpr int kCountSlice = 19456;  // tokens, a multiple of 32
__global__ void __launch_bounds__(kCountThreads) k_count_anew(const int* __restrict__ ids, const int* __restrict__ cu,
                                                              const int* __restrict__ prompt, int* __restrict__ counts,
                                                              uint32_t* __restrict__ seen, int n_ids, int vocab, int words, int slice) {
  extern __shared__ __align__(16) int s_slice[];  // counts from `pad` on, so that their 16-byte vectors are the table's; the bits
  pdl_launch_dependents();
  const int row = blockIdx.y, first = blockIdx.x * slice, n = min(slice, vocab - first), tid = threadIdx.x;
  int* to = counts + size_t(row) * vocab + first;
  const int pad = int((reinterpret_cast<uintptr_t>(to) >> 2) & 3);
  int* s_count = s_slice + pad;
  uint32_t* s_seen = reinterpret_cast<uint32_t*>(s_slice + slice + 4);
  for (int i = tid; i < (slice + 4 + slice / 32) / 4; i += kCountThreads) reinterpret_cast<int4*>(s_slice)[i] = make_int4(0, 0, 0, 0);
  __syncthreads();
  pdl_wait();
  const int lo = cu ? max(cu[row], 0) : row, hi = cu ? min(cu[row + 1], n_ids) : row + 1;
  const int p = prompt ? prompt[row] : 0;
  for (int64_t i0 = int64_t(lo) + tid; i0 < hi; i0 += 4 * kCountThreads) {
    int id[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) id[j] = i0 + j * kCountThreads < hi ? ids[i0 + j * kCountThreads] : -1;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int at = id[j] - first;
      if (id[j] < 0 || at < 0 || at >= n) continue;
      atomicOr(s_seen + (at >> 5), 1u << (at & 31));
      if (i0 + j * kCountThreads - lo >= p) atomicAdd(s_count + at, 1);
    }
  }
  __syncthreads();
  const int skip = min((4 - pad) & 3, n), nv = (n - skip) / 4;
  if (tid < skip) to[tid] = s_count[tid];
  for (int i = tid; i < nv; i += kCountThreads)
    reinterpret_cast<int4*>(to + skip)[i] = reinterpret_cast<const int4*>(s_count + skip)[i];
  for (int i = skip + 4 * nv + tid; i < n; i += kCountThreads) to[i] = s_count[i];
  for (int i = tid; i < (n + 31) / 32; i += kCountThreads) seen[size_t(row) * words + first / 32 + i] = s_seen[i];
}

// ---------------------------------------------------------------------------
// rules on the logits
// ---------------------------------------------------------------------------
struct Rules {
  const void* logits;
  void* out;     // same type, or null
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

// the top bits of bytes `s & 7` of v, each spread over a byte (a selector of 8 + byte)
__device__ __forceinline__ uint32_t spread_signs(uint32_t v, uint32_t s) {
  uint32_t r;
  asm("prmt.b32 %0, %1, 0, %2;" : "=r"(r) : "r"(v), "r"(s));
  return r;
}
// eight neighbouring logits as they lie, 16-byte aligned
template <typename T>
struct Eight;
template <>
struct Eight<__nv_bfloat16> {
  uint32_t w[4];
  __device__ __forceinline__ void load(const __nv_bfloat16* p) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
  }
  __device__ __forceinline__ void store(__nv_bfloat16* p) const { *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]); }
  __device__ __forceinline__ float get(int j) const { return __uint_as_float(j & 1 ? w[j >> 1] & 0xffff0000u : w[j >> 1] << 16); }
  // -inf where the bit is 0: four bits become the top bits of four bytes, which a byte permutation spreads over the halves
  __device__ __forceinline__ void keep(uint32_t bits) {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const uint32_t top = ((bits >> (4 * q) & 15u) * 0x10204080u) & 0x80808080u;
      const uint32_t m0 = spread_signs(top, 0x9988), m1 = spread_signs(top, 0xbbaa);
      w[2 * q] = (w[2 * q] & m0) | (~m0 & 0xff80ff80u);
      w[2 * q + 1] = (w[2 * q + 1] & m1) | (~m1 & 0xff80ff80u);
    }
  }
  __device__ __forceinline__ float top() const {  // (a NaN is passed over)
    auto h = [](uint32_t v) { return *reinterpret_cast<const __nv_bfloat162*>(&v); };
    const float2 m = __bfloat1622float2(__hmax2(__hmax2(h(w[0]), h(w[1])), __hmax2(h(w[2]), h(w[3]))));
    return fmaxf(m.x, m.y);
  }
};
template <>
struct Eight<float> {
  float x[8];
  __device__ __forceinline__ void load(const float* p) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
  }
  __device__ __forceinline__ void store(float* p) const {
    *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
  }
  __device__ __forceinline__ float get(int j) const { return x[j]; }
  __device__ __forceinline__ void keep(uint32_t bits) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (!(bits >> j & 1)) x[j] = -INFINITY;
  }
  __device__ __forceinline__ float top() const {
    return fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
  }
};
// the bytes that hold bits [at, at + 8)
__device__ __forceinline__ uint32_t two_bytes(const uint32_t* words, int at, bool both) {
  const uint8_t* p = reinterpret_cast<const uint8_t*>(words) + (at >> 3);
  uint32_t v = p[0];
  if (both) v |= uint32_t(p[1]) << 8;
  return v;
}

__device__ __forceinline__ void better(float& best, int& bi, float v, int i) {
  if (v > best || (v == best && i < bi)) {
    best = v;
    bi = i;
  }
}

// the same over a warp, as integers in the numbers' order (none of them NaN; -0 and 0 are equal)
__device__ __forceinline__ void warp_best(float& best, int& bi) {
  const uint32_t b = __float_as_uint(best + 0.f), key = b ^ (b >> 31 ? 0xffffffffu : 0x80000000u);
  const uint32_t top = __reduce_max_sync(0xffffffffu, key);
  bi = __reduce_min_sync(0xffffffffu, key == top ? bi : 0x7fffffff);
  best = __uint_as_float(top ^ (top >> 31 ? 0x80000000u : 0xffffffffu));
}

// A cluster of blocks shares a row.  Most tokens carry no rule but the mask, and those that do lie close together (frequent tokens
// have low ids), so there are two passes: the first takes eight neighbouring logits to a thread, 16 bytes of bf16, several such
// vectors on their way at a time, with a byte of each bit table; it lists the tokens that were seen, and leaves them
// and the ones with a bias aside.  The second gives a listed token to a thread, and a bias entry.  Of the maximum the
// first pass keeps the vector, and looks for the place in it at the end.  Each operation is rounded by itself (no fused multiply-add):
// the values are the formula's to the bit.  The blocks' maxima meet in the first block's shared memory.  Measured, 64 x 152064,
// us: one pass that branches into the penalties for every vector with a seen token 30; the seen words dealt out to warps 20.
constexpr int kRulesThreads = 512;
constexpr int kRulesShare = 8;    // blocks of a row at most
// Vectors that a thread takes at a time.  us with 2, 3, 4, 5, 6, 8: 64 x 152064 7.9, 8.1, 8.2, 7.8, 8.6, 13.7; 256 x 152064 25.1, 23.9, 24.1, 23.8,
// 25.8, 47; 64 x 50257 5.8, 6.1, 5.8, 5.9, 6.4, 9.4; 64 x 32000, where few threads have as many, 4.1, 4.4, 4.8, 4.9, 5.4, 7.5.
constexpr int kRulesLap = 5;
// Seen tokens of a block that are put off; what is beyond is dealt with on the spot.  1024 to 8192 take the same time, rows of 8000 tokens
// among them.
constexpr int kRulesList = 6144;
template <typename T, bool PICK>  // the arg max, or the logits under the rules
__global__ void __launch_bounds__(kRulesThreads, 2) k_logit_rules(const Rules a) {
  extern __shared__ uint32_t s_rules[];  // with biases: a bit per column that an entry names; the entries' columns and values
  __shared__ float s_v[kRulesThreads / 32];
  __shared__ int s_i[kRulesThreads / 32];
  __shared__ uint32_t s_all[kRulesShare][2];
  __shared__ int s_list[kRulesList];  // columns
  __shared__ int s_listed;
  pdl_launch_dependents();
  const int share = cluster_nctarank(), rank = cluster_ctarank(), row = blockIdx.x / share, tid = threadIdx.x, lane = tid & 31;
  const bool pen = a.penalties != nullptr;
  if (PICK) cluster_sync_all();  // the first block runs: its shared memory may be written
  uint32_t* s_named = s_rules;
  int* s_col = reinterpret_cast<int*>(s_rules + (a.n + 31) / 32);
  float* s_add = reinterpret_cast<float*>(s_col + a.n_bias);
  if (tid == 0) s_listed = 0;
  if (a.n_bias)
    for (int i = tid; i < (a.n + 31) / 32; i += kRulesThreads) s_named[i] = 0;
  __syncthreads();
  pdl_wait();
  if (a.n_bias) {
    for (int j = tid; j < a.n_bias; j += kRulesThreads) {
      const int id = a.bias_ids[size_t(row) * a.n_bias + j], at = id >= a.offset && id - a.offset < a.n ? id - a.offset : -1;
      s_col[j] = at;  // (below 0: none of this slice)
      s_add[j] = a.bias[size_t(row) * a.n_bias + j];
      if (at >= 0) atomicOr(s_named + (at >> 5), 1u << (at & 31));
    }
    __syncthreads();
  }
  const T* in = static_cast<const T*>(a.logits) + size_t(row) * a.ld;
  T* out = PICK ? nullptr : static_cast<T*>(a.out) + size_t(row) * a.ld_out;
  const uint32_t* seen = a.seen + size_t(row) * a.words;
  const uint32_t* mask = a.mask + size_t(row) * a.ld_mask;
  const int* counts = a.counts + size_t(row) * a.vocab + a.offset;
  const float again = pen ? a.penalties[row * 3] : 1.f, presence = pen ? a.penalties[row * 3 + 1] : 0.f,
              frequency = pen ? a.penalties[row * 3 + 2] : 0.f;
  auto penalised = [&](float x, int c) {
    x = x > 0.f ? __fdiv_rn(x, again) : __fmul_rn(x, again);
    return c > 0 ? __fsub_rn(__fsub_rn(x, __fmul_rn(frequency, float(c))), presence) : x;
  };
  float best = -INFINITY;
  int bi = 0x7fffffff;
  auto seen_token = [&](int i) {
    const float x = penalised(to_float<T>(in[i]), counts[i]);
    if (PICK) better(best, bi, x, i + a.offset);
    else out[i] = from_float<T>(x);
  };
  // vectors from the row's first 16-byte boundary on, as far as the vocabulary goes; the few columns around them one by one
  const int known = int(max(min(int64_t(a.n), int64_t(a.vocab) - a.offset), int64_t(0)));
  const int skip = min(int((16 - (reinterpret_cast<uintptr_t>(in) & 15)) % 16 / sizeof(T)), known), nvec = (known - skip) / 8;
  const bool vout = (reinterpret_cast<uintptr_t>(out + skip) & 15) == 0;
  const int sh = (a.offset + skip) & 7, lap = share * kRulesThreads;
  constexpr int U = sizeof(T) == 2 ? kRulesLap : 3;
  Eight<T> kept;  // the vector of the first pass's maximum
  float kept_top = -INFINITY;
  int kept_at = -1;
  // (a warp's 32 vectors in turn with the other blocks': frequent tokens lie together)
  for (int lap0 = 0; lap0 < nvec; lap0 += U * lap) {
    const int v0 = min(lap0 + ((tid >> 5) * share + rank) * 32 + lane, nvec - 1), mine0 = lap0 + ((tid >> 5) * share + rank) * 32 + lane;
    Eight<T> x[U];
    uint32_t okb[U], sb[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int v = mine0 + u * lap, i = skip + 8 * (v < nvec ? v : v0);
      x[u].load(in + i);
      okb[u] = a.mask ? two_bytes(mask, i + a.offset, sh != 0) : 0xffffu;
      sb[u] = pen ? two_bytes(seen, i + a.offset, sh != 0) : 0u;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int v = mine0 + u * lap, i = skip + 8 * v;
      if (v >= nvec) break;
      const uint32_t ok = okb[u] >> sh & 0xffu;
      uint32_t aside = sb[u] >> sh & 0xffu, mine = aside & ok;
      if (a.n_bias) {
        const uint32_t named = __funnelshift_r(s_named[i >> 5], s_named[min((i >> 5) + 1, (a.n - 1) >> 5)], i & 31);
        mine &= ~named;
        aside |= named;
      }
      x[u].keep(PICK ? ok & ~aside : ok);
      if (!PICK) {
        if (vout) x[u].store(out + i);
        else
#pragma unroll
          for (int j = 0; j < 8; ++j) out[i + j] = from_float<T>(x[u].get(j));
      }
      if (mine) {  // (behind the store, which has the token as it was)
        int at = atomicAdd(&s_listed, __popc(mine));
#pragma unroll 1
        for (; mine; mine &= mine - 1, ++at) {
          if (at < kRulesList) s_list[at] = i + __ffs(mine) - 1;
          else seen_token(i + __ffs(mine) - 1);
        }
      }
      if (PICK) {
        const float m = x[u].top();
        if (m > kept_top) {  // (ascending: the first of equals)
          kept_top = m;
          kept = x[u];
          kept_at = i;
        }
      }
    }
  }
  if (kept_at >= 0) {
    int at = 0;
#pragma unroll
    for (int j = 7; j >= 0; --j)
      if (kept.get(j) == kept_top) at = j;
    better(best, bi, kept_top, kept_at + at + a.offset);
  }
  __syncthreads();
  for (int e = tid, listed = min(s_listed, kRulesList); e < listed; e += kRulesThreads) seen_token(s_list[e]);
  const int tail = skip + 8 * nvec;
  for (int e = rank * kRulesThreads + tid; e < skip + a.n - tail; e += lap) {
    const int i = e < skip ? e : tail + e - skip, id = i + a.offset;
    const bool in_vocab = i < known;
    const bool ok = in_vocab && (!a.mask || (mask[id >> 5] >> (id & 31) & 1));
    const bool named = a.n_bias && (s_named[i >> 5] >> (i & 31) & 1);
    float x = ok ? to_float<T>(in[i]) : -INFINITY;
    if (ok && !named && pen && (seen[id >> 5] >> (id & 31) & 1)) x = penalised(x, counts[i]);
    if (!PICK) out[i] = from_float<T>(x);
    else if (!named) better(best, bi, x, id);
  }
  if (!PICK && a.n_bias) {
    // the bias entries overwrite what the first pass has copied, in whichever block
    __threadfence();
    __syncwarp();
    cluster_sync_all();
  }
  // (from the last warp on: the first ones have the list)
  for (int j = rank * kRulesThreads + kRulesThreads - 1 - tid; j < a.n_bias; j += lap) {
    const int col = s_col[j], id = col + a.offset;
    bool go = col >= 0;
    for (int e = 0; go && e < j; ++e) go = s_col[e] != col;  // the first entry of a token adds them all
    if (!go) continue;
    const bool in_vocab = col < known;
    const uint32_t mw = !in_vocab ? 0u : a.mask ? mask[id >> 5] : ~0u, sw = pen && in_vocab ? seen[id >> 5] : 0u;
    const int c = pen && in_vocab ? counts[col] : 0;
    float x = to_float<T>(in[col]);
    if (!(mw >> (id & 31) & 1)) continue;
    if (sw >> (id & 31) & 1) x = penalised(x, c);
    for (int e = j; e < a.n_bias; ++e)
      if (s_col[e] == col) x = __fadd_rn(x, s_add[e]);
    if (PICK) better(best, bi, x, id);
    else out[col] = from_float<T>(x);
  }
  if (!PICK) return;
  __syncwarp();
  warp_best(best, bi);
  if (lane == 0) {
    s_v[tid >> 5] = best;
    s_i[tid >> 5] = bi;
  }
  __syncthreads();
  if (tid < 32) {
    best = tid < kRulesThreads / 32 ? s_v[tid] : -INFINITY;
    bi = tid < kRulesThreads / 32 ? s_i[tid] : 0x7fffffff;
    warp_best(best, bi);
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
    if (best == -INFINITY) bi = 0x7fffffff;
    a.idx[row] = bi == 0x7fffffff ? -1 : bi;
    a.val[row] = best;
  }
}

}  // namespace bl

using namespace bl;

extern "C" int bl_paged_layout(const int* new_lens, const int* past_lens, int* block_tables, int* free_list, const int* free_range,
                               int* cu, int* positions, int* slots, int* ctx_lens, int* free_range_out, int batch, int max_blocks,
                               int n_free, int tokens, int block_size, int rows_per_request, void* stream, char* err, size_t errlen) {
  return bl_paged_layout_counting(new_lens, past_lens, block_tables, free_list, free_range, cu, positions, slots, ctx_lens, free_range_out, batch,
                                  max_blocks, n_free, tokens, block_size, rows_per_request, nullptr, stream, err, errlen);
}

extern "C" int bl_paged_layout_counting(const int* new_lens, const int* past_lens, int* block_tables, int* free_list, const int* free_range,
                                        int* cu, int* positions, int* slots, int* ctx_lens, int* free_range_out, int batch, int max_blocks,
                                        int n_free, int tokens, int block_size, int rows_per_request, int* lost, void* stream, char* err,
                                        size_t errlen) {
  if (batch < 1 || batch > kLayoutMaxBatch || max_blocks < 1 || n_free < 1 || tokens < 0 || tokens > 1 << 30 || block_size < 1 ||
      rows_per_request < 0) {
    set_err(err, errlen, "barlink: paged_layout takes 1 to %d requests, up to 2^30 tokens, a table and a list of free blocks", kLayoutMaxBatch);
    return -1;
  }
  if (int64_t(n_free) * block_size > 0x7fffffffLL || int64_t(batch) * max_blocks > 0x7fffffffLL) {
    set_err(err, errlen, "barlink: paged_layout: the cache's slots and the table's entries must fit 32 bits");
    return -1;
  }
  if (!new_lens || !past_lens || !block_tables || !free_list || !free_range || !cu || !ctx_lens || !free_range_out ||
      (tokens > 0 && (!positions || !slots))) {
    set_err(err, errlen, "barlink: paged_layout needs its lengths, table, list and range of free blocks, and all outputs");
    return -1;
  }
  RequestLayout a;
  a.new_lens = new_lens; a.past_lens = past_lens; a.tables = block_tables; a.ring = free_list; a.range = free_range;
  a.cu = cu; a.positions = positions; a.slots = slots; a.ctx_lens = ctx_lens; a.range_out = free_range_out;
  a.batch = batch; a.width = max_blocks; a.cap = n_free; a.tokens = tokens; a.block_size = block_size; a.per = rows_per_request;
  a.lost = lost;
  const int smem = int((size_t(batch) * 6 + 2) * sizeof(int));
  static bool attr[64] = {};
  const cudaError_t e = allow_smem(reinterpret_cast<const void*>(k_paged_layout<1024>), (kLayoutMaxBatch * 6 + 2) * int(sizeof(int)), attr);
  if (e != cudaSuccess) {
    set_err(err, errlen, "barlink: paged_layout shared memory opt-in failed: %s", cudaGetErrorString(e));
    return -1;
  }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  // A decode step: a block whose barriers are cheap, while it has a row and a request for each thread at most.  us, 256 and 1024 threads:
  // 64 requests of one token 3.1 and 3.7, 256 3.3 and 3.9, 256 of two 4.2 and 3.9, 512 4.9 and 4.1.
  const bool few = batch <= 256 && tokens <= 256;
  launch_k(few ? k_paged_layout<256> : k_paged_layout<1024>, dim3(1), dim3(few ? 256 : 1024), smem, st, a);
  SERVE_LAUNCH_CHECK("paged_layout");
  if (tokens > kLayoutAlone) {
    launch_k(k_layout_rows, dim3((tokens + 1023) / 1024), dim3(256), rows_per_request > 0 ? 0 : size_t(batch + 1) * sizeof(int), st, a);
    SERVE_LAUNCH_CHECK("layout_rows");
  }
  return 0;
}

extern "C" int bl_count_tokens(const int* ids, const int* cu, const int* prompt_lens, int* counts, void* seen, int rows, int n_ids,
                               int vocab, int reset, void* stream, char* err, size_t errlen) {
  if (rows < 1 || vocab < 1 || n_ids < 0 || !counts || !seen || (n_ids > 0 && !ids)) {
    set_err(err, errlen, "barlink: count_tokens needs ids, and tables of rows and a vocabulary");
    return -1;
  }
  if (!cu && n_ids != rows) {
    set_err(err, errlen, "barlink: count_tokens needs one id per row, or row offsets");
    return -1;
  }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int words = int((int64_t(vocab) + 31) / 32);
  if (rows > 65535) {
    set_err(err, errlen, "barlink: count_tokens takes at most 65535 rows");
    return -1;
  }
  if (reset) {
    // Four blocks for an SM, by slices of 1024 to kCountSlice tokens and up to 32 for a row: one row of 152064 in 8 and 32 slices 3.0 and 2.0 us,
    // 64 rows 9.4 and 12.5.  (64 rows: 9 slices of 16896, 576 blocks, of which shared memory lets three on an SM, 444 at once.)
    const int want = 4 * sm_count() / rows, most = want < 1 ? 1 : want > 32 ? 32 : want;
    const int64_t even = ((int64_t(vocab) + most - 1) / most + 127) / 128 * 128;
    const int slice = even < 1024 ? 1024 : even < kCountSlice ? int(even) : kCountSlice;
    const int smem = (slice + 4 + slice / 32) * 4;
    static bool attr[64] = {};
    const cudaError_t e = allow_smem(reinterpret_cast<const void*>(k_count_anew), (kCountSlice + 4 + kCountSlice / 32) * 4, attr);
    if (e != cudaSuccess) {
      set_err(err, errlen, "barlink: count_tokens shared memory opt-in failed: %s", cudaGetErrorString(e));
      return -1;
    }
    launch_k(k_count_anew, dim3(unsigned((int64_t(vocab) + slice - 1) / slice), rows), dim3(kCountThreads), smem, st, ids, cu, prompt_lens, counts,
             static_cast<uint32_t*>(seen), n_ids, vocab, words, slice);
  } else {
    const int x = cu ? int((int64_t(n_ids) / rows + kCountThreads - 1) / kCountThreads) : 1;
    launch_k(k_count_tokens, dim3(x < 1 ? 1 : x > 64 ? 64 : x, rows), dim3(kCountThreads), 0, st, ids, cu, prompt_lens, counts,
             static_cast<uint32_t*>(seen), n_ids, vocab, words);
  }
  SERVE_LAUNCH_CHECK("count_tokens");
  return 0;
}

extern "C" int bl_logit_rules(const blRulesArgs* r, void* stream, char* err, size_t errlen) {
  if (r->rows < 1 || r->n < 1 || !r->logits || r->n_bias < 0 || r->offset < 0 || !r->out == !r->idx || !r->idx != !r->val || (r->penalties && (!r->counts || !r->seen)) ||
      (r->n_bias > 0 && (!r->bias_ids || !r->bias)) || r->vocab < 0 ||
      (r->mask && int64_t(r->mask_words) * 32 < r->vocab)) {
    set_err(err, errlen, "barlink: logit rules need logits, an output, and the tables of the rules that are set");
    return -1;
  }
  Rules a;
  a.logits = r->logits; a.out = r->out; a.penalties = static_cast<const float*>(r->penalties);
  a.counts = static_cast<const int*>(r->counts); a.seen = static_cast<const uint32_t*>(r->seen);
  a.bias_ids = static_cast<const int*>(r->bias_ids); a.bias = static_cast<const float*>(r->bias);
  a.mask = static_cast<const uint32_t*>(r->mask);
  a.rows = r->rows; a.n = r->n; a.vocab = r->vocab; a.offset = r->offset; a.n_bias = r->n_bias;
  a.words = int((int64_t(r->vocab) + 31) / 32);
  a.ld = r->ld; a.ld_out = r->ld_out; a.ld_mask = r->ld_mask;
  a.idx = static_cast<int*>(r->idx); a.val = static_cast<float*>(r->val);
  // Blocks of a row: as many as leave all of them resident at once (two to an SM), none with less than 2048 logits.
  const int slots = 2 * sm_count();
  int share = 1;
  while (share < kRulesShare && r->rows * int64_t(2 * share) <= slots && r->n >= 2048 * 2 * share) share *= 2;
  const int64_t need = r->n_bias ? (int64_t(r->n) + 31) / 32 * 4 + int64_t(r->n_bias) * 8 : 0;
  if (need > 180 * 1024) {
    set_err(err, errlen, "barlink: logit rules: too many bias entries, or logits in a row with biases (n / 8 + 8 entries <= 184320)");
    return -1;
  }
  const int smem = int(need);
  const bool pick = !r->out;
  const auto kernel = r->fp32 ? pick ? k_logit_rules<float, true> : k_logit_rules<float, false>
                              : pick ? k_logit_rules<__nv_bfloat16, true> : k_logit_rules<__nv_bfloat16, false>;
  static bool attr[4][64] = {};
  cudaError_t e = smem > 4 * 1024 ? allow_smem(reinterpret_cast<const void*>(kernel), 180 * 1024, attr[2 * (r->fp32 ? 1 : 0) + pick]) : cudaSuccess;
  if (e == cudaSuccess)
    e = launch_cluster(kernel, dim3(unsigned(r->rows) * share), dim3(kRulesThreads), smem, share, static_cast<cudaStream_t>(stream), a);
  if (e != cudaSuccess) {
    set_err(err, errlen, "barlink: logit_rules launch failed: %s", cudaGetErrorString(e));
    return -1;
  }
  SERVE_LAUNCH_CHECK("logit_rules");
  return 0;
}
