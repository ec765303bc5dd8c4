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

// ---------------------------------------------------------------------------
// token histories to count tables
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(256) k_count_tokens(const int* __restrict__ ids, const int* __restrict__ cu,
                                                      const int* __restrict__ prompt, int* __restrict__ counts,
                                                      uint32_t* __restrict__ seen, int n_ids, int vocab, int words) {
  pdl_launch_dependents();
  pdl_wait();
  const int row = blockIdx.x;
  const int lo = cu ? max(cu[row], 0) : row, hi = cu ? min(cu[row + 1], n_ids) : row + 1;
  const int p = prompt ? prompt[row] : 0;
  for (int i = lo + blockIdx.y * blockDim.x + threadIdx.x; i < hi; i += gridDim.y * blockDim.x) {
    const int id = ids[i];
    if (id < 0 || id >= vocab) continue;
    atomicOr(seen + size_t(row) * words + (id >> 5), 1u << (id & 31));
    if (i - lo >= p) atomicAdd(counts + size_t(row) * vocab + id, 1);
  }
}

// ---------------------------------------------------------------------------
// rules on the logits
// ---------------------------------------------------------------------------
struct Rules {
  const void* logits;
  void* out;     // same type, or null
  float2* part;  // [chunks][rows] (value, token), or null
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

// grid (rows, chunks).  Each operation is rounded by itself (no fused multiply-add): the values are the formula's to the bit.
template <typename T>
__global__ void __launch_bounds__(256) k_logit_rules(const Rules a) {
  pdl_launch_dependents();
  pdl_wait();
  __shared__ float s_v[8];
  __shared__ int s_i[8];
  const int row = blockIdx.x, chunk = blockIdx.y, chunks = gridDim.y;
  const T* p = static_cast<const T*>(a.logits) + size_t(row) * a.ld;
  const int per = (a.n + chunks - 1) / chunks, lo = min(chunk * per, a.n), hi = min(lo + per, a.n);
  const bool pen = a.penalties != nullptr;
  const float again = pen ? a.penalties[row * 3] : 1.f, presence = pen ? a.penalties[row * 3 + 1] : 0.f,
              frequency = pen ? a.penalties[row * 3 + 2] : 0.f;
  float best = -INFINITY;
  int bi = 0x7fffffff;
  for (int i = lo + threadIdx.x; i < hi; i += blockDim.x) {
    const int id = i + a.offset;
    float x = to_float<T>(p[i]);
    const bool known = id >= 0 && id < a.vocab;
    if (pen && known && (a.seen[size_t(row) * a.words + (id >> 5)] >> (id & 31) & 1)) {
      x = x > 0.f ? __fdiv_rn(x, again) : __fmul_rn(x, again);
      const int c = a.counts[size_t(row) * a.vocab + id];
      if (c > 0) x = __fsub_rn(__fsub_rn(x, __fmul_rn(frequency, float(c))), presence);
    }
    for (int j = 0; j < a.n_bias; ++j)
      if (a.bias_ids[row * a.n_bias + j] == id) x = __fadd_rn(x, a.bias[row * a.n_bias + j]);
    if (a.mask && !(known && (a.mask[size_t(row) * a.ld_mask + (id >> 5)] >> (id & 31) & 1))) x = -INFINITY;
    if (a.out) static_cast<T*>(a.out)[size_t(row) * a.ld_out + i] = from_float<T>(x);
    if (x > best) {
      best = x;
      bi = id;
    }
  }
  if (!a.part) return;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float ov = __shfl_xor_sync(0xffffffffu, best, o);
    const int oi = __shfl_xor_sync(0xffffffffu, bi, o);
    if (ov > best || (ov == best && oi < bi)) {
      best = ov;
      bi = oi;
    }
  }
  if ((threadIdx.x & 31) == 0) {
    s_v[threadIdx.x >> 5] = best;
    s_i[threadIdx.x >> 5] = bi;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 8; ++w)
      if (s_v[w] > best || (s_v[w] == best && s_i[w] < bi)) {
        best = s_v[w];
        bi = s_i[w];
      }
    a.part[size_t(chunk) * a.rows + row] = make_float2(best, __int_as_float(bi));
  }
}

// (value, token) of a row's chunks -> the first of the greatest; -1 where nothing is left
__global__ void k_rules_pick(const float2* __restrict__ part, int chunks, int rows, int* __restrict__ idx, float* __restrict__ val) {
  pdl_launch_dependents();
  pdl_wait();
  const int r = blockIdx.x * blockDim.x + threadIdx.x;
  if (r >= rows) return;
  float best = -INFINITY;
  int bi = 0x7fffffff;
  for (int c = 0; c < chunks; ++c) {
    const float2 p = part[size_t(c) * rows + r];
    const int i = __float_as_int(p.y);
    if (p.x > best || (p.x == best && i < bi)) {
      best = p.x;
      bi = i;
    }
  }
  idx[r] = bi == 0x7fffffff ? -1 : bi;
  val[r] = best;
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
  launch_k(k_paged_layout, dim3(1), dim3(kLayoutThreads), smem, static_cast<cudaStream_t>(stream), a);
  SERVE_LAUNCH_CHECK("paged_layout");
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
  if (reset) {
    cudaMemsetAsync(counts, 0, size_t(rows) * vocab * 4, st);
    cudaMemsetAsync(seen, 0, size_t(rows) * words * 4, st);
  }
  const int y = cu ? (n_ids / rows + 1023) / 1024 : 1;
  launch_k(k_count_tokens, dim3(rows, y < 1 ? 1 : y > 64 ? 64 : y), dim3(256), 0, st, ids, cu, prompt_lens, counts,
           static_cast<uint32_t*>(seen), n_ids, vocab, words);
  SERVE_LAUNCH_CHECK("count_tokens");
  return 0;
}

extern "C" int bl_rules_chunks(int rows, int n) { (void)rows; (void)n; return 16; }

extern "C" int bl_logit_rules(const blRulesArgs* r, void* stream, char* err, size_t errlen) {
  if (r->rows < 1 || r->n < 1 || (!r->out && !r->part) || (r->penalties && (!r->counts || !r->seen)) ||
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
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const dim3 grid(r->rows, bl_rules_chunks(r->rows, r->n));
  launch_k(r->fp32 ? k_logit_rules<float> : k_logit_rules<__nv_bfloat16>, grid, dim3(256), 0, st, a);
  SERVE_LAUNCH_CHECK("logit_rules");
  if (r->part && r->idx) {
    launch_k(k_rules_pick, dim3((r->rows + 127) / 128), dim3(128), 0, st, static_cast<const float2*>(r->part), int(grid.y), r->rows,
             static_cast<int*>(r->idx), static_cast<float*>(r->val));
    SERVE_LAUNCH_CHECK("rules_pick");
  }
  return 0;
}
