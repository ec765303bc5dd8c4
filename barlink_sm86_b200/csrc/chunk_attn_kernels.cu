// SPDX-License-Identifier: MIT
//
// Attention of a chunk of new tokens of each request over its paged key/value cache (bf16, or in 4 bits: kv4.cuh), the chunk's own tokens
// included: token i of n new ones, of a request with c tokens in all, sees keys 0 .. c - n + i.
//
// The query heads that share a KV head, times T = 128 / (heads that share) tokens, are the 128 rows of a tile of tcgen05 products, so that a
// chunk of a few tokens reads its keys once for all of them.  Two tiles (a "pair") of 128 rows walk the keys together in steps of 64:
//
//   warp 0      asks for keys and values: boxes of up to 64 tokens of a block by TMA, or 16-token tiles of the 4-bit cache by bulk copies
//   warp 1      issues S = Q K^T (128 x 64 into TMEM, two buffers a tile) and O += P V (128 x hd in TMEM)
//   warp 2      asks for queries: one three-dimensional box is a tile (64 dims, the heads, T tokens)
//   warps 4-7   softmax of the first tile's rows, one row a thread: P (bf16) goes over S in TMEM, from where it is an operand
//   warps 8-11  the same for the second tile
//   warps 12-15 (4-bit cache) expand codes into bf16 tiles in the layout that TMA would leave
//
// Steps of all pairs of all requests and KV heads make one list, of which every block takes an equal run: lengths are known on the GPU only.  A pair
// that is cut leaves its pieces (sums, maxima) to a second kernel.  The chain of a run does not stop at a pair's end: scores are two steps
// ahead, also of the next pair; where a pair has one tile only (few new tokens: the case that is bound by memory) pairs take the two tiles'
// places in turn, and one's last products and output pass beside the next one's first scores.
//
// Tokens of table entries that name no block are left out (their boxes start behind the cache, so TMA fills in zeros).  What stands in the cache
// behind a request's last token may be anything: the values of the rest of its box are set to zero in shared memory.
//
// Every wait is bounded.  A run that gives up waits for its copies and products, leaves NaN for the rows of its run and sets the error word.
#include <cuda_bf16.h>
#include <stdint.h>

#include <atomic>

#include "attn_tc.cuh"
#include "bl_ops.h"
#include "heap.h"
#include "kv4.cuh"
#include "launch.h"
#include "ptx.cuh"

namespace bl {

constexpr int kChRows = 128;   // of a tile
constexpr int kChKeys = 64;    // of a step
constexpr int kChGran = 16;    // tokens that lie together in either cache
constexpr int kChStages = 4;   // K tiles and V tiles in flight, a ring each
constexpr int kChRaw = 3;      // steps of the 4-bit cache in flight
constexpr uint32_t kChTmemCols = 512;  // S of tile t, use parity p: 128 t + 64 p, P in its first half; O of tile t: 256 + 128 t
constexpr float kChRescale = 8.f;      // log2 units
constexpr uint32_t kChPolls = 1u << 24;

__device__ uint32_t g_chunk_err;  // set by a wait that ran out; one word per device

struct ChunkMeta {
  int count;                // pieces of the pair that begins in this run and ends in another; 0: none does
  int first;                // its first piece; piece k of the others is the first of run me + k
  int b, h, q0, tok0, ntok; // request, KV head, first row of the request, first token, tokens of the pair
};

struct Chunk {
  const int* cu;
  const int* ctx_lens;
  const int* tables;
  const uint8_t* cache4;
  __nv_bfloat16* out;
  float* part;   // [2 * runs][row_cap][hd], then [2 * runs][row_cap] (maximum, sum)
  ChunkMeta* meta;
  int tokens, batch, nq, nkv, G, T, block_size, n_blocks, max_blocks, row_cap, box;
  float scale_log2;
  uint32_t polls;
};

// A request's share of the list: tokens, positions, what its table can hold.
struct ChunkReq {
  int q0, n, past, cap;
};
__device__ __forceinline__ ChunkReq chunk_req(const Chunk& a, int b) {
  ChunkReq r;
  r.q0 = min(max(a.cu[b], 0), a.tokens);
  r.n = min(max(a.cu[b + 1], r.q0), a.tokens) - r.q0;
  const int ctx = min(max(a.ctx_lens[b], 0), 0x3fffffff);
  r.past = ctx - r.n;
  r.cap = min(ctx, a.max_blocks * a.block_size);
  return r;
}
// keys that the last of a pair's tokens sees
__device__ __forceinline__ int chunk_keys(const ChunkReq& r, int tok0, int ntok) { return min(max(r.past + tok0 + ntok, 0), r.cap); }
// (a pair that sees nothing has a step all the same: its rows are written)
__device__ __forceinline__ int chunk_steps(int keys) { return max(1, (keys + kChKeys - 1) / kChKeys); }

// Where a run stands: a pair and its steps.
struct ChunkAt {
  int b, h, tok0;
  int64_t start;   // of the pair in the list
  ChunkReq r;
  int ntok, keys, steps;
  __device__ __forceinline__ void fill(const Chunk& a) {
    ntok = min(2 * a.T, r.n - tok0);
    keys = chunk_keys(r, tok0, ntok);
    steps = chunk_steps(keys);
  }
  // the next pair (there is one)
  __device__ __forceinline__ void next(const Chunk& a) {
    start += steps;
    tok0 += 2 * a.T;
    if (tok0 >= r.n) {
      tok0 = 0;
      if (++h == a.nkv) {
        h = 0;
        do {
          ++b;
          if (b < a.batch) r = chunk_req(a, b);
        } while (b < a.batch && r.n == 0);
      }
    }
    fill(a);
  }
};

template <int HD, bool Q4>
struct ChunkShape {
  static constexpr int kThreads = Q4 ? 512 : 384;
  static constexpr uint32_t kQ = kChRows * HD * 2, kKV = kChKeys * HD * 2, kHalf = kChKeys * 128, kQHalf = kChRows * 128;
  static constexpr uint32_t kRawBytes = (kChKeys / kQ4Tokens) * q4_tile_bytes(HD);
  static constexpr uint32_t kOffK = 2 * kQ, kOffV = kOffK + kChStages * kKV, kOffRaw = kOffV + kChStages * kKV;
  static constexpr uint32_t kOffBar = kOffRaw + (Q4 ? kChRaw * kRawBytes : 0);
  static constexpr uint32_t kSmem = kOffBar + 512 + 1024;  // barriers and words; room to align
  static_assert(kSmem <= 232448, "attention tiles do not fit the shared memory of one block");
};

struct ChunkBars {
  uint64_t q_full[2], q_empty[2];
  uint64_t k_full[kChStages], k_empty[kChStages], v_full[kChStages], v_empty[kChStages];
  uint64_t raw_full[kChRaw], raw_empty[kChRaw];
  uint64_t s_ready[2][2], p_ready[2][2];  // [tile][use parity]
  uint64_t pv_done[2], o_final[2], o_free[2];
  uint64_t drained;
  uint32_t tmem, abort;
  uint32_t gone[8];  // granules of a step (by its number in the run, modulo 8) that have no block
};
static_assert(sizeof(ChunkBars) <= 512, "barriers");

template <int HD, bool Q4>
__global__ void __launch_bounds__(ChunkShape<HD, Q4>::kThreads, 1)
    k_chunk_attn(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k,
                 const __grid_constant__ CUtensorMap tmap_v, const Chunk a) {
  using S = ChunkShape<HD, Q4>;
  constexpr uint32_t kAll = 0xffffffffu;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* gen = smem_raw + (base - smem_u32(smem_raw));
  ChunkBars& bars = *reinterpret_cast<ChunkBars*>(gen + S::kOffBar);
  volatile uint32_t* s_abort = &bars.abort;
  __shared__ int64_t s_scan[S::kThreads / 32];
  __shared__ ChunkAt s_at;

  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int t = 0; t < 2; ++t) {
      mbar_init(&bars.q_full[t], 1);
      mbar_init(&bars.q_empty[t], 1);
      for (int p = 0; p < 2; ++p) {
        mbar_init(&bars.s_ready[t][p], 1);
        mbar_init(&bars.p_ready[t][p], kChRows);
      }
      mbar_init(&bars.pv_done[t], 1);
      mbar_init(&bars.o_final[t], 1);
      mbar_init(&bars.o_free[t], kChRows);
    }
    for (int s = 0; s < kChStages; ++s) {
      mbar_init(&bars.k_full[s], Q4 ? 4 : 1);
      mbar_init(&bars.k_empty[s], 1);
      mbar_init(&bars.v_full[s], Q4 ? 4 : 1);
      mbar_init(&bars.v_empty[s], 1);
    }
    for (int s = 0; s < kChRaw; ++s) {
      mbar_init(&bars.raw_full[s], 1);
      mbar_init(&bars.raw_empty[s], 4);
    }
    mbar_init(&bars.drained, 1);
    bars.abort = 0;
    for (int i = 0; i < 8; ++i) bars.gone[i] = 0;
    mbar_fence_init();
    tma_prefetch_desc(&tmap_q);
    if (!Q4) {
      tma_prefetch_desc(&tmap_k);
      tma_prefetch_desc(&tmap_v);
    }
  }
  if (warp == 1) {
    tmem_alloc(&bars.tmem, kChTmemCols);
    tmem_relinquish();
  }
  // lengths, tables, queries and the cache may come from the kernel just before this one
  pdl_wait();

  // ---- this block's run [lo, lo + count) of the list ----------------------------------------------------------------
  const int runs = gridDim.x, me = blockIdx.x;
  int64_t lo, run;
  int count;
  {
    const int per = (a.batch + S::kThreads - 1) / S::kThreads;
    const int b0 = min(int(threadIdx.x) * per, a.batch), b1 = min(b0 + per, a.batch);
    auto units_of = [&](const ChunkReq& r) {  // of one KV head
      int64_t u = 0;
      for (int t = 0; t < r.n; t += 2 * a.T) u += chunk_steps(chunk_keys(r, t, min(2 * a.T, r.n - t)));
      return u;
    };
    int64_t mine = 0;
    for (int b = b0; b < b1; ++b) mine += units_of(chunk_req(a, b)) * a.nkv;
    int64_t upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t u = __shfl_up_sync(kAll, upto, o);
      if (lane >= o) upto += u;
    }
    if (lane == 31) s_scan[warp] = upto;
    __syncthreads();
    int64_t total = 0;
#pragma unroll
    for (int w = 0; w < S::kThreads / 32; ++w) {
      if (w < warp) upto += s_scan[w];
      total += s_scan[w];
    }
    run = (total + runs - 1) / runs;
    lo = min(int64_t(me) * run, total);
    count = int(min(run, total - lo));
    int64_t at = upto - mine;
    if (count > 0 && at <= lo && lo < upto) {  // one thread's requests hold the first step
      ChunkAt s;
      s.b = b0;
      int64_t units;
      for (;; ++s.b) {
        s.r = chunk_req(a, s.b);
        units = units_of(s.r);
        if (lo < at + units * a.nkv) break;
        at += units * a.nkv;
      }
      s.h = int((lo - at) / units);
      s.start = at + s.h * units;
      s.tok0 = 0;
      s.fill(a);
      while (lo >= s.start + s.steps) {
        s.start += s.steps;
        s.tok0 += 2 * a.T;
        s.fill(a);
      }
      s_at = s;
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = bars.tmem;
  if (count == 0) {
    if (threadIdx.x == 0) a.meta[me].count = 0;
    __syncthreads();
    if (warp == 1) tmem_dealloc(tmem_base, kChTmemCols);
    return;
  }
  const ChunkAt first = s_at;
  // Every role walks the pairs of the run by itself: (pair, its first and last step + 1 in this run, its step 0 in the run's numbers, place).
  // place: the tile whose rows are a pair's only ones; 2: both tiles.  Pairs of one tile take the two places in turn.
  auto walk = [&](auto&& f) {
    ChunkAt s = first;
    int turn = 0;
    for (int i = 0;;) {
      const int j0 = int(lo + i - s.start), j1 = min(s.steps, j0 + count - i);
      int place = 2;
      if (s.ntok <= a.T) {
        place = turn;
        turn ^= 1;
      }
      if (!f(s, j0, j1, i, place)) return;
      i += j1 - j0;
      if (i >= count) return;
      s.next(a);
    }
  };

  if (warp == 0) {
    // ------------------------------ keys and values ------------------------------
    int kst = 0, issued_k = 0, issued_v = 0;  // (stages follow from the step's number)
    bool ok = true;
    uint32_t gone_before = 0;  // bit s: bars.gone[s] is set
    walk([&](const ChunkAt& s, int j0, int j1, int i0, int) {
      const int* table = a.tables + size_t(s.b) * a.max_blocks;
      // lane l: granule l of eight steps -- the row of the cache where it begins (tile of the 4-bit cache), -1: nothing visible, -2: no block
      auto look = [&](int j) {
        const int tok = j * kChKeys + lane * kChGran;
        int at = -1;
        if (tok < s.keys) {
          const int page = tok / a.block_size, blk = table[page], in = tok - page * a.block_size;
          at = blk < 0 || blk >= a.n_blocks ? -2 : Q4 ? (blk * a.nkv + s.h) * (a.block_size / kQ4Tokens) + in / kQ4Tokens : (blk * a.nkv + s.h) * a.block_size + in;
        }
        return at;
      };
      int ahead = look(j0), where = 0;
      const int none = a.n_blocks * a.nkv * a.block_size;  // behind the cache
      for (int j = j0; j < j1; ++j) {
        const int part = (j - j0) & 7, i = i0 + j - j0;
        if (part == 0) {
          where = ahead;
          ahead = look(j + 8);
        }
        const uint32_t lost = __ballot_sync(kAll, where == -2) >> (4 * part) & 15u;
        if constexpr (!Q4) {
          const int gr = lane & 3, half = lane >> 2 & 1;
          const int at = __shfl_sync(kAll, where, 4 * part + gr);
          const int y = at >= 0 ? at : none;
          const bool mine = lane < 4 * (HD / 64) && gr % (a.box / kChGran) == 0;
          const uint32_t off = uint32_t(half) * S::kHalf + uint32_t(gr) * (kChGran * 128);
          kst = i % kChStages;
          const uint32_t phase = uint32_t(i / kChStages) & 1u;
          ok = mbar_wait_bounded_warp(&bars.k_empty[kst], phase ^ 1u, s_abort, a.polls);
          if (!ok) break;
          if (lane == 0) {
            if (lost || (gone_before >> (i & 7) & 1u)) bars.gone[i & 7] = lost;
            mbar_expect_tx(&bars.k_full[kst], S::kKV);
          }
          gone_before = (gone_before & ~(1u << (i & 7))) | uint32_t(lost != 0) << (i & 7);
          __syncwarp();
          if (mine) tma_load_2d_hint_s(base + S::kOffK + kst * S::kKV + off, &tmap_k, smem_u32(&bars.k_full[kst]), half * 64, y, kHintEvictLast);
          issued_k = i + 1;
          ok = mbar_wait_bounded_warp(&bars.v_empty[kst], phase ^ 1u, s_abort, a.polls);
          if (!ok) break;
          if (lane == 0) mbar_expect_tx(&bars.v_full[kst], S::kKV);
          __syncwarp();
          if (mine) tma_load_2d_hint_s(base + S::kOffV + kst * S::kKV + off, &tmap_v, smem_u32(&bars.v_full[kst]), half * 64, y, kHintEvictLast);
          issued_v = i + 1;
        } else {
          const int at = __shfl_sync(kAll, where, 4 * part + (lane & 3));
          const uint32_t has = __ballot_sync(kAll, at >= 0) & 15u;
          const int rs = i % kChRaw;
          ok = mbar_wait_bounded_warp(&bars.raw_empty[rs], (uint32_t(i / kChRaw) & 1u) ^ 1u, s_abort, a.polls);
          if (!ok) break;
          if (lane == 0) {
            bars.gone[i & 7] = lost | (has ^ 15u) << 8;
            mbar_expect_tx(&bars.raw_full[rs], uint32_t(__popc(has)) * q4_tile_bytes(HD));
          }
          __syncwarp();
          bulk_load_warp(lane < 4 && at >= 0, base + S::kOffRaw + rs * S::kRawBytes + lane * q4_tile_bytes(HD),
                         a.cache4 + size_t(max(at, 0)) * q4_tile_bytes(HD), q4_tile_bytes(HD), smem_u32(&bars.raw_full[rs]), kHintEvictFirst);
          issued_k = i + 1;
        }
      }
      return ok;
    });
    // The block's shared memory is another's behind it: whatever is still on its way lands first, also after a wait that ran out.
    auto drain = [&](uint64_t* full, int issued, int stages) {
      for (int i = max(0, issued - stages); i < issued; ++i)
        for (uint32_t p = 0; p < (1u << 20); ++p)
          if (mbar_try_wait(&full[i % stages], uint32_t(i / stages) & 1u)) break;
    };
    if (*s_abort) {
      if constexpr (Q4) {
        drain(bars.raw_full, issued_k, kChRaw);
      } else {
        drain(bars.k_full, issued_k, kChStages);
        drain(bars.v_full, issued_v, kChStages);
      }
    }
  } else if (warp == 2) {
    // ------------------------------ queries ------------------------------
    const uint32_t bytes = uint32_t(a.G) * a.T * HD * 2;
    int n[2] = {0, 0};  // tiles asked for, by place
    walk([&](const ChunkAt& s, int, int, int, int place) {
      for (int t = 0; t < 2; ++t) {
        if (place != 2 && place != t) continue;
        if (!mbar_wait_bounded_warp(&bars.q_empty[t], (uint32_t(n[t]) & 1u) ^ 1u, s_abort, a.polls)) return false;
        if (lane == 0) {
          mbar_expect_tx(&bars.q_full[t], bytes);
#pragma unroll
          for (int h = 0; h < HD / 64; ++h)
            tma_load_3d_hint_s(base + t * S::kQ + h * S::kQHalf, &tmap_q, smem_u32(&bars.q_full[t]), h * 64, s.h * a.G,
                               s.r.q0 + s.tok0 + (place == 2 ? t * a.T : 0), kHintEvictFirst);
        }
        ++n[t];
      }
      return true;
    });
    if (*s_abort)
      for (int t = 0; t < 2; ++t)
        if (n[t] > 0)
          for (uint32_t p = 0; p < (1u << 20); ++p)
            if (mbar_try_wait(&bars.q_full[t], uint32_t(n[t] - 1) & 1u)) break;
  } else if (warp == 1) {
    // ------------------------------ products ------------------------------
    const uint32_t leader = elect_leader();
    const uint32_t idesc_s = umma_idesc_f16(kChRows, kChKeys, 1);
    const uint32_t idesc_o = umma_idesc_f16(kChRows, HD, 1) | kUmmaBMajorN;
    auto issue_s = [&](int t, int p, int st) {
      const uint64_t dq = umma_desc_k_sw128(base + t * S::kQ), dk = umma_desc_k_sw128(base + S::kOffK + st * S::kKV);
#pragma unroll
      for (int ks = 0; ks < HD / 16; ++ks)
        umma_f16_ss_warp(leader, tmem_base + uint32_t(t * 128 + p * kChKeys), dq + uint64_t((ks >> 2) * (S::kQHalf / 16) + 2 * (ks & 3)),
                         dk + uint64_t((ks >> 2) * (S::kHalf / 16) + 2 * (ks & 3)), idesc_s, ks > 0 ? 1u : 0u);
      umma_commit_warp(leader, &bars.s_ready[t][p]);
    };
    auto issue_pv = [&](int t, int p, int st, bool acc) {
      const uint64_t dv = umma_desc_mn_sw128(base + S::kOffV + st * S::kKV, S::kHalf);
#pragma unroll
      for (int ks = 0; ks < kChKeys / 16; ++ks)
        umma_f16_ts_warp(leader, tmem_base + 256u + uint32_t(t * 128), tmem_base + uint32_t(t * 128 + p * kChKeys + 8 * ks), dv + uint64_t(128 * ks), idesc_o,
                         (acc || ks > 0) ? 1u : 0u);
      umma_commit_warp(leader, &bars.pv_done[t]);
    };
    bool ok = true;
    // scores, two steps ahead of the products with values
    ChunkAt sa = first;
    int s_i = 0, s_pair = 0, s_turn = 0;           // step of the run, where its pair begins there, whose turn it is
    int s_uses[2] = {0, 0}, s_tiles[2] = {0, 0};   // uses and query tiles of either place so far
    int s_j0 = int(lo - sa.start), s_j1 = min(sa.steps, s_j0 + count), s_place = sa.ntok <= a.T ? s_turn : 2;
    if (s_place != 2) s_turn ^= 1;
    auto scores = [&] {
      if (s_i >= count) return true;
      if (s_i - s_pair >= s_j1 - s_j0) {
        s_pair = s_i;
        sa.next(a);
        s_j0 = 0;
        s_j1 = min(sa.steps, count - s_i);
        s_place = 2;
        if (sa.ntok <= a.T) {
          s_place = s_turn;
          s_turn ^= 1;
        }
      }
      const int st = s_i % kChStages;
      if (!mbar_wait_bounded_warp(&bars.k_full[st], uint32_t(s_i / kChStages) & 1u, s_abort, a.polls)) return false;
      const bool begins = s_i == s_pair, ends = s_i - s_pair + 1 == s_j1 - s_j0;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        if (s_place != 2 && s_place != t) continue;
        if (begins && !mbar_wait_bounded_warp(&bars.q_full[t], uint32_t(s_tiles[t]++) & 1u, s_abort, a.polls)) return false;
        tc_fence_after_sync();
        issue_s(t, s_uses[t]++ & 1, st);
        if (ends) umma_commit_warp(leader, &bars.q_empty[t]);
      }
      umma_commit_warp(leader, &bars.k_empty[st]);
      ++s_i;
      return true;
    };
    ok = scores() && scores();
    int uses[2] = {0, 0}, pairs[2] = {0, 0};
    if (ok)
      walk([&](const ChunkAt& s, int j0, int j1, int i0, int place) {
        for (int j = j0; j < j1; ++j) {
          const int i = i0 + j - j0, st = i % kChStages;
          bool waited = false;
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (place != 2 && place != t) continue;
            const int p = uses[t] & 1;
            bool here = mbar_wait_bounded(&bars.p_ready[t][p], uint32_t(uses[t] >> 1) & 1u, s_abort, a.polls);
            if (!waited) here = here && mbar_wait_bounded(&bars.v_full[st], uint32_t(i / kChStages) & 1u, s_abort, a.polls);
            // the sums of the place's pair before have been read
            if (j == j0) here = here && mbar_wait_bounded(&bars.o_free[t], (uint32_t(pairs[t]) & 1u) ^ 1u, s_abort, a.polls);
            if (!__all_sync(kAll, here)) return ok = false;
            if (!Q4 && !waited && (j + 1) * kChKeys > s.keys && s.keys % a.box) {
              // the rest of the last box: probabilities are zero there, values may be anything
              const int r0 = s.keys - j * kChKeys, r1 = (r0 + a.box - 1) / a.box * a.box;
              for (int k = lane + r0 * (HD / 8); k < r1 * (HD / 8); k += 32) {
                const int r = k / (HD / 8), c = k % (HD / 8);
                asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(base + S::kOffV + st * S::kKV + (c >> 3) * S::kHalf + r * 128 + (c & 7) * 16), "r"(0)
                             : "memory");
              }
              fence_proxy_async_smem();
              __syncwarp();
            }
            waited = true;
            tc_fence_after_sync();
            issue_pv(t, p, st, j > j0);
            if (j + 1 == j1) {
              umma_commit_warp(leader, &bars.o_final[t]);
              ++pairs[t];
            }
            ++uses[t];
          }
          umma_commit_warp(leader, &bars.v_empty[st]);
          if (!scores()) return ok = false;
        }
        return true;
      });
    if (!ok) {
      // products on their way read shared memory and write TMEM, which are given back below
      umma_commit_warp(leader, &bars.drained);
      mbar_wait_bounded_warp(&bars.drained, 0, s_abort, 1u << 20);
    }
  } else if (warp >= 12) {
    // ------------------------------ codes of the 4-bit cache to bf16 tiles ------------------------------
    if constexpr (Q4) {
      constexpr int NA = HD / kQ4Group;
      const int tid = threadIdx.x - 384;
      walk([&](const ChunkAt& s, int j0, int j1, int i0, int) {
        for (int j = j0; j < j1; ++j) {
          const int i = i0 + j - j0, rs = i % kChRaw, st = i % kChStages;
          if (!mbar_wait_bounded_warp(&bars.raw_full[rs], uint32_t(i / kChRaw) & 1u, s_abort, a.polls)) return false;
          const uint32_t none = bars.gone[i & 7] >> 8;  // granules without copies
          const int left = s.keys - j * kChKeys;        // tokens of this step
          const uint32_t raw = base + S::kOffRaw + rs * S::kRawBytes;
          auto words = [&](uint32_t addr, uint32_t (&w)[NA]) {
            if constexpr (NA == 4)
              asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(addr));
            else
              asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(addr));
          };
          // (16 bits 0x430c are the bf16 number 128 + c)
          auto value = [&](uint32_t two, __nv_bfloat162 step, __nv_bfloat162 low) {
            const uint32_t c = (two & 0x000f000fu) | 0x43004300u, k = 0xc300c300u;  // - 128
            const __nv_bfloat162 v = __hfma2(__hadd2(*reinterpret_cast<const __nv_bfloat162*>(&c), *reinterpret_cast<const __nv_bfloat162*>(&k)), step, low);
            return *reinterpret_cast<const uint32_t*>(&v);
          };
          auto twice = [](uint32_t w, int hi) {
            const uint32_t v = __byte_perm(w, 0, hi ? 0x3232 : 0x1010);
            return *reinterpret_cast<const __nv_bfloat162*>(&v);
          };
          auto store = [&](uint32_t tile, int key, int chunk, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
            asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(tile + (chunk >> 3) * S::kHalf + key * 128 + (((chunk & 7) ^ (key & 7)) << 4)), "r"(x), "r"(y), "r"(z), "r"(w)
                         : "memory");
          };
          if (!mbar_wait_bounded_warp(&bars.k_empty[st], (uint32_t(i / kChStages) & 1u) ^ 1u, s_abort, a.polls)) return false;
          const uint32_t kt = base + S::kOffK + st * S::kKV, vt = base + S::kOffV + st * S::kKV;
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int key = u * 32 + (tid >> 2), t = tid & 3, g = key >> 4;
            uint32_t w[NA] = {}, par[NA] = {};
            if (key < left && !(none >> g & 1u)) {
              words(raw + g * q4_tile_bytes(HD) + (key & 15) * (HD / 2) + t * NA * 4, w);
              words(raw + g * q4_tile_bytes(HD) + q4_k_params(HD) + (key & 15) * NA * 4, par);
            }
#pragma unroll
            for (int n = 0; n < NA; ++n) {
              const __nv_bfloat162 step = twice(par[n >> 1], n & 1), low = twice(par[NA / 2 + (n >> 1)], n & 1);
              // nibbles (0, 4), (1, 5), (2, 6), (3, 7)
              const uint32_t p0 = value(w[n], step, low), p1 = value(w[n] >> 4, step, low), p2 = value(w[n] >> 8, step, low), p3 = value(w[n] >> 12, step, low);
              store(kt, key, 4 * n + t, __byte_perm(p0, p1, 0x5410), __byte_perm(p2, p3, 0x5410), __byte_perm(p0, p1, 0x7632), __byte_perm(p2, p3, 0x7632));
            }
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&bars.k_full[st]);
          if (!mbar_wait_bounded_warp(&bars.v_empty[st], (uint32_t(i / kChStages) & 1u) ^ 1u, s_abort, a.polls)) return false;
          {
            // two tokens, eight dims of every group
            const int pair = tid >> 2, q = tid & 3, g = pair >> 3, key = 2 * pair;
            uint32_t w0[NA] = {}, w1[NA] = {}, pa[NA] = {}, pb[NA] = {};
            const bool one = key < left && !(none >> g & 1u), two = key + 1 < left && !(none >> g & 1u);
            const uint32_t tile = raw + g * q4_tile_bytes(HD);
            if (one) {
              words(tile + q4_v_codes(HD) + (pair & 7) * HD + 2 * q * NA * 4, w0);
              words(tile + q4_v_codes(HD) + (pair & 7) * HD + (2 * q + 1) * NA * 4, w1);
              words(tile + q4_v_params(HD) + (key & 15) * NA * 4, pa);
            }
            if (two) words(tile + q4_v_params(HD) + (key & 15) * NA * 4 + NA * 4, pb);
#pragma unroll
            for (int n = 0; n < NA; ++n) {
              // (the first token's nibble beside the second's)
              const uint32_t s2 = __byte_perm(pa[n >> 1], pb[n >> 1], n & 1 ? 0x7632 : 0x5410), l2 = __byte_perm(pa[NA / 2 + (n >> 1)], pb[NA / 2 + (n >> 1)], n & 1 ? 0x7632 : 0x5410);
              const __nv_bfloat162 step = *reinterpret_cast<const __nv_bfloat162*>(&s2), low = *reinterpret_cast<const __nv_bfloat162*>(&l2);
              uint32_t v[8];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                v[e] = value(w0[n] >> (4 * e), step, low);
                v[4 + e] = value(w1[n] >> (4 * e), step, low);
              }
              const int chunk = 4 * n + q;
              store(vt, key, chunk, __byte_perm(v[0], v[1], 0x5410), __byte_perm(v[2], v[3], 0x5410), __byte_perm(v[4], v[5], 0x5410), __byte_perm(v[6], v[7], 0x5410));
              store(vt, key + 1, chunk, __byte_perm(v[0], v[1], 0x7632), __byte_perm(v[2], v[3], 0x7632), __byte_perm(v[4], v[5], 0x7632), __byte_perm(v[6], v[7], 0x7632));
            }
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(&bars.v_full[st]);
            mbar_arrive(&bars.raw_empty[rs]);
          }
        }
        return true;
      });
    }
  } else if (warp >= 4) {
    // ------------------------------ softmax ------------------------------
    const int t = (warp - 4) >> 2, quarter = warp & 3, row = quarter * 32 + lane;  // TMEM lanes that this warp may touch
    const int tok = row / a.G, g = row - tok * a.G;
    const uint32_t lane_addr = tmem_base + (uint32_t(quarter * 32) << 16);
    const uint32_t o_addr = lane_addr + 256u + uint32_t(t * 128);
    int uses = 0, pairs = 0;
    bool ok = true;
    walk([&](const ChunkAt& s, int j0, int j1, int i0, int place) {
      if (place != 2 && place != t) return true;
      const int tk = s.tok0 + (place == 2 ? t * a.T : 0) + tok;  // token of the request
      const bool valid = tok < a.T && tk < s.r.n;
      const int lim = min(s.r.past + tk + 1, s.r.cap);           // keys [0, lim) are visible
      const bool busy = __any_sync(kAll, valid);
      float m_used = -INFINITY, l = 0.f;
      for (int j = j0; j < j1 && ok; ++j, ++uses) {
        const int p = uses & 1;
        if (!mbar_wait_bounded_warp(&bars.s_ready[t][p], uint32_t(uses >> 1) & 1u, s_abort, a.polls)) {
          ok = false;
          break;
        }
        if (!busy) {  // rows of no token: whatever their probabilities are
          mbar_arrive(&bars.p_ready[t][p]);
          continue;
        }
        tc_fence_after_sync();
        const uint32_t s_addr = lane_addr + uint32_t(t * 128 + p * kChKeys);
        float x[kChKeys];
        {
          uint32_t r0[32], r1[32];
          tmem_ld_32x32(s_addr, r0);
          tmem_ld_32x32(s_addr + 32, r1);
          tmem_ld_wait();
          const float2 sl = make_float2(a.scale_log2, a.scale_log2);
#pragma unroll
          for (int c = 0; c < 32; c += 2) {
            const float2 u = mul2(make_float2(__uint_as_float(r0[c]), __uint_as_float(r0[c + 1])), sl);
            const float2 v = mul2(make_float2(__uint_as_float(r1[c]), __uint_as_float(r1[c + 1])), sl);
            x[c] = u.x;
            x[c + 1] = u.y;
            x[c + 32] = v.x;
            x[c + 33] = v.y;
          }
        }
        const int kbase = j * kChKeys;
        if (kbase + kChKeys > lim) {
#pragma unroll
          for (int c = 0; c < kChKeys; ++c)
            if (kbase + c >= lim) x[c] = -INFINITY;
        }
        const uint32_t lost = *const_cast<volatile uint32_t*>(&bars.gone[(i0 + j - j0) & 7]) & 15u;
        if (lost) {
#pragma unroll
          for (int c = 0; c < kChKeys; ++c)
            if (lost >> (c / kChGran) & 1u) x[c] = -INFINITY;
        }
        // four chains: the maximum is on the way from the scores to everything else
        float mx4[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
        for (int c = 4; c < kChKeys; ++c) mx4[c & 3] = fmaxf(mx4[c & 3], x[c]);
        const float m_new = fmaxf(m_used, fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])));
        const bool grow = m_new > m_used + kChRescale;  // also true on the first finite maximum
        if (__any_sync(kAll, grow)) {
          const float alpha = (m_new == -INFINITY) ? 1.f : ex2_approx(m_used - m_new);
          if (j > j0) {
            // P V of the use before may still be running.  Parity tells its phase apart from its neighbours: the one behind needs this warp's own
            // P, and the one before is over, since it was issued ahead of the scores of this use by the same thread.
            if (!mbar_wait_bounded_warp(&bars.pv_done[t], uint32_t(uses - 1) & 1u, s_abort, a.polls)) {
              ok = false;
              break;
            }
            tc_fence_after_sync();
#pragma unroll 1
            for (int c0 = 0; c0 < HD; c0 += 32) {
              uint32_t r[32];
              tmem_ld_32x32(o_addr + c0, r);
              tmem_ld_wait();
#pragma unroll
              for (int c = 0; c < 32; ++c) r[c] = __float_as_uint(__uint_as_float(r[c]) * alpha);
              tmem_st_32x32(o_addr + c0, r);
            }
            tmem_st_wait();
          }
          l *= alpha;
          m_used = m_new;
        }
        const float mref = (m_used == -INFINITY) ? 0.f : m_used;
        const float2 neg = make_float2(-mref, -mref);
        float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        uint32_t pk[kChKeys / 2];
#pragma unroll
        for (int c = 0; c < kChKeys; c += 2) {
          const float2 u = add2(make_float2(x[c], x[c + 1]), neg);
          const float2 e = make_float2(ex2_approx(u.x), ex2_approx(u.y));
          sum[(c >> 1) & 1] = add2(sum[(c >> 1) & 1], e);
          // (P in bf16: the products want it; off by half a step, 2^-9, of every term)
          pk[c >> 1] = pack_bf16x2(e.x, e.y);
        }
        sum[0] = add2(sum[0], sum[1]);
        l += sum[0].x + sum[0].y;
        tmem_st_32x32(s_addr, pk);  // over the scores that it was made of
        tmem_st_wait();
        tc_fence_before_sync();
        mbar_arrive(&bars.p_ready[t][p]);
      }
      // ---- the pair's rows, or a piece of them ----
      if (ok && !mbar_wait_bounded_warp(&bars.o_final[t], uint32_t(pairs) & 1u, s_abort, a.polls)) ok = false;
      ++pairs;
      const bool whole = j0 == 0 && j1 == s.steps;
      const int piece = 2 * me + (i0 == 0 ? 0 : 1), at = (place == 2 ? t * kChRows : 0) + row;
      const float inv = !whole ? 1.f : l > 0.f ? 1.f / l : 0.f;
      __nv_bfloat16* orow = a.out + (size_t(s.r.q0 + tk) * a.nq + size_t(s.h) * a.G + g) * HD;
      float* prow = a.part + (size_t(piece) * a.row_cap + at) * HD;
      tc_fence_after_sync();
#pragma unroll 1
      for (int c0 = 0; c0 < HD; c0 += 32) {
        uint32_t r[32];
        if (ok) {
          tmem_ld_32x32(o_addr + c0, r);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int c = 0; c < 32; ++c) r[c] = 0x7fffffffu;
        }
        if (valid && whole) {
#pragma unroll
          for (int c = 0; c < 32; c += 8)
            *reinterpret_cast<uint4*>(orow + c0 + c) = make_uint4(
                pack_bf16x2(__uint_as_float(r[c]) * inv, __uint_as_float(r[c + 1]) * inv), pack_bf16x2(__uint_as_float(r[c + 2]) * inv, __uint_as_float(r[c + 3]) * inv),
                pack_bf16x2(__uint_as_float(r[c + 4]) * inv, __uint_as_float(r[c + 5]) * inv), pack_bf16x2(__uint_as_float(r[c + 6]) * inv, __uint_as_float(r[c + 7]) * inv));
        } else if (valid) {
#pragma unroll
          for (int c = 0; c < 32; c += 4) *reinterpret_cast<uint4*>(prow + c0 + c) = make_uint4(r[c], r[c + 1], r[c + 2], r[c + 3]);
        }
        __syncwarp();
      }
      if (!whole && valid)
        reinterpret_cast<float2*>(a.part + size_t(2 * runs) * a.row_cap * HD)[size_t(piece) * a.row_cap + at] = make_float2(m_used, ok ? l : NAN);
      tc_fence_before_sync();
      mbar_arrive(&bars.o_free[t]);
      return true;  // (a run that gave up goes on to leave NaN everywhere)
    });
  } else if (lane == 0) {
    // ------------------------------ what the second kernel needs to know ------------------------------
    ChunkMeta m = {};
    walk([&](const ChunkAt& s, int j0, int j1, int i0, int) {
      if (j0 == 0 && j1 < s.steps) m = {int((s.start + s.steps - 1) / run) - me + 1, 2 * me + (i0 == 0 ? 0 : 1), s.b, s.h, s.r.q0, s.tok0, s.ntok};
      return true;
    });
    a.meta[me] = m;
  }

  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, kChTmemCols);
  }
  if (threadIdx.x == 0 && *s_abort) g_chunk_err = 1;
}

// Pieces of a pair that was cut: block (run where it begins, rows).  Eight warps take a row each, or, with more pieces, share a row.
constexpr int kChMergeWarps = 8;
template <int HD>
__global__ void __launch_bounds__(kChMergeWarps * 32) k_chunk_merge(const Chunk a) {
  constexpr int D = HD / 32;
  __shared__ float s_o[kChMergeWarps][HD], s_m[kChMergeWarps], s_l[kChMergeWarps];
  pdl_launch_dependents();
  pdl_wait();
  const int me = blockIdx.x, runs = gridDim.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const ChunkMeta m = a.meta[me];
  // (every run leaves its words; lengths that another stream changes meanwhile, which nobody may, could leave some that fit nothing)
  if (m.count <= 0 || m.count > runs - me || m.ntok > 2 * a.T) return;
  const int ways = m.count <= 2 ? 1 : m.count <= 5 ? 2 : m.count <= 12 ? 4 : 8, per = kChMergeWarps / ways, w = warp % ways;
  const int rows = m.ntok * a.G;
  const float2* sums = reinterpret_cast<const float2*>(a.part + size_t(2 * runs) * a.row_cap * HD);
  for (int r0 = blockIdx.y * per; r0 < rows; r0 += gridDim.y * per) {
    const int r = r0 + warp / ways;
    const bool there = r < rows;
    const int tok = r / a.G, g = r - tok * a.G, at = (tok >= a.T ? kChRows + (tok - a.T) * a.G : tok * a.G) + g;
    float M = -INFINITY, L = 0.f, acc[D];
#pragma unroll
    for (int d = 0; d < D; ++d) acc[d] = 0.f;
    if (there) {
#pragma unroll 4
      for (int k = w; k < m.count; k += ways) {
        const size_t p = size_t(k == 0 ? m.first : 2 * (me + k)) * a.row_cap + at;
        const float2 ml = sums[p];
        float v[D];
        if constexpr (D == 4) {
          const float4 u = *reinterpret_cast<const float4*>(a.part + p * HD + 4 * lane);
          v[0] = u.x; v[1] = u.y; v[2] = u.z; v[3] = u.w;
        } else {
          const float2 u = *reinterpret_cast<const float2*>(a.part + p * HD + 2 * lane);
          v[0] = u.x; v[1] = u.y;
        }
        const float n = fmaxf(M, ml.x), ref = n == -INFINITY ? 0.f : n, s0 = ex2_approx(M - ref), s1 = ex2_approx(ml.x - ref);
        M = n;
        L = L * s0 + ml.y * s1;
#pragma unroll
        for (int d = 0; d < D; ++d) acc[d] = acc[d] * s0 + v[d] * s1;
      }
    }
    if (ways > 1) {
#pragma unroll
      for (int d = 0; d < D; ++d) s_o[warp][D * lane + d] = acc[d];
      if (lane == 0) {
        s_m[warp] = M;
        s_l[warp] = L;
      }
      __syncthreads();
      if (w == 0) {
        for (int i = 1; i < ways; ++i) {
          const float n = fmaxf(M, s_m[warp + i]), ref = n == -INFINITY ? 0.f : n, s0 = ex2_approx(M - ref), s1 = ex2_approx(s_m[warp + i] - ref);
          M = n;
          L = L * s0 + s_l[warp + i] * s1;
#pragma unroll
          for (int d = 0; d < D; ++d) acc[d] = acc[d] * s0 + s_o[warp + i][D * lane + d] * s1;
        }
      }
      __syncthreads();
    }
    if (there && w == 0) {
      const float inv = L == 0.f ? 0.f : 1.f / L;
      __nv_bfloat16* to = a.out + (size_t(m.q0 + m.tok0 + tok) * a.nq + size_t(m.h) * a.G + g) * HD + D * lane;
      if constexpr (D == 4)
        *reinterpret_cast<uint2*>(to) = make_uint2(pack_bf16x2(acc[0] * inv, acc[1] * inv), pack_bf16x2(acc[2] * inv, acc[3] * inv));
      else
        *reinterpret_cast<uint32_t*>(to) = pack_bf16x2(acc[0] * inv, acc[1] * inv);
    }
  }
}

}  // namespace bl

using namespace bl;

static std::atomic<uint32_t> g_chunk_polls{kChPolls};

static int chunk_error_rc(cudaError_t e, char* err, size_t errlen) {
  if (e != cudaSuccess) set_err(err, errlen, "barlink: chunk_attn_error: %s", cudaGetErrorString(e));
  return e == cudaSuccess ? 0 : -1;
}
extern "C" int bl_chunk_attn_error_async(unsigned* out, void* stream, char* err, size_t errlen) {
  return chunk_error_rc(cudaMemcpyFromSymbolAsync(out, g_chunk_err, sizeof(*out), 0, cudaMemcpyDeviceToHost, static_cast<cudaStream_t>(stream)), err, errlen);
}
extern "C" int bl_chunk_attn_error_clear(char* err, size_t errlen) {
  const unsigned none = 0;
  return chunk_error_rc(cudaMemcpyToSymbol(g_chunk_err, &none, sizeof(none)), err, errlen);
}
extern "C" unsigned bl_chunk_attn_wait_polls(unsigned polls) { return g_chunk_polls.exchange(polls); }

// tokens of a tile, and rows of a pair that a piece has room for
static int chunk_tile_tokens(int G) { return kChRows / G; }
static int chunk_row_cap(int tokens, int G) {
  const int T = chunk_tile_tokens(G);
  return tokens <= T ? tokens * G : 2 * kChRows;
}

extern "C" size_t bl_paged_attn_chunk_ws(int tokens, int nq, int nkv, int hd) {
  if (tokens < 1 || nkv < 1 || nq < nkv || nq / nkv > kChRows || (hd != 64 && hd != 128)) return 0;
  return size_t(sm_count()) * (2 * size_t(chunk_row_cap(tokens, nq / nkv)) * (hd + 2) * sizeof(float) + sizeof(ChunkMeta));
}

extern "C" int bl_paged_attn_chunk(const void* q, int q_stride, const void* k_cache, const void* v_cache, const void* cache4,
                                   const int* block_tables, const int* cu_q, const int* ctx_lens, void* out, int tokens, int batch, int nq,
                                   int nkv, int hd, int block_size, int n_blocks, int max_blocks, float scale, void* ws, size_t ws_bytes,
                                   void* stream, char* err, size_t errlen) {
  auto refuse = [&](const char* why) {
    set_err(err, errlen, "barlink: attention of a chunk over the paged cache %s", why);
    return -1;
  };
  if (hd != 64 && hd != 128) return refuse("is built for head_dim 64 and 128");
  if (nkv < 1 || nq < 1 || nq % nkv || nq / nkv > kChRows) return refuse("needs nq % nkv == 0 and at most 128 query heads per KV head");
  if (block_size < kChGran || block_size % kChGran) return refuse("needs a block size that is a multiple of 16");
  if (tokens < 0 || batch < 0 || max_blocks < 0) return refuse("needs sizes that are not below 0");
  if (tokens == 0 || batch == 0) return 0;
  if (n_blocks < 1) return refuse("needs a cache with a block");
  if (int64_t(n_blocks) * nkv * block_size > 0x7fffffffLL - kChKeys) return refuse("needs a cache whose rows (tokens times KV heads) fit 32 bits");
  if (int64_t(max_blocks) * block_size > 0x3fffffffLL) return refuse("needs tables of less than 2^30 tokens");
  if (q_stride % 8 || q_stride < 0 || (tokens > 1 && q_stride < int64_t(nq) * hd)) return refuse("needs rows of q on 16-byte boundaries that hold nq heads");
  if (!q || (cache4 ? k_cache || v_cache : !k_cache || !v_cache) || (!block_tables && max_blocks) || !cu_q || !ctx_lens || !out)
    return refuse("needs queries, one kind of cache, block tables, row offsets, context lengths and an output");
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache) | reinterpret_cast<uintptr_t>(cache4) |
       reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(ws)) & 15)
    return refuse("needs tensors on 16-byte boundaries");
  if (!(scale > 0.f) || scale > 3e38f) return refuse("needs a positive scale");
  if (!ws || ws_bytes < bl_paged_attn_chunk_ws(tokens, nq, nkv, hd)) return refuse("needs the workspace that bl_paged_attn_chunk_ws says");

  const int runs = sm_count();
  Chunk a;
  a.G = nq / nkv;
  a.T = chunk_tile_tokens(a.G);
  a.cu = cu_q;
  a.ctx_lens = ctx_lens;
  a.tables = block_tables;
  a.cache4 = static_cast<const uint8_t*>(cache4);
  a.out = static_cast<__nv_bfloat16*>(out);
  a.part = static_cast<float*>(ws);
  a.row_cap = chunk_row_cap(tokens, a.G);
  a.meta = reinterpret_cast<ChunkMeta*>(a.part + 2 * size_t(runs) * a.row_cap * (hd + 2));
  a.tokens = tokens; a.batch = batch; a.nq = nq; a.nkv = nkv; a.block_size = block_size; a.n_blocks = n_blocks; a.max_blocks = max_blocks;
  a.box = block_size % 64 == 0 ? 64 : block_size % 32 == 0 ? 32 : 16;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.polls = g_chunk_polls.load();

  const DriverApi* d = driver(err, errlen);
  if (!d) return -1;
  CUtensorMap tq, tk, tv;
  {
    const cuuint64_t dims[3] = {cuuint64_t(hd), cuuint64_t(nq), cuuint64_t(tokens)};
    const cuuint64_t strides[2] = {cuuint64_t(hd) * 2, cuuint64_t(tokens > 1 ? q_stride : nq * hd) * 2};
    const cuuint32_t box[3] = {64, cuuint32_t(a.G), cuuint32_t(a.T)}, step[3] = {1, 1, 1};
    const CUresult r = d->cuTensorMapEncodeTiled(&tq, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(q), dims, strides, box, step,
                                                 CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                                 CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return refuse("could not describe the queries to TMA");
  }
  if (cache4) {
    tk = tv = tq;
  } else {
    const uint64_t rows = uint64_t(n_blocks) * nkv * block_size;
    if (make_tmap_kmajor(k_cache, rows, uint64_t(hd), uint64_t(hd), uint32_t(a.box), 2, &tk, err, errlen) ||
        make_tmap_kmajor(v_cache, rows, uint64_t(hd), uint64_t(hd), uint32_t(a.box), 2, &tv, err, errlen))
      return -1;
  }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  static bool attr[4][64] = {};
  auto go = [&](auto* kernel, auto* merge, unsigned smem, unsigned threads, bool (&done)[64]) {
    cudaError_t e = allow_smem(reinterpret_cast<const void*>(kernel), int(smem), done);
    if (e == cudaSuccess) e = launch_k(kernel, dim3(runs), dim3(threads), smem, st, tq, tk, tv, a);
    if (e == cudaSuccess) e = launch_k(merge, dim3(runs, a.row_cap < 32 ? a.row_cap : 32), dim3(kChMergeWarps * 32), 0, st, a);
    return e;
  };
  cudaError_t e;
  if (hd == 128)
    e = cache4 ? go(k_chunk_attn<128, true>, k_chunk_merge<128>, ChunkShape<128, true>::kSmem, ChunkShape<128, true>::kThreads, attr[0])
               : go(k_chunk_attn<128, false>, k_chunk_merge<128>, ChunkShape<128, false>::kSmem, ChunkShape<128, false>::kThreads, attr[1]);
  else
    e = cache4 ? go(k_chunk_attn<64, true>, k_chunk_merge<64>, ChunkShape<64, true>::kSmem, ChunkShape<64, true>::kThreads, attr[2])
               : go(k_chunk_attn<64, false>, k_chunk_merge<64>, ChunkShape<64, false>::kSmem, ChunkShape<64, false>::kThreads, attr[3]);
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) {
    set_err(err, errlen, "barlink: attention of a chunk over the paged cache could not be launched: %s", cudaGetErrorString(e));
    return -1;
  }
  return 0;
}
