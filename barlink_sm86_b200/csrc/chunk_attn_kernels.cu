// SPDX-License-Identifier: MIT
//
// Attention of a chunk of new tokens of each request over its paged key/value cache (bf16, or in 4 bits: kv4.cuh), the chunk's own tokens
// included: token i of n new ones, of a request with c tokens in all, sees keys 0 .. c - n + i.
//
// The query heads that share a KV head, times T = 128 / (heads that share) tokens, are the 128 rows of a tile of tcgen05 products, so that a
// chunk of a few tokens reads its keys once for all of them.  A block has places for two tiles; the keys come in steps of 128.  Where a request has
// new tokens for more than a tile, the two hold neighbouring tiles ("a pair") and share every step's keys and values; where it has not (the
// case that is bound by memory and by the chain scores -> softmax -> values) both hold the same tile and take the steps in turn, and their
// sums are joined at the end.
//
//   warp 0      asks for keys, warp 3 for values: boxes of up to 64 tokens of a block by TMA; 4-bit cache: parts of 16-token tiles by bulk copies
//   warp 3      also walks the list, and asks for queries: one three-dimensional box is a tile (64 dims, the heads, T tokens)
//   warps 1, 2  issue S = Q K^T (128 x 64 into TMEM) and O += P V (128 x hd in TMEM) of a place each, the next S right behind P V
//   warps 4-7   softmax of the first place's rows, one row a thread: P (bf16) goes over S in TMEM, from where it is an operand
//   warps 8-11  the same for the second place
//   warps 12-19 (4-bit cache) expand codes into bf16 tiles in the layout that TMA would leave
//
// A step's scores come in halves of 64 keys, each with columns of its own, so that a place's softmax always finds scores while its products go on.  S of
// a half goes into the columns from which P V of the same half of the step before, issued ahead of it and not waited for, takes P: one thread
// issues both, and the tensor pipe works off a thread's products in the order in which they are issued.
//
// Steps of all pairs of all requests and KV heads make one list, of which every block takes an equal run: lengths are known on the GPU only.  A pair
// that is cut leaves its pieces (sums, maxima) to a second kernel.
//
// Measured, as captured and replayed (heads / KV heads x dims; ideal: bytes at the rate of a copy, or products at that of a large matrix product):
//   bf16   5 tokens on 333, 28/4x128             11 us          two launches and one step's chain: 5 us until the first keys are there, 2 for the pieces
//          64 requests of up to 8 on 1100        27 us (10)     1.8 pairs a block, of four steps each: the first one's start and every pair's end
//          9 of up to 700 on 5001, 14/2x128      89 us (42)     the chain below, and pairs' ends; 80 to 89 with other lengths
//          2048 on 16383, 40/8x128              559 us (387)    1.16 PFLOP/s; 650 us where it runs for long and the clock drops
//   4-bit  4 on 900, 28/4x128                    13 us          as the first, and the first keys' conversion
//          64 of up to 6 on 1100                 32 us (3.4)    as the 64 above, with longer steps
//          2 of up to 13 on 100000, 40/8x128    125 us (29)     3400 cycles a step (61 a block; 119 to 145 us with other lengths), in which a quarter of the SM
//                                                              issues 2200 warp instructions: 800 to expand codes, the softmax, and looks at barriers.  35 % of
//                                                              its slots stay empty: each half step's expansion is a chain of its own (a wait, loads, 200
//                                                              instructions that depend on one another, stores, a fence), one warp for keys and one for values
//          1500 on 9000, 28/4x128               221 us (106)    the same, and the softmax of full tiles
// Where new tokens fill tiles a step of two tiles takes some 3900 cycles of an SM; its products 2560 (S of 64 keys at a time reads its operands from shared
// memory at three quarters of the rate of 128, which would leave a place no scores to go on with), its exponentials 1540 of the unit for them.  The rest is
// the chain of a place's half step: products seen to be done, scores read, largest one, exponentials, P seen to be there.
//
// Tokens of table entries that name no block are left out (their boxes start behind the cache, so TMA fills in zeros).  What stands in the cache
// behind a request's last token may be anything: the values of the rest of its box are set to zero in shared memory.
//
// A pair's products go through the keys of its last token, so that a row meets up to 2 T - 1 values that it does not see; they weigh nothing, but 0 x
// infinity is NaN.  Rows that end up with a number that is none are looked at by the second kernel: where such a value is hidden from the row, the
// dims concerned are computed once more from what it sees.
//
// Every wait is bounded.  A run that gives up waits for its copies and products, leaves NaN for the rows of its run and sets the call's error word.
#include <cuda_bf16.h>
#include <stdint.h>

#include <algorithm>
#include <atomic>

#include "attn_tc.cuh"
#include "bl_ops.h"
#include "heap.h"
#include "kv4.cuh"
#include "launch.h"
#include "ptx.cuh"

namespace bl {

constexpr int kChRows = 128;   // of a tile
constexpr int kChKeys = 128;   // of a step
constexpr int kChGran = 16;    // tokens that lie together in either cache
constexpr int kChGrans = kChKeys / kChGran;
constexpr int kChRaw = 3;      // half steps of the 4-bit cache in flight
constexpr int kChHalf = kChKeys / 2;
constexpr uint32_t kChTmemCols = 512;  // S of place t, half h of a step: 128 t + 64 h, P in its first half; O of place t: 256 + 128 t
// Of four pairs of exponentials, those on the FMA pipe (bf16 cache).  2048 tokens on 16383: none 573 us, one 553, two 589; 9 requests of up to 700 on 5001: 94,
// 87, 91.  The 4-bit cache's blocks have no issue slots for them (1500 on 9000: none 214 us, one 224).
constexpr int kChPoly = 1;
// What a pair costs beside its steps (queries, sums, a chain that starts anew), in steps: that many empty ones, or one more, follow it in the list.
// 64 requests of up to 8 tokens on 1100 without any 36.5 us, with 2 or 3 25.7; 9 of up to 700 on 5001 without 138, 3: 91, 2: 89.5; 4-bit cache, 64 of up to 6 on
// 1100 without 42, 3: 33.0, 4: 32.6, 8: 41.
constexpr int chunk_over(bool q4) { return q4 ? 4 : 2; }
constexpr float kChRescale = 8.f;      // log2 units
constexpr uint32_t kChPolls = 1u << 24;

__device__ uint32_t g_chunk_err;  // set by a wait that ran out in a call without a word of its own; one per device

struct ChunkMeta {
  int count;                // pieces of the pair that begins in this run and ends in another; 0: none does
  int first;                // its first piece; piece k of the others is the first of run me + k
  int h, row, ntok;         // KV head, first row of q and out, tokens of the pair
  int odd;                  // whether this run wrote a row that holds an infinity or NaN
};

// n / d for 0 <= n < 2^31 by a product: with m = ceil(2^(31 + s) / d) and 2^s >= d, m d is above 2^(31 + s) by less than 2^s, which n times over stays
// below one quotient's step.
struct ChunkDiv {
  uint32_t m;
  int s;
  __device__ __forceinline__ int operator()(int n) const { return int(uint64_t(uint32_t(n)) * m >> (31 + s)); }
};
// n / d where the quotient is below 2^16 (the quotient in fp32 is off by less than one)
__device__ __forceinline__ int small_div(int n, int d) {
  int q = int(__fdividef(float(n), float(d)));
  const int r = n - q * d;
  return r < 0 ? q - 1 : r >= d ? q + 1 : q;
}

struct Chunk {
  const int* cu;
  const int* ctx_lens;
  const int* tables;
  const uint8_t* cache4;
  const __nv_bfloat16 *q, *k, *v;
  __nv_bfloat16* out;
  float* part;   // [2 * runs][row_cap][hd], then [2 * runs][row_cap] (maximum, sum)
  ChunkMeta* meta;
  uint32_t* error;  // the caller's word, or none
  size_t q_stride;
  int again;     // rows that hold an infinity or NaN are looked at (q is still there)
  int tokens, batch, nq, nkv, G, T, block_size, n_blocks, max_blocks, row_cap, box;
  float scale_log2;
  uint32_t polls;
  ChunkDiv by_runs, by_block, by_pair;
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
__device__ __forceinline__ int chunk_pairs(const Chunk& a, const ChunkReq& r) { return a.by_pair(r.n + 2 * a.T - 1); }
// Where pair p of a request begins in its part of the list: floor(sum of the keys of the pairs before / 128) + p (1 + over).  A pair of x keys has no more
// than floor(x / 128) + 1 steps, so that there is room for them and for `over` or one more empty ones; and the sum (keys grow evenly from pair to pair,
// between 0 and what the table holds) needs no loop.
__device__ __forceinline__ int chunk_upto(const Chunk& a, const ChunkReq& r, int p, int over) {
  const int q1 = r.cap > r.past ? min(p, a.by_pair(r.cap - r.past - 1)) : 0;  // pairs 1 .. q1 end below the table's end,
  const int q0 = r.past < 0 ? min(q1, a.by_pair(-r.past)) : 0;                // 1 .. q0 ahead of the first key
  const int64_t keys = int64_t(q1 - q0) * r.past + a.T * (int64_t(q1) * (q1 + 1) - int64_t(q0) * (q0 + 1)) + int64_t(p - q1) * r.cap;
  return int(keys >> 7) + p * (1 + over);
}

// A run's share of a pair, as the warp that walks the list leaves it for the others.
struct ChunkSeg {
  int b, h;
  int row, ntok;    // first row of q and out, tokens
  int keys;         // that the last token sees
  int lim, cap;     // the first token sees min(lim, cap) keys, and each one more, up to cap
  int j0, n, i0;    // first step, steps (0: the run is over), number of the first one in the run
  int piece;        // -1: the whole pair
  int cut;          // the last step has its first half only
};
constexpr int kChSegs = 4;

template <int HD, bool Q4>
struct ChunkShape {
  static constexpr int kThreads = Q4 ? 640 : 384, kOver = chunk_over(Q4);
  static constexpr uint32_t kQ = kChRows * HD * 2, kKV = kChKeys * HD * 2, kHalf = kChKeys * 128, kQHalf = kChRows * 128;
  static constexpr uint32_t kRawGran = 10 * HD, kRawBytes = (kChGrans / 2) * kRawGran;  // codes and params of a granule's keys, or of its values
  static constexpr uint32_t kOffK = 2 * kQ, kOffV = kOffK + 2 * kKV, kOffRaw = kOffV + 2 * kKV;
  static constexpr uint32_t kOffSums = kOffRaw + (Q4 ? 2 * kChRaw * kRawBytes : 0);  // (maximum, sum) of the second place's rows
  static constexpr uint32_t kOffBar = kOffSums + kChRows * 8;
  static constexpr uint32_t kSmem = kOffBar + 768 + 1024;  // barriers, words, shares of pairs; room to align
  static_assert(kSmem <= 232448 - 256, "attention tiles do not fit the shared memory of one block");
};

struct ChunkBars {
  uint64_t q_full[2], q_empty[2];
  uint64_t k_full[2][2], k_empty[2][2], v_full[2][2], v_empty[2][2];  // by slot and half
  uint64_t raw_full[2][kChRaw], raw_empty[2][kChRaw];  // keys, values
  uint64_t s_ready[2][2], p_ready[2][2];        // by place and half
  uint64_t pv_done[2], o_final[2], o_free[2];   // by place
  uint64_t met[2];   // see the products
  uint64_t sums;     // the second place's (maximum, sum) are there
  uint64_t drained[2];
  uint64_t seg_full[kChSegs], seg_empty[kChSegs];
  ChunkSeg segs[kChSegs];
  uint32_t tmem, abort;
  uint32_t never;    // set where a wait for the list ran out
  uint32_t has[2][kChRaw];  // 4-bit cache: granules that a raw half has copies of
  uint32_t gone[8];  // granules of a step (by its number in the run, modulo 8) that have no block
};
static_assert(sizeof(ChunkBars) <= 768, "barriers");

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// 2^x of two numbers on the FMA pipe: x = n + f, |f| <= 1/2, 2^f by the polynomial of degree 3 whose relative error is least (7.5e-5; P is rounded to
// 2^-8 behind it), 2^n by its bits.  Exactly 0 below -127, -inf included; NaN stays.
__device__ __forceinline__ float2 ex2_poly(float2 x) {
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(x.x) : "f"(-127.f));
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(x.y) : "f"(-127.f));
  const float2 magic = make_float2(12583039.f, 12583039.f);  // 1.5 * 2^23 + 127: adding it leaves n + 127 in the lowest bits
  const float2 t = add2(x, magic);
  const float2 f = add2(x, fma2(t, make_float2(-1.f, -1.f), magic));
  float2 p = fma2(f, make_float2(0.0551716685f, 0.0551716685f), make_float2(0.242611125f, 0.242611125f));
  p = fma2(p, f, make_float2(0.693260968f, 0.693260968f));
  p = fma2(p, f, make_float2(0.999928057f, 0.999928057f));
  return mul2(p, make_float2(__uint_as_float(__float_as_uint(t.x) << 23), __uint_as_float(__float_as_uint(t.y) << 23)));
}
// S of a tile: hd / 16 products, in both operands 64 dims to a half tile of 128 rows (16 KiB).  (Few instructions: predicates are made once, and only the low
// words of the operands' descriptors change.)
template <int HD>
__device__ __forceinline__ void umma_f16_ss_row_warp(uint32_t leader, uint32_t d, uint64_t qa, uint64_t kb, uint32_t idesc) {
  const uint32_t qlo = uint32_t(qa), qhi = uint32_t(qa >> 32), klo = uint32_t(kb), khi = uint32_t(kb >> 32);
  uint32_t acc = 0;
  asm volatile(
      "{\n\t.reg .pred q, f, t;\n\t.reg .b64 x, y;\n\t.reg .b32 u, v;\n\t"
      "setp.ne.b32 q, %6, 0;\n\tsetp.ne.b32 f, %7, 0;\n\tsetp.eq.b32 t, 0, 0;\n\t"
      "add.u32 u, %1, 0;\n\tadd.u32 v, %3, 0;\n\tmov.b64 x, {u, %2};\n\tmov.b64 y, {v, %4};\n\t@q tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %5, f;\n\t"
      "add.u32 u, %1, 2;\n\tadd.u32 v, %3, 2;\n\tmov.b64 x, {u, %2};\n\tmov.b64 y, {v, %4};\n\t@q tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %5, t;\n\t"
      "add.u32 u, %1, 4;\n\tadd.u32 v, %3, 4;\n\tmov.b64 x, {u, %2};\n\tmov.b64 y, {v, %4};\n\t@q tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %5, t;\n\t"
      "add.u32 u, %1, 6;\n\tadd.u32 v, %3, 6;\n\tmov.b64 x, {u, %2};\n\tmov.b64 y, {v, %4};\n\t@q tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %5, t;\n\t"
      "}" ::"r"(d),
      "r"(qlo), "r"(qhi), "r"(klo), "r"(khi), "r"(idesc), "r"(leader), "r"(acc)
      : "memory");
  if constexpr (HD == 128) {
    acc = 1;
    asm volatile(
      "{\n\t.reg .pred q, f, t;\n\t.reg .b64 x, y;\n\t.reg .b32 u, v;\n\t"
      "setp.ne.b32 q, %6, 0;\n\tsetp.ne.b32 f, %7, 0;\n\tsetp.eq.b32 t, 0, 0;\n\t"
      "add.u32 u, %1, 1024;\n\tadd.u32 v, %3, 1024;\n\tmov.b64 x, {u, %2};\n\tmov.b64 y, {v, %4};\n\t@q tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %5, f;\n\t"
      "add.u32 u, %1, 1026;\n\tadd.u32 v, %3, 1026;\n\tmov.b64 x, {u, %2};\n\tmov.b64 y, {v, %4};\n\t@q tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %5, t;\n\t"
      "add.u32 u, %1, 1028;\n\tadd.u32 v, %3, 1028;\n\tmov.b64 x, {u, %2};\n\tmov.b64 y, {v, %4};\n\t@q tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %5, t;\n\t"
      "add.u32 u, %1, 1030;\n\tadd.u32 v, %3, 1030;\n\tmov.b64 x, {u, %2};\n\tmov.b64 y, {v, %4};\n\t@q tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %5, t;\n\t"
      "}" ::"r"(d),
      "r"(qlo), "r"(qhi), "r"(klo), "r"(khi), "r"(idesc), "r"(leader), "r"(acc)
      : "memory");
  }
}
// P V of half a step: four products of 16 keys, P in 32 columns of TMEM, 16 keys of V 2 KiB apart
__device__ __forceinline__ void umma_f16_ts4_warp(uint32_t leader, uint32_t d, uint32_t pa, uint64_t vb, uint32_t idesc, uint32_t accumulate) {
  const uint32_t vlo = uint32_t(vb), vhi = uint32_t(vb >> 32);
  asm volatile(
      "{\n\t.reg .pred q, f, t;\n\t.reg .b64 y;\n\t.reg .b32 x, v;\n\t"
      "setp.ne.b32 q, %5, 0;\n\tsetp.ne.b32 f, %6, 0;\n\tsetp.eq.b32 t, 0, 0;\n\t"
      "add.u32 x, %1, 0;\n\tadd.u32 v, %2, 0;\n\tmov.b64 y, {v, %3};\n\t@q tcgen05.mma.cta_group::1.kind::f16 [%0], [x], y, %4, f;\n\t"
      "add.u32 x, %1, 8;\n\tadd.u32 v, %2, 128;\n\tmov.b64 y, {v, %3};\n\t@q tcgen05.mma.cta_group::1.kind::f16 [%0], [x], y, %4, t;\n\t"
      "add.u32 x, %1, 16;\n\tadd.u32 v, %2, 256;\n\tmov.b64 y, {v, %3};\n\t@q tcgen05.mma.cta_group::1.kind::f16 [%0], [x], y, %4, t;\n\t"
      "add.u32 x, %1, 24;\n\tadd.u32 v, %2, 384;\n\tmov.b64 y, {v, %3};\n\t@q tcgen05.mma.cta_group::1.kind::f16 [%0], [x], y, %4, t;\n\t"
      "}" ::"r"(d),
      "r"(pa), "r"(vlo), "r"(vhi), "r"(idesc), "r"(leader), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tmem_st_32x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
      "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// Keeps the compiler from making a copy of a loop for either value of a flag (what does not fit the instruction cache is fetched once a step).
__device__ __forceinline__ bool one_copy(bool flag) {
  int f = flag;
  asm volatile("" : "+r"(f));
  return f != 0;
}

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
  const uint32_t abort_at = smem_u32(&bars.abort), never_at = smem_u32(&bars.never);
  __shared__ int s_scan[S::kThreads / 32];
  int* s_upto = reinterpret_cast<int*>(gen + S::kOffK);  // (ahead of the first copy)

  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int t = 0; t < 2; ++t) {
      mbar_init(&bars.q_full[t], 1);
      mbar_init(&bars.q_empty[t], 1);
      for (int h = 0; h < 2; ++h) {
        mbar_init(&bars.s_ready[t][h], 1);
        mbar_init(&bars.p_ready[t][h], kChRows / 32);
      }
      mbar_init(&bars.pv_done[t], 1);
      mbar_init(&bars.o_final[t], 1);
      mbar_init(&bars.o_free[t], kChRows / 32);
    }
    for (int s = 0; s < 2; ++s) {
      for (int h = 0; h < 2; ++h) {
        mbar_init(&bars.k_full[s][h], Q4 ? 4 : 1);
        mbar_init(&bars.v_full[s][h], Q4 ? 4 : 1);
        mbar_init(&bars.k_empty[s][h], 2);
        mbar_init(&bars.v_empty[s][h], 2);
      }
      mbar_init(&bars.met[s], 1);
    }
    for (int s = 0; s < kChRaw; ++s)
      for (int v = 0; v < 2; ++v) {
        mbar_init(&bars.raw_full[v][s], 1);
        mbar_init(&bars.raw_empty[v][s], 4);
      }
    mbar_init(&bars.sums, kChRows / 32);
    for (int t = 0; t < 2; ++t) mbar_init(&bars.drained[t], 1);
    for (int i = 0; i < kChSegs; ++i) {
      mbar_init(&bars.seg_full[i], 1);
      mbar_init(&bars.seg_empty[i], S::kThreads / 32 - 1);  // all warps but the one that fills them
    }
    bars.abort = 0;
    bars.never = 0;
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

  // ---- the list's length, up to each thread's requests ----
  const int runs = gridDim.x, me = blockIdx.x, pair = 2 * a.T;
  const int per = (a.batch + S::kThreads - 1) / S::kThreads;
  {
    int upto = 0;
#pragma unroll 1
    for (int k = 0; k < per; ++k) {
      const int b = int(threadIdx.x) * per + k;
      if (b >= a.batch) break;
      const ChunkReq r = chunk_req(a, b);
      upto += chunk_upto(a, r, chunk_pairs(a, r), S::kOver) * a.nkv;
    }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(kAll, upto, o);
      if (lane >= o) upto += v;
    }
    s_upto[threadIdx.x] = upto;
    fence_proxy_async_smem();  // (copies go there behind the barriers)
    if (lane == 31) s_scan[warp] = upto;
    if (threadIdx.x == 0) a.meta[me].odd = 0;  // (ahead of the barrier; whoever sets it is behind)
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = bars.tmem;
  // Warp 3 finds the run's first step while the others wait here for its first share.
  auto begin = [] { asm volatile("bar.sync 0;" ::: "memory"); };
  // Step j of a share has slot j & 1 of the keys and of the values, so that a share with one tile has a slot to a place; a slot is filled and emptied by
  // halves, of which a pair's last step may have the first only, and a role knows a half's phase by how often it has been filled.
  struct Fills {
    uint32_t n[2][2] = {{0, 0}, {0, 0}};
    __device__ __forceinline__ uint32_t of(int j, int h) const {  // ahead of step j
      return (j & 1 ? (h ? n[1][1] : n[1][0]) : (h ? n[0][1] : n[0][0])) + uint32_t(j >> 1);
    }
    __device__ __forceinline__ void add(const ChunkSeg& s) {
      const uint32_t a = uint32_t(s.n + 1) >> 1, b = uint32_t(s.n) >> 1;
      n[0][0] += a;
      n[1][0] += b;
      n[0][1] += a - (s.cut && (s.n & 1) ? 1 : 0);
      n[1][1] += b - (s.cut && !(s.n & 1) ? 1 : 0);
    }
  };
  bool ok = true;
  // Softmax warps of the bf16 cache look at a barrier all the time (9 requests of up to 700 on 5001: 87 us; pausing between looks: 89).  With the 4-bit cache, whose
  // warps are short of issue slots, they pause, as its converting warps do (1500 on 9000: 217 us; looking all the time: 225).
  auto wait_for = [&](uint64_t* bar, uint32_t parity) {
    if constexpr (!Q4) return mbar_spin_warp(bar, parity & 1u, s_abort, a.polls);
    return mbar_wait_quick_warp(bar, parity & 1u, abort_at, a.polls);
  };
  // All roles are through; behind it `abort` stays as it is.
  auto settle = [&] {
    tc_fence_before_sync();
    asm volatile("bar.sync 0;" ::: "memory");
    return *s_abort != 0;
  };
  // Every role goes through the run's shares of pairs: f(share, whether it has two tiles).  After a wait that ran out they go on without work.
  auto each = [&](auto&& f) {
    begin();
#pragma unroll 1
    for (int k = 0;; ++k) {
      if (k > 0 && !mbar_wait_call(smem_u32(&bars.seg_full[k % kChSegs]), uint32_t(k / kChSegs) & 1u, never_at, 1u << 22)) {
        *s_abort = 1;
        return;
      }
      const ChunkSeg s = bars.segs[k % kChSegs];
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars.seg_empty[k % kChSegs]);
      if (s.n == 0) return;
      f(s, s.ntok > a.T);
    }
  };

  if (warp == 0 || warp == 3) {
    // ------------------------------ keys (warp 0); the list, queries and values (warp 3) ------------------------------
    const uint32_t leader = elect_leader();
    const int values = warp == 3;
    uint64_t (*full)[2] = values ? bars.v_full : bars.k_full;
    uint64_t (*empty)[2] = values ? bars.v_empty : bars.k_empty;
    const CUtensorMap* tmap = values ? &tmap_v : &tmap_k;
    const uint32_t ring = base + (Q4 ? S::kOffRaw + values * kChRaw * S::kRawBytes : values ? S::kOffV : S::kOffK);
    int rs = 0, issued = 0;  // (4-bit cache: a ring of its own)
    uint32_t rphase = 1;
    Fills fills;
    uint32_t asked00 = 0, asked01 = 0, asked10 = 0, asked11 = 0;  // of either slot's halves
    uint32_t gone_before = 0;  // bit s: bars.gone[s] is set
    auto load = [&](const ChunkSeg& s) {
      const int* table = a.tables + size_t(s.b) * a.max_blocks;
      // lane l: granule l of four steps -- the row of the cache where it begins (tile of the 4-bit cache), -1: nothing visible, -2: no block
      auto look = [&](int j) {
        const int tok = j * kChKeys + lane * kChGran;
        int at = -1;
        if (tok < s.keys) {
          const int page = a.by_block(tok), blk = table[page], in = tok - page * a.block_size;
          at = blk < 0 || blk >= a.n_blocks ? -2 : Q4 ? (blk * a.nkv + s.h) * (a.block_size / kQ4Tokens) + in / kQ4Tokens : (blk * a.nkv + s.h) * a.block_size + in;
        }
        return at;
      };
      int ahead = look(s.j0), where = 0;
      const int none = a.n_blocks * a.nkv * a.block_size;  // behind the cache
#pragma unroll 1
      for (int j = 0; j < s.n; ++j) {
        const int part = j & 3, i = s.i0 + j;
        if (part == 0) {
          where = ahead;
          ahead = look(s.j0 + j + 4);
        }
        const uint32_t lost = __ballot_sync(kAll, where == -2) >> (kChGrans * part) & 255u;
        const int st = j & 1;
#pragma unroll 1
        for (int h = 0; h < 2 - (s.cut && j == s.n - 1 ? 1 : 0); ++h) {
          uint64_t* bar = Q4 ? &bars.raw_full[values][rs] : &full[st][h];
          if (!(ok = mbar_wait_quick_warp(Q4 ? &bars.raw_empty[values][rs] : &empty[st][h], (Q4 ? rphase : fills.of(j, h) + 1u) & 1u, abort_at, a.polls))) return;
          if (!values && h == 0) {
            if (lane == 0 && (lost || (gone_before >> (i & 7) & 1u))) bars.gone[i & 7] = lost;
            gone_before = (gone_before & ~(1u << (i & 7))) | uint32_t(lost != 0) << (i & 7);
            __syncwarp();
          }
          if constexpr (!Q4) {
            // (the whole warp stays together and one lane issues)
            mbar_expect_tx_warp(leader, bar, S::kKV / 2);
#pragma unroll 1
            for (int gr = kChGrans / 2 * h; gr < kChGrans / 2 * (h + 1); gr += a.box / kChGran) {
              const int at = __shfl_sync(kAll, where, kChGrans * part + gr);
#pragma unroll
              for (int d = 0; d < HD / 64; ++d)
                tma_load_2d_hint_warp(leader, ring + st * S::kKV + d * S::kHalf + gr * (kChGran * 128), tmap, smem_u32(bar), d * 64, at >= 0 ? at : none, kHintEvictLast);
            }
            ++issued;
            if (st) {
              if (h) ++asked11; else ++asked10;
            } else {
              if (h) ++asked01; else ++asked00;
            }
          } else {
            // lanes 0..3 ask for the codes of a granule, 4..7 for its steps and least elements; one that is not there leaves what stood there before
            const int at = __shfl_sync(kAll, where, kChGrans * part + 4 * h + (lane & 3));
            const uint32_t has = __ballot_sync(kAll, at >= 0) & 15u;
            if (lane == 0) bars.has[values][rs] = has;
            __syncwarp();
            mbar_expect_tx_warp(leader, bar, uint32_t(__popc(has)) * S::kRawGran);
            const bool params = lane >= 4;
            const uint8_t* from = a.cache4 + size_t(max(at, 0)) * q4_tile_bytes(HD) + (values ? (params ? q4_v_params(HD) : q4_v_codes(HD)) : params ? q4_k_params(HD) : 0);
            bulk_load_warp(lane < 8 && at >= 0, ring + rs * S::kRawBytes + (lane & 3) * S::kRawGran + (params ? 8 * HD : 0), from, params ? 2 * HD : 8 * HD,
                           smem_u32(bar), kHintEvictFirst);
            ++issued;
            if (++rs == kChRaw) {
              rs = 0;
              rphase ^= 1u;
            }
          }
        }
      }
      fills.add(s);
    };
    const uint32_t bytes = uint32_t(a.G) * a.T * HD * 2;
    int asked[2] = {0, 0};  // query tiles asked for, by place
    ChunkMeta m = {};       // what the second kernel needs to know
    // ---- this block's run [lo, lo + count) of the list, and where it begins ----
    int b = 0, h = 0, p = 0, p_at = 0, j0 = 0, run = 0, lo = 0, count = 0;  // (pair p, which begins at p_at)
    ChunkReq r = {0, 0, 0, 0};
    if (values) {
      const int w = lane < S::kThreads / 32 ? s_scan[lane] : 0;  // (at most twenty warps)
      int at = w;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(kAll, at, o);
        if (lane >= o) at += v;
      }
      const int total = __shfl_sync(kAll, at, 31);
      run = a.by_runs(total + runs - 1);
      lo = min(me * run, total);
      count = min(run, total - lo);
      if (count > 0) {
        // (Lengths that another stream changes meanwhile, which nobody may, or row offsets that fall, whose sum may pass 31 bits, are to leave nothing
        // worse than wrong rows: what is found stays in range.)
        const int of = max(__ffs(__ballot_sync(kAll, lo < at)) - 1, 0);
        at = __shfl_sync(kAll, at - w, of);
        const int upto = at + s_upto[of * 32 + lane], src = max(__ffs(__ballot_sync(kAll, lo < upto)) - 1, 0);
        if (src > 0) at = __shfl_sync(kAll, upto, src - 1);
        // the request that holds the first step; its KV head, and the pair
        int u = 0;
        b = min((of * 32 + src) * per, a.batch - 1) - 1;
        do {
          at += u * a.nkv;
          r = chunk_req(a, ++b);
          u = chunk_upto(a, r, chunk_pairs(a, r), S::kOver);
        } while (lo >= at + u * a.nkv && b + 1 < a.batch);
        u = max(u, 1);
        h = min(max(small_div(lo - at, u), 0), a.nkv - 1);
        const int in = lo - at - h * u;
#pragma unroll 1
        for (int many = chunk_pairs(a, r); many > 1;) {
          const int stride = (many + 31) / 32;
          const int top = 31 - __clz(__ballot_sync(kAll, lane * stride < many && chunk_upto(a, r, p + lane * stride, S::kOver) <= in) | 1);
          p += top * stride;
          many = min(stride, many - top * stride);
        }
        p_at = chunk_upto(a, r, p, S::kOver);
        j0 = in - p_at;
      }
    }
#pragma unroll 1
    for (int k = 0, i = 0, done = 0;; ++k) {
      const uint32_t slot = k % kChSegs, turn = uint32_t(k / kChSegs) & 1u;
      if (k >= (values ? kChSegs : 1) && !mbar_wait_call(smem_u32(values ? &bars.seg_empty[slot] : &bars.seg_full[slot]), values ? turn ^ 1u : turn, never_at, 1u << 22)) {
        *s_abort = 1;
        break;
      }
      if (values && lane == 0) {
        // the next share of a pair
        ChunkSeg s = {};
#pragma unroll 1
        while (i < count && s.n == 0) {
          s.b = b;
          s.h = h;
          const int tok0 = p * pair;
          s.row = r.q0 + tok0;
          s.ntok = min(pair, r.n - tok0);
          s.keys = chunk_keys(r, tok0, s.ntok);
          s.lim = r.past + tok0 + 1;
          s.cap = r.cap;
          const int steps = chunk_steps(s.keys);
          s.j0 = j0;
          s.n = min(max(steps - j0, 0), count - i);  // (0: the run begins behind the pair's steps)
          s.i0 = done;
          s.cut = s.keys - (j0 + s.n - 1) * kChKeys <= kChHalf;
          s.piece = s.n == steps ? -1 : 2 * me + (i == 0 ? 0 : 1);
          if (j0 == 0 && s.n < steps) m = {small_div(lo + i + steps - 1, run) - me + 1, s.piece, h, s.row, s.ntok, 0};
          done += s.n;
          i -= p_at + j0;
          i += p_at = chunk_upto(a, r, ++p, S::kOver);
          j0 = 0;
          if (tok0 + pair >= r.n) {
            p = p_at = 0;
            if (++h == a.nkv && i < count) {
              h = 0;
              do
                if (++b < a.batch) r = chunk_req(a, b);
              while (b < a.batch && r.n == 0);
              if (b >= a.batch) i = count;  // (not with steps left, but see above)
            }
          }
        }
        bars.segs[slot] = s;
        mbar_arrive(&bars.seg_full[slot]);
      }
      __syncwarp();
      if (k == 0) begin();
      const ChunkSeg s = bars.segs[slot];
      __syncwarp();
      if (!values && lane == 0) mbar_arrive(&bars.seg_empty[slot]);
      if (s.n == 0) break;
      if (values) {
        const bool two = s.ntok > a.T;
#pragma unroll 1
        for (int t = 0; t < 2; ++t) {
          if (!ok || (t == 1 && !two && s.n < 2)) break;
          if (!(ok = mbar_wait_quick_warp(&bars.q_empty[t], (uint32_t(t ? asked[1] : asked[0]) & 1u) ^ 1u, abort_at, a.polls))) break;
          if (lane == 0) {
            mbar_expect_tx(&bars.q_full[t], bytes);
#pragma unroll
            for (int hh = 0; hh < HD / 64; ++hh)
              tma_load_3d_hint_s(base + t * S::kQ + hh * S::kQHalf, &tmap_q, smem_u32(&bars.q_full[t]), hh * 64, s.h * a.G, s.row + (two ? t * a.T : 0), kHintEvictFirst);
          }
          t ? ++asked[1] : ++asked[0];
        }
      }
      if (ok) load(s);
    }
    if (values && lane == 0) {
      ChunkMeta& to = a.meta[me];  // (all but `odd`)
      to.count = m.count;
      to.first = m.first;
      to.h = m.h;
      to.row = m.row;
      to.ntok = m.ntok;
    }
    // The block's shared memory is another's behind it: after a wait that ran out, anyone's, whatever is still on its way lands first.
    const bool gave_up = settle();
    if (gave_up && values)
#pragma unroll 1
      for (int t = 0; t < 2; ++t)
#pragma unroll 1
        for (uint32_t p = 0; asked[t] > 0 && p < (1u << 20); ++p)
          if (mbar_try_wait(&bars.q_full[t], uint32_t(asked[t] - 1) & 1u)) break;
    if (gave_up && issued > 0) {
#pragma unroll 1
      for (int i = 0; i < (Q4 ? kChRaw : 4); ++i) {
        uint64_t* bar = Q4 ? &bars.raw_full[values][i] : &full[i >> 1][i & 1];
        // (what was never asked for has nothing on its way; of the rest the last time counts)
        const uint32_t n = Q4 ? uint32_t((issued + kChRaw - 1 - i) / kChRaw) : i == 0 ? asked00 : i == 1 ? asked01 : i == 2 ? asked10 : asked11;
#pragma unroll 1
        for (uint32_t p = 0; n > 0 && p < (1u << 20); ++p)
          if (mbar_try_wait(bar, (n - 1) & 1u)) break;
      }
    }
  } else if (warp < 3) {
    // ------------------------------ products, a place's by a warp ------------------------------
    // (a wait takes as long as the tensor cores have queued products for: two warps, and one's products fill the other's waits)
    const uint32_t leader = elect_leader();
    const int t = warp - 1;
    const uint32_t idesc_s = umma_idesc_f16(kChRows, kChHalf, 1);
    const uint32_t idesc_o = umma_idesc_f16(kChRows, HD, 1) | kUmmaBMajorN;
    const uint64_t desc_q = umma_desc_k_sw128(base + t * S::kQ), desc_k = umma_desc_k_sw128(base + S::kOffK), desc_v = umma_desc_mn_sw128(base + S::kOffV, S::kHalf);
    const uint32_t s_at = tmem_base + uint32_t(t * 128), o_at = s_at + 256u;
    uint32_t uses[2] = {0, 0}, tiles = 0;  // halves of steps, pairs of this place so far
    Fills fills;
    uint32_t meets = 0;
    bool apart = false;
    auto wait = [&](uint64_t* bar, uint32_t parity) { return ok = mbar_spin_warp(bar, parity & 1u, s_abort, a.polls); };
    auto share = [&](const ChunkSeg& s, bool two) {
      const int every = two ? 1 : 2, n = s.n, begin = two ? 0 : t;  // this place's steps
      if (begin >= n) return;
      const int last = (n - 1 - begin) / every * every + begin;       // this place's last step
      const bool cut = s.cut && last == n - 1;                        // of which there is the first half only
      if (!wait(&bars.q_full[t], tiles)) return;
#pragma unroll 1
      for (int js = begin;; js += every) {
        const int j = js - every, sk = js & 1, sv = j & 1;
        const bool product = one_copy(js != begin), more = js <= last;
#pragma unroll 1
        for (int h = 0; h < 2; ++h) {
          // the scores of half h of step js, ahead of which that half of the place's step before is multiplied by its values
          const bool of = product && !(h == 1 && cut && j == last), next = more && !(h == 1 && cut && js == last), fresh = of && h == 0 && j == begin;
          if (of) {
            if (!wait(&bars.p_ready[t][h], h ? uses[1]++ : uses[0]++)) return;
            if (!wait(&bars.v_full[sv][h], fills.of(j, h))) return;
          }
          // (ahead of the product, behind which a wait takes longer; but the 4-bit cache's next keys may have to wait for the values that it reads)
          if ((!Q4 || !product) && next && !wait(&bars.k_full[sk][h], fills.of(js, h))) return;
          if (of) {
            if (!Q4 && j == last) {
              const int r0 = s.keys - (s.j0 + j) * kChKeys;
              if (r0 > kChHalf * h && r0 < kChHalf * (h + 1) && r0 % a.box) {
                // the rest of the last box: probabilities are zero there, values may be anything
                const int r1 = (r0 + a.box - 1) / a.box * a.box;
#pragma unroll 1
                for (int k = lane + r0 * (HD / 8); k < r1 * (HD / 8); k += 32) {
                  const int r = k / (HD / 8), c = k % (HD / 8);
                  asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(base + S::kOffV + sv * S::kKV + (c >> 3) * S::kHalf + r * 128 + (c & 7) * 16), "r"(0)
                               : "memory");
                }
                fence_proxy_async_smem();
                __syncwarp();
              }
            }
            // a place's first product of a pair: the sums of the pair before have been read
            if (fresh && !wait(&bars.o_free[t], tiles ^ 1u)) return;
            tc_fence_after_sync();
            umma_f16_ts4_warp(leader, o_at, s_at + uint32_t(kChHalf * h), desc_v + uint64_t(sv * int(S::kKV / 16) + h * (kChHalf * 128 / 16)), idesc_o, fresh ? 0u : 1u);
            umma_commit_warp(leader, &bars.pv_done[t]);
            umma_commit_warp(leader, &bars.v_empty[sv][h]);
            if (!two) umma_commit_warp(leader, &bars.v_empty[sv][h]);  // (for the other place)
          }
          if (next) {
            if (Q4 && product && !wait(&bars.k_full[sk][h], fills.of(js, h))) return;
            tc_fence_after_sync();
            umma_f16_ss_row_warp<HD>(leader, s_at + uint32_t(kChHalf * h), desc_q, desc_k + uint64_t(sk * int(S::kKV / 16) + h * (kChHalf * 128 / 16)), idesc_s);
            umma_commit_warp(leader, &bars.s_ready[t][h]);
            umma_commit_warp(leader, &bars.k_empty[sk][h]);
            if (!two) umma_commit_warp(leader, &bars.k_empty[sk][h]);
          }
          if (h == 1 && js == last) umma_commit_warp(leader, &bars.q_empty[t]);  // (the place's last use of the queries)
        }
        if (!more) break;
      }
      umma_commit_warp(leader, &bars.o_final[t]);
      ++tiles;
    };
    each([&](const ChunkSeg& s, bool two) {
      // Where the places go on together after steps apart, each has to know that the other has seen its slot's fills: a phase is told from
      // the one before it, not from older ones.
      if (two && apart) {
        if (lane == 0) mbar_arrive(&bars.met[t]);
        // (a place that has given up meets the other without having seen anything)
        if (ok && wait(&bars.met[t ^ 1], meets) && *s_abort) ok = false;
        ++meets;
      }
      apart = !two;
      if (ok) share(s, two);
      fills.add(s);
    });
    if (settle()) {
      // products on their way read shared memory and write TMEM, which are given back below
      umma_commit_warp(leader, &bars.drained[t]);
      mbar_wait_call(smem_u32(&bars.drained[t]), 0, never_at, 1u << 20);
    }
  } else if (warp >= 12) {
    // ------------------------------ codes of the 4-bit cache to bf16 tiles ------------------------------
    if constexpr (Q4) {
      constexpr int NA = HD / kQ4Group;
      auto words = [&](uint32_t addr, uint32_t (&w)[NA]) {
        if constexpr (NA == 4)
          asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(addr));
        else
          asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(addr));
      };
      auto pair_order = [](int i) { return (i >> 2) * 4 + (i >> 1 & 1) + (i & 1) * 2; };  // 0 2 1 3 4 6 5 7: neighbours are four tokens apart
      // (16 bits 0x430c are the bf16 number 128 + c; low + step * c is rounded once)
      auto value = [&](uint32_t two, __nv_bfloat162 step, __nv_bfloat162 low) {
        const uint32_t c = (two & 0x000f000fu) | 0x43004300u, k = 0xc300c300u;  // - 128
        const __nv_bfloat162 v = __hfma2(__hadd2(*reinterpret_cast<const __nv_bfloat162*>(&c), *reinterpret_cast<const __nv_bfloat162*>(&k)), step, low);
        return *reinterpret_cast<const uint32_t*>(&v);
      };
      auto pair_of = [](uint32_t x, uint32_t y, uint32_t how) {
        const uint32_t v = __byte_perm(x, y, how);
        return *reinterpret_cast<const __nv_bfloat162*>(&v);
      };
      // eight dims, 4 m + t of 8, of a key whose row's place for dims 8 t (swizzled) is `at`: t < 4, so that bit 2 of 4 m is bit 6 of the address
      auto store = [&](uint32_t at, int m, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
        asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"((m & 1 ? at ^ 64u : at) + (m >> 1) * S::kHalf), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
      };
      auto place = [](uint32_t tile, int key, int t) { return tile + uint32_t(key * 128 + ((t ^ (key & 7)) << 4)); };
      const int values = warp >= 16, cwarp = warp & 3;  // warps 12 to 15 keys, 16 to 19 values
      int rs = 0;
      uint32_t rphase = 0;
      Fills fills;
      each([&](const ChunkSeg& s, bool) {
        if (!ok) return;
#pragma unroll 1
        for (int j = 0; j < s.n; ++j) {
          const int left = s.keys - (s.j0 + j) * kChKeys;  // tokens of this step
          const int st = j & 1;
          const uint32_t tile = base + (values ? S::kOffV : S::kOffK) + st * S::kKV;
#pragma unroll 1
          for (int u = 0; u < 2 - (s.cut && j == s.n - 1 ? 1 : 0); ++u) {
            if (!wait_for(&bars.raw_full[values][rs], rphase) || !wait_for(values ? &bars.v_empty[st][u] : &bars.k_empty[st][u], fills.of(j, u) + 1u)) {
              ok = false;
              return;
            }
            const uint32_t has = *const_cast<volatile uint32_t*>(&bars.has[values][rs]);
            const uint32_t raw = base + S::kOffRaw + (values * kChRaw + rs) * S::kRawBytes;
            if (!values) {
#pragma unroll 1
              for (int v = 0; v < 2; ++v) {
                // a token, eight dims of every group; of eight neighbouring lanes four have a token four further on, so that a store of theirs meets all banks
                const int in = 32 * v + cwarp * 8 + (lane >> 3) + (lane & 4), t = lane & 3, g = in >> 4, key = 64 * u + in;
                const uint32_t gran = raw + g * S::kRawGran, to = place(tile, key, t);
                uint32_t w[NA] = {}, par[NA] = {};
                if (key < left && (has >> g & 1u)) {
                  words(gran + (in & 15) * (HD / 2) + t * NA * 4, w);
                  words(gran + 8 * HD + (in & 15) * NA * 4, par);
                }
#pragma unroll
                for (int m = 0; m < NA; ++m) {
                  const __nv_bfloat162 step = pair_of(par[m >> 1], 0, m & 1 ? 0x3232 : 0x1010), low = pair_of(par[NA / 2 + (m >> 1)], 0, m & 1 ? 0x3232 : 0x1010);
                  // nibbles (0, 4), (1, 5), (2, 6), (3, 7)
                  const uint32_t p0 = value(w[m], step, low), p1 = value(w[m] >> 4, step, low), p2 = value(w[m] >> 8, step, low), p3 = value(w[m] >> 12, step, low);
                  store(to, m, __byte_perm(p0, p1, 0x5410), __byte_perm(p2, p3, 0x5410), __byte_perm(p0, p1, 0x7632), __byte_perm(p2, p3, 0x7632));
                }
              }
            } else {
              // two tokens, eight dims of every group; lanes as above
              const int in = 2 * (cwarp * 8 + pair_order(lane >> 2)), q = lane & 3, g = in >> 4, key = 64 * u + in;
              const uint32_t gran = raw + g * S::kRawGran, to0 = place(tile, key, q), to1 = place(tile, key + 1, q);
              uint32_t w0[NA] = {}, w1[NA] = {}, pa[NA] = {}, pb[NA] = {};
              if (key < left && (has >> g & 1u)) {
                words(gran + (in >> 1 & 7) * HD + 2 * q * NA * 4, w0);
                words(gran + (in >> 1 & 7) * HD + (2 * q + 1) * NA * 4, w1);
                words(gran + 8 * HD + (in & 15) * NA * 4, pa);
                if (key + 1 < left) words(gran + 8 * HD + (in & 15) * NA * 4 + NA * 4, pb);
              }
#pragma unroll
              for (int m = 0; m < NA; ++m) {
                // (the first token's beside the second's)
                const uint32_t how = m & 1 ? 0x7632 : 0x5410;
                const __nv_bfloat162 step = pair_of(pa[m >> 1], pb[m >> 1], how), low = pair_of(pa[NA / 2 + (m >> 1)], pb[NA / 2 + (m >> 1)], how);
                uint32_t v[8];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  v[e] = value(w0[m] >> (4 * e), step, low);
                  v[4 + e] = value(w1[m] >> (4 * e), step, low);
                }
                store(to0, m, __byte_perm(v[0], v[1], 0x5410), __byte_perm(v[2], v[3], 0x5410), __byte_perm(v[4], v[5], 0x5410), __byte_perm(v[6], v[7], 0x5410));
                store(to1, m, __byte_perm(v[0], v[1], 0x7632), __byte_perm(v[2], v[3], 0x7632), __byte_perm(v[4], v[5], 0x7632), __byte_perm(v[6], v[7], 0x7632));
              }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              mbar_arrive(values ? &bars.v_full[st][u] : &bars.k_full[st][u]);
              mbar_arrive(&bars.raw_empty[values][rs]);
            }
            if (++rs == kChRaw) {
              rs = 0;
              rphase ^= 1u;
            }
          }
        }
        fills.add(s);
      });
      settle();
    }
  } else if (warp >= 4) {
    // ------------------------------ softmax ------------------------------
    constexpr int kCols = Q4 ? 16 : 32;  // of the sums, at a time
    const int t = (warp - 4) >> 2, quarter = warp & 3, row = quarter * 32 + lane;  // TMEM lanes that this warp may touch
    const int tok = row / a.G, g = row - tok * a.G;
    const uint32_t s_base = tmem_base + (uint32_t(quarter * 32) << 16) + uint32_t(t * 128);
    const uint32_t o_addr = tmem_base + (uint32_t(quarter * 32) << 16) + 256u + uint32_t(t * 128);
    float2* s_sums = reinterpret_cast<float2*>(gen + S::kOffSums);
    uint32_t uses[2] = {0, 0}, pairs = 0, others = 0, joins = 0, products = 0;
    each([&](const ChunkSeg& s, bool two) {
      const int n = s.n, tk = (two ? t * a.T : 0) + tok;  // token of the pair
      const bool valid = tok < a.T && tk < s.ntok;
      const int lim = min(s.lim + tk, s.cap);             // keys [0, lim) are visible
      const bool busy = __any_sync(kAll, valid);
      const int mine = two ? n : (n + 1 - t) >> 1;        // steps of this place
      // halves of steps; the last may be without its second one
      const int halves = 2 * mine - (s.cut && mine > 0 && (two || ((n - 1) & 1) == t) ? 1 : 0);
      float m_used = -INFINITY, l = 0.f;
#pragma unroll 1
      for (int k = 0; k < halves && ok; ++k, ++products) {
        const int j = one_copy(two) ? k >> 1 : (k & ~1) + t, half = k & 1;
        if (!wait_for(&bars.s_ready[t][half], half ? uses[1] : uses[0])) {
          ok = false;
          break;
        }
        half ? ++uses[1] : ++uses[0];
        if (!one_copy(busy)) {  // rows of no token: whatever their probabilities are
          if (lane == 0) mbar_arrive(&bars.p_ready[t][half]);
          continue;
        }
        tc_fence_after_sync();
        const uint32_t s_addr = s_base + uint32_t(kChHalf * half);
        const uint32_t lost = *const_cast<volatile uint32_t*>(&bars.gone[(s.i0 + j) & 7]) >> (kChGrans / 2 * half) & 15u;
        const int seen = lim - (s.j0 + j) * kChKeys - kChHalf * half;  // of these keys
        if (lost || __any_sync(kAll, valid && seen < kChHalf)) {
          // keys that a row does not see, or that no block holds: their scores are written over
#pragma unroll 1
          for (int c0 = 0; c0 < kChHalf; c0 += 16) {
            uint32_t r[16];
            tmem_ld_32x16(s_addr + c0, r);
            tmem_ld_wait();
#pragma unroll
            for (int c = 0; c < 16; ++c)
              if (c0 + c >= seen || (lost >> (c0 / kChGran) & 1u)) r[c] = 0xff800000u;
            tmem_st_32x16(s_addr + c0, r);
          }
          tmem_st_wait();
        }
        // (4-bit cache: 32 scores at a time, read once more for the exponentials: its 640 threads have 96 registers each)
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        uint32_t r0[32], r1[Q4 ? 1 : 32];
        tmem_ld_32x32(s_addr, r0);
        if constexpr (!Q4) {
          tmem_ld_32x32(s_addr + 32, r1);
          tmem_ld_wait();
#pragma unroll
          for (int c = 0; c < 32; c += 4)
#pragma unroll
            for (int e = 0; e < 4; ++e) mx[e] = max3(mx[e], __uint_as_float(r0[c + e]), __uint_as_float(r1[c + e]));
        } else {
#pragma unroll 1
          for (int c0 = 0; c0 < kChHalf; c0 += 32) {
            tmem_ld_wait();
#pragma unroll
            for (int c = 0; c < 32; c += 8)
#pragma unroll
              for (int e = 0; e < 4; ++e) mx[e] = max3(mx[e], __uint_as_float(r0[c + e]), __uint_as_float(r0[c + 4 + e]));
            tmem_ld_32x32(s_addr + (c0 ^ 32), r0);
          }
        }
        const float m_new = fmaxf(m_used, fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * a.scale_log2);
        // also true on the first finite maximum; rows of no token have no say (the warp's others would be rounded as they have it)
        const bool grow = valid && m_new > m_used + kChRescale;
        if (__any_sync(kAll, grow)) {
          const float alpha = (m_new == -INFINITY) ? 1.f : ex2_approx(m_used - m_new);
          if (k > 0) {
            // P V of the half before may still be running.  Parity tells its phase from its neighbours: the one behind needs this warp's own P,
            // and the one before it was issued ahead of these scores.
            // (a warp by itself: one whose wait runs out goes on with its group, and leaves NaN)
            if (!mbar_wait_quick_warp(&bars.pv_done[t], (products - 1) & 1u, abort_at, a.polls)) l = NAN;
            tc_fence_after_sync();
#pragma unroll 1
            for (int c0 = 0; c0 < HD; c0 += 16) {
              uint32_t r[16];
              tmem_ld_32x16(o_addr + c0, r);
              tmem_ld_wait();
#pragma unroll
              for (int c = 0; c < 16; ++c) r[c] = __float_as_uint(__uint_as_float(r[c]) * alpha);
              tmem_st_32x16(o_addr + c0, r);
            }
            tmem_st_wait();
          }
          l *= alpha;
          m_used = m_new;
        }
        const float mref = (m_used == -INFINITY) ? 0.f : m_used;
        const float2 neg = make_float2(-mref, -mref), sl = make_float2(a.scale_log2, a.scale_log2);
        float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        auto weigh = [&](const uint32_t (&r)[32], uint32_t to) {
          uint32_t pk[16];
#pragma unroll
          for (int c = 0; c < 32; c += 2) {
            const float2 u = fma2(make_float2(__uint_as_float(r[c]), __uint_as_float(r[c + 1])), sl, neg);
            const float2 e = !Q4 && (c >> 1) % 4 < kChPoly ? ex2_poly(u) : make_float2(ex2_approx(u.x), ex2_approx(u.y));
            sum[(c >> 1) & 1] = add2(sum[(c >> 1) & 1], e);
            // (P in bf16: the products want it; off by half a step, 2^-8 at most, of every term)
            pk[c >> 1] = pack_bf16x2(e.x, e.y);
          }
          tmem_st_32x16(to, pk);  // over the scores: P of 32 keys takes the columns of 16
        };
        if constexpr (!Q4) {
          weigh(r0, s_addr);
          weigh(r1, s_addr + 16);
        } else {
#pragma unroll 1
          for (int c0 = 0; c0 < kChHalf; c0 += 32) {
            tmem_ld_wait();
            weigh(r0, s_addr + c0 / 2);
            if (c0 == 0) tmem_ld_32x32(s_addr + 32, r0);
          }
        }
        sum[0] = add2(sum[0], sum[1]);
        l += sum[0].x + sum[0].y;
        tmem_st_wait();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.p_ready[t][half]);
      }
      // ---- the pair's rows, or a piece of them ----
      if (mine == 0) return;
      if (ok && !wait_for(&bars.o_final[t], pairs)) ok = false;
      ++pairs;
      const bool join = !two && n > 1;  // the sums of the same rows in two places
      if (join && t == 1) {
        s_sums[row] = make_float2(m_used, ok ? l : NAN);
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.sums);
        return;
      }
      float w0 = 1.f, w1 = 0.f;
      if (join) {
        if (ok && !(wait_for(&bars.sums, joins) && wait_for(&bars.o_final[1], others))) ok = false;
        ++joins;
        const float2 ml = s_sums[row];
        const float m = fmaxf(m_used, ml.x), ref = m == -INFINITY ? 0.f : m;
        w0 = ex2_approx(m_used - ref);
        w1 = ex2_approx(ml.x - ref);
        l = l * w0 + ml.y * w1;
        m_used = m;
      }
      if (t == 0 && (two || join)) ++others;
      const bool whole = s.piece < 0;
      const int at = (two ? t * kChRows : 0) + row;
      const float inv = !whole ? 1.f : l > 0.f ? 1.f / l : l == 0.f ? 0.f : NAN;
      w0 = ok ? w0 * inv : NAN;
      w1 *= inv;
      __nv_bfloat16* orow = a.out + (size_t(s.row + tk) * a.nq + size_t(s.h) * a.G + g) * HD;
      // (pieces: four dims of all rows beside one another, so that a warp's stores are whole lines)
      float4* prow = reinterpret_cast<float4*>(a.part) + size_t(s.piece) * (HD / 4) * a.row_cap + at;
      tc_fence_after_sync();
      if (busy) {
        float2 odd = make_float2(0.f, 0.f);  // NaN from the first number that is none
#pragma unroll 1
        for (int c0 = 0; c0 < HD; c0 += kCols) {
          uint32_t r[kCols / 16][16], q[kCols / 16][16];
#pragma unroll
          for (int d = 0; d < kCols / 16; ++d) tmem_ld_32x16(o_addr + c0 + 16 * d, r[d]);
          if (one_copy(join)) {
#pragma unroll
            for (int d = 0; d < kCols / 16; ++d) tmem_ld_32x16(o_addr + 128u + c0 + 16 * d, q[d]);
          } else {
#pragma unroll
            for (int c = 0; c < kCols; ++c) q[c >> 4][c & 15] = 0;
          }
          tmem_ld_wait();
          float v[kCols];
#pragma unroll
          for (int c = 0; c < kCols; ++c) v[c] = fmaf(__uint_as_float(q[c >> 4][c & 15]), w1, __uint_as_float(r[c >> 4][c & 15]) * w0);
#pragma unroll
          for (int c = 0; c < kCols; c += 2) odd = fma2(make_float2(v[c], v[c + 1]), make_float2(0.f, 0.f), odd);
          if (one_copy(valid && whole)) {
#pragma unroll
            for (int c = 0; c < kCols; c += 8)
              *reinterpret_cast<uint4*>(orow + c0 + c) =
                  make_uint4(pack_bf16x2(v[c], v[c + 1]), pack_bf16x2(v[c + 2], v[c + 3]), pack_bf16x2(v[c + 4], v[c + 5]), pack_bf16x2(v[c + 6], v[c + 7]));
          } else if (one_copy(valid)) {
#pragma unroll
            for (int c = 0; c < kCols; c += 4) prow[size_t((c0 + c) / 4) * a.row_cap] = make_float4(v[c], v[c + 1], v[c + 2], v[c + 3]);
          }
          __syncwarp();
        }
        if (!whole && valid)
          reinterpret_cast<float2*>(a.part + size_t(2 * runs) * a.row_cap * HD)[size_t(s.piece) * a.row_cap + at] = make_float2(m_used, ok ? l : NAN);
        if (whole && valid && odd.x + odd.y != 0.f) a.meta[me].odd = 1;
      }
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&bars.o_free[t]);
        if (join) mbar_arrive(&bars.o_free[1]);
      }
      // (a run that gave up goes on to leave NaN everywhere)
    });
    settle();
  }

  if (*s_abort) __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, kChTmemCols);
  }
  if (threadIdx.x == 0 && *s_abort) *(a.error ? a.error : &g_chunk_err) = 1;
}

// Numbers of one token's key or value as a lane of a warp holds them: dims V lane .. V lane + V - 1, V = HD / 32.
template <int HD>
struct ChunkLane {
  static constexpr int V = HD / 32, NA = HD / kQ4Group;
  static __device__ __forceinline__ void of(const __nv_bfloat16* row, float (&x)[V]) {
    uint32_t w[V / 2];
    if constexpr (V == 4) {
      const uint2 u = *reinterpret_cast<const uint2*>(row + V * (threadIdx.x & 31));
      w[0] = u.x;
      w[1] = u.y;
    } else {
      w[0] = *reinterpret_cast<const uint32_t*>(row + V * (threadIdx.x & 31));
    }
#pragma unroll
    for (int e = 0; e < V; ++e) x[e] = __uint_as_float(e & 1 ? w[e >> 1] & 0xffff0000u : w[e >> 1] << 16);
  }
  // token `r` of a tile of the 4-bit cache
  static __device__ __forceinline__ void of4(const uint8_t* tile, int r, bool value, float (&x)[V]) {
    const int d = V * (threadIdx.x & 31), ga = d / kQ4Group, in = d % kQ4Group;
    const uint8_t* codes = value ? tile + q4_v_codes(HD) + (r >> 1) * HD + ((in >> 2) * NA + ga) * 4 : tile + r * (HD / 2) + ((in >> 3) * NA + ga) * 4;
    const uint32_t w = *reinterpret_cast<const uint32_t*>(codes) >> 4 * (value ? (r & 1) * 4 + (in & 3) : in & 7);
    const __nv_bfloat16* par = reinterpret_cast<const __nv_bfloat16*>(tile + (value ? q4_v_params(HD) : q4_k_params(HD)) + r * NA * 4);
    const float step = __bfloat162float(par[ga]), low = __bfloat162float(par[NA + ga]);
#pragma unroll
    for (int e = 0; e < V; ++e) x[e] = __bfloat162float(__float2bfloat16(fmaf(step, float(w >> (4 * e) & 15u), low)));
  }
};
__device__ __forceinline__ bool chunk_odd(float x) { return !(fabsf(x) < INFINITY); }

// A warp looks at one row (token, query head) of the result.  Dims that hold an infinity or NaN, where a value of the pair's keys that the row does not
// see is one, are computed from the keys that it sees; where one of these is none either, the dim stays as it is.  As plain as can be, as no row of a sound
// cache comes here: 0.2 us a key and row (4-bit cache 0.4).  One NaN behind 2048 tokens on 16383, 40/8x128: 1880 rows, 12 ms (26).
template <int HD, bool Q4>
__device__ __noinline__ void chunk_again(const Chunk& a, int row, int head) {
  using L = ChunkLane<HD>;
  constexpr int V = L::V, kAhead = 8;
  constexpr uint32_t kAll = 0xffffffffu;
  const int lane = threadIdx.x & 31, h = head / a.G;
  __nv_bfloat16* to = a.out + (size_t(row) * a.nq + head) * HD;
  float x[V];
  L::of(to, x);
  uint32_t bad = 0;
#pragma unroll
  for (int e = 0; e < V; ++e) bad |= uint32_t(chunk_odd(x[e])) << e;
  if (!__any_sync(kAll, bad)) return;
  int b = -1;
#pragma unroll 1
  for (int b0 = 0; b0 < a.batch && b < 0; b0 += 32) {
    bool here = false;
    if (b0 + lane < a.batch) {
      const ChunkReq r = chunk_req(a, b0 + lane);
      here = row >= r.q0 && row - r.q0 < r.n;
    }
    const uint32_t found = __ballot_sync(kAll, here);
    if (found) b = b0 + __ffs(found) - 1;
  }
  if (b < 0) return;  // a row of no request: whatever stands there
  const ChunkReq r = chunk_req(a, b);
  const int tok = row - r.q0, tok0 = tok / (2 * a.T) * (2 * a.T);
  const int lim = max(min(r.past + tok + 1, r.cap), 0), keys = chunk_keys(r, tok0, min(2 * a.T, r.n - tok0));
  const int* table = a.tables + size_t(b) * a.max_blocks;
  // token t of the head: the row of the cache, -1: no block has it
  auto look = [&](int t) {
    const int page = t / a.block_size, blk = table[page];
    return blk < 0 || blk >= a.n_blocks ? -1 : (blk * a.nkv + h) * a.block_size + t - page * a.block_size;
  };
  // (-1: of some row, so that loads wait for no branch)
  auto load = [&](int at, bool value, float (&y)[V]) {
    at = max(at, 0);
    if constexpr (Q4)
      L::of4(a.cache4 + size_t(at / kQ4Tokens) * q4_tile_bytes(HD), at % kQ4Tokens, value, y);
    else
      L::of((value ? a.v : a.k) + size_t(at) * HD, y);
  };
  // ---- values that the row does not see ----
  uint32_t hidden = 0;
#pragma unroll 1
  for (int t0 = lim; t0 < keys; t0 += 32) {
    const int mine = t0 + lane < keys ? look(t0 + lane) : -1;
#pragma unroll kAhead
    for (int k = 0; k < 32; ++k) {
      const int at = __shfl_sync(kAll, mine, k);
      float y[V];
      load(at, true, y);
#pragma unroll
      for (int e = 0; e < V; ++e) hidden |= uint32_t(at >= 0 && chunk_odd(y[e])) << e;
    }
  }
  bad &= hidden;
  if (!__any_sync(kAll, bad)) return;
  // ---- the row from what it sees, the last key first ----
  float q[V], acc[V] = {}, m = -INFINITY, l = 0.f;
  L::of(a.q + size_t(row) * a.q_stride + size_t(head) * HD, q);
#pragma unroll 1
  for (int t1 = lim; t1 > 0; t1 -= 32) {
    const int mine = t1 - 1 - lane >= 0 ? look(t1 - 1 - lane) : -1;
#pragma unroll 1
    for (int k0 = 0; k0 < 32; k0 += kAhead) {
      float s[kAhead], y[kAhead][V], v[kAhead][V], top = m;
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int at = __shfl_sync(kAll, mine, k0 + k);
        load(at, false, y[k]);
        load(at, true, v[k]);
      }
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const bool there = __shfl_sync(kAll, mine, k0 + k) >= 0;
        s[k] = 0.f;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          s[k] = fmaf(q[e], y[k][e], s[k]);
          v[k][e] = there ? v[k][e] : 0.f;
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) s[k] += __shfl_xor_sync(kAll, s[k], o);
        s[k] = there ? s[k] * a.scale_log2 : -INFINITY;
        top = fmaxf(top, s[k]);
      }
      const float ref = top == -INFINITY ? 0.f : top, alpha = ex2_approx(m - ref);
      m = top;
      l *= alpha;
#pragma unroll
      for (int e = 0; e < V; ++e) acc[e] *= alpha;
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const float p = ex2_approx(s[k] - ref);
        l += p;
#pragma unroll
        for (int e = 0; e < V; ++e) acc[e] = fmaf(p, v[k][e], acc[e]);
      }
    }
    // dims of which the row sees a value that is none
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (chunk_odd(acc[e])) bad &= ~(1u << e);
    if (!__any_sync(kAll, bad)) return;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int e = 0; e < V; ++e)
    if (bad >> e & 1u) to[V * lane + e] = __float2bfloat16(acc[e] * inv);
}

// Pieces of a pair that was cut: block (run where it begins, 32 rows), a lane a row, a warp HD / 8 of its dims.
constexpr int kChMergeWarps = 8, kChMergeAhead = 4;  // pieces that are asked for at once
template <int HD>
__global__ void __launch_bounds__(kChMergeWarps * 32, 2) k_chunk_merge(const __grid_constant__ Chunk a) {
  constexpr int V = HD / 4 / kChMergeWarps;  // vectors of four dims
  pdl_launch_dependents();
  pdl_wait();
  const int me = blockIdx.x, runs = gridDim.x, warp = threadIdx.x >> 5;
  const ChunkMeta m = a.meta[me];
  const int r = blockIdx.y * 32 + (threadIdx.x & 31), tok = r / a.G, g = r - tok * a.G;
  // (every run leaves its words; lengths that another stream changes meanwhile, which nobody may, could leave some that fit nothing)
  int odd = m.odd;  // 1: rows that the run's first kernel wrote, 2: rows joined here
  const bool cut = m.count > 0 && m.count <= runs - me && m.ntok <= 2 * a.T;
  if (cut && tok < m.ntok) {
    const int at = (tok >= a.T ? kChRows + (tok - a.T) * a.G : tok * a.G) + g;
    const float2* sums = reinterpret_cast<const float2*>(a.part + size_t(2 * runs) * a.row_cap * HD) + at;
    const float4* part = reinterpret_cast<const float4*>(a.part) + size_t(warp * V) * a.row_cap + at;
    float M = -INFINITY, L = 0.f;
    float4 acc[V];
#pragma unroll
    for (int d = 0; d < V; ++d) acc[d] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
    for (int k = 0; k < m.count; k += kChMergeAhead) {
      float2 ml[kChMergeAhead];
      float4 v[kChMergeAhead][V];
#pragma unroll
      for (int e = 0; e < kChMergeAhead; ++e) {
        ml[e] = make_float2(-INFINITY, 0.f);
#pragma unroll
        for (int d = 0; d < V; ++d) v[e][d] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (k + e < m.count) {
          const size_t p = size_t(k + e == 0 ? m.first : 2 * (me + k + e)) * a.row_cap;
          ml[e] = sums[p];
#pragma unroll
          for (int d = 0; d < V; ++d) v[e][d] = part[p * (HD / 4) + size_t(d) * a.row_cap];
        }
      }
#pragma unroll
      for (int e = 0; e < kChMergeAhead; ++e) {
        const float n = fmaxf(M, ml[e].x), ref = n == -INFINITY ? 0.f : n, s0 = ex2_approx(M - ref), s1 = ex2_approx(ml[e].x - ref);
        M = n;
        L = L * s0 + ml[e].y * s1;
#pragma unroll
        for (int d = 0; d < V; ++d) {
          acc[d].x = acc[d].x * s0 + v[e][d].x * s1;
          acc[d].y = acc[d].y * s0 + v[e][d].y * s1;
          acc[d].z = acc[d].z * s0 + v[e][d].z * s1;
          acc[d].w = acc[d].w * s0 + v[e][d].w * s1;
        }
      }
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
    __nv_bfloat16* to = a.out + (size_t(m.row + tok) * a.nq + size_t(m.h) * a.G + g) * HD + 4 * V * warp;
#pragma unroll
    for (int d = 0; d < V; d += 2)
      *reinterpret_cast<uint4*>(to + 4 * d) = make_uint4(pack_bf16x2(acc[d].x * inv, acc[d].y * inv), pack_bf16x2(acc[d].z * inv, acc[d].w * inv),
                                                         pack_bf16x2(acc[d + 1].x * inv, acc[d + 1].y * inv), pack_bf16x2(acc[d + 1].z * inv, acc[d + 1].w * inv));
#pragma unroll
    for (int d = 0; d < V; ++d)
      if (chunk_odd(acc[d].x * inv) || chunk_odd(acc[d].y * inv) || chunk_odd(acc[d].z * inv) || chunk_odd(acc[d].w * inv)) odd |= 2;
  }
  // ---- numbers that are none ----
  auto again = [&](int row, int head) {
    if (a.cache4)
      chunk_again<HD, true>(a, row, head);
    else
      chunk_again<HD, false>(a, row, head);
  };
  if (!__syncthreads_or(odd) || !a.again) return;
  if (__syncthreads_or(odd & 2)) {
#pragma unroll 1
    for (int i = warp; i < 32; i += kChMergeWarps) {
      const int rr = blockIdx.y * 32 + i, t = rr / a.G;
      if (t < m.ntok) again(m.row + t, m.h * a.G + rr - t * a.G);
    }
  }
  if (odd & 1) {
    // all rows, shared out among the runs that have some
    int many = 0, mine = 0;
#pragma unroll 1
    for (int i = 0; i < runs; ++i) {
      const int has = a.meta[i].odd != 0;
      many += has;
      mine += i < me && has;
    }
    const int64_t rows = int64_t(a.tokens) * a.nq;
#pragma unroll 1
    for (int64_t i = (int64_t(mine) * gridDim.y + blockIdx.y) * kChMergeWarps + warp; i < rows; i += int64_t(many) * gridDim.y * kChMergeWarps) {
      const int row = int(i / a.nq), head = int(i - int64_t(row) * a.nq);
      // (pairs that were cut are their own blocks')
      bool other = false;
#pragma unroll 1
      for (int k = threadIdx.x & 31; k < runs; k += 32) {
        const ChunkMeta c = a.meta[k];
        other |= c.count > 0 && row >= c.row && row - c.row < c.ntok && head / a.G == c.h;
      }
      if (!__any_sync(0xffffffffu, other)) again(row, head);
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
  return bl_paged_attn_chunk_say(q, q_stride, k_cache, v_cache, cache4, block_tables, cu_q, ctx_lens, out, tokens, batch, nq, nkv, hd, block_size, n_blocks,
                                 max_blocks, scale, ws, ws_bytes, nullptr, stream, err, errlen);
}

extern "C" int bl_paged_attn_chunk_say(const void* q, int q_stride, const void* k_cache, const void* v_cache, const void* cache4,
                                       const int* block_tables, const int* cu_q, const int* ctx_lens, void* out, int tokens, int batch, int nq,
                                       int nkv, int hd, int block_size, int n_blocks, int max_blocks, float scale, void* ws, size_t ws_bytes,
                                       unsigned* error, void* stream, char* err, size_t errlen) {
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
  {
    const int64_t pairs = tokens / (2 * chunk_tile_tokens(nq / nkv)) + int64_t(batch), steps = int64_t(max_blocks) * block_size / kChKeys + 1 + chunk_over(true);
    if (pairs * nkv > 0x7fffffffLL / steps - sm_count()) return refuse("has too many tokens for its tables: steps of 128 keys, over all tiles and KV heads, must fit 31 bits");
  }
  if (q_stride % 8 || q_stride < 0 || (tokens > 1 && q_stride < int64_t(nq) * hd)) return refuse("needs rows of q on 16-byte boundaries that hold nq heads");
  if (!q || (cache4 ? k_cache || v_cache : !k_cache || !v_cache) || (!block_tables && max_blocks) || !cu_q || !ctx_lens || !out)
    return refuse("needs queries, one kind of cache, block tables, row offsets, context lengths and an output");
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache) | reinterpret_cast<uintptr_t>(cache4) |
       reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(ws)) & 15)
    return refuse("needs tensors on 16-byte boundaries");
  if (!(scale > 0.f) || scale > 3e38f) return refuse("needs a positive scale");
  if (reinterpret_cast<uintptr_t>(error) & 3) return refuse("needs an error word on its own boundary");
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
  a.error = error;
  a.q = static_cast<const __nv_bfloat16*>(q);
  a.k = static_cast<const __nv_bfloat16*>(k_cache);
  a.v = static_cast<const __nv_bfloat16*>(v_cache);
  a.q_stride = size_t(tokens > 1 ? q_stride : 0);
  {
    // (where the result takes the queries' place, none are left to compute anything with)
    const uintptr_t q0 = reinterpret_cast<uintptr_t>(q), o0 = reinterpret_cast<uintptr_t>(out);
    const uintptr_t q1 = q0 + (size_t(tokens - 1) * a.q_stride + size_t(nq) * hd) * 2, o1 = o0 + size_t(tokens) * nq * hd * 2;
    a.again = q1 <= o0 || o1 <= q0;
  }
  a.tokens = tokens; a.batch = batch; a.nq = nq; a.nkv = nkv; a.block_size = block_size; a.n_blocks = n_blocks; a.max_blocks = max_blocks;
  a.box = block_size % 64 == 0 ? 64 : block_size % 32 == 0 ? 32 : 16;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.polls = std::min(g_chunk_polls.load(), 1u << 27);  // (a poll of the warps that look all the time is 16 looks)
  auto divide_by = [](uint32_t d) {
    ChunkDiv r = {0, 0};
    while ((uint64_t(1) << r.s) < d) ++r.s;
    r.m = uint32_t(((uint64_t(1) << (31 + r.s)) + d - 1) / d);
    return r;
  };
  a.by_runs = divide_by(runs);
  a.by_block = divide_by(block_size);
  a.by_pair = divide_by(2 * a.T);

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
    if (e == cudaSuccess) e = launch_k(merge, dim3(runs, (a.row_cap + 31) / 32), dim3(kChMergeWarps * 32), 0, st, a);
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
