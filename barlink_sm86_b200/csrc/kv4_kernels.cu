// SPDX-License-Identifier: MIT
//
// The key/value cache in 4 bits (layout: kv4.cuh): writer, reader, and attention of one query token per request.
//
// A group of 32 dims of a token's key (after RoPE) or value, both rounded to bf16, is held as low = its least
// element (exact in bf16), step = bf16((greatest - low) / 15) and codes rint((x - low) / step).  A group whose range
// is no finite number is held as step 0, low NaN: it reads as NaN and leaves the other groups alone.
#include <math.h>
#include <stdio.h>

#include <atomic>

#include "bl_ops.h"
#include "heap.h"
#include "kv4.cuh"
#include "launch.h"
#include "ptx.cuh"

namespace bl {

#define KV4_LAUNCH_CHECK(what)                                                             \
  do {                                                                                     \
    cudaError_t _e = cudaGetLastError();                                                   \
    if (_e != cudaSuccess) {                                                               \
      set_err(err, errlen, "barlink: %s launch failed: %s", what, cudaGetErrorString(_e)); \
      return -1;                                                                           \
    }                                                                                      \
  } while (0)

// ---------------------------------------------------------------------------
// RoPE and the write into the cache
// ---------------------------------------------------------------------------
struct Q4Write {
  const __nv_bfloat16* qkv;  // rows of width (nq + 2 nkv) * hd, or null:
  const float* slabs;        // k-split slabs of the QKV linear, `slab` floats apart
  int nsplit;
  size_t slab;
  const __nv_bfloat16* bias;
  __nv_bfloat16* out;  // rotated rows (may be qkv)
  const int* positions;
  const int* slots;
  uint8_t* cache;
  int rows, nq, nkv, hd, block_size, n_blocks;
  double log2_theta;
};

// eight elements of a row from column `col`: the bf16 buffer (as it lies), or the slabs added in split order, then the bias,
// rounded to bf16 (as k_rope_kv_write does)
template <bool SLABS>
__device__ __forceinline__ uint4 q4_load8(const Q4Write& a, size_t row, int width, int col) {
  if constexpr (!SLABS) {
    return *reinterpret_cast<const uint4*>(a.qkv + row * width + col);
  } else {
    const float* p = a.slabs + row * width + col;
    float f[8] = {};
    for (int s0 = 0; s0 < a.nsplit; s0 += 4) {  // (four on their way at a time, added in order)
      float4 u[4], w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (s0 + i < a.nsplit) {
          u[i] = __ldcg(reinterpret_cast<const float4*>(p + (s0 + i) * a.slab));
          w[i] = __ldcg(reinterpret_cast<const float4*>(p + (s0 + i) * a.slab) + 1);
        }
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (s0 + i < a.nsplit) {
          f[0] += u[i].x; f[1] += u[i].y; f[2] += u[i].z; f[3] += u[i].w;
          f[4] += w[i].x; f[5] += w[i].y; f[6] += w[i].z; f[7] += w[i].w;
        }
    }
    if (a.bias) {
      const uint4 b = *reinterpret_cast<const uint4*>(a.bias + col);
      const uint32_t w[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 v = unpack_bf16x2(w[j]);
        f[2 * j] += v.x;
        f[2 * j + 1] += v.y;
      }
    }
    return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
  }
}
__device__ __forceinline__ void q4_unpack8(const uint4& v, float (&f)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    f[2 * j] = __uint_as_float(w[j] << 16);
    f[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
  }
}

// Eight of a group's 32 elements (bf16, as they lie), the rest with the other lanes of the quad -> codes (nibble e = element e), and
// the group's step and low as bf16 bits.  Least and greatest are taken in pairs, the least as the greatest of the negatives, so that
// one exchange carries both; a NaN or infinity comes out as a step that is no finite number.  The codes are those of the formula to the
// bit: a product with 1 / 15 or 1 / step is within 10^-5 of the quotient (or a few units in the last place of a step), and where
// that could round otherwise it is divided.
__device__ __forceinline__ uint32_t q4_quantise8(const uint4& raw, uint16_t& step_bits, uint16_t& low_bits) {
  auto h = [](uint32_t v) { return *reinterpret_cast<const __nv_bfloat162*>(&v); };
  auto u = [](__nv_bfloat162 v) { return *reinterpret_cast<const uint32_t*>(&v); };
  const uint32_t hi2 = u(__hmax2_nan(__hmax2_nan(h(raw.x), h(raw.y)), __hmax2_nan(h(raw.z), h(raw.w))));
  const uint32_t lo2 = u(__hmin2_nan(__hmin2_nan(h(raw.x), h(raw.y)), __hmin2_nan(h(raw.z), h(raw.w)))) ^ 0x80008000u;
  uint32_t m = u(__hmax2_nan(h(__byte_perm(lo2, hi2, 0x5410)), h(__byte_perm(lo2, hi2, 0x7632))));  // (-low, greatest)
  m = u(__hmax2_nan(h(m), h(__shfl_xor_sync(0xffffffffu, m, 1))));
  m = u(__hmax2_nan(h(m), h(__shfl_xor_sync(0xffffffffu, m, 2))));
  const float lo = -__uint_as_float(m << 16), range = __uint_as_float(m & 0xffff0000u) - lo;
  float q = range * (1.f / 15.f);
  if ((__float_as_uint(q) & 0xffffu) - 0x7ff8u < 16u) q = __fdiv_rn(range, 15.f);  // near the middle of two bf16 numbers
  const __nv_bfloat16 st = __float2bfloat16(q);
  const float step = __bfloat162float(st);
  const bool fine = isfinite(step);
  uint32_t w = 0;
  if (fine && step > 0.f) {
    float x[8];
    q4_unpack8(raw, x);
    const float inv = __fdividef(1.f, step);
    bool near = step < 1e-30f;  // (1 / step must be a finite number)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float v = (x[e] - lo) * inv, r = v + 12582912.f;  // 3 * 2^22: the sum's last bits are the rounded quotient
      near |= fabsf(v - (r - 12582912.f)) > 0.49999f;
      w |= (__float_as_uint(r) & 15u) << (4 * e);  // (at most 15: a step is no more than 2^-8 below a fifteenth of the range)
    }
    if (near) {
      w = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) w |= uint32_t(fminf(rintf(__fdiv_rn(x[e] - lo, step)), 15.f)) << (4 * e);
    }
  }
  step_bits = fine ? __bfloat16_as_ushort(st) : 0;
  low_bits = fine ? uint16_t((m & 0xffffu) ^ 0x8000u) : 0x7fc0;
  return w;
}

// One octet of a key (group a, lane t of the quad) or value into its token's tile.
__device__ __forceinline__ void q4_store8(uint8_t* tile, int r, int hd, bool value, int a, int t, uint32_t w, uint16_t step,
                                          uint16_t low) {
  const int na = hd / kQ4Group;
  if (!value) {
    *reinterpret_cast<uint32_t*>(tile + r * (hd / 2) + (t * na + a) * 4) = w;
  } else {
    uint8_t* p = tile + q4_v_codes(hd) + (r >> 1) * hd + (r & 1) * 2;
    *reinterpret_cast<uint16_t*>(p + ((2 * t) * na + a) * 4) = uint16_t(w);
    *reinterpret_cast<uint16_t*>(p + ((2 * t + 1) * na + a) * 4) = uint16_t(w >> 16);
  }
  if (t == 0) {
    uint16_t* q = reinterpret_cast<uint16_t*>(tile + (value ? q4_v_params(hd) : q4_k_params(hd)) + r * na * 4);
    q[a] = step;
    q[na + a] = low;
  }
}

// A block takes ROWS neighbouring rows, or, one row at a time, the blocks of grid.y share its heads; PER = THREADS / ROWS threads to a
// row.  A thread keeps one octet of the heads' lower halves and its rotation partner, and goes through the heads, BATCH of them
// requested at a time.  The angles of the block's rows are computed once, in 64 bits (a position of 10^5 leaves 32 bits no better than 0.01 radians), and the products are
// rounded one by one: the rotated elements are the formula's to the bit.
template <int HD, bool SLABS, int ROWS, int THREADS, int BATCH>
__global__ void __launch_bounds__(THREADS, ROWS > 1 ? 1024 / THREADS : 1) k_rope_kv_write_q4(const Q4Write a) {
  constexpr int HALF = HD / 2, OPH = HD / 16, PER = THREADS / ROWS, STEP = PER / OPH;  // octets of half a head; heads of a pass
  pdl_launch_dependents();
  pdl_wait();
  __shared__ __align__(16) float2 s_rot[ROWS][HALF];
  const int row0 = blockIdx.x * ROWS, rows = min(ROWS, a.rows - row0), heads = a.nq + 2 * a.nkv, width = heads * HD;
  {
    // (THREADS is a multiple of HALF: a thread has the same pair in every row that it visits)
    const int i = threadIdx.x % HALF;
    const double inv = exp2(-a.log2_theta * (double(2 * i) / HD)) * 0.15915494309189533577;
    for (int r = threadIdx.x / HALF; r < rows; r += THREADS / HALF) {
      const double turn = double(a.positions[row0 + r]) * inv;
      double sn, cs;
      sincospi(2.0 * (turn - rint(turn)), &sn, &cs);
      s_rot[r][i] = make_float2(float(cs), float(sn));
    }
  }
  const int r = threadIdx.x / PER, o = threadIdx.x % OPH, h0 = threadIdx.x % PER / OPH + (ROWS == 1 ? blockIdx.y * STEP : 0);
  const int all = ROWS == 1 ? gridDim.y * STEP : STEP;  // heads of a pass, over the blocks of a row
  const bool row_there = r < rows;  // (whole warps: PER is a multiple of 32)
  const size_t row = row0 + (row_there ? r : 0);
  const int slot = a.slots ? a.slots[row] : -1;
  __syncthreads();
  if (!row_there) return;
  const int blk = slot >= 0 ? slot / a.block_size : -1, in_block = slot >= 0 ? slot - blk * a.block_size : 0;
  const bool kept = blk >= 0 && blk < a.n_blocks;  // (no such block: not kept)
  for (int pass = 0; pass < heads; pass += all * BATCH) {
    const int hb = h0 + pass;
    uint4 lo[BATCH], hi[BATCH];
#pragma unroll
    for (int c = 0; c < BATCH; ++c) {
      const int h = hb + c * all;
      lo[c] = hi[c] = make_uint4(0, 0, 0, 0);
      if (h < heads) {
        lo[c] = q4_load8<SLABS>(a, row, width, h * HD + 8 * o);
        hi[c] = q4_load8<SLABS>(a, row, width, h * HD + 8 * o + HALF);
      }
    }
#pragma unroll
    for (int c = 0; c < BATCH; ++c) {
      const int h = hb + c * all;
      const bool there = h < heads;
      if (!__any_sync(0xffffffffu, there)) break;
      if (there && h < a.nq + a.nkv) {
        float x[8], y[8];
        q4_unpack8(lo[c], x);
        q4_unpack8(hi[c], y);
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
          const float4 cs = *reinterpret_cast<const float4*>(&s_rot[r][8 * o + j]);
          const float p0 = __fsub_rn(__fmul_rn(x[j], cs.x), __fmul_rn(y[j], cs.y)), q0 = __fadd_rn(__fmul_rn(y[j], cs.x), __fmul_rn(x[j], cs.y));
          const float p1 = __fsub_rn(__fmul_rn(x[j + 1], cs.z), __fmul_rn(y[j + 1], cs.w)),
                      q1 = __fadd_rn(__fmul_rn(y[j + 1], cs.z), __fmul_rn(x[j + 1], cs.w));
          (&lo[c].x)[j / 2] = pack_bf16x2(p0, p1);
          (&hi[c].x)[j / 2] = pack_bf16x2(q0, q1);
        }
      }
      if (there) {
        __nv_bfloat16* p = a.out + row * width + h * HD + 8 * o;
        *reinterpret_cast<uint4*>(p) = lo[c];
        *reinterpret_cast<uint4*>(p + HALF) = hi[c];
      }
      const bool keep = there && h >= a.nq && kept;
      if (!__any_sync(0xffffffffu, keep)) continue;
      uint16_t s0, l0, s1, l1;
      const uint32_t w0 = q4_quantise8(lo[c], s0, l0), w1 = q4_quantise8(hi[c], s1, l1);
      if (keep) {
        const bool value = h >= a.nq + a.nkv;
        uint8_t* tile = a.cache + q4_tile_offset(blk, in_block, h - a.nq - (value ? a.nkv : 0), a.nkv, a.block_size, HD);
        const int tr = in_block % kQ4Tokens;
        q4_store8(tile, tr, HD, value, o >> 2, o & 3, w0, s0, l0);
        q4_store8(tile, tr, HD, value, (o + OPH) >> 2, o & 3, w1, s1, l1);
      }
    }
  }
}

// Rows of the cache back as bf16 (zeros where a slot names none).  One octet of a key and of a value per thread; a block takes as many
// rows as it has threads for, so that the numbers that are divided are small (with 64-bit ones: 8.7 us for 8191 rows of 4 heads).
template <int HD>
__global__ void __launch_bounds__(256) k_kv4_read(const uint8_t* __restrict__ cache, const int* __restrict__ slots, __nv_bfloat16* __restrict__ k,
                                                  __nv_bfloat16* __restrict__ v, int rows, int block_rows, int nkv, int block_size, int n_blocks) {
  constexpr int OH = HD / 8, NA = HD / kQ4Group;
  pdl_launch_dependents();
  pdl_wait();
  const int row0 = blockIdx.x * block_rows, per = nkv * OH, count = min(block_rows, rows - row0) * per;
  for (int u = threadIdx.x; u < count; u += 256) {
    const int r0 = u / per, e = u - r0 * per, h = e / OH, o = e % OH, ga = o >> 2, t = o & 3;
    const int slot = slots[row0 + r0], blk = slot / block_size;
    uint4 ko = make_uint4(0, 0, 0, 0), vo = ko;
    if (slot >= 0 && blk < n_blocks) {
      const int in_block = slot - blk * block_size, r = in_block % kQ4Tokens;
      const uint8_t* tile = cache + q4_tile_offset(blk, in_block, h, nkv, block_size, HD);
      const uint32_t kw = *reinterpret_cast<const uint32_t*>(tile + r * (HD / 2) + (t * NA + ga) * 4);
      const uint8_t* vp = tile + q4_v_codes(HD) + (r >> 1) * HD + (r & 1) * 2;
      const uint32_t vw = *reinterpret_cast<const uint16_t*>(vp + ((2 * t) * NA + ga) * 4) |
                          uint32_t(*reinterpret_cast<const uint16_t*>(vp + ((2 * t + 1) * NA + ga) * 4)) << 16;
      const __nv_bfloat16* kp = reinterpret_cast<const __nv_bfloat16*>(tile + q4_k_params(HD) + r * NA * 4);
      const __nv_bfloat16* vq = reinterpret_cast<const __nv_bfloat16*>(tile + q4_v_params(HD) + r * NA * 4);
      const float ks = __bfloat162float(kp[ga]), kl = __bfloat162float(kp[NA + ga]);
      const float vs = __bfloat162float(vq[ga]), vl = __bfloat162float(vq[NA + ga]);
      uint32_t kk[4], vv[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        kk[j] = pack_bf16x2(kl + ks * float((kw >> (8 * j)) & 15), kl + ks * float((kw >> (8 * j + 4)) & 15));
        vv[j] = pack_bf16x2(vl + vs * float((vw >> (8 * j)) & 15), vl + vs * float((vw >> (8 * j + 4)) & 15));
      }
      ko = make_uint4(kk[0], kk[1], kk[2], kk[3]);
      vo = make_uint4(vv[0], vv[1], vv[2], vv[3]);
    }
    const size_t at = (size_t(row0) * per + u) * 8;
    *reinterpret_cast<uint4*>(k + at) = ko;
    *reinterpret_cast<uint4*>(v + at) = vo;
  }
}

// ---------------------------------------------------------------------------
// attention
// ---------------------------------------------------------------------------
// S = Q K^T and O = P V by mma.sync with the tokens (S) and the dims (O) on the 16-row side and up to eight query heads on the
// 8-column side, so that a group of 4 to 8 heads wastes little of a product; the codes come from shared memory in the order in
// which a lane needs them and become fp16 operands by one mask each: the 16 bits 0x000c are the subnormal number c * 2^-24,
// 0x00c0 is 16 c * 2^-24, and the powers of two are taken out of Q and of the result.  step and low never touch the codes:
//   s_t = sum over groups a of step_ta (sum q c) + low_ta (sum q)     -- one accumulator per group; the second sum is a product
//                                                                        of k = (parts of sum q) x groups in bf16, exact parts
//   o_d = sum over tokens of (p_t step_ta) c + p_t low_ta             -- p step rounded to fp16 (2^-11), the second sum in fp32
// Queries go in as fp16 of a power of two per head (exact: 2^-27 of the head's largest element is still whole).  The reference of
// the running softmax is the greatest of x_t + e_t, e_t = log2 of the token's largest step, so that p step stays within fp16 whatever the
// values' size, or of its largest |low| over 2^95, if that is more: a group of one value has no step, and p low has to stay within
// fp32.  It moves only when p step exceeds it by 2^8, when a lane's four tokens have next to no steps and lows that matter there, or when there
// is a low of 2^65 or more, which one vote per unit finds out.  Between the votes p is at most 2^29 where a token has less than 2^65, so
// that p low is below 2^97 and its sums are finite, whatever the context's length.  (What that costs: beside a low above 2^95, groups with steps below
// 2^-14 of low / 2^95 lose places.)
//
// Work: the units (two tiles) of all (request, KV head) pairs in one row, cut into equal runs, one for each warp; a warp has a
// ring of its own that the bulk copies fill across pairs, and shares nothing with others.  Lengths are on the GPU only, so every warp
// adds them up by itself.  Pairs that were cut are joined by k_q4_merge.  (A cluster of blocks for each pair, joined through distributed
// shared memory without a second kernel: one request of 333 tokens 5.9 us and 6.0 so, 64 of up to 1100 16.8 and 13.7.)
constexpr int kQ4MaxG = 16;
constexpr int kQ4Warps = 4;
constexpr float kQ4None = -3.402823466e38f;  // reference before the first token

// (whole 16-byte vectors)
__host__ __device__ constexpr size_t q4_part_floats(int G, int hd) { return size_t(G) * hd + (2 * G + 3) / 4 * 4; }

// set by a wait that ran out; one word per device
__device__ uint32_t g_kv4_err;
// polls of a wait for copies before it gives up
constexpr uint32_t kQ4Polls = 1u << 24;
static std::atomic<uint32_t> g_kv4_polls{kQ4Polls};

struct Q4Attn {
  const __nv_bfloat16* q;
  const uint8_t* cache;
  const int* tables;
  const int* ctx_lens;
  __nv_bfloat16* out;
  float* part;   // [2 * runs]: a run's first piece of a pair and its last; G * hd sums, G times (reference, sum of p)
  int2* meta;    // [batch * nkv]: a pair's first piece, and the number of its pieces (0: done); the others are the first of their runs
  int q_stride, batch, nq, nkv, block_size, n_blocks, max_blocks;
  float scale_log2;
  uint32_t polls;
};

__device__ __forceinline__ float q4_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void q4_mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// (the same with nothing to add to)
__device__ __forceinline__ void q4_mma_f16_0(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void q4_mma_bf16_0(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ uint32_t q4_transpose(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
template <int N>
__device__ __forceinline__ void lds_words(uint32_t addr, uint32_t (&w)[N]) {
  if constexpr (N == 4)
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(addr));
  else if constexpr (N == 2)
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(addr));
  else
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[0]) : "r"(addr));
}
__device__ __forceinline__ float bf16_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// Where a flat unit index stands: its pair begins at `start` and has `units`.
constexpr int kQ4Unit = 2 * kQ4Tokens;
struct Q4At {
  int b, h, start, units;
};
__device__ __forceinline__ int q4_context(const Q4Attn& a, int b) { return min(max(a.ctx_lens[b], 0), a.max_blocks * a.block_size); }
__device__ __forceinline__ int q4_units(const Q4Attn& a, int b) { return (q4_context(a, b) + kQ4Unit - 1) / kQ4Unit; }
__device__ __forceinline__ void q4_advance(const Q4Attn& a, Q4At& p, int idx) {
  while (idx >= p.start + p.units && p.b < a.batch) {
    p.start += p.units;
    if (++p.h == a.nkv) {
      p.h = 0;
      do {
        ++p.b;
      } while (p.b < a.batch && (p.units = q4_units(a, p.b)) == 0);
    }
  }
}

// The tensor core cuts its sums off, toward 0, and they grow with every unit while a mean over many tokens is small: 4.2 million tokens,
// 111 units a warp, were off by 1.0e-3 of the result's norm beside its rounding.  So they are put aside every kQ4Aside units, and
// added there by rounded additions: over n units of a pair in one run they lose at most n / 32 times 2^-24 of what was added in absolute
// value.  The sums of p and of p low are rounded additions all the way, two a unit: at most 2 n times 2^-24, which reaches the result's own
// rounding, 2^-9, with n = 16384, half a million tokens of a request for one warp (a request alone has 1184 of them).
constexpr int kQ4Aside = 32;

template <int HD, int NT, int STAGES>
constexpr int q4_smem_bytes() {
  return kQ4Warps * (STAGES * (2 * q4_tile_bytes(HD) + 8) + NT * HD * 8 * 4);
}

template <int HD, int NT, int STAGES>
__global__ void __launch_bounds__(kQ4Warps * 32, 2) k_paged_attn_q4(const Q4Attn a) {
  constexpr int NA = HD / kQ4Group, TB = q4_tile_bytes(HD);
  constexpr uint32_t kAll = 0xffffffffu;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ uint32_t s_abort[kQ4Warps];
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kQ4Warps * STAGES * 2 * TB) + warp * STAGES;
  const uint32_t ring = smem_u32(smem) + warp * STAGES * 2 * TB;
  // [NT * 2 NA * 4][lane]
  float* aside = reinterpret_cast<float*>(smem + kQ4Warps * STAGES * (2 * TB + 8)) + warp * (NT * HD * 8) + lane;
  if (lane == 0) {
#pragma unroll
    for (int i = 0; i < STAGES; ++i) mbar_init(bars + i, 1);
    mbar_fence_init();
    s_abort[warp] = 0;
  }
  __syncwarp();
  pdl_wait();

  // ---- this warp's run of units: [lo, hi) of all pairs' units (neighbouring runs on different SMs) ---------------
  const int G = a.nq / a.nkv, me = warp * gridDim.x + blockIdx.x, runs = gridDim.x * kQ4Warps;
  int lo, hi, run;
  Q4At seg;
  {
    const int per = (a.batch + 31) / 32, b0 = min(lane * per, a.batch), b1 = min(b0 + per, a.batch);
    int mine = 0;
    for (int b = b0; b < b1; ++b) mine += q4_units(a, b);
    mine *= a.nkv;
    int upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(kAll, upto, o);
      if (lane >= o) upto += u;
    }
    const int total = __shfl_sync(kAll, upto, 31);
    run = (total + runs - 1) / runs;
    lo = int(min(int64_t(me) * run, int64_t(total)));
    hi = min(lo + run, total);
    int b = b0, at = upto - mine, n = 0;
    const bool holds = at <= lo && lo < upto;  // one lane's requests hold the first unit
    if (holds)
      for (n = q4_units(a, b) * a.nkv; lo >= at + n; n = q4_units(a, ++b) * a.nkv) at += n;
    const uint32_t who = __ballot_sync(kAll, holds);
    const int src = who ? __ffs(who) - 1 : 0;
    seg.b = __shfl_sync(kAll, b, src);
    at = __shfl_sync(kAll, at, src);
    seg.units = max(__shfl_sync(kAll, n, src) / a.nkv, 1);
    seg.h = (lo - at) / seg.units;
    seg.start = at + seg.h * seg.units;
  }
  // requests without tokens
  for (int b = me; b < a.batch; b += runs)
    if (q4_units(a, b) == 0) {
      for (int i = lane; i < a.nq * HD / 8; i += 32) reinterpret_cast<uint4*>(a.out + size_t(b) * a.nq * HD)[i] = make_uint4(0, 0, 0, 0);
      for (int h = lane; h < a.nkv; h += 32) a.meta[size_t(b) * a.nkv + h] = make_int2(0, 0);
    }
  if (lo >= hi) return;

  // ---- copies: lane l knows where tile l of the next 16 units lies, and asks for it when its turn comes ------------
  const int count = hi - lo;
  Q4At ahead = seg;
  const uint8_t* from = nullptr;
  uint32_t have = 0;  // bit l: that tile has a block
  uint32_t gone = 0;  // bits 2 s, 2 s + 1: the tiles of stage s have none
  const uint32_t leader = elect_leader();
  auto issue = [&](int i, int stage) {  // (units in turn)
    if ((i & 15) == 0) {
      const int idx = lo + i + (lane >> 1);
      int tile = -1;
      if (idx < hi) {
        q4_advance(a, ahead, idx);
        const int tok = (idx - ahead.start) * kQ4Unit + (lane & 1) * kQ4Tokens;
        if (tok < q4_context(a, ahead.b)) {
          const int page = tok / a.block_size, blk = a.tables[size_t(ahead.b) * a.max_blocks + page];
          if (blk >= 0 && blk < a.n_blocks)
            tile = (blk * a.nkv + ahead.h) * (a.block_size / kQ4Tokens) + (tok - page * a.block_size) / kQ4Tokens;
        }
      }
      from = a.cache + size_t(max(tile, 0)) * TB;
      have = __ballot_sync(kAll, tile >= 0);
    }
    const uint32_t has = have >> (2 * (i & 15)) & 3u;
    if (has != 3 || gone) gone = (gone & ~(3u << (2 * stage))) | (has ^ 3u) << (2 * stage);
    mbar_expect_tx_warp(leader, bars + stage, TB * ((has & 1) + (has >> 1)));
    const uint32_t mine = (lane >> 1) == (i & 15) && (have >> lane & 1);
    bulk_load_warp(mine, ring + (stage * 2 + (lane & 1)) * TB, from, TB, smem_u32(bars + stage), kHintEvictFirst);
  };
  // (the queries first: behind the copies they would wait for what may be the whole cache)
  uint4 raw[NT][NA];
  auto ask_queries = [&](const Q4At& seg) {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int ga = 0; ga < NA; ++ga)
        raw[n][ga] = 8 * n + g < G ? *reinterpret_cast<const uint4*>(a.q + size_t(seg.b) * a.q_stride + (size_t(seg.h) * G + 8 * n + g) * HD + 32 * ga + 8 * t)
                                   : make_uint4(0, 0, 0, 0);
  };
  ask_queries(seg);
#pragma unroll 1
  for (int i = 0; i < STAGES; ++i)
    if (i < count) issue(i, i);

  int k = 0, stage = 0;  // unit of the run, its stage
  uint32_t phase = 0;
  bool dead = false;
  while (k < count && !dead) {
    const int seg_end = min(hi, seg.start + seg.units) - lo;
    const bool begins = lo + k == seg.start, whole = begins && lo + seg_end == seg.start + seg.units;
    const int piece = 2 * me + (k == 0 ? 0 : 1);
    const int ctx = q4_context(a, seg.b);
    // ---- queries of this pair: operands, factor, sums --------------------------------------------
    uint32_t qb[NT][NA][4], qs[NT][2];
    float f[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      uint32_t top = 0;  // the largest element's bits: magnitudes of bf16 compare as integers
#pragma unroll
      for (int ga = 0; ga < NA; ++ga)
        top = __vmaxu2(top, __vmaxu2(__vmaxu2(raw[n][ga].x & 0x7fff7fffu, raw[n][ga].y & 0x7fff7fffu), __vmaxu2(raw[n][ga].z & 0x7fff7fffu, raw[n][ga].w & 0x7fff7fffu)));
      top = max(top & 0xffffu, top >> 16);
      top = max(top, __shfl_xor_sync(kAll, top, 1));
      top = max(top, __shfl_xor_sync(kAll, top, 2));
      const int ex = min(max(int(top >> 7) - 127, -100), 127);
      const float up = __uint_as_float(uint32_t(14 - ex + 127) << 23);  // the largest element comes to 2^14 .. 2^15
      float sum[NA];
#pragma unroll
      for (int ga = 0; ga < NA; ++ga) {
        const float e0 = bf16_lo(raw[n][ga].x) * up, e1 = bf16_hi(raw[n][ga].x) * up, e2 = bf16_lo(raw[n][ga].y) * up, e3 = bf16_hi(raw[n][ga].y) * up,
                    e4 = bf16_lo(raw[n][ga].z) * up, e5 = bf16_hi(raw[n][ga].z) * up, e6 = bf16_lo(raw[n][ga].w) * up, e7 = bf16_hi(raw[n][ga].w) * up;
        qb[n][ga][0] = pack_f16x2(e0, e4);
        qb[n][ga][1] = pack_f16x2(e1 * 0.0625f, e5 * 0.0625f);
        qb[n][ga][2] = pack_f16x2(e2, e6);
        qb[n][ga][3] = pack_f16x2(e3 * 0.0625f, e7 * 0.0625f);
        float v = ((e0 + e1) + (e2 + e3)) + ((e4 + e5) + (e6 + e7));
        v += __shfl_xor_sync(kAll, v, 1);
        v += __shfl_xor_sync(kAll, v, 2);
        sum[ga] = v * 5.9604644775390625e-8f;  // 2^-24, as the codes have it
      }
      // three bf16 parts of every sum, along k = part * NA + group
      const int part0 = NA == 4 ? t >> 1 : t;
      float first[2], second[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float v = NA == 4 && (t & 1) ? sum[2 * (NA / 4) + j] : sum[j];
        const float p0 = __bfloat162float(__float2bfloat16(v)), p1 = __bfloat162float(__float2bfloat16(v - p0)), p2 = v - p0 - p1;
        first[j] = part0 == 0 ? p0 : part0 == 1 ? p1 : part0 == 2 ? p2 : 0.f;
        second[j] = NA == 4 && part0 == 0 ? p2 : 0.f;
      }
      qs[n][0] = pack_bf16x2(first[0], first[1]);
      qs[n][1] = pack_bf16x2(second[0], second[1]);
      // 2^24 * 2^(ex - 14); never 0, for it meets the infinity that stands for "behind the last token"
      const float fac = fmaxf(__uint_as_float(uint32_t(min(ex + 10, 127) + 127) << 23) * a.scale_log2, 1.17549435e-38f);
      f[n][0] = __shfl_sync(kAll, fac, 8 * t);
      f[n][1] = __shfl_sync(kAll, fac, 8 * t + 4);
    }
    // the next pair's queries, where there are registers for them: behind this pair's copies they take long
    constexpr bool AHEAD = NT == 1;
    Q4At next = seg;
    if (AHEAD && seg_end < count) {
      q4_advance(a, next, lo + seg_end);
      ask_queries(next);
    }
    float o[NT][2 * NA][4], vm[NT][NA][2], R[NT][2], l[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int i = 0; i < 2 * NA; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f;
#pragma unroll
      for (int i = 0; i < NA; ++i) vm[n][i][0] = vm[n][i][1] = 0.f;
      R[n][0] = R[n][1] = kQ4None;
      l[n][0] = l[n][1] = 0.f;
    }

    int fresh = 0;         // units in o
    bool put = false;      // sums stand aside
    auto each_sum = [&](auto&& f) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 2 * NA; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) f(o[n][i][j], aside[((n * 2 * NA + i) * 4 + j) * 32]);
    };
#pragma unroll 1
    for (; k < seg_end; ++k) {
      if (!mbar_wait_bounded_warp(bars + stage, phase, &s_abort[warp], a.polls)) {
        dead = true;
        break;
      }
      const uint32_t tile = ring + stage * 2 * TB;
      const int left = ctx - (lo + k - seg.start) * kQ4Unit;  // tokens of this unit

      // ---- scores, over the factor f: tokens g (c[.][.][0], [1]) and g + 8 of either tile, heads 2 t and 2 t + 1 ----
      // (the asm statements keep their order: products that wait for one another stand four apart)
      float c[2][NT][4];
      {
        uint32_t w0[2][NA], w1[2][NA], sl0[2][NA], sl1[2][NA];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          lds_words<NA>(tile + u * TB + q4_k_params(HD) + g * NA * 4, sl0[u]);  // step[NA], low[NA]
          lds_words<NA>(tile + u * TB + q4_k_params(HD) + (g + 8) * NA * 4, sl1[u]);
          lds_words<NA>(tile + u * TB + g * (HD / 2) + t * NA * 4, w0[u]);
          lds_words<NA>(tile + u * TB + (g + 8) * (HD / 2) + t * NA * 4, w1[u]);
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const uint32_t m0 = NA == 4 && (t & 1) ? sl0[u][NA - 1] : sl0[u][NA / 2], m1 = NA == 4 && (t & 1) ? sl1[u][NA - 1] : sl1[u][NA / 2];
#pragma unroll
          for (int n = 0; n < NT; ++n) q4_mma_bf16_0(c[u][n], m0, m1, m0, m1, qs[n][0], qs[n][1]);
        }
#pragma unroll
        for (int gp = 0; gp < NA; gp += 2) {
          float d[2][2][NT][4];
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
              for (int n = 0; n < NT; ++n)
                q4_mma_f16_0(d[i][u][n], w0[u][gp + i] & 0x000f000fu, w1[u][gp + i] & 0x000f000fu, w0[u][gp + i] & 0x00f000f0u, w1[u][gp + i] & 0x00f000f0u,
                             qb[n][gp + i][0], qb[n][gp + i][1]);
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              const uint32_t v0 = w0[u][gp + i] >> 8, v1 = w1[u][gp + i] >> 8;
#pragma unroll
              for (int n = 0; n < NT; ++n)
                q4_mma_f16(d[i][u][n], v0 & 0x000f000fu, v1 & 0x000f000fu, v0 & 0x00f000f0u, v1 & 0x00f000f0u, qb[n][gp + i][2], qb[n][gp + i][3]);
            }
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              const float s0 = i ? bf16_hi(sl0[u][gp >> 1]) : bf16_lo(sl0[u][gp >> 1]), s1 = i ? bf16_hi(sl1[u][gp >> 1]) : bf16_lo(sl1[u][gp >> 1]);
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                c[u][n][0] += s0 * d[i][u][n][0];
                c[u][n][1] += s0 * d[i][u][n][1];
                c[u][n][2] += s1 * d[i][u][n][2];
                c[u][n][3] += s1 * d[i][u][n][3];
              }
            }
        }
      }
      uint32_t vs0[2][NA], vs1[2][NA];  // step[NA], low[NA] of the values of tokens g and g + 8
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        lds_words<NA>(tile + u * TB + q4_v_params(HD) + g * NA * 4, vs0[u]);
        lds_words<NA>(tile + u * TB + q4_v_params(HD) + (g + 8) * NA * 4, vs1[u]);
      }
      const uint32_t no_block = gone >> (2 * stage) & 3u;
      if (left < kQ4Unit || no_block) {
        // behind the last token, and where there is no block: whatever stands there (NaN too) stays out
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int j = 0; j < 2; ++j)
            if (16 * u + 8 * j + g >= left || (no_block >> u & 1)) {
#pragma unroll
              for (int n = 0; n < NT; ++n) c[u][n][2 * j] = c[u][n][2 * j + 1] = -INFINITY;
#pragma unroll
              for (int i = 0; i < NA; ++i) (j ? vs1[u] : vs0[u])[i] = 0;
            }
      }
      // ---- probabilities; where one times step may leave fp16's range, a new reference first ----
      float steps, top;  // the largest of the steps here (bf16 above 0 compare as integers); the same, or 2^39 where it does not bound p low
      {
        uint32_t m = 0;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int i = 0; i < NA / 2; ++i) m = __vmaxu2(m, __vmaxu2(vs0[u][i], vs1[u][i]));
        steps = fmaxf(bf16_lo(m), bf16_hi(m));
        top = steps < 9.5367431640625e-7f ? 549755813888.f : steps;  // (2^-20: p up to 2^-30 passes, tokens that are not there among them)
      }
      const uint32_t lows = tile + (lane >> 4) * TB + q4_v_params(HD) + (lane & 15) * NA * 4 + NA * 2;  // of token `lane` of the unit
      uint32_t vast;  // one of 2^65 or more is among them: the two highest bits of its exponent
      {
        uint32_t w[NA / 2];
        lds_words<NA / 2>(lows, w);
        vast = w[0] & w[0] << 1;
        if constexpr (NA == 4) vast |= w[1] & w[1] << 1;
        vast &= lane < left && !(no_block >> (lane >> 4) & 1) ? 0x40004000u : 0u;
      }
      float p[2][NT][4];
      auto weigh = [&] {
        float most = 0.f;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              p[u][n][j] = q4_ex2(fmaf(c[u][n][j], f[n][j & 1], -R[n][j & 1]));
              most += p[u][n][j];  // (no less than the greatest; NaN if one of them is)
            }
        return most;
      };
      const float most = weigh();
      // (NaN too: it is of one head, and would hide what the lane's others ask for)
      bool move = __any_sync(kAll, !(most * top <= 512.f) || vast);
      if (move && !__any_sync(kAll, !(most * fmaxf(steps, 6.4623485355705287e-27f) <= 512.f))) {
        // next to no steps, and p at most 2^96: lows below 2^-2 (zeros, most of all) need no other reference
        uint32_t w[NA / 2], large = 0;
        lds_words<NA / 2>(lows, w);
#pragma unroll
        for (int i = 0; i < NA / 2; ++i) large |= __vcmpgeu2(w[i] & 0x7fff7fffu, 0x3e803e80u);
        move = __any_sync(kAll, large && lane < left && !(no_block >> (lane >> 4) & 1));
      }
      if (move) {
        float e[2][2];  // log2 of a token's largest step, rounded down, or that of its largest low less 95
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            uint32_t m = (j ? vs1[u] : vs0[u])[0];
            if constexpr (NA == 4) m = __vmaxu2(m, (j ? vs1[u] : vs0[u])[1]);
            e[u][j] = float(min(max(int(max(m & 0xffffu, m >> 16) >> 7) - 127, -90), 110));
          }
        if (__any_sync(kAll, vast || (top >= 549755813888.f && !(most <= 0.f)))) {
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              uint32_t m = 0;
#pragma unroll
              for (int i = NA / 2; i < NA; ++i) {
                const uint32_t low = (j ? vs1[u] : vs0[u])[i] & 0x7fff7fffu;
                m = __vmaxu2(m, low & __vcmpleu2(low, 0x7f7f7f7fu));  // (a group that is no number bounds nothing)
              }
              e[u][j] = fmaxf(e[u][j], float(int(max(m & 0xffffu, m >> 16) >> 7) - 127 - 95));
            }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float z = fmaxf(fmaxf(fmaf(c[0][n][j], f[n][j], e[0][0]), fmaf(c[0][n][2 + j], f[n][j], e[0][1])),
                            fmaxf(fmaf(c[1][n][j], f[n][j], e[1][0]), fmaf(c[1][n][2 + j], f[n][j], e[1][1])));
            z = fmaxf(z, __shfl_xor_sync(kAll, z, 4));
            z = fmaxf(z, __shfl_xor_sync(kAll, z, 8));
            z = fmaxf(fmaxf(z, __shfl_xor_sync(kAll, z, 16)), R[n][j]);
            const float al = q4_ex2(R[n][j] - z);
            R[n][j] = z;
            l[n][j] *= al;
#pragma unroll
            for (int i = 0; i < NA; ++i) vm[n][i][j] *= al;
#pragma unroll
            for (int i = 0; i < 2 * NA; ++i) {
              o[n][i][j] *= al;
              o[n][i][2 + j] *= al;
            }
            if (put) {
#pragma unroll
              for (int i = 0; i < 2 * NA; ++i) {
                aside[((n * 2 * NA + i) * 4 + j) * 32] *= al;
                aside[((n * 2 * NA + i) * 4 + 2 + j) * 32] *= al;
              }
            }
          }
        weigh();
      }
      // ---- values: p times step as the columns' operand, p times low beside it.  The rows g of a product take a byte's lower code, the
      // rows g + 8 the two together, lower + 16 upper: one instruction less for a word, and the difference is taken at the end (of the
      // two sums and not of the lower code's: what the tensor core cuts off its sums would come out sixteen times as large) ----
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        uint32_t w0[NA], w1[NA], pb[NT][NA][2];
        lds_words<NA>(tile + u * TB + q4_v_codes(HD) + t * HD + g * NA * 4, w0);
        lds_words<NA>(tile + u * TB + q4_v_codes(HD) + (t + 4) * HD + g * NA * 4, w1);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const float* q = p[u][n];
          l[n][0] += q[0] + q[2];
          l[n][1] += q[1] + q[3];
#pragma unroll
          for (int ga = 0; ga < NA; ++ga) {
            const float s0 = ga & 1 ? bf16_hi(vs0[u][ga >> 1]) : bf16_lo(vs0[u][ga >> 1]), s1 = ga & 1 ? bf16_hi(vs1[u][ga >> 1]) : bf16_lo(vs1[u][ga >> 1]);
            const uint32_t lw0 = vs0[u][NA / 2 + (ga >> 1)], lw1 = vs1[u][NA / 2 + (ga >> 1)];
            const float m0 = ga & 1 ? bf16_hi(lw0) : bf16_lo(lw0), m1 = ga & 1 ? bf16_hi(lw1) : bf16_lo(lw1);
            pb[n][ga][0] = q4_transpose(pack_f16x2(q[0] * s0, q[1] * s0));
            pb[n][ga][1] = q4_transpose(pack_f16x2(q[2] * s1, q[3] * s1));
            vm[n][ga][0] = fmaf(q[0], m0, fmaf(q[2], m1, vm[n][ga][0]));
            vm[n][ga][1] = fmaf(q[1], m0, fmaf(q[3], m1, vm[n][ga][1]));
          }
        }
#pragma unroll
        for (int ga = 0; ga < NA; ++ga) {
          const uint32_t v0 = __byte_perm(w0[ga], 0, 0x4341), v1 = __byte_perm(w1[ga], 0, 0x4341);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            q4_mma_f16(o[n][2 * ga], w0[ga] & 0x000f000fu, w0[ga] & 0x00ff00ffu, w1[ga] & 0x000f000fu, w1[ga] & 0x00ff00ffu, pb[n][ga][0], pb[n][ga][1]);
            q4_mma_f16(o[n][2 * ga + 1], v0 & 0x000f000fu, v0, v1 & 0x000f000fu, v1, pb[n][ga][0], pb[n][ga][1]);
          }
        }
      }
      if (++fresh == kQ4Aside) {
        each_sum([&](float& sum, float& there) {
          there = put ? there + sum : sum;
          sum = 0.f;
        });
        fresh = 0;
        put = true;
      }
      __syncwarp();  // all lanes have read the stage that the next copies fill
      if (k + STAGES < count) issue(k + STAGES, stage);
      if (++stage == STAGES) {
        stage = 0;
        phase ^= 1;
      }
    }
    if (dead) break;

    if (put) each_sum([&](float& sum, float& there) { sum += there; });
    // ---- out: the whole pair, or a piece of it ---------------------------------------------------------
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) {
          l[n][j] += __shfl_xor_sync(kAll, l[n][j], d);
#pragma unroll
          for (int i = 0; i < NA; ++i) vm[n][i][j] += __shfl_xor_sync(kAll, vm[n][i][j], d);
        }
        const int head = 8 * n + 2 * t + j;
        if (head >= G) continue;
        const float inv = !whole ? 1.f : l[n][j] == 0.f ? 0.f : 1.f / l[n][j];
        float* part = a.part + size_t(piece) * q4_part_floats(G, HD);
#pragma unroll
        for (int i = 0; i < NA; ++i) {  // 2^24, and the 16 of the odd dims
          const float *o0 = o[n][2 * i], *o1 = o[n][2 * i + 1], add = vm[n][i][j];
          const float v0 = fmaf(o0[j], 16777216.f, add) * inv, v1 = fmaf(o0[2 + j] - o0[j], 1048576.f, add) * inv,
                      v2 = fmaf(o1[j], 16777216.f, add) * inv, v3 = fmaf(o1[2 + j] - o1[j], 1048576.f, add) * inv;
          const int d = 4 * (8 * i + g);
          if (whole)
            *reinterpret_cast<uint2*>(a.out + (size_t(seg.b) * a.nq + size_t(seg.h) * G + head) * HD + d) =
                make_uint2(pack_bf16x2(v0, v1), pack_bf16x2(v2, v3));
          else
            *reinterpret_cast<float4*>(part + head * HD + d) = make_float4(v0, v1, v2, v3);
        }
        if (!whole && g == 0) *reinterpret_cast<float2*>(part + G * HD + 2 * head) = make_float2(R[n][j], l[n][j]);
      }
    if (begins && lane == 0)
      a.meta[size_t(seg.b) * a.nkv + seg.h] = make_int2(piece, whole ? 0 : (seg.start + seg.units - 1) / run - me + 1);
    if constexpr (AHEAD) {
      seg = next;
    } else if (k < count) {
      q4_advance(a, seg, lo + k);
      ask_queries(seg);
    }
  }
  if (dead) {
    // A copy did not arrive in time: say so, wait for all that are in flight (each as long as a wait may take: shared memory is another
    // block's behind this one), and leave NaN in place of this pair's result and of all that follow in this run.
    if (lane == 0) g_kv4_err = 1;
    for (int i = k; i < min(k + STAGES, count); ++i) {
      __syncwarp();
      if (lane == 0) s_abort[warp] = 0;
      __syncwarp();
      mbar_wait_bounded_warp(bars + stage, phase, &s_abort[warp]);
      if (++stage == STAGES) {
        stage = 0;
        phase ^= 1;
      }
    }
    for (;;) {
      const int seg_end = min(hi, seg.start + seg.units) - lo, piece = 2 * me + (seg.start > lo ? 1 : 0);
      const bool begins = seg.start >= lo, whole = begins && lo + seg_end == seg.start + seg.units;
      if (whole) {
        uint4* to = reinterpret_cast<uint4*>(a.out + (size_t(seg.b) * a.nq + size_t(seg.h) * G) * HD);
        for (int i = lane; i < G * HD / 8; i += 32) to[i] = make_uint4(0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu);
      } else {
        float* part = a.part + size_t(piece) * q4_part_floats(G, HD);
        for (int i = lane; i < G * HD; i += 32) part[i] = 0.f;
        for (int i = lane; i < G; i += 32) *reinterpret_cast<float2*>(part + G * HD + 2 * i) = make_float2(0.f, NAN);
      }
      if (begins && lane == 0) a.meta[size_t(seg.b) * a.nkv + seg.h] = make_int2(piece, whole ? 0 : (seg.start + seg.units - 1) / run - me + 1);
      if (seg_end >= count) break;
      q4_advance(a, seg, lo + seg_end);
    }
  }
}

// The pieces of a pair that was cut: block (pair, head), a warp takes every kQ4MergeWarps-th piece, a lane HD / 32 dims of it.
constexpr int kQ4MergeWarps = 8;
template <int HD>
__global__ void __launch_bounds__(kQ4MergeWarps * 32) k_q4_merge(const Q4Attn a, int G, int runs) {
  constexpr int D = HD / 32;
  pdl_launch_dependents();
  pdl_wait();
  __shared__ float s_o[kQ4MergeWarps][HD], s_m[kQ4MergeWarps], s_l[kQ4MergeWarps];
  const int2 m = a.meta[blockIdx.x];
  if (m.y == 0) return;
  // (every run leaves its words; lengths that another stream changes meanwhile, which nobody may, could leave some out: nothing there is followed)
  if (m.y < 0 || m.x < 0 || m.x >= 2 * runs || m.y > runs - (m.x >> 1)) return;
  const int head = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const size_t pitch = q4_part_floats(G, HD);
  auto at = [&](int i) { return a.part + size_t(i == 0 ? m.x : 2 * ((m.x >> 1) + i)) * pitch; };
  float M = kQ4None, L = 0.f, acc[D];
#pragma unroll
  for (int j = 0; j < D; ++j) acc[j] = 0.f;
#pragma unroll 4
  for (int i = warp; i < m.y; i += kQ4MergeWarps) {
    const float* p = at(i);
    const float2 rl = *reinterpret_cast<const float2*>(p + G * HD + 2 * head);
    float v[D];
    if constexpr (D == 4) {
      const float4 u = *reinterpret_cast<const float4*>(p + head * HD + 4 * lane);
      v[0] = u.x; v[1] = u.y; v[2] = u.z; v[3] = u.w;
    } else {
      const float2 u = *reinterpret_cast<const float2*>(p + head * HD + 2 * lane);
      v[0] = u.x; v[1] = u.y;
    }
    const float n = fmaxf(M, rl.x), s0 = q4_ex2(M - n), s1 = q4_ex2(rl.x - n);
    M = n;
    L = L * s0 + rl.y * s1;
#pragma unroll
    for (int j = 0; j < D; ++j) acc[j] = acc[j] * s0 + v[j] * s1;
  }
#pragma unroll
  for (int j = 0; j < D; ++j) s_o[warp][D * lane + j] = acc[j];
  if (lane == 0) {
    s_m[warp] = M;
    s_l[warp] = L;
  }
  __syncthreads();
  const int d = threadIdx.x;
  if (d >= HD) return;
  M = kQ4None;
#pragma unroll
  for (int w = 0; w < kQ4MergeWarps; ++w) M = fmaxf(M, s_m[w]);
  L = 0.f;
  float o = 0.f;
#pragma unroll
  for (int w = 0; w < kQ4MergeWarps; ++w) {
    const float sc = q4_ex2(s_m[w] - M);
    L += s_l[w] * sc;
    o += s_o[w][d] * sc;
  }
  a.out[(size_t(blockIdx.x) * G + head) * HD + d] = __float2bfloat16(L == 0.f ? 0.f : o / L);
}

}  // namespace bl

using namespace bl;

static int q4_shape(const char* what, int hd, int nkv, int block_size, int n_blocks, char* err, size_t errlen) {
  if ((hd != 64 && hd != 128) || block_size < kQ4Tokens || block_size % kQ4Tokens) {
    set_err(err, errlen, "barlink: %s is built for head_dim 64 and 128 and block sizes that are multiples of %d", what, kQ4Tokens);
    return -1;
  }
  if (n_blocks < 0 || int64_t(n_blocks) * block_size > 0x7fffffffLL || int64_t(n_blocks) * (block_size / kQ4Tokens) * nkv > 0x7fffffffLL) {
    set_err(err, errlen, "barlink: %s: the cache's slots and tiles must fit 32 bits", what);
    return -1;
  }
  return 0;
}

extern "C" size_t bl_kv4_tile_bytes(int hd) { return q4_tile_bytes(hd); }

extern "C" int bl_rope_kv_write_q4(const void* qkv, const void* slabs, int nsplit, size_t slab, const void* bias, void* out,
                                   const int* positions, const int* slots, void* cache, int rows, int nq, int nkv, int hd,
                                   int block_size, int n_blocks, double theta, void* stream, char* err, size_t errlen) {
  if (q4_shape("the 4-bit cache", hd, nkv, block_size, n_blocks, err, errlen)) return -1;
  if (rows < 0 || nq < 0 || nkv < 1 || (!qkv && (!slabs || nsplit < 1)) || !out || !positions || (slots && !cache) || !(theta > 0)) {
    set_err(err, errlen, "barlink: rope_kv_write_q4 needs the QKV rows or slabs, positions, an output and, with slots, a cache");
    return -1;
  }
  if (((reinterpret_cast<uintptr_t>(qkv) | reinterpret_cast<uintptr_t>(slabs) | reinterpret_cast<uintptr_t>(bias) |
        reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(cache)) & 15) || (slab & 3)) {
    set_err(err, errlen, "barlink: rope_kv_write_q4 needs tensors on 16-byte boundaries");
    return -1;
  }
  if (rows == 0) return 0;
  Q4Write a;
  a.qkv = static_cast<const __nv_bfloat16*>(qkv);
  a.slabs = qkv ? nullptr : static_cast<const float*>(slabs);
  a.nsplit = nsplit;
  a.slab = slab;
  a.bias = static_cast<const __nv_bfloat16*>(bias);
  a.out = static_cast<__nv_bfloat16*>(out);
  a.positions = positions;
  a.slots = slots;
  a.cache = static_cast<uint8_t*>(cache);
  a.rows = rows; a.nq = nq; a.nkv = nkv; a.hd = hd; a.block_size = block_size; a.n_blocks = n_blocks;
  a.log2_theta = log2(theta);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  // Many rows: four to a block, a warp each that goes through the heads (8191 rows of 36 heads: 35 us; two warps a row and three heads at
  // a time 37 to 48, by registers); few rows (a decode step) and slabs: a row's heads dealt out to blocks, each thread with one octet.
  // us, a row and four to a block: 36 heads of 128, 592 rows 5.9 and 7.1, 2000 rows 13.4 and 17.4, 3200 19.6 and 18.7, 4000 24.1 and 18.9; 56
  // heads, 2000 rows 18.2 and 26.7, 3200 29.8 and 29.4; 12 heads of 64, 900 rows 3.8 and 4.3, 1200 5.3 and 4.4.
  const bool many = rows > (hd == 128 ? 22 : 7) * sm_count() && !a.slabs;
  const int heads = nq + 2 * nkv, step = 128 / (hd / 16);
  const dim3 grid(many ? (rows + 3) / 4 : rows, many ? 1 : (heads + step - 1) / step), block(128);
  if (hd == 128) {
    if (a.slabs) launch_k(k_rope_kv_write_q4<128, true, 1, 128, 1>, grid, block, 0, st, a);
    else launch_k(many ? k_rope_kv_write_q4<128, false, 4, 128, 2> : k_rope_kv_write_q4<128, false, 1, 128, 1>, grid, block, 0, st, a);
  } else {
    if (a.slabs) launch_k(k_rope_kv_write_q4<64, true, 1, 128, 1>, grid, block, 0, st, a);
    else launch_k(many ? k_rope_kv_write_q4<64, false, 4, 128, 2> : k_rope_kv_write_q4<64, false, 1, 128, 1>, grid, block, 0, st, a);
  }
  KV4_LAUNCH_CHECK("rope_kv_write_q4");
  return 0;
}

extern "C" int bl_kv4_read(const void* cache, const int* slots, void* k, void* v, int rows, int nkv, int hd, int block_size,
                           int n_blocks, void* stream, char* err, size_t errlen) {
  if (q4_shape("the 4-bit cache", hd, nkv, block_size, n_blocks, err, errlen)) return -1;
  if (rows < 0 || rows > 1 << 30 || nkv < 1 || nkv > 1 << 20) {
    set_err(err, errlen, "barlink: kv4_read: rows and KV heads out of range");
    return -1;
  }
  if (rows == 0) return 0;
  if ((!cache && n_blocks) || !slots || !k || !v || ((reinterpret_cast<uintptr_t>(cache) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15)) {
    set_err(err, errlen, "barlink: kv4_read needs slots, and a cache and outputs on 16-byte boundaries");
    return -1;
  }
  const int per = nkv * (hd / 8), block_rows = per >= 256 ? 1 : 256 / per;
  launch_k(hd == 64 ? k_kv4_read<64> : k_kv4_read<128>, dim3((rows + block_rows - 1) / block_rows), dim3(256), 0, static_cast<cudaStream_t>(stream),
           static_cast<const uint8_t*>(cache), slots, static_cast<__nv_bfloat16*>(k), static_cast<__nv_bfloat16*>(v), rows, block_rows, nkv,
           block_size, n_blocks);
  KV4_LAUNCH_CHECK("kv4_read");
  return 0;
}

static int q4_error_rc(cudaError_t e, char* err, size_t errlen) {
  if (e != cudaSuccess) set_err(err, errlen, "barlink: kv4_error: %s", cudaGetErrorString(e));
  return e == cudaSuccess ? 0 : -1;
}
extern "C" int bl_kv4_error(unsigned* out, char* err, size_t errlen) {
  return q4_error_rc(cudaMemcpyFromSymbol(out, g_kv4_err, sizeof(*out)), err, errlen);
}
extern "C" int bl_kv4_error_async(unsigned* out, void* stream, char* err, size_t errlen) {
  return q4_error_rc(cudaMemcpyFromSymbolAsync(out, g_kv4_err, sizeof(*out), 0, cudaMemcpyDeviceToHost, static_cast<cudaStream_t>(stream)), err, errlen);
}
extern "C" int bl_kv4_error_clear(char* err, size_t errlen) {
  const unsigned none = 0;
  return q4_error_rc(cudaMemcpyToSymbol(g_kv4_err, &none, sizeof(none)), err, errlen);
}
extern "C" unsigned bl_kv4_wait_polls(unsigned polls) { return g_kv4_polls.exchange(polls); }

// Blocks of attention.  Two to an SM, with registers for two tiles at once: three and four of fewer registers (the last with spills) took
// 34.5 and 37.9 us where two take 32.7 (4 requests of up to 32767 tokens), 14.9 and 17.0 against 13.7 (64 of up to 1100).
static int q4_grid() { return sm_count() * 2; }

extern "C" size_t bl_paged_attn_decode_q4_ws(int batch, int nq, int nkv, int hd) {
  if (batch < 1 || nkv < 1 || nq < 1) return 0;
  const int G = nq / nkv;
  return 2 * size_t(q4_grid()) * kQ4Warps * q4_part_floats(G, hd) * sizeof(float) + size_t(batch) * nkv * sizeof(int2);
}

extern "C" int bl_paged_attn_decode_q4(const void* q, int q_stride, const void* cache, const int* block_tables, const int* ctx_lens,
                                       void* out, int batch, int nq, int nkv, int hd, int block_size, int n_blocks, int max_blocks,
                                       float scale, void* ws, size_t ws_bytes, void* stream, char* err, size_t errlen) {
  if (q4_shape("attention over the 4-bit cache", hd, nkv, block_size, n_blocks, err, errlen)) return -1;
  if (nkv < 1 || nq < 1 || nq % nkv || nq / nkv > kQ4MaxG) {
    set_err(err, errlen, "barlink: attention over the 4-bit cache needs nq %% nkv == 0 and at most %d query heads per KV head", kQ4MaxG);
    return -1;
  }
  if (batch < 0) {
    set_err(err, errlen, "barlink: attention over the 4-bit cache: a negative batch");
    return -1;
  }
  // (runs are counted in 32 bits, one of them beyond the last tile)
  if (int64_t(max_blocks) * block_size > 0x7fffffffLL - 16 || int64_t(max_blocks) * (block_size / kQ4Tokens) * batch * nkv > 0x3fffffffLL) {
    set_err(err, errlen, "barlink: attention over the 4-bit cache: the tables' tokens, times KV heads, must not exceed 2^34");
    return -1;
  }
  if (batch == 0) return 0;
  if (max_blocks < 1) {
    set_err(err, errlen, "barlink: attention over the 4-bit cache needs a table");
    return -1;
  }
  if (!q || (!cache && n_blocks) || !block_tables || !ctx_lens || !out) {
    set_err(err, errlen, "barlink: attention over the 4-bit cache needs queries, a cache, block tables, context lengths and an output");
    return -1;
  }
  if (((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(cache) | reinterpret_cast<uintptr_t>(out) |
        reinterpret_cast<uintptr_t>(ws)) & 15) || q_stride % 8) {
    set_err(err, errlen, "barlink: attention over the 4-bit cache needs tensors and rows on 16-byte boundaries");
    return -1;
  }
  if (!(scale > 0.f) || scale > 3e38f) {
    set_err(err, errlen, "barlink: attention over the 4-bit cache needs a positive scale");
    return -1;
  }
  const int G = nq / nkv, nt = G > 8 ? 2 : 1, grid = q4_grid();
  if (!ws || ws_bytes < bl_paged_attn_decode_q4_ws(batch, nq, nkv, hd)) {
    set_err(err, errlen, "barlink: attention over the 4-bit cache needs %zu bytes of workspace",
            bl_paged_attn_decode_q4_ws(batch, nq, nkv, hd));
    return -1;
  }
  Q4Attn a;
  a.q = static_cast<const __nv_bfloat16*>(q);
  a.cache = static_cast<const uint8_t*>(cache);
  a.tables = block_tables;
  a.ctx_lens = ctx_lens;
  a.out = static_cast<__nv_bfloat16*>(out);
  a.part = static_cast<float*>(ws);
  a.meta = reinterpret_cast<int2*>(a.part + 2 * size_t(grid) * kQ4Warps * q4_part_floats(G, hd));
  a.q_stride = q_stride; a.batch = batch; a.nq = nq; a.nkv = nkv; a.block_size = block_size; a.n_blocks = n_blocks;
  a.max_blocks = max_blocks;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.polls = g_kv4_polls.load();
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  static bool attr[4][64] = {};
  auto go = [&](auto* kernel, auto* merge, int smem, bool (&done)[64]) {
    const cudaError_t e = allow_smem(reinterpret_cast<const void*>(kernel), smem, done);
    if (e != cudaSuccess) return e;
    launch_k(kernel, dim3(grid), dim3(kQ4Warps * 32), smem, st, a);
    return launch_k(merge, dim3(batch * nkv, G), dim3(kQ4MergeWarps * 32), 0, st, a, G, grid * kQ4Warps);
  };
  cudaError_t e;
  if (hd == 128)
    e = nt == 1 ? go(k_paged_attn_q4<128, 1, 4>, k_q4_merge<128>, q4_smem_bytes<128, 1, 4>(), attr[0])
                : go(k_paged_attn_q4<128, 2, 3>, k_q4_merge<128>, q4_smem_bytes<128, 2, 3>(), attr[1]);
  else
    e = nt == 1 ? go(k_paged_attn_q4<64, 1, 4>, k_q4_merge<64>, q4_smem_bytes<64, 1, 4>(), attr[2])
                : go(k_paged_attn_q4<64, 2, 4>, k_q4_merge<64>, q4_smem_bytes<64, 2, 4>(), attr[3]);
  if (e != cudaSuccess) {
    set_err(err, errlen, "barlink: attention over the 4-bit cache could not be launched: %s", cudaGetErrorString(e));
    return -1;
  }
  KV4_LAUNCH_CHECK("paged_attn_decode_q4");
  return 0;
}
