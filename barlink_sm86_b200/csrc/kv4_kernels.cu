// SPDX-License-Identifier: MIT
//
// The key/value cache in 4 bits (layout: kv4.cuh): writer, reader, and attention of one query token per request.
//
// A group of 32 dims of a token's key (after RoPE) or value, both rounded to bf16, is held as low = its least
// element (exact in bf16), step = bf16((greatest - low) / 15) and codes rint((x - low) / step).  A group whose range
// is no finite number is held as step 0, low NaN: it reads as NaN and leaves the other groups alone.
#include <math.h>
#include <stdio.h>

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

// eight elements of a row from column `col`: the bf16 buffer, or the slabs added in split order, then the bias,
// rounded to bf16 (as k_rope_kv_write does)
__device__ __forceinline__ void q4_load8(const Q4Write& a, int row, int width, int col, float (&f)[8]) {
  if (a.slabs) {
    const float* p = a.slabs + size_t(row) * width + col;
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = 0.f;
    for (int s = 0; s < a.nsplit; ++s) {
      const float4 u = __ldcg(reinterpret_cast<const float4*>(p + s * a.slab));
      const float4 w = __ldcg(reinterpret_cast<const float4*>(p + s * a.slab) + 1);
      f[0] += u.x; f[1] += u.y; f[2] += u.z; f[3] += u.w;
      f[4] += w.x; f[5] += w.y; f[6] += w.z; f[7] += w.w;
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
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = __bfloat162float(__float2bfloat16(f[j]));
    return;
  }
  const uint4 b = *reinterpret_cast<const uint4*>(a.qkv + size_t(row) * width + col);
  const uint32_t w[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 v = unpack_bf16x2(w[j]);
    f[2 * j] = v.x;
    f[2 * j + 1] = v.y;
  }
}

__device__ __forceinline__ float quad_min(float v) {
  v = fminf(v, __shfl_xor_sync(0xffffffffu, v, 1));
  return fminf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}
__device__ __forceinline__ float quad_max(float v) {
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}

// Eight of a group's 32 elements, the rest with the other lanes of the quad -> codes (nibble e = element e), and the
// group's step and low as bf16 bits.  (x - low) / step is divided, not multiplied by a reciprocal: the codes are
// those of the formula to the bit.
__device__ __forceinline__ uint32_t q4_quantise8(const float (&x)[8], uint16_t& step_bits, uint16_t& low_bits) {
  float lo = x[0], hi = x[0], nan = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    lo = fminf(lo, x[e]);
    hi = fmaxf(hi, x[e]);
    nan += x[e] * 0.f;  // NaN where an element is no finite number (minimum and maximum pass over NaN)
  }
  lo = quad_min(lo);
  hi = quad_max(hi);
  nan += __shfl_xor_sync(0xffffffffu, nan, 1);
  nan += __shfl_xor_sync(0xffffffffu, nan, 2);
  __nv_bfloat16 st = __float2bfloat16(__fdiv_rn(hi - lo, 15.f));
  float step = __bfloat162float(st);
  const bool fine = nan == 0.f && isfinite(step);
  if (!fine) step = 0.f;
  uint32_t w = 0;
  if (step > 0.f) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float c = fminf(rintf(__fdiv_rn(x[e] - lo, step)), 15.f);
      w |= uint32_t(c) << (4 * e);
    }
  }
  step_bits = fine ? __bfloat16_as_ushort(st) : 0;
  low_bits = fine ? __bfloat16_as_ushort(__float2bfloat16(lo)) : 0x7fc0;
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

// One block per row.  A thread takes an octet of a head's lower half and its rotation partner; the angles of the row are
// computed once, in 64 bits (a position of 10^5 leaves 32 bits no better than 0.01 radians), and the products are
// rounded one by one: the rotated elements are the formula's to the bit.
__global__ void __launch_bounds__(256) k_rope_kv_write_q4(const Q4Write a) {
  pdl_launch_dependents();
  pdl_wait();
  __shared__ float2 s_rot[128];
  const int row = blockIdx.x, half = a.hd >> 1, width = (a.nq + 2 * a.nkv) * a.hd;
  for (int i = threadIdx.x; i < half; i += blockDim.x) {
    const double turn = double(a.positions[row]) * exp2(-a.log2_theta * (double(2 * i) / a.hd)) * 0.15915494309189533577;
    double sn, cs;
    sincospi(2.0 * (turn - rint(turn)), &sn, &cs);
    s_rot[i] = make_float2(float(cs), float(sn));
  }
  __syncthreads();
  int slot = a.slots ? a.slots[row] : -1;
  const int blk = slot >= 0 ? slot / a.block_size : 0, in_block = slot >= 0 ? slot % a.block_size : 0;
  if (blk >= a.n_blocks) slot = -1;  // no such block: not kept
  const int oph = a.hd >> 4;  // octets of half a head
  const int units = (a.nq + 2 * a.nkv) * oph;
  for (int u0 = 0; u0 < units; u0 += blockDim.x) {
    const int u = u0 + threadIdx.x;
    const bool there = u < units;  // (whole quads: oph is a multiple of 4)
    const int h = there ? u / oph : 0, o = there ? u % oph : 0, col = h * a.hd + 8 * o;
    float x[8] = {}, y[8] = {};
    if (there) {
      q4_load8(a, row, width, col, x);
      q4_load8(a, row, width, col + half, y);
      uint32_t ox[4], oy[4];
      if (h < a.nq + a.nkv) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float2 cs = s_rot[8 * o + j];
          const float p = __fsub_rn(__fmul_rn(x[j], cs.x), __fmul_rn(y[j], cs.y));
          const float q = __fadd_rn(__fmul_rn(y[j], cs.x), __fmul_rn(x[j], cs.y));
          x[j] = __bfloat162float(__float2bfloat16(p));
          y[j] = __bfloat162float(__float2bfloat16(q));
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        ox[j] = pack_bf16x2(x[2 * j], x[2 * j + 1]);
        oy[j] = pack_bf16x2(y[2 * j], y[2 * j + 1]);
      }
      __nv_bfloat16* p = a.out + size_t(row) * width + col;
      *reinterpret_cast<uint4*>(p) = make_uint4(ox[0], ox[1], ox[2], ox[3]);
      *reinterpret_cast<uint4*>(p + half) = make_uint4(oy[0], oy[1], oy[2], oy[3]);
    }
    const bool keep = there && h >= a.nq && slot >= 0;
    if (!__any_sync(0xffffffffu, keep)) continue;
    uint16_t s0, l0, s1, l1;
    const uint32_t w0 = q4_quantise8(x, s0, l0), w1 = q4_quantise8(y, s1, l1);
    if (keep) {
      const bool value = h >= a.nq + a.nkv;
      uint8_t* tile = a.cache + q4_tile_offset(blk, in_block, h - a.nq - (value ? a.nkv : 0), a.nkv, a.block_size, a.hd);
      const int r = in_block % kQ4Tokens;
      q4_store8(tile, r, a.hd, value, o >> 2, o & 3, w0, s0, l0);
      q4_store8(tile, r, a.hd, value, (o + oph) >> 2, o & 3, w1, s1, l1);
    }
  }
}

// Rows of the cache back as bf16 (zeros where a slot names none).  One octet of a key and of a value per thread.
__global__ void __launch_bounds__(256) k_kv4_read(const uint8_t* __restrict__ cache, const int* __restrict__ slots,
                                                  __nv_bfloat16* __restrict__ k, __nv_bfloat16* __restrict__ v, size_t units, int nkv,
                                                  int hd, int block_size, int n_blocks) {
  pdl_launch_dependents();
  pdl_wait();
  const size_t u = size_t(blockIdx.x) * blockDim.x + threadIdx.x;
  if (u >= units) return;
  const int oh = hd >> 3, o = int(u % oh), h = int(u / oh % nkv), na = hd / kQ4Group, ga = o >> 2, t = o & 3;
  const size_t row = u / oh / nkv;
  const int slot = slots[row];
  uint4 ko = make_uint4(0, 0, 0, 0), vo = ko;
  if (slot >= 0 && slot / block_size < n_blocks) {
    const int in_block = slot % block_size, r = in_block % kQ4Tokens;
    const uint8_t* tile = cache + q4_tile_offset(slot / block_size, in_block, h, nkv, block_size, hd);
    const uint32_t kw = *reinterpret_cast<const uint32_t*>(tile + r * (hd / 2) + (t * na + ga) * 4);
    const uint8_t* vp = tile + q4_v_codes(hd) + (r >> 1) * hd + (r & 1) * 2;
    const uint32_t vw = *reinterpret_cast<const uint16_t*>(vp + ((2 * t) * na + ga) * 4) |
                        uint32_t(*reinterpret_cast<const uint16_t*>(vp + ((2 * t + 1) * na + ga) * 4)) << 16;
    const __nv_bfloat16* kp = reinterpret_cast<const __nv_bfloat16*>(tile + q4_k_params(hd) + r * na * 4);
    const __nv_bfloat16* vq = reinterpret_cast<const __nv_bfloat16*>(tile + q4_v_params(hd) + r * na * 4);
    const float ks = __bfloat162float(kp[ga]), kl = __bfloat162float(kp[na + ga]);
    const float vs = __bfloat162float(vq[ga]), vl = __bfloat162float(vq[na + ga]);
    uint32_t kk[4], vv[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      kk[j] = pack_bf16x2(kl + ks * float((kw >> (8 * j)) & 15), kl + ks * float((kw >> (8 * j + 4)) & 15));
      vv[j] = pack_bf16x2(vl + vs * float((vw >> (8 * j)) & 15), vl + vs * float((vw >> (8 * j + 4)) & 15));
    }
    ko = make_uint4(kk[0], kk[1], kk[2], kk[3]);
    vo = make_uint4(vv[0], vv[1], vv[2], vv[3]);
  }
  *reinterpret_cast<uint4*>(k + u * 8) = ko;
  *reinterpret_cast<uint4*>(v + u * 8) = vo;
}

// ---------------------------------------------------------------------------
// attention
// ---------------------------------------------------------------------------
// One block per (request, KV head); a warp takes every fourth token, a lane hd / 32 dims of it.
constexpr int kQ4MaxG = 16;
template <int HD>
__global__ void __launch_bounds__(128) k_paged_attn_q4(const __nv_bfloat16* __restrict__ q, int q_stride,
                                                       const uint8_t* __restrict__ cache, const int* __restrict__ tables,
                                                       const int* __restrict__ ctx_lens, __nv_bfloat16* __restrict__ out, int nq,
                                                       int nkv, int block_size, int n_blocks, int max_blocks, float scale_log2) {
  constexpr int NA = HD / kQ4Group, D = HD / 32;  // a lane's dims are D * lane ..
  pdl_launch_dependents();
  pdl_wait();
  __shared__ float s_o[4][HD];
  __shared__ float s_m[4], s_l[4];
  const int h = blockIdx.x, b = blockIdx.y, G = nq / nkv, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int ctx = min(ctx_lens[b], max_blocks * block_size);
  float m[kQ4MaxG], l[kQ4MaxG], o[kQ4MaxG][D];
#pragma unroll
  for (int g = 0; g < kQ4MaxG; ++g) {
    m[g] = -INFINITY;
    l[g] = 0.f;
#pragma unroll
    for (int j = 0; j < D; ++j) o[g][j] = 0.f;
  }
  const __nv_bfloat16* qb = q + size_t(b) * q_stride + size_t(h) * G * HD + D * lane;
  const int d0 = D * lane, ga = d0 / kQ4Group;
  for (int tok = warp; tok < ctx; tok += 4) {
    const int blk = tables[size_t(b) * max_blocks + tok / block_size];
    if (blk < 0 || blk >= n_blocks) continue;
    const int in_block = tok % block_size, r = in_block % kQ4Tokens;
    const uint8_t* tile = cache + q4_tile_offset(blk, in_block, h, nkv, block_size, HD);
    const uint32_t kw = *reinterpret_cast<const uint32_t*>(tile + r * (HD / 2) + (((d0 >> 3) & 3) * NA + ga) * 4) >> (4 * (d0 & 7));
    const uint32_t vw = *reinterpret_cast<const uint16_t*>(tile + q4_v_codes(HD) + (r >> 1) * HD + (r & 1) * 2 +
                                                           (((d0 >> 2) & 7) * NA + ga) * 4) >> (4 * (d0 & 3));
    const __nv_bfloat16* kp = reinterpret_cast<const __nv_bfloat16*>(tile + q4_k_params(HD) + r * NA * 4);
    const __nv_bfloat16* vp = reinterpret_cast<const __nv_bfloat16*>(tile + q4_v_params(HD) + r * NA * 4);
    float k[D], v[D];
#pragma unroll
    for (int j = 0; j < D; ++j) {
      k[j] = __bfloat162float(kp[NA + ga]) + __bfloat162float(kp[ga]) * float((kw >> (4 * j)) & 15);
      v[j] = __bfloat162float(vp[NA + ga]) + __bfloat162float(vp[ga]) * float((vw >> (4 * j)) & 15);
    }
#pragma unroll
    for (int g = 0; g < kQ4MaxG; ++g) {
      if (g >= G) break;
      float s = 0.f;
#pragma unroll
      for (int j = 0; j < D; ++j) s += __bfloat162float(qb[g * HD + j]) * k[j];
      s = warp_sum(s) * scale_log2;
      const float n = fmaxf(m[g], s);
      const float al = exp2f(m[g] - n), p = exp2f(s - n);
      m[g] = n;
      l[g] = l[g] * al + p;
#pragma unroll
      for (int j = 0; j < D; ++j) o[g][j] = o[g][j] * al + p * v[j];
    }
  }
#pragma unroll
  for (int g = 0; g < kQ4MaxG; ++g) {
    if (g >= G) break;
    __syncthreads();
    if (lane == 0) {
      s_m[warp] = m[g];
      s_l[warp] = l[g];
    }
#pragma unroll
    for (int j = 0; j < D; ++j) s_o[warp][d0 + j] = o[g][j];
    __syncthreads();
    if (threadIdx.x < HD) {
      const float M = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
      float L = 0.f, acc = 0.f;
      for (int w = 0; w < 4; ++w) {
        const float f = s_m[w] == -INFINITY ? 0.f : exp2f(s_m[w] - M);
        L += s_l[w] * f;
        acc += s_o[w][threadIdx.x] * f;
      }
      out[(size_t(b) * nq + h * G + g) * HD + threadIdx.x] = __float2bfloat16(L == 0.f ? 0.f : acc / L);
    }
  }
}

}  // namespace bl

using namespace bl;

static int q4_shape(const char* what, int hd, int block_size, int n_blocks, char* err, size_t errlen) {
  if ((hd != 64 && hd != 128) || block_size < kQ4Tokens || block_size % kQ4Tokens) {
    set_err(err, errlen, "barlink: %s is built for head_dim 64 and 128 and block sizes that are multiples of %d", what, kQ4Tokens);
    return -1;
  }
  if (n_blocks < 0 || int64_t(n_blocks) * block_size > 0x7fffffffLL) {
    set_err(err, errlen, "barlink: %s: the cache's slots do not fit 32 bits", what);
    return -1;
  }
  return 0;
}

extern "C" size_t bl_kv4_tile_bytes(int hd) { return q4_tile_bytes(hd); }

extern "C" int bl_rope_kv_write_q4(const void* qkv, const void* slabs, int nsplit, size_t slab, const void* bias, void* out,
                                   const int* positions, const int* slots, void* cache, int rows, int nq, int nkv, int hd,
                                   int block_size, int n_blocks, double theta, void* stream, char* err, size_t errlen) {
  if (q4_shape("the 4-bit cache", hd, block_size, n_blocks, err, errlen)) return -1;
  if (rows < 0 || nq < 0 || nkv < 1 || (!qkv && (!slabs || nsplit < 1)) || !out || !positions || (slots && !cache) || !(theta > 0)) {
    set_err(err, errlen, "barlink: rope_kv_write_q4 needs the QKV rows or slabs, positions, an output and, with slots, a cache");
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
  launch_k(k_rope_kv_write_q4, dim3(rows), dim3(256), 0, static_cast<cudaStream_t>(stream), a);
  KV4_LAUNCH_CHECK("rope_kv_write_q4");
  return 0;
}

extern "C" int bl_kv4_read(const void* cache, const int* slots, void* k, void* v, int rows, int nkv, int hd, int block_size,
                           int n_blocks, void* stream, char* err, size_t errlen) {
  if (q4_shape("the 4-bit cache", hd, block_size, n_blocks, err, errlen)) return -1;
  const size_t units = size_t(rows) * nkv * (hd / 8);
  if (units == 0) return 0;
  launch_k(k_kv4_read, dim3(unsigned((units + 255) / 256)), dim3(256), 0, static_cast<cudaStream_t>(stream),
           static_cast<const uint8_t*>(cache), slots, static_cast<__nv_bfloat16*>(k), static_cast<__nv_bfloat16*>(v), units, nkv,
           hd, block_size, n_blocks);
  KV4_LAUNCH_CHECK("kv4_read");
  return 0;
}

extern "C" int bl_paged_attn_decode_q4(const void* q, int q_stride, const void* cache, const int* block_tables, const int* ctx_lens,
                                       void* out, int batch, int nq, int nkv, int hd, int block_size, int n_blocks, int max_blocks,
                                       float scale, void* ws, size_t ws_bytes, void* stream, char* err, size_t errlen) {
  if (q4_shape("attention over the 4-bit cache", hd, block_size, n_blocks, err, errlen)) return -1;
  if (nkv < 1 || nq < 1 || nq % nkv || nq / nkv > kQ4MaxG) {
    set_err(err, errlen, "barlink: attention over the 4-bit cache needs nq %% nkv == 0 and at most %d query heads per KV head", kQ4MaxG);
    return -1;
  }
  if (int64_t(max_blocks) * block_size > 0x7fffffffLL || batch > 65535) {
    set_err(err, errlen, "barlink: attention over the 4-bit cache: contexts must fit 32 bits, and at most 65535 requests");
    return -1;
  }
  if (batch == 0) return 0;
  (void)ws; (void)ws_bytes;
  const float scale_log2 = scale * 1.4426950408889634f;
  launch_k(hd == 64 ? k_paged_attn_q4<64> : k_paged_attn_q4<128>, dim3(nkv, batch), dim3(128), 0, static_cast<cudaStream_t>(stream),
           static_cast<const __nv_bfloat16*>(q), q_stride, static_cast<const uint8_t*>(cache), block_tables, ctx_lens,
           static_cast<__nv_bfloat16*>(out), nq, nkv, block_size, n_blocks, max_blocks, scale_log2);
  KV4_LAUNCH_CHECK("paged_attn_decode_q4");
  return 0;
}
