// SPDX-License-Identifier: MIT
//
// Third part of the `_C` binding: the 4-bit key/value cache, request layouts, rules on logits.  Workspaces are
// allocated by each call from the caching allocator, so that calls on several streams and captured graphs share none.
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/utils/pybind.h>
#include <torch/extension.h>

#include <tuple>

#include "bl_ops.h"

namespace py = pybind11;

// (Numbers go into the messages of TORCH_CHECK as text, std::to_string, see binding_extra.cc.)

namespace {

constexpr size_t kErr = 512;
#define BL_CHECK(expr)                                                 \
  do {                                                                 \
    char _e[kErr] = {0};                                               \
    char* err = _e;                                                    \
    size_t errlen = kErr;                                              \
    (void)err; (void)errlen;                                           \
    int _rc = (expr);                                                  \
    TORCH_CHECK(_rc == 0, _e[0] ? _e : "barlink: call failed: " #expr); \
  } while (0)

void* stream_of(const at::Tensor& t) {
  return at::cuda::getCurrentCUDAStream(t.device().index()).stream();
}
using OptTensor = c10::optional<at::Tensor>;

// Small calls are bound by the host: a tensor costs half as much from the allocator directly, and parts of one buffer a tenth.
at::Tensor fresh(at::IntArrayRef size, at::ScalarType type, const at::Tensor& like) {
  return at::Tensor(at::detail::empty_cuda(size, type, like.device(), c10::nullopt));
}
at::Tensor part_of(const at::Tensor& buf, at::ScalarType type, int64_t byte_offset, at::IntArrayRef size) {
  at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(buf.storage()), buf.key_set(), c10::scalarTypeToTypeMeta(type));
  t.unsafeGetTensorImpl()->set_storage_offset(byte_offset / int64_t(c10::elementSize(type)));
  t.unsafeGetTensorImpl()->set_sizes_contiguous(size);
  return t;
}
int64_t to16(int64_t bytes) { return (bytes + 15) / 16 * 16; }

void check_on(const at::Tensor& t, const at::Tensor& like, const char* name) {
  TORCH_CHECK(t.is_cuda() && t.device() == like.device(), "barlink: ", name, " must be on the same GPU as the other tensors");
}
const int* i32(const at::Tensor& t, const at::Tensor& like, int64_t n, const char* name) {
  check_on(t, like, name);
  TORCH_CHECK(t.scalar_type() == at::kInt && t.is_contiguous(), "barlink: ", name, " must be contiguous int32");
  TORCH_CHECK(n < 0 || t.numel() == n, "barlink: ", name, " must have ", std::to_string(n), " elements");
  return t.data_ptr<int>();
}
bool aligned16(const at::Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }
int small(int64_t n, const char* name) {
  TORCH_CHECK(n >= 0 && n <= 0x7fffffff, "barlink: ", name, " does not fit 32 bits");
  return int(n);
}

// [blocks, nkv, block_size / 16, tile bytes] uint8
void check_cache(const at::Tensor& cache, const at::Tensor& like, int nkv, int hd, int block_size) {
  check_on(cache, like, "cache");
  TORCH_CHECK(hd == 64 || hd == 128, "barlink: the 4-bit cache is built for head_dim 64 and 128");
  TORCH_CHECK(block_size >= 16 && block_size % 16 == 0, "barlink: the 4-bit cache needs a block size that is a multiple of 16");
  TORCH_CHECK(cache.scalar_type() == at::kByte && cache.is_contiguous() && cache.dim() == 4 && cache.size(1) == nkv &&
                  cache.size(2) == block_size / 16 && cache.size(3) == int64_t(bl_kv4_tile_bytes(hd)) && aligned16(cache),
              "barlink: the 4-bit cache is a contiguous uint8 [blocks, nkv, block_size / 16, tile bytes] as kv4_cache makes it");
}

at::Tensor rope_kv_write_q4(const at::Tensor& qkv, const at::Tensor& positions, const OptTensor& slots, const OptTensor& cache,
                            int nq, int nkv, int hd, int block_size, double theta, const OptTensor& bias, const OptTensor& out_opt) {
  const bool slabs = qkv.scalar_type() == at::kFloat;
  TORCH_CHECK(nq >= 0 && nkv >= 1 && (hd == 64 || hd == 128), "barlink: rope_kv_write_q4 needs KV heads of head_dim 64 or 128");
  TORCH_CHECK(qkv.is_cuda() && qkv.is_contiguous() && aligned16(qkv) &&
                  (slabs ? qkv.dim() == 3 && qkv.size(0) >= 1 : qkv.scalar_type() == at::kBFloat16 && qkv.dim() == 2),
              "barlink: qkv must be a contiguous, 16-byte aligned CUDA tensor: bfloat16 [rows, width] or float32 slabs [splits, rows, width]");
  const int rows = small(qkv.size(slabs ? 1 : 0), "rows");
  const int64_t width = (int64_t(nq) + 2 * int64_t(nkv)) * hd;
  TORCH_CHECK(qkv.size(slabs ? 2 : 1) == width && width <= 0x7fffffff, "barlink: qkv rows must hold nq + 2 nkv heads");
  TORCH_CHECK(theta > 0, "barlink: theta must be positive");
  TORCH_CHECK(!bias || slabs, "barlink: bias is applied only when the input is split-K slabs");
  const int* pos = i32(positions, qkv, rows, "positions");
  if (bias) {
    check_on(*bias, qkv, "bias");
    TORCH_CHECK(bias->scalar_type() == at::kBFloat16 && bias->is_contiguous() && bias->numel() == width && aligned16(*bias),
                "barlink: bias must be a contiguous, 16-byte aligned bfloat16 tensor of one entry per qkv column");
  }
  const int* sl = nullptr;
  void* cp = nullptr;
  int n_blocks = 0;
  TORCH_CHECK(bool(slots) == bool(cache), "barlink: slots and the cache go together");
  if (slots) {
    sl = i32(*slots, qkv, rows, "slots");
    check_cache(*cache, qkv, nkv, hd, block_size);
    cp = cache->data_ptr();
    n_blocks = small(cache->size(0), "blocks");
  } else {
    block_size = 16;
  }
  c10::cuda::CUDAGuard guard(qkv.device());
  at::Tensor out = out_opt ? *out_opt : slabs ? fresh({rows, width}, at::kBFloat16, qkv) : qkv;
  check_on(out, qkv, "out");
  TORCH_CHECK(out.scalar_type() == at::kBFloat16 && out.is_contiguous() && out.dim() == 2 && out.size(0) == rows && out.size(1) == width &&
                  aligned16(out),
              "barlink: out must be a contiguous, 16-byte aligned bfloat16 [rows, width]");
  if (rows > 0)
    BL_CHECK(bl_rope_kv_write_q4(slabs ? nullptr : qkv.data_ptr(), slabs ? qkv.data_ptr() : nullptr, slabs ? int(qkv.size(0)) : 0,
                                 size_t(rows) * width, bias ? bias->data_ptr() : nullptr, out.data_ptr(), pos, sl, cp, rows, nq, nkv, hd,
                                 block_size, n_blocks, theta, stream_of(qkv), err, errlen));
  return out;
}

std::tuple<at::Tensor, at::Tensor> kv4_read(const at::Tensor& cache, const at::Tensor& slots, int hd, int block_size) {
  TORCH_CHECK(cache.is_cuda() && cache.dim() == 4, "barlink: the 4-bit cache must be a 4-D CUDA tensor");
  const int nkv = small(cache.size(1), "KV heads");
  check_cache(cache, cache, nkv, hd, block_size);
  const int rows = small(slots.numel(), "rows");
  const int* sl = i32(slots, cache, -1, "slots");
  c10::cuda::CUDAGuard guard(cache.device());
  const int64_t half = int64_t(rows) * nkv * hd * 2;  // (hd: a multiple of 16 bytes)
  at::Tensor both = fresh({2 * half}, at::kByte, cache);
  at::Tensor k = part_of(both, at::kBFloat16, 0, {rows, nkv, hd}), v = part_of(both, at::kBFloat16, half, {rows, nkv, hd});
  if (rows > 0)
    BL_CHECK(bl_kv4_read(cache.data_ptr(), sl, k.data_ptr(), v.data_ptr(), rows, nkv, hd, block_size, small(cache.size(0), "blocks"),
                         stream_of(cache), err, errlen));
  return {k, v};
}

// 1: a kernel of this device gave up waiting for its copies
int kv4_error_flag(int dev) {
  c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(dev));
  unsigned v = 0;
  BL_CHECK(bl_kv4_error(&v, err, errlen));
  return int(v);
}
void kv4_error_clear(int dev) {
  c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(dev));
  BL_CHECK(bl_kv4_error_clear(err, errlen));
}
// The same word, into a pinned int32 tensor on the current stream of a device: the caller reads it once the stream has come that far.
void kv4_error_into(const at::Tensor& out, int dev) {
  TORCH_CHECK(out.is_cpu() && out.is_pinned() && out.scalar_type() == at::kInt && out.numel() == 1, "barlink: kv4_error_into needs a pinned int32 element");
  c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(dev));
  BL_CHECK(bl_kv4_error_async(static_cast<unsigned*>(out.data_ptr()), at::cuda::getCurrentCUDAStream(dev).stream(), err, errlen));
}

at::Tensor paged_attn_decode_q4(const at::Tensor& q, const at::Tensor& cache, const at::Tensor& block_tables, const at::Tensor& ctx_lens,
                                int nq, int nkv, int hd, double scale, const OptTensor& out_opt) {
  TORCH_CHECK(q.is_cuda() && q.scalar_type() == at::kBFloat16 && q.dim() == 2 && q.stride(1) == 1 && q.stride(0) % 8 == 0 && aligned16(q),
              "barlink: q/qkv must be a 2-D bfloat16 CUDA tensor whose rows start on 16-byte boundaries");
  TORCH_CHECK(nkv >= 1 && nq >= 1 && nq % nkv == 0 && nq / nkv <= 16,
              "barlink: attention over the 4-bit cache needs nq % nkv == 0 and at most 16 query heads per KV head");
  TORCH_CHECK(cache.dim() == 4, "barlink: the 4-bit cache must be a 4-D CUDA tensor");
  const int block_size = small(cache.size(2) * 16, "block size");
  check_cache(cache, q, nkv, hd, block_size);
  const int batch = small(q.size(0), "batch");
  TORCH_CHECK(q.size(1) >= int64_t(nq) * hd && (batch < 2 || q.stride(0) >= int64_t(nq) * hd) && q.stride(0) <= 0x7fffffff,
              "barlink: q rows too short");
  TORCH_CHECK(block_tables.dim() == 2 && block_tables.size(0) == batch, "barlink: block_tables must be int32 [batch, max_blocks]");
  const int* bt = i32(block_tables, q, -1, "block_tables");
  const int* cl = i32(ctx_lens, q, batch, "ctx_lens");
  c10::cuda::CUDAGuard guard(q.device());
  at::Tensor out = out_opt ? *out_opt : fresh({batch, int64_t(nq) * hd}, at::kBFloat16, q);
  check_on(out, q, "out");
  TORCH_CHECK(out.scalar_type() == at::kBFloat16 && out.is_contiguous() && out.dim() == 2 && out.size(0) == batch &&
                  out.size(1) == int64_t(nq) * hd && aligned16(out),
              "barlink: out must be a contiguous, 16-byte aligned bfloat16 [batch, nq * hd]");
  if (batch > 0 && block_tables.size(1) == 0) {
    out.zero_();
  } else if (batch > 0) {
    const int max_blocks = small(block_tables.size(1), "max_blocks");
    const size_t bytes = bl_paged_attn_decode_q4_ws(batch, nq, nkv, hd);
    at::Tensor ws = fresh({int64_t(bytes)}, at::kByte, cache);
    BL_CHECK(bl_paged_attn_decode_q4(q.data_ptr(), int(q.stride(0)), cache.data_ptr(), bt, cl, out.data_ptr(), batch, nq, nkv, hd,
                                     block_size, small(cache.size(0), "blocks"), max_blocks, float(scale),
                                     ws.data_ptr(), bytes, stream_of(q), err, errlen));
  }
  return out;
}

// [cu, positions, slots, ctx_lens, free_range]; `into`: the same five to write to
std::vector<at::Tensor> paged_layout(const at::Tensor& new_lens, const at::Tensor& past_lens, const at::Tensor& block_tables,
                                     const at::Tensor& free_list, const at::Tensor& free_range, int64_t tokens, int block_size, int rows_per_request,
                                     const c10::optional<std::vector<at::Tensor>>& into, const OptTensor& lost) {
  TORCH_CHECK(new_lens.is_cuda() && new_lens.dim() == 1, "barlink: new_lens must be a 1-D CUDA tensor");
  const int batch = small(new_lens.numel(), "batch"), rows = small(tokens, "tokens");
  const int* nl = i32(new_lens, new_lens, -1, "new_lens");
  const int* pl = i32(past_lens, new_lens, batch, "past_lens");
  TORCH_CHECK(block_tables.dim() == 2 && block_tables.size(0) == batch, "barlink: block_tables must be int32 [batch, max_blocks]");
  i32(block_tables, new_lens, -1, "block_tables");
  i32(free_list, new_lens, -1, "free_list");
  const int* fr = i32(free_range, new_lens, 3, "free_range");
  TORCH_CHECK(block_size >= 1 && rows_per_request >= 0, "barlink: block_size must be positive, rows_per_request not below 0");
  c10::cuda::CUDAGuard guard(new_lens.device());
  std::vector<at::Tensor> r;
  if (into) {
    r = *into;
    TORCH_CHECK(r.size() == 5, "barlink: paged_layout writes cu, positions, slots, ctx_lens and free_range");
  } else {
    const int64_t n[5] = {int64_t(batch) + 1, rows, rows, batch, 3};
    int64_t at[6] = {0};
    for (int i = 0; i < 5; ++i) at[i + 1] = at[i] + to16(4 * n[i]);
    const at::Tensor all = fresh({at[5]}, at::kByte, new_lens);
    for (int i = 0; i < 5; ++i) r.push_back(part_of(all, at::kInt, at[i], {n[i]}));
  }
  i32(r[0], new_lens, batch + 1, "cu");
  i32(r[1], new_lens, rows, "positions");
  i32(r[2], new_lens, rows, "slots");
  i32(r[3], new_lens, batch, "ctx_lens");
  i32(r[4], new_lens, 3, "free_range");
  if (lost) i32(*lost, new_lens, 1, "lost");
  BL_CHECK(bl_paged_layout_counting(nl, pl, block_tables.data_ptr<int>(), free_list.data_ptr<int>(), fr, r[0].data_ptr<int>(),
                           r[1].data_ptr<int>(), r[2].data_ptr<int>(), r[3].data_ptr<int>(), r[4].data_ptr<int>(), batch,
                           small(block_tables.size(1), "max_blocks"), small(free_list.numel(), "free_list"), rows, block_size, rows_per_request,
                           lost ? lost->data_ptr<int>() : nullptr, stream_of(new_lens), err, errlen));
  return r;
}

void count_tokens(const at::Tensor& counts, const at::Tensor& seen, const at::Tensor& ids, const OptTensor& cu,
                  const OptTensor& prompt_lens, bool reset) {
  TORCH_CHECK(counts.is_cuda() && counts.dim() == 2 && seen.dim() == 2 && seen.size(0) == counts.size(0) &&
                  seen.size(1) == (counts.size(1) + 31) / 32,
              "barlink: counts must be int32 [rows, vocab] and seen int32 [rows, ceil(vocab / 32)] on a GPU");
  i32(counts, counts, -1, "counts");
  i32(seen, counts, -1, "seen");
  const int rows = small(counts.size(0), "rows"), vocab = small(counts.size(1), "vocab");
  const int* id = i32(ids, counts, cu ? -1 : rows, "ids");
  const int* c = cu ? i32(*cu, counts, int64_t(rows) + 1, "cu") : nullptr;
  const int* p = prompt_lens ? i32(*prompt_lens, counts, rows, "prompt_lens") : nullptr;
  c10::cuda::CUDAGuard guard(counts.device());
  if (rows > 0 && vocab > 0)
    BL_CHECK(bl_count_tokens(id, c, p, counts.data_ptr<int>(), seen.data_ptr(), rows, small(ids.numel(), "ids"), vocab, reset ? 1 : 0,
                             stream_of(counts), err, errlen));
}

// pick: (token, value) of the arg max; else the logits under the rules (into out, or a new tensor)
std::vector<at::Tensor> logit_rules(const at::Tensor& logits, bool pick, int64_t vocab, int offset, const OptTensor& penalties,
                                    const OptTensor& counts, const OptTensor& seen, const OptTensor& bias_ids, const OptTensor& bias,
                                    const OptTensor& mask, const OptTensor& out_opt) {
  const bool fp32 = logits.scalar_type() == at::kFloat;
  TORCH_CHECK(logits.is_cuda() && (fp32 || logits.scalar_type() == at::kBFloat16) && logits.dim() == 2 && logits.stride(1) == 1 &&
                  (logits.size(0) < 2 || logits.stride(0) >= logits.size(1)),
              "barlink: logit rules need 2-D bfloat16 or float32 CUDA logits with dense rows");
  blRulesArgs a = {};
  a.rows = small(logits.size(0), "rows");
  a.n = small(logits.size(1), "columns");
  a.fp32 = fp32;
  a.vocab = small(vocab, "vocab");
  a.offset = offset;
  TORCH_CHECK(offset >= 0 && int64_t(offset) + a.n <= 0x7fffffff && a.n >= 1, "barlink: token ids must fit 32 bits");
  a.logits = logits.data_ptr();
  a.ld = size_t(logits.stride(0));
  const int64_t words = (vocab + 31) / 32;
  auto f32 = [&](const at::Tensor& t, int64_t n, const char* name) {
    check_on(t, logits, name);
    TORCH_CHECK(t.scalar_type() == at::kFloat && t.is_contiguous() && t.numel() == n, "barlink: ", name, " must be contiguous float32 of ",
                std::to_string(n), " elements");
    return t.data_ptr();
  };
  if (penalties) {
    TORCH_CHECK(counts && seen, "barlink: penalties need the counts and seen tables");
    a.penalties = f32(*penalties, int64_t(a.rows) * 3, "penalties");
    a.counts = i32(*counts, logits, a.rows * vocab, "counts");
    a.seen = i32(*seen, logits, a.rows * words, "seen");
  }
  TORCH_CHECK(bool(bias_ids) == bool(bias), "barlink: bias_ids and bias go together");
  if (bias && bias->numel() > 0) {
    TORCH_CHECK(bias_ids->dim() == 2 && bias_ids->size(0) == a.rows, "barlink: bias_ids must be int32 [rows, entries]");
    a.n_bias = small(bias_ids->size(1), "bias entries");
    TORCH_CHECK(a.n_bias <= 4096, "barlink: at most 4096 bias entries per row");
    a.bias_ids = i32(*bias_ids, logits, -1, "bias_ids");
    a.bias = f32(*bias, bias_ids->numel(), "bias");
  }
  if (mask) {
    check_on(*mask, logits, "mask");
    TORCH_CHECK(mask->scalar_type() == at::kInt && mask->dim() == 2 && mask->size(0) == a.rows && mask->size(1) >= words &&
                    (mask->stride(1) == 1 || mask->size(1) == 1) && (mask->stride(0) >= mask->size(1) || a.rows < 2 || mask->stride(0) == 0),
                "barlink: mask must be int32 [rows, >= ceil(vocab / 32)] with dense rows");
    a.mask = mask->data_ptr();
    a.mask_words = small(mask->size(1), "mask");
    a.ld_mask = size_t(mask->stride(0));
  }
  c10::cuda::CUDAGuard guard(logits.device());
  std::vector<at::Tensor> r;
  if (!pick) {
    at::Tensor out = out_opt ? *out_opt : fresh({a.rows, a.n}, logits.scalar_type(), logits);
    check_on(out, logits, "out");
    TORCH_CHECK(out.scalar_type() == logits.scalar_type() && out.dim() == 2 && out.size(0) == a.rows && out.size(1) == a.n && out.stride(1) == 1 &&
                    (a.rows < 2 || out.stride(0) >= a.n),
                "barlink: out must have the logits' shape and type, with dense rows");
    a.out = out.data_ptr();
    a.ld_out = size_t(out.stride(0));
    r = {out};
  } else {
    const at::Tensor both = fresh({2 * to16(4 * int64_t(a.rows))}, at::kByte, logits);
    r = {part_of(both, at::kInt, 0, {a.rows}), part_of(both, at::kFloat, to16(4 * int64_t(a.rows)), {a.rows})};
    a.idx = r[0].data_ptr();
    a.val = r[1].data_ptr();
  }
  if (a.rows > 0) BL_CHECK(bl_logit_rules(&a, stream_of(logits), err, errlen));
  return r;
}

}  // namespace

void bind_serve(py::module_& m) {
  m.def("kv4_tile_bytes", &bl_kv4_tile_bytes, py::arg("hd"));
  m.def("rope_kv_write_q4", &rope_kv_write_q4, py::arg("qkv"), py::arg("positions"), py::arg("slots"), py::arg("cache"), py::arg("nq"),
        py::arg("nkv"), py::arg("hd"), py::arg("block_size"), py::arg("theta"), py::arg("bias") = py::none(), py::arg("out") = py::none());
  m.def("kv4_read", &kv4_read, py::arg("cache"), py::arg("slots"), py::arg("hd"), py::arg("block_size"));
  m.def("paged_attn_decode_q4", &paged_attn_decode_q4, py::arg("q"), py::arg("cache"), py::arg("block_tables"), py::arg("ctx_lens"),
        py::arg("nq"), py::arg("nkv"), py::arg("hd"), py::arg("scale"), py::arg("out") = py::none());
  m.def("kv4_error_flag", &kv4_error_flag, py::arg("device") = 0);
  m.def("kv4_error_clear", &kv4_error_clear, py::arg("device") = 0);
  m.def("kv4_error_into", &kv4_error_into, py::arg("out"), py::arg("device") = 0);
  m.def("kv4_wait_polls", &bl_kv4_wait_polls, py::arg("polls"));
  m.def("paged_layout", &paged_layout, py::arg("new_lens"), py::arg("past_lens"), py::arg("block_tables"), py::arg("free_list"),
        py::arg("free_range"), py::arg("tokens"), py::arg("block_size"), py::arg("rows_per_request") = 0, py::arg("into") = py::none(), py::arg("lost") = py::none());
  m.def("count_tokens", &count_tokens, py::arg("counts"), py::arg("seen"), py::arg("ids"), py::arg("cu") = py::none(),
        py::arg("prompt_lens") = py::none(), py::arg("reset") = false);
  m.def("logit_rules", &logit_rules, py::arg("logits"), py::arg("pick"), py::arg("vocab"), py::arg("offset") = 0,
        py::arg("penalties") = py::none(), py::arg("counts") = py::none(), py::arg("seen") = py::none(), py::arg("bias_ids") = py::none(),
        py::arg("bias") = py::none(), py::arg("mask") = py::none(), py::arg("out") = py::none());
}
