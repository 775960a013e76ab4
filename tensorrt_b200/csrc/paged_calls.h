// The calls of the paged key-value cache and its attention on torch tensors: checks of the arguments, outputs, one b200q_* call on
// the current stream.  Shared by the torch.library shim (torch_ops.cpp) and the native Python calls (python_calls.cpp).
#pragma once

#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <cuda_runtime_api.h>

#include <algorithm>
#include <cmath>
#include <map>
#include <mutex>
#include <optional>
#include <tuple>
#include <utility>

#include "b200q.h"

namespace b200q_calls {
namespace {

using at::Tensor;

void must_be_ok(int rc, const char* what) { TORCH_CHECK(rc == B200Q_OK, what, " failed: ", b200q_status_string(rc), " (status ", rc, ")"); }
b200q_stream_t stream_of_call() { return static_cast<b200q_stream_t>(at::cuda::getCurrentCUDAStream().stream()); }
Tensor f32_on(const Tensor& t, const Tensor& like) {
  return t.scalar_type() == at::kFloat && t.is_contiguous() && t.device() == like.device() ? t : t.to(like.device(), at::kFloat).contiguous();
}

// Pages [pages, kv heads, rows, D] (any strides with D contiguous), block table [B, pages per sequence] int32, lens [B] int32.
struct CacheArgs {
  b200q_paged_cache c{};
  Tensor k_amax, v_amax;     // keep the converted ranges alive
  const int32_t* table;
  int64_t table_stride, table_width, B;
  const int32_t* lens;
};

bool rows_16(const Tensor& t) {
  const int64_t unit = 16 / t.element_size();
  if (t.dim() == 0 || (t.size(-1) > 1 && t.stride(-1) != 1) || reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 != 0) return false;
  for (int64_t i = 0; i + 1 < t.dim(); ++i)
    if (t.size(i) > 1 && t.stride(i) % unit != 0) return false;
  return true;
}
Tensor rows_of_16(const Tensor& t) { return rows_16(t) ? t : t.clone(at::MemoryFormat::Contiguous); }
// the same, and no two rows in one place: a tensor map has no stride of zero
Tensor rows_apart(const Tensor& t) {
  for (int64_t i = 0; i + 1 < t.dim(); ++i)
    if (t.size(i) > 1 && t.stride(i) == 0) return t.clone(at::MemoryFormat::Contiguous);
  return rows_of_16(t);
}
int64_t outer_stride(const Tensor& t, int64_t dim) { return t.size(dim) > 1 ? t.stride(dim) : 0; }   // torch leaves any value where there is one

void check_table(const Tensor& t, const Tensor& like, const char* what, const char* op) {
  TORCH_CHECK(t.device() == like.device() && t.scalar_type() == at::kInt && t.dim() == 2 && (t.size(1) <= 1 || t.stride(1) == 1), op, ": ", what,
              " must be int32 [B, pages] on the device of the pages, a line contiguous, got ", t.sizes(), " of ", t.scalar_type());
}
const int32_t* check_lens(const std::optional<Tensor>& t, int64_t n, const Tensor& like, const char* what, const char* op) {
  if (!t.has_value()) return nullptr;
  TORCH_CHECK(t->device() == like.device() && t->scalar_type() == at::kInt && t->dim() == 1 && t->size(0) == n && t->is_contiguous(), op, ": ", what,
              " must be ", n, " contiguous int32 values on the device of the inputs, got ", t->sizes(), " of ", t->scalar_type());
  return t->data_ptr<int32_t>();
}

CacheArgs cache_args(const Tensor& k_pages, const Tensor& v_pages, const Tensor& table, const Tensor& lens, const std::optional<Tensor>& k_amax,
                     const std::optional<Tensor>& v_amax, bool moves, const char* op) {
  TORCH_CHECK(k_pages.is_cuda(), op, ": b200q operates on CUDA tensors only; there is no CPU implementation");
  TORCH_CHECK(k_pages.dim() == 4 && k_pages.sizes() == v_pages.sizes() && k_pages.scalar_type() == v_pages.scalar_type() &&
                  v_pages.device() == k_pages.device(),
              op, ": expected k_pages and v_pages [pages, kv heads, rows, D] of one type, got ", k_pages.sizes(), " and ", v_pages.sizes());
  CacheArgs a;
  switch (k_pages.scalar_type()) {
    case at::kHalf: a.c.dtype = B200Q_F16; break;
    case at::kBFloat16: a.c.dtype = B200Q_BF16; break;
    case at::kByte:
    case at::kFloat8_e4m3fn: a.c.dtype = B200Q_E4M3; break;
    default: TORCH_CHECK_VALUE(false, op, " received pages of ", k_pages.scalar_type(), " type. Supported types: float16 | bfloat16 | float8_e4m3fn | uint8 (its codes)");
  }
  TORCH_CHECK_VALUE(k_pages.size(3) % 16 == 0 && k_pages.size(3) > 0 && k_pages.size(3) <= 128 && k_pages.size(2) > 0, op,
                    ": need a head dimension that is a multiple of 16 up to 128 and pages of at least one row, got pages ", k_pages.sizes());
  TORCH_CHECK(rows_16(k_pages) && rows_16(v_pages), op, ": rows of pages must be contiguous, 16-byte aligned and multiples of 16 bytes apart, got strides ",
              k_pages.strides(), " and ", v_pages.strides());
  check_table(table, k_pages, "block_table", op);
  a.B = table.size(0);
  TORCH_CHECK(lens.dim() == 1, op, ": lens must be int32 [B]");
  a.lens = check_lens(lens, a.B, k_pages, "lens", op);
  a.table = table.data_ptr<int32_t>();
  a.table_stride = outer_stride(table, 0);
  a.table_width = table.size(1);
  a.c.k_pages = k_pages.data_ptr();
  a.c.v_pages = v_pages.data_ptr();
  a.c.num_pages = k_pages.size(0);
  a.c.heads = k_pages.size(1);
  a.c.page_size = static_cast<int32_t>(std::min<int64_t>(k_pages.size(2), 0x7fffffff));
  a.c.D = k_pages.size(3);
  for (int i = 0; i < 3; ++i) a.c.k_strides[i] = outer_stride(k_pages, i), a.c.v_strides[i] = outer_stride(v_pages, i);
  if (!moves) {
    const bool codes = a.c.dtype == B200Q_E4M3;
    TORCH_CHECK_VALUE(codes == k_amax.has_value() && codes == v_amax.has_value(), op, ": pages of FP8 codes need k_amax and v_amax, other pages take none");
    if (codes) {
      TORCH_CHECK_VALUE(k_amax->numel() == v_amax->numel() && (k_amax->numel() == 1 || k_amax->numel() == a.c.heads), op,
                        ": k_amax and v_amax must hold one value or one per kv head (", a.c.heads, "), got ", k_amax->sizes(), " and ", v_amax->sizes());
      a.k_amax = f32_on(*k_amax, k_pages);
      a.v_amax = f32_on(*v_amax, k_pages);
      a.c.k_amax = a.k_amax.data_ptr<float>();
      a.c.v_amax = a.v_amax.data_ptr<float>();
      a.c.amax_numel = a.k_amax.numel();
    }
  }
  return a;
}

// scale 0 = 1 / sqrt(D)
float softmax_scale(double scale, int64_t D, const char* op) {
  TORCH_CHECK_VALUE(scale >= 0.0 && std::isfinite(scale), op, ": scale must be positive (0: 1 / sqrt(D)), got ", scale);
  return scale > 0.0 ? static_cast<float>(scale) : 1.0f / std::sqrt(static_cast<float>(D));
}

// dtype code of tokens that meet the cache
int token_dtype(const Tensor& x, const CacheArgs& a, const Tensor& pages, const char* op) {
  TORCH_CHECK_VALUE(x.scalar_type() == at::kHalf || x.scalar_type() == at::kBFloat16, op, " received an input of ", x.scalar_type(),
                    " type. Supported types: float16 | bfloat16");
  TORCH_CHECK_VALUE(a.c.dtype == B200Q_E4M3 || x.scalar_type() == pages.scalar_type(), op, ": the inputs (", x.scalar_type(), ") and the pages (",
                    pages.scalar_type(), ") must share a type unless the pages hold FP8 codes");
  TORCH_CHECK(x.device() == pages.device(), op, ": inputs and pages must be on one device");
  return x.scalar_type() == at::kHalf ? B200Q_F16 : B200Q_BF16;
}

void paged_append(const Tensor& k_in, const Tensor& v_in, const Tensor& k_pages, const Tensor& v_pages, const Tensor& table, const Tensor& lens,
                       const std::optional<Tensor>& cu_new, const std::optional<Tensor>& k_amax, const std::optional<Tensor>& v_amax) {
  const char* op = "b200_paged_append";
  c10::cuda::CUDAGuard guard(k_pages.device());
  CacheArgs a = cache_args(k_pages, v_pages, table, lens, k_amax, v_amax, false, op);
  const int dt = token_dtype(k_in, a, k_pages, op);
  TORCH_CHECK(k_in.dim() == 3 && k_in.sizes() == v_in.sizes() && k_in.scalar_type() == v_in.scalar_type() && v_in.device() == k_in.device() &&
                  k_in.size(1) == a.c.heads && k_in.size(2) == a.c.D,
              op, ": expected k and v [tokens, ", a.c.heads, ", ", a.c.D, "] of one type, got ", k_in.sizes(), " and ", v_in.sizes());
  const int32_t* cu = check_lens(cu_new, a.B + 1, k_pages, "cu_new", op);
  TORCH_CHECK(cu != nullptr || k_in.size(0) == a.B, op, ": without cu_new there is one token of every sequence (", a.B, "), got ", k_in.size(0));
  if (k_in.size(0) == 0) return;
  Tensor k = rows_of_16(k_in), v = rows_of_16(v_in);
  const int64_t strides[4] = {outer_stride(k, 0), outer_stride(k, 1), outer_stride(v, 0), outer_stride(v, 1)};
  must_be_ok(b200q_paged_append(k.data_ptr(), v.data_ptr(), dt, strides, k.size(0), cu, &a.c, a.table, a.table_stride, a.table_width, a.lens, a.B,
                                  stream_of_call()),
               "b200q_paged_append");
}

// A workspace whose head is zero, which the kernels leave as they found it: one per device and stream, kept for the life of the
// process.  A graph may be replayed on any stream beside that one, so a stream that is being captured gets one of the graph's own, which
// the graph clears where it first uses it; held here until the stream's next capture, then the graph's memory pool alone has it.
Tensor attention_workspace(const Tensor& like) {
  struct Kept {
    unsigned long long capture = 0;
    Tensor workspace;
  };
  static std::mutex mu;
  static auto* kept = new std::map<std::tuple<int, cudaStream_t, bool>, Kept>;      // not destroyed: the context may be gone by then
  const cudaStream_t stream = at::cuda::getCurrentCUDAStream().stream();
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  unsigned long long capture = 0;
  TORCH_CHECK(cudaStreamGetCaptureInfo(stream, &status, &capture) == cudaSuccess, "b200_paged_attention: cudaStreamGetCaptureInfo failed");
  const bool captured = status == cudaStreamCaptureStatusActive;
  if (!captured) capture = 0;
  std::lock_guard<std::mutex> lk(mu);
  Kept& k = (*kept)[{like.get_device(), stream, captured}];
  if (!k.workspace.defined() || k.capture != capture) {
    k.workspace = Tensor();
    k.workspace = at::empty({static_cast<int64_t>(b200q_paged_attention_workspace_bytes())}, like.options().dtype(at::kByte));
    k.workspace.narrow(0, 0, B200Q_PAGED_ATTENTION_ZERO_BYTES).zero_();
    k.capture = capture;
  }
  return k.workspace;
}

Tensor paged_attention(const Tensor& q_in, const Tensor& k_pages, const Tensor& v_pages, const Tensor& table, const Tensor& lens,
                            const std::optional<Tensor>& weights, const std::optional<Tensor>& k_amax, const std::optional<Tensor>& v_amax,
                            double scale, int64_t window, int64_t sinks) {
  const char* op = "b200_paged_attention";
  c10::cuda::CUDAGuard guard(k_pages.device());
  CacheArgs a = cache_args(k_pages, v_pages, table, lens, k_amax, v_amax, false, op);
  const int dt = token_dtype(q_in, a, k_pages, op);
  TORCH_CHECK(q_in.dim() == 3 && q_in.size(0) == a.B && q_in.size(2) == a.c.D, op, ": expected q [", a.B, ", query heads, ", a.c.D, "], got ", q_in.sizes());
  const int64_t Hq = q_in.size(1);
  TORCH_CHECK_VALUE(Hq > 0 && Hq % a.c.heads == 0, op, ": query heads (", Hq, ") must be a multiple of the kv heads (", a.c.heads, ")");
  TORCH_CHECK_VALUE(sinks >= 0, op, ": sinks must not be negative, got ", sinks);
  float* w = nullptr;
  int64_t wl = 0;
  Tensor scratch;
  if (weights.has_value()) {
    TORCH_CHECK(weights->device() == k_pages.device() && weights->scalar_type() == at::kFloat && weights->dim() == 3 && weights->size(0) == a.B &&
                    weights->size(1) == a.c.heads && weights->is_contiguous(),
                op, ": weights must be contiguous float32 [", a.B, ", ", a.c.heads, ", keys], got ", weights->sizes(), " of ", weights->scalar_type());
    w = weights->data_ptr<float>();
    wl = weights->size(2);
    int64_t keys = std::min<int64_t>(wl, a.table_width * a.c.page_size);       // logits of what a token can see
    if (window > 0 && window < keys && sinks < keys) keys = std::min(keys, window + sinks);
    scratch = at::empty({static_cast<int64_t>(b200q_paged_attention_scratch_bytes(a.B, Hq, keys))}, q_in.options().dtype(at::kByte));
  }
  Tensor out = at::empty(q_in.sizes(), q_in.options());
  if (a.B == 0) return out;
  Tensor q = rows_of_16(q_in);
  const int64_t strides[2] = {outer_stride(q, 0), outer_stride(q, 1)};
  Tensor ws = attention_workspace(q);
  const float sm = softmax_scale(scale, a.c.D, op);
  must_be_ok(b200q_paged_attention(q.data_ptr(), dt, strides, &a.c, a.table, a.table_stride, a.table_width, a.lens, a.B, Hq, sm, window, sinks,
                                     out.data_ptr(), w, wl, ws.data_ptr(), static_cast<size_t>(ws.numel()), w ? scratch.data_ptr() : nullptr,
                                     w ? static_cast<size_t>(scratch.numel()) : 0, stream_of_call()),
               "b200q_paged_attention");
  return out;
}

std::tuple<Tensor, Tensor, Tensor> paged_evict(const Tensor& k_pages, const Tensor& v_pages, const Tensor& table, const Tensor& lens,
                                                    const Tensor& weights, const Tensor& out_table, int64_t keep, int64_t recent, int64_t sinks) {
  const char* op = "b200_paged_evict";
  c10::cuda::CUDAGuard guard(k_pages.device());
  CacheArgs a = cache_args(k_pages, v_pages, table, lens, std::nullopt, std::nullopt, true, op);
  TORCH_CHECK(weights.device() == k_pages.device() && weights.scalar_type() == at::kFloat && weights.dim() == 3 && weights.size(0) == a.B &&
                  weights.size(1) == a.c.heads && weights.is_contiguous(),
              op, ": weights must be contiguous float32 [", a.B, ", ", a.c.heads, ", keys], got ", weights.sizes(), " of ", weights.scalar_type());
  check_table(out_table, k_pages, "out_table", op);
  TORCH_CHECK_VALUE(keep >= 0 && recent >= 0 && sinks >= 0 && recent + sinks <= keep, op, ": need recent + sinks <= keep, none negative, got ", recent, ", ",
                    sinks, ", ", keep);
  TORCH_CHECK_VALUE(keep <= weights.size(2) && out_table.size(0) == a.B && out_table.size(1) * k_pages.size(2) >= keep, op, ": weights [.., keys] and out_table ",
                    out_table.sizes(), " must have room for ", keep, " tokens of each of ", a.B, " sequences");
  Tensor kept = at::empty({a.B, a.c.heads, keep}, table.options()), new_lens = at::empty({a.B}, lens.options()), new_weights = at::empty_like(weights);
  must_be_ok(b200q_paged_evict(&a.c, a.table, a.table_stride, a.table_width, a.lens, weights.data_ptr<float>(), weights.size(2),
                                 out_table.data_ptr<int32_t>(), outer_stride(out_table, 0), out_table.size(1), a.B, keep, recent, sinks,
                                 kept.data_ptr<int32_t>(), new_lens.data_ptr<int32_t>(), new_weights.data_ptr<float>(), stream_of_call()),
               "b200q_paged_evict");
  return {kept, new_lens, new_weights};
}

Tensor like_queries(const Tensor& q) {
  // token-major queries (a slice of a projection) give a token-major result: the O projection reads it as it lies
  if (q.size(1) > 1 && q.size(2) > 1 && q.stride(1) < q.stride(2))
    return at::empty({q.size(0), q.size(2), q.size(1), q.size(3)}, q.options()).transpose(1, 2);
  return at::empty(q.sizes(), q.options());
}
Tensor window_attention(const Tensor& q_in, const Tensor& k_in, const Tensor& v_in, const std::optional<Tensor>& q_lens,
                             const std::optional<Tensor>& k_lens, double scale, int64_t window, int64_t sinks) {
  const char* op = "b200_window_attention";
  TORCH_CHECK(q_in.is_cuda(), op, ": b200q operates on CUDA tensors only; there is no CPU implementation");
  TORCH_CHECK_VALUE(q_in.scalar_type() == at::kHalf || q_in.scalar_type() == at::kBFloat16, op, " received an input of ", q_in.scalar_type(),
                    " type. Supported types: float16 | bfloat16");
  TORCH_CHECK(q_in.dim() == 4 && k_in.dim() == 4 && k_in.sizes() == v_in.sizes() && q_in.size(0) == k_in.size(0) && q_in.size(3) == k_in.size(3), op,
              ": expected q [B, Hq, Sq, D] and k, v [B, Hkv, Sk, D], got ", q_in.sizes(), ", ", k_in.sizes(), ", ", v_in.sizes());
  TORCH_CHECK(k_in.scalar_type() == q_in.scalar_type() && v_in.scalar_type() == q_in.scalar_type() && k_in.device() == q_in.device() &&
                  v_in.device() == q_in.device(),
              op, ": q, k, v must share a type and a device");
  const int64_t B = q_in.size(0), Hq = q_in.size(1), Sq = q_in.size(2), D = q_in.size(3), Hkv = k_in.size(1), Sk = k_in.size(2);
  TORCH_CHECK_VALUE(Hkv > 0 && Hq > 0 && Hq % Hkv == 0 && D % 16 == 0 && D > 0 && D <= 128, op,
                    ": need Hq % Hkv == 0 and a head dimension that is a multiple of 16 up to 128");
  TORCH_CHECK_VALUE(sinks >= 0, op, ": sinks must not be negative, got ", sinks);
  c10::cuda::CUDAGuard guard(q_in.device());
  const int32_t* nq = check_lens(q_lens, B, q_in, "q_lens", op);
  const int32_t* nk = check_lens(k_lens, B, q_in, "k_lens", op);
  Tensor out = like_queries(q_in);
  if (out.numel() == 0) return out;
  Tensor q = rows_apart(q_in), k = rows_apart(k_in), v = rows_apart(v_in);
  int64_t strides[9], out_strides[3];
  for (int i = 0; i < 3; ++i)
    strides[i] = outer_stride(q, i), strides[3 + i] = outer_stride(k, i), strides[6 + i] = outer_stride(v, i), out_strides[i] = outer_stride(out, i);
  const float sm = softmax_scale(scale, D, op);
  must_be_ok(b200q_window_attention(q.data_ptr(), k.data_ptr(), v.data_ptr(), q_in.scalar_type() == at::kHalf ? B200Q_F16 : B200Q_BF16, strides,
                                      out.data_ptr(), out_strides, nq, nk, B, Hq, Hkv, Sq, Sk, D, sm, window, sinks, stream_of_call()),
               "b200q_window_attention");
  return out;
}

}  // namespace
}  // namespace b200q_calls
