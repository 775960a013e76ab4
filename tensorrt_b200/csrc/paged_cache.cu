// Rows in and out of the paged key-value cache: append and evict.
#include "paged.cuh"

namespace b200q {
namespace {

using paged::Cache;

struct AppendParams {
  Cache c;
  const char* k;
  const char* v;
  int64_t k_token, k_head, v_token, v_head;   // bytes
  const int32_t* cu_new;
  int64_t T;
  int B;
};

__device__ __forceinline__ int ld_i32(const int32_t* p) {
  int v;
  asm volatile("ld.global.b32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}

// One thread per 16 elements of a row of K or V.
template <typename T, bool CODES>
__global__ void __launch_bounds__(256) append_kernel(const __grid_constant__ AppendParams p) {
  const int parts = p.c.D / 16, per_token = p.c.heads * parts;
  const int64_t at = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (at >= p.T * per_token * 2) return;
  const int part = static_cast<int>(at % parts);
  const int head = static_cast<int>(at / parts % p.c.heads);
  const bool is_v = (at / per_token) & 1;
  const int64_t t = at / per_token / 2;
  int b, i, fresh;
  if (p.cu_new == nullptr) {
    b = static_cast<int>(t), i = 0, fresh = 1;
  } else {
    int lo = 0, hi = p.B;                       // cu_new[lo] <= t < cu_new[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (ld_i32(p.cu_new + mid) <= t) lo = mid; else hi = mid;
    }
    b = lo;
    const int first = ld_i32(p.cu_new + lo);
    i = static_cast<int>(t - first), fresh = ld_i32(p.cu_new + lo + 1) - first;
  }
  const int64_t token = static_cast<int64_t>(ld_i32(p.c.lens + b)) - fresh + i;
  if (token < 0 || token >= p.c.capacity) return;
  const int page = paged::page_of(p.c.table + b * p.c.table_stride, static_cast<int>(token), p.c);
  if (page < 0) return;
  const char* src = is_v ? p.v + t * p.v_token + head * p.v_head : p.k + t * p.k_token + head * p.k_head;
  char* dst = paged::row_at(is_v ? p.c.v : p.c.k, page, head, static_cast<int>(token % p.c.page_size));
  Raw16<T, false> raw;
  raw.load(reinterpret_cast<const T*>(src) + part * 16);
  if constexpr (CODES) {
    const float scale = paged::head_scale(is_v ? p.c.v_amax : p.c.k_amax, p.c.amax_stride, head);
    *reinterpret_cast<uint4*>(dst + part * 16) =
        e4m3_of_16(raw, scale, __frcp_rn(scale), scale * 512.0f, b200q_div_fast_ok(scale));
  } else {
    uint4* d = reinterpret_cast<uint4*>(dst + part * 32);
    d[0] = make_uint4(raw.w[0].v[0], raw.w[0].v[1], raw.w[0].v[2], raw.w[0].v[3]);
    d[1] = make_uint4(raw.w[0].v[4], raw.w[0].v[5], raw.w[0].v[6], raw.w[0].v[7]);
  }
}

struct EvictParams {
  Cache c;
  const float* weights;
  int64_t L;
  const int32_t* out_table;
  int64_t out_stride;
  int keep, recent, sinks;
  int32_t* kept;
  int32_t* new_lens;
  float* new_weights;
  int row_bytes;
};

// Order of weights as unsigned numbers: larger weight, larger number; -0 and 0 are equal, NaN is -inf.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) w = -INFINITY;
  if (w == 0.0f) w = 0.0f;
  const uint32_t u = __float_as_uint(w);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// One CTA per sequence and kv head.  The smallest kept key is found bit by bit; then one pass in the order of the tokens.
__global__ void __launch_bounds__(256) evict_kernel(const __grid_constant__ EvictParams p) {
  __shared__ int counts[8];
  const int b = blockIdx.y, h = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int n = paged::cached_tokens(p.c, b, p.L), m = min(n, p.keep);
  const int64_t line = (static_cast<int64_t>(b) * p.c.heads + h);
  const float* w = p.weights + line * p.L;
  float* nw = p.new_weights + line * p.L;
  int32_t* kept = p.kept + line * p.keep;
  if (h == 0 && tid == 0) p.new_lens[b] = m;
  const int lo = min(p.sinks, n), hi = max(lo, n - p.recent);       // candidates: [lo, hi)
  const int want = m - lo - (n - hi);                               // of them stay
  auto total = [&](int v) {
    v = __reduce_add_sync(0xffffffffu, v);
    if (lane == 0) counts[warp] = v;
    __syncthreads();
    int s = 0;
    for (int i = 0; i < 8; ++i) s += counts[i];
    __syncthreads();
    return s;
  };
  uint32_t least = 0;                                               // the largest key that `want` candidates reach
  for (int bit = 31; bit >= 0 && want > 0; --bit) {
    const uint32_t probe = least | (1u << bit);
    int v = 0;
    for (int t = lo + tid; t < hi; t += 256) v += weight_key(w[t]) >= probe;
    if (total(v) >= want) least = probe;
  }
  int above = 0;
  for (int t = lo + tid; t < hi; t += 256) above += weight_key(w[t]) > least;
  const int equal = want - total(above);                            // of the candidates equal to it: the first ones
  __shared__ int warp_kept[8], warp_equal[8];
  int done = 0, done_equal = 0;
  for (int t0 = 0; t0 < n; t0 += 256) {
    const int t = t0 + tid;
    const bool fixed = t < n && (t < lo || t >= hi), inside = t < n && !fixed;
    const uint32_t key = inside ? weight_key(w[t]) : 0;
    const unsigned eq = __ballot_sync(0xffffffffu, inside && want > 0 && key == least);
    if (lane == 0) warp_equal[warp] = __popc(eq);
    __syncthreads();
    int rank = done_equal + __popc(eq & ((1u << lane) - 1));
    for (int i = 0; i < warp; ++i) rank += warp_equal[i];
    const bool stay = fixed || (inside && want > 0 && (key > least || (key == least && rank < equal)));
    const unsigned st = __ballot_sync(0xffffffffu, stay);
    if (lane == 0) warp_kept[warp] = __popc(st);
    __syncthreads();
    int at = done + __popc(st & ((1u << lane) - 1));
    for (int i = 0; i < warp; ++i) at += warp_kept[i];
    if (stay) kept[at] = t, nw[at] = w[t];
    for (int i = 0; i < 8; ++i) done += warp_kept[i], done_equal += warp_equal[i];
    __syncthreads();
  }
  for (int j = m + tid; j < p.keep; j += 256) kept[j] = -1;
  for (int64_t j = m + tid; j < p.L; j += 256) nw[j] = 0.0f;
  __syncthreads();
  const int pieces = p.row_bytes / 16;
  const int32_t* from = p.c.table + b * p.c.table_stride;
  const int32_t* to = p.out_table + b * p.out_stride;
  for (int64_t i = tid; i < static_cast<int64_t>(m) * pieces; i += 256) {
    const int j = static_cast<int>(i / pieces), piece = static_cast<int>(i % pieces) * 16, t = kept[j];
    const int sp = paged::page_of(from, t, p.c), dp = paged::page_of(to, j, p.c);
    if (sp < 0 || dp < 0) continue;
    const int sr = t % p.c.page_size, dr = j % p.c.page_size;
    *reinterpret_cast<uint4*>(paged::row_at(p.c.k, dp, h, dr) + piece) = *reinterpret_cast<const uint4*>(paged::row_at(p.c.k, sp, h, sr) + piece);
    *reinterpret_cast<uint4*>(paged::row_at(p.c.v, dp, h, dr) + piece) = *reinterpret_cast<const uint4*>(paged::row_at(p.c.v, sp, h, sr) + piece);
  }
}

}  // namespace
}  // namespace b200q

using namespace b200q;

extern "C" {

int b200q_paged_append(const void* k, const void* v, int dtype, const int64_t* strides, int64_t T, const int32_t* cu_new,
                       const b200q_paged_cache* cache, const int32_t* block_table, int64_t table_stride, int64_t table_width,
                       const int32_t* lens, int64_t B, b200q_stream_t stream) {
  AppendParams p{};
  if (int rc = paged::make_cache(&p.c, cache, dtype, block_table, table_stride, table_width, lens, B)) return rc;
  if (T < 0 || T > 0x7fffffffLL || (cu_new == nullptr && T != B) || (B == 0 && T != 0)) return B200Q_ERR_INVALID;
  if (T == 0 || table_width == 0) return B200Q_OK;
  if (k == nullptr || v == nullptr || strides == nullptr) return B200Q_ERR_INVALID;
  if (!aligned(k, 16) || !aligned(v, 16) || !paged::strides_ok(strides, 4, 8)) return B200Q_ERR_ALIGN;
  const int64_t threads = T * p.c.heads * (p.c.D / 16) * 2, blocks = (threads + 255) / 256;
  if (blocks > 0x7fffffffLL) return B200Q_ERR_INVALID;
  if (int rc = check_arch()) return rc;
  p.k = static_cast<const char*>(k);
  p.v = static_cast<const char*>(v);
  p.k_token = strides[0] * 2, p.k_head = strides[1] * 2, p.v_token = strides[2] * 2, p.v_head = strides[3] * 2;
  p.cu_new = cu_new;
  p.T = T;
  p.B = static_cast<int>(B);
  const auto st = static_cast<cudaStream_t>(stream);
  const auto n = static_cast<unsigned>(blocks);
  const bool half = dtype == B200Q_F16;
  if (p.c.codes) {
    if (half) append_kernel<__half, true><<<n, 256, 0, st>>>(p); else append_kernel<__nv_bfloat16, true><<<n, 256, 0, st>>>(p);
  } else {
    if (half) append_kernel<__half, false><<<n, 256, 0, st>>>(p); else append_kernel<__nv_bfloat16, false><<<n, 256, 0, st>>>(p);
  }
  return check_launch();
}

int b200q_paged_evict(const b200q_paged_cache* cache, const int32_t* block_table, int64_t table_stride, int64_t table_width,
                      const int32_t* lens, const float* weights, int64_t weights_len, const int32_t* out_table, int64_t out_stride,
                      int64_t out_width, int64_t B, int64_t keep, int64_t recent, int64_t sinks, int32_t* kept, int32_t* new_lens,
                      float* new_weights, b200q_stream_t stream) {
  EvictParams p{};
  if (int rc = paged::make_cache(&p.c, cache, -1, block_table, table_stride, table_width, lens, B)) return rc;
  if (keep < 0 || recent < 0 || sinks < 0 || recent + sinks > keep || weights_len < keep || weights_len > 0x7fffff00LL) return B200Q_ERR_INVALID;
  if (out_width < 0 || out_width > 0x7fffffffLL || out_stride < 0 || out_width * p.c.page_size < keep) return B200Q_ERR_INVALID;
  if (B > 65535) return B200Q_ERR_INVALID;
  if (B == 0) return B200Q_OK;
  if (new_lens == nullptr || (weights_len > 0 && (weights == nullptr || new_weights == nullptr || new_weights == weights))) return B200Q_ERR_INVALID;
  if (keep > 0 && (kept == nullptr || out_table == nullptr)) return B200Q_ERR_INVALID;
  if (int rc = check_arch()) return rc;
  p.weights = weights;
  p.L = weights_len;
  p.out_table = out_table;
  p.out_stride = out_stride;
  p.keep = static_cast<int>(keep), p.recent = static_cast<int>(recent), p.sinks = static_cast<int>(sinks);
  p.kept = kept;
  p.new_lens = new_lens;
  p.new_weights = new_weights;
  p.row_bytes = p.c.D * (p.c.codes ? 1 : 2);
  evict_kernel<<<dim3(p.c.heads, static_cast<unsigned>(B)), 256, 0, static_cast<cudaStream_t>(stream)>>>(p);
  return check_launch();
}

}  // extern "C"
