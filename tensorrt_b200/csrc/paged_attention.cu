// Attention of one new token of every sequence over its pages of the key-value cache.
#include "paged.cuh"

namespace b200q {
namespace {

using paged::Cache;

struct DecodeParams {
  Cache c;
  const char* q;
  int64_t q_batch, q_head;   // bytes
  void* out;
  float* weights;
  int64_t weights_len;
  int Hq, group;
  float scale;
  int64_t window, sinks;
};

__device__ __forceinline__ void load4(const __nv_bfloat16* p, float* f) {
  const uint2 u = *reinterpret_cast<const uint2*>(p);
  f[0] = __uint_as_float(u.x << 16), f[1] = __uint_as_float(u.x & 0xffff0000u);
  f[2] = __uint_as_float(u.y << 16), f[3] = __uint_as_float(u.y & 0xffff0000u);
}
__device__ __forceinline__ void load4(const __half* p, float* f) {
  const uint2 u = *reinterpret_cast<const uint2*>(p);
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&u.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&u.y));
  f[0] = a.x, f[1] = a.y, f[2] = b.x, f[3] = b.y;
}
__device__ __forceinline__ void load4(const uint8_t* p, float* f) {
  const uint32_t u = *reinterpret_cast<const uint32_t*>(p);
  const float2 a = e4m3x2_to_f32x2(u & 0xffffu), b = e4m3x2_to_f32x2(u >> 16);
  f[0] = a.x, f[1] = a.y, f[2] = b.x, f[3] = b.y;
}

// One CTA per sequence and kv head, one query head after the other; a warp takes every fourth key, a lane four elements of a row.
template <typename T, typename KV>
__global__ void __launch_bounds__(128) decode_kernel(const __grid_constant__ DecodeParams p) {
  __shared__ float sm[4], sl[4], so[4][paged::kMaxD];
  const int b = blockIdx.y, h = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int n = paged::cached_tokens(p.c, b, 0x7fffffff);
  const int first = p.window > 0 && n > p.window ? static_cast<int>(n - p.window) : 0;
  const int sinks = static_cast<int>(min(p.sinks, static_cast<int64_t>(first))), gap = first - sinks, seen = n - gap;
  const int32_t* line = p.c.table + b * p.c.table_stride;
  const bool mine = lane * 4 < p.c.D;
  const float ks = p.c.codes ? paged::head_scale(p.c.k_amax, p.c.amax_stride, h) : 1.0f;
  const float vs = p.c.codes ? paged::head_scale(p.c.v_amax, p.c.amax_stride, h) : 1.0f;
  for (int g = 0; g < p.group; ++g) {
    const int hq = h * p.group + g;
    float q[4] = {}, o[4] = {}, m = -INFINITY, l = 0.0f;
    bool any = false;
    if (mine) load4(reinterpret_cast<const T*>(p.q + b * p.q_batch + hq * p.q_head) + lane * 4, q);
    auto logit = [&](int i, int* page, int* row) {
      const int t = i < sinks ? i : i + gap;
      *page = paged::page_of(line, t, p.c), *row = t % p.c.page_size;
      float k[4] = {}, s = 0.0f;
      if (*page >= 0 && mine) load4(reinterpret_cast<const KV*>(paged::row_at(p.c.k, *page, h, *row)) + lane * 4, k);
      for (int e = 0; e < 4; ++e) s += q[e] * k[e];
      for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
      return s * (ks * p.scale);
    };
    for (int i = warp; i < seen; i += 4) {
      int page, row;
      const float s = logit(i, &page, &row);
      if (page < 0) continue;
      any = true;
      const float mn = fmaxf(m, s), safe = mn == -INFINITY ? 0.0f : mn, f = expf(m - safe), e = expf(s - safe);
      float v[4] = {};
      if (mine) load4(reinterpret_cast<const KV*>(paged::row_at(p.c.v, page, h, row)) + lane * 4, v);
      for (int x = 0; x < 4; ++x) o[x] = o[x] * f + e * v[x];
      l = l * f + e, m = mn;
    }
    if (lane == 0) sm[warp] = m, sl[warp] = l;
    for (int x = 0; x < 4; ++x) if (mine) so[warp][lane * 4 + x] = o[x];
    any = __syncthreads_or(any);
    float top = sm[0], total = 0.0f;
    for (int w = 1; w < 4; ++w) top = fmaxf(top, sm[w]);
    if (top == -INFINITY) top = 0.0f;
    for (int w = 0; w < 4; ++w) total += sl[w] * expf(sm[w] - top);
    for (int d = threadIdx.x; d < p.c.D; d += 128) {
      float acc = 0.0f;
      for (int w = 0; w < 4; ++w) acc += so[w][d] * expf(sm[w] - top);
      const float r = !any ? 0.0f : acc * vs / total;
      static_cast<T*>(p.out)[(static_cast<int64_t>(b) * p.Hq + hq) * p.c.D + d] = static_cast<T>(r);
    }
    if (p.weights != nullptr) {
      float* w = p.weights + (static_cast<int64_t>(b) * p.c.heads + h) * p.weights_len;
      for (int i = warp; i < seen; i += 4) {
        int page, row;
        const float s = logit(i, &page, &row);
        const int t = i < sinks ? i : i + gap;
        if (lane == 0 && page >= 0 && t < p.weights_len) w[t] += expf(s - top) / total;
      }
    }
    __syncthreads();
  }
}

}  // namespace
}  // namespace b200q

using namespace b200q;

extern "C" {

size_t b200q_paged_attention_workspace_bytes(void) { return 16; }
size_t b200q_paged_attention_scratch_bytes(int64_t, int64_t, int64_t) { return 16; }

int b200q_paged_attention(const void* q, int dtype, const int64_t* q_strides, const b200q_paged_cache* cache, const int32_t* block_table,
                          int64_t table_stride, int64_t table_width, const int32_t* lens, int64_t B, int64_t Hq, float scale,
                          int64_t window, int64_t sinks, void* out, float* weights, int64_t weights_len, void* workspace,
                          size_t workspace_bytes, void* scratch, size_t scratch_bytes, b200q_stream_t stream) {
  DecodeParams p{};
  if (int rc = paged::make_cache(&p.c, cache, dtype, block_table, table_stride, table_width, lens, B)) return rc;
  if (Hq <= 0 || Hq > 65535 || Hq % p.c.heads != 0 || sinks < 0 || !(scale == scale) || B > 65535) return B200Q_ERR_INVALID;
  if (B == 0) return B200Q_OK;
  if (q == nullptr || q_strides == nullptr || out == nullptr || (weights != nullptr && weights_len < 0)) return B200Q_ERR_INVALID;
  if (!aligned(q, 16) || !aligned(out, 16) || !paged::strides_ok(q_strides, 2, 8)) return B200Q_ERR_ALIGN;
  if (workspace == nullptr || workspace_bytes < b200q_paged_attention_workspace_bytes()) return B200Q_ERR_WORKSPACE;
  if (weights != nullptr && (scratch == nullptr || scratch_bytes < b200q_paged_attention_scratch_bytes(B, Hq, weights_len))) return B200Q_ERR_WORKSPACE;
  if (!aligned(workspace, 16) || !aligned(scratch, 16)) return B200Q_ERR_ALIGN;
  if (int rc = check_arch()) return rc;
  p.q = static_cast<const char*>(q);
  p.q_batch = q_strides[0] * 2, p.q_head = q_strides[1] * 2;
  p.out = out;
  p.weights = weights;
  p.weights_len = weights_len;
  p.Hq = static_cast<int>(Hq), p.group = static_cast<int>(Hq / p.c.heads);
  p.scale = scale;
  p.window = window, p.sinks = sinks;
  const dim3 grid(p.c.heads, static_cast<unsigned>(B));
  const auto st = static_cast<cudaStream_t>(stream);
  if (dtype == B200Q_BF16) {
    if (p.c.codes) decode_kernel<__nv_bfloat16, uint8_t><<<grid, 128, 0, st>>>(p); else decode_kernel<__nv_bfloat16, __nv_bfloat16><<<grid, 128, 0, st>>>(p);
  } else {
    if (p.c.codes) decode_kernel<__half, uint8_t><<<grid, 128, 0, st>>>(p); else decode_kernel<__half, __half><<<grid, 128, 0, st>>>(p);
  }
  return check_launch();
}

}  // extern "C"
