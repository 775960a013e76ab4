// Causal attention with a sliding window and sinks over contiguous K and V.
#include "common.cuh"

namespace b200q {
namespace {

struct WindowParams {
  const char* q;
  const char* k;
  const char* v;
  char* out;
  int64_t q_s[3], k_s[3], v_s[3], o_s[3];   // batch, head, row; elements
  const int32_t* q_lens;
  const int32_t* k_lens;
  int Hq, group, Sq, Sk, D;
  float scale;
  int64_t window, sinks;
};

__device__ __forceinline__ int length_of(const int32_t* lens, int b, int most) {
  if (lens == nullptr) return most;
  int n;
  asm volatile("ld.global.b32 %0, [%1];" : "=r"(n) : "l"(lens + b) : "memory");
  return min(max(n, 0), most);
}

template <typename T>
__device__ __forceinline__ void load4(const T* p, float* f) {
  const uint2 u = *reinterpret_cast<const uint2*>(p);
  if constexpr (std::is_same<T, __half>::value) {
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&u.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&u.y));
    f[0] = a.x, f[1] = a.y, f[2] = b.x, f[3] = b.y;
  } else {
    f[0] = __uint_as_float(u.x << 16), f[1] = __uint_as_float(u.x & 0xffff0000u);
    f[2] = __uint_as_float(u.y << 16), f[3] = __uint_as_float(u.y & 0xffff0000u);
  }
}

// One warp per query row, a lane four elements of a row, one key after the other.
template <typename T>
__global__ void __launch_bounds__(128) window_kernel(const __grid_constant__ WindowParams p) {
  const int lane = threadIdx.x & 31, row = blockIdx.x * 4 + (threadIdx.x >> 5), b = blockIdx.y / p.Hq, h = blockIdx.y % p.Hq;
  if (row >= p.Sq) return;
  const int nq = length_of(p.q_lens, b, p.Sq), nk = length_of(p.k_lens, b, p.Sk);
  const int at = row < nq ? row + nk - nq : -1;
  const bool mine = lane * 4 < p.D;
  const T* k = reinterpret_cast<const T*>(p.k) + b * p.k_s[0] + h / p.group * p.k_s[1] + lane * 4;
  const T* v = reinterpret_cast<const T*>(p.v) + b * p.v_s[0] + h / p.group * p.v_s[1] + lane * 4;
  float q[4] = {}, o[4] = {}, m = -INFINITY, l = 0.0f;
  if (mine) load4(reinterpret_cast<const T*>(p.q) + b * p.q_s[0] + h * p.q_s[1] + row * p.q_s[2] + lane * 4, q);
  for (int j = 0; j <= at; ++j) {
    if (p.window > 0 && j >= p.sinks && at - j >= p.window) {
      j = static_cast<int>(at - p.window);
      continue;
    }
    float x[4] = {}, y[4] = {}, s = 0.0f;
    if (mine) load4(k + j * p.k_s[2], x), load4(v + j * p.v_s[2], y);
    for (int e = 0; e < 4; ++e) s += q[e] * x[e];
    for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    s *= p.scale;
    const float mn = fmaxf(m, s), safe = mn == -INFINITY ? 0.0f : mn, f = expf(m - safe), e = expf(s - safe);
    for (int i = 0; i < 4; ++i) o[i] = o[i] * f + e * y[i];
    l = l * f + e, m = mn;
  }
  T* out = reinterpret_cast<T*>(p.out) + b * p.o_s[0] + h * p.o_s[1] + row * p.o_s[2] + lane * 4;
  if (mine)
    for (int i = 0; i < 4; ++i) out[i] = static_cast<T>(at < 0 ? 0.0f : o[i] / l);
}

}  // namespace
}  // namespace b200q

using namespace b200q;

extern "C" {

int b200q_window_attention(const void* q, const void* k, const void* v, int dtype, const int64_t* strides, void* out, const int64_t* out_strides,
                           const int32_t* q_lens, const int32_t* k_lens, int64_t B, int64_t Hq, int64_t Hkv, int64_t Sq, int64_t Sk, int64_t D,
                           float scale, int64_t window, int64_t sinks, b200q_stream_t stream) {
  if (dtype != B200Q_F16 && dtype != B200Q_BF16) return B200Q_ERR_INVALID;
  if (B < 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0 || Sq < 0 || Sk < 0 || Sq > 0x7fffff00LL || Sk > 0x7fffff00LL || D <= 0 || D > 128 ||
      D % 16 != 0 || sinks < 0 || !(scale == scale) || B > 65535 || B * Hq > 65535)
    return B200Q_ERR_INVALID;
  if (B == 0 || Sq == 0) return B200Q_OK;
  if (q == nullptr || out == nullptr || strides == nullptr || out_strides == nullptr || (Sk > 0 && (k == nullptr || v == nullptr))) return B200Q_ERR_INVALID;
  if (!aligned(q, 16) || !aligned(k, 16) || !aligned(v, 16) || !aligned(out, 16)) return B200Q_ERR_ALIGN;
  for (int i = 0; i < 9; ++i)
    if (strides[i] < 0 || strides[i] % 8 != 0) return B200Q_ERR_ALIGN;
  for (int i = 0; i < 3; ++i)
    if (out_strides[i] < 0 || out_strides[i] % 8 != 0) return B200Q_ERR_ALIGN;
  if (int rc = check_arch()) return rc;
  WindowParams p{};
  p.q = static_cast<const char*>(q), p.k = static_cast<const char*>(k), p.v = static_cast<const char*>(v), p.out = static_cast<char*>(out);
  for (int i = 0; i < 3; ++i) p.q_s[i] = strides[i], p.k_s[i] = strides[3 + i], p.v_s[i] = strides[6 + i], p.o_s[i] = out_strides[i];
  p.q_lens = q_lens, p.k_lens = k_lens;
  p.Hq = static_cast<int>(Hq), p.group = static_cast<int>(Hq / Hkv), p.Sq = static_cast<int>(Sq), p.Sk = static_cast<int>(Sk), p.D = static_cast<int>(D);
  p.scale = scale, p.window = window, p.sinks = sinks;
  const dim3 grid(static_cast<unsigned>((Sq + 3) / 4), static_cast<unsigned>(B * Hq));
  const auto st = static_cast<cudaStream_t>(stream);
  if (dtype == B200Q_BF16) window_kernel<__nv_bfloat16><<<grid, 128, 0, st>>>(p); else window_kernel<__half><<<grid, 128, 0, st>>>(p);
  return check_launch();
}

}  // extern "C"
