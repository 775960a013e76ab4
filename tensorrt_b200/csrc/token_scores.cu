// What ranks the continuations of a prompt, from the logits of a step: log probability of a given token, entropy, the most likely tokens.
//
//   z_j = (x_j - max x) * scale,  S = sum_j exp(z_j),  log p_t = z_t - log S,  H = log S - sum_j exp(z_j) z_j / S
//
// Every logit is read once and takes part in one exponential and some ten other operations, so the memory binds the kernel, with the
// special-function unit not far behind for 16-bit logits (16 exponentials a clock, 12 logits a clock at the copy rate).
//
// A row is one CTA's, or, where there are few rows, a cluster's of up to eight.  A CTA takes 256 x 8 pieces of 16 bytes at once and keeps them in
// registers.  A thread follows its own maximum, sum S and sum of exp(z) z, so that nothing but the end of the row makes threads wait for one another.
//
// The most likely tokens.  An element is a number of 64 bits, unlike any other of its row: the logit in the order of numbers (NaN above all), then
// the complement of its place, so that equal logits rank by the lower place.  Of a tile the maxima of 64 groups of four threads are ranked; the
// k-th largest of them has at least k elements at or above it, and elements at or above it lie in k groups only.  Those, a few more than k as
// a rule, are put in a list, which is ranked by counting.  Where they are too many (the largest all in one thread's hands), a threshold that
// leaves enough and not too many is searched by halving.
#include "common.cuh"
#include "ex2.cuh"
#include "tcgen05.cuh"

namespace b200q {
namespace {

constexpr int kThreads = 256, kVectors = 8, kGroups = 64, kMostParts = 8;
constexpr int kMostTop = 64, kRoom = 2048;          // entries of a list; a tile of 256 pieces, all of it, has room
constexpr int kEdges = 14;                          // elements in front of and behind the aligned pieces

struct ScoreParams {
  const char* logits;
  int64_t row_bytes;
  const void* tokens;
  int wide_tokens;
  float* log_probs;
  float* entropy;
  float* top_log_probs;
  int32_t* top_tokens;
  int64_t rows;
  int vocabulary, top, parts;
  float scale;
};

template <typename T>
struct Logits;
template <>
struct Logits<__nv_bfloat16> {
  static constexpr int kPer = 8;
  static constexpr uint32_t kNone = 0xff80ff80u;
  __device__ static __forceinline__ float one(const char* p) { return __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(p)); }
  __device__ static __forceinline__ void widen(const uint4& v, float* f) { Elem<__nv_bfloat16>::unpack(v, f); }
};
template <>
struct Logits<__half> {
  static constexpr int kPer = 8;
  static constexpr uint32_t kNone = 0xfc00fc00u;
  __device__ static __forceinline__ float one(const char* p) { return __half2float(*reinterpret_cast<const __half*>(p)); }
  __device__ static __forceinline__ void widen(const uint4& v, float* f) { Elem<__half>::unpack(v, f); }
};
template <>
struct Logits<float> {
  static constexpr int kPer = 4;
  static constexpr uint32_t kNone = 0xff800000u;
  __device__ static __forceinline__ float one(const char* p) { return *reinterpret_cast<const float*>(p); }
  __device__ static __forceinline__ void widen(const uint4& v, float* f) {
    f[0] = __uint_as_float(v.x), f[1] = __uint_as_float(v.y), f[2] = __uint_as_float(v.z), f[3] = __uint_as_float(v.w);
  }
};

// 2^x and the natural logarithm's factor
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kLeast = -200.0f;                   // 2^-200 is zero here, and its product with what it belongs to too

__device__ __forceinline__ float exp2_of(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Maximum, sum of 2^y and sum of 2^y y with y = (x - maximum) * scale * log2 e.
struct Stats {
  float m, s, t;
};
__device__ __forceinline__ void refer(Stats& a, float m, float c) {      // to a maximum that is not below its own
  const float d = fmaxf((a.m - m) * c, kLeast), f = exp2_of(d);
  if (a.s > 0.0f) a.t = f * fmaf(a.s, d, a.t), a.s *= f;
  a.m = m;
}
__device__ __forceinline__ Stats both(Stats a, Stats b, float c) {
  const float m = max_nan(a.m, b.m);
  refer(a, m, c), refer(b, m, c);
  return Stats{m, a.s + b.s, a.t + b.t};
}

__device__ __forceinline__ uint32_t rank_of(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t b = __float_as_uint(x + 0.0f);                          // -0 is 0
  return b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t rank) {
  if (rank == 0xffffffffu) return __uint_as_float(0x7fffffffu);
  return __uint_as_float(rank & 0x80000000u ? rank ^ 0x80000000u : ~rank);
}
__device__ __forceinline__ uint64_t element(float x, uint32_t place) { return static_cast<uint64_t>(rank_of(x)) << 32 | static_cast<uint32_t>(~place); }

__device__ __forceinline__ float ld_shared_cluster(const float* p, unsigned cta) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(ptx::mapa_u32(ptx::smem_u32(p), cta)) : "memory");
  return v;
}
__device__ __forceinline__ int ld_shared_cluster(const int* p, unsigned cta) {
  int v;
  asm volatile("ld.shared::cluster.b32 %0, [%1];" : "=r"(v) : "r"(ptx::mapa_u32(ptx::smem_u32(p), cta)) : "memory");
  return v;
}
__device__ __forceinline__ uint64_t ld_shared_cluster(const uint64_t* p, unsigned cta) {
  uint64_t v;
  asm volatile("ld.shared::cluster.b64 %0, [%1];" : "=l"(v) : "r"(ptx::mapa_u32(ptx::smem_u32(p), cta)) : "memory");
  return v;
}

struct Lists {
  uint64_t found[kRoom];                             // of the tile
  uint64_t best[2][kMostTop + 2];                    // of the row so far, ranked
  uint64_t edges[kEdges + 2];
  uint64_t groups[kGroups];
  uint64_t threshold;
  int count;
};

template <typename T, bool TOP>
__global__ void __launch_bounds__(kThreads, TOP ? 2 : 3) token_scores_kernel(const __grid_constant__ ScoreParams p) {
  using E = Logits<T>;
  __shared__ float warps[3][kThreads / 32];
  __shared__ Stats whole;
  __shared__ int have_of;
  __shared__ std::conditional_t<TOP, Lists, int> lists_;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t row = blockIdx.x / p.parts;
  const int part = static_cast<int>(blockIdx.x - row * p.parts);
  const float c = p.scale * kLog2e;
  pdl_launch_dependents();
  pdl_wait();
  const char* const x0 = p.logits + row * p.row_bytes;
  const int lead = min(static_cast<int>((16 - (reinterpret_cast<uintptr_t>(x0) & 15)) & 15) / static_cast<int>(sizeof(T)), p.vocabulary);
  const int vectors = (p.vocabulary - lead) / E::kPer, tail = p.vocabulary - lead - vectors * E::kPer;
  const char* const body = x0 + lead * sizeof(T);
  const int v0 = static_cast<int>(static_cast<int64_t>(vectors) * part / p.parts), v1 = static_cast<int>(static_cast<int64_t>(vectors) * (part + 1) / p.parts);

  Stats mine{-INFINITY, 0.0f, 0.0f};
  int have = 0, side = 0, edges = 0;                   // entries of best[side], and of the edges that are not among them yet
  if (part == 0) {
    edges = lead + tail;
    if (tid < edges) {
      const int place = tid < lead ? tid : p.vocabulary - edges + tid;
      const float x = E::one(x0 + static_cast<int64_t>(place) * sizeof(T));
      mine = Stats{x, x == -INFINITY ? 0.0f : 1.0f, 0.0f};
      if constexpr (TOP) lists_.edges[tid] = element(x, place);
    }
  }
  if constexpr (TOP) {
    if (tid == 0) lists_.count = 0, lists_.threshold = 0;
    __syncthreads();
  }
  for (int at = v0; at < v1 || (TOP && edges > 0); at += kThreads * kVectors) {
    uint4 v[kVectors];
#pragma unroll
    for (int k = 0; k < kVectors; ++k) {
      const int i = at + k * kThreads + tid;
      v[k] = make_uint4(E::kNone, E::kNone, E::kNone, E::kNone);
      if (i < v1) v[k] = ld_nc_128(body + static_cast<int64_t>(i) * 16);
    }
    // ------------------------------------------------------------- maximum and sums
    float top = -INFINITY, tops[kVectors];
#pragma unroll
    for (int k = 0; k < kVectors; ++k) {
      float f[E::kPer];
      E::widen(v[k], f);
      tops[k] = f[0];
#pragma unroll
      for (int e = 1; e < E::kPer; ++e) tops[k] = max_nan(tops[k], f[e]);
      top = max_nan(top, tops[k]);
    }
    const float m = max_nan(mine.m, top);
    refer(mine, m, c);
    const float base = m == -INFINITY ? 0.0f : m;
    float s[2] = {}, t[2] = {};
#pragma unroll
    for (int k = 0; k < kVectors; ++k) {
      float f[E::kPer];
      E::widen(v[k], f);
#pragma unroll
      for (int e = 0; e < E::kPer; ++e) {
        const float y = fmaxf((f[e] - base) * c, kLeast), w = exp2_of(y);
        s[e & 1] += w, t[e & 1] = fmaf(w, y, t[e & 1]);
      }
    }
    mine.s += s[0] + s[1], mine.t += t[0] + t[1];
    // ------------------------------------------------------------- the largest
    if constexpr (TOP) {
      Lists& l = lists_;
      int which = 0;                                  // the first piece that holds the maximum
#pragma unroll
      for (int k = kVectors - 1; k >= 0; --k) which = rank_of(tops[k]) == rank_of(top) ? k : which;
      auto place_of = [&](int k) { return static_cast<uint32_t>(lead + (at + k * kThreads + tid) * E::kPer); };
      // no place of that piece lies behind its last one: the threshold admits the maximum wherever it is
      uint64_t most = at + tid < v1 ? element(top, place_of(which) + E::kPer - 1) : 0;
#pragma unroll
      for (int d = 1; d < 4; d <<= 1) {
        const uint64_t o = __shfl_xor_sync(0xffffffffu, most, d);
        most = o > most ? o : most;
      }
      if ((lane & 3) == 0) l.groups[tid >> 2] = most;
      __syncthreads();
      if (tid < kGroups) {
        const uint64_t g = l.groups[tid];
        int above = 0;
#pragma unroll 8
        for (int i = 0; i < kGroups; ++i) above += l.groups[i] > g;
        if (above == p.top - 1) l.threshold = g;      // several where groups are empty: zero, everything
      }
      __syncthreads();
      uint64_t threshold = l.threshold;
      const uint64_t last = have == p.top ? l.best[side][p.top - 1] : 0;
      threshold = last > threshold ? last : threshold;
      // All of the tile's elements at or above the threshold.  Where they are too many, the threshold is searched between it and what none reaches.
      int n;
      for (uint64_t low = threshold, high = ~uint64_t{0}, limit = threshold;;) {
        const float from = value_of(static_cast<uint32_t>(limit >> 32));
        if (limit == 0 || !(top < from)) {
#pragma unroll
          for (int k = 0; k < kVectors; ++k) {
            if (at + k * kThreads + tid >= v1) break;
            float x[E::kPer];
            E::widen(v[k], x);
#pragma unroll
            for (int e = 0; e < E::kPer; ++e) {
              if (limit != 0 && x[e] < from) continue;
              const uint64_t it = element(x[e], place_of(k) + e);
              if (it < limit) continue;
              const int to = atomicAdd(&l.count, 1);
              if (to < kRoom) l.found[to] = it;
            }
          }
        }
        __syncthreads();
        n = l.count;
        if (n > kRoom) low = limit;
        else if (limit != threshold && n < p.top) high = limit;
        else break;
        limit = low + (high - low) / 2;
        __syncthreads();
        if (tid == 0) l.count = 0;
        __syncthreads();
      }
      if (n + edges > 0) {
        auto entry = [&](int i) { return i < n ? l.found[i] : (i < n + have ? l.best[side][i - n] : l.edges[i - n - have]); };
        const int all = n + have + edges;
        for (int i = tid; i < all; i += kThreads) {
          const uint64_t it = entry(i);
          int above = 0;
          for (int k = 0; k < n; ++k) above += l.found[k] > it;
          for (int k = 0; k < have; ++k) above += l.best[side][k] > it;
          for (int k = 0; k < edges; ++k) above += l.edges[k] > it;
          if (above < p.top) l.best[side ^ 1][above] = it;
        }
        side ^= 1, have = min(all, p.top), edges = 0;
      }
      __syncthreads();
      if (tid == 0) l.count = 0, l.threshold = 0;     // seen behind the next tile's first barrier
    }
  }

  // ------------------------------------------------------------- the CTA's threads, then the cluster's CTAs
#pragma unroll
  for (int d = 16; d > 0; d >>= 1)
    mine = both(mine, Stats{__shfl_xor_sync(0xffffffffu, mine.m, d), __shfl_xor_sync(0xffffffffu, mine.s, d), __shfl_xor_sync(0xffffffffu, mine.t, d)}, c);
  if (lane == 0) warps[0][warp] = mine.m, warps[1][warp] = mine.s, warps[2][warp] = mine.t;
  __syncthreads();
  if (tid == 0) {
#pragma unroll
    for (int w = 1; w < kThreads / 32; ++w) mine = both(mine, Stats{warps[0][w], warps[1][w], warps[2][w]}, c);
    whole = mine;
    have_of = have | side << 16;
  }
  if (p.parts > 1) ptx::cluster_sync();
  else __syncthreads();
  if (part == 0) {
    Stats all = whole;
    for (int i = 1; i < p.parts; ++i)
      all = both(all, Stats{ld_shared_cluster(&whole.m, i), ld_shared_cluster(&whole.s, i), ld_shared_cluster(&whole.t, i)}, c);
    // a row without a finite maximum has no distribution
    const float none = __uint_as_float(0x7fffffffu), log_sum = logf(all.s);
    const bool sound = fabsf(all.m) < INFINITY;
    if (tid == 0) {
      if (p.entropy != nullptr) p.entropy[row] = sound ? fmaxf(log_sum - kLn2 * (all.t / all.s), 0.0f) : none;
      if (p.log_probs != nullptr) {
        const int64_t token = p.wide_tokens ? static_cast<const int64_t*>(p.tokens)[row] : static_cast<const int32_t*>(p.tokens)[row];
        float lp = 0.0f;                                // no token
        if (token >= 0 && token < p.vocabulary) lp = sound ? (E::one(x0 + token * sizeof(T)) - all.m) * p.scale - log_sum : none;
        p.log_probs[row] = lp;
      }
    }
    if constexpr (TOP) {
      Lists& l = lists_;
      int n = 0;
      for (int i = 0; i < p.parts; ++i) {               // ranked lists, one behind the other
        const int word = i == 0 ? have_of : ld_shared_cluster(&have_of, i), count = word & 0xffff;
        for (int k = tid; k < count; k += kThreads)
          l.found[n + k] = i == 0 ? l.best[word >> 16][k] : ld_shared_cluster(&l.best[word >> 16][k], i);
        n += count;
      }
      __syncthreads();
      for (int i = tid; i < n; i += kThreads) {
        const uint64_t it = l.found[i];
        int above = 0;
        for (int k = 0; k < n; ++k) above += l.found[k] > it;
        if (above < p.top) {
          p.top_tokens[row * p.top + above] = static_cast<int32_t>(~static_cast<uint32_t>(it));
          p.top_log_probs[row * p.top + above] = sound ? (value_of(static_cast<uint32_t>(it >> 32)) - all.m) * p.scale - log_sum : none;
        }
      }
    }
  }
  if (p.parts > 1) ptx::cluster_sync();               // nobody leaves while its part may still be read
}

template <typename T, bool TOP>
int launch_scores(const ScoreParams& p, cudaStream_t st) {
  auto kernel = token_scores_kernel<T, TOP>;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(p.rows * p.parts));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (p.parts > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = static_cast<unsigned>(p.parts), attr[n].val.clusterDim.y = 1, attr[n].val.clusterDim.z = 1;
    ++n;
  }
  if (pdl_enabled()) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  if (cudaLaunchKernelEx(&cfg, kernel, p) != cudaSuccess) return B200Q_ERR_CUDA;
  return check_launch();
}

}  // namespace
}  // namespace b200q

using namespace b200q;

extern "C" {

int b200q_token_log_probs(const void* logits, int dtype, int64_t rows, int64_t vocabulary, int64_t row_stride, const void* tokens, int token_bytes,
                          float scale, float* log_probs, float* entropy, int64_t top, float* top_log_probs, int32_t* top_tokens,
                          b200q_stream_t stream) {
  if (dtype != B200Q_F32 && dtype != B200Q_F16 && dtype != B200Q_BF16) return B200Q_ERR_INVALID;
  if (rows < 0 || rows > 0x0fffffffLL || vocabulary <= 0 || vocabulary > 0x3fffffffLL || row_stride < 0 || row_stride > (1LL << 46) || top < 0 ||
      top > kMostTop || top > vocabulary || !(scale > 0.0f) || !(scale < INFINITY))
    return B200Q_ERR_INVALID;
  if (rows == 0) return B200Q_OK;
  if (logits == nullptr || (tokens == nullptr) != (log_probs == nullptr) || (top > 0 && (top_log_probs == nullptr || top_tokens == nullptr)) ||
      (tokens != nullptr && token_bytes != 4 && token_bytes != 8))
    return B200Q_ERR_INVALID;
  const size_t size = dtype == B200Q_F32 ? 4 : 2;
  if (!aligned(logits, size) || (tokens != nullptr && !aligned(tokens, static_cast<size_t>(token_bytes)))) return B200Q_ERR_ALIGN;
  if (int rc = check_arch()) return rc;
  ScoreParams p{};
  p.logits = static_cast<const char*>(logits);
  p.row_bytes = row_stride * static_cast<int64_t>(size);
  p.tokens = tokens, p.wide_tokens = token_bytes == 8;
  p.log_probs = log_probs, p.entropy = entropy, p.top_log_probs = top_log_probs, p.top_tokens = top_tokens;
  p.rows = rows, p.vocabulary = static_cast<int>(vocabulary), p.top = static_cast<int>(top), p.scale = scale;
  // CTAs for all places of the device, four to an SM, as long as each has a round of pieces
  p.parts = 1;
  while (p.parts < kMostParts && rows * p.parts < 4 * sm_count() && vocabulary * static_cast<int64_t>(size) / 16 >= 2 * p.parts * kThreads) p.parts *= 2;
  const auto st = static_cast<cudaStream_t>(stream);
  if (dtype == B200Q_BF16) return top > 0 ? launch_scores<__nv_bfloat16, true>(p, st) : launch_scores<__nv_bfloat16, false>(p, st);
  if (dtype == B200Q_F16) return top > 0 ? launch_scores<__half, true>(p, st) : launch_scores<__half, false>(p, st);
  return top > 0 ? launch_scores<float, true>(p, st) : launch_scores<float, false>(p, st);
}

}  // extern "C"
