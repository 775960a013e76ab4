// What ranks the continuations of a prompt, from the logits of a step: log probability of a given token, entropy, the most likely tokens.
//
//   z_j = (x_j - max x) * scale,  S = sum_j exp(z_j),  log p_t = z_t - log S,  H = log S - sum_j exp(z_j) z_j / S
//
// Every logit is read once and takes part in one exponential and some ten other operations, so the memory binds the kernel, with the
// special-function unit not far behind for 16-bit logits (16 exponentials a clock, 12 logits a clock at the copy rate).
//
// A row is one CTA's, or, where there are few rows, a cluster's of up to eight.  A CTA takes 256 x 8 pieces of 16 bytes at once, into registers, and asks
// for the next ones when it is done with them: its loads and its work take turns, which the two or three other CTAs of its SM hide in part.  A thread follows its own
// maximum, sum S and sum of exp(z) z, so that for these nothing but the end of the row makes threads wait for one another.  The CTAs of a cluster write what they have found
// into the first one's shared memory.  What runs once a row stands in loops and functions: a short call waits for its code (50 KB of it: 10 us).
//
// The most likely tokens.  An element is a number of 64 bits, unlike any other of its row: the logit in the order of numbers (NaN above all), then
// the complement of its place, so that equal logits rank by the lower place.  Elements at or above a threshold go into a list, which is cut to the k
// largest, by counting, now and then; the last of them is the threshold from then on.  The first threshold, and one where too many pass: of the maxima
// of 64 groups of four threads the k-th largest has at least k elements at or above it, and elements at or above it lie in k groups only, a few
// more than k as a rule.  Where they are too many (the largest all in one group's hands), a threshold that leaves enough and not too many is
// searched by halving.
//
// Measured (us; the bytes at the copy rate): 2000 rows of 50001 bf16 logits, no list 44 (31); 200 rows of 100003 fp32 logits, most of them -inf, 8 of
// the list 29 (12): four and seven tiles to a CTA, with nothing on its way while one is worked on.  64 rows of 128000 bf16, 20 of the list 17 (2.5), two
// tiles to a CTA of a cluster of four, and 3 rows of 32000, 6 of the list 8.9 (0.03): the chain of a row's load, threshold, list, cut and exchange, and the code
// from memory.  CTAs that stay for the next row were slower.
// The difference taken first (scale x largest logit from 2^26 / log2 e on): 1.7, 1.4 and 1.2 times the time of the first three.
#include "common.cuh"
#include "ex2.cuh"
#include "softmax_tc.cuh"

namespace b200q {
namespace {

constexpr int kThreads = 256, kVectors = 8, kGroups = 64, kMostParts = 8;
constexpr int kMostTop = 64;
constexpr int kEdges = 14;                          // elements in front of and behind the aligned pieces
constexpr int kRoom = 2048 + kMostTop + kEdges + 2; // entries of a list: 256 pieces, all of them, behind what is there
constexpr int kLong = 192;                          // entries from which on it is cut

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
  __device__ static __forceinline__ float one(const char* p) { return __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(p)); }
  __device__ static __forceinline__ void widen(const uint4& v, float* f) { Elem<__nv_bfloat16>::unpack(v, f); }
  __device__ static __forceinline__ float most(const uint4& v) {          // a NaN where there is one
    const auto* h = reinterpret_cast<const __nv_bfloat162*>(&v);
    const __nv_bfloat162 m = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
    return __bfloat162float(__hmax_nan(m.x, m.y));
  }
  static constexpr float kFloor = -1e30f;              // no logit counts as less
  __device__ static __forceinline__ uint4 floored(uint4 v) {
    auto* h = reinterpret_cast<__nv_bfloat162*>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __hmax2(h[i], __float2bfloat162_rn(kFloor));
    return v;
  }
};
template <>
struct Logits<__half> {
  static constexpr int kPer = 8;
  __device__ static __forceinline__ float one(const char* p) { return __half2float(*reinterpret_cast<const __half*>(p)); }
  __device__ static __forceinline__ void widen(const uint4& v, float* f) { Elem<__half>::unpack(v, f); }
  __device__ static __forceinline__ float most(const uint4& v) {
    const auto* h = reinterpret_cast<const __half2*>(&v);
    const __half2 m = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
    return __half2float(__hmax_nan(m.x, m.y));
  }
  static constexpr float kFloor = -65504.0f;
  __device__ static __forceinline__ uint4 floored(uint4 v) {
    auto* h = reinterpret_cast<__half2*>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __hmax2(h[i], __float2half2_rn(kFloor));
    return v;
  }
};
template <>
struct Logits<float> {
  static constexpr int kPer = 4;
  __device__ static __forceinline__ float one(const char* p) { return *reinterpret_cast<const float*>(p); }
  __device__ static __forceinline__ void widen(const uint4& v, float* f) {
    f[0] = __uint_as_float(v.x), f[1] = __uint_as_float(v.y), f[2] = __uint_as_float(v.z), f[3] = __uint_as_float(v.w);
  }
  __device__ static __forceinline__ float most(const uint4& v) {
    return max_nan(max_nan(__uint_as_float(v.x), __uint_as_float(v.y)), max_nan(__uint_as_float(v.z), __uint_as_float(v.w)));
  }
  static constexpr float kFloor = -1e30f;
  __device__ static __forceinline__ uint4 floored(const uint4& v) {
    return make_uint4(__float_as_uint(fmaxf(__uint_as_float(v.x), kFloor)), __float_as_uint(fmaxf(__uint_as_float(v.y), kFloor)),
                      __float_as_uint(fmaxf(__uint_as_float(v.z), kFloor)), __float_as_uint(fmaxf(__uint_as_float(v.w), kFloor)));
  }
};

// 2^x and the natural logarithm's factor
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kLeast = -200.0f;                   // 2^-200 is zero here, and its product with what it belongs to too

// Maximum, sum of 2^y and sum of 2^y y with y = (x - maximum) * scale * log2 e.
struct Stats {
  float m, s, t;
};
// By the scale first: its product with log2 e may lie beyond the type.
__device__ __forceinline__ void refer(Stats& a, float m, float scale) {  // to a maximum that is not below its own
  const float d = fmaxf((a.m - m) * scale * kLog2e, kLeast), f = exp2_fast(d);
  if (a.s > 0.0f) a.t = f * fmaf(a.s, d, a.t), a.s *= f;
  a.m = m;
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

__device__ __forceinline__ void st_cluster(uint64_t* p, unsigned cta, uint64_t v) {
  asm volatile("st.shared::cluster.b64 [%0], %1;" ::"r"(ptx::mapa_u32(ptx::smem_u32(p), cta)), "l"(v) : "memory");
}
__device__ __forceinline__ void st_cluster(float* p, unsigned cta, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(ptx::mapa_u32(ptx::smem_u32(p), cta)), "f"(v) : "memory");
}
// Over the first `lanes` lanes of a warp, a power of two, in each of them: the maximum first, then two plain sums.
__device__ __forceinline__ Stats over_lanes(Stats a, float scale, int lanes) {
  float m = a.m;
#pragma unroll 1
  for (int d = lanes >> 1; d > 0; d >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, d));
  refer(a, m, scale);
#pragma unroll 1
  for (int d = lanes >> 1; d > 0; d >>= 1) a.s += __shfl_xor_sync(0xffffffffu, a.s, d), a.t += __shfl_xor_sync(0xffffffffu, a.t, d);
  return a;
}

struct Lists {
  uint64_t list[kRoom];                              // the row's largest so far
  uint64_t best[kMostParts][kMostTop];               // ranked, of each CTA
  uint64_t groups[kGroups];
  uint64_t threshold;
  int count;                                         // of the list; more than kRoom: there was no room
  float counts[kMostParts];                          // of `best`
};

// The `top` largest of the list, ranked, into best[0] of CTA `to` of the cluster (or this one's best[0], to < 0), all threads.
__device__ __noinline__ int rank_list(Lists& l, int n, int top, int part, int to) {
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const uint64_t it = l.list[i];
    int above = 0;
#pragma unroll 4
    for (int k = 0; k < n; ++k) above += l.list[k] > it;
    if (above < top) {
      if (to < 0) l.best[part][above] = it;
      else st_cluster(&l.best[part][above], to, it);
    }
  }
  return min(n, top);
}
// The list cut to its `top` largest; the last of them is the threshold from then on.
__device__ __noinline__ int cut(Lists& l, int n, int top) {
  n = rank_list(l, n, top, 0, -1);
  __syncthreads();
  const int tid = threadIdx.x;
  if (tid < n) l.list[tid] = l.best[0][tid];
  if (tid == 0) l.count = n;
  if (tid == 0 && n == top) l.threshold = l.best[0][n - 1];
  __syncthreads();
  return n;
}
// The k-th largest of the maxima of 64 groups of four threads, or 0 where there are fewer groups; all threads.
__device__ __noinline__ uint64_t of_groups(Lists& l, uint64_t most, int top) {
  const int tid = threadIdx.x;
#pragma unroll
  for (int d = 1; d < 4; d <<= 1) {
    const uint64_t o = __shfl_xor_sync(0xffffffffu, most, d);
    most = o > most ? o : most;
  }
  if ((tid & 3) == 0) l.groups[tid >> 2] = most;
  if (tid == 0) l.threshold = 0;
  __syncthreads();
  if (tid < kGroups) {
    const uint64_t g = l.groups[tid];
    int above = 0;
#pragma unroll 8
    for (int i = 0; i < kGroups; ++i) above += l.groups[i] > g;
    if (above == top - 1) l.threshold = g;             // several where groups are empty: zero, everything
  }
  __syncthreads();
  return l.threshold;
}
// The elements of a piece at or above the limit into the list; `from`: the limit's logit, a NaN lets all through to the second look.
template <typename T>
__device__ __noinline__ void list_piece(Lists& l, uint4 v, uint32_t place, uint64_t limit, float from) {
  float x[Logits<T>::kPer];
  Logits<T>::widen(v, x);
  unsigned near = 0;
#pragma unroll
  for (int e = 0; e < Logits<T>::kPer; ++e) near |= x[e] < from ? 0u : 1u << e;
#pragma unroll 1
  for (; near != 0; near &= near - 1) {
    const int e = __ffs(near) - 1;
    float of = x[0];
#pragma unroll
    for (int k = 1; k < Logits<T>::kPer; ++k) of = k == e ? x[k] : of;
    const uint64_t it = element(of, place + e);
    if (it < limit) continue;
    const int to = atomicAdd(&l.count, 1);
    if (to < kRoom) l.list[to] = it;
  }
}

// Sums of 2^y and of 2^y y over a piece, y = (x - base) scale log2 e.
template <typename T>
__device__ __noinline__ float2 sums_of(uint4 v, float base, float scale) {
  float f[Logits<T>::kPer];
  float2 sum = make_float2(0.0f, 0.0f);
  Logits<T>::widen(v, f);
#pragma unroll
  for (int e = 0; e < Logits<T>::kPer; ++e) {
    const float y = fmaxf((f[e] - base) * scale * kLog2e, kLeast), w = exp2_fast(y);
    sum.x += w, sum.y = fmaf(w, y, sum.y);
  }
  return sum;
}
template <int N>
__device__ __forceinline__ uint4 pick(const uint4 (&v)[N], int k) {
  uint4 of = v[0];
#pragma unroll
  for (int i = 1; i < N; ++i)
    if (k == i) of = v[i];
  return of;
}

constexpr int per_sm(bool top) { return top ? 3 : 4; }

template <typename T, bool TOP>
__global__ void __launch_bounds__(kThreads, per_sm(TOP)) token_scores_kernel(const __grid_constant__ ScoreParams p) {
  using E = Logits<T>;
  __shared__ float warps[3][kThreads / 32];
  __shared__ float sums[3][kMostParts];               // of the CTAs of a cluster
  __shared__ std::conditional_t<TOP, Lists, int> lists_;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int part = p.parts > 1 ? static_cast<int>(ptx::cluster_ctarank()) : 0;
  const float c = p.scale * kLog2e;
  if (p.parts > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  pdl_launch_dependents();

  // elements in front of the first 16-byte boundary, pieces of 16 bytes (v0 .. v1 - 1 are this CTA's), elements behind
  const int64_t row = p.parts > 1 ? blockIdx.x / p.parts : blockIdx.x;
  const char* const begin = p.logits + row * p.row_bytes;
  const int lead = min(static_cast<int>((16 - (reinterpret_cast<uintptr_t>(begin) & 15)) & 15) / static_cast<int>(sizeof(T)), p.vocabulary);
  const int vectors = (p.vocabulary - lead) / E::kPer, edges = p.vocabulary - vectors * E::kPer;
  const uint4* const pieces = reinterpret_cast<const uint4*>(begin + lead * sizeof(T)) + tid;
  const int v0 = static_cast<int>(static_cast<int64_t>(vectors) * part / p.parts), v1 = static_cast<int>(static_cast<int64_t>(vectors) * (part + 1) / p.parts);
  const int mine_to = v1 - tid;                        // this thread's pieces: v0 + k * 256 below it
  uint4 v[kVectors];
  auto load = [&](int at) {
#pragma unroll
    for (int k = 0; k < kVectors; ++k)
      if (at + k * kThreads < mine_to) v[k] = ld_nc_128(pieces + at + k * kThreads);
  };
  pdl_wait();
  load(v0);
  // the row's token and its logit, and the elements that no piece holds, behind the loads of the pieces
  float taken = 0.0f;
  bool is_taken = false;
  if (part == 0 && tid == kThreads - 1 && p.log_probs != nullptr) {
    const int64_t token = p.wide_tokens ? static_cast<const int64_t*>(p.tokens)[row] : static_cast<const int32_t*>(p.tokens)[row];
    is_taken = token >= 0 && token < p.vocabulary;
    if (is_taken) taken = E::one(begin + token * sizeof(T));
  }
  Stats mine{-INFINITY, 0.0f, 0.0f};
  int held = part == 0 ? edges : 0;        // entries of the list in front of this round's
  if (tid < held) {
    const int place = tid < lead ? tid : p.vocabulary - held + tid;
    const float x = E::one(begin + static_cast<int64_t>(place) * sizeof(T));
    mine = Stats{x, x == -INFINITY ? 0.0f : 1.0f, 0.0f};
    if constexpr (TOP) lists_.list[tid] = element(x, place);
  }
  if constexpr (TOP) {
    if (tid == 0) lists_.threshold = 0, lists_.count = held;
    __syncthreads();
  }
#pragma unroll 1
  for (int at = v0; at < v1; at += kThreads * kVectors) {
    // ----------------------------------------------------------- maximum and sums
    float top = -INFINITY, tops[kVectors];
#pragma unroll
    for (int k = 0; k < kVectors; ++k) {
      tops[k] = at + k * kThreads < mine_to ? E::most(v[k]) : -INFINITY;
      top = max_nan(top, tops[k]);
    }
    const float m = max_nan(mine.m, top);
    if (!(m == mine.m)) refer(mine, m, p.scale);
    const float base = m == -INFINITY ? 0.0f : m;
    // y = x c - base c in one step: base c is rounded once for all, and what that left out goes onto the sums behind.  It is up to half a unit in the last
    // place of base c: from 2^26 on more than 2, where 2^left and y + left would take their digits from the sums.  The difference first, then.
    const float shift = -base * c, left = fmaf(-base, c, -shift);
    float s[2] = {}, t[2] = {};
    // 0 times the -inf of a masked logit would be NaN: a floor under the logits, far enough below the maximum that its term is nothing, and not so far
    // that its product is beyond the type
    const float depth = (base - E::kFloor) * c;
    if (fabsf(shift) < 0x1p26f && base < 1e30f && depth > 150.0f && depth < 1e38f) {
#pragma unroll
      for (int k = 0; k < kVectors; ++k) {
        if (at + k * kThreads >= mine_to) break;
        float f[E::kPer];
        E::widen(E::floored(v[k]), f);
#pragma unroll
        for (int e = 0; e < E::kPer; ++e) {
          const float y = fmaf(f[e], c, shift), w = exp2_fast(y);
          s[e & 1] += w, t[e & 1] = fmaf(w, y, t[e & 1]);
        }
      }
      // sum of 2^(y + left) = 2^left s, and of 2^(y + left) (y + left) = 2^left (t + left s)
      const float s1 = s[0] + s[1], grown = exp2_fast(left);
      mine.s = fmaf(s1, grown, mine.s), mine.t = fmaf(fmaf(s1, left, t[0] + t[1]), grown, mine.t);
    } else {                                         // products beyond the type, and no distribution
#pragma unroll 1
      for (int k = 0; k < kVectors; ++k)
        if (at + k * kThreads < mine_to) {
          const float2 of = sums_of<T>(pick(v, k), base, p.scale);
          mine.s += of.x, mine.t += of.y;
        }
    }
    // ----------------------------------------------------------- the largest
    if constexpr (TOP) {
      Lists& l = lists_;
      auto place_of = [&](int k) { return static_cast<uint32_t>(lead + (at + k * kThreads + tid) * E::kPer); };
      uint64_t low = l.threshold, limit = low, high = ~uint64_t{0};
      bool grouped = false;
      int n = kRoom + 1;
#pragma unroll 1
      for (;;) {
        if (limit != 0 || grouped) {                  // all of the tile's elements at or above the limit into the list
          const float from = limit != 0 ? value_of(static_cast<uint32_t>(limit >> 32)) : __uint_as_float(0x7fffffffu);
          if (!(top < from)) {
#pragma unroll
            for (int k = 0; k < kVectors; ++k)
              if (at + k * kThreads < mine_to && !(tops[k] < from)) list_piece<T>(l, v[k], place_of(k), limit, from);
          }
          __syncthreads();
          n = l.count;
        }
        if (n <= kRoom && (!grouped || limit == low || n - held >= p.top)) break;
        // too many passed (or there was no threshold), or too few
        __syncthreads();
        if (tid == 0) l.count = held;
        if (!grouped) {
          grouped = true;
          int which = 0;                              // the first piece that holds the maximum
#pragma unroll
          for (int k = kVectors - 1; k >= 0; --k) which = tops[k] == top || tops[k] != tops[k] ? k : which;
          // no place of that piece lies behind its last one: the threshold admits the maximum wherever it is
          const uint64_t of = of_groups(l, at < mine_to ? element(top, place_of(which) + E::kPer - 1) : 0, p.top);
          low = limit = of > low ? of : low;
        } else {
          if (n > kRoom) low = limit;
          else high = limit;
          limit = low + (high - low) / 2;
        }
        __syncthreads();
      }
      if (n > kLong) n = cut(l, n, p.top);
      else if (tid == 0 && grouped) l.threshold = limit;
      held = n;
      __syncthreads();
    }
    if (at + kThreads * kVectors < v1) load(at + kThreads * kVectors);
  }
  // ------------------------------------------------------------- the CTA's threads, then the cluster's CTAs
  if (p.parts > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");      // the first CTA is there
  mine = over_lanes(mine, p.scale, 32);
  if (lane == 0) warps[0][warp] = mine.m, warps[1][warp] = mine.s, warps[2][warp] = mine.t;
  int listed = 0;
  if constexpr (TOP) listed = rank_list(lists_, held, p.top, part, p.parts > 1 ? 0 : -1);
  __syncthreads();
  const bool writes = warp == kThreads / 32 - 1;
  Stats all{-INFINITY, 0.0f, 0.0f};
  if (TOP || writes) {
    if (lane < kThreads / 32) all = Stats{warps[0][lane], warps[1][lane], warps[2][lane]};
    all = over_lanes(all, p.scale, kThreads / 32);
  }
  if (p.parts > 1) {
    if (writes && lane == 0) {
      st_cluster(&sums[0][part], 0, all.m), st_cluster(&sums[1][part], 0, all.s), st_cluster(&sums[2][part], 0, all.t);
      if constexpr (TOP) st_cluster(&lists_.counts[part], 0, static_cast<float>(listed));
    }
    ptx::cluster_sync();
    if (part > 0) return;                            // nothing of it is read from here on
    all = Stats{-INFINITY, 0.0f, 0.0f};
    if (lane < p.parts) all = Stats{sums[0][lane], sums[1][lane], sums[2][lane]};
    all = over_lanes(all, p.scale, kMostParts);
  }
  all.m = __shfl_sync(0xffffffffu, all.m, 0), all.s = __shfl_sync(0xffffffffu, all.s, 0), all.t = __shfl_sync(0xffffffffu, all.t, 0);
  // a row without a finite maximum has no distribution
  const float none = __uint_as_float(0x7fffffffu), log_sum = logf(all.s);
  const bool sound = fabsf(all.m) < INFINITY;
  if (tid == kThreads - 1) {
    if (p.entropy != nullptr) p.entropy[row] = sound ? fmaxf(log_sum - kLn2 * (all.t / all.s), 0.0f) : none;
    if (p.log_probs != nullptr) p.log_probs[row] = !is_taken ? 0.0f : (sound ? (taken - all.m) * p.scale - log_sum : none);      // 0: no token
  }
  if constexpr (TOP) {
    Lists& l = lists_;
    for (int k = tid; k < kMostTop * p.parts; k += kThreads) {
      const int i = k / kMostTop, at = k % kMostTop;
      if (at >= (p.parts > 1 ? static_cast<int>(l.counts[i]) : listed)) continue;
      const uint64_t it = l.best[i][at];
      int above = at;                                 // and those of the other lists, which are ranked too
#pragma unroll 1
      for (int o = 0; o < p.parts; ++o) {
        if (o == i) continue;
        int low = 0, high = static_cast<int>(l.counts[o]);
        while (low < high) {
          const int mid = (low + high) >> 1;
          if (l.best[o][mid] > it) low = mid + 1;
          else high = mid;
        }
        above += low;
      }
      if (above < p.top) {
        p.top_tokens[row * p.top + above] = static_cast<int32_t>(~static_cast<uint32_t>(it));
        p.top_log_probs[row * p.top + above] = sound ? (value_of(static_cast<uint32_t>(it >> 32)) - all.m) * p.scale - log_sum : none;
      }
    }
  }
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
  // As many CTAs to a row as the device holds at once, with some room (a cluster wants its places side by side), as long as each has a piece a thread.
  const int64_t places = static_cast<int64_t>(per_sm(top > 0)) * sm_count();
  for (p.parts = 1; p.parts < kMostParts; p.parts *= 2) {
    const int more = 2 * p.parts, percent = more == 2 ? 95 : (more == 4 ? 90 : 80);
    if (rows * more * 100 > places * percent || vocabulary * static_cast<int64_t>(size) / 16 < more * kThreads) break;
  }
  const auto st = static_cast<cudaStream_t>(stream);
  if (dtype == B200Q_BF16) return top > 0 ? launch_scores<__nv_bfloat16, true>(p, st) : launch_scores<__nv_bfloat16, false>(p, st);
  if (dtype == B200Q_F16) return top > 0 ? launch_scores<__half, true>(p, st) : launch_scores<__half, false>(p, st);
  return top > 0 ? launch_scores<float, true>(p, st) : launch_scores<float, false>(p, st);
}

}  // extern "C"
