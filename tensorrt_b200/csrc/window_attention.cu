// Causal attention with a sliding window and sinks over contiguous K and V.
//
//   x_ij = (q_i . k_j) * scale over the keys j that row i sees: j <= p_i with j > p_i - window or j < sinks
//   out_i = sum_j exp(x_ij - m_i) v_j / sum_j exp(x_ij - m_i)
//
// 4 D operations a pair of row and key that see each other, and one exponential: for D = 128 the tensor cores and the special-function
// units of an SM need the same time (a tile of 128 rows and 128 keys is 1024 clocks of both), so the two have to run under each
// other all the time.
//
// A CTA holds two tiles of 128 query rows: of two heads that share their K and V where the group is even, of one head
// otherwise; with few queries a tile holds the rows of several heads.  One warp loads (TMA; Q once, then K and V tiles of 128
// keys through a ring), one issues tcgen05.mma (S = Q K^T into tensor memory, O += P V with P read from tensor memory), and four
// warps for each query tile run its softmax, one thread to a row, so that maximum and sum need no exchange: while one tile is in its softmax
// the tensor cores work on the other.  The one issuing warp takes the two tiles in turn, and that keeps them in opposite phase; with a warp
// each, or with P beside S so that the next scores could be made early (D 64), both softmaxes ran at once on the same
// special-function units and the tensor cores idled (2 x 32 x 8192 rows of 128, window 4096: 722 -> 816 us; of 64: 606 -> 757).  P takes the place
// of the S it came from.  Only key tiles that some row of the CTA sees are visited, and a query tile passes over those that none of
// its own rows sees; the mask, a word for 32 keys, is applied to tiles at an edge of it.  Where that is shorter a CTA holds one query tile, two to an
// SM, or the CTAs of a cluster share the keys of one (choose_shape).
//
// Measured (us a call, bf16): 2 x 32 / 8 heads, 8192 rows of 128, window 4096 with 4 sinks 722 at full clock, 820 call after call under the power
// cap (1143 and 1006 TFLOP/s; the library's dense product 1633 and 1382); 32 / 8 heads, 4096 rows, no window 126 (1090).  A key tile of both query tiles
// takes about 3300 clocks: 2100 of softmax, the rest the second half of P V, Q K^T (79 clocks a product of 64 ideal) and barriers.  Counters at the
// latter: tensor pipe 54 % active, special-function pipe 48 %, issue slots 43 %.  Two threads to a row 1085 us, scores read twice
// instead of held in registers 802, persistent CTAs in a fixed order 800; exponentials on the FMA pipe, of 16 pairs: none 715, 2 714, 4 733, 8 823.
// 8 sequences of up to 1500, 12 / 12 heads of 80, window 512 41.8.  What runs once or rarely in a CTA (rescaling, the way out) stays in loops: short
// calls pay for fetching the code, and registers spill less (43.9 with those unrolled).  A branch that took a tile of sinks alone as 32 keys cost
// more than it saved there (42.7; 8192 rows the same).
//
// The running maximum is followed lazily: O and the sum stay referred to an older maximum while the new one is at most 2^8 (fp16: 2^4)
// times larger, which 32-bit sums and the types' exponents hold; so the rescaling of O in tensor memory is
// rare.  Rounding: S, the softmax, O and the sums are 32-bit; P is rounded to 16 bits for the second product, an error of one rounding
// of each term, of the size of the result's own; in fp16 that holds for terms down to 2^-25 of the largest, and those below are off by up to
// 2^-36 of it (kRaise; with P of at most one, 2^-14 and 2^-25).
//
// A masked key has P = 0, and 0 times an infinity or a NaN of its V row would be a NaN: rows whose result is not finite are computed
// again, by one warp each, over the keys that they see.  That costs nothing where all is finite; where nothing is, a call takes hundreds of times
// as long, so padding behind ragged K and V is better cleared than left as it was allocated.
#include <cuda.h>

#include <atomic>

#include "common.cuh"
#include "ex2.cuh"
#include "gemm_host.cuh"
#include "tcgen05.cuh"

namespace b200q {
namespace {

constexpr int kTileRows = 128, kTileKeys = 128;
// log2 of how far the reference of the sums may lie below the maximum, and of the factor that P, the sums and O carry beside it: fp16 is a
// normal number from 2^-14 on only, so P is raised by 2^11 there and stays below 2^15.  bf16 has the range.
template <typename T>
constexpr float kLazy = std::is_same<T, __half>::value ? 4.0f : 8.0f;
template <typename T>
constexpr float kRaise = std::is_same<T, __half>::value ? 11.0f : 0.0f;
// The term of the reference is 2^kRaise, and the sum is no less, but for logits from 2^24 on: there the reference is rounded by a power of two or more,
// which cancels where the exponents of P hold it.  fp16's do not, so rows with a smaller sum (and those where P is infinite) are computed again.
template <typename T>
constexpr float kLeast = std::is_same<T, __half>::value ? 1024.0f : 0.0f;
constexpr int kPolyPairs = 2;   // of 16 pairs of exponentials: on the FMA pipe

// Division of numbers below 2^31 by one that the host knows: n / d = (mulhi(n, mul) + n) >> shift.
struct Divisor {
  uint32_t d, mul;
  int shift;
};
Divisor divisor(uint32_t d) {
  int shift = 0;
  while ((1ull << shift) < d) ++shift;
  return Divisor{d, static_cast<uint32_t>(((1ull << 32) * ((1ull << shift) - d)) / d + 1), shift};
}
__device__ __forceinline__ int divide(int n, const Divisor& v, int* rest) {
  const uint32_t q = (__umulhi(static_cast<uint32_t>(n), v.mul) + static_cast<uint32_t>(n)) >> v.shift;
  *rest = n - static_cast<int>(q * v.d);
  return static_cast<int>(q);
}

struct WindowParams {
  const char* q;
  const char* k;
  const char* v;
  char* out;
  int64_t q_s[3], k_s[3], v_s[3], o_s[3];   // batch, head, row; elements
  const int32_t* q_lens;
  const int32_t* k_lens;
  int Hq, Hkv, group, Sq, Sk, D;
  float scale;
  int window, sinks;         // window 0: none
  int rp, rp_log2, nh;       // rows of one head and heads in a query tile, rp * nh = 128
  Divisor by_block, by_split, by_unit, by_head;   // query blocks, splits, units, kv heads in the number of a CTA
  int pair_heads;            // the second query tile: the next heads (1) or the next rows (0)
  int units;                 // CTAs that share a kv head and rows
  int q_blocks;
  int splits;                // CTAs of a cluster that share an item's key tiles (one query tile a CTA)
  int B;
  int* status;
};

__device__ __forceinline__ void timed_out(int* status, int where) { atomicCAS(status, 0, where); }

__device__ __forceinline__ int length_of(const int32_t* lens, int b, int most) {
  if (lens == nullptr) return most;
  int n;
  asm volatile("ld.global.b32 %0, [%1];" : "=r"(n) : "l"(lens + b) : "memory");
  return min(max(n, 0), most);
}

// 4-D tiled load into this CTA's shared memory, completion on this CTA's own barrier.
__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* m, uint64_t* bar, int32_t x, int32_t y, int32_t z, int32_t w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(ptx::smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(m)), "r"(ptx::smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}
// kind::f16, fp32 accumulator; format 0 = fp16, 1 = bf16 for both operands; B K-major or N-major
__device__ __forceinline__ uint32_t idesc_16(int format, int m, int n, int b_n_major) {
  return (1u << 4) | (static_cast<uint32_t>(format) << 7) | (static_cast<uint32_t>(format) << 10) | (static_cast<uint32_t>(b_n_major) << 16) |
         (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float2 ld_cluster_f2(const float2* p, unsigned cta) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(ptx::mapa_u32(ptx::smem_u32(p), cta)) : "memory");
  return v;
}
__device__ __forceinline__ float4 ld_cluster_f4(const float* p, unsigned cta) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(ptx::mapa_u32(ptx::smem_u32(p), cta)) : "memory");
  return v;
}
// true in one lane of a converged warp
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r != 0;
}
// the n lowest bits, n of any size
__device__ __forceinline__ uint32_t low_bits(int n) { return n <= 0 ? 0u : (n >= 32 ? 0xffffffffu : (1u << n) - 1u); }
template <typename T>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  uint32_t r;
  if constexpr (std::is_same<T, __half>::value) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
template <typename T>
__device__ __forceinline__ void load4(const T* p, float* f) {
  uint2 u;
  asm volatile("ld.global.v2.b32 {%0, %1}, [%2];" : "=r"(u.x), "=r"(u.y) : "l"(p) : "memory");
  if constexpr (std::is_same<T, __half>::value) {
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&u.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&u.y));
    f[0] = a.x, f[1] = a.y, f[2] = b.x, f[3] = b.y;
  } else {
    f[0] = __uint_as_float(u.x << 16), f[1] = __uint_as_float(u.x & 0xffff0000u);
    f[2] = __uint_as_float(u.y << 16), f[3] = __uint_as_float(u.y & 0xffff0000u);
  }
}

// What a CTA works on: NQ query tiles.
template <int NQ>
struct Work {
  int b, kv_head, nq, off;                  // off: position of query 0
  int head[NQ], q0[NQ], lowest[NQ], highest[NQ];  // per query tile: first head, first query, positions of its rows (highest < 0: none)
  int sink_tiles, first, begin, tiles;      // key tiles 0 .. sink_tiles - 1, then first, first + 1, ..; of them `tiles` from the `begin`-th on
  __device__ __forceinline__ int tile(int j) const { return begin + j < sink_tiles ? begin + j : first + begin + j - sink_tiles; }
};
// Whether rows at positions lowest .. highest see a key of tile t.
__device__ __forceinline__ bool needs(const WindowParams& p, int lowest, int highest, int t) {
  const int k0 = t * kTileKeys;
  return k0 <= highest && (p.window == 0 || k0 + kTileKeys - 1 > lowest - p.window || k0 < p.sinks);
}

template <int NQ>
__device__ __forceinline__ Work<NQ> work_of(const WindowParams& p) {
  Work<NQ> w;
  int part, at, unit;
  const int item = divide(static_cast<int>(blockIdx.x), p.by_split, &part);
  const int block = p.q_blocks - 1 - divide(item, p.by_block, &at);        // the last queries first: they see most
  w.b = divide(divide(at, p.by_unit, &unit), p.by_head, &w.kv_head);
  w.nq = length_of(p.q_lens, w.b, p.Sq);
  const int nk = length_of(p.k_lens, w.b, p.Sk);
  w.off = nk - w.nq;
  int low = 0x7fffffff, high = -1;
#pragma unroll
  for (int s = 0; s < NQ; ++s) {
    w.head[s] = w.kv_head * p.group + (p.pair_heads ? NQ * unit + s : unit) * p.nh;
    w.q0[s] = p.pair_heads ? block * p.rp : (NQ * block + s) * p.rp;
    w.lowest[s] = max(w.q0[s] + w.off, 0);
    w.highest[s] = w.q0[s] < w.nq ? min(w.q0[s] + p.rp, w.nq) - 1 + w.off : -1;
    if (w.highest[s] >= 0) low = min(low, w.lowest[s]), high = max(high, w.highest[s]);
  }
  w.sink_tiles = w.first = w.begin = w.tiles = 0;
  if (high >= 0) {
    if (p.window > 0) {
      w.first = max(0, low - p.window + 1) / kTileKeys;
      w.sink_tiles = min((min(p.sinks, high + 1) + kTileKeys - 1) / kTileKeys, w.first);
    }
    w.tiles = w.sink_tiles + high / kTileKeys - w.first + 1;
  }
  const int all = w.tiles;
  w.begin = all * part / p.splits;
  w.tiles = all * (part + 1) / p.splits - w.begin;
  return w;
}

template <int DPAD, int NQ>
struct Layout {
  static constexpr int kBoxes = DPAD / 64, kBoxBytes = 128 * 128, kTileBytes = kBoxes * kBoxBytes;
  static constexpr int kPerSm = NQ == 1 ? 2 : 1;
  static constexpr int kStages = NQ == 2 ? (DPAD == 128 ? 5 : 8) : (DPAD == 128 ? 2 : 4);
  static constexpr int kBars = 2 * kStages + NQ + 4 * NQ + 1;
  static constexpr int kSmem = 1024 + (NQ + kStages) * kTileBytes + kBars * 8 + 16;
  static constexpr int kAlone = NQ == 1 ? 120 * 1024 : kSmem;
  static constexpr int kMmaWarp = 4 * NQ, kLoadWarp = kMmaWarp + 1, kThreads = 128 * (NQ + 1);
  static constexpr int kTmemCols = 256 * NQ;       // S of each query tile, then O of each
  // registers of a thread: 65536 / kPerSm for all; a softmax thread holds 128 scores
  static constexpr int kSoftmaxRegs = NQ == 2 ? 192 : 184, kOtherRegs = NQ == 2 ? 120 : 72;
};

// One row over the keys that it sees, by one warp, four elements a lane: for rows that a masked key spoiled.
template <typename T>
__device__ __noinline__ void row_again(const WindowParams& p, int b, int h, int row, int at) {
  const int lane = threadIdx.x & 31;
  const bool mine = lane * 4 < p.D;
  const T* k = reinterpret_cast<const T*>(p.k) + b * p.k_s[0] + h / p.group * p.k_s[1] + lane * 4;
  const T* v = reinterpret_cast<const T*>(p.v) + b * p.v_s[0] + h / p.group * p.v_s[1] + lane * 4;
  float q[4] = {}, o[4] = {}, m = -INFINITY, l = 0.0f;
  if (mine) load4(reinterpret_cast<const T*>(p.q) + b * p.q_s[0] + h * p.q_s[1] + row * p.q_s[2] + lane * 4, q);
  for (int j = 0; j <= at; ++j) {
    if (p.window > 0 && j >= p.sinks && at - j >= p.window) {
      j = at - p.window;
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
  if (mine) {
    const uint2 r = make_uint2(pack16<T>(o[0] / l, o[1] / l), pack16<T>(o[2] / l, o[3] / l));
    *reinterpret_cast<uint2*>(reinterpret_cast<T*>(p.out) + b * p.o_s[0] + h * p.o_s[1] + row * p.o_s[2] + lane * 4) = r;
  }
}

// The rows of this CTA from the parts of its cluster, by its first four warps: a warp takes 8 / SPLITS rows at once, so that eight loads are
// on their way together.
template <typename T, int DPAD, int SPLITS>
__device__ __noinline__ void join_rows(const WindowParams& p, const float* part, const float2* part_ml, int b, int head, int q0, int nq, int off) {
  constexpr int kRows = 8 / SPLITS, kPerWarp = kTileRows / SPLITS / 4;
  const int lane = threadIdx.x & 31, first = static_cast<int>(ptx::cluster_ctarank()) * (kTileRows / SPLITS) + (threadIdx.x >> 5) * kPerWarp;
  const int d = min(lane * 4, DPAD - 4);
  const float sl = fmaxf(p.scale * 1.4426950408889634f, 1e-30f);
  unsigned bad = 0;
#pragma unroll 1
  for (int r0 = 0; r0 < kPerWarp; r0 += kRows) {
    float2 ml[kRows][SPLITS];
    float4 o[kRows][SPLITS];
#pragma unroll
    for (int r = 0; r < kRows; ++r)
#pragma unroll
      for (int k = 0; k < SPLITS; ++k) {
        const int row = first + r0 + r;
        ml[r][k] = ld_cluster_f2(part_ml + row, k);
        o[r][k] = ld_cluster_f4(part + row * DPAD + (d ^ ((row & 7) * 4)), k);
      }
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const int row = first + r0 + r, h = head + (row >> p.rp_log2), i = q0 + (row & (p.rp - 1)), at = i < nq ? i + off : -1;
      float top = ml[r][0].x, l = 0.0f, y[4] = {};
      bool small = false;
#pragma unroll
      for (int k = 1; k < SPLITS; ++k) top = fmaxf(top, ml[r][k].x);
      const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll
      for (int k = 0; k < SPLITS; ++k) {
        const float f = exp2_fast((ml[r][k].x - base) * sl);
        l += ml[r][k].y * f;
        small |= ml[r][k].x != -INFINITY && ml[r][k].y < kLeast<T>;
        y[0] += o[r][k].x * f, y[1] += o[r][k].y * f, y[2] += o[r][k].z * f, y[3] += o[r][k].w * f;
      }
      const float f = 1.0f / l;
      float probe = 0.0f;
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] *= f, probe = fmaf(y[e], 0.0f, probe);
      if (__any_sync(0xffffffffu, small || (lane * 4 < p.D && probe != probe)) && at >= 0 && i < p.Sq) bad |= 1u << (r0 + r);
      if (lane * 4 < p.D && i < p.Sq) {
        uint2 u = make_uint2(0, 0);
        if (at >= 0) u = make_uint2(pack16<T>(y[0], y[1]), pack16<T>(y[2], y[3]));
        *reinterpret_cast<uint2*>(reinterpret_cast<T*>(p.out) + b * p.o_s[0] + h * p.o_s[1] + static_cast<int64_t>(i) * p.o_s[2] + lane * 4) = u;
      }
    }
  }
  for (; bad; bad &= bad - 1) {
    const int row = first + __ffs(bad) - 1, i = q0 + (row & (p.rp - 1));
    row_again<T>(p, b, head + (row >> p.rp_log2), i, i + off);
  }
}

template <typename T, int DPAD, int NQ>
__global__ void __launch_bounds__(Layout<DPAD, NQ>::kThreads, Layout<DPAD, NQ>::kPerSm)
window_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
              const __grid_constant__ WindowParams p) {
  using L = Layout<DPAD, NQ>;
  extern __shared__ char smem_raw[];
  char* const base = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t{1023});
  char* const sq = base;
  char* const ring = base + NQ * L::kTileBytes;
  uint64_t* const bars = reinterpret_cast<uint64_t*>(ring + L::kStages * L::kTileBytes);
  uint64_t* const full = bars;
  uint64_t* const empty = bars + L::kStages;
  uint64_t* const q_full = empty + L::kStages;
  uint64_t* const s_full = q_full + NQ;
  uint64_t* const p_full = s_full + NQ;
  uint64_t* const p_half = p_full + NQ;
  uint64_t* const o_full = p_half + NQ;
  uint64_t* const done = o_full + NQ;
  uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(done + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (warp == L::kMmaWarp) {
    ptx::tmem_alloc<1>(tmem_slot, L::kTmemCols);
    ptx::tmem_relinquish<1>();
  } else if (threadIdx.x == 0) {
    for (int i = 0; i < 2 * L::kStages + NQ; ++i) ptx::mbar_init(bars + i, 1);
    for (int s = 0; s < NQ; ++s) ptx::mbar_init(s_full + s, 1), ptx::mbar_init(p_full + s, 4), ptx::mbar_init(p_half + s, 4), ptx::mbar_init(o_full + s, 1);
    ptx::mbar_init(done, 1);
    ptx::fence_barrier_init();
    ptx::prefetch_tmap(&tq);
    ptx::prefetch_tmap(&tk);
    ptx::prefetch_tmap(&tv);
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_launch_dependents();
  pdl_wait();
  const Work<NQ> w = work_of<NQ>(p);

  if (warp >= L::kMmaWarp) {
    ptx::setmaxnreg_dec<L::kOtherRegs>();          // two query tiles: 128 x 120 + 256 x 192 = 384 x 168, one: 128 x (72 + 184) = 256 x 128, as launched
    if (warp == L::kLoadWarp) {
    // ------------------------------------------------------------- loads
    if (lane == 0 && w.tiles > 0) {
      auto load_q = [&](int s, int q0, int head) {
        ptx::mbar_arrive_expect_tx(q_full + s, L::kTileBytes);
        for (int x = 0; x < L::kBoxes; ++x) tma_load_4d(sq + s * L::kTileBytes + x * L::kBoxBytes, &tq, q_full + s, x * 64, q0, head, w.b);
      };
      load_q(0, w.q0[0], w.head[0]);
      int st = 0, issued = 0;
      uint32_t ph = 0;
      bool ok = true;
      for (int j = 0; j < w.tiles && ok; ++j) {
        const int row = w.tile(j) * kTileKeys;
        for (int kv = 0; kv < 2; ++kv) {
          if (!ptx::mbar_wait(empty + st, ph ^ 1u)) {
            timed_out(p.status, 80);
            ok = false;
            break;
          }
          ptx::mbar_arrive_expect_tx(full + st, L::kTileBytes);
          for (int x = 0; x < L::kBoxes; ++x)
            tma_load_4d(ring + st * L::kTileBytes + x * L::kBoxBytes, kv == 0 ? &tk : &tv, full + st, x * 64, row, w.kv_head, w.b);
          if (++issued == 1 && NQ == 2) load_q(1, w.q0[NQ - 1], w.head[NQ - 1]);      // the first product waits for the first query tile and the first keys
          if (++st == L::kStages) st = 0, ph ^= 1u;
        }
      }
      // no copy may be under way when the CTA ends, whatever became of its readers
      if (!ptx::mbar_wait(q_full, 0) || (NQ == 2 && issued > 0 && !ptx::mbar_wait(q_full + 1, 0))) timed_out(p.status, 81);
      for (int i = max(0, issued - L::kStages); i < issued; ++i)
        if (!ptx::mbar_wait(full + i % L::kStages, (i / L::kStages) & 1)) timed_out(p.status, 81);
    }
  } else if (warp == L::kMmaWarp) {
    // ------------------------------------------------------------- products
    // The warp walks the loop together, so that barriers, phases and descriptors stay in uniform registers; one lane issues.
    if (w.tiles > 0) {
      constexpr int kFormat = std::is_same<T, __half>::value ? 0 : 1;
      const uint32_t id_s = idesc_16(kFormat, 128, kTileKeys, 0), id_o = idesc_16(kFormat, 128, p.D, 1);
      const int steps = p.D / 16;
      // V as the second operand: rows of 64 elements of D, 8 keys to 1024 bytes, the next 64 elements a box further on
      constexpr uint32_t kHiV = (1024u >> 4) | (1u << 14) | (2u << 29);
      constexpr uint32_t kLeadV = (L::kBoxBytes >> 4) << 16;
      const uint32_t ring_lo = (ptx::smem_u32(ring) >> 4) & 0x3fffu, q_lo = ptx::desc_lo_sw128(ptx::smem_u32(sq));
      const bool leader = elect_one();
      bool ok = true;
      uint32_t p_phase[NQ] = {};
      bool waiting[NQ] = {}, begun[NQ] = {};   // a P that is to be multiplied; O holds something
      int stage = 0, v_stage = 0;                                    // of this tile's K; of the V of the tile before
      uint32_t phase = 0, v_phase = 0;
      for (int j = 0; j <= w.tiles && ok; ++j) {
        const bool more = j < w.tiles;
        const int t = more ? w.tile(j) : 0;
        // a stage is given back only once its copy has arrived, read or not
        if (more) ok = ptx::mbar_wait(full + stage, phase);
        if (j > 0) ok = ok && ptx::mbar_wait(full + v_stage, v_phase);
        if (!ok) {
          timed_out(p.status, 84);
          break;
        }
        ptx::tc_fence_after();
        const uint32_t v_lo = (ring_lo + v_stage * (L::kTileBytes >> 4)) | kLeadV, k_lo = (ring_lo + stage * (L::kTileBytes >> 4)) | (1u << 16);
#pragma unroll
        for (int s = 0; s < NQ; ++s) {
          if (waiting[s]) {
            // the first half of the keys as soon as it is there
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              ok = ok && ptx::mbar_wait((half == 0 ? p_half : p_full) + s, p_phase[s]);
              ptx::tc_fence_after();
              if (leader) {
#pragma unroll
                for (int k = 0; k < kTileKeys / 32; ++k)
                  mma_ts(tmem + (NQ + s) * 128, tmem + s * 128 + half * 32 + k * 8, ptx::desc_join(v_lo + (half * 4 + k) * (2048 >> 4), kHiV), id_o,
                         half > 0 || k > 0 ? 1u : (begun[s] ? 1u : 0u));
              }
              __syncwarp();
            }
            p_phase[s] ^= 1u;
            begun[s] = true;
            waiting[s] = false;
          }
          if (!more && leader) ptx::tc_commit<1>(o_full + s);
          __syncwarp();
          if (j == 0 && ok && !ptx::mbar_wait(q_full + s, 0)) ok = false;
          if (ok && more && needs(p, w.lowest[s], w.highest[s], t)) {
            if (j == 0) ptx::tc_fence_after();
            if (leader) {
#pragma unroll
              for (int k = 0; k < DPAD / 16; ++k) {
                const uint32_t at = ((k >> 2) * L::kBoxBytes + (k & 3) * 32) >> 4;
                if (k < steps)
                  mma_ss(tmem + s * 128, ptx::desc_join(q_lo + s * (L::kTileBytes >> 4) + at, ptx::kDescHiSw128), ptx::desc_join(k_lo + at, ptx::kDescHiSw128), id_s,
                         k > 0);
              }
              ptx::tc_commit<1>(s_full + s);
            }
            __syncwarp();
            waiting[s] = true;
          }
        }
        if (!ok) {
          timed_out(p.status, 83);
          break;
        }
        if (leader) {
          if (j > 0) ptx::tc_commit<1>(empty + v_stage);
          if (more) ptx::tc_commit<1>(empty + stage);
        }
        __syncwarp();
        v_stage = stage + 1, v_phase = phase;
        if (v_stage == L::kStages) v_stage = 0, v_phase ^= 1u;
        stage = v_stage + 1, phase = v_phase;
        if (stage == L::kStages) stage = 0, phase ^= 1u;
      }
      if (leader) ptx::tc_commit<1>(done);
      __syncwarp();
      if (!ptx::mbar_wait(done, 0)) timed_out(p.status, 85);
    }
    }
  } else {
    // ------------------------------------------------------------- softmax of query tile s, one thread to a row
    ptx::setmaxnreg_inc<L::kSoftmaxRegs>();
    const int s = NQ == 1 ? 0 : warp >> 2, r = threadIdx.x & 127;
    const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;     // this warp's 32 lanes of tensor memory
    const uint32_t ts = tmem + s * 128 + lanes, to = tmem + (NQ + s) * 128 + lanes;
    const int q0 = s ? w.q0[NQ - 1] : w.q0[0], lowest = s ? w.lowest[NQ - 1] : w.lowest[0], highest = s ? w.highest[NQ - 1] : w.highest[0];
    const int h = (s ? w.head[NQ - 1] : w.head[0]) + (r >> p.rp_log2), i = q0 + (r & (p.rp - 1));
    const int at = i < w.nq ? i + w.off : -1;                         // position; < 0: sees nothing
    const float sl = fmaxf(p.scale * 1.4426950408889634f, 1e-30f);    // 0 times a masked -inf would be NaN
    const uint64_t sl2 = pack2(sl, sl);
    float m = -INFINITY, l = 0.0f;
    bool ok = true, begun = false;
    uint32_t phase = 0;
    for (int j = 0; j < w.tiles && ok; ++j) {
      const int t = w.tile(j), k0 = t * kTileKeys;
      if (!needs(p, lowest, highest, t)) continue;
      ok = ptx::mbar_wait(s_full + s, phase);
      if (!ok) {
        timed_out(p.status, 86);
        break;
      }
      phase ^= 1u;
      ptx::tc_fence_after();
      uint32_t x[kTileKeys];
#pragma unroll
      for (int c = 0; c < 4; ++c) ptx::tmem_ld_32x32(ts + c * 32, x + c * 32);
      ptx::tmem_ld_wait();
      // no row of this tile that sees anything is at an edge; the others are not written
      const bool inside = k0 + kTileKeys - 1 <= lowest && (p.window == 0 || k0 > highest - p.window || k0 + kTileKeys <= p.sinks);
      if (!inside) {
        const int last = at - k0, first = p.window > 0 ? last - p.window : -1, sinks = p.sinks - k0;   // seen: c <= last with c > first or c < sinks
#pragma unroll
        for (int c = 0; c < kTileKeys; c += 32) {
          const uint32_t seen = low_bits(last + 1 - c) & (~low_bits(first + 1 - c) | low_bits(sinks - c));
#pragma unroll
          for (int e = 0; e < 32; ++e) x[c + e] = seen & (1u << e) ? x[c + e] : 0xff800000u;
        }
      }
      float top[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) top[c] = fmaxf(__uint_as_float(x[c]), __uint_as_float(x[4 + c]));
#pragma unroll
      for (int c = 8; c < kTileKeys; c += 8)
#pragma unroll
        for (int e = 0; e < 4; ++e) top[e] = fmaxf(top[e], fmaxf(__uint_as_float(x[c + e]), __uint_as_float(x[c + 4 + e])));
      const float mx = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
      if (!begun) {
        m = mx;
        begun = true;
      } else if (__any_sync(0xffffffffu, (mx - m) * sl > kLazy<T>)) {
        // O is complete up to the tile before: its product was issued in front of the S that has just arrived
        const float now = fmaxf(m, mx), f = now == -INFINITY ? 1.0f : exp2_fast((m - now) * sl);
        m = now;
        l *= f;
#pragma unroll 1
        for (int c = 0; c < DPAD / 32; ++c) {
          uint32_t o[32];
          ptx::tmem_ld_32x32(to + c * 32, o);
          ptx::tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
          ptx::tmem_st_32x32_x16(to + c * 32, o);
          ptx::tmem_st_32x32_x16(to + c * 32 + 16, o + 16);
        }
      }
      const float back = m == -INFINITY ? 0.0f : kRaise<T> - m * sl;
      const uint64_t back2 = pack2(back, back);
      uint64_t sum0 = 0, sum1 = 0;
#pragma unroll
      for (int c = 0; c < kTileKeys; c += 32) {
        uint32_t pk[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const uint64_t y = fma2(pack2(__uint_as_float(x[c + 2 * e]), __uint_as_float(x[c + 2 * e + 1])), sl2, back2);
          uint64_t v;
          if ((e + 1) * kPolyPairs / 16 != e * kPolyPairs / 16) {
            v = ex2_poly2(y);
          } else {
            const float2 a = unpack2(y);
            v = pack2(exp2_fast(a.x), exp2_fast(a.y));
          }
          if (e & 1) sum1 = add2(sum1, v); else sum0 = add2(sum0, v);
          const float2 a = unpack2(v);
          pk[e] = pack16<T>(a.x, a.y);
        }
        ptx::tmem_st_32x32_x16(ts + c / 2, pk);
        if (c == 32) {
          ptx::tmem_st_wait();
          ptx::tc_fence_before();
          __syncwarp();
          if (lane == 0) ptx::mbar_arrive(p_half + s);
        }
      }
      const float2 s0 = unpack2(sum0), s1 = unpack2(sum1);
      l += (s0.x + s0.y) + (s1.x + s1.y);
      ptx::tmem_st_wait();
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(p_full + s);
    }
    if (ok && w.tiles > 0 && !ptx::mbar_wait(o_full + s, 0)) {
      timed_out(p.status, 87);
      ok = false;
    }
    if (ok) {
      ptx::tc_fence_after();
      if (NQ == 1 && p.splits > 1) {
        // this CTA's part of the row: O, referred to m, over the ring (its last tile has been read); m and l over the queries
        float* const rows = reinterpret_cast<float*>(ring) + r * DPAD;
        reinterpret_cast<float2*>(sq)[r] = make_float2(m, l);
#pragma unroll 1
        for (int c = 0; c < DPAD / 32; ++c) {
          uint32_t o[32] = {};
          if (begun) {
            ptx::tmem_ld_32x32(to + c * 32, o);
            ptx::tmem_ld_wait();
          }
#pragma unroll
          for (int e = 0; e < 32; e += 4)            // pieces of 16 bytes turned by the row: 32 rows in one instruction
            *reinterpret_cast<uint4*>(rows + ((c * 32 + e) ^ ((r & 7) * 4))) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
        }
      } else {
      const float f = 1.0f / l;
      float probe = 0.0f;
      // Through the place of this tile's queries, which no product reads any more: a thread has a whole row, and 32 rows' pieces of 16 bytes
      // in one store instruction are 32 lines (5700 clocks for a tile; so 1000).
      constexpr int kRowBytes = DPAD * 2, kPieces = kRowBytes / 16;
      char* const rows = sq + s * L::kTileBytes;
#pragma unroll 1
      for (int c = 0; c < DPAD / 32; ++c) {
        uint32_t o[32];
        if (begun) {
          ptx::tmem_ld_32x32(to + c * 32, o);
          ptx::tmem_ld_wait();
        }
#pragma unroll
        for (int e = 0; e < 32; e += 8) {
          uint4 u = make_uint4(0, 0, 0, 0);
          if (at >= 0) {
            float y[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              y[k] = __uint_as_float(o[e + k]) * f;
              if (c * 32 + e < p.D) probe = fmaf(y[k], 0.0f, probe);
            }
            u = make_uint4(pack16<T>(y[0], y[1]), pack16<T>(y[2], y[3]), pack16<T>(y[4], y[5]), pack16<T>(y[6], y[7]));
          }
          *reinterpret_cast<uint4*>(rows + r * kRowBytes + (((c * 4 + e / 8) ^ (r & 7)) * 16)) = u;
        }
      }
      __syncwarp();
      const int64_t row_at = w.b * p.o_s[0] + h * p.o_s[1] + static_cast<int64_t>(i) * p.o_s[2];
#pragma unroll 4
      for (int k = 0; k < 32; k += 32 / kPieces) {
        const int from = k + lane / kPieces, piece = lane % kPieces;        // row of this warp
        const int64_t dst = __shfl_sync(0xffffffffu, row_at, from);
        const bool there = __shfl_sync(0xffffffffu, i, from) < p.Sq && piece * 8 < p.D;
        const int row = (r & ~31) + from;
        if (there)
          *reinterpret_cast<uint4*>(reinterpret_cast<T*>(p.out) + dst + piece * 8) =
              *reinterpret_cast<const uint4*>(rows + row * kRowBytes + ((piece ^ (row & 7)) * 16));
      }
      __syncwarp();
      for (unsigned bad = __ballot_sync(0xffffffffu, at >= 0 && (probe != probe || l < kLeast<T>)); bad; bad &= bad - 1) {
        const int who = __ffs(bad) - 1;
        row_again<T>(p, w.b, __shfl_sync(0xffffffffu, h, who), __shfl_sync(0xffffffffu, i, who), __shfl_sync(0xffffffffu, at, who));
      }
      }
    }
  }
  if (NQ == 1 && p.splits > 1) {
    // ------------------------------------------------------------- the parts of a cluster together: each CTA some of the rows, a warp a row
    __syncwarp();
    ptx::cluster_sync();
    if (warp < 4) {
      const float* const o = reinterpret_cast<const float*>(ring);
      const float2* const ml = reinterpret_cast<const float2*>(sq);
      if (p.splits == 2) join_rows<T, DPAD, 2>(p, o, ml, w.b, w.head[0], w.q0[0], w.nq, w.off);
      else if (p.splits == 4) join_rows<T, DPAD, 4>(p, o, ml, w.b, w.head[0], w.q0[0], w.nq, w.off);
      else join_rows<T, DPAD, 8>(p, o, ml, w.b, w.head[0], w.q0[0], w.nq, w.off);
    }
    __syncwarp();
    ptx::cluster_sync();                          // nobody leaves while its part may still be read
  }
  ptx::tc_fence_before();
  __syncthreads();
  if (warp == L::kMmaWarp) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc<1>(tmem, L::kTmemCols);
  }
}

// [D, rows, heads, batches] of 16-bit elements -> boxes of 64 x box_rows x box_heads, 128-byte swizzle, zeros out of bounds
int make_map(CUtensorMap* map, const void* base, int dtype, int64_t D, int64_t rows, int64_t heads, int64_t B, const int64_t* s, int box_rows, int box_heads) {
  gemm::EncodeTiledFn fn = gemm::encode_tiled();
  if (fn == nullptr) return B200Q_ERR_CUDA;
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(rows), static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(B)};
  // where there is one only, any stride will do
  const cuuint64_t strides[3] = {static_cast<cuuint64_t>(rows > 1 ? 2 * s[2] : 2 * D), static_cast<cuuint64_t>(heads > 1 ? 2 * s[1] : 2 * D),
                                 static_cast<cuuint64_t>(B > 1 ? 2 * s[0] : 2 * D)};
  const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(box_rows), static_cast<cuuint32_t>(box_heads), 1};
  const cuuint32_t unit[4] = {1, 1, 1, 1};
  const CUresult r = fn(map, dtype == B200Q_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base), dims, strides,
                        box, unit, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? B200Q_OK : B200Q_ERR_CUDA;
}

// Query tiles of a CTA and CTAs that share an item's keys.
//
// Two query tiles keep the tensor cores busy on their own and read K and V once for 256 rows; one query tile, two CTAs to an SM,
// hides start and end of a CTA behind its neighbour and wastes fewer rows and keys; splitting an item's keys over a cluster shortens the chain
// of its tiles where there are few items.  The costs in us are fitted to 190 shapes (1 to 8 sequences, groups of 1, 4 and 8, D 64 and
// 128, 61 to 4096 queries, 61 to 16000 keys, windows of 256, 1024 and none).  Of the form that is chosen they are 0.62 to 1.56 times what 79 other
// shapes take (median 1.2; most above one where a call is short), good enough to tell forms apart that differ by more than that.  They go by the
// tensors' sizes, since the lengths are on the device: ragged sequences are taken for whole ones.  One / two query tiles measured: 4096 queries without a window,
// 32 / 8 heads of 128 135 / 124, window 256 52 / 51, 12 / 12 heads of 64 x 8 sequences window 256 111 / 126; 300 queries of 4000 keys, 12 / 12
// heads x 8 84 / 116 (288 and 192 items on 296 and 148 places); 61 queries of 16000 keys, 32 / 8 heads 204 / 210, split over 8 CTAs 43;
// of 1999 keys behind a window of 1024 20.3 / 21.9, split 14.5.
struct Shape {
  int nq, splits;
};
int64_t blocks_of(const WindowParams& p, int nq) {
  const int rows = nq == 2 && p.group % (2 * p.nh) != 0 ? 2 * p.rp : p.rp;
  return (p.Sq + rows - 1) / rows;
}
Shape choose_shape(const WindowParams& p) {
  const int sms = sm_count();
  const bool narrow = p.D <= 64, pairs = p.group % (2 * p.nh) == 0;
  const double items1 = static_cast<double>(blocks_of(p, 1)) * p.B * p.Hkv * (p.group / p.nh);
  const double items2 = static_cast<double>(blocks_of(p, 2)) * p.B * p.Hkv * (p.group / (pairs ? 2 * p.nh : p.nh));
  // key tiles of a query tile, on average
  double keys = p.Sk - 0.5 * p.Sq;
  if (keys < 1.0) keys = 1.0;
  if (p.window > 0 && static_cast<double>(p.window) + p.rp + p.sinks < keys) keys = static_cast<double>(p.window) + p.rp + p.sinks;
  const double tiles1 = keys / kTileKeys + 0.5, tiles2 = tiles1 + (pairs ? 0.0 : static_cast<double>(p.rp) / kTileKeys);
  auto rounds = [](double x) { return x <= 1.0 ? 1.0 : (x <= 2.0 ? 2.0 : (x <= 3.0 ? 3.0 : x + 0.5)); };
  Shape best{2, 1};
  double least = rounds(items2 / sms) * ((narrow ? 7.7 : 8.0) + (narrow ? 1.4 : 1.75) * tiles2);
  for (int k = 1; k <= 8; k *= 2) {
    const double ctas = items1 * k;
    if (k > 1 && ctas > 1.75 * sms) break;       // a cluster that has to wait for its places gains nothing
    const double tile = ctas <= sms ? (narrow ? 1.4 : 1.6) : (narrow ? 1.55 : 2.1), join = k == 1 ? 0.0 : (k == 2 ? 5.5 : (k == 4 ? 3.6 : 2.8));
    const double mine = tiles1 / k < 1.0 ? 1.0 : tiles1 / k;
    const double cost = rounds(ctas / (2 * sms)) * ((narrow ? 6.3 : 7.5) + tile * mine) + join;
    if (cost < least) least = cost, best = Shape{1, k};
  }
  return best;
}

bool sizes_ok(int64_t B, int64_t Hq, int64_t Hkv, int64_t Sq, int64_t Sk, int64_t D, int64_t sinks) {
  return !(B < 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0 || Sq < 0 || Sk < 0 || Sq > 0x3fffff00LL || Sk > 0x3fffff00LL || D <= 0 || D > 128 ||
           D % 16 != 0 || sinks < 0 || B > 65535 || Hq > 0x7fffffffLL || B * Hq > 65535);
}

// The sizes of a call, what a query tile holds, and its form.
Shape plan(WindowParams* p, int64_t B, int64_t Hq, int64_t Hkv, int64_t Sq, int64_t Sk, int64_t D, int64_t window, int64_t sinks) {
  p->Hq = static_cast<int>(Hq), p->Hkv = static_cast<int>(Hkv), p->group = static_cast<int>(Hq / Hkv);
  p->Sq = static_cast<int>(Sq), p->Sk = static_cast<int>(Sk), p->D = static_cast<int>(D), p->B = static_cast<int>(B);
  p->window = window <= 0 || window >= Sk ? 0 : static_cast<int>(window);     // as wide as the keys: none
  p->sinks = static_cast<int>(sinks < Sk ? sinks : Sk);
  // few queries: the rows of several heads of a group in one tile
  p->rp = kTileRows, p->nh = 1;
  while (p->rp > 8 && Sq <= p->rp / 2 && p->group % (2 * p->nh) == 0) p->rp /= 2, p->nh *= 2;
  const Shape shape = choose_shape(*p);
  p->pair_heads = shape.nq == 2 && p->group % (2 * p->nh) == 0 ? 1 : 0;
  p->units = p->group / (p->pair_heads ? 2 * p->nh : p->nh);
  p->q_blocks = static_cast<int>(blocks_of(*p, shape.nq));
  p->splits = shape.splits;
  return shape;
}

template <typename T, int DPAD, int NQ>
int launch_window(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const WindowParams& p, unsigned ctas, cudaStream_t st) {
  using L = Layout<DPAD, NQ>;
  auto kernel = window_kernel<T, DPAD, NQ>;
  static std::atomic<bool> ready[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return B200Q_ERR_CUDA;
  if (dev < 0 || dev >= 64 || !ready[dev].load(std::memory_order_relaxed)) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kAlone) != cudaSuccess) return B200Q_ERR_CUDA;
    if (dev >= 0 && dev < 64) ready[dev].store(true, std::memory_order_relaxed);
  }
  // CTAs of a programmatic launch pile up on the SMs that the kernel in front left first: where one to an SM is enough, more shared
  // memory than two of them can have
  const int smem = NQ == 1 && p.splits == 1 && ctas <= static_cast<unsigned>(sm_count()) ? L::kAlone : L::kSmem;
  if (NQ == 2 || p.splits == 1) {
    if (launch_pdl(kernel, dim3(ctas), dim3(L::kThreads), smem, st, tq, tk, tv, p) != cudaSuccess) return B200Q_ERR_CUDA;
    return check_launch();
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(L::kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(p.splits), attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  if (cudaLaunchKernelEx(&cfg, kernel, tq, tk, tv, p) != cudaSuccess) return B200Q_ERR_CUDA;
  return check_launch();
}

template <typename T>
int launch_window_n(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const WindowParams& p, int nq, unsigned ctas, cudaStream_t st) {
  if (p.D <= 64) return nq == 2 ? launch_window<T, 64, 2>(tq, tk, tv, p, ctas, st) : launch_window<T, 64, 1>(tq, tk, tv, p, ctas, st);
  return nq == 2 ? launch_window<T, 128, 2>(tq, tk, tv, p, ctas, st) : launch_window<T, 128, 1>(tq, tk, tv, p, ctas, st);
}

}  // namespace
}  // namespace b200q

using namespace b200q;

extern "C" {

int b200q_window_attention_form(int64_t B, int64_t Hq, int64_t Hkv, int64_t Sq, int64_t Sk, int64_t D, int64_t window, int64_t sinks, int32_t form[3]) {
  if (!sizes_ok(B, Hq, Hkv, Sq, Sk, D, sinks) || B == 0 || Sq == 0 || form == nullptr) return B200Q_ERR_INVALID;
  if (int rc = check_arch()) return rc;
  WindowParams p{};
  const Shape shape = plan(&p, B, Hq, Hkv, Sq, Sk, D, window, sinks);
  form[0] = shape.nq, form[1] = shape.splits, form[2] = p.pair_heads;
  return B200Q_OK;
}

int b200q_window_attention(const void* q, const void* k, const void* v, int dtype, const int64_t* strides, void* out, const int64_t* out_strides,
                           const int32_t* q_lens, const int32_t* k_lens, int64_t B, int64_t Hq, int64_t Hkv, int64_t Sq, int64_t Sk, int64_t D,
                           float scale, int64_t window, int64_t sinks, b200q_stream_t stream) {
  if (dtype != B200Q_F16 && dtype != B200Q_BF16) return B200Q_ERR_INVALID;
  if (!sizes_ok(B, Hq, Hkv, Sq, Sk, D, sinks) || !(scale >= 0.0f)) return B200Q_ERR_INVALID;
  if (B == 0 || Sq == 0) return B200Q_OK;
  if (q == nullptr || out == nullptr || strides == nullptr || out_strides == nullptr || (Sk > 0 && (k == nullptr || v == nullptr))) return B200Q_ERR_INVALID;
  if (!aligned(q, 16) || !aligned(k, 16) || !aligned(v, 16) || !aligned(out, 16)) return B200Q_ERR_ALIGN;
  const int64_t sizes[9] = {B, Hq, Sq, B, Hkv, Sk, B, Hkv, Sk};
  for (int i = 0; i < 9; ++i)
    if (strides[i] < 0 || strides[i] % 8 != 0 || strides[i] >= (1LL << 39) || (sizes[i] > 1 && strides[i] == 0)) return B200Q_ERR_ALIGN;
  for (int i = 0; i < 3; ++i)
    if (out_strides[i] < 0 || out_strides[i] % 8 != 0) return B200Q_ERR_ALIGN;
  if (int rc = check_arch()) return rc;
  WindowParams p{};
  p.q = static_cast<const char*>(q), p.k = static_cast<const char*>(k), p.v = static_cast<const char*>(v), p.out = static_cast<char*>(out);
  for (int i = 0; i < 3; ++i) p.q_s[i] = strides[i], p.k_s[i] = strides[3 + i], p.v_s[i] = strides[6 + i], p.o_s[i] = out_strides[i];
  p.q_lens = q_lens, p.k_lens = k_lens;
  p.scale = scale;
  p.status = gemm::device_status_word();
  if (p.status == nullptr) return B200Q_ERR_CUDA;
  const Shape shape = plan(&p, B, Hq, Hkv, Sq, Sk, D, window, sinks);
  while ((1 << p.rp_log2) < p.rp) ++p.rp_log2;
  p.by_split = divisor(static_cast<uint32_t>(p.splits));
  p.by_block = divisor(static_cast<uint32_t>(B * Hkv * p.units));
  p.by_unit = divisor(static_cast<uint32_t>(p.units));
  p.by_head = divisor(static_cast<uint32_t>(Hkv));
  const int64_t ctas = static_cast<int64_t>(p.q_blocks) * B * Hkv * p.units * p.splits;
  if (ctas > 0x7fffffffLL) return B200Q_ERR_INVALID;
  CUtensorMap tq, tk, tv;
  if (int rc = make_map(&tq, q, dtype, D, Sq, Hq, B, strides, p.rp, p.nh)) return rc;
  // no keys: nothing is loaded, but the maps have to be valid
  if (int rc = make_map(&tk, Sk > 0 ? k : q, dtype, D, Sk > 0 ? Sk : Sq, Sk > 0 ? Hkv : Hq, B, Sk > 0 ? strides + 3 : strides, kTileKeys, 1)) return rc;
  if (int rc = make_map(&tv, Sk > 0 ? v : q, dtype, D, Sk > 0 ? Sk : Sq, Sk > 0 ? Hkv : Hq, B, Sk > 0 ? strides + 6 : strides, kTileKeys, 1)) return rc;
  const auto st = static_cast<cudaStream_t>(stream);
  const auto n = static_cast<unsigned>(ctas);
  return dtype == B200Q_BF16 ? launch_window_n<__nv_bfloat16>(tq, tk, tv, p, shape.nq, n, st) : launch_window_n<__half>(tq, tk, tv, p, shape.nq, n, st);
}

}  // extern "C"
