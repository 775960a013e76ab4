// Attention of one new token of every sequence, where groups of sequences share the pages of a prefix.
//
//   x_j = (q . k_j) * scale,  out = sum_j exp(x_j - m) v_j / sum_j exp(x_j - m),  m = max_j x_j
//
// The keys j < tokens of a group's prefix are the same for all of its sequences, so the rows of a group (its sequences times the query heads of a
// kv head) meet them as one matrix product, S = Q K^T and O = P V on tcgen05, and every K and V row is read once for up to 256 rows.  The keys behind
// the prefix belong to one sequence each: the kernel of paged_attention.cu attends to them, in parts.  A last kernel joins all parts of a row:
// with m = max_i m_i, sum = sum_i l_i 2^(m_i - m), out = sum_i o_i 2^(m_i - m) / sum.
//
// Work: shared_prefix.cuh, a CTA to an SM, pieces from the plan (found by the CTAs themselves they cost 3 us in front of every call).  Two times four
// warps run the softmax of a tile of 128 x 128 scores each, one thread to a row; one warp issues the products of both in turn, so that the tensor
// cores work on one while the other is in its softmax; one asks for K and V rows, which pages scatter, box by box (tensor maps); two copy queries
// (by the softmax's threads, through registers, that took 3 to 10 us in front of the first product: their code came from memory first); codes
// are widened to fp16, exactly, by four more warps in the place that they came to.  P takes the place of the scores that it came from in tensor memory.
//
// What bounds it.  Long prefixes: the softmax.  A step of 256 rows x 128 keys x 128 takes 2.4 us (1030 TFLOP/s): a warp needs 24 clocks for a pair
// of scores, alone on its quarter of the SM, whatever the order of its instructions, and the two tiles take turns with 1800 clocks of it each.
// Tried in vain, at 64 sequences x 8 heads behind 32768 tokens (80 us then, 74 now): one exponential in eight, in four, in two on the FMA pipe (80,
// 87, 97 us), the maximum in the addend of the scaling instead of a subtraction in front (81), two threads to a row (135: 104 registers spill).
// Short ones: what stands in front of the first product, some 4 us (launch, code from memory, queries, the first boxes), and the two kernels behind.
// 64 sequences behind 8192 tokens, 64 / 8 heads of 128: prefix 27 us, own keys 11, join 10, 42 in a row; 16 behind 100000 tokens of codes: 77, 15
// and 11, 99 in a row.
//
// Rounding: S, the softmax, O and the sums are 32-bit; P is rounded to 16 bits for the second product, an error of one rounding of each term,
// of the size of the result's own.  fp16 (fp16 pages and codes): P is raised by 2^11, so that holds for terms down to 2^-25 of the largest.  bf16
// queries in front of codes are scaled by a power of two into fp16's range, which loses nothing above 2^-38 of a row's largest.
#include <atomic>
#include <cfloat>

#include "gemm_host.cuh"
#include "shared_prefix.cuh"
#include "softmax_tc.cuh"

namespace b200q {
namespace {

using paged::Cache;
using paged::PlanLayout;
using paged::Prefix;
using paged::kPrefixKeys;
using paged::kPrefixRows;

struct PrefixParams {
  Cache c;
  Prefix x;
  int page_shift;            // log2 of the page size, or -1
  int box_rows, box_shift;   // rows of a page that a copy by tensor map takes, a power of two, and its logarithm
  const char* q;
  int64_t q_batch, q_head;   // bytes
  float scale;
  int* status;
};

// log2 of how far the reference of the sums may lie below the maximum, and of the factor that P, the sums and O carry beside it: fp16 is a normal
// number from 2^-14 on only, so P is raised by 2^11 there and stays below 2^15.  bf16 has the range.
template <bool HALF>
constexpr float kLazy = HALF ? 4.0f : 8.0f;
template <bool HALF>
constexpr float kRaise = HALF ? 11.0f : 0.0f;

template <int DPAD, bool CODES>
struct Layout {
  static constexpr int kBoxes = DPAD / 64, kBoxBytes = 128 * 128, kTileBytes = kBoxes * kBoxBytes;
  static constexpr int kTiles = DPAD == 128 ? 7 : 10;   // queries, then the ring; a second tile of queries takes a stage of it
  static constexpr int kMostStages = kTiles - 1;
  static constexpr int kBars = 3 * kMostStages + 12;
  static constexpr int kSlots = 16;                     // of tiles whose masks are kept
  static constexpr int kSmem = 1024 + kTiles * kTileBytes + kBars * 8 + 16 + kSlots * 16 + 16 + 512;
  static constexpr int kThreads = CODES ? 512 : 384, kMmaWarp = 8, kLoadWarp = 9, kQueryWarp = 10, kWidenWarp = 12, kWidenWarps = 4;
  static constexpr int kLoadWarps = kThreads / 32 - kLoadWarp;        // where threads load
  static constexpr int kTmemCols = 512;                 // the scores of both tiles, then O of both
  // registers at launch: 384 x 168 = 256 x 192 + 128 x 120, 512 x 128 = 256 x 192 + 256 x 64
  static constexpr int kSoftmaxRegs = 192, kOtherRegs = CODES ? 64 : 120;
};

// A wait whose long way stands in the code once: what a short call runs it also fetches, 40 KB of it in 5 us.
__device__ __noinline__ bool wait_on(uint64_t* bar, uint32_t parity, int* status, int where) {
  if (ptx::mbar_wait(bar, parity)) return true;
  timed_out(status, where);
  return false;
}
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, int* status, int where) {
  return ptx::mbar_try_wait(bar, parity) || wait_on(bar, parity, status, where);
}

// A CTA's way along its piece of the line, item after item.
struct Walk {
  int left;                  // steps from here to the end of the piece
  int item;                  // number of the item
  int g, h, block, step;     // the item, and the first step of this CTA's part of it
  int first, n, tokens, leader;   // of the group
  int tiles, rows;           // key tiles and rows of the group
  bool paired;
  __device__ __forceinline__ int steps() const { return paired ? tiles : (tiles + 1) >> 1; }
  __device__ __forceinline__ int blocks() const { return paired ? (rows + 255) >> 8 : (rows + 127) >> 7; }
  __device__ __forceinline__ int count() const { return min(left, steps() - step); }
  // first row of tile s, first key tile of step j of it; whether there are any
  __device__ __forceinline__ int row0(int s) const { return paired ? block * 256 + s * 128 : block * 128; }
  __device__ __forceinline__ int tile(int j, int s) const { return paired ? step + j : 2 * (step + j) + s; }
  __device__ __forceinline__ bool has(int j, int s) const { return s == 0 || (paired ? row0(1) < rows : tile(j, 1) < tiles); }
  // rows of half s of a part; where row r of it lies, or a place behind all parts
  __device__ __forceinline__ int half_rows(int s) const { return min(rows - row0(s), 128); }
  __device__ __forceinline__ unsigned place_of(const PrefixParams& p, int cta, int s, int r) const {
    if (item < 0 || item >= p.x.items || r >= half_rows(s)) return ~0u;
    const int whole = paired ? min(rows - row0(0), 256) : 2 * half_rows(0);
    return static_cast<unsigned>(paged::ld_index(p.x.plan + p.x.at.places + PlanLayout::kPlace * item) + cta * whole + s * half_rows(0) + r);
  }
  // key tiles of the first `count` steps that are loaded
  __device__ __forceinline__ int loaded(int count) const { return paired ? count : 2 * count - (has(count - 1, 1) ? 0 : 1); }
  // of the group: place of its first sequence, sequences, tokens, leader
  __device__ __forceinline__ void set_group(const PrefixParams& p, const int4& of) {
    first = min(max(of.x, 0), p.x.B), n = min(max(min(of.y, p.x.largest), 0), p.x.B - first);
    tokens = min(max(of.z, 0), 0x7fffff00), leader = of.w;
    tiles = (tokens + kPrefixKeys - 1) / kPrefixKeys, rows = n * p.x.group;
  }
  __device__ __forceinline__ void next(const PrefixParams& p) {
    left -= count() + paged::kItemSteps;
    step = 0;
    if (left <= 0) return;
    ++item;
    if (++block < blocks()) return;
    block = 0;
    if (++h < p.x.heads) return;
    h = 0;
    do {
      if (++g >= p.x.groups) {
        left = 0;
        return;
      }
      set_group(p, paged::ld_index4(p.x.plan + p.x.at.groups + PlanLayout::kGroup * g));
    } while (tiles == 0 || rows == 0);
  }
};

// The piece of CTA `cta`, empty where there is none.
__device__ __forceinline__ Walk find_start(const PrefixParams& p, int cta) {
  const int32_t* const at = p.x.plan + p.x.at.ctas + PlanLayout::kCta * cta;
  const int4 a = paged::ld_index4(at), b = paged::ld_index4(at + 4), of = paged::ld_index4(at + 8);
  Walk w;
  w.paired = paged::ld_index(p.x.plan + p.x.at.head) != 0;
  w.left = a.x, w.item = a.y, w.g = a.z, w.h = a.w, w.block = b.x, w.step = b.y;
  w.set_group(p, of);
  if (w.g < 0 || w.g >= p.x.groups || w.h < 0 || w.h >= p.x.heads || w.block < 0 || w.block >= w.blocks() || w.step < 0 || w.step >= w.steps()) w.left = 0;
  return w;
}

// A place in the ring of stages.
struct Ring {
  int stage, stages;
  uint32_t phase;
  __device__ __forceinline__ void advance(int n) {
    stage += n;
    if (stage >= stages) stage -= stages, phase ^= 1u;
  }
};

__device__ __forceinline__ void copy16(uint32_t dst, const char* src, int bytes) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
// one arrival of this thread once all of its copies so far are there
__device__ __forceinline__ void arrive_with_copies(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(ptx::smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void sts128(uint32_t a, uint4 v) {
  asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
// four codes -> four fp16 values, two and two
__device__ __forceinline__ void widen(uint32_t v, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}" : "=r"(lo), "=r"(hi) : "r"(v));
}
// Place of 16 bytes (piece c of a row) in a tile of 128 rows: boxes of 64 elements, 128-byte swizzle.
__device__ __forceinline__ uint32_t tile_at(int row, int c) {
  return static_cast<uint32_t>((c >> 3) * (128 * 128) + row * 128 + (((c & 7) ^ (row & 7)) * 16));
}

__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 r;
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(a) : "memory");
  return r;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
  uint2 r;
  asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(r.x), "=r"(r.y) : "r"(a) : "memory");
  return r;
}
// Rows of codes, each in the first bytes of 128, to rows of fp16 in their tile: a row's place takes its own codes' place, so nothing but the warp that
// widens it need have read it.  Rows without a key become zeros.  `first`: of the warp's 32 rows; `there`: a bit for each of them.
// Eight lanes to a row, 8 codes each of either half of it; odd rows take the halves in the other order, so that two rows meet no bank twice.
template <int DPAD>
__device__ __forceinline__ void widen_rows(uint32_t tile, int first, uint32_t there) {
  constexpr int kBatch = 4;
  const int lane = threadIdx.x & 31, c = lane & 7, turn = DPAD == 128 ? (lane >> 3) & 1 : 0;
  const uint32_t codes = tile + (DPAD == 128 ? 128 * 128 : 0);
#pragma unroll
  for (int r0 = 0; r0 < 32; r0 += 4 * kBatch) {
    uint2 v[kBatch][2];
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int i = r0 + k * 4 + (lane >> 3);
#pragma unroll
      for (int half = 0; half < DPAD / 64; ++half)
        v[k][half] = (there >> i) & 1 ? lds64(codes + (first + i) * 128 + (half ^ turn) * 64 + c * 8) : make_uint2(0, 0);
    }
    __syncwarp();
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int r = first + r0 + k * 4 + (lane >> 3);
#pragma unroll
      for (int half = 0; half < DPAD / 64; ++half) {
        uint4 a;
        widen(v[k][half].x, a.x, a.y), widen(v[k][half].y, a.z, a.w);
        sts128(tile + tile_at(r, (half ^ turn) * 8 + c), a);        // behind D: zeros, as they came
      }
    }
  }
}

// -inf in the place of the scores of keys that are not there, a bit for each key; all of a warp.  Rare: once an item, at holes in a table.
__device__ __forceinline__ void mask_scores(uint32_t scores, uint4 there) {
#pragma unroll 1
  for (int c = 0; c < 4; ++c) {
    const uint32_t word = c == 0 ? there.x : (c == 1 ? there.y : (c == 2 ? there.z : there.w));
    uint32_t x[32];
    ptx::tmem_ld_32x32(scores + c * 32, x);
    ptx::tmem_ld_wait();
#pragma unroll
    for (int e = 0; e < 32; ++e) x[e] = word & (1u << e) ? x[e] : 0xff800000u;
    ptx::tmem_st_32x32_x16(scores + c * 32, x);
    ptx::tmem_st_32x32_x16(scores + c * 32 + 16, x + 16);
  }
  ptx::tmem_st_wait();
}
// The first `left` of `rows` rows of a page into a tile of V, zeros behind, by one warp.
template <int DPAD>
__device__ __noinline__ void rows_by_hand(const PrefixParams& p, uint32_t tile, const char* src, int first, int rows, int left) {
  for (int k = threadIdx.x & 31; k < rows * (DPAD / 8); k += 32) {
    const int r = k / (DPAD / 8), c = k % (DPAD / 8);
    uint4 v = make_uint4(0, 0, 0, 0);
    if (r < left && c * 8 < p.c.D) v = ld_128(src + r * p.c.v.row + c * 16);
    sts128(tile + tile_at(first + r, c), v);
  }
  ptx::fence_proxy_async();
  __syncwarp();
}

// MAPS: K and V rows come by tensor maps, box_rows of a page at once (pages of a multiple of eight rows); otherwise by threads, 16 bytes each.
template <typename T, bool CODES, int DPAD, bool MAPS>
__global__ void __launch_bounds__(Layout<DPAD, CODES>::kThreads, 1)
prefix_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv, const __grid_constant__ PrefixParams p) {
  using L = Layout<DPAD, CODES>;
  constexpr bool kHalf = CODES || std::is_same<T, __half>::value;
  using E = std::conditional_t<kHalf, __half, __nv_bfloat16>;       // of the products
  extern __shared__ char smem_raw[];
  char* const base = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t{1023});
  char* const sq = base;
  uint64_t* const bars = reinterpret_cast<uint64_t*>(base + L::kTiles * L::kTileBytes);
  uint64_t* const full = bars;
  uint64_t* const empty = full + L::kMostStages;
  uint64_t* const raw = empty + L::kMostStages;          // codes are there
  uint64_t* const q_full = raw + L::kMostStages;
  uint64_t* const s_full = q_full + 2;
  uint64_t* const p_half = s_full + 2;
  uint64_t* const p_full = p_half + 2;
  uint64_t* const o_full = p_full + 2;
  uint64_t* const q_empty = o_full + 2;
  uint64_t* const done = q_empty + 1;
  uint4* const there = reinterpret_cast<uint4*>((reinterpret_cast<uintptr_t>(done + 1) + 15) & ~uintptr_t{15});   // which keys of a tile exist
  uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(there + L::kSlots);
  int8_t* const ups = reinterpret_cast<int8_t*>(tmem_slot + 4);      // [items by turns][tiles][rows] powers of two that queries in front of codes are scaled by
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (warp == L::kMmaWarp) {
    ptx::tmem_alloc<1>(tmem_slot, L::kTmemCols);
    ptx::tmem_relinquish<1>();
  } else if (threadIdx.x == 0) {
    // a stage is full when its boxes are there (codes: when four warps have widened them); or each loading thread's copies, and the mask is written
    for (int i = 0; i < L::kMostStages; ++i)
      ptx::mbar_init(full + i, MAPS ? (CODES ? L::kWidenWarps : 1) : 32 * L::kLoadWarps + 1), ptx::mbar_init(empty + i, 1), ptx::mbar_init(raw + i, 1);
    for (int s = 0; s < 2; ++s)
      ptx::mbar_init(q_full + s, 64), ptx::mbar_init(s_full + s, 2), ptx::mbar_init(p_half + s, 4), ptx::mbar_init(p_full + s, 4), ptx::mbar_init(o_full + s, 1);
    ptx::mbar_init(q_empty, 1), ptx::mbar_init(done, 1);
    ptx::fence_barrier_init();
    if constexpr (MAPS) {
      ptx::prefetch_tmap(&tk);
      ptx::prefetch_tmap(&tv);
    }
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int cta = static_cast<int>(blockIdx.x);

  if (warp >= L::kMmaWarp) {
    ptx::setmaxnreg_dec<L::kOtherRegs>();
    pdl_enter(true);         // the kernel behind starts once everything in front of this one has completed, and reads that without a wait
    Walk walk = find_start(p, cta);
    // paired: two tiles of queries, a stage less
    char* const ring_at = base + (walk.paired ? 2 : 1) * L::kTileBytes;
    Ring ring{0, walk.paired ? L::kMostStages - 1 : L::kMostStages, 0};
    // The item's queries, half of each tile's rows a warp: all copies under way at once, by a few instructions in a loop.
    bool q_turn = false;
    auto load_queries = [&](const Walk& walk) {
      constexpr bool kScaled = CODES && !std::is_same<T, __half>::value;
      constexpr int kLanes = DPAD / 8, kRowsAtOnce = 32 / kLanes;        // a row's pieces of 16 bytes by neighbouring lanes
      const int mine = (warp - L::kQueryWarp) * 64, c = lane % kLanes;
      if (!wait(q_empty, q_turn ? 0u : 1u, p.status, 89)) return false;
#pragma unroll 1
      for (int s = 0; s < 2; ++s) {
        if (s == 1 && (!walk.paired || !walk.has(0, 1))) break;
        int64_t off[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int at = walk.row0(s) + mine + u * 32 + lane, place = at / p.x.group;
          off[u] = -1;
          if (place < walk.n) {
            const int b = paged::ld_index(p.x.plan + p.x.at.order + walk.first + place);
            if (b >= 0 && b < p.x.B) off[u] = b * p.q_batch + (walk.h * p.x.group + at - place * p.x.group) * p.q_head;
          }
        }
        const uint32_t dst = ptx::smem_u32(sq) + s * L::kTileBytes;
#pragma unroll 4
        for (int i = 0; i < 64; i += kRowsAtOnce) {
          const int r = i + lane / kLanes;
          const int64_t from = __shfl_sync(0xffffffffu, i < 32 ? off[0] : off[1], r & 31);
          copy16(dst + tile_at(mine + r, c), p.q + (from < 0 ? 0 : from) + c * 16, from < 0 || c * 8 >= p.c.D ? 0 : 16);
        }
        if constexpr (kScaled) {
          // 2^(13 - exponent): the largest lands in [2^13, 2^14); zero, infinity and NaN stay as they are.  A lane has a row, so that no lane waits for
          // another (a row's pieces by neighbouring lanes took 6 us for two tiles).
          asm volatile("cp.async.wait_all;" ::: "memory");
          __syncwarp();
#pragma unroll 1
          for (int r = mine + lane; r < mine + 64; r += 32) {
            __nv_bfloat162 tops = __float2bfloat162_rn(0.0f);
#pragma unroll 4
            for (int k = 0; k < kLanes; ++k) {
              const uint4 v = lds128(dst + tile_at(r, k));
              const auto* h = reinterpret_cast<const __nv_bfloat162*>(&v);
#pragma unroll
              for (int u = 0; u < 4; ++u) tops = __hmax2(tops, __habs2(h[u]));
            }
            const float top = __bfloat162float(__hmax(tops.x, tops.y));
            const int e = static_cast<int>(__float_as_uint(top) >> 23), up = top != 0.0f && e < 255 ? min(max(140 - max(e, 1), -125), 124) : 0;
            const float f = __uint_as_float(static_cast<uint32_t>(up + 127) << 23);
#pragma unroll 4
            for (int k = 0; k < kLanes; ++k) {
              uint4 v = lds128(dst + tile_at(r, k));
              uint32_t* w = &v.x;
#pragma unroll
              for (int u = 0; u < 4; ++u) w[u] = pack16<__half>(__uint_as_float(w[u] << 16) * f, __uint_as_float(w[u] & 0xffff0000u) * f);
              sts128(dst + tile_at(r, k), v);
            }
            ups[(q_turn * 2 + s) * 128 + r] = static_cast<int8_t>(up);
          }
          ptx::fence_proxy_async();
          ptx::mbar_arrive(q_full + s);
        } else {
          arrive_with_copies(q_full + s);
        }
      }
      q_turn = !q_turn;
      return true;
    };
    if (MAPS && (warp == L::kQueryWarp || warp == L::kQueryWarp + 1)) {
      // ------------------------------------------------------------- queries
      for (bool ok = true; walk.left > 0 && ok; walk.next(p)) ok = load_queries(walk);
      asm volatile("cp.async.wait_all;" ::: "memory");       // no copy may be under way when the CTA ends
    } else if (MAPS && warp == L::kLoadWarp) {
      // ------------------------------------------------------------- loads: a lane asks for a box of each tile
      const int boxes = kPrefixKeys >> p.box_shift, rows = p.box_rows;
      uint64_t* const arrival = CODES ? raw : full;
      bool ok = true;
      int n = 0, issued = 0;                          // tiles so far; stages filled
      for (; walk.left > 0 && ok; walk.next(p)) {
        const int count = walk.count(), tokens = walk.tokens;
        const bool named = walk.leader >= 0 && walk.leader < p.x.B && tokens <= p.c.capacity;
        const int32_t* line = p.c.table + (named ? walk.leader : 0) * p.c.table_stride;
        int page[2], row[2];                          // of this lane's box, of each tile of a step
        auto find = [&](int j) {
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            if (s == 1 && walk.paired) break;
            const int t = walk.tile(j, s) * kPrefixKeys + lane * rows;
            page[s] = -1, row[s] = 0;
            if (named && lane < boxes && t < tokens) {
              const int at = p.page_shift >= 0 ? t >> p.page_shift : t / p.c.page_size;
              page[s] = paged::ld_index(line + at);
              row[s] = t - at * p.c.page_size;
            }
          }
        };
        find(0);
        for (int j = 0; j < count && ok; ++j) {
          const int tiles = walk.paired || !walk.has(j, 1) ? 1 : 2;
          int z[2], y[2], held[2];
          unsigned cut[2];
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            if (s >= tiles) break;
            const int t = walk.tile(j, s) * kPrefixKeys + lane * rows;
            const bool exists = static_cast<unsigned>(page[s]) < static_cast<unsigned>(p.c.num_pages);
            held[s] = exists ? min(rows, tokens - t) : 0;
            z[s] = exists ? page[s] : p.c.num_pages, y[s] = row[s];        // behind the last page: zeros
            // a box that the prefix ends in: what lies behind may be anything, and 0 times a NaN of V would be one
            cut[s] = __ballot_sync(0xffffffffu, held[s] > 0 && held[s] < rows);
            uint4 words = make_uint4(~0u, ~0u, ~0u, ~0u);
            if (!__all_sync(0xffffffffu, lane >= boxes || held[s] == rows)) {
              uint32_t w[4];
#pragma unroll
              for (int u = 0; u < 4; ++u) {
                const int key = u * 32 + lane;
                w[u] = __ballot_sync(0xffffffffu, (key & (rows - 1)) < __shfl_sync(0xffffffffu, held[s], key >> p.box_shift));
              }
              words = make_uint4(w[0], w[1], w[2], w[3]);
            }
            if (lane == 0) there[(n + s) % L::kSlots] = words;
          }
          n += tiles;
          if (j + 1 < count) find(j + 1);
#pragma unroll 1
          for (int i = 0; i < 2 * tiles; ++i) {       // K of the step's tiles, then V
            const int kv = i >= tiles, s = kv ? i - tiles : i;
            if (!ok) continue;
            const int page_at = s ? z[1] : z[0], row_at = s ? y[1] : y[0];
            if (!wait(empty + ring.stage, ring.phase ^ 1u, p.status, 90)) {
              ok = false;
              continue;
            }
            uint64_t* const bar = arrival + ring.stage;
            const uint32_t dst = ptx::smem_u32(ring_at + ring.stage * L::kTileBytes);
            const bool by_rows = !CODES && kv == 1 && (s ? cut[1] : cut[0]) != 0;      // one box at most: the last
            if (by_rows) {
              const int who = __ffs(s ? cut[1] : cut[0]) - 1, left = __shfl_sync(0xffffffffu, s ? held[1] : held[0], who);
              const int64_t off = __shfl_sync(0xffffffffu, page_at, who) * p.c.v.page + __shfl_sync(0xffffffffu, row_at, who) * p.c.v.row + walk.h * p.c.v.head;
              rows_by_hand<DPAD>(p, dst, p.c.v.base + off, who * rows, rows, left);
            }
            if (lane == 0) ptx::mbar_arrive_expect_tx(bar, (CODES ? 128 * 128 : L::kTileBytes) - (by_rows ? rows * L::kBoxes * 128 : 0));
            __syncwarp();
            if (lane < boxes && !(by_rows && (s ? cut[1] : cut[0]) >> lane & 1)) {
              const uint32_t to = dst + lane * rows * 128;
              if constexpr (CODES) {
                tma_load_4d(to + (DPAD == 128 ? 128 * 128 : 0), kv == 0 ? &tk : &tv, bar, 0, row_at, walk.h, page_at);
              } else {
#pragma unroll
                for (int x = 0; x < L::kBoxes; ++x) tma_load_4d(to + x * L::kBoxBytes, kv == 0 ? &tk : &tv, bar, x * 64, row_at, walk.h, page_at);
              }
            }
            ++issued;
            ring.advance(1);
          }
        }
      }
      // no copy may be under way when the CTA ends, whatever became of its readers
      for (int i = max(0, issued - ring.stages); i < issued; ++i)
        wait(arrival + i % ring.stages, (i / ring.stages) & 1, p.status, 91);
    } else if (MAPS && CODES && warp >= L::kWidenWarp) {
      // ------------------------------------------------------------- codes to fp16, a quarter of a tile's rows a warp
      bool ok = true;
      int n = 0;
      for (; walk.left > 0 && ok; walk.next(p)) {
        const int count = walk.count();
        for (int j = 0; j < count && ok; ++j) {
          const int tiles = walk.paired || !walk.has(j, 1) ? 1 : 2;
#pragma unroll 1
          for (int i = 0; i < 2 * tiles; ++i) {
            if (!wait(raw + ring.stage, ring.phase, p.status, 92)) {
              ok = false;
              break;
            }
            const uint32_t* const words = reinterpret_cast<const uint32_t*>(there + (n + (tiles == 2 ? i & 1 : 0)) % L::kSlots);
            widen_rows<DPAD>(ptx::smem_u32(ring_at + ring.stage * L::kTileBytes), (warp - L::kWidenWarp) * 32, words[warp - L::kWidenWarp]);
            ptx::fence_proxy_async();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(full + ring.stage);
            ring.advance(1);
          }
          n += tiles;
        }
      }
    } else if (!MAPS && warp >= L::kLoadWarp) {
      // ------------------------------------------------------------- loads by threads
      const int loader = warp - L::kLoadWarp;
      bool ok = true;
      int n = 0;
      for (; walk.left > 0 && ok; walk.next(p)) {
        if (warp == L::kQueryWarp || warp == L::kQueryWarp + 1) ok = load_queries(walk);
        const int count = walk.count(), tokens = walk.tokens;
        const bool named = walk.leader >= 0 && walk.leader < p.x.B && tokens <= p.c.capacity;
        const int32_t* line = p.c.table + (named ? walk.leader : 0) * p.c.table_stride;
        int page[4], row[4];                          // of keys lane, lane + 32, .. of a tile: page (-1: none), row
        auto find = [&](int tile) {
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const int t = tile * kPrefixKeys + u * 32 + lane;
            page[u] = -1, row[u] = 0;
            if (named && t < tokens) {
              const int at = p.page_shift >= 0 ? t >> p.page_shift : t / p.c.page_size;
              page[u] = paged::ld_index(line + at);
              row[u] = t - at * p.c.page_size;
            }
          }
        };
        find(walk.tile(0, 0));
        for (int j = 0; j < count && ok; ++j) {
          const int tiles = walk.paired || !walk.has(j, 1) ? 1 : 2;
#pragma unroll 1
          for (int i = 0; i < 2 * tiles; ++i) {       // K of the step's tiles, then V
            const int kv = i >= tiles, s = kv ? i - tiles : i;
            const int64_t page_step = kv ? p.c.v.page : p.c.k.page, row_step = kv ? p.c.v.row : p.c.k.row;
            const char* const src = kv ? p.c.v.base + walk.h * p.c.v.head : p.c.k.base + walk.h * p.c.k.head;
            uint32_t words[4];
            int64_t at[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              const bool exists = static_cast<unsigned>(page[u]) < static_cast<unsigned>(p.c.num_pages);
              words[u] = __ballot_sync(0xffffffffu, exists);
              at[u] = exists ? page[u] * page_step + row[u] * row_step : -1;
            }
            if (i + 1 < 2 * tiles) find(walk.tile(j, i + 1 >= tiles ? i + 1 - tiles : i + 1));
            else if (j + 1 < count) find(walk.tile(j + 1, 0));
            if (!kv && loader == 0 && lane == 0) there[(n + s) % L::kSlots] = make_uint4(words[0], words[1], words[2], words[3]);
            if (!wait(empty + ring.stage, ring.phase ^ 1u, p.status, 90)) {
              ok = false;
              break;
            }
            const uint32_t dst = ptx::smem_u32(ring_at + ring.stage * L::kTileBytes);
            constexpr int kLanes = DPAD / (CODES ? 16 : 8), kRowsAtOnce = 32 / kLanes;      // lanes to a row
            const int c = lane % kLanes;
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              for (int r0 = loader * kRowsAtOnce; r0 < 32; r0 += L::kLoadWarps * kRowsAtOnce) {
                const int r = r0 + lane / kLanes;
                const int64_t off = __shfl_sync(0xffffffffu, at[u], r);
                if constexpr (CODES) {
                  if (c * 16 < p.c.D) {
                    uint4 v = make_uint4(0, 0, 0, 0), a, b;
                    if (off >= 0) v = ld_128(src + off + c * 16);
                    widen(v.x, a.x, a.y), widen(v.y, a.z, a.w), widen(v.z, b.x, b.y), widen(v.w, b.z, b.w);
                    sts128(dst + tile_at(u * 32 + r, 2 * c), a);
                    sts128(dst + tile_at(u * 32 + r, 2 * c + 1), b);
                  }
                } else {
                  if (c * 8 < p.c.D) copy16(dst + tile_at(u * 32 + r, c), src + (off < 0 ? 0 : off) + c * 16, off < 0 ? 0 : 16);
                }
              }
            }
            if constexpr (CODES) {
              ptx::fence_proxy_async();
              ptx::mbar_arrive(full + ring.stage);
            } else {
              arrive_with_copies(full + ring.stage);
            }
            if (loader == 0 && lane == 0) ptx::mbar_arrive(full + ring.stage);       // behind the mask
            ring.advance(1);
          }
          n += tiles;
        }
      }
      asm volatile("cp.async.wait_all;" ::: "memory");       // no copy may be under way when the CTA ends
    } else if (warp == L::kMmaWarp) {
      // ------------------------------------------------------------- products
      // The warp walks the loop together, so that barriers, phases and descriptors stay in uniform registers; one lane issues.
      constexpr int kFormat = kHalf ? 0 : 1;
      const uint32_t id_s = idesc_16(kFormat, 128, kPrefixKeys, 0), id_o = idesc_16(kFormat, 128, p.c.D, 1);
      const int steps = p.c.D / 16;
      // V as the second operand: rows of 64 elements of D, 8 keys to 1024 bytes, the next 64 elements a box further on
      constexpr uint32_t kHiV = (1024u >> 4) | (1u << 14) | (2u << 29);
      constexpr uint32_t kLeadV = (L::kBoxBytes >> 4) << 16;
      const uint32_t ring_lo = (ptx::smem_u32(ring_at) >> 4) & 0x3fffu, q_lo = ptx::desc_lo_sw128(ptx::smem_u32(sq));
      const bool leader = elect_one(), paired = walk.paired;
      bool ok = true;
      uint32_t p_phase[2] = {}, q_phase[2] = {};
      const bool any = walk.left > 0;
      for (; walk.left > 0 && ok; walk.next(p)) {
        const int count = walk.count();
        bool waiting[2] = {}, begun[2] = {};                         // a P that is to be multiplied; O holds something
        Ring v_at[2] = {ring, ring};                                 // its V
        for (int j = 0; j <= count && ok; ++j) {
          const bool more = j < count;
          const bool two = more && walk.has(j, 1);
          Ring k_at[2] = {ring, ring}, v_next[2] = {ring, ring};
          if (paired) {
            v_next[0].advance(1);
            v_next[1] = v_next[0];
          } else {
            k_at[1].advance(1);
            v_next[0].advance(two ? 2 : 1);
            v_next[1] = v_next[0];
            v_next[1].advance(1);
          }
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            if (waiting[s]) {
              ok = ok && wait(full + v_at[s].stage, v_at[s].phase, p.status, 93);
              ptx::fence_proxy_async();                // rows that threads have written, read by the tensor cores
              const uint32_t v_lo = (ring_lo + v_at[s].stage * (L::kTileBytes >> 4)) | kLeadV;
              // the first half of the keys as soon as it is there
#pragma unroll
              for (int half = 0; half < 2; ++half) {
                ok = ok && wait((half == 0 ? p_half : p_full) + s, p_phase[s], p.status, 94);
                ptx::tc_fence_after();
                if (leader && ok) {
#pragma unroll
                  for (int k = 0; k < kPrefixKeys / 32; ++k)
                    mma_ts(tmem + (2 + s) * 128, tmem + s * 128 + half * 32 + k * 8, ptx::desc_join(v_lo + (half * 4 + k) * (2048 >> 4), kHiV), id_o,
                           half > 0 || k > 0 ? 1u : (begun[s] ? 1u : 0u));
                }
                __syncwarp();
              }
              p_phase[s] ^= 1u;
              begun[s] = true;
              waiting[s] = false;
              if (leader && ok && (!paired || s == 1 || !walk.has(0, 1))) ptx::tc_commit<1>(empty + v_at[s].stage);
            }
            if (!more && begun[s] && leader && ok) ptx::tc_commit<1>(o_full + s);
            __syncwarp();
            if (more && (s == 0 || two) && ok) {
              if (j == 0 && (s == 0 || paired)) {
                ok = wait(q_full + s, q_phase[s], p.status, 95);
                q_phase[s] ^= 1u;
              }
              ok = ok && wait(full + k_at[s].stage, k_at[s].phase, p.status, 93);
              ptx::fence_proxy_async();
              ptx::tc_fence_after();
              if (leader && ok) {
                const uint32_t k_lo = (ring_lo + k_at[s].stage * (L::kTileBytes >> 4)) | (1u << 16), mine = q_lo + (paired ? s * (L::kTileBytes >> 4) : 0);
#pragma unroll
                for (int k = 0; k < DPAD / 16; ++k) {
                  const uint32_t at = ((k >> 2) * L::kBoxBytes + (k & 3) * 32) >> 4;
                  if (k < steps) mma_ss(tmem + s * 128, ptx::desc_join(mine + at, ptx::kDescHiSw128), ptx::desc_join(k_lo + at, ptx::kDescHiSw128), id_s, k > 0);
                }
                ptx::tc_commit<1>(s_full + s);
                ptx::mbar_arrive(s_full + s);          // the mask of the tile goes along
                if (!paired || s == 1 || !two) ptx::tc_commit<1>(empty + k_at[s].stage);
              }
              __syncwarp();
              waiting[s] = true;
              v_at[s] = v_next[s];
            }
          }
          if (j == count - 1 && leader && ok) ptx::tc_commit<1>(q_empty);
          __syncwarp();
          if (more) ring.advance(paired ? 2 : (two ? 4 : 2));
        }
      }
      if (any) {
        if (leader) ptx::tc_commit<1>(done);
        __syncwarp();
        wait(done, 0, p.status, 98);
      }
    }
  } else {
    // ------------------------------------------------------------- softmax of tile s, one thread to a row
    ptx::setmaxnreg_inc<L::kSoftmaxRegs>();
    const int s = warp >> 2, r = threadIdx.x & 127;
    const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;     // this warp's 32 lanes of tensor memory
    const uint32_t ts = tmem + s * 128 + lanes, to = tmem + (2 + s) * 128 + lanes;
    bool ok = true;
    uint32_t phase = 0, o_phase = 0;
    int n = 0;                                         // tiles loaded so far
    // The first pass is dry: it waits for nothing, writes nothing and fetches the code below from memory, which takes longer than a tile, while the kernel in
    // front still runs.
    bool dry = p.x.heads > 0, q_turn = false;
    constexpr bool kScaled = CODES && !std::is_same<T, __half>::value;
    Walk walk{};
    walk.left = 1, walk.tiles = 2;
    while (walk.left > 0 && ok) {
      const int count = walk.count();
      bool mine = false;
      float sl = p.scale * 1.4426950408889634f;
      if (!dry) {
        if (!walk.has(0, s)) {                           // no row (which nobody asks for), or no second tile of keys in this part
          const unsigned row = walk.place_of(p, cta, s, r);
          if (!walk.paired && row < p.x.rows) p.x.stats[row] = make_float2(-INFINITY, -1.0f);
          n += walk.loaded(count);
          walk.next(p);
          q_turn = !q_turn;
          continue;
        }
        const int at = walk.row0(s) + r, place = at / p.x.group;
        if (place < walk.n) {
          const int b = paged::ld_index(p.x.plan + p.x.at.order + walk.first + place);
          mine = b >= 0 && b < p.x.B && paged::cached_tokens(p.c, b, 0x7fffffff) >= walk.tokens;
        }
        if constexpr (CODES) sl *= paged::head_scale(p.c.k_amax, p.c.amax_stride, walk.h);
      }
      const bool works = dry || __any_sync(0xffffffffu, mine);
      if (!kScaled) sl = fmaxf(sl, FLT_MIN);            // 0 times a masked -inf would be NaN
      float m = -INFINITY, l = 0.0f;
      bool begun = false, any = false;
      for (int j = 0; j < count && ok; ++j) {
        if (!walk.has(j, s)) break;                    // the last step of an item may have one tile of keys
        if (!dry) {
          ok = ptx::mbar_wait(s_full + s, phase);
          if (!ok) {
            timed_out(p.status, 96);
            break;
          }
          phase ^= 1u;
        }
        if (kScaled && j == 0) {                       // the queries, and how far they were raised, are there as S is
          sl = fmaxf(sl * __uint_as_float(static_cast<uint32_t>(127 - ups[(q_turn * 2 + (walk.paired ? s : 0)) * 128 + r]) << 23), FLT_MIN);
        }
        ptx::tc_fence_after();
        const uint4 words = there[(n + (walk.paired ? j : 2 * j + s)) % L::kSlots];
        any = any || (words.x | words.y | words.z | words.w) != 0;
        if (works) {
          if (!dry && (words.x & words.y & words.z & words.w) != 0xffffffffu) mask_scores(ts, words);
          uint32_t x[kPrefixKeys];
#pragma unroll
          for (int c = 0; c < 4; ++c) ptx::tmem_ld_32x32(ts + c * 32, x + c * 32);
          ptx::tmem_ld_wait();
          float top[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) top[c] = fmaxf(__uint_as_float(x[c]), __uint_as_float(x[4 + c]));
#pragma unroll
          for (int c = 8; c < kPrefixKeys; c += 8)
#pragma unroll
            for (int e = 0; e < 4; ++e) top[e] = fmaxf(top[e], fmaxf(__uint_as_float(x[c + e]), __uint_as_float(x[c + 4 + e])));
          const float mx = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
          if (!begun) {
            m = mx;
            begun = true;
          } else if (__any_sync(0xffffffffu, (mx - m) * sl > kLazy<kHalf>)) {
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
              if (!dry) {
                ptx::tmem_st_32x32_x16(to + c * 32, o);
                ptx::tmem_st_32x32_x16(to + c * 32 + 16, o + 16);
              }
            }
          }
          // the difference first: logits of 2^24 and more would lose the factor
          const float back = m == -INFINITY ? 0.0f : -m;
          const uint64_t back2 = pack2(back, back), sl2 = pack2(sl, sl), raise2 = pack2(kRaise<kHalf>, kRaise<kHalf>);
          uint64_t sum0 = 0, sum1 = 0;
#pragma unroll
          for (int c = 0; c < kPrefixKeys; c += 32) {
            uint32_t pk[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const uint64_t y = fma2(add2(pack2(__uint_as_float(x[c + 2 * e]), __uint_as_float(x[c + 2 * e + 1])), back2), sl2, raise2);
              const float2 a = unpack2(y);
              const float px = exp2_fast(a.x), py = exp2_fast(a.y);
              if (e & 1) sum1 = add2(sum1, pack2(px, py)); else sum0 = add2(sum0, pack2(px, py));
              pk[e] = pack16<E>(px, py);
            }
            if (!dry) ptx::tmem_st_32x32_x16(ts + c / 2, pk);
            if (c == 32) {
              ptx::tmem_st_wait();
              ptx::tc_fence_before();
              __syncwarp();
              if (lane == 0 && !dry) ptx::mbar_arrive(p_half + s);
            }
          }
          const float2 s0 = unpack2(sum0), s1 = unpack2(sum1);
          l += (s0.x + s0.y) + (s1.x + s1.y);
          ptx::tmem_st_wait();
          ptx::tc_fence_before();
          __syncwarp();
          if (lane == 0 && !dry) ptx::mbar_arrive(p_full + s);
        } else if (lane == 0) {                        // rows of nobody: what their P holds reaches their own O only
          ptx::mbar_arrive(p_half + s);
          ptx::mbar_arrive(p_full + s);
        }
      }
      if (dry) {
        pdl_wait();
        walk = find_start(p, cta);
        dry = false;
        continue;
      }
      q_turn = !q_turn;
      n += walk.loaded(count);
      const unsigned row = walk.place_of(p, cta, s, r);
      if (ok && !ptx::mbar_wait(o_full + s, o_phase)) {
        timed_out(p.status, 97);
        ok = false;
      }
      o_phase ^= 1u;
      if (!ok) break;
      ptx::tc_fence_after();
      const bool keeps = row < p.x.rows;
      if (keeps) p.x.stats[row] = make_float2(m == -INFINITY ? m : m * sl - kRaise<kHalf>, mine && any ? l : -1.0f);
      if (works) {
        float* const dst = p.x.parts + static_cast<int64_t>(row) * DPAD;
#pragma unroll 1
        for (int c = 0; c < DPAD / 32; ++c) {
          U32x8 o[4];
          ptx::tmem_ld_32x32(to + c * 32, &o[0].v[0]);
          ptx::tmem_ld_wait();
          if (keeps && mine) {
#pragma unroll
            for (int e = 0; e < 4; ++e) st_256(dst + c * 32 + e * 8, o[e]);
          }
        }
      }
      ptx::tc_fence_before();                          // these reads of O in front of the next item's products
      walk.next(p);
    }
  }
  ptx::tc_fence_before();
  __syncthreads();
  if (warp == L::kMmaWarp) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc<1>(tmem, L::kTmemCols);
  }
}

// The parts of every row together, in the order of the keys: those of its prefix, then those of its own keys.  A row has 1, 2, 4 or 8 of a CTA's warps, a
// share of the parts each.
struct JoinParams {
  Cache c;
  Prefix x;
  void* out;
  int B, Hq, rows_log2;      // rows of a CTA
};
constexpr int kJoinWarps = 8;

struct PartSum {
  float top, sum, acc[4];
  bool has;
  template <int N>
  __device__ __forceinline__ void add(const float2 (&s)[N], const float4 (&v)[N]) {
    float now = top;
#pragma unroll
    for (int k = 0; k < N; ++k)
      if (!(s[k].y < 0.0f)) now = fmaxf(now, s[k].x), has = true;
    const float base = now == -INFINITY ? 0.0f : now, f0 = exp2_fast(top - base);
    sum *= f0, acc[0] *= f0, acc[1] *= f0, acc[2] *= f0, acc[3] *= f0, top = now;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      if (s[k].y < 0.0f) continue;
      const float f = exp2_fast(s[k].x - base);
      sum += s[k].y * f;
      acc[0] += v[k].x * f, acc[1] += v[k].y * f, acc[2] += v[k].z * f, acc[3] += v[k].w * f;
    }
  }
};

template <typename T, int DPAD>
__global__ void __launch_bounds__(kJoinWarps * 32, 3) join_kernel(const __grid_constant__ JoinParams p) {
  __shared__ float4 acc_of[kJoinWarps][32];
  __shared__ float2 stats_of[kJoinWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, share_log2 = 3 - p.rows_log2, share = warp & ((1 << share_log2) - 1);
  const int id = static_cast<int>(blockIdx.x << p.rows_log2) + (warp >> share_log2);
  const bool there = id < p.B * p.Hq;
  const int b = there ? id / p.Hq : 0, hq = there ? id - b * p.Hq : 0, h = hq / p.x.group, head = hq - h * p.x.group, d = lane * 4;
  pdl_launch_dependents();
  pdl_wait();
  PartSum a{-INFINITY, 0.0f, {}, false};
  if (there) {
    // its prefix: of each part the half that holds the row, or (not paired) both
    const int4 of = paged::ld_index4(p.x.plan + p.x.at.sequences + PlanLayout::kSequence * b);
    const bool paired = paged::ld_index(p.x.plan + p.x.at.head) != 0;
    const int held = paged::cached_tokens(p.c, b, 0x7fffffff);
    const int64_t own_total = __ldcg(p.x.own_lines + p.B);
    const int own_ctas = static_cast<int>(__ldcg(p.x.own_lines + p.B + 1));
    const int64_t own_begin = __ldcg(p.x.own_lines + b);
    const int shared = paged::prefix_tokens(of.x, held), row = of.w + head, item = of.y + h * of.z + (row >> (paired ? 8 : 7)), r = row & 127;
    int parts = 0, apart = 0;
    int64_t at = 0;                                    // the first, in rows
    if (shared > 0 && row >= 0 && item >= 0 && item < p.x.items) {
      const int32_t* const entry = p.x.plan + p.x.at.items + PlanLayout::kItem * item;
      const int c0 = min(max(paged::ld_index(entry), 0), paged::kPrefixCtas), ctas = min(max(paged::ld_index(entry + 1), 0), paged::kPrefixCtas - c0);
      const int2 place = make_int2(paged::ld_index(p.x.plan + p.x.at.places + PlanLayout::kPlace * item), min(max(paged::ld_index(p.x.plan + p.x.at.places + PlanLayout::kPlace * item + 1), 0), 256));
      parts = paired ? ctas : 2 * ctas, apart = paired ? place.y : place.y / 2;
      at = static_cast<int64_t>(place.x) + c0 * place.y + (paired ? row & 128 : 0) + r;
      if (at < 0 || at + static_cast<int64_t>(parts) * apart - apart >= p.x.rows) parts = 0;
    }
    // its own keys
    const int own_tiles = held > shared ? (held - shared + 15) / 16 : 1, own_block = head / p.x.own_rows;
    const int64_t own_start = own_begin + static_cast<int64_t>(h * p.x.own_blocks + own_block) * (own_tiles + paged::kOwnItemTiles) + paged::kOwnItemTiles;
    const int o0 = holder(own_total, own_start, own_ctas), o1 = holder(own_total, own_start + own_tiles - 1, own_ctas);
    const int64_t own_at = ((static_cast<int64_t>(b) * p.c.heads + h) * p.x.own_blocks + own_block + o0) * p.x.own_rows + head - own_block * p.x.own_rows;
    const int all = parts + o1 - o0 + 1, from = all * share >> share_log2, to = all * (share + 1) >> share_log2;
    constexpr int kAtOnce = 8;
#pragma unroll 1
    for (int i = from; i < to; i += kAtOnce) {
      float2 s[kAtOnce];
      float4 v[kAtOnce];
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k) {              // the loads first: they do not wait for one another
        s[k].y = -1.0f;
        const int n = i + k;
        if (n >= to) continue;
        const int64_t of = n < parts ? at + static_cast<int64_t>(n) * apart : own_at + static_cast<int64_t>(n - parts) * p.x.own_rows;
        s[k] = __ldcg((n < parts ? p.x.stats : p.x.own_stats) + of);
        if (d < DPAD) v[k] = __ldcg(reinterpret_cast<const float4*>((n < parts ? p.x.parts : p.x.own) + of * DPAD + d));
      }
      a.add(s, v);
    }
  }
  if (share_log2 > 0) {
    acc_of[warp][lane] = make_float4(a.acc[0], a.acc[1], a.acc[2], a.acc[3]);
    if (lane == 0) stats_of[warp] = make_float2(a.top, a.has ? a.sum : -1.0f);
    __syncthreads();
    if (share > 0) return;
#pragma unroll 1
    for (int k = 1; k < 1 << share_log2; ++k) {
      const float2 s[1] = {stats_of[warp + k]};
      const float4 v[1] = {acc_of[warp + k][lane]};
      a.add(s, v);
    }
  }
  if (!there || d >= p.c.D) return;
  uint2 u = make_uint2(0, 0);
  if (a.has) {
    const float f = (p.c.codes ? paged::head_scale(p.c.v_amax, p.c.amax_stride, h) : 1.0f) / a.sum;
    u = make_uint2(pack16<T>(a.acc[0] * f, a.acc[1] * f), pack16<T>(a.acc[2] * f, a.acc[3] * f));
  }
  *reinterpret_cast<uint2*>(static_cast<T*>(p.out) + static_cast<int64_t>(id) * p.c.D + d) = u;
}

// [D, rows, heads, pages] -> boxes of 128 bytes x box_rows of one head and page, zeros out of bounds; false where a tensor map cannot hold the strides
bool make_map(CUtensorMap* map, const paged::Pool& pool, const Cache& c, int dtype, int box_rows) {
  gemm::EncodeTiledFn fn = gemm::encode_tiled();
  if (fn == nullptr) return false;
  const int size = c.codes ? 1 : 2;
  const int64_t strides_in[3] = {pool.row, pool.head, pool.page}, counts[3] = {c.page_size, c.heads, c.num_pages};
  cuuint64_t strides[3];
  for (int i = 0; i < 3; ++i) {
    if (counts[i] > 1 && (strides_in[i] <= 0 || strides_in[i] >= (1LL << 40))) return false;
    strides[i] = static_cast<cuuint64_t>(counts[i] > 1 ? strides_in[i] : 256);       // where there is one only, any stride will do
  }
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(c.D), static_cast<cuuint64_t>(c.page_size), static_cast<cuuint64_t>(c.heads),
                              static_cast<cuuint64_t>(c.num_pages)};
  const cuuint32_t box[4] = {static_cast<cuuint32_t>(128 / size), static_cast<cuuint32_t>(box_rows), 1, 1}, unit[4] = {1, 1, 1, 1};
  const CUtensorMapDataType type = c.codes ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : (dtype == B200Q_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16);
  return fn(map, type, 4, pool.base, dims, strides, box, unit, CU_TENSOR_MAP_INTERLEAVE_NONE, c.codes ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, bool CODES, int DPAD, bool MAPS>
int launch_prefix(const CUtensorMap& tk, const CUtensorMap& tv, const PrefixParams& p, cudaStream_t st) {
  using L = Layout<DPAD, CODES>;
  auto kernel = prefix_kernel<T, CODES, DPAD, MAPS>;
  static std::atomic<bool> ready[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return B200Q_ERR_CUDA;
  if (dev < 0 || dev >= 64 || !ready[dev].load(std::memory_order_relaxed)) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kSmem) != cudaSuccess) return B200Q_ERR_CUDA;
    if (dev >= 0 && dev < 64) ready[dev].store(true, std::memory_order_relaxed);
  }
  if (launch_pdl(kernel, dim3(paged::kPrefixCtas), dim3(L::kThreads), L::kSmem, st, tk, tv, p) != cudaSuccess) return B200Q_ERR_CUDA;
  return check_launch();
}
template <typename T, bool CODES>
int launch_prefix_d(bool maps, const CUtensorMap& tk, const CUtensorMap& tv, const PrefixParams& p, cudaStream_t st) {
  if (p.c.D <= 64) return maps ? launch_prefix<T, CODES, 64, true>(tk, tv, p, st) : launch_prefix<T, CODES, 64, false>(tk, tv, p, st);
  return maps ? launch_prefix<T, CODES, 128, true>(tk, tv, p, st) : launch_prefix<T, CODES, 128, false>(tk, tv, p, st);
}

template <typename T>
int launch_join(const JoinParams& p, cudaStream_t st) {
  const int64_t rows = static_cast<int64_t>(p.B) * p.Hq, ctas = (rows + (1 << p.rows_log2) - 1) >> p.rows_log2;
  auto kernel = p.c.D <= 64 ? join_kernel<T, 64> : join_kernel<T, 128>;
  if (launch_pdl(kernel, dim3(static_cast<unsigned>(ctas)), dim3(kJoinWarps * 32), 0, st, p) != cudaSuccess) return B200Q_ERR_CUDA;
  return check_launch();
}

// Items of a call, at most, the rows of their parts, and the bytes of the workspace.
struct Sizes {
  int64_t rows, items, parts, stats, own, own_stats, own_lines, bytes;
  int own_rows, own_blocks;
};
bool sizes_of(int64_t B, int64_t Hq, int64_t heads, int64_t D, int64_t groups, int64_t largest, Sizes* s) {
  if (B <= 0 || Hq <= 0 || heads <= 0 || Hq % heads != 0 || D <= 0 || D > paged::kMaxD || groups < 0 || groups > B || largest < 0 || largest > B ||
      B > 65535 || Hq > 65535 || B * Hq > 0x3fffffffLL)
    return false;
  const int64_t group = Hq / heads, up = D <= 64 ? 64 : 128;
  // sum over the groups of ceil(sequences * group / 128), each at most its own number of row tiles, all together one more than full ones each
  const int64_t most = groups * ((largest * group + kPrefixRows - 1) / kPrefixRows), all = B * group / kPrefixRows + groups;
  s->items = heads * (most < all ? most : all);
  if (s->items > 0x3fffffffLL) return false;
  // not paired: two halves of every row; and of one more part to each CTA, which begins within an item
  const int64_t sharing = groups * largest < B ? groups * largest : B, part = 2 * largest * group < 256 ? 2 * largest * group : 256;
  s->rows = 2 * sharing * Hq + paged::kPrefixCtas * part;
  if (s->rows > 0x7fffffffLL) return false;
  const auto round = [](int64_t n) { return (n + 255) / 256 * 256; };
  s->stats = round(s->rows * 8);
  int64_t own_slots;
  paged::own_shape(B, Hq, heads, &s->own_rows, &s->own_blocks, &own_slots);
  s->own_lines = round((B + 2) * 8);
  s->own_stats = round(own_slots * s->own_rows * 8);
  s->own = round(own_slots * s->own_rows * up * 4);
  s->parts = round(s->rows * up * 4);
  s->bytes = s->stats + s->own_lines + s->own_stats + s->own + s->parts + 256;      // the tables begin at a multiple of 256, parts are written 32 bytes at once
  return true;
}

}  // namespace
}  // namespace b200q

using namespace b200q;

extern "C" {

int64_t b200q_shared_prefix_plan_values(int64_t B, int64_t Hq, int64_t heads, int64_t groups, int64_t largest) {
  Sizes s;
  return sizes_of(B, Hq, heads, 128, groups, largest, &s) ? paged::plan_layout(B, groups, s.items).values : 0;
}

int b200q_shared_prefix_plan(const int32_t* members, const int32_t* cu, const int32_t* tokens, int64_t B, int64_t Hq, int64_t heads, int64_t groups,
                             int64_t largest, int32_t* plan) {
  Sizes s;
  if (!sizes_of(B, Hq, heads, 128, groups, largest, &s) || plan == nullptr) return B200Q_ERR_INVALID;
  if (groups > 0 && (cu == nullptr || tokens == nullptr || members == nullptr || cu[0] != 0)) return B200Q_ERR_INVALID;
  for (int64_t g = 0; g < groups; ++g)
    if (cu[g + 1] < cu[g] || cu[g + 1] > B || cu[g + 1] - cu[g] > largest || tokens[g] < 0) return B200Q_ERR_INVALID;
  const PlanLayout l = paged::plan_layout(B, groups, s.items);
  const int64_t group = Hq / heads;
  for (int64_t i = 0; i < l.values; ++i) plan[i] = 0;
  for (int64_t b = 0; b < B; ++b) plan[l.order + b] = -1;
  for (int64_t g = 0; g < groups; ++g) {
    int32_t* const of = plan + l.groups + PlanLayout::kGroup * g;
    of[0] = cu[g], of[1] = cu[g + 1] - cu[g], of[2] = tokens[g], of[3] = of[1] > 0 ? members[cu[g]] : -1;
    for (int32_t i = cu[g]; i < cu[g + 1]; ++i) {
      const int32_t b = members[i];
      if (b < 0 || b >= B || plan[l.sequences + PlanLayout::kSequence * b + 2] != 0) return B200Q_ERR_INVALID;      // of the batch, and in one group
      int32_t* const seq = plan + l.sequences + PlanLayout::kSequence * b;
      seq[0] = tokens[g], seq[2] = 1, seq[3] = static_cast<int32_t>((i - cu[g]) * group);
      plan[l.order + i] = b;
    }
  }
  // Steps and blocks of a group, one way and the other, and the least longest piece, each item that is begun taken for kItemSteps more.
  const auto steps = [&](int64_t g, bool paired) { const int64_t t = (static_cast<int64_t>(tokens[g]) + 127) / 128; return paired ? t : (t + 1) / 2; };
  const auto blocks = [&](int64_t g, bool paired) {
    const int64_t rows = (cu[g + 1] - cu[g]) * group, of = paired ? 256 : 128;
    return tokens[g] > 0 ? (rows + of - 1) / of : 0;
  };
  const auto needed = [&](bool paired, int64_t longest) {    // pieces of up to that length
    int64_t pieces = 0, room = 0;
    for (int64_t g = 0; g < groups; ++g) {
      const int64_t n = heads * blocks(g, paired), all = steps(g, paired);
      for (int64_t i = 0; i < n; ++i) {
        int64_t left = all;
        if (room > paged::kItemSteps) {
          const int64_t take = room - paged::kItemSteps < left ? room - paged::kItemSteps : left;
          left -= take, room -= take + paged::kItemSteps;
        }
        if (left > 0) {
          const int64_t full = (left - 1) / (longest - paged::kItemSteps);
          left -= full * (longest - paged::kItemSteps);
          pieces += full + 1, room = longest - paged::kItemSteps - left;
        }
        if (pieces > paged::kPrefixCtas) return pieces;
      }
    }
    return pieces;
  };
  int64_t best[2];
  for (int paired = 0; paired < 2; ++paired) {
    int64_t total = 0;
    for (int64_t g = 0; g < groups; ++g) total += heads * blocks(g, paired) * (steps(g, paired) + paged::kItemSteps);
    int64_t low = paged::kItemSteps, high = total + paged::kItemSteps + 1;      // too short, long enough
    while (high - low > 1) {
      const int64_t mid = low + (high - low) / 2;
      if (needed(paired, mid) <= paged::kPrefixCtas) high = mid;
      else low = mid;
    }
    best[paired] = high;
  }
  const bool paired = best[1] <= best[0];
  const int64_t longest = best[paired];
  if (longest > 0x3fffffffLL) return B200Q_ERR_INVALID;
  plan[l.head] = paired;
  int64_t item = 0, room = 0, cta = -1, place = 0;
  for (int64_t g = 0; g < groups; ++g) {
    const int64_t n = blocks(g, paired), all = steps(g, paired);
    const int32_t* const of = plan + l.groups + PlanLayout::kGroup * g;
    for (int32_t i = cu[g]; i < cu[g + 1]; ++i) {
      int32_t* const seq = plan + l.sequences + PlanLayout::kSequence * members[i];
      seq[1] = static_cast<int32_t>(item), seq[2] = static_cast<int32_t>(n);
    }
    for (int64_t k = 0; k < heads * n; ++k, ++item) {
      int32_t* const entry = plan + l.items + PlanLayout::kItem * item;
      const int64_t full = paired ? 256 : 128, left = (cu[g + 1] - cu[g]) * group - k % n * full, rows = (left < full ? left : full) * (paired ? 1 : 2);
      int64_t at = 0;
      bool begun = false;
      while (at < all) {
        int32_t* mine = plan + l.ctas + PlanLayout::kCta * cta;
        if (at == 0 && !begun && room > paged::kItemSteps) {                    // behind the item before
          room -= paged::kItemSteps, mine[0] += paged::kItemSteps;
        } else {
          ++cta, room = longest - paged::kItemSteps, mine = plan + l.ctas + PlanLayout::kCta * cta;
          mine[1] = static_cast<int32_t>(item), mine[2] = static_cast<int32_t>(g), mine[3] = static_cast<int32_t>(k / n), mine[4] = static_cast<int32_t>(k % n);
          mine[5] = static_cast<int32_t>(at);
          for (int e = 0; e < 4; ++e) mine[8 + e] = of[e];
        }
        const int64_t take = room < all - at ? room : all - at;
        mine[0] += static_cast<int32_t>(take), room -= take, at += take;
        if (!begun) {
          entry[0] = static_cast<int32_t>(cta), begun = true;
          plan[l.places + PlanLayout::kPlace * item] = static_cast<int32_t>(place - cta * rows), plan[l.places + PlanLayout::kPlace * item + 1] = static_cast<int32_t>(rows);
        }
        entry[1] = static_cast<int32_t>(cta - entry[0] + 1);
        place += rows;
      }
    }
  }
  return B200Q_OK;
}

size_t b200q_shared_prefix_workspace_bytes(int64_t B, int64_t Hq, int64_t heads, int64_t D, int64_t groups, int64_t largest) {
  Sizes s;
  return sizes_of(B, Hq, heads, D, groups, largest, &s) ? static_cast<size_t>(s.bytes) : 0;
}

int b200q_shared_prefix_attention(const void* q, int dtype, const int64_t* q_strides, const b200q_paged_cache* cache, const int32_t* block_table,
                                  int64_t table_stride, int64_t table_width, const int32_t* lens, int64_t B, int64_t Hq, const int32_t* plan,
                                  int64_t groups, int64_t largest, float scale, void* out, void* attention_workspace, size_t attention_workspace_bytes,
                                  void* workspace, size_t workspace_bytes, b200q_stream_t stream) {
  if (groups == 0)           // nothing is shared
    return b200q_paged_attention(q, dtype, q_strides, cache, block_table, table_stride, table_width, lens, B, Hq, scale, 0, 0, out, nullptr, 0,
                                 attention_workspace, attention_workspace_bytes, nullptr, 0, stream);
  PrefixParams p{};
  if (int rc = paged::make_cache(&p.c, cache, dtype, block_table, table_stride, table_width, lens, B)) return rc;
  Sizes s;
  if (!sizes_of(B, Hq, p.c.heads, p.c.D, groups, largest, &s) || largest == 0 || !(scale >= 0.0f)) return B200Q_ERR_INVALID;
  if (q == nullptr || q_strides == nullptr || out == nullptr || plan == nullptr) return B200Q_ERR_INVALID;
  if (!aligned(q, 16) || !aligned(out, 16) || !paged::strides_ok(q_strides, 2, 8)) return B200Q_ERR_ALIGN;
  if (attention_workspace == nullptr || attention_workspace_bytes < b200q_paged_attention_workspace_bytes() || workspace == nullptr ||
      workspace_bytes < static_cast<size_t>(s.bytes))
    return B200Q_ERR_WORKSPACE;
  if (!aligned(attention_workspace, 16) || !aligned(workspace, 16) || !aligned(plan, 16)) return B200Q_ERR_ALIGN;
  if (int rc = check_arch()) return rc;
  p.page_shift = -1;
  if ((p.c.page_size & (p.c.page_size - 1)) == 0)
    for (p.page_shift = 0; (1 << p.page_shift) < p.c.page_size;) ++p.page_shift;
  p.q = static_cast<const char*>(q);
  p.q_batch = q_strides[0] * 2, p.q_head = q_strides[1] * 2;
  p.scale = scale;
  p.status = gemm::device_status_word();
  if (p.status == nullptr) return B200Q_ERR_CUDA;
  char* at = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(workspace) + 255) & ~uintptr_t{255});
  const auto take = [&at](int64_t n) { char* const here = at; at += n; return here; };
  p.x.plan = plan, p.x.at = paged::plan_layout(B, groups, s.items);
  p.x.B = static_cast<int>(B), p.x.groups = static_cast<int>(groups), p.x.largest = static_cast<int>(largest);
  p.x.heads = p.c.heads, p.x.group = static_cast<int>(Hq / p.c.heads), p.x.rows = static_cast<unsigned>(s.rows), p.x.items = static_cast<int>(s.items);
  p.x.stats = reinterpret_cast<float2*>(take(s.stats));
  p.x.own_rows = s.own_rows, p.x.own_blocks = s.own_blocks;
  p.x.own_lines = reinterpret_cast<int64_t*>(take(s.own_lines));
  p.x.own_stats = reinterpret_cast<float2*>(take(s.own_stats));
  p.x.own = reinterpret_cast<float*>(take(s.own));
  p.x.parts = reinterpret_cast<float*>(take(s.parts));
  const auto st = static_cast<cudaStream_t>(stream);
  CUtensorMap tk{}, tv{};
  for (p.box_rows = 1; p.box_rows < kPrefixKeys && p.c.page_size % (2 * p.box_rows) == 0;) p.box_rows *= 2, ++p.box_shift;
  const bool maps = p.box_rows >= 8 && p.c.num_pages > 0 && make_map(&tk, p.c.k, p.c, dtype, p.box_rows) && make_map(&tv, p.c.v, p.c, dtype, p.box_rows);
  int rc;
  if (dtype == B200Q_BF16) rc = p.c.codes ? launch_prefix_d<__nv_bfloat16, true>(maps, tk, tv, p, st) : launch_prefix_d<__nv_bfloat16, false>(maps, tk, tv, p, st);
  else rc = p.c.codes ? launch_prefix_d<__half, true>(maps, tk, tv, p, st) : launch_prefix_d<__half, false>(maps, tk, tv, p, st);
  if (rc == B200Q_OK) rc = paged::attend_behind_prefix(p.c, p.x, q, dtype, q_strides, B, Hq, scale, attention_workspace, st);
  if (rc != B200Q_OK) return rc;
  // a warp to a row where there are rows for all SMs, up to eight otherwise
  JoinParams join{p.c, p.x, out, static_cast<int>(B), static_cast<int>(Hq), 3};
  while (join.rows_log2 > 0 && (B * Hq) >> join.rows_log2 < 2 * sm_count()) --join.rows_log2;
  return dtype == B200Q_BF16 ? launch_join<__nv_bfloat16>(join, st) : launch_join<__half>(join, st);
}

}  // extern "C"
