// Attention of one new token of every sequence, where groups of sequences share the pages of a prefix.
//
//   x_j = (q . k_j) * scale,  out = sum_j exp(x_j - m) v_j / sum_j exp(x_j - m),  m = max_j x_j
//
// The keys j < tokens of a group's prefix are the same for all of its sequences, so the rows of a group (its sequences times the query heads of a
// kv head) meet them as one matrix product, S = Q K^T and O = P V on tcgen05, and every K and V row is read once for up to 128 rows.  The keys behind
// the prefix belong to one sequence each: the kernel of paged_attention.cu attends to them, and joins its result with the parts left here:
// with m = max_i m_i, sum = sum_i l_i 2^(m_i - m), out = sum_i o_i 2^(m_i - m) / sum.
//
// Work: items (shared_prefix.cuh) cut into tiles of 128 keys, and the line of all tiles into equal pieces, one for each resident CTA, two to an SM.  A
// CTA: four warps run the softmax, one thread to a row; one warp issues the products; three load K and V rows, which pages scatter, into
// swizzled tiles (8-bit codes are widened to fp16 on the way, exactly).  P takes the place of the scores it came from in tensor memory.
//
// Rounding: S, the softmax, O and the sums are 32-bit; P is rounded to 16 bits for the second product, an error of one rounding of each term,
// of the size of the result's own.  fp16 (fp16 pages and codes): P is raised by 2^11, so that holds for terms down to 2^-25 of the largest.  bf16
// queries in front of codes are scaled by a power of two into fp16's range, which loses nothing above 2^-38 of a row's largest.
#include <atomic>

#include "gemm_host.cuh"
#include "shared_prefix.cuh"
#include "softmax_tc.cuh"

namespace b200q {
namespace {

using paged::Cache;
using paged::GroupWork;
using paged::Prefix;
using paged::kPrefixKeys;
using paged::kPrefixRows;

constexpr int kLoadWarps = 3;
constexpr int kPerSm = 2;
constexpr int kMostCtas = 320;                   // of a launch

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

template <int DPAD>
struct Layout {
  static constexpr int kBoxes = DPAD / 64, kBoxBytes = 128 * 128, kTileBytes = kBoxes * kBoxBytes;
  static constexpr int kStages = DPAD == 128 ? 2 : 4;
  static constexpr int kBars = 3 * kStages + 6;
  static constexpr int kSlots = 8;                      // of tiles whose masks are kept
  static constexpr int kSmem = 1024 + (1 + kStages) * kTileBytes + kBars * 8 + kSlots * 16 + 16;
  static constexpr int kMmaWarp = 4, kThreads = 128 + 32 * (1 + kLoadWarps);
  static constexpr int kTmemCols = 256;                 // S, then O
  // 256 x 128 registers at launch = 128 x (184 + 72)
  static constexpr int kSoftmaxRegs = 184, kOtherRegs = 72;
};

// A CTA's way along its piece of the line, item after item.
struct Walk {
  int64_t left;              // tiles from here to the end of the piece
  int g, h, row_tile, tile;  // the item, and the first tile of this CTA's part of it
  int64_t item;              // its number
  GroupWork w;
  __device__ __forceinline__ int count() const { return static_cast<int>(left < w.tiles - tile ? left : w.tiles - tile); }
  __device__ __forceinline__ void next(const PrefixParams& p) {
    left -= count();
    tile = 0;
    if (left <= 0) return;
    ++item;
    if (++row_tile < w.row_tiles) return;
    row_tile = 0;
    if (++h < p.x.heads) return;
    h = 0;
    do {
      if (++g >= p.x.groups) {
        left = 0;
        return;
      }
      w = paged::group_work(p.x, p.c, g);
    } while (w.tiles == 0);
  }
};

// Adds up the tiles of all groups and finds the one that holds the first tile of this CTA's piece; all threads take part.  CTA 0 leaves the sums
// where the kernel behind finds them.
template <int THREADS>
__device__ __forceinline__ Walk find_start(const PrefixParams& p, int cta, int ctas) {
  constexpr int kWarps = THREADS / 32;
  __shared__ int64_t sums[2][kWarps];
  __shared__ int64_t found[3];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int64_t tiles = 0, items = 0, mine_tiles = 0, mine_items = 0;      // in front of and of this thread's group
  auto group = [&](int g) {
    mine_tiles = mine_items = 0;
    if (g < p.x.groups) {
      const GroupWork w = paged::group_work(p.x, p.c, g);
      if (w.tiles > 0) mine_items = static_cast<int64_t>(p.x.heads) * w.row_tiles, mine_tiles = mine_items * w.tiles;
    }
  };
  auto scan = [&](int64_t* all_tiles, int64_t* all_items) {
    int64_t a = mine_tiles, b = mine_items;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t oa = __shfl_up_sync(0xffffffffu, a, d), ob = __shfl_up_sync(0xffffffffu, b, d);
      if (lane >= d) a += oa, b += ob;
    }
    if (lane == 31) sums[0][warp] = a, sums[1][warp] = b;
    __syncthreads();
    int64_t ta = 0, tb = 0;
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) a += sums[0][w], b += sums[1][w];
      ta += sums[0][w], tb += sums[1][w];
    }
    __syncthreads();
    tiles = a - mine_tiles, items = b - mine_items;
    *all_tiles = ta, *all_items = tb;
  };
  int64_t total = 0, ignored = 0, items_before = 0;
  for (int base = 0; base < p.x.groups; base += THREADS) {
    int64_t t, n;
    group(base + tid);
    scan(&t, &n);
    if (cta == 0 && base + tid < p.x.groups) {
      p.x.lines[2 * (base + tid)] = total + tiles;
      p.x.lines[2 * (base + tid) + 1] = items_before + items;
    }
    total += t, items_before += n;
  }
  if (total < ctas) ctas = static_cast<int>(total);
  if (cta == 0 && tid == 0) p.x.lines[2 * p.x.groups] = total, p.x.lines[2 * p.x.groups + 1] = ctas;
  Walk walk{};
  if (cta >= ctas) return walk;
  const int64_t want = piece(total, cta, ctas);
  int64_t before = 0;
  items_before = 0;
  for (int base = 0; base < p.x.groups; base += THREADS) {
    int64_t t, n;
    if (p.x.groups > THREADS) {
      group(base + tid);
      scan(&t, &n);
    } else {
      t = total, n = ignored;
    }
    if (want >= before + tiles && want < before + tiles + mine_tiles) found[0] = base + tid, found[1] = before + tiles, found[2] = items_before + items;
    before += t, items_before += n;
    if (before > want) break;
  }
  __syncthreads();
  walk.g = static_cast<int>(found[0]);
  walk.w = paged::group_work(p.x, p.c, walk.g);
  const int64_t rel = want - found[1], item = divide(rel, walk.w.tiles);
  walk.tile = static_cast<int>(rel - item * walk.w.tiles);
  walk.h = static_cast<int>(divide(item, walk.w.row_tiles));
  walk.row_tile = static_cast<int>(item - static_cast<int64_t>(walk.h) * walk.w.row_tiles);
  walk.item = found[2] + item;
  walk.left = piece(total, cta + 1, ctas) - want;
  return walk;
}

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
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 r;
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(a) : "memory");
  return r;
}
// 4-D tiled load into this CTA's shared memory, completion on this CTA's own barrier.
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* m, uint64_t* bar, int32_t x, int32_t y, int32_t z, int32_t w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(m)), "r"(ptx::smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}
// Place of 16 bytes (piece c of a row) in a tile of 128 rows: boxes of 64 elements, 128-byte swizzle.
__device__ __forceinline__ uint32_t tile_at(int row, int c) {
  return static_cast<uint32_t>((c >> 3) * (128 * 128) + row * 128 + (((c & 7) ^ (row & 7)) * 16));
}

// Rows of codes, each in the first bytes of 128, to rows of fp16 in their tile: a row's place takes its own codes' place, so nothing but the warp that
// widens it need have read it.  Rows without a key become zeros.  `first`: of the warp's rows; `there`: 32 bits for 32 keys.
template <int DPAD, int ROWS>
__device__ __forceinline__ void widen_rows(uint32_t tile, int first, int D, const uint4& there) {
  constexpr int kLanes = DPAD / 16, kAtOnce = 32 / kLanes, kBatch = 4;
  const int lane = threadIdx.x & 31, c = lane % kLanes;
  const uint32_t codes = tile + (DPAD == 128 ? 128 * 128 : 0);
  const uint32_t words[4] = {there.x, there.y, there.z, there.w};
#pragma unroll 1
  for (int r0 = first; r0 < first + ROWS; r0 += kAtOnce * kBatch) {
    uint4 v[kBatch];
    const uint32_t word = words[r0 >> 5] >> (r0 & 31);
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int i = k * kAtOnce + lane / kLanes;
      v[k] = (word >> i) & 1 ? lds128(codes + (r0 + i) * 128 + c * 16) : make_uint4(0, 0, 0, 0);
    }
    __syncwarp();
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int r = r0 + k * kAtOnce + lane / kLanes;
      uint4 a, b;
      widen(v[k].x, a.x, a.y), widen(v[k].y, a.z, a.w), widen(v[k].z, b.x, b.y), widen(v[k].w, b.z, b.w);
      if (c * 16 < D) sts128(tile + tile_at(r, 2 * c), a), sts128(tile + tile_at(r, 2 * c + 1), b);
    }
    __syncwarp();
  }
}

// MAPS: K and V rows come by tensor maps, box_rows of a page at once (pages of a multiple of eight rows); otherwise by threads, 16 bytes each.
template <typename T, bool CODES, int DPAD, bool MAPS>
__global__ void __launch_bounds__(Layout<DPAD>::kThreads, kPerSm)
prefix_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv, const __grid_constant__ PrefixParams p) {
  using L = Layout<DPAD>;
  constexpr bool kHalf = CODES || std::is_same<T, __half>::value;
  using E = std::conditional_t<kHalf, __half, __nv_bfloat16>;       // of the products
  extern __shared__ char smem_raw[];
  char* const base = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t{1023});
  char* const sq = base;
  char* const ring = base + L::kTileBytes;
  uint64_t* const bars = reinterpret_cast<uint64_t*>(ring + L::kStages * L::kTileBytes);
  uint64_t* const full = bars;
  uint64_t* const empty = bars + L::kStages;
  uint64_t* const raw = empty + L::kStages;            // codes are there
  uint64_t* const q_full = raw + L::kStages;
  uint64_t* const s_full = q_full + 1;
  uint64_t* const p_half = s_full + 1;
  uint64_t* const p_full = p_half + 1;
  uint64_t* const o_full = p_full + 1;
  uint64_t* const done = o_full + 1;
  uint4* const there = reinterpret_cast<uint4*>((reinterpret_cast<uintptr_t>(done + 1) + 15) & ~uintptr_t{15});   // which keys of a tile exist
  uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(there + L::kSlots);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (warp == L::kMmaWarp) {
    ptx::tmem_alloc<1>(tmem_slot, L::kTmemCols);
    ptx::tmem_relinquish<1>();
  } else if (threadIdx.x == 0) {
    // a stage is full when its boxes are there (codes: when two warps have widened them); or each loading thread's copies, and the mask is written
    for (int i = 0; i < L::kStages; ++i)
      ptx::mbar_init(full + i, MAPS ? (CODES ? 2 : 1) : 32 * kLoadWarps + 1), ptx::mbar_init(empty + i, 1), ptx::mbar_init(raw + i, 1);
    ptx::mbar_init(q_full, 4);
    ptx::mbar_init(s_full, 2);
    ptx::mbar_init(p_half, 4);
    ptx::mbar_init(p_full, 4);
    ptx::mbar_init(o_full, 1);
    ptx::mbar_init(done, 1);
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
  pdl_enter(true);           // the kernel behind starts once everything in front of this one has completed, and reads that without a wait
  const int cta = static_cast<int>(blockIdx.x);
  Walk walk = find_start<L::kThreads>(p, cta, static_cast<int>(gridDim.x));

  if (warp >= L::kMmaWarp) {
    ptx::setmaxnreg_dec<L::kOtherRegs>();
    if (MAPS && warp == L::kMmaWarp + 1) {
      // ------------------------------------------------------------- loads: a lane asks for a box of each tile
      const int boxes = kPrefixKeys >> p.box_shift, rows = p.box_rows;
      uint64_t* const arrival = CODES ? raw : full;
      bool ok = true;
      int st = 0, n = 0, issued = 0;
      uint32_t ph = 0;
      for (; walk.left > 0 && ok; walk.next(p)) {
        const int count = walk.count(), tokens = walk.w.tokens;
        const int leader = paged::ld_index(p.x.order + walk.w.first);
        const bool named = leader >= 0 && leader < p.x.B;
        const int32_t* line = p.c.table + (named ? leader : 0) * p.c.table_stride;
        int page, row;                                // of this lane's box
        auto find = [&](int tile) {
          const int t = tile * kPrefixKeys + lane * rows;
          page = -1, row = 0;
          if (named && lane < boxes && t < tokens) {
            const int at = p.page_shift >= 0 ? t >> p.page_shift : t / p.c.page_size;
            page = paged::ld_index(line + at);
            row = t - at * p.c.page_size;
          }
        };
        find(walk.tile);
        for (int j = 0; j < count && ok; ++j) {
          const int t = (walk.tile + j) * kPrefixKeys + lane * rows;
          const bool exists = static_cast<unsigned>(page) < static_cast<unsigned>(p.c.num_pages);
          const int there_rows = exists ? min(rows, tokens - t) : 0;
          const int z = exists ? page : p.c.num_pages, y = row;      // behind the last page: zeros
          if (j + 1 < count) find(walk.tile + j + 1);
          // a box that the prefix ends in: what lies behind may be anything, and 0 times a NaN of V would be one
          const unsigned cut = __ballot_sync(0xffffffffu, there_rows > 0 && there_rows < rows);
          uint4 words = make_uint4(~0u, ~0u, ~0u, ~0u);
          if (!__all_sync(0xffffffffu, lane >= boxes || there_rows == rows)) {
            uint32_t w[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              const int key = u * 32 + lane;
              w[u] = __ballot_sync(0xffffffffu, (key & (rows - 1)) < __shfl_sync(0xffffffffu, there_rows, key >> p.box_shift));
            }
            words = make_uint4(w[0], w[1], w[2], w[3]);
          }
          if (lane == 0) there[n % L::kSlots] = words;
          ++n;
#pragma unroll 1
          for (int kv = 0; kv < 2; ++kv) {
            if (!ptx::mbar_wait(empty + st, ph ^ 1u)) {
              timed_out(p.status, 90);
              ok = false;
              break;
            }
            const uint32_t dst = ptx::smem_u32(ring + st * L::kTileBytes);
            const bool by_rows = !CODES && kv == 1 && cut != 0;      // one box at most: the last
            if (by_rows) {
              const int who = __ffs(cut) - 1, left = __shfl_sync(0xffffffffu, there_rows, who);
              const int64_t off = __shfl_sync(0xffffffffu, z, who) * p.c.v.page + __shfl_sync(0xffffffffu, y, who) * p.c.v.row + walk.h * p.c.v.head;
              for (int i = lane; i < rows * (DPAD / 8); i += 32) {
                const int r = i / (DPAD / 8), c = i % (DPAD / 8);
                uint4 v = make_uint4(0, 0, 0, 0);
                if (r < left && c * 8 < p.c.D) v = ld_128(p.c.v.base + off + r * p.c.v.row + c * 16);
                sts128(dst + tile_at(who * rows + r, c), v);
              }
              ptx::fence_proxy_async();
              __syncwarp();
            }
            if (lane == 0) ptx::mbar_arrive_expect_tx(arrival + st, (CODES ? 128 * 128 : L::kTileBytes) - (by_rows ? rows * L::kBoxes * 128 : 0));
            __syncwarp();
            if (lane < boxes && !(by_rows && cut >> lane & 1)) {
              const uint32_t to = dst + lane * rows * 128;
              if constexpr (CODES) {
                tma_load_4d(to + (DPAD == 128 ? 128 * 128 : 0), kv == 0 ? &tk : &tv, raw + st, 0, y, walk.h, z);
              } else {
#pragma unroll
                for (int x = 0; x < L::kBoxes; ++x) tma_load_4d(to + x * L::kBoxBytes, kv == 0 ? &tk : &tv, full + st, x * 64, y, walk.h, z);
              }
            }
            ++issued;
            if (++st == L::kStages) st = 0, ph ^= 1u;
          }
        }
      }
      // no copy may be under way when the CTA ends, whatever became of its readers
      for (int i = max(0, issued - L::kStages); i < issued; ++i)
        if (!ptx::mbar_wait(arrival + i % L::kStages, (i / L::kStages) & 1)) timed_out(p.status, 91);
    } else if (MAPS && warp > L::kMmaWarp) {
      // ------------------------------------------------------------- codes to fp16, half of a tile's rows a warp
      if constexpr (CODES) {
        bool ok = true;
        int st = 0, n = 0;
        uint32_t ph = 0;
        for (; walk.left > 0 && ok; walk.next(p)) {
          const int count = walk.count();
          for (int j = 0; j < count && ok; ++j, ++n) {
#pragma unroll 1
            for (int kv = 0; kv < 2; ++kv) {
              if (!ptx::mbar_wait(raw + st, ph)) {
                timed_out(p.status, 92);
                ok = false;
                break;
              }
              widen_rows<DPAD, 64>(ptx::smem_u32(ring + st * L::kTileBytes), (warp - L::kMmaWarp - 2) * 64, p.c.D, there[n % L::kSlots]);
              ptx::fence_proxy_async();
              __syncwarp();
              if (lane == 0) ptx::mbar_arrive(full + st);
              if (++st == L::kStages) st = 0, ph ^= 1u;
            }
          }
        }
      }
    } else if (warp > L::kMmaWarp) {
      // ------------------------------------------------------------- loads by threads
      const int loader = warp - L::kMmaWarp - 1;
      bool ok = true;
      int st = 0, n = 0;                              // stage; tiles so far
      uint32_t ph = 0;
      for (; walk.left > 0 && ok; walk.next(p)) {
        const int count = walk.count(), tokens = walk.w.tokens;
        const int leader = paged::ld_index(p.x.order + walk.w.first);
        const bool named = leader >= 0 && leader < p.x.B;
        const int32_t* line = p.c.table + (named ? leader : 0) * p.c.table_stride;
        int page[4], row[4];                          // of keys lane, lane + 32, .. of the tile: page (-1: none), row
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
        find(walk.tile);
        for (int j = 0; j < count && ok; ++j) {
          uint32_t words[4];
          int64_t k_row[4], v_row[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const bool exists = static_cast<unsigned>(page[u]) < static_cast<unsigned>(p.c.num_pages);
            words[u] = __ballot_sync(0xffffffffu, exists);
            k_row[u] = exists ? page[u] * p.c.k.page + row[u] * p.c.k.row : -1;
            v_row[u] = exists ? page[u] * p.c.v.page + row[u] * p.c.v.row : -1;
          }
          if (j + 1 < count) find(walk.tile + j + 1);
          if (loader == 0 && lane == 0) there[n % L::kSlots] = make_uint4(words[0], words[1], words[2], words[3]);
          ++n;
#pragma unroll 1
          for (int kv = 0; kv < 2; ++kv) {
            if (!ptx::mbar_wait(empty + st, ph ^ 1u)) {
              timed_out(p.status, 90);
              ok = false;
              break;
            }
            const uint32_t dst = ptx::smem_u32(ring + st * L::kTileBytes);
            const char* const src = kv == 0 ? p.c.k.base + walk.h * p.c.k.head : p.c.v.base + walk.h * p.c.v.head;
            if constexpr (!CODES) {
              constexpr int kLanes = DPAD / 8, kRowsAtOnce = 32 / kLanes;      // lanes to a row
              const int c = lane % kLanes;
#pragma unroll
              for (int u = 0; u < 4; ++u) {
                for (int r0 = loader * kRowsAtOnce; r0 < 32; r0 += kLoadWarps * kRowsAtOnce) {
                  const int r = r0 + lane / kLanes;
                  const int64_t off = __shfl_sync(0xffffffffu, kv == 0 ? k_row[u] : v_row[u], r);
                  if (c * 8 < p.c.D) copy16(dst + tile_at(u * 32 + r, c), src + (off < 0 ? 0 : off) + c * 16, off < 0 ? 0 : 16);
                }
              }
              arrive_with_copies(full + st);
            } else {
              constexpr int kLanes = DPAD / 16, kRowsAtOnce = 32 / kLanes;
              const int c = lane % kLanes;
#pragma unroll
              for (int u = 0; u < 4; ++u) {
                for (int r0 = loader * kRowsAtOnce; r0 < 32; r0 += kLoadWarps * kRowsAtOnce) {
                  const int r = r0 + lane / kLanes;
                  const int64_t off = __shfl_sync(0xffffffffu, kv == 0 ? k_row[u] : v_row[u], r);
                  if (c * 16 < p.c.D) {
                    uint4 v = make_uint4(0, 0, 0, 0);
                    if (off >= 0) v = ld_128(src + off + c * 16);
                    uint4 a, b;
                    widen(v.x, a.x, a.y), widen(v.y, a.z, a.w), widen(v.z, b.x, b.y), widen(v.w, b.z, b.w);
                    sts128(dst + tile_at(u * 32 + r, 2 * c), a);
                    sts128(dst + tile_at(u * 32 + r, 2 * c + 1), b);
                  }
                }
              }
              ptx::fence_proxy_async();
              ptx::mbar_arrive(full + st);
            }
            if (loader == 0 && lane == 0) ptx::mbar_arrive(full + st);       // behind the mask
            if (++st == L::kStages) st = 0, ph ^= 1u;
          }
        }
      }
      asm volatile("cp.async.wait_all;" ::: "memory");       // no copy may be under way when the CTA ends
    } else {
      // ------------------------------------------------------------- products
      constexpr int kFormat = kHalf ? 0 : 1;
      const uint32_t id_s = idesc_16(kFormat, 128, kPrefixKeys, 0), id_o = idesc_16(kFormat, 128, p.c.D, 1);
      const int steps = p.c.D / 16;
      // V as the second operand: rows of 64 elements of D, 8 keys to 1024 bytes, the next 64 elements a box further on
      constexpr uint32_t kHiV = (1024u >> 4) | (1u << 14) | (2u << 29);
      constexpr uint32_t kLeadV = (L::kBoxBytes >> 4) << 16;
      const uint32_t ring_lo = (ptx::smem_u32(ring) >> 4) & 0x3fffu, q_lo = ptx::desc_lo_sw128(ptx::smem_u32(sq));
      const bool leader = elect_one();
      bool ok = true;
      uint32_t p_phase = 0, q_phase = 0;
      int stage = 0, v_stage = 0;                                    // of this tile's K; of the V of the tile before
      uint32_t phase = 0, v_phase = 0;
      const bool any = walk.left > 0;
      for (; walk.left > 0 && ok; walk.next(p)) {
        const int count = walk.count();
        if (!ptx::mbar_wait(q_full, q_phase)) ok = false;
        q_phase ^= 1u;
        for (int j = 0; j <= count && ok; ++j) {
          const bool more = j < count;
          if (more) ok = ptx::mbar_wait(full + stage, phase);
          if (j > 0) ok = ok && ptx::mbar_wait(full + v_stage, v_phase);
          if (!ok) break;
          ptx::fence_proxy_async();                    // rows written by asynchronous copies of threads, read by the tensor cores
          ptx::tc_fence_after();
          const uint32_t v_lo = (ring_lo + v_stage * (L::kTileBytes >> 4)) | kLeadV, k_lo = (ring_lo + stage * (L::kTileBytes >> 4)) | (1u << 16);
          if (j > 0) {
            // the first half of the keys as soon as it is there
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              ok = ok && ptx::mbar_wait(half == 0 ? p_half : p_full, p_phase);
              ptx::tc_fence_after();
              if (leader && ok) {
#pragma unroll
                for (int k = 0; k < kPrefixKeys / 32; ++k)
                  mma_ts(tmem + 128, tmem + half * 32 + k * 8, ptx::desc_join(v_lo + (half * 4 + k) * (2048 >> 4), kHiV), id_o, half > 0 || k > 0 || j > 1 ? 1u : 0u);
              }
              __syncwarp();
            }
            p_phase ^= 1u;
            if (!more && leader) ptx::tc_commit<1>(o_full);
            __syncwarp();
          }
          if (more && ok) {
            if (leader) {
#pragma unroll
              for (int k = 0; k < DPAD / 16; ++k) {
                const uint32_t at = ((k >> 2) * L::kBoxBytes + (k & 3) * 32) >> 4;
                if (k < steps) mma_ss(tmem, ptx::desc_join(q_lo + at, ptx::kDescHiSw128), ptx::desc_join(k_lo + at, ptx::kDescHiSw128), id_s, k > 0);
              }
              ptx::tc_commit<1>(s_full);
              ptx::mbar_arrive(s_full);                // the mask of the tile goes along
            }
            __syncwarp();
          }
          if (!ok) break;
          if (leader) {
            if (j > 0) ptx::tc_commit<1>(empty + v_stage);
            if (more) ptx::tc_commit<1>(empty + stage);
          }
          __syncwarp();
          if (more) {
            v_stage = stage + 1, v_phase = phase;
            if (v_stage == L::kStages) v_stage = 0, v_phase ^= 1u;
            stage = v_stage + 1, phase = v_phase;
            if (stage == L::kStages) stage = 0, phase ^= 1u;
          }
        }
        if (!ok) timed_out(p.status, 94);
      }
      if (any) {
        if (leader) ptx::tc_commit<1>(done);
        __syncwarp();
        if (!ptx::mbar_wait(done, 0)) timed_out(p.status, 95);
      }
    }
  } else {
    // ------------------------------------------------------------- softmax, one thread to a row
    ptx::setmaxnreg_inc<L::kSoftmaxRegs>();
    const int r = threadIdx.x;
    const uint32_t lanes = static_cast<uint32_t>(warp) << 21;         // this warp's 32 lanes of tensor memory
    const uint32_t ts = tmem + lanes, to = tmem + 128 + lanes;
    bool ok = true;
    uint32_t phase = 0, o_phase = 0;
    int n = 0;
    for (; walk.left > 0 && ok; walk.next(p)) {
      const int count = walk.count();
      // the row's query: products with those of the item before have ended (its last scores are here)
      const int at = walk.row_tile * kPrefixRows + r, place = at / p.x.group;
      int b = -1;
      if (place < walk.w.n) b = paged::ld_index(p.x.order + walk.w.first + place);
      const bool mine = b >= 0 && b < p.x.B && paged::cached_tokens(p.c, b, 0x7fffffff) >= walk.w.tokens;
      float sl = p.scale * 1.4426950408889634f;
      {
        const char* src = p.q + (mine ? b : 0) * p.q_batch + (walk.h * p.x.group + at - place * p.x.group) * p.q_head;
        uint4 u[DPAD / 8];
#pragma unroll
        for (int c = 0; c < DPAD / 8; ++c) {
          u[c] = make_uint4(0, 0, 0, 0);
          if (mine && c * 8 < p.c.D) u[c] = ld_128(src + c * 16);
        }
        if constexpr (CODES) {
          sl *= paged::head_scale(p.c.k_amax, p.c.amax_stride, walk.h);
          if constexpr (!std::is_same<T, __half>::value) {
            uint32_t* w = &u[0].x;
            float top = 0.0f;
#pragma unroll
            for (int i = 0; i < DPAD / 2; ++i) top = fmaxf(top, fmaxf(fabsf(__uint_as_float(w[i] << 16)), fabsf(__uint_as_float(w[i] & 0xffff0000u))));
            // 2^(13 - exponent): the largest lands in [2^13, 2^14); zero, infinity and NaN stay as they are
            const int e = static_cast<int>(__float_as_uint(top) >> 23);
            float f = 1.0f;
            if (top != 0.0f && e < 255) {
              const int s = min(140 - max(e, 1), 124);
              f = __uint_as_float(static_cast<uint32_t>(max(s, -125) + 127) << 23);
            }
            sl *= 1.0f / f;
#pragma unroll
            for (int i = 0; i < DPAD / 2; ++i) w[i] = pack16<__half>(__uint_as_float(w[i] << 16) * f, __uint_as_float(w[i] & 0xffff0000u) * f);
          }
        }
        const uint32_t dst = ptx::smem_u32(sq);
#pragma unroll
        for (int c = 0; c < DPAD / 8; ++c) sts128(dst + tile_at(r, c), u[c]);
      }
      ptx::fence_proxy_async();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(q_full);
      sl = fmaxf(sl, 1e-30f);                                         // 0 times a masked -inf would be NaN
      const bool works = __any_sync(0xffffffffu, mine);
      const uint64_t sl2 = pack2(sl, sl);
      float m = -INFINITY, l = 0.0f;
      bool begun = false, any = false;
      for (int j = 0; j < count && ok; ++j) {
        ok = ptx::mbar_wait(s_full, phase);
        if (!ok) {
          timed_out(p.status, 96);
          break;
        }
        phase ^= 1u;
        ptx::tc_fence_after();
        const uint4 words = there[n++ % L::kSlots];
        any = any || (words.x | words.y | words.z | words.w) != 0;
        if (works) {
          uint32_t x[kPrefixKeys];
#pragma unroll
          for (int c = 0; c < 4; ++c) ptx::tmem_ld_32x32(ts + c * 32, x + c * 32);
          ptx::tmem_ld_wait();
          if ((words.x & words.y & words.z & words.w) != 0xffffffffu) {
            const uint32_t seen[4] = {words.x, words.y, words.z, words.w};
#pragma unroll
            for (int c = 0; c < kPrefixKeys; ++c) x[c] = seen[c / 32] & (1u << (c % 32)) ? x[c] : 0xff800000u;
          }
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
              ptx::tmem_st_32x32_x16(to + c * 32, o);
              ptx::tmem_st_32x32_x16(to + c * 32 + 16, o + 16);
            }
          }
          // the difference first: logits of 2^24 and more would lose the factor
          const float back = m == -INFINITY ? 0.0f : -m;
          const uint64_t back2 = pack2(back, back), raise2 = pack2(kRaise<kHalf>, kRaise<kHalf>);
          uint64_t sum0 = 0, sum1 = 0;
#pragma unroll
          for (int c = 0; c < kPrefixKeys; c += 32) {
            uint32_t pk[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const float2 y = unpack2(fma2(add2(pack2(__uint_as_float(x[c + 2 * e]), __uint_as_float(x[c + 2 * e + 1])), back2), sl2, raise2));
              const uint64_t v = pack2(exp2_fast(y.x), exp2_fast(y.y));
              if (e & 1) sum1 = add2(sum1, v); else sum0 = add2(sum0, v);
              const float2 a = unpack2(v);
              pk[e] = pack16<E>(a.x, a.y);
            }
            ptx::tmem_st_32x32_x16(ts + c / 2, pk);
            if (c == 32) {
              ptx::tmem_st_wait();
              ptx::tc_fence_before();
              __syncwarp();
              if (lane == 0) ptx::mbar_arrive(p_half);
            }
          }
          const float2 s0 = unpack2(sum0), s1 = unpack2(sum1);
          l += (s0.x + s0.y) + (s1.x + s1.y);
          ptx::tmem_st_wait();
          ptx::tc_fence_before();
          __syncwarp();
          if (lane == 0) ptx::mbar_arrive(p_full);
        } else if (lane == 0) {                        // rows of nobody: what their P holds reaches their own O only
          ptx::mbar_arrive(p_half);
          ptx::mbar_arrive(p_full);
        }
      }
      if (ok && !ptx::mbar_wait(o_full, o_phase)) {
        timed_out(p.status, 97);
        ok = false;
      }
      o_phase ^= 1u;
      if (!ok) break;
      ptx::tc_fence_after();
      const int64_t slot = walk.item + cta;
      const bool keeps = r < p.x.rows && slot < p.x.slots;
      if (keeps) p.x.stats[slot * p.x.rows + r] = make_float2(m == -INFINITY ? m : m * sl - kRaise<kHalf>, mine && any ? l : -1.0f);
      if (works) {
        float* const dst = p.x.parts + (slot * p.x.rows + r) * DPAD;
#pragma unroll 1
        for (int c = 0; c < DPAD / 32; ++c) {
          uint32_t o[32];
          ptx::tmem_ld_32x32(to + c * 32, o);
          ptx::tmem_ld_wait();
          if (keeps && mine) {
#pragma unroll
            for (int e = 0; e < 32; e += 4) *reinterpret_cast<uint4*>(dst + c * 32 + e) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
          }
        }
      }
      ptx::tc_fence_before();                          // these reads of O in front of the next item's products
    }
  }
  ptx::tc_fence_before();
  __syncthreads();
  if (warp == L::kMmaWarp) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc<1>(tmem, L::kTmemCols);
  }
}

// The parts of every row together: those of its prefix, in the order of the keys, and that of its own keys.  A row has 1, 2, 4 or 8 of a CTA's warps, a
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
  __device__ __forceinline__ void add(const float2& s, const float4& v) {
    if (s.y < 0.0f) return;
    has = true;
    const float now = fmaxf(top, s.x), base = now == -INFINITY ? 0.0f : now, f0 = exp2_fast(top - base), f1 = exp2_fast(s.x - base);
    sum = sum * f0 + s.y * f1;
    acc[0] = acc[0] * f0 + v.x * f1, acc[1] = acc[1] * f0 + v.y * f1;
    acc[2] = acc[2] * f0 + v.z * f1, acc[3] = acc[3] * f0 + v.w * f1;
    top = now;
  }
};

template <typename T, int DPAD>
__global__ void __launch_bounds__(kJoinWarps * 32) join_kernel(const __grid_constant__ JoinParams p) {
  __shared__ float4 acc_of[kJoinWarps][32];
  __shared__ float2 stats_of[kJoinWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, share_log2 = 3 - p.rows_log2, share = warp & ((1 << share_log2) - 1);
  const int64_t id = (static_cast<int64_t>(blockIdx.x) << p.rows_log2) + (warp >> share_log2);
  const bool there = id < static_cast<int64_t>(p.B) * p.Hq;
  const int b = there ? static_cast<int>(id / p.Hq) : 0, hq = there ? static_cast<int>(id - static_cast<int64_t>(b) * p.Hq) : 0;
  const int h = hq / p.x.group, d = lane * 4;
  pdl_launch_dependents();
  pdl_wait();
  PartSum a{-INFINITY, 0.0f, {}, false};
  if (there) {
    const int g = paged::ld_index(p.x.group_of + b), place = paged::ld_index(p.x.place_of + b);
    const bool grouped = paged::prefix_tokens(p.x, b, paged::cached_tokens(p.c, b, 0x7fffffff)) > 0 && g >= 0 && g < p.x.groups;
    const GroupWork w = grouped ? paged::group_work(p.x, p.c, g) : GroupWork{};
    if (grouped && w.tiles > 0 && place >= 0 && place < w.n) {
      const int64_t total = __ldcg(p.x.lines + 2 * p.x.groups);
      const int ctas = static_cast<int>(__ldcg(p.x.lines + 2 * p.x.groups + 1));
      const int row = place * p.x.group + hq - h * p.x.group, tile = row / kPrefixRows, r = row % kPrefixRows;
      const int64_t items = static_cast<int64_t>(h) * w.row_tiles + tile, start = __ldcg(p.x.lines + 2 * g) + items * w.tiles;
      const int64_t slot0 = __ldcg(p.x.lines + 2 * g + 1) + items;
      const int c0 = holder(total, start, ctas), c1 = holder(total, start + w.tiles - 1, ctas);
      const int parts = c1 - c0 + 1, from = c0 + (parts * share >> share_log2), to = c0 + (parts * (share + 1) >> share_log2);
      constexpr int kAtOnce = 8;
#pragma unroll 1
      for (int c = from; c < to; c += kAtOnce) {
        float2 s[kAtOnce];
        float4 v[kAtOnce];
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) {            // the loads first: they do not wait for one another
          s[k].y = -1.0f;
          const int64_t slot = slot0 + c + k;
          if (c + k >= to || r >= p.x.rows || slot >= p.x.slots) continue;
          s[k] = __ldcg(p.x.stats + slot * p.x.rows + r);
          if (d < DPAD) v[k] = __ldcg(reinterpret_cast<const float4*>(p.x.parts + (slot * p.x.rows + r) * DPAD + d));
        }
#pragma unroll
        for (int k = 0; k < kAtOnce; ++k) a.add(s[k], v[k]);
      }
    }
    if (share == (1 << share_log2) - 1) {              // behind the prefix
      float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (d < DPAD) v = __ldcg(reinterpret_cast<const float4*>(p.x.own + id * DPAD + d));
      a.add(__ldcg(p.x.own_stats + id), v);
    }
  }
  if (share_log2 > 0) {
    acc_of[warp][lane] = make_float4(a.acc[0], a.acc[1], a.acc[2], a.acc[3]);
    if (lane == 0) stats_of[warp] = make_float2(a.top, a.has ? a.sum : -1.0f);
    __syncthreads();
    if (share > 0) return;
    for (int k = 1; k < 1 << share_log2; ++k) a.add(stats_of[warp + k], acc_of[warp + k][lane]);
  }
  if (!there || d >= p.c.D) return;
  uint2 u = make_uint2(0, 0);
  if (a.has) {
    const float f = (p.c.codes ? paged::head_scale(p.c.v_amax, p.c.amax_stride, h) : 1.0f) / a.sum;
    u = make_uint2(pack16<T>(a.acc[0] * f, a.acc[1] * f), pack16<T>(a.acc[2] * f, a.acc[3] * f));
  }
  *reinterpret_cast<uint2*>(static_cast<T*>(p.out) + id * p.c.D + d) = u;
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
  using L = Layout<DPAD>;
  auto kernel = prefix_kernel<T, CODES, DPAD, MAPS>;
  static std::atomic<bool> ready[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return B200Q_ERR_CUDA;
  if (dev < 0 || dev >= 64 || !ready[dev].load(std::memory_order_relaxed)) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kSmem) != cudaSuccess) return B200Q_ERR_CUDA;
    if (dev >= 0 && dev < 64) ready[dev].store(true, std::memory_order_relaxed);
  }
  const int ctas = kPerSm * sm_count() < kMostCtas ? kPerSm * sm_count() : kMostCtas;
  if (launch_pdl(kernel, dim3(static_cast<unsigned>(ctas)), dim3(L::kThreads), L::kSmem, st, tk, tv, p) != cudaSuccess) return B200Q_ERR_CUDA;
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

// Parts of a call, at most, and the rows of each: all of its CTAs' and all items.
struct Sizes {
  int64_t rows, slots, parts, stats, lines, own, own_stats, bytes;
};
bool sizes_of(int64_t B, int64_t Hq, int64_t heads, int64_t D, int64_t groups, int64_t largest, Sizes* s) {
  if (B <= 0 || Hq <= 0 || heads <= 0 || Hq % heads != 0 || D <= 0 || D > paged::kMaxD || groups < 0 || groups > B || largest < 0 || largest > B ||
      B > 65535 || Hq > 65535 || B * Hq > 0x3fffffffLL)
    return false;
  const int64_t group = Hq / heads, up = D <= 64 ? 64 : 128;
  s->rows = largest * group < kPrefixRows ? largest * group : kPrefixRows;
  // sum over the groups of ceil(sequences * group / 128), each at most its own number of row tiles, all together one more than full ones each
  const int64_t most = groups * ((largest * group + kPrefixRows - 1) / kPrefixRows), all = B * group / kPrefixRows + groups;
  s->slots = heads * (most < all ? most : all) + kMostCtas;
  const auto round = [](int64_t n) { return (n + 255) / 256 * 256; };
  s->lines = round((2 * groups + 2) * 8);
  s->stats = round(s->slots * s->rows * 8);
  s->own_stats = round(B * Hq * 8);
  s->own = round(B * Hq * up * 4);
  s->parts = round(s->slots * s->rows * up * 4);
  s->bytes = s->lines + s->stats + s->own_stats + s->own + s->parts;
  return true;
}

}  // namespace
}  // namespace b200q

using namespace b200q;

extern "C" {

int64_t b200q_shared_prefix_plan_values(int64_t B, int64_t groups) { return B < 0 || groups < 0 || groups > B ? 0 : 4 * B + 2 * groups + 1; }

int b200q_shared_prefix_plan(const int32_t* members, const int32_t* cu, const int32_t* tokens, int64_t groups, int64_t B, int32_t* plan) {
  if (groups < 0 || B < 0 || B > 65535 || groups > B || plan == nullptr) return B200Q_ERR_INVALID;
  if (groups > 0 && (cu == nullptr || tokens == nullptr || members == nullptr)) return B200Q_ERR_INVALID;
  if (groups > 0 && cu[0] != 0) return B200Q_ERR_INVALID;
  for (int64_t g = 0; g < groups; ++g)
    if (cu[g + 1] < cu[g] || cu[g + 1] > B || tokens[g] < 0) return B200Q_ERR_INVALID;
  int32_t *const tokens_of = plan, *const group_of = plan + B, *const place_of = plan + 2 * B, *const order = plan + 3 * B, *const begin = plan + 4 * B,
          *const shared = begin + groups + 1;
  for (int64_t b = 0; b < B; ++b) tokens_of[b] = 0, group_of[b] = place_of[b] = order[b] = -1;
  begin[0] = 0;
  for (int64_t g = 0; g < groups; ++g) {
    begin[g + 1] = cu[g + 1], shared[g] = tokens[g];
    for (int32_t i = cu[g]; i < cu[g + 1]; ++i) {
      const int32_t b = members[i];
      if (b < 0 || b >= B || group_of[b] >= 0) return B200Q_ERR_INVALID;      // of the batch, and in one group
      order[i] = b, tokens_of[b] = tokens[g], group_of[b] = static_cast<int32_t>(g), place_of[b] = i - cu[g];
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
  if (!aligned(attention_workspace, 16) || !aligned(workspace, 16)) return B200Q_ERR_ALIGN;
  if (int rc = check_arch()) return rc;
  p.page_shift = -1;
  if ((p.c.page_size & (p.c.page_size - 1)) == 0)
    for (p.page_shift = 0; (1 << p.page_shift) < p.c.page_size;) ++p.page_shift;
  p.q = static_cast<const char*>(q);
  p.q_batch = q_strides[0] * 2, p.q_head = q_strides[1] * 2;
  p.scale = scale;
  p.status = gemm::device_status_word();
  if (p.status == nullptr) return B200Q_ERR_CUDA;
  char* at = static_cast<char*>(workspace);
  const auto take = [&at](int64_t n) { char* const here = at; at += n; return here; };
  p.x = Prefix{plan, plan + B, plan + 2 * B, plan + 3 * B, plan + 4 * B, plan + 4 * B + groups + 1, static_cast<int>(B), static_cast<int>(groups),
               static_cast<int>(largest), p.c.heads, static_cast<int>(Hq / p.c.heads), static_cast<int>(s.rows), s.slots};
  p.x.lines = reinterpret_cast<int64_t*>(take(s.lines));
  p.x.stats = reinterpret_cast<float2*>(take(s.stats));
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
