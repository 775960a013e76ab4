// The prefix that groups of sequences share, as its own kernel and the kernel behind it see it: a line of key tiles cut into equal pieces, and
// where the parts of a row lie.
#pragma once

#include "paged.cuh"

namespace b200q {

// a / b of numbers that are not negative; a division of 64 bits takes some hundred clocks, one of 32 bits a third of that
static __device__ __noinline__ int64_t divide_wide(int64_t a, int64_t b) { return a / b; }
__device__ __forceinline__ int64_t divide(int64_t a, int64_t b) {
  return (a | b) >> 32 == 0 ? static_cast<int64_t>(static_cast<uint32_t>(a) / static_cast<uint32_t>(b)) : divide_wide(a, b);
}
// Where the piece of CTA c of `ctas` begins in the line of tiles, ctas <= tiles; no piece is empty.
__device__ __forceinline__ int64_t piece(int64_t tiles, int c, int ctas) { return divide(tiles * c, ctas); }
// The CTA whose piece holds tile x.
__device__ __forceinline__ int holder(int64_t tiles, int64_t x, int ctas) { return static_cast<int>(divide((x + 1) * ctas - 1, tiles)); }

namespace paged {

constexpr int kPrefixRows = 128, kPrefixKeys = 128;      // of a tile
constexpr int kOwnItemTiles = 2;                         // what beginning another item costs a warp, in tiles: room in front of each in the line
constexpr int kItemSteps = 2;                            // the same for a prefix's items, in steps
constexpr int kPrefixCtas = 148;                         // SMs of a B200; any other number of them works through the same CTAs

__device__ __forceinline__ int ld_index(const int32_t* p) {
  int v;
  asm volatile("ld.global.b32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ int4 ld_index4(const int32_t* p) {
  int4 v;
  asm volatile("ld.global.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
  return v;
}

// The rows of a group at a kv head: its sequences, one behind the other, each with the query heads of the kv head.  A CTA works on two tiles of
// scores at once: of 256 rows and the same 128 keys ("paired"), or, where that is more, of 128 rows and two times 128 keys.  An item is a group,
// a kv head and a block of that many rows, its keys are steps of 128 or 256.  The steps of all items stand in one line, which the plan, made on the
// host, cuts into a piece for each CTA, all as long as can be (with what it costs to begin another item); what a CTA computes of an item is
// a part, of two halves: the rows of each of the two tiles, or the same rows with every other 128 keys.  Parts lie one behind the other in the order of the
// line, each with as many rows as its item has (twice as many where it is not paired), so those of an item are equally far apart: what a call has to
// have room for are the rows of its batch, and of one more item to each CTA, however many groups there may be.
//
// The plan: 32-bit integers, each table at a multiple of four of them.  What is read of it is checked against the sizes of the call where an address
// hangs on it.
struct PlanLayout {
  int64_t head, sequences, order, groups, ctas, items, places, values;
  static constexpr int kHead = 4;                        // whether paired
  static constexpr int kSequence = 4;                    // tokens of its prefix (0: none), first item, items of a kv head, its first row there
  static constexpr int kGroup = 4;                       // place of its first sequence in `order`, sequences, tokens, the sequence whose line names them
  static constexpr int kCta = 12;                        // steps (0: none), item, group, kv head, block, first step; of the group as above
  static constexpr int kItem = 2;                        // first CTA, CTAs
  static constexpr int kPlace = 2;                       // of an item: first row of the part that CTA 0 would have of it, rows of a part
};
inline PlanLayout plan_layout(int64_t B, int64_t groups, int64_t items) {
  const auto up = [](int64_t n) { return (n + 3) / 4 * 4; };
  PlanLayout l{};
  l.head = 0;
  l.sequences = PlanLayout::kHead;
  l.order = l.sequences + PlanLayout::kSequence * B;
  l.groups = l.order + up(B);
  l.ctas = l.groups + PlanLayout::kGroup * groups;
  l.items = l.ctas + PlanLayout::kCta * kPrefixCtas;
  l.places = l.items + up(PlanLayout::kItem * items);
  l.values = l.places + up(PlanLayout::kPlace * items);
  return l;
}

struct Prefix {
  const int32_t* plan;
  PlanLayout at;
  int B, groups, largest;       // largest: sequences of a group, at most
  int heads, group;             // kv heads, query heads of each
  unsigned rows;                // of all parts, at most
  int items;                    // at most
  float* parts;                 // [rows][D up to 64 or 128], unnormalised
  float2* stats;                // [rows] base-2 logarithm of what they are referred to, sum (-1: no key)
  // The keys that a sequence has to itself: items are a sequence, a kv head and a block of its query heads, tiles are of 16 keys, and every warp has
  // a piece of their line, which it finds itself: the lengths are on the device.
  int own_rows, own_blocks;     // query heads of an item, items of a kv head
  float* own;                   // [slots][own_rows][D up to 64 or 128]
  float2* own_stats;            // [slots][own_rows]
  int64_t* own_lines;           // [B] tiles in front of each sequence; behind them: tiles of all, warps
};

// Tokens of sequence b that are attended to with its group: of n in the cache, all of the prefix or (a sequence that has been cut or released) none.
__device__ __forceinline__ int prefix_tokens(int shared, int n) { return shared > 0 && shared <= n ? shared : 0; }
__device__ __forceinline__ int prefix_tokens(const Prefix& x, int b, int n) {
  return prefix_tokens(ld_index(x.plan + x.at.sequences + PlanLayout::kSequence * b), n);
}

// Rows and blocks of the kernel below, and its slots.
void own_shape(int64_t B, int64_t Hq, int64_t heads, int* rows, int* blocks, int64_t* slots);
// Behind the kernel of the prefixes: single-token attention over the keys that a sequence has to itself, in parts.
int attend_behind_prefix(const Cache& c, const Prefix& x, const void* q, int dtype, const int64_t* q_strides, int64_t B, int64_t Hq, float scale,
                         void* workspace, cudaStream_t st);

}  // namespace paged
}  // namespace b200q
