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
constexpr int kOwnItemTiles = 2;                         // the same for a sequence's own keys, in their tiles
constexpr int kItemSteps = 2;                            // what beginning another item costs a CTA, in steps: room in front of each item in the line

__device__ __forceinline__ int ld_index(const int32_t* p) {
  int v;
  asm volatile("ld.global.b32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}

// The rows of a group at a kv head: its sequences, one behind the other, each with the query heads of the kv head.  A CTA works on two tiles of
// scores at once: of 256 rows and the same 128 keys ("paired"), or, where that is more, of 128 rows and two times 128 keys.  An item is a group,
// a kv head and a block of that many rows, its keys are steps of 128 or 256.  The steps of all items stand in one line, which the CTAs cut into
// equal pieces (each item with some room in front, which stands for its queries and its results); what a CTA computes of an item is a part, of two halves: the rows of each of the two tiles, or the same rows with every other 128
// keys.  Along the line either the item or the CTA is another one from part to part, so item + CTA numbers the parts: their slots.
struct Prefix {
  const int32_t* tokens_of;     // [B] the plan (b200q_shared_prefix_plan): of each sequence, the tokens of its prefix,
  const int32_t* group_of;      // [B] its group
  const int32_t* place_of;      // [B] and its place there
  const int32_t* order;         // [B] the sequences of all groups
  const int32_t* cu;            // [groups + 1] where each begins there
  const int32_t* tokens;        // [groups]
  int B, groups, largest;       // largest: sequences of a group, at most
  int heads, group;             // kv heads, query heads of each
  int rows;                     // of half a part
  int64_t slots;
  float* parts;                 // [slots][2][rows][D up to 64 or 128], unnormalised
  float2* stats;                // [slots][2][rows] base-2 logarithm of what they are referred to, sum (-1: no key)
  int64_t* lines;               // [groups][2] steps and items in front of each group; behind them: steps of all, CTAs, whether paired
  // The keys that a sequence has to itself, the same way: items are a sequence, a kv head and a block of its query heads, tiles are of 16 keys, and
  // every warp has a piece of the line.
  int own_rows, own_blocks;     // query heads of an item, items of a kv head
  float* own;                   // [slots][own_rows][D up to 64 or 128]
  float2* own_stats;            // [slots][own_rows]
  int64_t* own_lines;           // [B] tiles in front of each sequence; behind them: tiles of all, warps
};

struct GroupWork {
  int first, n, tokens, tiles, rows;         // place of its first sequence, sequences, keys and their tiles of 128, rows of a kv head
  __device__ __forceinline__ int steps(bool paired) const { return paired ? tiles : (tiles + 1) >> 1; }
  __device__ __forceinline__ int blocks(bool paired) const { return paired ? (rows + 255) >> 8 : (rows + 127) >> 7; }
};
__device__ __forceinline__ GroupWork group_work(const Prefix& x, const Cache& c, int g) {
  GroupWork w;
  w.first = min(max(ld_index(x.cu + g), 0), x.B);
  w.n = min(min(max(ld_index(x.cu + g + 1), w.first), x.B) - w.first, x.largest);
  const int t = ld_index(x.tokens + g);
  w.tokens = t > 0 && t <= c.capacity && w.n > 0 ? t : 0;
  w.tiles = (w.tokens + kPrefixKeys - 1) / kPrefixKeys;
  w.rows = w.n * x.group;
  return w;
}

// Tokens of sequence b that are attended to with its group: of n in the cache, all of the prefix or (a sequence that has been cut or released) none.
__device__ __forceinline__ int prefix_tokens(const Prefix& x, int b, int n) {
  const int t = ld_index(x.tokens_of + b);
  return t > 0 && t <= n ? t : 0;
}

// Rows and blocks of the kernel below, and its slots.
void own_shape(int64_t B, int64_t Hq, int64_t heads, int* rows, int* blocks, int64_t* slots);
// Behind the kernel of the prefixes: single-token attention over the keys that a sequence has to itself, in parts.
int attend_behind_prefix(const Cache& c, const Prefix& x, const void* q, int dtype, const int64_t* q_strides, int64_t B, int64_t Hq, float scale,
                         void* workspace, cudaStream_t st);

}  // namespace paged
}  // namespace b200q
