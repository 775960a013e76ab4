// The prefix that groups of sequences share, as its own kernel and the kernel behind it see it: a line of key tiles cut into equal pieces, and
// where the parts of a row lie.
#pragma once

#include "paged.cuh"

namespace b200q {

// a / b of numbers that are not negative; a division of 64 bits takes some hundred clocks, one of 32 bits a third of that
__device__ __forceinline__ int64_t divide(int64_t a, int64_t b) {
  return (a | b) >> 32 == 0 ? static_cast<int64_t>(static_cast<uint32_t>(a) / static_cast<uint32_t>(b)) : a / b;
}
// Where the piece of CTA c of `ctas` begins in the line of tiles, ctas <= tiles; no piece is empty.
__device__ __forceinline__ int64_t piece(int64_t tiles, int c, int ctas) { return divide(tiles * c, ctas); }
// The CTA whose piece holds tile x.
__device__ __forceinline__ int holder(int64_t tiles, int64_t x, int ctas) { return static_cast<int>(divide((x + 1) * ctas - 1, tiles)); }

namespace paged {

constexpr int kPrefixRows = 128, kPrefixKeys = 128;      // of a tile

__device__ __forceinline__ int ld_index(const int32_t* p) {
  int v;
  asm volatile("ld.global.b32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}

// An item is a group, a kv head and up to 128 of the group's rows there (a row: a sequence and one of the query heads of the kv head, the sequences
// one behind the other).  The key tiles of all items stand in one line, which the CTAs cut into equal pieces; what a CTA computes of an
// item is a part.  Along the line either the item or the CTA is another one from part to part, so item + CTA numbers the parts: their slots.
struct Prefix {
  const int32_t* tokens_of;     // [B] the plan (b200q_shared_prefix_plan): of each sequence, the tokens of its prefix,
  const int32_t* group_of;      // [B] its group
  const int32_t* place_of;      // [B] and its place there
  const int32_t* order;         // [B] the sequences of all groups
  const int32_t* cu;            // [groups + 1] where each begins there
  const int32_t* tokens;        // [groups]
  int B, groups, largest;       // largest: sequences of a group, at most
  int heads, group;             // kv heads, query heads of each
  int rows;                     // of a slot
  int64_t slots;
  float* parts;                 // [slots][rows][D up to 64 or 128], unnormalised
  float2* stats;                // [slots][rows] base-2 logarithm of what they are referred to, sum (-1: no key)
  int64_t* lines;               // [groups][2] tiles and items in front of each group; behind them: tiles of all, CTAs
  float* own;                   // [B][Hq][D up to 64 or 128] the part of each row's own keys
  float2* own_stats;            // [B][Hq]
};

struct GroupWork {
  int first, n, tokens, tiles, row_tiles;    // place of its first sequence, sequences, keys and their tiles, items of a kv head
};
__device__ __forceinline__ GroupWork group_work(const Prefix& x, const Cache& c, int g) {
  GroupWork w;
  w.first = min(max(ld_index(x.cu + g), 0), x.B);
  w.n = min(min(max(ld_index(x.cu + g + 1), w.first), x.B) - w.first, x.largest);
  const int t = ld_index(x.tokens + g);
  w.tokens = t > 0 && t <= c.capacity && w.n > 0 ? t : 0;
  w.tiles = (w.tokens + kPrefixKeys - 1) / kPrefixKeys;
  w.row_tiles = (w.n * x.group + kPrefixRows - 1) / kPrefixRows;
  return w;
}

// Tokens of sequence b that are attended to with its group: of n in the cache, all of the prefix or (a sequence that has been cut or released) none.
__device__ __forceinline__ int prefix_tokens(const Prefix& x, int b, int n) {
  const int t = ld_index(x.tokens_of + b);
  return t > 0 && t <= n ? t : 0;
}

// Behind the kernel of the prefixes: single-token attention over the keys that a sequence has to itself, into `own` and `own_stats`.
int attend_behind_prefix(const Cache& c, const Prefix& x, const void* q, int dtype, const int64_t* q_strides, int64_t B, int64_t Hq, float scale,
                         void* workspace, cudaStream_t st);

}  // namespace paged
}  // namespace b200q
