// Attention of one new token of every sequence over its pages of the key-value cache.
//
//   x_j = (q . k_j) * scale,  out = sum_j exp(x_j - m) v_j / sum_j exp(x_j - m),  m = max_j x_j
//
// over the keys j that the token sees, in one pass with a running maximum and sum.  Every K and V row is read once for up to 16
// query heads (a larger group is several items, each of which reads it) and takes part in 4 * D operations per query head, so the
// memory binds the kernel: what has to be found is enough bytes in flight on every SM, and work of the same size for each of them.
//
// Work.  An item is a sequence, a kv head and up to 16 of its query heads; its keys are tiles of 64.  The tiles of all items
// stand in one line, which the resident CTAs cut into equal pieces (the lengths are on the device, so every CTA adds them up
// for itself).  A CTA that ends inside an item leaves its part (maximum, sum, unnormalised result, 32 bits) in the workspace; the
// CTA that arrives last joins the parts in the order of the keys, so that results do not depend on who is last.  More than 16 parts are
// joined in two steps (one sequence of 100000, 8 / 1 heads of 128, 444 parts 25 us instead of 78; of 30000, 64 / 4 heads, 8-bit pages 28.6 instead of 51;
// of 4000, 32 / 8 heads 11.0 instead of 12.3).
//
// A warp takes 16 of a tile's 64 keys through a ring of its own in shared memory, filled by asynchronous copies of 16 bytes, and
// has its own maximum, sum and result; nothing but the end of an item makes warps wait for one another.  The products run on
// mma.sync with K and V^T as the 16-row operand and 8 or 16 query heads as the columns, S^T = K Q^T and O^T = V^T P^T: with so few
// columns a tensor-memory accumulator has nothing to gain (the products need a tenth of the mma.sync rate), and register fragments
// let 8-bit codes be widened between shared memory and the product.  P^T turns from the result of one product into the operand
// of the next by an 8 x 8 transpose among the lanes.
//
// Measured (us a call): 64 sequences of 1 to 8190 tokens, 64 / 8 heads of 128, bf16 174 (6.18 TB/s, 0.94 of the copy rate; DRAM 6.1 TB/s, issue
// slots 28 %); 3 of 60000 to 131071, 8-bit pages 106 (5.5 TB/s: widening codes takes issue slots, 58 %); 32 of 900 to 16000, 16 / 16 heads of 64, window
// 2048 48 (5.5 TB/s); one of 411 tokens 7.3, the chain from the lengths to the joined parts.  With the query heads as the 16-row
// operand 187 / 144 / 69 / 8.3.  The loop in three or six copies, one for each stage of the ring, made short calls longer (instructions are
// fetched once) and long ones no shorter; four CTAs to an SM for 8-bit pages 111.
//
// Rounding.  Products are summed in 32 bits, the softmax is 32-bit.  P is rounded to the 16-bit type of V's operand for the second
// product: an error of one rounding of each term, of the size of the result's own; in fp16 that holds for terms down to 2^-25 of the largest
// one of their warp's keys, and those below are off by up to 2^-36 of it (Reference).  8-bit K and V are exact in fp16; bf16
// queries in front of them are scaled by a power of two into fp16's range, which loses nothing above 2^-38 of the largest.
// Sums of P V are unnormalised: bf16 values up to 2^100 leave them room (P up to 2^8, 2^17 keys).
#include <atomic>

#include "paged.cuh"

namespace b200q {
namespace {

using paged::Cache;

constexpr int kThreads = 128, kWarps = 4, kRows = 16, kTile = 64, kKeys = 16;   // kRows: most query heads of an item; kKeys: of one warp
constexpr int kMaxCtas = 512;                                                  // of a launch
constexpr int kGroupsFrom = 16;                                                 // parts are joined in two steps from one more on
static_assert(2 * kMaxCtas * sizeof(unsigned) == B200Q_PAGED_ATTENTION_ZERO_BYTES, "the header says how much has to be zero");

struct DecodeParams {
  Cache c;
  int page_shift;            // log2 of the page size, or -1
  bool one_layout;           // K and V pages have the same strides
  const char* q;
  int64_t q_batch, q_head;   // bytes
  void* out;
  float* logits;             // with weights: [B, Hq, logits_stride], by the place among the keys seen
  float* lse;                // [B, Hq]
  int64_t logits_stride, weights_len;
  int B, Hq, group, blocks, rows;   // `blocks` of up to `rows` query heads per kv head
  float scale;
  int64_t window, sinks;
  unsigned* tickets;         // [2][kMaxCtas], of items and of groups, zero between calls: B200Q_PAGED_ATTENTION_ZERO_BYTES
  float* parts;              // [kMaxCtas][2][kPart]
};

// What P is referred to.  fp16 (fp16 pages, and codes, which are widened to fp16): set 2^11 below the largest term, so that P is rounded like
// any normal number down to 2^-25 of it (2^-14 if it were set at it), and kept until a term is 2^15 above, within fp16's range.  bf16 has the range.
template <bool HALF>
struct Reference {
  static constexpr float kBelow = HALF ? 11.0f : 0.0f;
  static constexpr float kMost = HALF ? 15.0f : 8.0f;
  // Logits from 2^24 on stand so far apart that a sum of two numbers is rounded to more than it should be.
  __device__ static __forceinline__ float of(float top) {
    const float r = top - kBelow;
    return top - r > kMost ? top : r;
  }
  __device__ static __forceinline__ float most(float r) {
    const float limit = r + kMost;
    return limit - r > kMost ? r : limit;
  }
};
constexpr int kPart = kRows * paged::kMaxD + 4 * kRows;   // result rows, maxima, sums; maxima and sums of a group

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
// 16 bytes to shared memory: `bytes` of them from `src`, zeros behind.
__device__ __forceinline__ void copy16(uint32_t dst, const char* src, int bytes) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

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
__device__ __forceinline__ void ldmatrix_trans(uint32_t a, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
template <bool HALF>
__device__ __forceinline__ void mma(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  if constexpr (HALF)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <bool HALF>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  uint32_t r;
  if constexpr (HALF) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// four codes -> four fp16 values, two and two
__device__ __forceinline__ void widen(uint32_t v, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}" : "=r"(lo), "=r"(hi) : "r"(v));
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float quad_max(float v) {
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}
// over the lanes that share a place in their quads
__device__ __forceinline__ float column_max(float v) {
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
}
__device__ __forceinline__ float column_sum(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 4);
  v += __shfl_xor_sync(0xffffffffu, v, 8);
  return v + __shfl_xor_sync(0xffffffffu, v, 16);
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// The keys that the newest token of a sequence sees: `seen` of them, the first `sinks` in place, the others `gap` further on.
struct Seen {
  int seen, sinks, gap;
  __device__ __forceinline__ int token(int i) const { return i < sinks ? i : i + gap; }
  __device__ __forceinline__ int tiles() const { return seen > 0 ? (seen + kTile - 1) / kTile : 1; }   // 1: somebody writes the zeros
};
__device__ __forceinline__ Seen keys_seen(const DecodeParams& p, int b) {
  const int n = paged::cached_tokens(p.c, b, 0x7fffffff);
  const int first = p.window > 0 && n > p.window ? static_cast<int>(n - p.window) : 0;
  const int sinks = p.sinks < first ? static_cast<int>(p.sinks) : first;
  return Seen{n - (first - sinks), sinks, first - sinks};
}

// Layout of one warp's stage: 16 rows of K, then 16 of V, 16-byte chunks swizzled so that the reads below meet no bank twice.
template <bool CODES, int DPAD, int BLOCKS8>
struct Stage {
  static constexpr int kRowBytes = DPAD * (CODES ? 1 : 2);
  static constexpr int kChunks = kRowBytes / 16;
  static constexpr int kBytes = 2 * kKeys * kRowBytes;
  static constexpr int kPerSm = kBytes >= 8192 || BLOCKS8 == 2 ? 2 : 3;           // CTAs that share an SM
  static constexpr int kDepth = kBytes >= 8192 ? 3 : (kBytes >= 4096 ? (kPerSm == 3 ? 4 : 6) : 8);
  __device__ static __forceinline__ int k_chunk(int key, int c) { return kRowBytes == 64 ? c : c ^ ((key & 1) << 2); }
  __device__ static __forceinline__ int v_chunk(int key, int c) {
    if (!CODES) return c ^ (key & 7);
    return kRowBytes == 64 ? c ^ ((key >> 1) & 3) : c ^ (((key >> 1) & 3) << 1);
  }
};

// a / b of numbers that are not negative; a division of 64 bits takes some hundred clocks, one of 32 bits a third of that
__device__ __forceinline__ int64_t divide(int64_t a, int64_t b) {
  return (a | b) >> 32 == 0 ? static_cast<int64_t>(static_cast<uint32_t>(a) / static_cast<uint32_t>(b)) : a / b;
}
// Where the piece of CTA c of `ctas` begins in the line of tiles, ctas <= tiles; no piece is empty.
__device__ __forceinline__ int64_t piece(int64_t tiles, int c, int ctas) { return divide(tiles * c, ctas); }
// The CTA whose piece holds tile x.
__device__ __forceinline__ int holder(int64_t tiles, int64_t x, int ctas) { return static_cast<int>(divide((x + 1) * ctas - 1, tiles)); }

// Adds up the tiles of all sequences and finds the one that holds the first tile of this CTA's piece; all threads take part.
// `ctas`: of those launched, as many as there are tiles.
__device__ __forceinline__ int64_t find_start(const DecodeParams& p, int cta, int* ctas, int* b_out, int64_t* before_out, Seen* seen_out) {
  __shared__ int64_t sums[kWarps];
  __shared__ int64_t found[2];
  __shared__ Seen found_keys;
  Seen keys{0, 0, 0};
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t per = static_cast<int64_t>(p.c.heads) * p.blocks;
  int64_t total = 0, inclusive = 0, mine = 0;
  auto scan = [&](int64_t v) {                        // inclusive over the CTA; returns the sum
    int64_t s = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t o = __shfl_up_sync(0xffffffffu, s, d);
      if (lane >= d) s += o;
    }
    if (lane == 31) sums[warp] = s;
    __syncthreads();
    int64_t all = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) s += sums[w];
      all += sums[w];
    }
    __syncthreads();
    inclusive = s;
    return all;
  };
  for (int base = 0; base < p.B; base += kThreads) {
    if (base + tid < p.B) keys = keys_seen(p, base + tid);
    mine = base + tid < p.B ? keys.tiles() * per : 0;
    total += scan(mine);
  }
  if (total < *ctas) *ctas = static_cast<int>(total);
  if (cta >= *ctas) return total;
  const int64_t want = piece(total, cta, *ctas);
  if (p.B <= kThreads) {
    if (want >= inclusive - mine && want < inclusive) found[0] = tid, found[1] = inclusive - mine, found_keys = keys;
    __syncthreads();
  } else {
    int64_t before = 0;
    for (int base = 0; base < p.B; base += kThreads) {
      if (base + tid < p.B) keys = keys_seen(p, base + tid);
      mine = base + tid < p.B ? keys.tiles() * per : 0;
      const int64_t all = scan(mine);
      if (want >= before + inclusive - mine && want < before + inclusive)
        found[0] = base + tid, found[1] = before + inclusive - mine, found_keys = keys;
      before += all;
      if (before > want) break;
    }
    __syncthreads();
  }
  *b_out = static_cast<int>(found[0]);
  *before_out = found[1];
  *seen_out = found_keys;
  return total;
}

// BLOCKS8: query heads of an item in blocks of 8.
template <typename T, bool CODES, int DPAD, int BLOCKS8>
__global__ void __launch_bounds__(kThreads, Stage<CODES, DPAD, BLOCKS8>::kPerSm) decode_kernel(const __grid_constant__ DecodeParams p) {
  using S = Stage<CODES, DPAD, BLOCKS8>;
  constexpr bool kHalf = CODES || std::is_same<T, __half>::value;
  constexpr int kSteps = DPAD / 16;
  using R = Reference<kHalf>;
  extern __shared__ __align__(128) char smem[];
  __shared__ float row_max[kWarps][kRows], row_sum[kWarps][kRows];
  __shared__ uint32_t there[kWarps][S::kDepth];        // which of the 16 keys of a stage exist
  __shared__ int last_one;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const int cta = blockIdx.x;
  int ctas = gridDim.x;
  char* const ring = smem + warp * S::kDepth * S::kBytes;
  const uint32_t ring_u32 = smem_u32(ring);
  pdl_launch_dependents();
  pdl_wait();

  int b;
  int64_t before;
  Seen see;
  const int64_t total = find_start(p, cta, &ctas, &b, &before, &see);
  if (cta >= ctas) return;
  int64_t at = piece(total, cta, ctas);
  const int64_t first_tile = at, end = piece(total, cta + 1, ctas);
  // the item: kv head and block of query heads, within sequence b
  int64_t item = divide(at - before, see.tiles());
  int h = static_cast<int>(divide(item, p.blocks)), block = static_cast<int>(item) - h * p.blocks;
  int64_t item_start = before + item * see.tiles();
  while (at < end) {
    const int tiles = see.tiles();
    const int64_t item_end = item_start + tiles;
    const int tile0 = static_cast<int>(at - item_start), tile1 = static_cast<int>((end < item_end ? end : item_end) - item_start);
    const int head0 = h * p.group + block * p.rows, rows = min(p.rows, p.group - block * p.rows);
    const int32_t* line = p.c.table + b * p.c.table_stride;
    const char* const k_lane = p.c.k.base + h * p.c.k.head + lane % (S::kChunks < 8 ? S::kChunks : 8) * 16;
    const char* const v_lane = p.c.v.base + h * p.c.v.head + lane % (S::kChunks < 8 ? S::kChunks : 8) * 16;

    // ------------------------------------------------------------- copies of a warp's 16 keys of a tile
    // lane: of key lane % 16, its page (-1: none) and its row within it
    auto find_page = [&](int tile) {
      const int i = tile * kTile + warp * kKeys + (lane & 15);
      int page = -1, row = 0;
      if (tile < tile1 && i < see.seen) {
        const int token = see.token(i), n = p.page_shift >= 0 ? token >> p.page_shift : token / p.c.page_size;
        asm volatile("ld.global.b32 %0, [%1];" : "=r"(page) : "l"(line + n) : "memory");
        row = token - n * p.c.page_size;
      }
      return make_int2(page, row);
    };
    auto issue = [&](int slot, int2 where) {
      const bool exists = static_cast<unsigned>(where.x) < static_cast<unsigned>(p.c.num_pages);
      constexpr int kLanes = S::kChunks < 8 ? S::kChunks : 8, kPer = 32 / kLanes;     // lanes to a row, rows to an instruction
      const int64_t k_row = exists ? where.x * p.c.k.page + where.y * p.c.k.row : -1;
      const int64_t v_row = p.one_layout ? k_row : (exists ? where.x * p.c.v.page + where.y * p.c.v.row : -1);
      const uint32_t kdst = ring_u32 + slot * S::kBytes, vdst = kdst + kKeys * S::kRowBytes;
#pragma unroll
      for (int j = 0; j < kKeys / kPer; ++j) {
        const int key = j * kPer + lane / kLanes;
        int64_t k_off = __shfl_sync(0xffffffffu, k_row, key);
        const int there_bytes = k_off < 0 ? 0 : 16;
        k_off = k_off < 0 ? 0 : k_off;                  // an aligned address even where nothing is read
        int64_t v_off = k_off;
        if (!p.one_layout) v_off = max(__shfl_sync(0xffffffffu, v_row, key), int64_t{0});
#pragma unroll
        for (int c0 = 0; c0 < S::kChunks; c0 += kLanes) {
          const int c = c0 + lane % kLanes;
          const int bytes = c * 16 < p.c.D * (CODES ? 1 : 2) ? there_bytes : 0;      // 0: nothing is read, zeros are written
          copy16(kdst + key * S::kRowBytes + S::k_chunk(key, c) * 16, k_lane + k_off + c0 * 16, bytes);
          copy16(vdst + key * S::kRowBytes + S::v_chunk(key, c) * 16, v_lane + v_off + c0 * 16, bytes);
        }
      }
      const uint32_t keys = __ballot_sync(0xffffffffu, exists && lane < 16);
      if (lane == 0) there[warp][slot] = keys;
    };
    // ------------------------------------------------------------- queries: head g of each block, the elements that this lane's K chunks meet
    uint32_t q[BLOCKS8][kSteps][2];
    float unit[BLOCKS8];
    int2 page0 = find_page(tile0), page1 = find_page(tile0 + 1), page2 = find_page(tile0 + 2);   // three ahead: a load from the table takes as long as a tile
    {
      const char* base = p.q + b * p.q_batch + head0 * p.q_head;
#pragma unroll
      for (int r = 0; r < BLOCKS8; ++r) {
        const int row = g + 8 * r;
        const char* src = base + row * p.q_head;
        uint32_t* w = &q[r][0][0];                      // step s of the product takes words 2 s and 2 s + 1
#pragma unroll
        for (int i = 0; i < kSteps / 2; ++i) {          // 8 elements each
          const int e = CODES ? (i / 2) * 64 + t * 16 + (i % 2) * 8 : i * 32 + t * 8;
          uint4 u = make_uint4(0, 0, 0, 0);
          if (row < rows && e < p.c.D) u = ld_128(src + e * 2);
          w[4 * i] = u.x, w[4 * i + 1] = u.y, w[4 * i + 2] = u.z, w[4 * i + 3] = u.w;
        }
      }
    }
    {
#pragma unroll
      for (int r = 0; r < BLOCKS8; ++r) {
        uint32_t* w = &q[r][0][0];
        unit[r] = 1.0f;
        if constexpr (CODES && !std::is_same<T, __half>::value) {
          float top = 0.0f;
#pragma unroll
          for (int i = 0; i < 2 * kSteps; ++i)
            top = fmaxf(top, fmaxf(fabsf(__uint_as_float(w[i] << 16)), fabsf(__uint_as_float(w[i] & 0xffff0000u))));
          top = quad_max(top);
          // 2^(13 - exponent): the largest lands in [2^13, 2^14); zero, infinity and NaN stay as they are
          const int e = static_cast<int>(__float_as_uint(top) >> 23);
          float f = 1.0f;
          if (top != 0.0f && e < 255) {
            const int s = min(140 - max(e, 1), 124);
            f = __uint_as_float(static_cast<uint32_t>(max(s, -125) + 127) << 23);
          }
          unit[r] = 1.0f / f;
#pragma unroll
          for (int i = 0; i < 2 * kSteps; ++i)
            w[i] = pack16<true>(__uint_as_float(w[i] << 16) * f, __uint_as_float(w[i] & 0xffff0000u) * f);
        }
      }
    }
    const float k_scale = CODES ? paged::head_scale(p.c.k_amax, p.c.amax_stride, h) : 1.0f;
    const float v_scale = CODES ? paged::head_scale(p.c.v_amax, p.c.amax_stride, h) : 1.0f;
    const float log2_scale = p.scale * k_scale * 1.4426950408889634f;
    float sl[BLOCKS8][2];                               // of heads 2 t and 2 t + 1, the columns of this lane's products
#pragma unroll
    for (int r = 0; r < BLOCKS8; ++r)
#pragma unroll
      for (int e = 0; e < 2; ++e) sl[r][e] = log2_scale * __shfl_sync(0xffffffffu, unit[r], (2 * t + e) * 4);

    // ------------------------------------------------------------- the keys
    float o[BLOCKS8][kSteps][4];                        // O^T: rows of 16 elements, heads 2 t and 2 t + 1
    float m[BLOCKS8][2], most[BLOCKS8][2], l[BLOCKS8][2];     // reference, up to which logit it stays, sum
#pragma unroll
    for (int r = 0; r < BLOCKS8; ++r) {
#pragma unroll
      for (int i = 0; i < kSteps; ++i) o[r][i][0] = o[r][i][1] = o[r][i][2] = o[r][i][3] = 0.0f;
      m[r][0] = m[r][1] = most[r][0] = most[r][1] = -INFINITY, l[r][0] = l[r][1] = 0.0f;
    }
    bool any = false;
    int slot = 0;                                       // of the tile that is requested; the next one holds the oldest
#pragma unroll 1
    for (int ahead = tile0; ahead < tile1 + S::kDepth - 1; ++ahead) {
      if (ahead < tile1) issue(slot, page0);
      copy_commit();                                // an empty group behind the last tile
      page0 = page1, page1 = page2, page2 = find_page(ahead + 3);
      slot = slot + 1 == S::kDepth ? 0 : slot + 1;
      const int tile = ahead - (S::kDepth - 1);
      if (tile < tile0) continue;
      copy_wait<S::kDepth - 1>();
      __syncwarp();
      const uint32_t ks = ring_u32 + slot * S::kBytes, vs = ks + kKeys * S::kRowBytes, keys = there[warp][slot];
      any = any || keys != 0;
      // S^T: keys g and g + 8, heads 2 t and 2 t + 1; two chains of sums, the products of one wait for each other
      float x[BLOCKS8][4], y[BLOCKS8][4];
#pragma unroll
      for (int r = 0; r < BLOCKS8; ++r) x[r][0] = x[r][1] = x[r][2] = x[r][3] = y[r][0] = y[r][1] = y[r][2] = y[r][3] = 0.0f;
#pragma unroll
      for (int i = 0; i < kSteps / (CODES ? 4 : 2); ++i) {
        const uint4 u = lds128(ks + g * S::kRowBytes + S::k_chunk(g, i * 4 + t) * 16);
        const uint4 v = lds128(ks + (g + 8) * S::kRowBytes + S::k_chunk(g + 8, i * 4 + t) * 16);
        if constexpr (CODES) {
          const uint32_t uw[4] = {u.x, u.y, u.z, u.w}, vw[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            uint32_t a[4];
            widen(uw[e], a[0], a[2]);
            widen(vw[e], a[1], a[3]);
#pragma unroll
            for (int r = 0; r < BLOCKS8; ++r) mma<kHalf>(e & 1 ? y[r] : x[r], a, q[r][i * 4 + e][0], q[r][i * 4 + e][1]);
          }
        } else {
          const uint32_t a0[4] = {u.x, v.x, u.y, v.y}, a1[4] = {u.z, v.z, u.w, v.w};
#pragma unroll
          for (int r = 0; r < BLOCKS8; ++r) {
            mma<kHalf>(x[r], a0, q[r][i * 2][0], q[r][i * 2][1]);
            mma<kHalf>(y[r], a1, q[r][i * 2 + 1][0], q[r][i * 2 + 1][1]);
          }
        }
      }
      const bool there0 = (keys >> g) & 1, there1 = (keys >> (g + 8)) & 1;
      uint32_t pt[BLOCKS8][2];
#pragma unroll
      for (int r = 0; r < BLOCKS8; ++r) {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[r][e] = (e < 2 ? there0 : there1) ? (x[r][e] + y[r][e]) * sl[r][e & 1] : -INFINITY;
        if (p.logits != nullptr) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int i = tile * kTile + warp * kKeys + g + 8 * (e >> 1), row = 8 * r + 2 * t + (e & 1);
            if (row < rows && i < see.seen && see.token(i) < p.weights_len)
              p.logits[(static_cast<int64_t>(b) * p.Hq + head0 + row) * p.logits_stride + i] = x[r][e];
          }
        }
        // the reference stays while no logit is too far above it: sums and P hold that, and the exchange among lanes is rare
        if (__any_sync(0xffffffffu, fmaxf(x[r][0], x[r][2]) > most[r][0] || fmaxf(x[r][1], x[r][3]) > most[r][1])) {
          const float m0 = fmaxf(m[r][0], R::of(column_max(fmaxf(x[r][0], x[r][2])))), m1 = fmaxf(m[r][1], R::of(column_max(fmaxf(x[r][1], x[r][3]))));
          const float f0 = m0 == -INFINITY ? 1.0f : exp2_fast(m[r][0] - m0), f1 = m1 == -INFINITY ? 1.0f : exp2_fast(m[r][1] - m1);
          l[r][0] *= f0, l[r][1] *= f1, m[r][0] = m0, m[r][1] = m1, most[r][0] = R::most(m0), most[r][1] = R::most(m1);
#pragma unroll
          for (int i = 0; i < kSteps; ++i) o[r][i][0] *= f0, o[r][i][1] *= f1, o[r][i][2] *= f0, o[r][i][3] *= f1;
        }
        const float base0 = m[r][0] == -INFINITY ? 0.0f : m[r][0], base1 = m[r][1] == -INFINITY ? 0.0f : m[r][1];
        x[r][0] = exp2_fast(x[r][0] - base0), x[r][1] = exp2_fast(x[r][1] - base1);
        x[r][2] = exp2_fast(x[r][2] - base0), x[r][3] = exp2_fast(x[r][3] - base1);
        l[r][0] += x[r][0] + x[r][2], l[r][1] += x[r][1] + x[r][3];
        pt[r][0] = transpose8x8(pack16<kHalf>(x[r][0], x[r][1]));
        pt[r][1] = transpose8x8(pack16<kHalf>(x[r][2], x[r][3]));
      }
      if constexpr (CODES) {
        constexpr int kWords = DPAD / 32;           // of the row pieces that this lane widens
        uint32_t w[4][kWords];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int key = t * 2 + (k & 1) + (k >> 1) * 8;
          if constexpr (DPAD == 128) {
            const uint4 u = lds128(vs + key * S::kRowBytes + S::v_chunk(key, g) * 16);
            w[k][0] = u.x, w[k][1] = u.y, w[k][2] = u.z, w[k][3] = u.w;
          } else {
            const uint2 u = lds64(vs + key * S::kRowBytes + S::v_chunk(key, g >> 1) * 16 + (g & 1) * 8);
            w[k][0] = u.x, w[k][1] = u.y;
          }
        }
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
          const uint32_t lo0 = __byte_perm(w[0][i], w[1][i], 0x5140), hi0 = __byte_perm(w[0][i], w[1][i], 0x7362);
          const uint32_t lo1 = __byte_perm(w[2][i], w[3][i], 0x5140), hi1 = __byte_perm(w[2][i], w[3][i], 0x7362);
          uint32_t a0[4], a1[4];
          widen(lo0, a0[0], a0[1]), widen(lo1, a0[2], a0[3]);
          widen(hi0, a1[0], a1[1]), widen(hi1, a1[2], a1[3]);
#pragma unroll
          for (int r = 0; r < BLOCKS8; ++r) {
            mma<kHalf>(o[r][2 * i], a0, pt[r][0], pt[r][1]);
            mma<kHalf>(o[r][2 * i + 1], a1, pt[r][0], pt[r][1]);
          }
        }
      } else {
        const int key = (lane & 7) + ((lane >> 4) & 1) * 8;
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
          uint32_t a[4];
          ldmatrix_trans(vs + key * S::kRowBytes + S::v_chunk(key, 2 * i + ((lane >> 3) & 1)) * 16, a);
#pragma unroll
          for (int r = 0; r < BLOCKS8; ++r) mma<kHalf>(o[r][i], a, pt[r][0], pt[r][1]);
        }
      }
      __syncwarp();
    }

    // ------------------------------------------------------------- the four warps' parts together
    float* mine = reinterpret_cast<float*>(ring);     // rows of DPAD: the ring is empty
#pragma unroll
    for (int r = 0; r < BLOCKS8; ++r)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = 8 * r + 2 * t + e;
        const float sum = column_sum(l[r][e]);
        if (g == 0) row_max[warp][row] = m[r][e], row_sum[warp][row] = any ? sum : -1.0f;   // -1: no key at all
#pragma unroll
        for (int i = 0; i < kSteps; ++i)
#pragma unroll
          for (int half = 0; half < 2; ++half)
            mine[row * DPAD + (CODES ? g * (DPAD / 8) + 2 * i + half : 16 * i + 8 * half + g)] = o[r][i][2 * half + e];
      }
    __syncthreads();
    const bool whole = tile0 == 0 && tile1 == tiles;
    // CTAs that share the item: c0 .. c1, those with a piece of it; the counter of the one that begins it
    const int c0 = whole ? cta : holder(total, item_start, ctas), c1 = whole ? cta : holder(total, item_end - 1, ctas);
    float* part = p.parts + (static_cast<int64_t>(cta) * 2 + (at == first_tile ? 0 : 1)) * kPart;
    constexpr int kQuads = DPAD / 4;
    for (int i = tid; i < rows * kQuads; i += kThreads) {
      const int row = i / kQuads, d = (i % kQuads) * 4;
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) top = fmaxf(top, row_max[w][row]);
      const float base = top == -INFINITY ? 0.0f : top;
      float sum = 0.0f, acc[4] = {};
      bool has = false;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        if (row_sum[w][row] < 0.0f) continue;
        has = true;
        const float f = exp2_fast(row_max[w][row] - base);
        sum += row_sum[w][row] * f;
        const float4 v = *reinterpret_cast<const float4*>(smem + w * S::kDepth * S::kBytes + (row * DPAD + d) * 4);
        acc[0] += v.x * f, acc[1] += v.y * f, acc[2] += v.z * f, acc[3] += v.w * f;
      }
      if (whole) {
        if (d < p.c.D) {
          const float f = v_scale / sum;
          T* dst = static_cast<T*>(p.out) + (static_cast<int64_t>(b) * p.Hq + head0 + row) * p.c.D + d;
          uint2 r = make_uint2(0, 0);
          if (has) {
            r.x = pack16<std::is_same<T, __half>::value>(acc[0] * f, acc[1] * f);
            r.y = pack16<std::is_same<T, __half>::value>(acc[2] * f, acc[3] * f);
          }
          *reinterpret_cast<uint2*>(dst) = r;
        }
        if (d == 0 && p.lse != nullptr) p.lse[static_cast<int64_t>(b) * p.Hq + head0 + row] = has ? base + log2f(sum) : 0.0f;
      } else {
        *reinterpret_cast<float4*>(part + row * DPAD + d) = make_float4(acc[0], acc[1], acc[2], acc[3]);
        if (d == 0) part[kRows * DPAD + row] = top, part[kRows * DPAD + kRows + row] = has ? sum : -1.0f;
      }
    }
    // ------------------------------------------------------------- the CTAs' parts together, by the one that comes last
    // Many parts in two steps: 8 or 16 neighbours by the last of them, into the place of the first, then the groups.
    if (!whole) {
      const int more = c1 - c0, group = more < kGroupsFrom ? 0 : (more < 128 ? 3 : 4);     // log2 of the parts of a group, 0: no groups
      int lo = group > 0 ? c0 + ((cta - c0) >> group << group) : c0, hi = group > 0 ? min(lo + (1 << group) - 1, c1) : c1, step = 1;
#pragma unroll 1
      for (bool grouping = group > 0;; grouping = false) {
        __syncthreads();
        if (tid == 0) {
          __threadfence();                             // what the CTA has written, seen through the barrier, in front of the ticket
          unsigned* const ticket = p.tickets + (grouping ? kMaxCtas : 0) + lo;
          last_one = lo == hi || atomicAdd(ticket, 1u) == static_cast<unsigned>((hi - lo) >> (step > 1 ? group : 0));
          if (last_one && lo != hi) *ticket = 0;
        }
        __syncthreads();
        if (!last_one) break;
        __threadfence();
        const bool second = piece(total, c0, ctas) < item_start;     // the item is not the first that CTA c0 worked on
        for (int i = tid; i < rows * kQuads; i += kThreads) {
          const int row = i / kQuads, d = (i % kQuads) * 4;
          const int from = kRows * DPAD + (step > 1 ? 2 * kRows : 0) + row;        // of the maxima
          float top = -INFINITY, sum = 0.0f, acc[4] = {};
          bool has = false;
          constexpr int kAtOnce = 8;
#pragma unroll 1
          for (int c = lo; c <= hi; c += kAtOnce * step) {
            float pm[kAtOnce], ps[kAtOnce];
            float4 v[kAtOnce];
#pragma unroll
            for (int k = 0; k < kAtOnce; ++k) {        // the loads first: they do not wait for one another
              ps[k] = -1.0f;
              const int of = c + k * step;
              if (of > hi) continue;
              const float* src = p.parts + (static_cast<int64_t>(of) * 2 + (of == c0 && second ? 1 : 0)) * kPart;
              pm[k] = __ldcg(src + from), ps[k] = __ldcg(src + from + kRows);
              v[k] = __ldcg(reinterpret_cast<const float4*>(src + row * DPAD + d));
            }
#pragma unroll
            for (int k = 0; k < kAtOnce; ++k) {
              if (ps[k] < 0.0f) continue;
              has = true;
              const float now = fmaxf(top, pm[k]), base = now == -INFINITY ? 0.0f : now, f0 = exp2_fast(top - base), f1 = exp2_fast(pm[k] - base);
              sum = sum * f0 + ps[k] * f1;
              acc[0] = acc[0] * f0 + v[k].x * f1, acc[1] = acc[1] * f0 + v[k].y * f1;
              acc[2] = acc[2] * f0 + v[k].z * f1, acc[3] = acc[3] * f0 + v[k].w * f1;
              top = now;
            }
          }
          if (grouping) {
            float* dst = p.parts + (static_cast<int64_t>(lo) * 2 + (lo == c0 && second ? 1 : 0)) * kPart;
            *reinterpret_cast<float4*>(dst + row * DPAD + d) = make_float4(acc[0], acc[1], acc[2], acc[3]);
            if (d == 0) dst[kRows * DPAD + 2 * kRows + row] = top, dst[kRows * DPAD + 3 * kRows + row] = has ? sum : -1.0f;
            continue;
          }
          if (d < p.c.D) {
            const float f = v_scale / sum;
            T* dst = static_cast<T*>(p.out) + (static_cast<int64_t>(b) * p.Hq + head0 + row) * p.c.D + d;
            uint2 r = make_uint2(0, 0);
            if (has) {
              r.x = pack16<std::is_same<T, __half>::value>(acc[0] * f, acc[1] * f);
              r.y = pack16<std::is_same<T, __half>::value>(acc[2] * f, acc[3] * f);
            }
            *reinterpret_cast<uint2*>(dst) = r;
          }
          if (d == 0 && p.lse != nullptr)
            p.lse[static_cast<int64_t>(b) * p.Hq + head0 + row] = has ? (top == -INFINITY ? 0.0f : top) + log2f(sum) : 0.0f;
        }
        if (!grouping) break;
        lo = c0, hi = c0 + (more >> group << group), step = 1 << group;
      }
    }
    __syncthreads();
    at += tile1 - tile0;
    if (at >= end) break;
    item_start = item_end;
    if (++block == p.blocks) {
      block = 0;
      if (++h == p.c.heads) h = 0, see = keys_seen(p, ++b);
    }
  }
}

// weights[b, h, token] += sum over the query heads of P, from the logits that the kernel above left and their normalisers.
__global__ void __launch_bounds__(256) weights_kernel(const __grid_constant__ DecodeParams p, float* weights) {
  pdl_launch_dependents();
  pdl_wait();
  const int b = blockIdx.z, h = blockIdx.y;
  const Seen see = keys_seen(p, b);
  const int64_t first = static_cast<int64_t>(b) * p.Hq + h * p.group;
  float* w = weights + (static_cast<int64_t>(b) * p.c.heads + h) * p.weights_len;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < see.seen; i += static_cast<int64_t>(gridDim.x) * 256) {
    const int token = see.token(static_cast<int>(i));
    if (token >= p.weights_len) return;
    const float old = w[token];            // read beside the logits, not behind them (1 us of 41)
    float sum = 0.0f;
    for (int g = 0; g < p.group; ++g) sum += exp2_fast(p.logits[(first + g) * p.logits_stride + i] - p.lse[first + g]);
    w[token] = old + sum;
  }
}

template <typename T, bool CODES, int DPAD, int BLOCKS8>
int launch_decode(const DecodeParams& p, int64_t most_tiles, cudaStream_t st) {
  using S = Stage<CODES, DPAD, BLOCKS8>;
  constexpr int kSmem = kWarps * S::kDepth * S::kBytes;
  static_assert(S::kDepth * S::kBytes >= 8 * BLOCKS8 * DPAD * 4, "a warp's result takes its ring");
  auto kernel = decode_kernel<T, CODES, DPAD, BLOCKS8>;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return B200Q_ERR_CUDA;
  static std::atomic<int> resident[64];                // CTAs that one SM holds; 0: not asked yet
  int per_sm = dev >= 0 && dev < 64 ? resident[dev].load(std::memory_order_relaxed) : 0;
  if (per_sm == 0) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem) != cudaSuccess) return B200Q_ERR_CUDA;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, kThreads, kSmem) != cudaSuccess || per_sm < 1) return B200Q_ERR_CUDA;
    if (dev >= 0 && dev < 64) resident[dev].store(per_sm, std::memory_order_relaxed);
  }
  int64_t ctas = static_cast<int64_t>(per_sm) * sm_count();
  ctas = ctas < kMaxCtas ? ctas : kMaxCtas;
  ctas = ctas < most_tiles ? ctas : most_tiles;
  if (launch_pdl(kernel, dim3(static_cast<unsigned>(ctas)), dim3(kThreads), kSmem, st, p) != cudaSuccess) return B200Q_ERR_CUDA;
  return check_launch();
}

template <typename T, bool CODES>
int launch_decode_d(const DecodeParams& p, int64_t most_tiles, cudaStream_t st) {
  if (p.rows <= 8) return p.c.D <= 64 ? launch_decode<T, CODES, 64, 1>(p, most_tiles, st) : launch_decode<T, CODES, 128, 1>(p, most_tiles, st);
  return p.c.D <= 64 ? launch_decode<T, CODES, 64, 2>(p, most_tiles, st) : launch_decode<T, CODES, 128, 2>(p, most_tiles, st);
}

int64_t round4(int64_t n) { return (n + 3) / 4 * 4; }

}  // namespace
}  // namespace b200q

using namespace b200q;

extern "C" {

size_t b200q_paged_attention_workspace_bytes(void) { return 2 * kMaxCtas * sizeof(unsigned) + static_cast<size_t>(kMaxCtas) * 2 * kPart * sizeof(float); }

size_t b200q_paged_attention_scratch_bytes(int64_t B, int64_t Hq, int64_t keys) {
  if (B <= 0 || Hq <= 0 || keys < 0) return 16;
  return static_cast<size_t>(B * Hq) * (round4(keys) + 1) * sizeof(float) + 16;
}

int b200q_paged_attention(const void* q, int dtype, const int64_t* q_strides, const b200q_paged_cache* cache, const int32_t* block_table,
                          int64_t table_stride, int64_t table_width, const int32_t* lens, int64_t B, int64_t Hq, float scale,
                          int64_t window, int64_t sinks, void* out, float* weights, int64_t weights_len, void* workspace,
                          size_t workspace_bytes, void* scratch, size_t scratch_bytes, b200q_stream_t stream) {
  DecodeParams p{};
  if (int rc = paged::make_cache(&p.c, cache, dtype, block_table, table_stride, table_width, lens, B)) return rc;
  if (Hq <= 0 || Hq > 65535 || Hq % p.c.heads != 0 || sinks < 0 || !(scale >= 0.0f) || B > 65535) return B200Q_ERR_INVALID;
  if (B == 0) return B200Q_OK;
  if (q == nullptr || q_strides == nullptr || out == nullptr || (weights != nullptr && (weights_len < 0 || weights_len > 0x7fffff00LL)))
    return B200Q_ERR_INVALID;
  if (!aligned(q, 16) || !aligned(out, 16) || !paged::strides_ok(q_strides, 2, 8)) return B200Q_ERR_ALIGN;
  if (workspace == nullptr || workspace_bytes < b200q_paged_attention_workspace_bytes()) return B200Q_ERR_WORKSPACE;
  // keys that a token of the longest sequence in the table sees
  const int64_t most = window > 0 && sinks < (1LL << 40) && window < (1LL << 40) && window + sinks < p.c.capacity ? window + sinks : p.c.capacity;
  const int64_t keys = most < weights_len ? most : weights_len;
  if (weights != nullptr && (scratch == nullptr || scratch_bytes < b200q_paged_attention_scratch_bytes(B, Hq, keys))) return B200Q_ERR_WORKSPACE;
  if (!aligned(workspace, 16) || !aligned(scratch, 16)) return B200Q_ERR_ALIGN;
  if (int rc = check_arch()) return rc;
  p.page_shift = -1;
  if ((p.c.page_size & (p.c.page_size - 1)) == 0)
    for (p.page_shift = 0; (1 << p.page_shift) < p.c.page_size;) ++p.page_shift;
  p.one_layout = p.c.k.page == p.c.v.page && p.c.k.row == p.c.v.row;
  p.q = static_cast<const char*>(q);
  p.q_batch = q_strides[0] * 2, p.q_head = q_strides[1] * 2;
  p.out = out;
  p.B = static_cast<int>(B), p.Hq = static_cast<int>(Hq), p.group = static_cast<int>(Hq / p.c.heads);
  p.blocks = (p.group + kRows - 1) / kRows;
  p.rows = (p.group + p.blocks - 1) / p.blocks;
  p.blocks = (p.group + p.rows - 1) / p.rows;
  p.scale = scale;
  p.window = window, p.sinks = sinks;
  p.tickets = static_cast<unsigned*>(workspace);
  p.parts = reinterpret_cast<float*>(p.tickets + 2 * kMaxCtas);
  if (weights != nullptr && weights_len > 0) {
    p.logits_stride = round4(keys);
    p.weights_len = weights_len;
    p.logits = static_cast<float*>(scratch);
    p.lse = p.logits + B * Hq * p.logits_stride;
  }
  // no more CTAs than tiles
  const int64_t tiles = (most > 0 ? (most + kTile - 1) / kTile : 1) * B * p.c.heads * p.blocks;
  const auto st = static_cast<cudaStream_t>(stream);
  const int rc = dtype == B200Q_BF16 ? (p.c.codes ? launch_decode_d<__nv_bfloat16, true>(p, tiles, st) : launch_decode_d<__nv_bfloat16, false>(p, tiles, st))
                                     : (p.c.codes ? launch_decode_d<__half, true>(p, tiles, st) : launch_decode_d<__half, false>(p, tiles, st));
  if (rc != B200Q_OK || p.logits == nullptr) return rc;
  const int64_t chunks = (keys + 255) / 256;
  const dim3 grid(static_cast<unsigned>(chunks < 1 ? 1 : (chunks < 65535 ? chunks : 65535)), static_cast<unsigned>(p.c.heads), static_cast<unsigned>(B));
  if (launch_pdl(weights_kernel, grid, dim3(256), 0, st, p, weights) != cudaSuccess) return B200Q_ERR_CUDA;
  return check_launch();
}

}  // extern "C"
