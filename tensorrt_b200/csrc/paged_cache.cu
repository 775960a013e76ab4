// Rows in and out of the paged key-value cache: append and evict.
#include "paged.cuh"
#include "tcgen05.cuh"

namespace b200q {
namespace {

using paged::Cache;

struct AppendParams {
  Cache c;
  const char* k;
  const char* v;
  int64_t k_token, k_head, v_token, v_head;   // bytes
  const int32_t* cu_new;
  int64_t T;
  int B;
};

__device__ __forceinline__ int ld_i32(const int32_t* p) {
  int v;
  asm volatile("ld.global.b32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}

// A thread moves 16 elements of K and of V, read first; the pages of the CTA's tokens are found while they come: a warp
// looks for the sequence of its first token, whose other tokens it holds as well, and so on; then a lane finds the page of a token.
// Bound by the memory for prompts (9620 tokens of 8 heads of 128, bf16, 79 MB: 16.9 us, 4.7 TB/s; the copy rate gives 12.0), by three loads that
// wait for one another (lengths, table, rows) for a decode step (64 tokens 2.4 us, of which an empty launch is most).  Many small CTAs: two or
// four pieces a thread take the registers of others (18.4 and 21.8 us; pages first and four pieces 19.0), 256 threads 17.3, 64 threads 16.6 but
// more rounds for wide rows.  32000 tokens of one head of 64 to 8-bit pages 4.9 us; with a search to each token 12.2.
constexpr int kAppendThreads = 128, kAppendTokens = 64;
static_assert(kAppendTokens <= kAppendThreads, "a lane finds one token");

template <typename T, bool CODES>
__global__ void __launch_bounds__(kAppendThreads) append_kernel(const __grid_constant__ AppendParams p, int tokens) {
  __shared__ int2 place[kAppendTokens];       // page (-1: none) and row
  const int tid = threadIdx.x, lane = tid & 31;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * tokens;
  const int here = static_cast<int>(p.T - first < tokens ? p.T - first : tokens);
  pdl_launch_dependents();
  pdl_wait();
  auto find_places = [&] {
    const int share = (here + kAppendThreads / 32 - 1) / (kAppendThreads / 32), i = (tid >> 5) * share + lane;    // at most 32 tokens to a warp
    const bool mine = lane < share && i < here;
    const int t = static_cast<int>(first) + i;
    int b = t, at = 0, fresh = 1;
    if (p.cu_new != nullptr) {
      unsigned left = __ballot_sync(0xffffffffu, mine);
      while (left != 0) {                     // the sequence of the first token left, and all the tokens that it holds
        const int leader = __ffs(left) - 1, of = __shfl_sync(0xffffffffu, t, leader);
        int lo = 0, span = p.B;               // the last that begins at or before it, 32 candidates a step: one of lo .. lo + span - 1
        while (span > 1) {
          const int step = (span + 31) / 32, probe = lo + lane * step;
          const unsigned below = __ballot_sync(0xffffffffu, lane * step < span && ld_i32(p.cu_new + min(probe, p.B)) <= of);
          const int last = 31 - __clz(below | 1u);
          span = min(step, span - last * step);
          lo += last * step;
        }
        const int begin = ld_i32(p.cu_new + lo), end = ld_i32(p.cu_new + lo + 1);
        const bool here_too = lane == leader || ((left >> lane) & 1 && t < end);
        if (here_too) b = lo, at = t - begin, fresh = end - begin;
        left &= ~__ballot_sync(0xffffffffu, here_too);
      }
    }
    if (mine) {
      const int64_t token = static_cast<int64_t>(ld_i32(p.c.lens + b)) - fresh + at;
      int2 found = make_int2(-1, 0);
      if (at >= 0 && at < fresh && token >= 0 && token < p.c.capacity)      // else: a row that no sequence brings
        found = make_int2(paged::page_of(p.c.table + b * p.c.table_stride, static_cast<int>(token), p.c), static_cast<int>(token % p.c.page_size));
      place[i] = found;
    }
    __syncthreads();
  };
  const int parts = p.c.D / 16, per_token = p.c.heads * parts, all = here * per_token;
  for (int base = 0; base < all; base += kAppendThreads) {
    const int i = base + tid, token = i / per_token, rest = i - token * per_token, head = rest / parts, part = rest - head * parts;
    Raw16<T, false> kr, vr;
    if (i < all) {
      kr.load(reinterpret_cast<const T*>(p.k + (first + token) * p.k_token + head * p.k_head) + part * 16);
      vr.load(reinterpret_cast<const T*>(p.v + (first + token) * p.v_token + head * p.v_head) + part * 16);
    }
    if (base == 0) find_places();
    const int2 to = i < all ? place[token] : make_int2(-1, 0);
    if (to.x < 0) continue;
    char* const kd = paged::row_at(p.c.k, to.x, head, to.y);
    char* const vd = paged::row_at(p.c.v, to.x, head, to.y);
    if constexpr (CODES) {
      const float ks = paged::head_scale(p.c.k_amax, p.c.amax_stride, head), vs = paged::head_scale(p.c.v_amax, p.c.amax_stride, head);
      *reinterpret_cast<uint4*>(kd + part * 16) = e4m3_of_16(kr, ks, __frcp_rn(ks), ks * 512.0f, b200q_div_fast_ok(ks));
      *reinterpret_cast<uint4*>(vd + part * 16) = e4m3_of_16(vr, vs, __frcp_rn(vs), vs * 512.0f, b200q_div_fast_ok(vs));
    } else {
      uint4* const k4 = reinterpret_cast<uint4*>(kd + part * 32);
      uint4* const v4 = reinterpret_cast<uint4*>(vd + part * 32);
      const U32x8 &kw = kr.w[0], &vw = vr.w[0];
      k4[0] = make_uint4(kw.v[0], kw.v[1], kw.v[2], kw.v[3]), k4[1] = make_uint4(kw.v[4], kw.v[5], kw.v[6], kw.v[7]);
      v4[0] = make_uint4(vw.v[0], vw.v[1], vw.v[2], vw.v[3]), v4[1] = make_uint4(vw.v[4], vw.v[5], vw.v[6], vw.v[7]);
    }
  }
}

struct EvictParams {
  Cache c;
  const float* weights;
  int64_t L;
  const int32_t* out_table;
  int64_t out_stride;
  int64_t table_width;
  int keep, recent, sinks;
  int32_t* kept;
  int32_t* new_lens;
  float* new_weights;
  int row_bytes;
};

// Order of weights as unsigned numbers: larger weight, larger number; -0 and 0 are equal, NaN is -inf.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) w = -INFINITY;
  if (w == 0.0f) w = 0.0f;
  const uint32_t u = __float_as_uint(w);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Which tokens stay.  A cluster of CTAs per sequence and kv head, each with a part of the tokens, their keys in shared memory (up to
// kHeldKeys, else read again on each walk).  Sinks and recent tokens have a key above all others, so the m largest keys stay.  The m-th
// largest key is found eight bits at a time, from the top: every CTA counts the digits of its keys that agree with the bits found so
// far and writes the counts into every CTA of the cluster (reading the others' from there instead takes 1850 clocks a digit, not 400);
// one warp adds them, and all CTAs step to the same digit, up to the digit whose keys all stay.  Lanes count in 16 columns: attention
// weights share a few exponents, and 32 lanes adding to the same few words wait for one another; 8 columns are no faster.
// The counts also say how many tokens a CTA keeps in front of the next, so that two more walks in the order of the tokens, a run of them
// to each warp, write the list; a weight is its key read backwards, since a load from memory in that loop takes 5000 clocks in all.
// Bound by latency and, since all of it runs a few times only, by the size of the code: what unrolling more loops saves is lost to
// instruction fetches (34.6 us for the first of these calls became 40.3).  32000 tokens to 8192, 8 heads: about 19 us of the call's 32.3 (clusters of 4: 5 us
// more); 24 sequences of 1500 to 6000 to 2048, 8 heads: 19 of 53.7.  Of 30000 clocks there 17000 are the four digits, 7000 the keys.  The table
// is looked through for pages that are not there: 0.3 us of either call, 2 us more where its entries are read behind the length.
constexpr int kSelectThreads = 512, kSelectWarps = kSelectThreads / 32, kMaxCluster = 8, kColumns = 16;
constexpr uint32_t kStays = 0xffffffffu, kLowest = 0x007fffffu, kZero = 0x80000000u;      // no weight's key; that of -inf and NaN; that of 0 and -0

__device__ __forceinline__ int ld_cluster_i32(const int* p, unsigned cta) {
  int v;
  asm volatile("ld.shared::cluster.b32 %0, [%1];" : "=r"(v) : "r"(ptx::mapa_u32(ptx::smem_u32(p), cta)) : "memory");
  return v;
}
__device__ __forceinline__ void st_cluster_i32(int* p, unsigned cta, int v) {
  asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(ptx::mapa_u32(ptx::smem_u32(p), cta)), "r"(v) : "memory");
}
__device__ __forceinline__ float ld_f32(const float* p) {
  float v;
  asm volatile("ld.global.f32 %0, [%1];" : "=f"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ unsigned cluster_size() {
  unsigned r;
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(r));
  return r;
}

// What fits beside the counts: 320 rows of 45000 keys, one CTA to an SM, 187 us a call, 242 from memory; of 30 x 16 rows of 15000 93 and 138.
constexpr int kHeldKeys = 49152;
template <bool HELD>
__global__ void __launch_bounds__(kSelectThreads) evict_select_kernel(const __grid_constant__ EvictParams p) {
  extern __shared__ __align__(16) uint32_t keys[];  // HELD: those of the part, zeros up to a multiple of 4
  __shared__ __align__(16) int columns[256 * kColumns];       // [digit][lane & 15]
  __shared__ __align__(16) int counts[2][kMaxCluster][256];   // [round & 1][CTA][255 - digit], written by the CTA that they are of
  __shared__ int found[4];                          // digit; how many of its keys are wanted; this CTA's keys above it; its own of them if all stay, else -1
  __shared__ int published[2];                      // of this CTA's part: tokens kept for sure, keys equal to the smallest kept key
  __shared__ int warp_sum[2][kSelectWarps];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = static_cast<int>(ptx::cluster_ctarank()), ctas = static_cast<int>(cluster_size());
  const int b = blockIdx.y, h = blockIdx.x / ctas;
  for (int i = tid; i < 256 * kColumns / 4; i += kSelectThreads) reinterpret_cast<int4*>(columns)[i] = make_int4(0, 0, 0, 0);
  pdl_launch_dependents();
  pdl_wait();
  // Tokens whose page the table does not name are not there, so they are not among those that stay: their key is zero, below every weight's.
  // The first entries are read beside the length, not behind it.
  constexpr int kAhead = 4;
  const int32_t* const table = p.c.table + b * p.c.table_stride;
  int entry[kAhead], gone = 0;
#pragma unroll
  for (int u = 0; u < kAhead; ++u) entry[u] = tid + u * kSelectThreads < p.table_width ? ld_i32(table + tid + u * kSelectThreads) : 0;
  const int n = paged::cached_tokens(p.c, b, p.L);
  const int64_t line = static_cast<int64_t>(b) * p.c.heads + h;
  auto gone_of = [&](int64_t i, int page) {
    const int64_t left = n - i * p.c.page_size;
    return left > 0 && static_cast<unsigned>(page) >= static_cast<unsigned>(p.c.num_pages) ? static_cast<int>(left < p.c.page_size ? left : p.c.page_size) : 0;
  };
#pragma unroll
  for (int u = 0; u < kAhead; ++u) gone += gone_of(tid + u * kSelectThreads, entry[u]);
#pragma unroll 1
  for (int64_t i = tid + kAhead * kSelectThreads; i * p.c.page_size < n; i += kSelectThreads) gone += gone_of(i, ld_i32(table + i));
  const bool holes = __syncthreads_or(gone);
  if (holes) {
    gone = __reduce_add_sync(0xffffffffu, gone);
    if (lane == 0) warp_sum[0][warp] = gone;
    __syncthreads();
    gone = 0;
    for (int i = 0; i < kSelectWarps; ++i) gone += warp_sum[0][i];
  }
  const int m = min(n - gone, p.keep);
  const float* w = p.weights + line * p.L;
  float* nw = p.new_weights + line * p.L;
  int32_t* kept = p.kept + line * p.keep;
  if (h == 0 && rank == 0 && tid == 0) p.new_lens[b] = m;
  const int part = (n + ctas - 1) / ctas, t0 = min(rank * part, n), size = min(t0 + part, n) - t0;
  const int c0 = min(p.sinks, n) - t0, c1 = max(p.sinks, n - p.recent) - t0;      // the others of the part stay
  auto weight_at = [&](int i) { return (i >= c0) & (i < c1) ? weight_key(ld_f32(w + t0 + i)) : kStays; };
  auto key_at = [&](int i) { return holes && paged::page_of(table, t0 + i, p.c) < 0 ? 0u : weight_at(i); };
  auto key_of = [&](int i) { return HELD ? keys[i] : key_at(i); };
  if (m == n) {                                     // the same for the whole cluster
#pragma unroll 4
    for (int i = tid; i < size; i += kSelectThreads) kept[t0 + i] = t0 + i, nw[t0 + i] = ld_f32(w + t0 + i);
  } else if (HELD) {
#pragma unroll 4
    for (int i = tid; i < size; i += kSelectThreads) keys[i] = weight_at(i);
    if (holes)
#pragma unroll 1
      for (int i = tid; i < size; i += kSelectThreads)
        if (paged::page_of(table, t0 + i, p.c) < 0) keys[i] = 0;
    if (tid < (-size & 3)) keys[size + tid] = 0;
  }
  for (int64_t j = m + rank * kSelectThreads + tid; j < p.keep; j += ctas * kSelectThreads) kept[j] = -1;
  for (int64_t j = m + rank * kSelectThreads + tid; j < p.L; j += ctas * kSelectThreads) nw[j] = 0.0f;
  if (m == n || m == 0) return;
  if (ctas > 1) ptx::cluster_sync(); else __syncthreads();           // the others run, and may be written to
  uint32_t least = 0, agree = 0;                // the bits found, and which they are
  int left = m, above = 0, equals = 0;          // wanted among the keys that agree so far; this part's keys above them, and of those that agree
#pragma unroll 1
  for (int d = 0; d < 4; ++d) {
    const int shift = 24 - 8 * d;
    auto count = [&](uint32_t key) {
      if ((key & agree) == least) atomicAdd(&columns[((key >> shift) & 255) * kColumns + (lane & (kColumns - 1))], 1);
    };
    if (HELD) {
#pragma unroll 1
      for (int i = tid; i < (size + 3) / 4; i += kSelectThreads) {
        const uint4 four = reinterpret_cast<const uint4*>(keys)[i];
        count(four.x), count(four.y), count(four.z), count(four.w);
      }
    } else {
#pragma unroll 4
      for (int i = tid; i < size; i += kSelectThreads) count(key_at(i));
    }
    __syncthreads();
    {                                           // two threads to a digit, half of its columns each, turned so that no two meet a bank; cleared for the next
      int4* mine = reinterpret_cast<int4*>(columns) + tid * 2;
      int sum = 0;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        int4* at = mine + (i ^ ((tid >> 2) & 1));
        const int4 v = *at;
        *at = make_int4(0, 0, 0, 0);
        sum += v.x + v.y + v.z + v.w;
      }
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      int* const slot = &counts[d & 1][rank][255 - (tid >> 1)];       // the largest digit first
      if (ctas == 1) {
        if ((tid & 1) == 0) *slot = sum;
      } else {
#pragma unroll 1
        for (int r = tid & 1; r < ctas; r += 2) st_cluster_i32(slot, r, sum);
      }
    }
    if (ctas > 1) ptx::cluster_sync(); else __syncthreads();
    if (warp == 0) {                            // a lane has eight digits: their keys, here and in the cluster, and those of the lanes in front
      int own[8], all[8] = {};
#pragma unroll 1
      for (int r = 0; r < ctas; ++r) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int4 v = *reinterpret_cast<const int4*>(&counts[d & 1][r][lane * 8 + i * 4]);
          const int of[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            all[4 * i + j] += of[j];
            if (r == rank) own[4 * i + j] = of[j];
          }
        }
      }
      int own_up = 0, all_up = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) own_up += own[i], all_up += all[i];
      const int own_sum = own_up, all_sum = all_up;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, own_up, o), y = __shfl_up_sync(0xffffffffu, all_up, o);
        if (lane >= o) own_up += x, all_up += y;
      }
      own_up -= own_sum, all_up -= all_sum;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (all_up < left && left <= all_up + all[i]) {
          const int rest = left - all_up;
          found[0] = 255 - lane * 8 - i, found[1] = rest, found[2] = own_up, found[3] = rest == all[i] ? own[i] : -1;
        }
        own_up += own[i], all_up += all[i];
      }
    }
    __syncthreads();
    left = found[1];
    above += found[2];
    least |= static_cast<uint32_t>(found[0]) << shift;
    if (found[3] >= 0) {                        // every key with these bits stays: nothing is left to tell apart
      above += found[3], left = 0;
      break;
    }
    agree |= 255u << shift;
    equals = counts[d & 1][rank][255 - found[0]];
  }
  if (tid == 0) published[0] = above, published[1] = left > 0 ? equals : 0;
  // each warp a run of the part, 32 tokens at a time
  const bool some = left > 0;                   // of the keys that equal the least, the first `left` stay
  const int run = ((size + kSelectWarps - 1) / kSelectWarps + 31) & ~31, r0 = min(warp * run, size), r1 = min(r0 + run, size);
  auto classify = [&](int i, unsigned* sure_lanes, unsigned* equal_lanes) {
    const bool inside = i < r1;
    const uint32_t key = key_of(min(i, size - 1));
    const bool equal = key == least && some;
    *sure_lanes = __ballot_sync(0xffffffffu, inside && key >= least && !equal);
    *equal_lanes = __ballot_sync(0xffffffffu, inside && equal);
    return key;
  };
  int my_sure = 0, my_equal = 0;
#pragma unroll 1
  for (int base = r0; base < r1; base += 32) {
    unsigned as, es;
    classify(base + lane, &as, &es);
    my_sure += __popc(as), my_equal += __popc(es);
  }
  if (lane == 0) warp_sum[0][warp] = my_sure, warp_sum[1][warp] = my_equal;
  if (ctas > 1) ptx::cluster_sync(); else __syncthreads();
  int sure = 0, equal = 0;                      // in the parts and runs in front
#pragma unroll
  for (int r = 0; r < kMaxCluster - 1; ++r)
    if (r < rank) sure += ld_cluster_i32(&published[0], r), equal += ld_cluster_i32(&published[1], r);
  for (int i = 0; i < warp; ++i) sure += warp_sum[0][i], equal += warp_sum[1][i];
#pragma unroll 1
  for (int base = r0; base < r1; base += 32) {
    unsigned as, es;
    const uint32_t key = classify(base + lane, &as, &es);
    const unsigned me = 1u << lane, below = me - 1;
    const int eq = equal + __popc(es & below);  // equal keys in front; the first `left` stay
    if (((as & me) != 0) | (((es & me) != 0) & (eq < left))) {
      const int at = sure + __popc(as & below) + min(eq, left);
      float weight = __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
      if (key == kStays || key == kLowest || key == kZero) weight = ld_f32(w + t0 + base + lane);
      kept[at] = t0 + base + lane, nw[at] = weight;
    }
    sure += __popc(as), equal += __popc(es);
  }
  if (ctas > 1) ptx::cluster_sync();            // nobody leaves while its counts may still be read
}

// The kept rows to their new pages: 16 bytes of K and of V a thread and row, two rows at once.  Bound by the memory
// (24 x 8 heads, 2048 rows of 128 bytes, 200 MB: 34 us, 5.9 TB/s).  Four rows at once take registers from other CTAs (the two calls 34.8 and
// 56.5 us, not 31.4 and 52.9), one leaves too little on its way (31.1 and 56.6).
constexpr int kMoveThreads = 128, kMoveRows = 2;
__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(const __grid_constant__ EvictParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int b = blockIdx.z, h = blockIdx.y;
  const int m = min(paged::cached_tokens(p.c, b, p.L), p.keep);
  const int pieces = p.row_bytes / 16, per = kMoveThreads / pieces;       // rows that the CTA takes at once
  const int r = static_cast<int>(threadIdx.x) / pieces, piece = (static_cast<int>(threadIdx.x) % pieces) * 16;
  const int32_t* kept = p.kept + (static_cast<int64_t>(b) * p.c.heads + h) * p.keep;
  const int32_t* from = p.c.table + b * p.c.table_stride;
  const int32_t* to = p.out_table + b * p.out_stride;
  if (r >= per) return;
  const int first = static_cast<int>(blockIdx.x) * per * kMoveRows + r;
  uint4 kv[kMoveRows], vv[kMoveRows];
  int token[kMoveRows], sp[kMoveRows], dp[kMoveRows];
#pragma unroll
  for (int u = 0; u < kMoveRows; ++u) {
    const int j = first + u * per;
    token[u] = j < m ? ld_i32(kept + j) : -1;
  }
#pragma unroll
  for (int u = 0; u < kMoveRows; ++u) {
    sp[u] = token[u] >= 0 ? paged::page_of(from, token[u], p.c) : -1;
    dp[u] = token[u] >= 0 ? paged::page_of(to, first + u * per, p.c) : -1;
    if (dp[u] < 0) sp[u] = -1;
  }
#pragma unroll
  for (int u = 0; u < kMoveRows; ++u)
    if (sp[u] >= 0) {
      const int row = token[u] % p.c.page_size;
      kv[u] = ld_128(paged::row_at(p.c.k, sp[u], h, row) + piece);
      vv[u] = ld_128(paged::row_at(p.c.v, sp[u], h, row) + piece);
    }
#pragma unroll
  for (int u = 0; u < kMoveRows; ++u)
    if (sp[u] >= 0) {
      const int row = (first + u * per) % p.c.page_size;
      *reinterpret_cast<uint4*>(paged::row_at(p.c.k, dp[u], h, row) + piece) = kv[u];
      *reinterpret_cast<uint4*>(paged::row_at(p.c.v, dp[u], h, row) + piece) = vv[u];
    }
}

}  // namespace
}  // namespace b200q

using namespace b200q;

extern "C" {

int b200q_paged_append(const void* k, const void* v, int dtype, const int64_t* strides, int64_t T, const int32_t* cu_new,
                       const b200q_paged_cache* cache, const int32_t* block_table, int64_t table_stride, int64_t table_width,
                       const int32_t* lens, int64_t B, b200q_stream_t stream) {
  AppendParams p{};
  if (int rc = paged::make_cache(&p.c, cache, dtype, block_table, table_stride, table_width, lens, B)) return rc;
  if (T < 0 || T > 0x7fffffffLL || (cu_new == nullptr && T != B) || (B == 0 && T != 0)) return B200Q_ERR_INVALID;
  if (T == 0 || table_width == 0) return B200Q_OK;
  if (k == nullptr || v == nullptr || strides == nullptr) return B200Q_ERR_INVALID;
  if (!aligned(k, 16) || !aligned(v, 16) || !paged::strides_ok(strides, 4, 8)) return B200Q_ERR_ALIGN;
  if (int rc = check_arch()) return rc;
  p.k = static_cast<const char*>(k);
  p.v = static_cast<const char*>(v);
  p.k_token = strides[0] * 2, p.k_head = strides[1] * 2, p.v_token = strides[2] * 2, p.v_head = strides[3] * 2;
  p.cu_new = cu_new;
  p.T = T;
  p.B = static_cast<int>(B);
  const auto st = static_cast<cudaStream_t>(stream);
  // tokens of a CTA: what keeps its threads busy once, fewer where that leaves SMs without a CTA
  const int64_t pieces = static_cast<int64_t>(p.c.heads) * (p.c.D / 16), fill = kAppendThreads / pieces, spread = T / (2 * sm_count());
  int64_t tokens = fill < spread ? fill : spread;
  tokens = tokens < 1 ? 1 : (tokens > kAppendTokens ? kAppendTokens : tokens);
  const dim3 grid(static_cast<unsigned>((T + tokens - 1) / tokens)), block(kAppendThreads);
  const int n = static_cast<int>(tokens);
  const bool half = dtype == B200Q_F16;
  cudaError_t e;
  if (p.c.codes) e = half ? launch_pdl(append_kernel<__half, true>, grid, block, 0, st, p, n) : launch_pdl(append_kernel<__nv_bfloat16, true>, grid, block, 0, st, p, n);
  else e = half ? launch_pdl(append_kernel<__half, false>, grid, block, 0, st, p, n) : launch_pdl(append_kernel<__nv_bfloat16, false>, grid, block, 0, st, p, n);
  return e == cudaSuccess ? check_launch() : B200Q_ERR_CUDA;
}

int b200q_paged_evict(const b200q_paged_cache* cache, const int32_t* block_table, int64_t table_stride, int64_t table_width,
                      const int32_t* lens, const float* weights, int64_t weights_len, const int32_t* out_table, int64_t out_stride,
                      int64_t out_width, int64_t B, int64_t keep, int64_t recent, int64_t sinks, int32_t* kept, int32_t* new_lens,
                      float* new_weights, b200q_stream_t stream) {
  EvictParams p{};
  if (int rc = paged::make_cache(&p.c, cache, -1, block_table, table_stride, table_width, lens, B)) return rc;
  if (keep < 0 || recent < 0 || sinks < 0 || recent + sinks > keep || weights_len < keep || weights_len > 0x7fffff00LL) return B200Q_ERR_INVALID;
  if (out_width < 0 || out_width > 0x7fffffffLL || out_stride < 0 || out_width * p.c.page_size < keep) return B200Q_ERR_INVALID;
  if (B > 65535) return B200Q_ERR_INVALID;
  if (B == 0) return B200Q_OK;
  if (new_lens == nullptr || (weights_len > 0 && (weights == nullptr || new_weights == nullptr || new_weights == weights))) return B200Q_ERR_INVALID;
  if (keep > 0 && (kept == nullptr || out_table == nullptr)) return B200Q_ERR_INVALID;
  if (int rc = check_arch()) return rc;
  p.weights = weights;
  p.L = weights_len;
  p.out_table = out_table;
  p.out_stride = out_stride;
  p.table_width = table_width;
  p.keep = static_cast<int>(keep), p.recent = static_cast<int>(recent), p.sinks = static_cast<int>(sinks);
  p.kept = kept;
  p.new_lens = new_lens;
  p.new_weights = new_weights;
  p.row_bytes = p.c.D * (p.c.codes ? 1 : 2);
  const auto st = static_cast<cudaStream_t>(stream);
  // a row of tokens over as many CTAs as the GPU has room for, but not less than 2048 tokens to each
  const int64_t rows = B * p.c.heads;
  int ctas = 1;
  while (ctas < kMaxCluster && rows * ctas * 2 <= 2 * sm_count() && weights_len >= 2048 * ctas * 2) ctas *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(p.c.heads * ctas), static_cast<unsigned>(B));
  cfg.blockDim = dim3(kSelectThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = static_cast<unsigned>(ctas), attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  const int64_t part = (weights_len + ctas - 1) / ctas;
  const int held = part <= kHeldKeys ? static_cast<int>((part + 3) & ~int64_t{3}) : 0;      // a longer part is not held at all
  cfg.dynamicSmemBytes = held * sizeof(uint32_t);
  if (held > 0 && cudaFuncSetAttribute(evict_select_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, kHeldKeys * sizeof(uint32_t)) != cudaSuccess)
    return B200Q_ERR_CUDA;
  if (cudaLaunchKernelEx(&cfg, held > 0 ? evict_select_kernel<true> : evict_select_kernel<false>, p) != cudaSuccess) return B200Q_ERR_CUDA;
  if (int rc = check_launch()) return rc;
  if (keep == 0 || table_width == 0) return B200Q_OK;
  const int64_t per = kMoveThreads / (p.row_bytes / 16) * kMoveRows, blocks = (keep + per - 1) / per;
  if (blocks > 0x7fffffffLL) return B200Q_ERR_INVALID;
  if (launch_pdl(evict_move_kernel, dim3(static_cast<unsigned>(blocks), static_cast<unsigned>(p.c.heads), static_cast<unsigned>(B)), dim3(kMoveThreads), 0, st, p) != cudaSuccess)
    return B200Q_ERR_CUDA;
  return check_launch();
}

}  // extern "C"
