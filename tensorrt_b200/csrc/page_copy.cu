// Pages of the key-value cache copied to other pages, in the pools of all layers at once.
//
// Nothing is computed: every byte is read once and written once, so the memory binds a large call and the launch a small one.  Page numbers
// are the host's (it hands pages out), so they travel in the kernel's parameters: no transfer in front of the launch, and a captured call keeps
// them.  A CTA copies up to 8 KB of one page of one pool, every thread four pieces of 16 bytes, all read before the first is written.
//
// Measured: 400 pages of 8 x 64 rows of 128 codes in 8 pools 64.8 us, 0.99 of the copy rate; the first 5 to 15 rows of 48 pages in 64 pools 14.6 us (10.9 at that
// rate: one wave of small CTAs and a launch); one page in 4 pools 4.8 us, the launch.
#include <vector>

#include "paged.cuh"

namespace b200q {
namespace {

constexpr int kThreads = 128, kPieces = 4;

struct Geometry {
  int64_t page, outer_stride, inner_stride;    // bytes
  int outer, inner, pieces;                    // heads and rows of a page (or rows and heads: `inner` lie closer together), pieces of 16 bytes of a row
  bool rows_inner;
};

template <int POOLS, int PAIRS>
struct CopyParams {
  Geometry g;
  char* pools[POOLS];
  int32_t src[PAIRS], dst[PAIRS], rows[PAIRS];
};

template <int POOLS, int PAIRS>
__global__ void __launch_bounds__(kThreads) page_copy_kernel(const __grid_constant__ CopyParams<POOLS, PAIRS> p) {
  pdl_launch_dependents();
  const int pair = blockIdx.y, rows = p.rows[pair];
  const unsigned inner = p.g.rows_inner ? rows : p.g.inner, outer = p.g.rows_inner ? p.g.outer : rows;
  const unsigned line = inner * p.g.pieces, all = line * outer, first = blockIdx.x * (kThreads * kPieces) + threadIdx.x;
  char* const pool = p.pools[blockIdx.z];
  const char* const src = pool + p.src[pair] * p.g.page;
  char* const dst = pool + p.dst[pair] * p.g.page;
  const bool packed = p.g.inner_stride == 16 * p.g.pieces;
  pdl_wait();
  uint4 v[kPieces];
  int64_t at[kPieces];
#pragma unroll
  for (int k = 0; k < kPieces; ++k) {
    const unsigned i = first + k * kThreads;
    if (i >= all) break;
    const unsigned z = i / line, rest = i - z * line;
    if (packed) {
      at[k] = z * p.g.outer_stride + rest * 16;
    } else {
      const unsigned y = rest / p.g.pieces;
      at[k] = z * p.g.outer_stride + y * p.g.inner_stride + (rest - y * p.g.pieces) * 16;
    }
    v[k] = ld_128(src + at[k]);
  }
#pragma unroll
  for (int k = 0; k < kPieces; ++k) {
    if (first + k * kThreads >= all) break;
    *reinterpret_cast<uint4*>(dst + at[k]) = v[k];
  }
}

template <int POOLS, int PAIRS>
int launch_copy(const Geometry& g, void* const* pools, int64_t n_pools, const int32_t* src, const int32_t* dst, const int32_t* rows, int64_t pairs,
                int page_size, cudaStream_t st) {
  CopyParams<POOLS, PAIRS> p;
  p.g = g;
  for (int64_t at = 0; at < n_pools; at += POOLS) {
    const int here = static_cast<int>(n_pools - at < POOLS ? n_pools - at : POOLS);
    for (int i = 0; i < here; ++i) p.pools[i] = static_cast<char*>(pools[at + i]);
    for (int64_t from = 0; from < pairs; from += PAIRS) {
      const int n = static_cast<int>(pairs - from < PAIRS ? pairs - from : PAIRS);
      int most = 0;
      for (int i = 0; i < n; ++i) {
        p.src[i] = src[from + i], p.dst[i] = dst[from + i], p.rows[i] = rows == nullptr ? page_size : rows[from + i];
        most = p.rows[i] > most ? p.rows[i] : most;
      }
      const int64_t all = static_cast<int64_t>(most) * (g.rows_inner ? g.outer : g.inner) * g.pieces;
      const int64_t slices = (all + kThreads * kPieces - 1) / (kThreads * kPieces);
      if (slices == 0) continue;
      const dim3 grid(static_cast<unsigned>(slices), static_cast<unsigned>(n), static_cast<unsigned>(here));
      if (launch_pdl(page_copy_kernel<POOLS, PAIRS>, grid, dim3(kThreads), 0, st, p) != cudaSuccess) return B200Q_ERR_CUDA;
      if (int rc = check_launch()) return rc;
    }
  }
  return B200Q_OK;
}

// Every page within the pool, no page written twice, none written that is read: the order of the copies does not matter then.
bool pairs_ok(const int32_t* src, const int32_t* dst, const int32_t* rows, int64_t pairs, int64_t num_pages, int page_size) {
  for (int64_t i = 0; i < pairs; ++i) {
    if (src[i] < 0 || src[i] >= num_pages || dst[i] < 0 || dst[i] >= num_pages) return false;
    if (rows != nullptr && (rows[i] < 0 || rows[i] > page_size)) return false;
  }
  if (pairs <= 16) {
    for (int64_t i = 0; i < pairs; ++i)
      for (int64_t k = 0; k < pairs; ++k)
        if (src[k] == dst[i] || (k != i && dst[k] == dst[i])) return false;
    return true;
  }
  std::vector<bool> written(static_cast<size_t>(num_pages));
  for (int64_t i = 0; i < pairs; ++i) {
    if (written[dst[i]]) return false;
    written[dst[i]] = true;
  }
  for (int64_t i = 0; i < pairs; ++i)
    if (written[src[i]]) return false;
  return true;
}

}  // namespace
}  // namespace b200q

using namespace b200q;

extern "C" {

int b200q_paged_copy(void* const* pools, int64_t n_pools, int64_t num_pages, int64_t heads, int32_t page_size, int64_t row_bytes,
                     const int64_t* strides, const int32_t* src, const int32_t* dst, const int32_t* rows, int64_t pairs, b200q_stream_t stream) {
  if (n_pools < 0 || pairs < 0 || num_pages < 0 || num_pages > 0x7fffffffLL || heads <= 0 || heads > 65535 || page_size <= 0 || page_size > (1 << 20) ||
      row_bytes <= 0 || row_bytes > 256 || strides == nullptr || pairs > num_pages)
    return B200Q_ERR_INVALID;
  if (row_bytes % 16 != 0) return B200Q_ERR_ALIGN;
  if (heads * page_size * (row_bytes / 16) > 0x3fffffffLL) return B200Q_ERR_INVALID;
  if (n_pools > 0 && pools == nullptr) return B200Q_ERR_INVALID;
  if (pairs > 0 && (src == nullptr || dst == nullptr)) return B200Q_ERR_INVALID;
  if (!paged::strides_ok(strides, 3, 16)) return B200Q_ERR_ALIGN;
  for (int64_t i = 0; i < n_pools; ++i) {
    if (pools[i] == nullptr && pairs > 0) return B200Q_ERR_INVALID;
    if (!aligned(pools[i], 16)) return B200Q_ERR_ALIGN;
  }
  try {
    if (!pairs_ok(src, dst, rows, pairs, num_pages, page_size)) return B200Q_ERR_INVALID;
  } catch (...) {            // no memory for the marks
    return B200Q_ERR_TOO_LARGE;
  }
  if (n_pools == 0 || pairs == 0) return B200Q_OK;
  if (int rc = check_arch()) return rc;
  Geometry g{};
  g.page = strides[0];
  g.pieces = static_cast<int>(row_bytes / 16);
  g.rows_inner = strides[2] <= strides[1] || heads == 1;
  g.outer = g.rows_inner ? static_cast<int>(heads) : page_size, g.inner = g.rows_inner ? page_size : static_cast<int>(heads);
  g.outer_stride = g.rows_inner ? strides[1] : strides[2], g.inner_stride = g.rows_inner ? strides[2] : strides[1];
  const auto st = static_cast<cudaStream_t>(stream);
  if (pairs <= 64 && n_pools <= 64) return launch_copy<64, 64>(g, pools, n_pools, src, dst, rows, pairs, page_size, st);
  return launch_copy<256, 1024>(g, pools, n_pools, src, dst, rows, pairs, page_size, st);
}

}  // extern "C"
