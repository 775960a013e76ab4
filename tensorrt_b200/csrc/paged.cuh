// The paged key-value cache as the kernels see it: addresses of rows, element types, checks of the host entry points.
#pragma once

#include "common.cuh"

namespace b200q {
namespace paged {

constexpr int kMaxD = 128;

// One of K and V.
struct Pool {
  char* base;
  int64_t page, head, row;   // bytes
};

struct Cache {
  Pool k, v;
  const float* k_amax;       // pages of codes only
  const float* v_amax;
  bool codes;
  int amax_stride;           // 0: one value for all heads
  int page_size;
  int num_pages;
  int heads, D;
  const int32_t* table;
  int64_t table_stride;
  int64_t capacity;          // rows that a line of the table can name
  const int32_t* lens;
};

// Tokens of sequence b, cut to what its line of the table and `limit` can hold.
__device__ __forceinline__ int cached_tokens(const Cache& c, int b, int64_t limit) {
  int n;
  asm volatile("ld.global.b32 %0, [%1];" : "=r"(n) : "l"(c.lens + b) : "memory");   // stays behind a pdl_wait()
  const int64_t most = c.capacity < limit ? c.capacity : limit;
  return n < 0 ? 0 : (n < most ? n : static_cast<int>(most));
}

// Page of token t of sequence b, or -1 where the table names none.
__device__ __forceinline__ int page_of(const int32_t* line, int t, const Cache& c) {
  int p;
  asm volatile("ld.global.b32 %0, [%1];" : "=r"(p) : "l"(line + t / c.page_size) : "memory");
  return static_cast<unsigned>(p) < static_cast<unsigned>(c.num_pages) ? p : -1;
}

__device__ __forceinline__ char* row_at(const Pool& p, int page, int head, int row) {
  return p.base + page * p.page + head * p.head + row * p.row;
}

__device__ __forceinline__ float head_scale(const float* amax, int stride, int head) {
  return fp8_scale_from_amax(ld_dependent(amax + static_cast<int64_t>(head) * stride));
}

// ---------------------------------------------------------------- host side
inline bool strides_ok(const int64_t* s, int n, int64_t unit) {
  for (int i = 0; i < n; ++i)
    if (s[i] < 0 || s[i] % unit != 0 || s[i] > (1LL << 46)) return false;
  return true;
}

// Fills `c` from a cache, its table and lengths.  `dtype`: the type of the tokens that meet it, or -1 where rows only move.
inline int make_cache(Cache* c, const b200q_paged_cache* in, int dtype, const int32_t* table, int64_t table_stride, int64_t table_width,
                      const int32_t* lens, int64_t B) {
  if (in == nullptr || B < 0 || B > 0x7fffffLL || table_width < 0 || table_width > 0x7fffffffLL || table_stride < 0) return B200Q_ERR_INVALID;
  if (in->page_size <= 0 || in->page_size > (1 << 20) || in->num_pages < 0 || in->num_pages > 0x7fffffffLL || in->heads <= 0 ||
      in->heads > 65535 || in->D <= 0 || in->D > kMaxD || in->D % 16 != 0)
    return B200Q_ERR_INVALID;
  const bool codes = in->dtype == B200Q_E4M3;
  if (!codes && in->dtype != B200Q_F16 && in->dtype != B200Q_BF16) return B200Q_ERR_INVALID;
  const bool moves = dtype == -1;
  if (!moves && dtype != B200Q_F16 && dtype != B200Q_BF16) return B200Q_ERR_INVALID;
  if (!moves && !codes && in->dtype != dtype) return B200Q_ERR_INVALID;
  if (!moves && codes && (in->k_amax == nullptr || in->v_amax == nullptr || (in->amax_numel != 1 && in->amax_numel != in->heads))) return B200Q_ERR_INVALID;
  if (in->num_pages > 0 && (in->k_pages == nullptr || in->v_pages == nullptr)) return B200Q_ERR_INVALID;
  if (B > 0 && (lens == nullptr || (table_width > 0 && table == nullptr))) return B200Q_ERR_INVALID;
  const int64_t size = codes ? 1 : 2, unit = 16 / size;
  if (!aligned(in->k_pages, 16) || !aligned(in->v_pages, 16) || !strides_ok(in->k_strides, 3, unit) || !strides_ok(in->v_strides, 3, unit))
    return B200Q_ERR_ALIGN;
  c->k = Pool{static_cast<char*>(in->k_pages), in->k_strides[0] * size, in->k_strides[1] * size, in->k_strides[2] * size};
  c->v = Pool{static_cast<char*>(in->v_pages), in->v_strides[0] * size, in->v_strides[1] * size, in->v_strides[2] * size};
  c->k_amax = in->k_amax;
  c->v_amax = in->v_amax;
  c->codes = codes;
  c->amax_stride = in->amax_numel == 1 ? 0 : 1;
  c->page_size = in->page_size;
  c->num_pages = static_cast<int>(in->num_pages);
  c->heads = static_cast<int>(in->heads);
  c->D = static_cast<int>(in->D);
  c->table = table;
  c->table_stride = table_stride;
  const int64_t rows = table_width * in->page_size;
  c->capacity = rows < 0x7fffff00LL ? rows : 0x7fffff00LL;
  c->lens = lens;
  return B200Q_OK;
}

}  // namespace paged
}  // namespace b200q
