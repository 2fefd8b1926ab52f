// dcr_paged.cuh — addressing of a paged key-value cache, shared by the paged operators.
//
// A pool holds num_pages pages of page_size slots; page p keeps, for every KV head, its
// slots' rows of D elements: element d of slot s of head h is at
//   base + p * sp + h * sh + s * sr + d        (strides in elements; rows contiguous)
// so pages laid out [page][head][slot][D] and [page][slot][head][D] are both strides. A
// sequence's slot i lives in page table[b][i / page_size] at i % page_size. A negative table
// entry marks a page that is not mapped; one >= num_pages is an error that raises the device
// status. Neither is ever dereferenced.
#pragma once

#include "dcr_common.cuh"
#include "dcr_internal.h"
#include "dcr_tables.h"

namespace dcr {

// n / d for 0 <= n < 2^31 by one multiplication: with s = ceil(log2 d) and
// m = ceil(2^(31+s) / d), the error m*d - 2^(31+s) is below d <= 2^s, so n times it stays
// below 2^(31+s) and the floor is exact.
struct FastDiv {
  uint32_t mul;
  uint32_t shift;
  uint32_t d;
  static FastDiv make(uint32_t d) {
    FastDiv f;
    uint32_t s = 0;
    while ((1ull << s) < d) ++s;
    f.shift = 31 + s;
    f.mul = static_cast<uint32_t>(((1ull << f.shift) + d - 1) / d);
    f.d = d;
    return f;
  }
  __device__ __forceinline__ uint32_t div(uint32_t n) const {
    return static_cast<uint32_t>((static_cast<uint64_t>(n) * mul) >> shift);
  }
};

struct PagePool {
  const void* k;
  const void* v;
  int64_t ksp, ksh, ksr;  // element strides of page, head and slot
  int64_t vsp, vsh, vsr;
  const int32_t* table;   // [sequences][max_pages], row stride tstride
  int64_t tstride;
  int num_pages;
  int max_pages;
  FastDiv page;           // page.d slots a page
};

// A table's entry as a page, or -1 (unmapped, or out of range: raises the status).
__device__ __forceinline__ int checked_page(const PagePool& c, int pg) {
  if (pg >= c.num_pages) {
    raise_status(DCR_ERR_DEVICE_INDEX);
    return -1;
  }
  return pg < 0 ? -1 : pg;
}

// Page page_index (below max_pages) of sequence b, or -1 as above.
__device__ __forceinline__ int page_of(const PagePool& c, int b, uint32_t page_index) {
  return checked_page(c, c.table[b * c.tstride + page_index]);
}

// A sequence's length, held to [0, max_pages * page_size] (beyond it: raises the status).
__device__ __forceinline__ int checked_length(const PagePool& c, int n) {
  const int cap = c.max_pages * static_cast<int>(c.page.d);
  if (n > cap) {
    raise_status(DCR_ERR_DEVICE_INDEX);
    return cap;
  }
  return n < 0 ? 0 : n;
}

// Host-side checks of a pool's description (a dcr_status).
inline int check_pool(const void* k, const void* v, int dtype, int64_t ksp, int64_t ksh,
                      int64_t ksr, int64_t vsp, int64_t vsh, int64_t vsr, int num_pages,
                      int page_size, const void* table, int64_t table_stride, int max_pages,
                      int H_kv, int D) {
  if (k == nullptr || v == nullptr || table == nullptr) return DCR_ERR_NULL;
  int64_t per16;
  switch (dtype) {
    case DCR_DTYPE_BF16:
    case DCR_DTYPE_F16: per16 = 8; break;
    case DCR_DTYPE_F32: per16 = 4; break;
    default: return DCR_ERR_DTYPE;
  }
  if (D != 64 && D != 128) return DCR_ERR_SHAPE;
  if (H_kv <= 0 || num_pages <= 0 || page_size <= 0 || max_pages <= 0) return DCR_ERR_SHAPE;
  if (static_cast<int64_t>(max_pages) * page_size > (1ll << 29)) return DCR_ERR_SHAPE;
  if (table_stride < max_pages) return DCR_ERR_SHAPE;
  const int64_t st[6] = {ksp, ksh, ksr, vsp, vsh, vsr};
  for (int i = 0; i < 6; ++i) {
    if (st[i] < 0) return DCR_ERR_SHAPE;
    if (st[i] % per16 != 0) return DCR_ERR_ALIGN;
  }
  // two slots of a head, or two heads of a slot, must not share elements
  if (page_size > 1 && (ksr < D || vsr < D)) return DCR_ERR_SHAPE;
  if (H_kv > 1 && (ksh < D || vsh < D)) return DCR_ERR_SHAPE;
  if (num_pages > 1 && (ksp < D || vsp < D)) return DCR_ERR_SHAPE;
  if (misaligned(16, k, v) || misaligned(4, table)) return DCR_ERR_ALIGN;
  return DCR_OK;
}

inline PagePool make_pool(const void* k, const void* v, int64_t ksp, int64_t ksh, int64_t ksr,
                          int64_t vsp, int64_t vsh, int64_t vsr, int num_pages, int page_size,
                          const int32_t* table, int64_t table_stride, int max_pages) {
  PagePool c;
  c.k = k;
  c.v = v;
  c.ksp = ksp;
  c.ksh = ksh;
  c.ksr = ksr;
  c.vsp = vsp;
  c.vsh = vsh;
  c.vsr = vsr;
  c.table = table;
  c.tstride = table_stride;
  c.num_pages = num_pages;
  c.max_pages = max_pages;
  c.page = FastDiv::make(static_cast<uint32_t>(page_size));
  return c;
}

}  // namespace dcr
