// dcr_tables.h — whether tables of strided rows share memory (host only; no CUDA, no torch).
//
// A table's row (b, h) is `slots` neighbouring elements at b * sb + h * sh: a slot's entries of 4
// bytes, or the logits of a row.
#pragma once

#include <stdint.h>

namespace dcr {

// Whether no two of the n_b * n_h rows share an element: one dimension's stride has to span all
// rows of the other, as in any slice or permutation of a dense tensor. What is written has to be
// so, or several CTAs would write one element.
inline bool rows_apart(int64_t n_b, int64_t n_h, int64_t slots, int64_t sb, int64_t sh) {
  if (n_b <= 1) return n_h <= 1 || sh >= slots;
  if (n_h <= 1) return sb >= slots;
  return (sh >= slots && sb >= slots && (sb - slots) / (n_h - 1) >= sh) ||
         (sb >= slots && sh >= slots && (sh - slots) / (n_b - 1) >= sb);
}

// A table as bytes.
struct TableSpan {
  const char* data;
  int64_t n_b, n_h, bytes, sb, sh;  // rows, a row's bytes, strides in bytes

  TableSpan(const void* table, int64_t nb, int64_t nh, int64_t slots, int64_t stride_b,
            int64_t stride_h, int64_t element = 4)
      : data(static_cast<const char*>(table)), n_b(nb), n_h(nh), bytes(element * slots),
        sb(nb > 1 ? element * stride_b : 0), sh(nh > 1 ? element * stride_h : 0) {}
  int64_t size() const { return (n_b - 1) * sb + (n_h - 1) * sh + bytes; }
};

// Whether a row of `a` shares a byte with a row of `b`, whose own rows are apart. Tables that lie
// one after the other, the usual case, need two comparisons; rows that lie between one another's
// are compared by division, a few of `b` for each of `a`.
inline bool tables_meet(const TableSpan& a, const TableSpan& b) {
  const int64_t off = static_cast<int64_t>(reinterpret_cast<uintptr_t>(a.data) -
                                           reinterpret_cast<uintptr_t>(b.data));
  if (off >= b.size() || -off >= a.size()) return false;
  const bool b_outer = b.n_h <= 1 || (b.n_b > 1 && b.sb >= b.sh);
  const int64_t n_out = b_outer ? b.n_b : b.n_h, n_in = b_outer ? b.n_h : b.n_b;
  const int64_t s_out = b_outer ? b.sb : b.sh, s_in = b_outer ? b.sh : b.sb;
  const int64_t block = (n_in - 1) * s_in + b.bytes;  // an outer index's rows
  // the indexes whose [i * stride, i * stride + size) may meet [x, x + a.bytes)
  auto first = [](int64_t x, int64_t size, int64_t stride) {
    return x < size || stride == 0 ? 0 : (x - size) / stride + 1;
  };
  auto last = [&](int64_t x, int64_t stride, int64_t n) {
    const int64_t end = x + a.bytes - 1;
    if (end < 0) return static_cast<int64_t>(-1);
    return stride == 0 || end / stride >= n ? n - 1 : end / stride;
  };
  for (int64_t i = 0; i < a.n_b; ++i)
    for (int64_t j = 0; j < a.n_h; ++j) {
      const int64_t x = off + i * a.sb + j * a.sh;
      for (int64_t o = first(x, block, s_out); o <= last(x, s_out, n_out); ++o) {
        const int64_t y = x - o * s_out;
        if (first(y, b.bytes, s_in) <= last(y, s_in, n_in)) return true;
      }
    }
  return false;
}

// Whether contiguous output rows [n, heads, D] reach into the strided rows that they are computed
// from. In place, row for row, is fine: a row is written after all reads of it.
inline bool rows_meet(const void* from, int64_t stride_n, int64_t stride_h, const void* to, int64_t n,
                      int64_t heads, int64_t D, int64_t element) {
  if (from == to && (n <= 1 || stride_n == heads * D) && (heads <= 1 || stride_h == D)) return false;
  return tables_meet(TableSpan(from, n, heads, D, stride_n, stride_h, element),
                     TableSpan(to, n, heads, D, heads * D, D, element));
}

// Whether rows [B, V] processed into rows of other strides or another address would be read after
// they are written. In place, row for row, is fine.
inline bool logits_meet(const void* from, int64_t from_stride, const void* to, int64_t to_stride,
                        int64_t B, int64_t V, int64_t element) {
  if (from == to && (B <= 1 || from_stride == to_stride)) return false;
  return tables_meet(TableSpan(from, B, 1, V, from_stride, 0, element),
                     TableSpan(to, B, 1, V, to_stride, 0, element));
}

}  // namespace dcr
