// dcr_tables.h — whether per-slot tables share memory (host only; no CUDA, no torch).
//
// A table's row (b, h) is `slots` neighbouring 4-byte elements at b * sb + h * sh.
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

}  // namespace dcr
