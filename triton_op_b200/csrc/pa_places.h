// Whether the entries of tensors that a call writes have places of their own.
#pragma once

#include <stdint.h>

namespace pa_places {

// Entries (i, j), i < n0 and j < n1, of one tensor at i * s0 + j * s1: false where two of them share a place by a
// stride of zero.
inline bool distinct(int64_t n0, int64_t n1, int64_t s0, int64_t s1) { return !((n0 > 1 && s0 == 0) || (n1 > 1 && s1 == 0)); }

// Whether an entry of one such tensor is an entry of another with the same strides, `apart` elements further on.
inline bool meet(int64_t apart, int64_t n0, int64_t n1, int64_t s0, int64_t s1) {
  const int64_t a0 = s0 < 0 ? -s0 : s0, a1 = s1 < 0 ? -s1 : s1;
  const int64_t reach = (n0 - 1) * a0 + (n1 - 1) * a1;
  if (apart > reach || -apart > reach) return false;
  for (int64_t j = 1 - n1; j < n1; ++j) {
    const int64_t rest = apart - j * s1;
    if (a0 == 0 ? rest == 0 : (rest % a0 == 0 && rest / a0 < n0 && -rest / a0 < n0)) return true;
  }
  return false;
}

}  // namespace pa_places
