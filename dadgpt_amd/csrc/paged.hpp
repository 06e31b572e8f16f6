// What the kernels over paged caches share: where a sequence's new rows lie, and which page a token is
// in.
#pragma once

#include "common.hpp"
#include "serving.hpp"

namespace dadgpt {
namespace paged {

// An element of an array that no kernel of a step writes, at an index that is the same in every lane, as a
// scalar load: what follows from it (pages, addresses, whether there is anything to do) stays in scalar
// registers and branches. Through the kernel's arguments alone the compiler takes it for a vector load,
// which also waits behind the tiles in flight.
__device__ __forceinline__ int ld_uniform(const int* p) {
  typedef __attribute__((address_space(4))) const int constant_int;
  return *reinterpret_cast<constant_int*>(reinterpret_cast<uintptr_t>(p));
}

// The new rows of sequence s (UNIFORM: the same in every lane): rows first .. first + count - 1 of the step
// (clamped, so that no value of the device arrays leads out of a buffer), the token number of the first,
// and the tokens after the last. Token numbers are below 0 where the count exceeds the length.
struct NewRows {
  int first, count, token, len;
  template <bool UNIFORM>
  __device__ __forceinline__ static NewRows of(const PagedStep& p, int s) {
    if constexpr (UNIFORM)
      return NewRows(p, ld_uniform(p.row_start + s), ld_uniform(p.row_start + s + 1),
                     ld_uniform(p.lens + s));
    else
      return NewRows(p, p.row_start[s], p.row_start[s + 1], p.lens[s]);
  }
  __device__ __forceinline__ NewRows(const PagedStep& p, int a, int b, int n) {
    const int most = p.max_pages * p.page;
    len = n < 0 ? 0 : (n > most ? most : n);
    first = a < 0 ? 0 : (a > p.rows ? p.rows : a);
    const int end = b < first ? first : (b > p.rows ? p.rows : b);
    token = len - (end - first);
    count = min(end - first, p.max_rows);
    len = min(len, token + count);  // tokens of rows that are left out are not there
  }
};

// First element of head `head` of slot `slot` of page `id`.
__device__ __forceinline__ size_t page_row(const PagedStep& p, int id, int head, int slot) {
  return (((size_t)id * p.Hkv + head) * p.page + slot) * p.D;
}
__device__ __forceinline__ bool is_page(const PagedStep& p, int id) {
  return (unsigned)id < (unsigned)p.n_pages;
}

}  // namespace paged
}  // namespace dadgpt
