// What the kernels over paged caches share: where a sequence's new rows lie, and which page a token is
// in.
#pragma once

#include "common.hpp"
#include "serving.hpp"

namespace dadgpt {
namespace paged {

// The new rows of sequence s: rows first .. first + count - 1 of the step (clamped, so that no value
// of the device arrays leads out of a buffer), the token number of the first, and the tokens after the
// last. Token numbers are below 0 where the count exceeds the length.
struct NewRows {
  int first, count, token, len;
  __device__ __forceinline__ NewRows(const PagedStep& p, int s) {
    const int a = p.row_start[s], b = p.row_start[s + 1], n = p.lens[s];
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
