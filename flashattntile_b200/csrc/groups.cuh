// Groups of consecutive sequences that share their first tokens (whole pages).
#pragma once

#include <stdint.h>

namespace fat {

struct Groups {
  const int* cu;          // [count + 1] first sequence of each group, non-decreasing from 0
  const int* prefix;      // [count] shared tokens (cut to whole pages here)
  int count;
  int batch, page_size, cap_tokens;
  int max_size;           // what the launch has room for: a larger group shares nothing

  // Sequences of group g, cut to the batch.
  __device__ __forceinline__ int first(int g) const { return min(max(__ldg(cu + g), 0), batch); }
  __device__ __forceinline__ int size(int g) const { return max(first(g + 1) - first(g), 0); }

  // Shared tokens of group g: whole pages inside the page table.
  __device__ __forceinline__ int tokens(int g) const {
    const int t = min(max(__ldg(prefix + g), 0), cap_tokens);
    return size(g) <= max_size ? t - t % page_size : 0;
  }

  // What the edges promise: they rise, to at most the batch, by at most max_size.
  __device__ __forceinline__ bool sound(int g) const {
    const int a = __ldg(cu + g), b = __ldg(cu + g + 1);
    return a >= 0 && b >= a && b <= batch && b - a <= max_size;
  }

  // The last group that starts at or before b (empty groups start where the next one does).
  __device__ __forceinline__ int near(int b) const {
    int lo = 0, hi = count - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (__ldg(cu + mid) <= b) lo = mid;
      else hi = mid - 1;
    }
    return lo;
  }

  // Whether group g, whatever the edges hold, has b inside and no more sequences than the
  // launch has room for, so that b's rows have a place in it.
  __device__ __forceinline__ bool has(int g, int b) const {
    const int a = first(g), e = first(g + 1);
    return b >= a && b < e && e - a <= max_size;
  }

  // Shared tokens of sequence b (0 without a group).  Its loads are independent after the search.
  __device__ __forceinline__ int tokens_of(int b) const {
    if (count <= 0) return 0;
    const int g = near(b), t = tokens(g);
    return has(g, b) ? t : 0;
  }
};

}  // namespace fat
