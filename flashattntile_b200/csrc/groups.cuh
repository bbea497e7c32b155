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

  // The group of sequence b, or -1.  The search takes the last group that starts at or
  // before b (empty groups start where the next one does); whatever the edges hold, the
  // group that it returns has b inside, so that a row's place in its group is one that
  // the launch has room for.
  __device__ __forceinline__ int of(int b) const {
    if (count <= 0 || b >= __ldg(cu + count)) return -1;
    int lo = 0, hi = count - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (__ldg(cu + mid) <= b) lo = mid;
      else hi = mid - 1;
    }
    const int a = first(lo), e = first(lo + 1);
    return b >= a && b < e && e - a <= max_size ? lo : -1;
  }

  // Shared tokens of sequence b (0 without a group).
  __device__ __forceinline__ int tokens_of(int b) const {
    const int g = of(b);
    return g < 0 ? 0 : tokens(g);
  }
};

}  // namespace fat
