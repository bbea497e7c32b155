// Pages shared between sequences: copying, forking, reserving (copy on write),
// releasing and compacting the pages of a paged KV cache, on the device.
//
// State beside the cache: refs[page], how many table entries hold the page
// (0: free), and owned[row], how many leading entries of a row hold pages (later
// entries are never read, and become 0, a valid page id, where a row gives pages back).
// Optionally released[row], 1 from a row's release until it is forked to or reserved by name: a reserve of all rows
// may leave such rows out, so that a captured step can run while rows are idle.
// Every operation is defined by whole numbers alone (the lowest free page id
// first, rows in the order given), so its result does not depend on the order
// in which threads run: integer counts commute, and every choice is made from
// prefix sums.
//
//   fork     row dst <- row src: table entries of the pages src's length
//            reaches, their counts + 1; what dst held is released.  No K/V moves.
//   reserve  a row may append `tokens` tokens: a shared, partly filled tail page
//            is copied to a free page (the last sharer in the call keeps it when
//            every holder is in the call), pages that are missing are taken.
//   release  counts - 1, entries 0, length 0.
//   compact  with L live pages, the k-th live page with id >= L moves to the
//            k-th free id below L; tables and counts follow.
#include <algorithm>

#include "common.cuh"
#include "host_util.h"
#include "pages.h"

namespace fat {
namespace pg {

constexpr int kSeg = 1024;      // page counts per segment (one block scans one segment)
constexpr int kMaxSegs = 8192;  // segments the allocating block scans in shared memory
constexpr int kCopyThreads = 256;
constexpr int kBlock = 1024;

// The operations are short kernels in a row: each is launched beside the one before it
// and waits here for its end, so that a launch costs a wait instead of a start.  Every
// block calls it first; what an earlier kernel may have written is not read through the
// read-only path, which assumes that it stays as it is while a kernel runs.
__device__ __forceinline__ void chained() {
  grid_allow_dependents();
  grid_dependency_wait();
}

// ---------------------------------------------------------------------------
// Copying
// ---------------------------------------------------------------------------
// A page of one tensor as runs of contiguous bytes: n1 runs stride1 apart, each
// of n2 runs stride2 apart, `vecs` vectors of the launch's width each.
struct Runs {
  int n1, n2, vecs;
  long long stride1, stride2;
};

struct CopyParams {
  uint8_t* k;
  uint8_t* v;
  long long sp;
  Runs runs;
  long long num_pages;
  const int* src;
  const int* dst;
  int n;             // pairs
  const int* n_dev;  // or their number on the device
  int pair_stride;   // ints between pairs (2: src and dst interleaved)
  int skip_negative; // a pair (-1, -1) stands for no copy
  float* k_scale;
  float* v_scale;
  long long scale_sp;
  int heads;
  int chunk_vecs;    // vectors a block copies at a time (a multiple of its threads)
  int chunks;        // chunks per (pair, tensor)
  int* err;
};

template <typename V>
__device__ __forceinline__ V ld_stream(const V* p) {
  return __ldcs(p);
}

// kUnroll vectors per thread are loaded before the first is stored: bytes in
// flight are what a copy's rate depends on.
template <typename V, int kUnroll>
__device__ __forceinline__ void copy_body(const CopyParams& p) {
  const int n = p.n_dev != nullptr ? min(__ldcg(p.n_dev), p.n) : p.n;
  const int page_vecs = p.runs.n1 * p.runs.n2 * p.runs.vecs;
  const long long jobs = (long long)n * 2 * p.chunks;
  for (long long job = blockIdx.x; job < jobs; job += gridDim.x) {
    const int chunk = int(job % p.chunks);
    const long long pt = job / p.chunks;
    const int pair = int(pt >> 1), which = int(pt & 1);
    const int s = __ldcg(p.src + pair * p.pair_stride), d = __ldcg(p.dst + pair * p.pair_stride);
    if (s < 0 && d < 0 && p.skip_negative) continue;
    if (s < 0 || d < 0 || s >= p.num_pages || d >= p.num_pages) {
      if (threadIdx.x == 0) raise_error(p.err, FAT_DEVERR_BAD_PAGE);
      continue;
    }
    uint8_t* base = which ? p.v : p.k;
    const uint8_t* from = base + (long long)s * p.sp;
    uint8_t* to = base + (long long)d * p.sp;
    const int i0 = chunk * p.chunk_vecs + threadIdx.x;
    const int i1 = min(page_vecs, (chunk + 1) * p.chunk_vecs);
    if (p.runs.n1 * p.runs.n2 == 1) {  // one contiguous run
      for (int i = i0; i < i1; i += kUnroll * kCopyThreads) {
        V x[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
          if (i + u * kCopyThreads < i1) x[u] = ld_stream(reinterpret_cast<const V*>(from) + i + u * kCopyThreads);
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
          if (i + u * kCopyThreads < i1) reinterpret_cast<V*>(to)[i + u * kCopyThreads] = x[u];
      }
    } else {
      for (int i = i0; i < i1; i += kCopyThreads) {
        const int run = i / p.runs.vecs, x = i - run * p.runs.vecs;
        const int r1 = run / p.runs.n2, r2 = run - r1 * p.runs.n2;
        const long long off = r1 * p.runs.stride1 + r2 * p.runs.stride2 + (long long)x * (long long)sizeof(V);
        *reinterpret_cast<V*>(to + off) = *reinterpret_cast<const V*>(from + off);
      }
    }
    if (p.k_scale != nullptr && chunk == 0) {
      float* sc = which ? p.v_scale : p.k_scale;
      for (int h = threadIdx.x; h < p.heads; h += kCopyThreads)
        sc[(long long)d * p.scale_sp + h] = sc[(long long)s * p.scale_sp + h];
    }
  }
}

template <typename V, int kUnroll>
__global__ void __launch_bounds__(kCopyThreads) copy_pages_kernel(const CopyParams p) {
  chained();
  copy_body<V, kUnroll>(p);
}

// ---------------------------------------------------------------------------
// Rows
// ---------------------------------------------------------------------------
struct RowParams {
  int* table;
  long long pt_sb;
  int max_pages;
  int* lens;
  int* owned;
  int* refs;
  int* released;  // null: not kept
  bool skip_released;
  int batch;
  long long num_pages;
  int page_size;
  int* err;
};

__device__ __forceinline__ bool row_ok(const RowParams& p, int row) {
  if (row >= 0 && row < p.batch) return true;
  raise_error(p.err, FAT_DEVERR_BAD_ROW);
  return false;
}

__device__ __forceinline__ bool page_ok(const RowParams& p, int page) {
  if (page >= 0 && page < p.num_pages) return true;
  raise_error(p.err, FAT_DEVERR_BAD_PAGE);
  return false;
}

// Pages that row `row` shares when forked: those its length reaches.
__device__ __forceinline__ int used_pages(const RowParams& p, int row) {
  const int len = max(p.lens[row], 0);
  return min(min((len + p.page_size - 1) / p.page_size, p.owned[row]), p.max_pages);
}

// True in every thread of the last block of the grid to get here; the ticket is
// zero again afterwards.  The fence before it publishes the block's writes.
__device__ __forceinline__ bool last_block(int* ticket) {
  __shared__ int last;
  if (gridDim.x == 1) {
    __syncthreads();
    return true;
  }
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) {
    last = atomicAdd(ticket, 1) == int(gridDim.x) - 1;
    if (last) {
      *ticket = 0;
      __threadfence();
    }
  }
  __syncthreads();
  return last != 0;
}

// One block takes `cols` columns of every forked row: it reads all the source
// entries before it writes any row, so a row may be source and destination at
// once (beams).  Many rows fork from one, so a page's count changes by as many at once:
// a warp takes 32 rows of a column and adds once per page among them.  Lengths are
// written by the last block, after every block has read them.
__global__ void __launch_bounds__(kBlock) fork_kernel(const RowParams p, const int* src, const int* dst, int n,
                                                      int cols, int* ticket) {
  extern __shared__ int stage[];  // [n][cols] entries, [n][cols] entries before; then [n] lengths, [n] owned counts
  chained();
  int* before = stage + n * cols;
  const int c0 = blockIdx.x * cols, lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i < n * cols; i += blockDim.x) {
    const int d = i / cols, c = c0 + i - d * cols;
    const int s = __ldcg(src + d);
    int e = -1;  // past the pages to share
    if (s >= 0 && s < p.batch && c < used_pages(p, s)) e = p.table[(long long)s * p.pt_sb + c];
    stage[i] = e;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n * cols; i += blockDim.x) {
    const int d = i / cols, c = c0 + i - d * cols;
    const int s = __ldcg(src + d), row = __ldcg(dst + d);
    int old = -1, now = -1;
    if (c < p.max_pages && s >= 0 && s < p.batch && row >= 0 && row < p.batch && s != row) {
      int* at = p.table + (long long)row * p.pt_sb + c;
      now = stage[i];
      if (c < p.owned[row]) old = *at;
      if (old == now) old = now = -1;
      else *at = max(now, 0);
      if (now >= 0 && !page_ok(p, now)) now = -1;
      if (old >= 0 && !page_ok(p, old)) old = -1;
    }
    stage[i] = now;
    before[i] = old;
  }
  __syncthreads();
  const int groups = (n + 31) / 32;
  for (int j = threadIdx.x >> 5; j < groups * cols; j += kBlock / 32) {
    const int d = j / cols * 32 + lane, at = d * cols + j % cols;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int page = d < n ? (k ? before[at] : stage[at]) : -1;
      const unsigned same = __match_any_sync(0xffffffffu, page);
      if (page >= 0 && lane == __ffs(same) - 1) atomicAdd(p.refs + page, k ? -__popc(same) : __popc(same));
    }
  }
  if (!last_block(ticket)) return;
  // All lengths are read before any is written; a row owns what its length
  // reaches, or the source's own pages when it holds fewer.  Length -1 stands for a source
  // that is released: so is its copy.
  int* len = stage;
  int* own = stage + n;
  for (int d = threadIdx.x; d < n; d += blockDim.x) {
    const int s = __ldcg(src + d);
    const bool ok = row_ok(p, s);
    len[d] = ok ? (p.released != nullptr && p.released[s] != 0 ? -1 : max(p.lens[s], 0)) : 0;
    own[d] = ok ? used_pages(p, s) : 0;
  }
  __syncthreads();
  for (int d = threadIdx.x; d < n; d += blockDim.x) {
    const int s = __ldcg(src + d), row = __ldcg(dst + d);
    if (s < 0 || s >= p.batch || !row_ok(p, row) || s == row) continue;
    p.lens[row] = max(len[d], 0);
    p.owned[row] = own[d];
    if (p.released != nullptr) p.released[row] = len[d] < 0;
  }
}

// One block per row.  owned is taken with an exchange, so a row listed twice is
// released once.
__global__ void __launch_bounds__(kBlock) release_kernel(const RowParams p, const int* rows) {
  __shared__ int own_s;
  chained();
  const int row = __ldcg(rows + blockIdx.x);
  if (row < 0 || row >= p.batch) {
    if (threadIdx.x == 0) raise_error(p.err, FAT_DEVERR_BAD_ROW);
    return;
  }
  if (threadIdx.x == 0) {
    own_s = min(atomicExch(p.owned + row, 0), p.max_pages);
    p.lens[row] = 0;
    if (p.released != nullptr) p.released[row] = 1;
  }
  __syncthreads();
  int* at = p.table + (long long)row * p.pt_sb;
  constexpr int kU = 4;
  for (int c = threadIdx.x; c < own_s; c += kU * kBlock) {
    int e[kU];
#pragma unroll
    for (int u = 0; u < kU; ++u) e[u] = c + u * kBlock < own_s ? at[c + u * kBlock] : -1;
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      if (c + u * kBlock >= own_s) continue;
      if (page_ok(p, e[u])) atomicSub(p.refs + e[u], 1);
      at[c + u * kBlock] = 0;
    }
  }
}

// ---------------------------------------------------------------------------
// Block scans
// ---------------------------------------------------------------------------
// Exclusive prefix sum of one value per thread over a block of kBlock threads;
// `total` receives the sum.  Ends with a barrier, so it can be called again.
__device__ __forceinline__ int block_scan(int v, int& total) {
  __shared__ int sums[kBlock / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) sums[warp] = x;
  __syncthreads();
  if (warp == 0) {
    int w = sums[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += y;
    }
    sums[lane] = w;
  }
  __syncthreads();
  const int before = warp > 0 ? sums[warp - 1] : 0;
  total = sums[kBlock / 32 - 1];
  __syncthreads();
  return before + x - v;
}

// A page is live while a table entry holds it.
__device__ __forceinline__ bool is_live(int refs) { return refs > 0; }

// Live (or free) pages of each segment of the block, eight segments' loads at a time.
__device__ __forceinline__ void count_segments(const int* refs, long long num_pages, int segs, bool live, int* counts) {
  constexpr int kAhead = 8;
  for (int s0 = blockIdx.x; s0 < segs; s0 += kAhead * gridDim.x) {
    int r[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const long long page = (long long)(s0 + k * int(gridDim.x)) * kSeg + threadIdx.x;
      r[k] = page < num_pages ? __ldcg(refs + page) : (live ? 0 : 1);  // past the pool: not counted
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int s = s0 + k * int(gridDim.x);
      if (s >= segs) break;
      const int here = __syncthreads_count(is_live(r[k]) == live);
      if (threadIdx.x == 0) counts[s] = here;
    }
  }
}

// Exclusive prefix sums of counts[0, segs) into pre[0, segs], by one block.
__device__ void scan_segments(const int* counts, int* pre, int segs) {
  int carry = 0;
  for (int s0 = 0; s0 < segs; s0 += kBlock) {
    const int s = s0 + threadIdx.x;
    int total;
    const int x = block_scan(s < segs ? __ldcg(counts + s) : 0, total);
    if (s < segs) pre[s] = carry + x;
    carry += total;
  }
  if (threadIdx.x == 0) pre[segs] = carry;
  __syncthreads();
}

// Scratch of the pool operations: counters first (zero between calls), then
// per-page words of which `sharers` and `latest` are zero between calls.
struct Scratch {
  int* ticket;    // [4]
  int* sharers;   // [num_pages] rows of this call with the page as shared tail
  int* latest;    // [num_pages] 1 + the last of them
  int* seg;       // [segs + 1]
  int* list;      // [num_pages] free pages in order | holes
  int* movers;    // [num_pages]
  int* rank;      // [num_pages]
  int* kept;      // [num_pages] refs of the movers
  int* pairs;     // [2 * batch] copies of a reserve
  int* info;      // [4] compact: live pages, moved pages, live below the live count
};

// ---------------------------------------------------------------------------
// Reserve
// ---------------------------------------------------------------------------
// What row i of the call needs.  tail: its shared, partly filled tail page (-1:
// none), which `held` table entries hold; fresh: pages missing for `tokens` more tokens.
struct Need {
  int row = -1, at = 0, tail = -1, held = 0, own = 0, fresh = 0;
  bool ok = false, idle = false;  // idle: left out on purpose
};

__device__ __forceinline__ Need row_need(const RowParams& p, const int* rows, int i, int tokens) {
  Need x;
  const int row = rows != nullptr ? __ldcg(rows + i) : i;
  if (row < 0 || row >= p.batch) return x;
  x.row = row;
  x.idle = rows == nullptr && p.skip_released && p.released[row] != 0;
  if (x.idle) return x;
  const int len = p.lens[row];
  x.own = p.owned[row];
  const long long want = ((long long)len + tokens + p.page_size - 1) / p.page_size;
  if (len < 0 || want > p.max_pages) return x;
  x.ok = true;
  x.at = len / p.page_size;
  x.fresh = max(int(want) - x.own, 0);
  if (len % p.page_size != 0 && x.at < x.own) {
    const int e = p.table[(long long)row * p.pt_sb + x.at];
    if (e >= 0 && e < p.num_pages) {
      x.held = __ldcg(p.refs + e);
      if (x.held > 1) x.tail = e;
    } else {
      x.ok = false;
    }
  }
  return x;
}

// Blocks count the free pages of their segments (counting_blocks); the last one to
// finish hands them out.  Copies asked for go to w.pairs (-1, -1 where a row needs none).
__global__ void __launch_bounds__(kBlock) reserve_kernel(const RowParams p, const Scratch w, const int* rows, int n,
                                                         int tokens, int segs) {
  chained();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // The needs of the first kBlock rows, which is mostly all, are looked up once, beside
  // the counting (only the last block changes what they depend on).
  const Need mine = tid < n ? row_need(p, rows, tid, tokens) : Need{};
  auto need_of = [&](int i) { return i < kBlock ? mine : row_need(p, rows, i, tokens); };
  count_segments(p.refs, p.num_pages, segs, false, w.seg);
  if (!last_block(w.ticket)) return;

  __shared__ int offs[kBlock + 1];
  constexpr int kNear = 2 * kBlock;  // free pages listed in shared memory; more go to w.list
  __shared__ int near_s[kNear];
  auto listed = [&](int k) { return k < kNear ? near_s[k] : w.list[k]; };
  scan_segments(w.seg, w.seg, segs);  // in place: each count is read before its sum is written
  const int free_total = __ldcg(w.seg + segs);

  // Which rows share a tail page with others of the call.
  for (int i = tid; i < n; i += kBlock) {
    const Need x = need_of(i);
    if (x.row < 0) raise_error(p.err, FAT_DEVERR_BAD_ROW);
    else if (!x.ok && !x.idle) raise_error(p.err, FAT_DEVERR_BAD_LENGTH);
    if (x.ok && x.tail >= 0) {
      atomicAdd(w.sharers + x.tail, 1);
      atomicMax(w.latest + x.tail, i + 1);
    }
  }
  __threadfence_block();
  __syncthreads();
  // The last sharer keeps the page if every holder of it is in the call.
  auto moves = [&](const Need& x, int i) {
    return x.ok && x.tail >= 0 &&
           !(__ldcg(w.sharers + x.tail) == x.held && __ldcg(w.latest + x.tail) == i + 1);
  };

  // Pages needed in all (rows past the free pages get none).
  int total = 0;
  for (int i0 = 0; i0 < n; i0 += kBlock) {
    const int i = i0 + tid;
    int need = 0;
    if (i < n) {
      const Need x = need_of(i);
      need = x.ok ? x.fresh + (moves(x, i) ? 1 : 0) : 0;
    }
    int sum;
    block_scan(need, sum);
    total += sum;
  }
  const int wanted = min(total, free_total);
  // The first `wanted` free pages, in order: a warp lists one segment.
  for (int s = warp; s < segs; s += kBlock / 32) {
    const int r0 = __ldcg(w.seg + s);
    if (r0 >= wanted) break;
    if (__ldcg(w.seg + s + 1) == r0) continue;
    int e[kSeg / 32];
#pragma unroll
    for (int j = 0; j < kSeg / 32; ++j) {
      const long long page = (long long)s * kSeg + j * 32 + lane;
      e[j] = page < p.num_pages ? __ldcg(p.refs + page) : 1;
    }
    int r = r0;
#pragma unroll
    for (int j = 0; j < kSeg / 32; ++j) {
      const bool fr = !is_live(e[j]);
      const unsigned m = __ballot_sync(0xffffffffu, fr);
      const int k = r + __popc(m & ((1u << lane) - 1u));
      if (fr && k < wanted) (k < kNear ? near_s[k] : w.list[k]) = s * kSeg + j * 32 + lane;
      r += __popc(m);
    }
  }
  __threadfence_block();
  __syncthreads();

  int base = 0;
  for (int i0 = 0; i0 < n; i0 += kBlock) {
    const int i = i0 + tid;
    Need x;
    bool mv = false;
    if (i < n) {
      x = need_of(i);
      mv = moves(x, i);
    }
    const int need = x.ok ? x.fresh + (mv ? 1 : 0) : 0;
    int sum;
    const int off = base + block_scan(need, sum);
    const bool got = off + need <= free_total;
    if (!got && need > 0) raise_error(p.err, FAT_DEVERR_NO_PAGE);
    __syncthreads();
    // Every row of the round has read the counts above; now they change.
    int from = -1, to = -1;
    if (got && mv) {
      from = x.tail;
      to = listed(off);
      p.table[(long long)x.row * p.pt_sb + x.at] = to;
      p.refs[to] = 1;
    }
    if (i < n) {
      w.pairs[2 * i] = from;
      w.pairs[2 * i + 1] = to;
      if (got && x.ok && x.fresh > 0) p.owned[x.row] = x.own + x.fresh;
      if (got && x.ok && rows != nullptr && p.released != nullptr) p.released[x.row] = 0;
    }
    // Missing pages, one thread each: offs finds the row of a page.
    offs[tid] = off + (mv ? 1 : 0) - base;
    if (tid == 0) offs[kBlock] = sum;
    __shared__ int own_s[kBlock], row_s[kBlock], fresh_s[kBlock];
    own_s[tid] = x.own;
    row_s[tid] = x.row;
    fresh_s[tid] = got && x.ok ? x.fresh : 0;
    __syncthreads();
    for (int k = tid; k < sum; k += kBlock) {
      // The last row whose first missing page is at or before k.
      int lo = 0, hi = kBlock - 1;
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (offs[mid] <= k) lo = mid;
        else hi = mid - 1;
      }
      const int j = k - offs[lo];
      if (j >= 0 && j < fresh_s[lo]) {
        const int page = listed(base + k);
        p.table[(long long)row_s[lo] * p.pt_sb + own_s[lo] + j] = page;
        p.refs[page] = 1;
      }
    }
    base += sum;
    __syncthreads();
  }
  // The copied tails lose a holder; the marks go back to zero (a kept tail is
  // still in its row's table).
  for (int i = tid; i < n; i += kBlock) {
    int page = w.pairs[2 * i];
    if (page >= 0) {
      atomicSub(p.refs + page, 1);
    } else if (i < kBlock) {
      page = mine.ok ? mine.tail : -1;
    } else {
      const int row = rows != nullptr ? __ldcg(rows + i) : i;
      if (row < 0 || row >= p.batch) continue;
      const int at = max(p.lens[row], 0) / p.page_size;
      page = at < p.max_pages ? p.table[(long long)row * p.pt_sb + at] : -1;
    }
    if (page >= 0 && page < p.num_pages) {
      w.sharers[page] = 0;
      w.latest[page] = 0;
    }
  }
}

// ---------------------------------------------------------------------------
// Compact
// ---------------------------------------------------------------------------
// Live pages before each segment, in all, and below the live count (the last
// block to finish).
__global__ void __launch_bounds__(kBlock) live_kernel(const RowParams p, const Scratch w, int* live_out, int segs) {
  chained();
  count_segments(p.refs, p.num_pages, segs, true, w.seg);
  if (!last_block(w.ticket)) return;
  scan_segments(w.seg, w.seg, segs);
  const int live = w.seg[segs];
  const int s = live / kSeg;  // the segment that page `live` is in
  const long long page = (long long)s * kSeg + threadIdx.x;
  const int part = __syncthreads_count(page < min((long long)live, p.num_pages) && is_live(__ldcg(p.refs + page)));
  if (threadIdx.x == 0) {
    const int below = (s < segs ? w.seg[s] : live) + part;
    w.info[0] = live;
    w.info[1] = live - below;
    w.info[2] = below;
    if (live_out != nullptr) *live_out = live;
  }
}

// One block per segment lists its pages: the k-th free page below the live count
// in w.list, the k-th live page at or above it in w.movers (with its count).
__global__ void __launch_bounds__(kBlock) list_kernel(const RowParams p, const Scratch w) {
  chained();
  const int live = w.info[0], below = w.info[2];
  const long long page = (long long)blockIdx.x * kSeg + threadIdx.x;
  const int refs = page < p.num_pages ? p.refs[page] : 0;
  int total;
  const int before = w.seg[blockIdx.x] + block_scan(is_live(refs) ? 1 : 0, total);
  if (page >= p.num_pages) return;
  if (page < live) {
    if (!is_live(refs)) w.list[int(page) - before] = int(page);
  } else if (is_live(refs)) {
    const int k = before - below;
    w.movers[k] = int(page);
    w.kept[k] = refs;
    w.rank[page] = k;
  }
}

// Tables and counts follow the pages.
__device__ __forceinline__ void follow_body(const RowParams& p, const Scratch& w, int* table_out,
                                            long long pt_out_sb, int* refs_out) {
  const int live = w.info[0], moved = w.info[1];
  const long long stride = (long long)gridDim.x * blockDim.x;
  const long long first = (long long)blockIdx.x * blockDim.x + threadIdx.x;
  for (long long i = first; i < (long long)p.batch * p.max_pages; i += stride) {
    const int row = int(i / p.max_pages), c = int(i - (long long)row * p.max_pages);
    const int e = p.table[(long long)row * p.pt_sb + c];
    int to = e;
    // An entry past what its row owns may hold anything: only a page on the
    // movers' list under its own rank is renamed.
    if (e >= live && e < p.num_pages) {
      const int k = w.rank[e];
      if (k >= 0 && k < moved && w.movers[k] == e) to = w.list[k];
    }
    if (table_out != p.table || to != e) table_out[(long long)row * pt_out_sb + c] = to;
  }
  for (long long i = first; i < p.num_pages; i += stride) {
    if (i >= live) refs_out[i] = 0;
    else if (refs_out != p.refs && is_live(p.refs[i])) refs_out[i] = p.refs[i];
  }
  for (long long k = first; k < moved; k += stride) refs_out[w.list[k]] = w.kept[k];
}

// The pages move beside it.  Sources lie at or above the live count and targets below
// it, so no page is both.
template <typename V, int kUnroll>
__global__ void __launch_bounds__(kCopyThreads) move_pages_kernel(const CopyParams c, const RowParams p,
                                                                  const Scratch w, int* table_out,
                                                                  long long pt_out_sb, int* refs_out) {
  chained();
  follow_body(p, w, table_out, pt_out_sb, refs_out);
  copy_body<V, kUnroll>(c);
}

}  // namespace pg

// =============================================================================
// Host side
// =============================================================================
namespace {

size_t align_up(size_t x, size_t a) { return (x + a - 1) / a * a; }

// Blocks that count the segments of a pool: one while a single round of loads does (up to
// 8,192 pages; it needs no agreement with other blocks: a small compaction takes 8.7 us,
// 9.3 with the agreement; at 8 segments both ways measure the same).
int counting_blocks(int segs, int sms) { return segs <= 8 ? 1 : std::min(segs, sms); }

int segments(int64_t num_pages) { return int((num_pages + pg::kSeg - 1) / pg::kSeg); }

// Scratch layout; counters and the two mark arrays first (zero between calls).
pg::Scratch carve(void* base, int64_t num_pages, int batch, size_t* total) {
  uint8_t* at = static_cast<uint8_t*>(base);
  size_t off = 0;
  auto take = [&](size_t ints) {
    int* x = reinterpret_cast<int*>(at + off);
    off = align_up(off + ints * sizeof(int), 256);
    return x;
  };
  const size_t n = size_t(num_pages);
  pg::Scratch w;
  w.ticket = take(4);
  w.sharers = take(n);
  w.latest = take(n);
  w.seg = take(size_t(segments(num_pages)) + 1);
  w.list = take(n);
  w.movers = take(n);
  w.rank = take(n);
  w.kept = take(n);
  w.pairs = take(2 * size_t(batch));
  w.info = take(4);
  *total = off;
  return w;
}

int check_store(const char* what, const PageStore& s) {
  const std::string w = what;
  if (s.num_pages <= 0 || s.num_kv_heads <= 0 || s.page_size <= 0 || s.row_bytes <= 0)
    return invalid(w + ": the pool's sizes must be positive");
  if (s.num_pages > (int64_t(1) << 31) - 1) return unsupported(w + ": too many pages");
  if (s.k == nullptr || s.v == nullptr) return invalid(w + ": null pointer argument");
  if ((s.k_scale == nullptr) != (s.v_scale == nullptr)) return invalid(w + ": give both scales or neither");
  const int64_t vecs = int64_t(s.page_size) * s.num_kv_heads * s.row_bytes;
  if (vecs > (int64_t(1) << 30)) return unsupported(w + ": a page larger than 1 GiB");
  return FAT_OK;
}

int check_rows(const char* what, const PageStore& s, const PageRows& r) {
  const std::string w = what;
  if (r.batch <= 0 || r.max_pages <= 0) return invalid(w + ": empty page table");
  if (r.max_pages > (int64_t(1) << 30)) return unsupported(w + ": page table too wide");
  if (r.table == nullptr || r.seq_lens == nullptr || r.owned == nullptr || r.refs == nullptr)
    return invalid(w + ": null pointer argument");
  if (segments(s.num_pages) > pg::kMaxSegs)
    return unsupported(w + ": pools are limited to " + std::to_string(pg::kMaxSegs * pg::kSeg) + " pages");
  return FAT_OK;
}

pg::RowParams row_params(const PageStore& s, const PageRows& r, int32_t* err) {
  pg::RowParams p{};
  p.table = r.table;
  p.pt_sb = r.pt_sb;
  p.max_pages = int(r.max_pages);
  p.lens = r.seq_lens;
  p.owned = r.owned;
  p.refs = r.refs;
  p.released = r.released;
  p.skip_released = r.skip_released && r.released != nullptr;
  p.batch = r.batch;
  p.num_pages = s.num_pages;
  p.page_size = s.page_size;
  p.err = err;
  return p;
}

int check_scratch(const char* what, void* scratch, size_t have, size_t need) {
  if (scratch == nullptr) return invalid(std::string(what) + ": null scratch");
  if (have >= need) return FAT_OK;
  set_last_error(std::string(what) + ": scratch holds " + std::to_string(have) + " bytes, needs " +
                 std::to_string(need));
  return FAT_ERR_WORKSPACE;
}

// Compacting: what follows the pages (rows.table null: nothing, a copy alone).
struct Follow {
  pg::RowParams rows;
  pg::Scratch w;
  int* table_out;
  long long pt_out_sb;
  int* refs_out;
};

template <typename V>
int copy_launch(const PageStore& s, pg::CopyParams p, const Follow* f, const char* what, cudaStream_t stream) {
  // Runs: the widest contiguous pieces of a page.
  const long long row = s.row_bytes;
  pg::Runs& r = p.runs;
  if (s.sh_bytes == row && s.ss_bytes == row * s.num_kv_heads) {
    r = {1, 1, int(row * s.num_kv_heads * s.page_size / (long long)sizeof(V)), 0, 0};
  } else if (s.sh_bytes == row) {
    r = {1, s.page_size, int(row * s.num_kv_heads / (long long)sizeof(V)), 0, s.ss_bytes};
  } else {
    r = {s.page_size, s.num_kv_heads, int(row / (long long)sizeof(V)), s.ss_bytes, s.sh_bytes};
  }
  const int page_vecs = r.n1 * r.n2 * r.vecs;
  // Four times the blocks that fit at once: 4,000 pages of 64 KB take 86 us, 92 us with
  // as many as fit (one long block at the end costs more than a start).
  const int grid_max = sm_count(current_device()) * 32;
  constexpr int kUnroll = 4;
  p.chunk_vecs = kUnroll * pg::kCopyThreads;
  p.chunks = (page_vecs + p.chunk_vecs - 1) / p.chunk_vecs;
  const long long jobs = (long long)p.n * 2 * p.chunks;
  cudaError_t e;
  if (f == nullptr) {
    e = launch_dependent(pg::copy_pages_kernel<V, kUnroll>, dim3(unsigned(std::min<long long>(jobs, grid_max))),
                         pg::kCopyThreads, 0, stream, p);
  } else {
    const long long entries = std::max<long long>((long long)f->rows.batch * f->rows.max_pages, f->rows.num_pages);
    const long long blocks = std::max(jobs, (entries + pg::kCopyThreads - 1) / pg::kCopyThreads);
    e = launch_dependent(pg::move_pages_kernel<V, kUnroll>, dim3(unsigned(std::min<long long>(blocks, grid_max))),
                         pg::kCopyThreads, 0, stream, p, f->rows, f->w, f->table_out, f->pt_out_sb, f->refs_out);
  }
  if (e != cudaSuccess) return cuda_failure(what, e);
  return FAT_OK;
}

int copy_pairs(const PageStore& s, const int* src, const int* dst, int n, const int* n_dev, bool interleaved,
               const Follow* f, int32_t* err, const char* what, cudaStream_t stream) {
  pg::CopyParams p{};
  p.k = static_cast<uint8_t*>(s.k);
  p.v = static_cast<uint8_t*>(s.v);
  p.sp = s.sp_bytes;
  p.num_pages = s.num_pages;
  p.src = src;
  p.dst = dst;
  p.n = n;
  p.n_dev = n_dev;
  p.pair_stride = interleaved ? 2 : 1;
  p.skip_negative = interleaved;
  p.k_scale = s.k_scale;
  p.v_scale = s.v_scale;
  p.scale_sp = s.scale_sp;
  p.heads = s.num_kv_heads;
  p.err = err;
  const uintptr_t bits = reinterpret_cast<uintptr_t>(s.k) | reinterpret_cast<uintptr_t>(s.v) |
                         uintptr_t(s.sp_bytes) | uintptr_t(s.ss_bytes) | uintptr_t(s.sh_bytes) |
                         uintptr_t(s.row_bytes);
  if ((bits & 15u) == 0) return copy_launch<uint4>(s, p, f, what, stream);
  if ((bits & 3u) == 0) return copy_launch<uint32_t>(s, p, f, what, stream);
  return copy_launch<uint8_t>(s, p, f, what, stream);
}

}  // namespace

size_t page_scratch_bytes(int64_t num_pages, int batch) {
  if (num_pages <= 0 || batch <= 0) return 0;
  size_t total = 0;
  carve(nullptr, num_pages, batch, &total);
  return total;
}

int launch_copy_pages(const PageStore& s, const int32_t* src, const int32_t* dst, int n, int32_t* err,
                      cudaStream_t stream) {
  if (n < 0) return invalid("copy_pages: the number of pages must be non-negative");
  const int rc = check_store("copy_pages", s);
  if (rc != FAT_OK || n == 0) return rc;
  if (src == nullptr || dst == nullptr) return invalid("copy_pages: null pointer argument");
  return copy_pairs(s, src, dst, n, nullptr, false, nullptr, err, "copy_pages launch", stream);
}

int launch_fork_rows(const PageStore& s, const PageRows& r, const int32_t* src, const int32_t* dst, int n,
                     void* scratch, size_t scratch_bytes, int32_t* err, cudaStream_t stream) {
  if (n < 0) return invalid("fork: the number of rows must be non-negative");
  int rc = check_store("fork", s);
  if (rc == FAT_OK) rc = check_rows("fork", s, r);
  if (rc != FAT_OK || n == 0) return rc;
  if (src == nullptr || dst == nullptr) return invalid("fork: null pointer argument");
  size_t need = 0;
  const pg::Scratch w = carve(scratch, s.num_pages, r.batch, &need);
  rc = check_scratch("fork", scratch, scratch_bytes, need);
  if (rc != FAT_OK) return rc;
  // All rows of a column tile are staged before any is written: 8 columns (one 32-byte
  // sector per row) while they fit, fewer for very many rows.  Releasing, forking and
  // reserving 256 rows of 1,000 pages takes 30 us so, 62 us with 32 columns (a line).
  constexpr size_t kLimit = 96 * 1024;
  int cols = 8;
  while (cols > 1 && 2 * size_t(n) * cols * sizeof(int) > kLimit) cols >>= 1;
  const size_t smem = 2 * size_t(n) * cols * sizeof(int);
  if (smem > kLimit) return unsupported("fork: at most " + std::to_string(kLimit / 8) + " rows in one call");
  cudaError_t e = ensure_smem_limit(reinterpret_cast<const void*>(pg::fork_kernel), int(kLimit), current_device());
  if (e != cudaSuccess) return cuda_failure("cudaFuncSetAttribute(fork)", e);
  const int grid = int((r.max_pages + cols - 1) / cols);
  e = launch_dependent(pg::fork_kernel, dim3(unsigned(grid)), pg::kBlock, smem, stream, row_params(s, r, err), src, dst,
                       n, cols, w.ticket);
  if (e != cudaSuccess) return cuda_failure("fork launch", e);
  return FAT_OK;
}

int launch_release_rows(const PageStore& s, const PageRows& r, const int32_t* rows, int n, int32_t* err,
                        cudaStream_t stream) {
  if (n < 0) return invalid("release: the number of rows must be non-negative");
  int rc = check_store("release", s);
  if (rc == FAT_OK) rc = check_rows("release", s, r);
  if (rc != FAT_OK || n == 0) return rc;
  if (rows == nullptr) return invalid("release: null pointer argument");
  const cudaError_t e =
      launch_dependent(pg::release_kernel, dim3(unsigned(n)), pg::kBlock, 0, stream, row_params(s, r, err), rows);
  if (e != cudaSuccess) return cuda_failure("release launch", e);
  return FAT_OK;
}

int launch_reserve_tokens(const PageStore& s, const PageRows& r, const int32_t* rows, int n, int tokens,
                          void* scratch, size_t scratch_bytes, int32_t* err, cudaStream_t stream) {
  if (n < 0 || tokens < 0) return invalid("reserve: rows and tokens must be non-negative");
  int rc = check_store("reserve", s);
  if (rc == FAT_OK) rc = check_rows("reserve", s, r);
  if (rc != FAT_OK || n == 0) return rc;
  if (n > r.batch) return invalid("reserve: more rows than the page table has");
  size_t need = 0;
  const pg::Scratch w = carve(scratch, s.num_pages, r.batch, &need);
  rc = check_scratch("reserve", scratch, scratch_bytes, need);
  if (rc != FAT_OK) return rc;
  const int segs = segments(s.num_pages);
  const int grid = counting_blocks(segs, sm_count(current_device()));
  const cudaError_t e = launch_dependent(pg::reserve_kernel, dim3(unsigned(grid)), pg::kBlock, 0, stream,
                                         row_params(s, r, err), w, rows, n, tokens, segs);
  if (e != cudaSuccess) return cuda_failure("reserve launch", e);
  return copy_pairs(s, w.pairs, w.pairs + 1, n, nullptr, true, nullptr, err, "reserve copy launch", stream);
}

int launch_compact_pages(const PageStore& s, const PageRows& r, int32_t* table_out, int64_t pt_out_sb,
                         int32_t* refs_out, int32_t* live_out, void* scratch, size_t scratch_bytes, int32_t* err,
                         cudaStream_t stream) {
  int rc = check_store("compact", s);
  if (rc == FAT_OK) rc = check_rows("compact", s, r);
  if (rc != FAT_OK) return rc;
  if (table_out == nullptr || refs_out == nullptr) return invalid("compact: null pointer argument");
  size_t need = 0;
  const pg::Scratch w = carve(scratch, s.num_pages, r.batch, &need);
  rc = check_scratch("compact", scratch, scratch_bytes, need);
  if (rc != FAT_OK) return rc;
  const int segs = segments(s.num_pages);
  const int sms = sm_count(current_device());
  const pg::RowParams p = row_params(s, r, err);
  cudaError_t e = launch_dependent(pg::live_kernel, dim3(unsigned(counting_blocks(segs, sms))), pg::kBlock, 0, stream, p, w,
                                   live_out, segs);
  if (e == cudaSuccess) e = launch_dependent(pg::list_kernel, dim3(unsigned(segs)), pg::kBlock, 0, stream, p, w);
  if (e != cudaSuccess) return cuda_failure("compact launch", e);
  const Follow f{p, w, table_out, pt_out_sb, refs_out};
  // At most half of the pool can move.
  return copy_pairs(s, w.movers, w.list, int(s.num_pages / 2 + 1), w.info + 1, false, &f, err, "compact copy launch",
                    stream);
}

}  // namespace fat
