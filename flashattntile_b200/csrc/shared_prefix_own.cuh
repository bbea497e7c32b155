// Shared-prefix decode: the tokens that each sequence holds alone.
//
// These parts are many, short and of unequal length (a few tokens to some
// thousand), so the unit of work is small and independent: a *piece* is up to
// piece_tokens tokens of one (sequence, KV head, 8 query heads), and one warp
// takes it from its first byte to its partial (o, m, l).  Warps claim pieces from a
// counter, so CTAs that finish their prefix early take more; a piece's partial goes
// to the piece's own place, so the result does not depend on who took it.
//
// A warp keeps its own ring of stages of token rows, filled by TMA (K and V of a
// stage on one mbarrier): it consumes a stage, refills it with the stage kStages
// ahead -- across pieces -- and then looks up the one after that, so that page ids
// are in registers when a stage comes free.  Nothing is shared between warps.
// Scores and P.V run on mma.sync m16n8k16 with the tokens (then the output columns) as
// the 16 rows and the query heads as the 8 columns, so that no row is idle: S^T = K Q^T,
// O^T = V^T P^T.  P goes in as two 16-bit parts (it keeps about 2^-22); a piece of at
// most 4 heads has both in one product, each head in two columns.  The softmax state
// stays in registers: a lane holds two heads, so O is rescaled without a shuffle, and
// only a vote asks whether a maximum has grown.
#pragma once

#include <math_constants.h>

#include <type_traits>

#include "common.cuh"
#include "groups.cuh"
#include "widen.cuh"

namespace fat {
namespace own {

constexpr int kRows = 8;             // query heads per piece
constexpr float kRescaleLog2 = 8.f;  // running-max slack before O is rescaled
constexpr float kLift = 64.f;        // 8-bit: P is held in units of 1 / kLift
constexpr int kPiecesPerWarp = 4;    // pieces for each of 8 warps per CTA at most (and one per unit)

template <int KVT>
constexpr int elem_bytes() {
  return (KVT == FAT_DTYPE_I8 || KVT == FAT_DTYPE_E4M3) ? 1 : 2;
}

template <int D, int EB>
struct Layout {
  static constexpr int kRowBytes = D * EB;
  static constexpr int kBoxBytes = kRowBytes >= 128 ? 128 : kRowBytes;  // column block of a copy
  static constexpr int kCB = kRowBytes / kBoxBytes;
  static constexpr int kTokens = kRowBytes >= 256 ? 16 : (kRowBytes >= 128 ? 32 : 64);  // per stage
  static constexpr int kTile = kTokens * kRowBytes;  // K (or V) of a stage
  // As many warps as have two stages in flight each (12: all of a 16-bit CTA's; against
  // eight with three stages, 64 sequences with 1,024 own tokens went from 66.1 to 64.5 us).
  static constexpr int kWarps = kRowBytes >= 512 ? 4 : (D <= 128 ? 12 : 8);
  static constexpr int kBudget = 220 * 1024 / kWarps;
  static constexpr int kStages = kBudget / (2 * kTile) > 4 ? 4 : kBudget / (2 * kTile);
  static constexpr int kNoteInts = 6 + (EB == 1 ? 2 * (kTokens / 8) : 0) + 2;
  static constexpr int kNote = (kNoteInts + 3) / 4 * 4;  // ints per stage beside the tiles
  static constexpr size_t kData = size_t(kWarps) * kStages * 2 * kTile;
  static constexpr size_t kSmem = 1024 + kData + size_t(kWarps) * kStages * (8 + 4 * kNote) + 32;
  static_assert(kStages >= 2 && kSmem <= 227 * 1024, "own-token stages");

  // Shared address of byte column `bc` of token row `row` of a tile stored as
  // [row][column block][128 B] under the 128-byte swizzle.
  static __device__ __forceinline__ uint32_t addr(uint32_t tile, int row, int bc) {
    if constexpr (kBoxBytes == 128) {
      const uint32_t seg = uint32_t(row * kCB + (bc >> 7));
      return tile + seg * 128u + ((uint32_t((bc & 127) >> 4) ^ (seg & 7u)) << 4) + uint32_t(bc & 15);
    } else {
      return tile + uint32_t(row * kBoxBytes + bc);
    }
  }
};

struct Params {
  const void* q;
  long long q_sb, q_sh;
  const int* page_table;
  long long pt_sb;
  const int* seq_lens;
  const float* k_scale;
  const float* v_scale;
  long long s_sp;
  Groups groups;
  int num_kv_heads, group, head_groups, num_pages, box_rows, max_pages;
  int rows;             // rows of a piece's partial: min(8, group)
  int workers;          // eight per CTA of the grid: what pieces are sized for
  float scale_log2;
  // Partials by piece: [piece][D / 4][rows][4] and [piece][rows][2] (m, l).
  float* part_o;
  float* part_ml;
  int* counter;         // [0] pieces claimed, [1] 1 + their number once known (zero when the kernel starts)
  int* err;
  unsigned long long wait_ns;
  int expire;
};

// Tokens of sequence b past its group's prefix; `skip` receives the table entries before them.
__device__ __forceinline__ int own_tokens(const Groups& g, const int* seq_lens, int b, int* skip) {
  const int len = min(max(__ldg(seq_lens + b), 0), g.cap_tokens);
  const int shared = g.tokens_of(b);
  *skip = shared / g.page_size;
  return max(len - shared, 0);
}

// Tokens per piece: so many that the warps of the grid get kPiecesPerWarp each (eight
// measure the same to 1%), whole stages, and at least 64: 32 costs up to 17% (33 sequences
// of up to 700 own tokens, e4m3: 69.5 us, 59.3); 128 gains up to 3% there and costs up to
// 5% where own tokens prevail (balance).
__device__ __forceinline__ int piece_tokens(long long own_total, int units, int workers, int stage) {
  const unsigned long long work = (unsigned long long)own_total * unsigned(units);
  const unsigned parts = unsigned(workers) * kPiecesPerWarp;
  const long long want = (work >> 32 ? (long long)(work / parts) : (long long)(unsigned(work) / parts)) + 1;
  return int(min((long long)1 << 30, max((long long)64, (want + stage - 1) / stage * stage)));
}

// Maps pieces, in rising order, to sequences: one warp, 32 sequences at a time.
struct Cursor {
  int c0, before;       // first sequence of the chunk, pieces before it
  int n, incl, len, skip;  // this lane's sequence: parts per unit, pieces up to and with it, tokens, entries skipped

  __device__ __forceinline__ void load(const Params& p, int units, int tokens, int lane) {
    n = len = skip = 0;
    if (c0 + lane < p.groups.batch) len = own_tokens(p.groups, p.seq_lens, c0 + lane, &skip);
    n = (len + tokens - 1) / tokens;
    incl = n * units;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += y;
    }
  }
};

// The 8x8 matrix of 16-bit elements that a warp holds (row lane / 4, columns of lane % 4), transposed.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

template <typename T, int D, int KVT>
__device__ __forceinline__ void own_body(const CUtensorMap& tm_k, const CUtensorMap& tm_v, const Params& p,
                                         const int tokens_per_piece) {
  constexpr int EB = elem_bytes<KVT>();
  using L = Layout<D, EB>;
  constexpr int NT = D / 16;  // 16-column tiles of the output
  // 8-bit caches compute in fp16: codes widen exactly, and a bf16 query row is
  // brought into fp16 exactly by a power of two that returns in the score multiplier.
  using Tc = typename std::conditional<EB == 1, __half, T>::type;
  constexpr bool kQConv = EB == 1 && !std::is_same<T, __half>::value;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t ring = smem_u32(smem) + uint32_t(warp) * L::kStages * 2 * L::kTile;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kData);  // [kWarps][kStages], then `never`
  const uint32_t full = smem_u32(bars) + uint32_t(warp) * L::kStages * 8;
  const uint32_t never = smem_u32(bars) + L::kWarps * L::kStages * 8;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bars + L::kWarps * L::kStages + 1);
  int* notes = reinterpret_cast<int*>(bars + L::kWarps * L::kStages + 2) + warp * L::kStages * L::kNote;
  if (lane == 0) {
    for (int s = 0; s < L::kStages; ++s) mbar_init(full + 8 * s, 1);
    if (warp == 0) {
      mbar_init(never, 1);
      *abort_flag = 0;
    }
    fence_barrier_init();
  }
  asm volatile("bar.sync 1, %0;" ::"n"(L::kWarps * 32) : "memory");

  const int units = p.num_kv_heads * p.head_groups;
  // ---- what is issued next ----
  Cursor cur{0, 0, 0, 0, 0, 0};
  cur.load(p, units, tokens_per_piece, lane);
  int claimed = 0;
  if (lane == 0) claimed = atomicAdd(p.counter, 1);
  struct Next {
    int piece, b, unit, tok, end, len, skip;  // tokens [tok, end) of the piece's len-token sequence are left
    int page, slot;                           // lane's box: table entry, token in it (-1: no rows)
  } nx;
  nx.piece = -1;
  nx.tok = nx.end = 0;
  bool more = true;
  // The stage after the one just issued: the rest of the piece, or the next claimed
  // piece; then this lane's page of it.
  auto look_ahead = [&]() {
    if (nx.tok >= nx.end) {
      const int x = __shfl_sync(0xffffffffu, claimed, 0);
      while (true) {
        const int total = __shfl_sync(0xffffffffu, cur.incl, 31);
        if (x < cur.before + total) break;
        cur.before += total;
        cur.c0 += 32;
        if (cur.c0 >= p.groups.batch) {
          more = false;
          return;
        }
        cur.load(p, units, tokens_per_piece, lane);
      }
      if (lane == 0) claimed = atomicAdd(p.counter, 1);
      const int src = __ffs(__ballot_sync(0xffffffffu, cur.before + cur.incl > x)) - 1;
      const int n = __shfl_sync(0xffffffffu, cur.n, src);
      const int off = x - cur.before - __shfl_sync(0xffffffffu, cur.incl, src) + n * units;
      nx.piece = x;
      nx.b = cur.c0 + src;
      nx.len = __shfl_sync(0xffffffffu, cur.len, src);
      nx.skip = __shfl_sync(0xffffffffu, cur.skip, src);
      nx.unit = off / n;
      nx.tok = (off - nx.unit * n) * tokens_per_piece;
      nx.end = min(nx.len, nx.tok + tokens_per_piece);
    }
    nx.page = 0;
    nx.slot = -1;
    const int t = nx.tok + lane * p.box_rows;
    if (lane * p.box_rows < L::kTokens && t < nx.end) {
      const int lp = t / p.groups.page_size;
      nx.slot = t - lp * p.groups.page_size;
      const int entry = nx.skip + lp;
      // Checked in issue(): a use here would wait for the load.
      nx.page = -1;
      if (entry < p.max_pages) nx.page = __ldg(p.page_table + (long long)nx.b * p.pt_sb + entry);
    }
  };
  int issued = 0, fresh = 1;  // fresh: the stage begins a piece
  const uint64_t policy = policy_evict_first();
  auto issue = [&]() {
    const int s = issued % L::kStages;
    const bool listed = nx.page >= 0 && nx.page < p.num_pages, ok = nx.slot >= 0 && listed;
    if (nx.slot >= 0 && !listed) raise_error(p.err, FAT_DEVERR_BAD_PAGE);
    const unsigned okmask = __ballot_sync(0xffffffffu, ok);
    const int kvh = nx.unit / p.head_groups;
    const int n = min(L::kTokens, nx.end - nx.tok);
    int* note = notes + s * L::kNote;
    if constexpr (EB == 1) {
      // One scale pair per 8 tokens; 0 where no page is, so that no stale value counts.
      const int per8 = p.box_rows / 8;
      const int page = __shfl_sync(0xffffffffu, ok ? nx.page : -1, (lane / per8) & 31);
      if (lane < L::kTokens / 8) {
        int* at = note + 8 + 2 * lane;
        if (page >= 0) {
          cp_async_4(smem_u32(at), p.k_scale + (long long)page * p.s_sp + kvh);
          cp_async_4(smem_u32(at + 1), p.v_scale + (long long)page * p.s_sp + kvh);
        } else {
          at[0] = at[1] = 0;
        }
      }
    }
    cp_async_commit();
    const uint32_t bar = full + 8 * s;
    if (lane == 0) {
      note[0] = nx.piece;
      note[1] = nx.b;
      note[2] = nx.unit;
      note[3] = n;
      note[4] = (fresh ? 1 : 0) | (nx.tok + n >= nx.end ? 2 : 0);
      mbar_arrive_expect_tx(bar, uint32_t(__popc(okmask)) * uint32_t(p.box_rows) * L::kRowBytes * 2u);
    }
    __syncwarp();
    if (ok) {
      const uint32_t dst = ring + uint32_t(s) * 2 * L::kTile + uint32_t(lane * p.box_rows * L::kRowBytes);
      tma_load_5d_hint(dst, &tm_k, bar, 0, 0, kvh, nx.slot, nx.page, policy);
      tma_load_5d_hint(dst + L::kTile, &tm_v, bar, 0, 0, kvh, nx.slot, nx.page, policy);
    }
    ++issued;
    nx.tok += n;
    fresh = nx.tok >= nx.end;
  };

  if (p.expire && warp == 0) mbar_wait_bounded(never, 0, p.err, abort_flag, p.wait_ns);
  look_ahead();
  for (int i = 0; i < L::kStages && more; ++i) {
    issue();
    look_ahead();
  }

  // ---- consume ----
  const int g = lane >> 2, c = lane & 3;
  const bool twice = p.rows <= kRows / 2;  // columns 4-7 repeat the heads of columns 0-3
  float o[NT][4];                          // columns d of rows g, g + 8 of the tile; heads 2c, 2c + 1
  float m0 = -CUDART_INF_F, m1 = -CUDART_INF_F, l0 = 0.f, l1 = 0.f;  // of heads 2c, 2c + 1
  float qmul0 = 1.f, qmul1 = 1.f;
  // 8-bit: P carries the V scale in units of a power of two above every one of the piece so
  // far, times kLift, so that it neither leaves fp16 nor loses bits, whatever V's size.
  float vunit = 0.f, vinv = 0.f;
  uint32_t qb[D / 16][2];
  int done = 0;
  while (done < issued) {
    const int s = done % L::kStages;
    if (!mbar_wait_bounded(full + 8 * s, uint32_t((done / L::kStages) & 1), p.err, abort_flag, p.wait_ns)) break;
    if constexpr (EB == 1) {
      cp_async_wait<L::kStages - 1>();
      __syncwarp();
    }
    const int* note = notes + s * L::kNote;
    const int flags = note[4], n_valid = note[3];
    if (flags & 1) {
      m0 = m1 = -CUDART_INF_F;
      l0 = l1 = 0.f;
      vunit = vinv = 0.f;
#pragma unroll
      for (int n = 0; n < NT; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
      const int b = note[1], unit = note[2];
      const int kvh = unit / p.head_groups, hg = unit - kvh * p.head_groups;
      const int head = twice ? g & 3 : g;
      const bool row = head < min(kRows, p.group - hg * kRows);
      const T* qs = reinterpret_cast<const T*>(p.q) + (long long)b * p.q_sb +
                    (long long)(kvh * p.group + hg * kRows + (row ? head : 0)) * p.q_sh;
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        // 8-bit caches use a permuted reduction order (see the K fragments below).
        const int d0 = (EB == 2) ? ks * 16 + 2 * c : c * (D / 4) + 4 * ks;
        const int d1 = (EB == 2) ? ks * 16 + 8 + 2 * c : c * (D / 4) + 4 * ks + 2;
        qb[ks][0] = row ? __ldg(reinterpret_cast<const unsigned*>(qs + d0)) : 0u;
        qb[ks][1] = row ? __ldg(reinterpret_cast<const unsigned*>(qs + d1)) : 0u;
      }
      if constexpr (kQConv) {
        // The power of two that puts the row's largest magnitude in [2^14, 2^15).
        float mx = 0.f;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
          float x0, x1, x2, x3;
          unpack2<T>(qb[ks][0], x0, x1);
          unpack2<T>(qb[ks][1], x2, x3);
          mx = fmaxf(mx, fmaxf(fmaxf(fabsf(x0), fabsf(x1)), fmaxf(fabsf(x2), fabsf(x3))));
        }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        int e = 0;
        if (mx > 0.f && mx < CUDART_INF_F) e = max(-126, min(126, ((__float_as_int(mx) >> 23) & 0xFF) - 127 - 14));
        const float down = __int_as_float((127 - e) << 23);
        const float up = __int_as_float((127 + e) << 23);
        qmul0 = __shfl_sync(0xffffffffu, up, 8 * c);  // lanes of head 2c, 2c + 1
        qmul1 = __shfl_sync(0xffffffffu, up, 8 * c + 4);
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float x0, x1;
            unpack2<T>(qb[ks][h], x0, x1);
            qb[ks][h] = pack2<__half>(x0 * down, x1 * down);
          }
        }
      }
    }
    const uint32_t kt = ring + uint32_t(s) * 2 * L::kTile, vt = kt + L::kTile;
    // 16 tokens are one step of the MMAs; where a stage holds more, two steps go side by
    // side, so that one's latencies pass under the other's.
    constexpr int kSteps = L::kTokens >= 32 ? 2 : 1;
#pragma unroll 1
    for (int wrow = 0; wrow < n_valid; wrow += 16 * kSteps) {
      const int nvalid = n_valid - wrow;
      if (nvalid < 16 * kSteps) {
        // Rows past the tokens may hold anything: zero their V so that p = 0 adds nothing.
        constexpr int kVecPerRow = L::kRowBytes / 16;
        for (int i = lane; i < (16 * kSteps - nvalid) * kVecPerRow; i += 32) {
          const int r = nvalid + i / kVecPerRow;
          st_shared_v4(L::addr(vt, wrow + r, (i % kVecPerRow) * 16), 0u, 0u, 0u, 0u);
        }
        __syncwarp();
      }
      // ---- S^T = K Q^T; two accumulators per step, for a shorter chain ----
      float sacc[kSteps][2][4];
#pragma unroll
      for (int j = 0; j < kSteps; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) sacc[j][0][i] = sacc[j][1][i] = 0.f;
      if constexpr (EB == 2) {
        const int row = wrow + (lane & 15);
        const int khalf = (lane >> 4) * 8;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
#pragma unroll
          for (int j = 0; j < kSteps; ++j) {
            uint32_t a[4];
            ldsm_x4(L::addr(kt, row + 16 * j, (ks * 16 + khalf) * 2), a[0], a[1], a[2], a[3]);
            MmaOp<Tc>::run(sacc[j][ks & 1], a, qb[ks][0], qb[ks][1]);
          }
        }
      } else {
        // Lane (g, c) owns the reduction slice d in [c*D/4, (c+1)*D/4) of token rows g
        // and g+8: k-step ks maps its k-slots (2c, 2c+1) to dims c*D/4 + 4ks + {0,1} and
        // (2c+8, 2c+9) to + {2,3}, as the query fragments do; each lane reads contiguous bytes.
        constexpr int kSlice = D / 4;
        constexpr int kVec = kSlice >= 16 ? 4 : 2;  // words per load
#pragma unroll
        for (int v = 0; v < kSlice / (4 * kVec); ++v) {
          uint32_t wv[2 * kSteps][4];
#pragma unroll
          for (int j = 0; j < 2 * kSteps; ++j) {
            const uint32_t at = L::addr(kt, wrow + j * 8 + g, c * kSlice + v * 4 * kVec);
            if constexpr (kVec == 4) {
              asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                           : "=r"(wv[j][0]), "=r"(wv[j][1]), "=r"(wv[j][2]), "=r"(wv[j][3])
                           : "r"(at));
            } else {
              asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(wv[j][0]), "=r"(wv[j][1]) : "r"(at));
            }
          }
#pragma unroll
          for (int i = 0; i < kVec; ++i) {
            const int ks = v * kVec + i;
#pragma unroll
            for (int j = 0; j < kSteps; ++j) {
              uint32_t a[4];
              Widen<Tc, KVT>::run(wv[2 * j][i], a[0], a[2]);
              Widen<Tc, KVT>::run(wv[2 * j + 1][i], a[1], a[3]);
              MmaOp<Tc>::run(sacc[j][ks & 1], a, qb[ks][0], qb[ks][1]);
            }
          }
        }
      }
      // 8-bit: V's words are on the way during the softmax.  Lane (g, c) owns output dims
      // [g*D/8, (g+1)*D/8) (rows g and g + 8 of tile n are dims g*D/8 + 2n and + 1) and
      // reads token rows 2c, 2c+1, 2c+8, 2c+9 of a step.
      constexpr int kSliceV = D / 8;
      [[maybe_unused]] uint32_t rw[EB == 1 ? 4 * kSteps : 1][EB == 1 ? kSliceV / 4 : 1];
      if constexpr (EB == 1) {
#pragma unroll
        for (int r = 0; r < 4 * kSteps; ++r) {
          const int row = wrow + 2 * c + (r & 1) + (r >> 1) * 8;
#pragma unroll
          for (int v = 0; v < kSliceV / 4; v += 4) {
            const uint32_t a = L::addr(vt, row, g * kSliceV + v * 4);
            if constexpr (kSliceV >= 16) {
              asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                           : "=r"(rw[r][v]), "=r"(rw[r][v + 1]), "=r"(rw[r][v + 2]), "=r"(rw[r][v + 3])
                           : "r"(a));
            } else if constexpr (kSliceV >= 8) {
              asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(rw[r][v]), "=r"(rw[r][v + 1]) : "r"(a));
            } else {
              asm volatile("ld.shared.u32 %0, [%1];" : "=r"(rw[r][v]) : "r"(a));
            }
          }
        }
      }
      // ---- online softmax on the fragment (rows: tokens; columns 2c, 2c + 1: heads) ----
      // Row half r: tokens 8 r + g of the step(s).
      float s0[2 * kSteps], s1[2 * kSteps], vf[2 * kSteps];
      float mx0 = -CUDART_INF_F, mx1 = -CUDART_INF_F;
#pragma unroll
      for (int r = 0; r < 2 * kSteps; ++r) {
        float f0 = p.scale_log2, f1 = p.scale_log2;
        vf[r] = 1.f;
        if constexpr (EB == 1) {
          const float* sc = reinterpret_cast<const float*>(note + 8) + 2 * (wrow / 8 + r);
          f0 = p.scale_log2 * qmul0 * sc[0];
          f1 = p.scale_log2 * qmul1 * sc[0];
          vf[r] = sc[1];
        }
        const float(&x)[2][4] = sacc[r >> 1];
        const int i = 2 * (r & 1);
        const bool in = 8 * r + g < nvalid;
        s0[r] = in ? (x[0][i] + x[1][i]) * f0 : -CUDART_INF_F;
        s1[r] = in ? (x[0][i + 1] + x[1][i + 1]) * f1 : -CUDART_INF_F;
        mx0 = fmaxf(mx0, s0[r]);
        mx1 = fmaxf(mx1, s1[r]);
      }
      if constexpr (EB == 1) {
        float vm = 0.f;  // the same in every lane
#pragma unroll
        for (int r = 0; r < 2 * kSteps; ++r) {
          const float f = fabsf(vf[r]);
          vm = fmaxf(vm, f >= 1.17549435e-38f && f < CUDART_INF_F ? f : 0.f);
        }
        if (vm > vunit) {
          const int e = min(253, ((__float_as_int(vm) >> 23) & 0xFF) + 1);
          const float up = __int_as_float(e << 23), a = vunit / up;  // o is 0 before the first unit
          vunit = up;
          vinv = __int_as_float((254 - e) << 23);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int i = 0; i < 4; ++i) o[n][i] *= a;
          }
        }
#pragma unroll
        for (int r = 0; r < 2 * kSteps; ++r) vf[r] = vf[r] * vinv * kLift;  // in this order: vinv may be 2^125
      }
      if (__any_sync(0xffffffffu, mx0 > m0 + kRescaleLog2 || mx1 > m1 + kRescaleLog2)) {
#pragma unroll
        for (int k = 4; k < 32; k <<= 1) {
          mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, k));
          mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, k));
        }
        const float n0 = mx0 > m0 + kRescaleLog2 ? mx0 : m0, n1 = mx1 > m1 + kRescaleLog2 ? mx1 : m1;
        const float a0 = m0 == -CUDART_INF_F ? 1.f : fast_exp2(m0 - n0);
        const float a1 = m1 == -CUDART_INF_F ? 1.f : fast_exp2(m1 - n1);
        m0 = n0;
        m1 = n1;
        l0 *= a0;
        l1 *= a1;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          o[n][0] *= a0;
          o[n][1] *= a1;
          o[n][2] *= a0;
          o[n][3] *= a1;
        }
      }
      const float b0 = m0 == -CUDART_INF_F ? 0.f : m0, b1 = m1 == -CUDART_INF_F ? 0.f : m1;
      // P rounded to 16 bits, and the remainder, as columns of the second product.
      uint32_t hi[2 * kSteps], lo[2 * kSteps];
#pragma unroll
      for (int r = 0; r < 2 * kSteps; ++r) {
        const float p0 = fast_exp2(s0[r] - b0), p1 = fast_exp2(s1[r] - b1);
        l0 += p0;
        l1 += p1;
        split_hi_lo<Tc>(p0 * vf[r], p1 * vf[r], hi[r], lo[r]);
        hi[r] = transpose8x8(twice && c >= 2 ? lo[r] : hi[r]);
        if (!twice) lo[r] = transpose8x8(lo[r]);
      }
      // ---- O^T += V^T P^T ----
      auto add_pv = [&](float(&acc)[4], const uint32_t(&a)[4], int j) {
        MmaOp<Tc>::run(acc, a, hi[2 * j], hi[2 * j + 1]);
        if (!twice) MmaOp<Tc>::run(acc, a, lo[2 * j], lo[2 * j + 1]);
      };
      if constexpr (EB == 2) {
        const int row = wrow + ((lane >> 4) << 3) + (lane & 7);
        const int dsel = ((lane >> 3) & 1) << 3;
#pragma unroll
        for (int j = 0; j < kSteps; ++j) {
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            uint32_t a[4];
            ldsm_x4_t(L::addr(vt, row + 16 * j, (n * 16 + dsel) * 2), a[0], a[1], a[2], a[3]);
            add_pv(o[n], a, j);
          }
        }
      } else {
        // A byte of two token rows makes the pair of one A register.
#pragma unroll
        for (int j = 0; j < kSteps; ++j) {
          const uint32_t(&x)[kSliceV / 4] = rw[4 * j], (&y)[kSliceV / 4] = rw[4 * j + 1];
          const uint32_t(&z)[kSliceV / 4] = rw[4 * j + 2], (&t)[kSliceV / 4] = rw[4 * j + 3];
#pragma unroll
          for (int w = 0; w < kSliceV / 4; ++w) {
            uint32_t a[2][4];
            Widen<Tc, KVT>::run(__byte_perm(x[w], y[w], 0x5140), a[0][0], a[0][1]);
            Widen<Tc, KVT>::run(__byte_perm(x[w], y[w], 0x7362), a[1][0], a[1][1]);
            Widen<Tc, KVT>::run(__byte_perm(z[w], t[w], 0x5140), a[0][2], a[0][3]);
            Widen<Tc, KVT>::run(__byte_perm(z[w], t[w], 0x7362), a[1][2], a[1][3]);
            add_pv(o[2 * w], a[0], j);
            add_pv(o[2 * w + 1], a[1], j);
          }
        }
      }
    }
    constexpr int kWhole = 16 * kSteps;
    if (n_valid % kWhole != 0) fence_proxy_async_smem();  // zeroed rows: the stage is copied to again

    if (flags & 2) {
      // ---- the piece's partial ----
      const int unit = note[2];
      const long long x = note[0];
      const int kvh = unit / p.head_groups, hg = unit - kvh * p.head_groups;
      const int rows = min(kRows, p.group - hg * kRows);
#pragma unroll
      for (int k = 4; k < 32; k <<= 1) {
        l0 += __shfl_xor_sync(0xffffffffu, l0, k);
        l1 += __shfl_xor_sync(0xffffffffu, l1, k);
      }
      // Where columns repeat heads, lanes c and c ^ 2 hold the two parts' sums: each adds
      // up one of its two rows.
      const int h0 = twice ? 2 * (c & 1) : 2 * c;
      float* at = p.part_o + (x * (D / 4) * p.rows + h0) * 4;
      auto put = [&](int d, float y0, float y1) {
        float* to = at + (long long)(d >> 2) * p.rows * 4 + (d & 3);
        if constexpr (EB == 1) {
          y0 *= vunit * (1.f / kLift);
          y1 *= vunit * (1.f / kLift);
        }
        if (h0 < rows) to[0] = y0;
        if (h0 + 1 < rows) to[4] = y1;
      };
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int d0 = EB == 2 ? n * 16 + g : g * (D / 8) + 2 * n, d1 = EB == 2 ? d0 + 8 : d0 + 1;
        if (twice) {
          const bool low = c < 2;
          const float y0 = (low ? o[n][0] : o[n][2]) + __shfl_xor_sync(0xffffffffu, low ? o[n][2] : o[n][0], 2);
          const float y1 = (low ? o[n][1] : o[n][3]) + __shfl_xor_sync(0xffffffffu, low ? o[n][3] : o[n][1], 2);
          put(low ? d0 : d1, y0, y1);
        } else {
          put(d0, o[n][0], o[n][1]);
          put(d1, o[n][2], o[n][3]);
        }
      }
      if (g == 0 && (!twice || c < 2)) {
        float2* ml = reinterpret_cast<float2*>(p.part_ml + (x * p.rows + h0) * 2);
        if (h0 < rows) ml[0] = make_float2(m0, l0);
        if (h0 + 1 < rows) ml[1] = make_float2(m1, l1);
      }
    }
    __syncwarp();
    ++done;
    if (more) {
      issue();
      look_ahead();
    }
  }
  cp_async_wait<0>();
  if (*abort_flag) {
    // Drain this warp's own copies before the shared memory goes away.
    for (int j = max(done, issued - L::kStages); j < issued; ++j)
      mbar_wait_bounded(full + 8 * (j % L::kStages), uint32_t((j / L::kStages) & 1), nullptr, nullptr, p.wait_ns);
  }
}

}  // namespace own
}  // namespace fat
