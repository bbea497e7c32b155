// Decode attention for groups of sequences that share a prefix (sm_100a).
//
// The n sequences of a group hold the same pages for their first S tokens.  Per
// KV head, the n * G query rows that read it (G query heads per KV head) make one
// matrix product with the prefix, so every prefix byte is read once per group
// (and per 256 rows) instead of once per sequence, on the tensor cores at an
// intensity of n * G FLOP per byte (16-bit cache).  The tokens that a sequence
// holds alone are taken by single warps in small pieces (shared_prefix_own.cuh), and
// a small kernel joins the partials by log-sum-exp:
//   out = (sum_i o_i 2^(m_i - M)) / (sum_i l_i 2^(m_i - M)),  M = max_i m_i,
// over the partials i of a row: o_i = sum_t 2^(s_t - m_i) v_t, l_i = sum_t 2^(s_t - m_i).
//
// One launch does both, one CTA per SM: some CTAs begin with a share of the prefix,
// in proportion to the work that every CTA counts from the lengths, and all CTAs
// claim pieces of the own tokens until none is left.  So the latencies of the two
// parts pass side by side, and CTAs that finish early take more.
//
// Prefix CTAs: the KV tiles of all (group, KV head) units lie on one line that is
// cut evenly over them; a group with more rows than a CTA holds takes several CTAs
// per cut (a gang), which walk the same tiles side by side.  Warp-specialised:
//   softmax warpgroups (one per stream): thread r owns row r (tensor-memory lane r);
//   producer warps: page ids and K/V tiles by TMA; MMA issuer: one thread;
//   8-bit caches: converter warpgroups (one for K, one for V) widen raw tiles to fp16
//   (exactly).
// Two streams overlap softmax with the tensor core.  With more than 128 rows a
// stream is a row tile (both read each K/V tile: its bytes serve 256 rows); with up
// to 128 rows the streams take the two halves of each tile's tokens for the one row
// tile.  head_dim 256 fills tensor memory with one stream.  A stream takes 64 tokens
// at a time (a unit) and has two buffers of scores, so that the scores of the next
// unit are computed while the softmax works on these.
// Tensor memory: the buffers of S_t at columns 128 t and 128 t + 64 (P is written over
// them), O_t from column 256.
// Every wait is bounded; on a timeout the CTA records FAT_DEVERR_TIMEOUT, drains
// its copies and MMAs, frees tensor memory and exits.
//
// What bounds it, and what it measured (one call after another, the join included; copies
// run at 6.5 TB/s):
//   8 sequences of 133k tokens, 131k shared, 64/8 heads of 128, fp16: 568 MB in 134 to
//     140 us, 4.1 TB/s (116 us in short runs of a graph).  5 us of start, 9 us of join; the
//     second part of P costs 4 to 17 us of it, the more the longer such calls run.
//   64 sequences of 8k + up to 1k tokens, 32/8 heads, bf16: 196 MB in 60 us.  The own
//     tokens are two thirds of the bytes: latency of single warps.
//   128 sequences of 16k + up to 512, 32/8 heads, int8: 101 MB in 109 us: a 16k prefix
//     against 512 rows is compute, in long dependent chains: 40% of the issue slots and 26%
//     of the tensor pipe are used.
// MMA issue: one elected thread; a branch on the lane number instead made each MMA cost
// about 80 cycles of issue, and a unit of both streams 1.6 us instead of 1.05.
#pragma once

#include <math_constants.h>

#include <algorithm>
#include <string>
#include <type_traits>

#include "common.cuh"
#include "groups.cuh"
#include "host_util.h"
#include "shared_prefix.h"
#include "shared_prefix_own.cuh"
#include "tcgen05.cuh"
#include "widen.cuh"

namespace fat {
namespace spx {

constexpr int BM = 128;                // rows per tile (the MMA's M)
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kColO = 256;
constexpr float kRescaleLog2 = 8.f;    // running-max slack before O is rescaled
// P is held in units of 2^-7, so at most 2^15: what is small beside a heavy key stays
// normal in fp16 for as long as it can.
constexpr float kLiftLog2 = 7.f;
// 8-bit: a V scale below the normal floats, or below 2^-100 of a larger one before it or in
// its tile, counts as 0 (P in units of the larger one would leave fp32).
constexpr float kLeastScale = 1.17549435e-38f;
constexpr float kLeastRatio = 7.8886091e-31f;
constexpr long long kMaxTiles = (1ll << 31) - 1;  // tiles on the line (2^38 tokens times KV heads)

// Streams: two row tiles, one row tile with half of each tile's tokens each, or one
// stream.  The rule is the group's rows: up to 128 a second row tile would be empty (an
// e4m3 case of 32 rows: 59 us, 78 as a pair), past it one row tile per CTA would read and
// widen every prefix byte once more (512 rows of 16k shared tokens, int8, head_dim 64:
// 80 us, 91 so).
enum Mode { kRowPair, kAlternate, kSolo };

enum KvType { kKv16, kKvI8, kKvE4M3 };

constexpr int kUnit = 64;  // tokens whose scores are taken at a time: two buffers per stream

template <int D, Mode kMode, bool k8>
struct Layout {
  static constexpr int kStreams = kMode == kSolo ? 1 : 2;
  static constexpr int kRowTiles = kMode == kRowPair ? 2 : 1;
  static constexpr int kRows = BM * kRowTiles;        // rows per CTA
  static constexpr int BN = D <= 128 ? 128 : 64;      // tokens per K/V tile
  static constexpr int kUnits = kMode == kRowPair ? BN / kUnit : 1;  // units of a tile, per stream
  static constexpr int kCB = D / 64;                  // 128-byte column blocks (16-bit elements)
  static constexpr int kQTile = BM * D * 2;
  static constexpr int kStage = k8 ? kUnit : BN;      // tokens of a stage of 16-bit K or V
  static constexpr int kHalves = BN / kStage;         // stages of a tile
  static constexpr int kTile = kStage * D * 2;        // one stage
  static constexpr int kRaw = BN * D;                 // one 8-bit K or V tile
  // As many stages as shared memory holds beside Q: bytes in flight set the
  // streaming rate.  8-bit: a few small 16-bit stages of each, the rest raw.
  static constexpr int kBudget = 224 * 1024 - kRowTiles * kQTile;
  static constexpr int kStagesK = k8 ? (kMode == kSolo ? 2 : kMode == kRowPair ? 3 : 4) : std::min(8, (kBudget / kTile + 1) / 2);
  static constexpr int kStagesV = k8 ? (kMode == kSolo ? 2 : kMode == kRowPair ? 3 : 4) : std::min(8, kBudget / kTile / 2);
  static constexpr int kStagesRaw = k8 ? std::min(8, (kBudget - 2 * kStagesK * kTile) / kRaw) / 2 * 2 : 0;
  static_assert(!k8 || kStagesRaw >= 2, "raw ring needs a K and a V stage");
  static_assert(kStagesK >= 2 && kStagesV >= 2, "rings too small");
  // 8-bit: tiles whose scales are in shared memory.  The producer writes those of
  // tile j once the raw K stage of tile j - kStagesRaw / 2 is free, so its K is
  // converted, so the scores of tile i = j - kStagesRaw / 2 - (K stages in tiles) were
  // issued, so P of tile i - 2 was written: its scales are read.
  static constexpr int kScaleSlots = k8 ? kStagesRaw / 2 + (kStagesK + kHalves - 1) / kHalves + 2 : 1;
  static constexpr int kSoftmaxThreads = 128 * kStreams;
  static constexpr int kProducerWarp = 4 * kStreams;
  static constexpr int kMmaWarp = kProducerWarp + 1;
  static constexpr int kVProducerWarp = kProducerWarp + 2;
  static constexpr int kQWarp = kProducerWarp + 3;
  static constexpr int kConvWarp = kProducerWarp + 4;
  static constexpr int kConvWarps = k8 ? (kStreams == 2 ? 8 : 4) : 0;  // four each for K and V, or for both
  static constexpr int kThreads = kSoftmaxThreads + 128 + kConvWarps * 32;
  // Registers.  16-bit: 384 threads launch at 168; the softmax holds 64 scores and their
  // working set: 208 * 256 + 88 * 128 = 384 * 168; for the own tokens all twelve warps
  // return to 168.  8-bit: 640 threads launch at 96:
  // 144 * 256 + 64 * 384 = 640 * 96, and the own tokens' twelve warps get
  // 144 * 384 + 24 * 256 = 640 * 96.
  static constexpr bool kSplitRegs = kStreams == 2;
  static constexpr int kRegsSoftmax = k8 ? 144 : 208;
  static constexpr int kRegsOther = k8 ? 64 : 88;
  static constexpr int kRegsOwn = k8 ? 144 : 168;
  static constexpr int kRegsIdle = k8 ? 24 : 168;
  static constexpr int kLaunchRegs = k8 ? 96 : 168;
  static_assert(!kSplitRegs || 256 * kRegsSoftmax + (kThreads - 256) * kRegsOther <= kThreads * kLaunchRegs,
                "register split exceeds the launch");
  static_assert(!kSplitRegs || !k8 || 384 * kRegsOwn + (kThreads - 384) * kRegsIdle <= kThreads * kLaunchRegs,
                "register split exceeds the launch");
  // What a tile costs a CTA, in units of 32 KB of own tokens.  Swept over sixteen shapes:
  // half or twice them costs up to 50%; over 28 more (head_dim 64 and 128), up to 1.35
  // times them measures within 3%.  What matters is on which side of a step the whole
  // units (choose_gangs) fall, and that enough CTAs begin with the own tokens, since a
  // prefix CTA comes to them late: 512 rows, 16k shared and up to 512 own tokens, int8, take
  // 105 us, 115 at 3.0; 24 sequences, 16 heads of 64, 16k shared and up to 64 own, fp16,
  // 24 us, 28 at 1.95.
  static constexpr float kTileCost =
      (kMode == kRowPair ? (k8 ? 2.6f : 3.3f) : (k8 ? 1.4f : 1.7f)) * (D == 64 ? 0.75f : 1.f);
  static constexpr int kBars = 4 + 2 * kStagesK + 2 * kStagesV + 6 * kStreams + 3 + 2 * kStagesRaw +
                               (k8 ? kScaleSlots : 0);
  // Per 8 tokens: K scale, log2 of the V scale's size in units, its reciprocal; then the
  // unit and the K and V masks (bits 0-15 zero, 16-31 negative).
  static constexpr int kScaleRow = 3 * (BN / 8) + 4;
  static constexpr int kScaleFloats = k8 ? kScaleSlots * kScaleRow : 0;
  static constexpr size_t kData = size_t(kRowTiles) * kQTile + size_t(kStagesK + kStagesV) * kTile +
                                  size_t(kStagesRaw) * kRaw;
  static constexpr size_t kSmem = 1024 + kData + size_t(kScaleFloats) * 4 + size_t(kBars) * 8 + 48 + 32 * 4 * kStreams;
  static_assert(kSmem <= 227 * 1024, "shared memory");
};

struct Params {
  int q_bf16;            // 8-bit caches: q is bf16 (brought into fp16 by a power of two)
  int q_negate;          // the softmax scale is negative: its sign moves into q
  int tile_rows;         // rows of a row tile: as many whole sequences as 128 rows hold
  float scale_log2;      // |softmax scale| * log2(e)
  Groups groups;
  const int* page_table;
  long long pt_sb;
  const int* seq_lens;
  int max_pages, num_pages, page_size, box_rows;
  int num_kv_heads, group, head_dim;
  const float* k_scale;
  const float* v_scale;
  long long s_sp;
  int per_gang;          // CTAs that walk the same tiles, for groups of more rows than a CTA holds
  int* info;             // what the joining kernel needs: the number of gangs,
  int2* first_piece;     // [batch] own pieces before a sequence, and its pieces per unit
  // Partials.  Slots: [CTA][2][D / 4][256 rows][4] and [CTA][2][256][2] (m, l).
  // Home (units that one gang covers): [streams' parts][kv head][D / 4][row][4], row = first * group + r.
  float* slot_o;
  float* slot_ml;
  float* home_o;
  float* home_ml;
  long long home_rows;
  int* err;
  unsigned long long wait_ns;
  int expire;
};

// The line of K/V tiles: group by group, KV head by KV head, tile by tile.
struct Line {
  const Groups& g;
  int bn, heads;
  __device__ __forceinline__ int tiles(int i) const {
    return g.size(i) > 0 ? (g.tokens(i) + bn - 1) / bn : 0;
  }
};

// Where range c of n begins on a line of `total`; the 64-bit quotient takes several
// times as long, on the way of every CTA's first copy.
__device__ __forceinline__ long long cut(long long c, long long total, int n) {
  const unsigned long long x = (unsigned long long)(c * total);
  return x >> 32 ? (long long)(x / unsigned(n)) : (long long)(unsigned(x) / unsigned(n));
}

// A CTA's piece of one unit.
struct Piece {
  int first, kvh, rows, row0;  // first sequence, KV head, this CTA's rows and the first of them
  int t0, t1, n, tokens;       // tiles [t0, t1) of the unit's n, shared tokens
  int leading;                 // the piece starts the CTA's range (its slot is 0)
};

// Walks the pieces of the range [x, x1); every role walks on its own.  Positions
// fit 32 bits (a longer line is refused when the range is found).
struct Walk {
  int x, x1, x0, base;
  int g, n, first, size, tokens;  // the group at x: its tiles per unit, sequences, shared tokens

  __device__ __forceinline__ void load(const Params& p, int bn) {
    first = p.groups.first(g);
    size = p.groups.size(g);
    tokens = p.groups.tokens(g);
    n = size > 0 ? (tokens + bn - 1) / bn : 0;
  }

  template <int kRowTiles>
  __device__ __forceinline__ bool next(const Params& p, int bn, int member, Piece& w) {
    const int cta_rows = kRowTiles * p.tile_rows;
    while (x < x1) {
      if (x >= base + n * p.num_kv_heads) {
        base += n * p.num_kv_heads;
        if (++g >= p.groups.count) return false;
        load(p, bn);
        continue;
      }
      const int off = x - base;
      w.kvh = off / n;
      w.t0 = off - w.kvh * n;
      w.t1 = min(n, w.t0 + (x1 - x));
      w.n = n;
      w.leading = x == x0;
      x += w.t1 - w.t0;
      w.row0 = member * cta_rows;
      w.rows = min(cta_rows, size * p.group - w.row0);
      if (w.rows <= 0) continue;  // a smaller group than the gang is made for
      w.first = first;
      w.tokens = tokens;
      return true;
    }
    return false;
  }
};

// Two probabilities for P.V, as two 16-bit parts in two products: what the type keeps of
// them (cut: bf16 8 bits, fp16 11) and the remainder, of which 2^-17 or 2^-21 of the whole
// is left out; s0 and s1 sum them in 32 bits.  One part alone costs a result up to as much
// again as its own rounding to the type, and in 8-bit caches, where P carries the V scale,
// a group whose scale is far below its neighbours' would vanish from a sum of rounded P.
// The second product costs nothing where own tokens prevail, 4 to 6% in 8-bit documents and
// up to 14% where the prefix is most of an fp16 call.
template <typename T>
__device__ __forceinline__ uint32_t split_p(float p0, float p1, float& s0, float& s1, uint32_t& rest) {
  constexpr uint32_t kKeep = std::is_same<T, __nv_bfloat16>::value ? 0xffff0000u : 0xffffe000u;
  float r0 = p0, r1 = p1;  // less the cut values: probabilities have no sign, so one operation each
  add2(r0, r1, __uint_as_float((__float_as_uint(p0) & kKeep) | 0x80000000u),
       __uint_as_float((__float_as_uint(p1) & kKeep) | 0x80000000u));
  add2(s0, s1, p0, p1);
  rest = pack2<T>(r0, r1);
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    return __byte_perm(__float_as_uint(p0), __float_as_uint(p1), 0x7632);
  uint32_t h;
  asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(h) : "f"(p1), "f"(p0));
  return h;
}

// True in one thread of a whole warp, in a form that the compiler knows to be one thread.
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(one));
  return one != 0;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

template <int Regs>
__device__ __forceinline__ void regs_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Regs));
}
template <int Regs>
__device__ __forceinline__ void regs_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Regs));
}

__device__ __forceinline__ uint4 ld_shared_v4(uint32_t addr) {
  uint4 x;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "r"(addr));
  return x;
}

// Eight 8-bit codes -> eight fp16 values (exact).
template <KvType kKv>
__device__ __forceinline__ uint4 widen8(uint2 raw) {
  using W = Widen<__half, kKv == kKvI8 ? FAT_DTYPE_I8 : FAT_DTYPE_E4M3>;
  uint4 o;
  W::run(raw.x, o.x, o.y);
  W::run(raw.y, o.z, o.w);
  return o;
}

// T: the MMA operands' type (the cache's for 16-bit caches, fp16 for 8-bit ones).
// CTA `cta` is member cta % per_gang of gang cta / per_gang of `gangs`.
template <typename T, int D, Mode kMode, KvType kKv>
__device__ __forceinline__ void prefix_body(const CUtensorMap& tm_q, const CUtensorMap& tm_k,
                                            const CUtensorMap& tm_v, const Params& p, const int cta,
                                            const int gangs) {
  constexpr bool k8 = kKv != kKv16;
  using L = Layout<D, kMode, k8>;
  constexpr int BN = L::BN, SK = L::kStagesK, SV = L::kStagesV, SR = L::kStagesRaw;
  constexpr int NS = L::kStreams;
  constexpr int fmt = std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
  constexpr uint32_t kIdescQK = tc::idesc_f16(BM, kUnit, fmt, 0, 0);
  constexpr uint32_t kIdescPV = tc::idesc_f16(BM, D, fmt, 0, 1);
  constexpr int kGroups8 = BN / 8;  // 8-token groups of a tile (a page holds whole ones)
  // Query rows that change on the way: bf16 ones of an 8-bit cache, a negative softmax scale.
  const bool touch_q = (k8 && p.q_bf16) || p.q_negate;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sQ = smem_u32(smem);
  const uint32_t sK = sQ + L::kRowTiles * L::kQTile;
  const uint32_t sV = sK + SK * L::kTile;
  const uint32_t sR = sV + SV * L::kTile;
  float* scales = reinterpret_cast<float*>(smem + L::kData);  // [slot][kScaleRow]
  uint64_t* bars = reinterpret_cast<uint64_t*>(scales + L::kScaleFloats);
  const uint32_t bar0 = smem_u32(bars);
  const uint32_t q_full = bar0;               // the piece's Q rows are in shared memory
  const uint32_t q_raw = q_full + 8;          // the same, where they are changed in place first
  const uint32_t q_seen = q_raw + 8;          // both streams' threads have read their raw row
  const uint32_t q_empty = q_seen + 8;        // the piece's last Q.K^T completed
  const uint32_t k_full = q_empty + 8;        // [SK]
  const uint32_t k_empty = k_full + 8 * SK;   // [SK]
  const uint32_t v_full = k_empty + 8 * SK;   // [SV]
  const uint32_t v_empty = v_full + 8 * SV;   // [SV]
  const uint32_t s_full = v_empty + 8 * SV;   // [NS][2]: the scores of a unit are complete
  const uint32_t p_full = s_full + 16 * NS;   // [NS][2]: its P is written, O_t rescaled
  const uint32_t o_full = p_full + 16 * NS;   // [NS][2]: its P.V is complete
  const uint32_t drain = o_full + 16 * NS;
  const uint32_t vtail = drain + 8;           // 16-bit: a partly valid V tile landed
  const uint32_t never = vtail + 8;           // nothing arrives on it (failure-path tests)
  const uint32_t r_full = never + 8;          // [SR]: raw tiles
  const uint32_t r_empty = r_full + 8 * SR;   // [SR]
  const uint32_t sc_full = r_empty + 8 * SR;  // [scale slots]: a tile's scales are in shared memory
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(bars + L::kBars);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* sh = reinterpret_cast<volatile int*>(tmem_slot + 2);  // [8] where the CTA's range starts
  volatile int* held = sh + 8;                                        // [softmax warp][8], see below

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int gang = cta / p.per_gang, member = cta - gang * p.per_gang;

  if (warp == L::kMmaWarp) {
    tc::tmem_alloc(smem_u32(const_cast<uint32_t*>(tmem_slot)), kTmemCols);
    tc::tmem_relinquish();
  }
  if (tid == 32) {
    mbar_init(q_full, touch_q ? L::kSoftmaxThreads : 1);
    mbar_init(q_raw, 1);
    mbar_init(q_seen, L::kSoftmaxThreads);
    mbar_init(q_empty, 1);
    for (int s = 0; s < SK; ++s) {
      mbar_init(k_full + 8 * s, k8 ? 128 : 1);
      mbar_init(k_empty + 8 * s, 1);
    }
    for (int s = 0; s < SV; ++s) {
      mbar_init(v_full + 8 * s, k8 ? 128 : 1);
      mbar_init(v_empty + 8 * s, 1);
    }
    for (int t = 0; t < NS; ++t) {
      for (int b = 0; b < 2; ++b) {
        mbar_init(s_full + 16 * t + 8 * b, 1);
        mbar_init(p_full + 16 * t + 8 * b, 128);
        mbar_init(o_full + 16 * t + 8 * b, 1);
      }
    }
    mbar_init(drain, 1);
    mbar_init(vtail, 1);
    mbar_init(never, 1);
    for (int s = 0; s < SR; ++s) {
      mbar_init(r_full + 8 * s, 1);
      mbar_init(r_empty + 8 * s, 128);
    }
    if (k8)
      for (int s = 0; s < L::kScaleSlots; ++s) mbar_init(sc_full + 8 * s, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  // Where this gang's range starts on the line (warp 0): the tiles in all, then the
  // group that holds the range's first tile (up to 32 groups stay in registers).
  if (warp == 0) {
    Walk mine{};
    mine.g = lane;
    if (lane < p.groups.count) mine.load(p, BN);
    long long total = mine.n;
    for (int g = lane + 32; g < p.groups.count; g += 32) total += Line{p.groups, BN, p.num_kv_heads}.tiles(g);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    total *= p.num_kv_heads;
    if (total > kMaxTiles) {
      if (lane == 0) raise_error(p.err, FAT_DEVERR_BAD_LENGTH);
      total = 0;
    }
    const int x0 = int(cut(gang, total, gangs)), x1 = int(cut(gang + 1, total, gangs));
    if (lane == 0) {
      sh[0] = x0;
      sh[1] = x0;  // no tile: an empty range
    }
    __syncwarp();
    int base = 0;
    for (int g0 = 0; g0 < p.groups.count && x0 < x1; g0 += 32) {
      if (g0 > 0) {
        mine = Walk{};
        mine.g = g0 + lane;
        if (mine.g < p.groups.count) mine.load(p, BN);
      }
      const int n = mine.n * p.num_kv_heads;
      int incl = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += y;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, base + incl > x0);
      if (hit != 0u) {
        if (lane == __ffs(hit) - 1) {
          sh[1] = x1;
          sh[2] = base + incl - n;
          sh[3] = mine.g;
          sh[4] = mine.n;
          sh[5] = mine.first;
          sh[6] = mine.size;
          sh[7] = mine.tokens;
        }
        break;
      }
      base += __shfl_sync(0xffffffffu, incl, 31);
    }
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  Walk walk;
  walk.x0 = walk.x = sh[0];
  walk.x1 = sh[1];
  walk.base = sh[2];
  walk.g = sh[3];
  walk.n = sh[4];
  walk.first = sh[5];
  walk.size = sh[6];
  walk.tokens = sh[7];
  auto wait = [&](uint32_t bar, uint32_t parity) { return mbar_wait_bounded(bar, parity, p.err, abort_flag, p.wait_ns); };

  if (warp >= L::kProducerWarp) {
    if constexpr (L::kSplitRegs) regs_dec<L::kRegsOther>();
    if (warp == L::kProducerWarp || (!k8 && warp == L::kVProducerWarp)) {
      // ============================ TMA producers ============================
      // 16-bit: one warp for K and one for V, so that neither ring waits for the
      // other's stages.  8-bit: one warp for the raw ring (K, V alternate) and the
      // scales.  Lane l brings rows [i_page * box_rows, + box_rows) of a tile (16-bit:
      // of column block cb) from their page; page ids are read two tiles ahead.
      constexpr int kCols = k8 ? 1 : L::kCB;
      const bool is_v = warp == L::kVProducerWarp;
      const CUtensorMap* tm = is_v ? &tm_v : &tm_k;
      const int i_page = lane / kCols, cb = lane - i_page * kCols;
      const int pages_per_tile = BN / p.box_rows;
      const int row0 = i_page * p.box_rows;
      const uint32_t box_bytes = uint32_t(p.box_rows) * (k8 ? uint32_t(p.head_dim) : 128u);
      int issued = 0;  // tiles
      int tails = 0;
      bool ok = true;
      Piece w;
      while (ok && walk.next<L::kRowTiles>(p, BN, member, w)) {
        const int* table = p.page_table + (long long)w.first * p.pt_sb;
        const int first_len = __ldg(p.seq_lens + w.first);
        auto page_of = [&](int j, int& slot0) -> int {
          slot0 = -1;
          const int tok = j * BN + row0;
          if (i_page >= pages_per_tile || j >= w.t1 || tok >= w.tokens) return 0;  // no rows there
          const int lp = tok / p.page_size;
          slot0 = tok - lp * p.page_size;
          return __ldg(table + lp);  // checked a tile later: a use here would wait for the load
        };
        auto checked = [&](int page, int slot0) -> int {
          return slot0 < 0 ? -2 : (page >= 0 && page < p.num_pages ? page : -1);
        };
        auto scales_of = [&](int page, float& ks, float& vs) {
          ks = vs = 0.f;
          if (k8 && page >= 0) {
            ks = __ldg(p.k_scale + (long long)page * p.s_sp + w.kvh);
            vs = __ldg(p.v_scale + (long long)page * p.s_sp + w.kvh);
          }
        };
        int slot1, slot2;
        int page1 = page_of(w.t0, slot1), page2 = page_of(w.t0 + 1, slot2);
        if (first_len < w.tokens) {
          // The first sequence does not hold the prefix (any more: it may have been
          // released); the table is that of the first one that does.
          for (int i0 = 0; i0 < walk.size; i0 += 32) {
            const int b = w.first + i0 + lane;
            const unsigned holds =
                __ballot_sync(0xffffffffu, i0 + lane < walk.size && __ldg(p.seq_lens + b) >= w.tokens);
            if (holds != 0u) {
              table = p.page_table + (long long)(w.first + i0 + __ffs(holds) - 1) * p.pt_sb;
              break;
            }
          }
          page1 = page_of(w.t0, slot1);
          page2 = page_of(w.t0 + 1, slot2);
        }
        page1 = checked(page1, slot1);
        float ks1, vs1;
        scales_of(page1, ks1, vs1);
        [[maybe_unused]] float unit = 0.f;  // 8-bit: what O is in units of (the piece's V scales so far)
        for (int j = w.t0; j < w.t1; ++j) {
          const int page = page1, slot0 = slot1;
          [[maybe_unused]] const float ks = ks1, vs = vs1;
          page1 = checked(page2, slot2);
          slot1 = slot2;
          page2 = page_of(j + 2, slot2);
          scales_of(page1, ks1, vs1);
          if (page == -1) raise_error(p.err, FAT_DEVERR_BAD_PAGE);
          const unsigned loaded = __ballot_sync(0xffffffffu, page >= 0);
          const uint32_t bytes = uint32_t(__popc(loaded)) * box_bytes;
          if constexpr (!k8) {
            const int depth = is_v ? SV : SK;
            const int st = issued % depth;
            const uint32_t full = (is_v ? v_full : k_full) + 8 * st;
            const uint32_t tile = (is_v ? sV : sK) + st * L::kTile;
            // Rows no copy fills are zeroed in V: p = 0 there adds exactly nothing.
            const bool tail = is_v && __popc(loaded) * p.box_rows < BN * kCols;
            if (lane == 0) ok = wait((is_v ? v_empty : k_empty) + 8 * st, ((issued / depth) & 1) ^ 1);
            ok = __shfl_sync(0xffffffffu, ok, 0);
            if (!ok) break;
            const uint32_t bar = tail ? vtail : full;
            if (lane == 0) mbar_arrive_expect_tx(bar, bytes);
            __syncwarp();
            if (page >= 0)
              tma_load_4d(tile + cb * BN * 128 + row0 * 128, tm, bar, cb * 64, w.kvh, slot0, page);
            ++issued;
            if (tail) {
              ++tails;
              if (lane == 0) ok = wait(vtail, (tails - 1) & 1);
              ok = __shfl_sync(0xffffffffu, ok, 0);
              if (!ok) break;
              const int valid_rows = min(BN, w.tokens - j * BN);
              for (int i = lane; i < L::kCB * BN * 8; i += 32) {
                const int c2 = i / (BN * 8), r = (i / 8) % BN;
                const bool filled = ((loaded >> ((r / p.box_rows) * L::kCB)) & 1u) != 0;
                if (!filled || r >= valid_rows)
                  st_shared_v4(tile + uint32_t(c2 * BN * 128 + r * 128 + (i % 8) * 16), 0u, 0u, 0u, 0u);
              }
              fence_proxy_async_smem();
              __syncwarp();
              if (lane == 0) mbar_arrive(full);
            }
          } else {
            // Raw K, then raw V; beside them, per 8 tokens: the K scale, and for the V
            // scale f in units of `unit`, a power of two above every f of the piece so far,
            // log2(f / unit) (P f / unit = 2^(x + log2(f / unit)): no product per element)
            // and unit / f (which takes f out of the sum of P again); then the unit.
            // Where no page is, or where a scale is 0, the tile's codes count as zeros; P of
            // a zero V scale is in the unit itself, so that it is as finite as the others'.
            const int slot = issued % L::kScaleSlots;
            const int per8 = p.box_rows / 8;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
              const int c = 2 * issued + t, sr = c % SR;
              if (lane == 0) ok = wait(r_empty + 8 * sr, ((c / SR) & 1) ^ 1);
              ok = __shfl_sync(0xffffffffu, ok, 0);
              if (!ok) break;
              if (t == 0) {
                // The slot's previous tile left the softmax before its raw stage came free.
                const float kg = __shfl_sync(0xffffffffu, ks, (lane / per8) & 31);
                const float vg = __shfl_sync(0xffffffffu, vs, (lane / per8) & 31);
                const float f = fabsf(vg);
                float vm = lane < kGroups8 && f >= kLeastScale && f < CUDART_INF_F ? f : 0.f;
#pragma unroll
                for (int o = 8; o > 0; o >>= 1) vm = fmaxf(vm, __shfl_xor_sync(0xffffffffu, vm, o));
                vm = __shfl_sync(0xffffffffu, vm, 0);
                if (vm > unit) unit = __int_as_float(min(254, ((__float_as_int(vm) >> 23) & 0xFF) + 1) << 23);
                float* sc = scales + slot * L::kScaleRow;
                const bool none = f < fmaxf(kLeastScale, unit * kLeastRatio);
                const unsigned in = (1u << kGroups8) - 1u;
                const unsigned kmask = (__ballot_sync(0xffffffffu, kg == 0.f) & in) |
                                       ((__ballot_sync(0xffffffffu, kg < 0.f) & in) << 16);
                const unsigned vmask = (__ballot_sync(0xffffffffu, none) & in) |
                                       ((__ballot_sync(0xffffffffu, vg < 0.f) & in) << 16);
                if (lane < kGroups8) {
                  sc[lane] = fabsf(kg);
                  sc[kGroups8 + lane] = none ? 0.f : log2f(f) - float((__float_as_int(unit) >> 23) - 127);
                  sc[2 * kGroups8 + lane] = none ? 1.f : unit / f;
                }
                if (lane == 0) {
                  sc[3 * kGroups8] = unit;
                  sc[3 * kGroups8 + 1] = __uint_as_float(kmask);
                  sc[3 * kGroups8 + 2] = __uint_as_float(vmask);
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(sc_full + 8 * slot);
              }
              if (lane == 0) mbar_arrive_expect_tx(r_full + 8 * sr, bytes);
              __syncwarp();
              if (page >= 0)
                tma_load_4d(sR + sr * L::kRaw + row0 * p.head_dim, t ? &tm_v : &tm_k, r_full + 8 * sr, 0, w.kvh, slot0,
                            page);
            }
            if (!ok) break;
            ++issued;
          }
        }
      }
      if (*abort_flag && lane == 0) {
        // Drain this warp's own copies before the shared memory goes away.
        if constexpr (!k8) {
          const int depth = is_v ? SV : SK;
          for (int j = max(0, issued - depth); j < issued; ++j)
            mbar_wait_bounded((is_v ? v_full : k_full) + 8 * (j % depth), (j / depth) & 1, nullptr, nullptr, p.wait_ns);
          if (tails > 0) mbar_wait_bounded(vtail, (tails - 1) & 1, nullptr, nullptr, p.wait_ns);
        } else {
          for (int c = max(0, 2 * issued + 1 - SR); c <= 2 * issued; ++c)
            mbar_wait_bounded(r_full + 8 * (c % SR), (c / SR) & 1, nullptr, nullptr, p.wait_ns);
        }
      }
    } else if (warp == L::kQWarp && lane == 0) {
      // ============================ queries ============================
      // The next piece's rows come as soon as the last Q.K^T of the piece before has
      // read its own, beside that piece's last softmax and its partial.  A box is the
      // group's heads of one KV head of as many sequences as a row tile holds; rows
      // past the piece's are other sequences' (or zeros) and go nowhere.
      int items = 0;
      Piece w;
      const uint32_t bar = touch_q ? q_raw : q_full;
      while (walk.next<L::kRowTiles>(p, BN, member, w)) {
        if (items > 0 && !wait(q_empty, (items - 1) & 1)) break;
        ++items;
        const int tiles = w.rows > p.tile_rows ? 2 : 1;
        mbar_arrive_expect_tx(bar, uint32_t(tiles * p.tile_rows) * 128u * L::kCB);
        for (int t = 0; t < tiles; ++t)
#pragma unroll
          for (int c = 0; c < L::kCB; ++c)
            tma_load_3d(sQ + t * L::kQTile + c * BM * 128, &tm_q, bar, c * 64, w.kvh * p.group,
                        w.first + (w.row0 + t * p.tile_rows) / p.group);
      }
      if (*abort_flag && items > 0) mbar_wait_bounded(bar, (items - 1) & 1, nullptr, nullptr, p.wait_ns);
    } else if (warp == L::kMmaWarp && elect_one()) {
      // ============================ MMA issuer ============================
      // Descriptor words are built once; operands move by adding (byte offset
      // >> 4) to the start-address field of the low word.
      const uint64_t dK = tc::sdesc_sw128(sK, 16, 1024);  // Q uses the same layout words
      const uint64_t dV = tc::sdesc_sw128(sV, L::kStage * 128, 1024);
      const uint32_t hiK = uint32_t(dK >> 32), loK0 = uint32_t(dK);
      const uint32_t hiV = uint32_t(dV >> 32), loV0 = uint32_t(dV);
      const uint32_t loQ0 = uint32_t(tc::sdesc_sw128(sQ, 16, 1024));
      constexpr uint32_t kTileDesc = uint32_t(L::kTile) >> 4;
      auto desc = [](uint32_t lo, uint32_t hi) { return (uint64_t(hi) << 32) | lo; };
      // The scores of half `h` of a K tile into buffer b of stream t; the P there with
      // half h of a V tile.
      auto issue_s = [&](int t, int b, uint32_t loK, int h) {
        const uint32_t loQ = loQ0 + (kMode == kRowPair ? uint32_t(t) * (uint32_t(L::kQTile) >> 4) : 0u);
        loK += uint32_t(h) * (uint32_t(kUnit * 128) >> 4);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint32_t offq = uint32_t(((kk >> 2) * (BM * 128) + (kk & 3) * 32) >> 4);
          const uint32_t offk = uint32_t(((kk >> 2) * (L::kStage * 128) + (kk & 3) * 32) >> 4);
          tc::mma_ss(tmem + 128 * t + kUnit * b, desc(loQ + offq, hiK), desc(loK + offk, hiK), kIdescQK,
                     kk > 0 ? 1u : 0u);
        }
      };
      auto issue_pv = [&](int t, int b, uint32_t loV, int h, bool acc) {
        loV += uint32_t(h) * (uint32_t(kUnit * 128) >> 4);
#pragma unroll
        for (int kk = 0; kk < 2 * kUnit / 16; ++kk) {
          const int tok = kk % (kUnit / 16) * 16;  // the remainders of P follow the cut values
          tc::mma_ts(tmem + kColO + 128 * t, tmem + 128 * t + kUnit * b + kk * 8,
                     desc(loV + uint32_t((tok * 128) >> 4), hiV), kIdescPV, (acc || kk > 0) ? 1u : 0u);
        }
      };
      int sk = 0, kph = 0, sv = 0, vph = 0, items = 0;
      int units[2] = {0, 0};  // of earlier pieces, by stream
      auto next_k = [&]() {
        tc::commit(k_empty + 8 * sk);
        if (++sk == SK) {
          sk = 0;
          kph ^= 1;
        }
      };
      auto next_v = [&]() {
        tc::commit(v_empty + 8 * sv);
        if (++sv == SV) {
          sv = 0;
          vph ^= 1;
        }
      };
      if (p.expire) wait(never, 0);
      bool ok = true;
      Piece w;
      while (ok && walk.next<L::kRowTiles>(p, BN, member, w)) {
        const int n = w.t1 - w.t0;
        if (!wait(q_full, items & 1)) break;
        ++items;
        tc::fence_after_sync();
        // Unit u of a stream: O += P(u) V(u), then the scores of unit u + 2 into the
        // buffer that P(u) leaves; the scores of unit u + 1 are there meanwhile.
        const int streams = kMode == kRowPair && w.rows <= p.tile_rows ? 1 : NS;
        const int U = n * L::kUnits;
        // A stage holds: 16-bit, the tile; 8-bit, a unit (of one stream where they alternate).
        constexpr int kStageUnits = L::kUnits / L::kHalves > 0 ? L::kUnits / L::kHalves : 1;
        constexpr bool kStreamStage = kMode == kAlternate && k8;
        auto half_of = [&](int t, int i) { return k8 ? 0 : (kMode == kAlternate ? t : i % L::kUnits); };
        for (int u = -2; ok && u < U; ++u) {
          const int s = u + 2;
#pragma unroll
          for (int t = 0; t < NS; ++t) {
            if (!ok || t >= streams) continue;
            const int x = units[t] + s, b = x & 1;
            const bool first = t == 0 || kStreamStage, last = t == streams - 1 || kStreamStage;
            if (u >= 0) {
              if ((first && u % kStageUnits == 0 && !wait(v_full + 8 * sv, vph)) ||
                  !wait(p_full + 16 * t + 8 * b, ((x >> 1) & 1) ^ 1)) {
                ok = false;
                continue;
              }
              tc::fence_after_sync();
              issue_pv(t, b, loV0 + uint32_t(sv) * kTileDesc, half_of(t, u), u > 0);
              tc::commit(o_full + 16 * t + 8 * b);
              if (last && u % kStageUnits == kStageUnits - 1) next_v();
            }
            if (s < U) {
              if (first && s % kStageUnits == 0 && !wait(k_full + 8 * sk, kph)) {
                ok = false;
                continue;
              }
              tc::fence_after_sync();
              issue_s(t, b, loK0 + uint32_t(sk) * kTileDesc, half_of(t, s));
              tc::commit(s_full + 16 * t + 8 * b);
              if (last && s % kStageUnits == kStageUnits - 1) next_k();
            }
          }
          if (ok && s == U - 1) tc::commit(q_empty);
        }
        for (int t = 0; t < streams; ++t) units[t] += U;
      }
      // Every MMA this thread issued has finished once `drain` completes.
      tc::commit(drain);
      mbar_wait_bounded(drain, 0, nullptr, nullptr, p.wait_ns);
    } else if constexpr (k8) {
      if (warp >= L::kConvWarp) {
        // ============================ converters ============================
        // Thread i takes 16 codes at a time, piece ch of every kStep-th row: two 16-byte
        // chunks, of which half of the threads write the odd one first, so that a quarter
        // warp writes eight different chunks of the swizzle (no bank conflicts).  A
        // stage's loads come before its stores.  Groups of scale 0 (or without a page) are
        // written as zeros; a scale's sign moves into the codes.
        const int ct = (tid - L::kConvWarp * 32) & 127;
        constexpr bool kBoth = L::kConvWarps == 4;
        const int first = kBoth ? 0 : (warp - L::kConvWarp) / 4;  // 0: K, 1: V
        constexpr int kLanes = D / 16;             // threads of a row
        constexpr int kStep = 128 / kLanes;        // rows between a thread's items
        constexpr int kItems = L::kStage / kStep;
        const int row0 = ct / kLanes, ch = ct % kLanes;
        const int hd = D == 64 ? p.head_dim : D;   // 32 goes as 64, the rest zeros
        const bool data = D > 64 || ch * 16 < hd;
        const uint32_t odd = (ch >> 2) & 1;        // the first chunk written
        int sk = 0, kph = 1, sv = 0, vph = 1, tile = 0;
        bool ok = true;
        Piece w;
        while (ok && walk.next<L::kRowTiles>(p, BN, member, w)) {
          for (int j = w.t0; ok && j < w.t1; ++j, ++tile) {
#pragma unroll 1
            for (int i = 0; i < (kBoth ? 2 : 1) * L::kHalves; ++i) {
              // Both: K's halves, then V's.
              const int t = kBoth ? i / L::kHalves : first, half = i % L::kHalves;
              const int c = 2 * tile + t, sr = c % SR;
              if ((half == 0 && !wait(r_full + 8 * sr, (c / SR) & 1)) ||
                  !wait(t ? v_empty + 8 * sv : k_empty + 8 * sk, t ? vph : kph)) {
                ok = false;
                break;
              }
              const uint32_t dst = t ? sV + sv * L::kTile : sK + sk * L::kTile;
              const uint32_t src = sR + sr * L::kRaw + uint32_t((half * L::kStage + row0) * hd + ch * 16);
              // Which 8-token groups count as zeros, and which change sign.
              const unsigned mask =
                  __float_as_uint(scales[(tile % L::kScaleSlots) * L::kScaleRow + 3 * kGroups8 + 1 + t]);
              uint4 raw[kItems];
#pragma unroll
              for (int u = 0; u < kItems; ++u) {
                raw[u] = make_uint4(0u, 0u, 0u, 0u);
                if (data) raw[u] = ld_shared_v4(src + uint32_t(u * kStep * hd));
              }
              const uint32_t block = dst + uint32_t((ch >> 2) * L::kStage * 128);
              auto put = [&](int r, const uint4& x, uint32_t keep, uint32_t flip) {
                uint4 lo = widen8<kKv>(make_uint2(x.x, x.y)), hi = widen8<kKv>(make_uint2(x.z, x.w));
                if (keep != 0xffffffffu || flip != 0u) {
                  lo = make_uint4((lo.x ^ flip) & keep, (lo.y ^ flip) & keep, (lo.z ^ flip) & keep, (lo.w ^ flip) & keep);
                  hi = make_uint4((hi.x ^ flip) & keep, (hi.y ^ flip) & keep, (hi.z ^ flip) & keep, (hi.w ^ flip) & keep);
                }
                const uint32_t c0 = 2u * (ch & 3) + odd, c1 = c0 ^ 1u;
                const uint4 a = odd ? hi : lo, b = odd ? lo : hi;
                st_shared_v4(block + swz128(uint32_t(r), c0), a.x, a.y, a.z, a.w);
                st_shared_v4(block + swz128(uint32_t(r), c1), b.x, b.y, b.z, b.w);
              };
              if (mask == 0u && data) {
#pragma unroll
                for (int u = 0; u < kItems; ++u) put(row0 + u * kStep, raw[u], 0xffffffffu, 0u);
              } else {
                const unsigned zero = (mask & 0xffffu) >> (half * (L::kStage / 8));
                const unsigned neg = mask >> (16 + half * (L::kStage / 8));
#pragma unroll
                for (int u = 0; u < kItems; ++u) {
                  const int r = row0 + u * kStep;
                  put(r, raw[u], (((zero >> (r >> 3)) & 1u) == 0u && data) ? 0xffffffffu : 0u,
                      ((neg >> (r >> 3)) & 1u) ? 0x80008000u : 0u);
                }
              }
              fence_proxy_async_smem();
              mbar_arrive(t ? v_full + 8 * sv : k_full + 8 * sk);
              if (half == L::kHalves - 1) mbar_arrive(r_empty + 8 * sr);
              if (t == 0) {
                if (++sk == SK) {
                  sk = 0;
                  kph ^= 1;
                }
              } else if (++sv == SV) {
                sv = 0;
                vph ^= 1;
              }
            }
          }
        }
      }
    }
  } else {
    if constexpr (L::kSplitRegs) regs_inc<L::kRegsSoftmax>();
    // ============================ softmax warpgroups ============================
    const int t = warp >> 2;    // stream
    const int row = tid & 127;  // row of the stream's tile = tensor-memory lane
    const uint32_t lane_base = tmem + (uint32_t((warp & 3) * 32) << 16);
    const uint32_t colO = kColO + 128 * t;
    const uint32_t sbar = s_full + 16 * t, pbar = p_full + 16 * t, obar = o_full + 16 * t;
    int items = 0, tile = 0;
    int x = 0;  // units of this stream
    bool ok = true;
    auto pv_done = [&]() { return wait(obar + 8 * ((x - 1) & 1), ((x - 1) >> 1) & 1); };  // of unit x - 1
    Piece w;
    while (ok && walk.next<L::kRowTiles>(p, BN, member, w)) {
      const int n = w.t1 - w.t0;
      ++items;
      float qmul = 1.f;
      if (touch_q) {
        // This row, in place.  bf16 queries of an 8-bit cache go to fp16 times the power
        // of two that puts the row's largest magnitude in [2^14, 2^15): exact, and so is
        // the conversion down to 2^-28 of that magnitude; the power returns in the score
        // multiplier.  Alternating streams see the same row: each takes half of it.
        if (!wait(q_raw, (items - 1) & 1)) break;
        const uint32_t qt = sQ + (kMode == kRowPair ? t * L::kQTile : 0);
        const uint32_t flip = p.q_negate ? 0x80008000u : 0u;
        auto chunk = [&](int c) { return qt + uint32_t((c >> 3) * BM * 128) + swz128(uint32_t(row), uint32_t(c & 7)); };
        // A row's chunks are read once and stay in registers.
        constexpr int kOwn = kMode == kAlternate ? D / 16 : (D <= 128 ? D / 8 : D / 16);  // chunks at a time
        const int c0 = kMode == kAlternate ? t * kOwn : 0;
        uint4 own[kOwn];
#pragma unroll
        for (int c = 0; c < kOwn; ++c) own[c] = ld_shared_v4(chunk(c0 + c));
        float down = 1.f;
        if (k8 && p.q_bf16) {
          // The largest magnitude's bits: as integers, the order of bf16 magnitudes (NaN last).
          uint32_t mx2 = 0u;
          auto take = [&](const uint4& x) {
            mx2 = __vmaxu2(__vmaxu2(mx2, x.x & 0x7fff7fffu), x.y & 0x7fff7fffu);
            mx2 = __vmaxu2(__vmaxu2(mx2, x.z & 0x7fff7fffu), x.w & 0x7fff7fffu);
          };
#pragma unroll
          for (int c = 0; c < kOwn; ++c) take(own[c]);
          if (kOwn < D / 8) {
#pragma unroll
            for (int c = 0; c < D / 8 - kOwn; ++c) take(ld_shared_v4(chunk((c0 + kOwn + c) % (D / 8))));
          }
          const int mx = int(max(mx2 & 0xffffu, mx2 >> 16));
          int e = 0;
          if (mx > 0 && mx < 0x7f80) e = max(-126, min(126, (mx >> 7) - 127 - 14));
          down = __int_as_float((127 - e) << 23);
          qmul = __int_as_float((127 + e) << 23);
        }
        if (kMode == kAlternate) {
          mbar_arrive(q_seen);
          if (!wait(q_seen, (items - 1) & 1)) break;
        }
        auto put = [&](int c, uint4 x) {
          if (k8 && p.q_bf16) {
            auto half2_of = [&](uint32_t v) {
              return pack2<__half>(__uint_as_float(v << 16) * down, __uint_as_float(v & 0xffff0000u) * down);
            };
            x = make_uint4(half2_of(x.x), half2_of(x.y), half2_of(x.z), half2_of(x.w));
          }
          st_shared_v4(chunk(c), x.x ^ flip, x.y ^ flip, x.z ^ flip, x.w ^ flip);
        };
#pragma unroll
        for (int c = 0; c < kOwn; ++c) put(c0 + c, own[c]);
        if (kMode != kAlternate && kOwn < D / 8) {
#pragma unroll 4
          for (int c = kOwn; c < D / 8; ++c) put(c, ld_shared_v4(chunk(c)));
        }
        fence_proxy_async_smem();
        mbar_arrive(q_full);
      }
      // What the partial's place depends on waits in shared memory, not in
      // registers: the row of scores needs them.
      volatile int* note = held + warp * 8;
      if (lane == 0) {
        note[0] = w.first;
        note[1] = w.kvh;
        note[2] = w.row0;
        note[3] = w.rows;
        note[4] = w.t0 == 0 && w.t1 == w.n;
        note[5] = w.leading;
      }
      __syncwarp();
      const bool active = kMode != kRowPair || t * p.tile_rows < w.rows;
      const int left = w.tokens - w.t0 * BN;  // shared tokens from the piece's first tile on
      float m_used = -CUDART_INF_F, l_sum = 0.f;
      float vref = 0.f;  // 8-bit: O is in units of this power of two (0: of any, it is all zeros)
      const int U = active ? n * L::kUnits : 0;
      for (int u = 0; u < U; ++u, ++x) {
        const int b = x & 1;
        const int j = u / L::kUnits, half = kMode == kAlternate ? t : u % L::kUnits;
        const uint32_t colS = 128 * t + kUnit * b;
        if (!wait(sbar + 8 * b, (x >> 1) & 1)) {
          ok = false;
          break;
        }
        const int lim = left - j * BN - half * kUnit;  // valid tokens of the unit
        // The running maximum moves only by more than 2^8 at a time;
        // O_t is rescaled in place, once it holds the P.V of the unit before.
        float factor = 1.f;
        bool grow = false;
        auto raise_max = [&](float mx) {
          if (mx > m_used + kRescaleLog2) {
            factor = (m_used == -CUDART_INF_F) ? 1.f : fast_exp2(m_used - mx);
            grow = m_used != -CUDART_INF_F;
            m_used = mx;
            l_sum *= factor;
          }
        };
        auto rescale = [&]() -> bool {
          if (__any_sync(0xffffffffu, grow)) {
            if (!pv_done()) return false;
            tc::fence_after_sync();
#pragma unroll
            for (int c = 0; c < D / 32; ++c) {
              uint32_t r[32];
              tc::ld32(lane_base + colO + 32 * c, r);
              tc::wait_ld();
#pragma unroll
              for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * factor);
              tc::st32(lane_base + colO + 32 * c, r);
            }
          }
          return true;
        };
        float sum0 = 0.f, sum1 = 0.f, sum2 = 0.f, sum3 = 0.f;
        if constexpr (!k8) {
          tc::fence_after_sync();
          float s[kUnit];
          {
            uint32_t r[2][32];
            tc::ld32(lane_base + colS, r[0]);
            tc::ld32(lane_base + colS + 32, r[1]);
            tc::wait_ld();
#pragma unroll
            for (int i = 0; i < kUnit; ++i) s[i] = __uint_as_float(r[i / 32][i % 32]);
          }
          float mul = p.scale_log2;
          if (lim < kUnit) {
            // Masked after the product: the scale may be 0.
            mul = 1.f;
#pragma unroll
            for (int i = 0; i < kUnit; ++i) s[i] = i < lim ? s[i] * p.scale_log2 : -CUDART_INF_F;
          }
          {
            float a0 = fmaxf(s[0], s[4]), a1 = fmaxf(s[1], s[5]), a2 = fmaxf(s[2], s[6]), a3 = fmaxf(s[3], s[7]);
#pragma unroll
            for (int i = 8; i < kUnit; i += 8) {
              a0 = max3(a0, s[i], s[i + 4]);
              a1 = max3(a1, s[i + 1], s[i + 5]);
              a2 = max3(a2, s[i + 2], s[i + 6]);
              a3 = max3(a3, s[i + 3], s[i + 7]);
            }
            raise_max(fmaxf(max3(a0, a1, a2), a3) * mul);
          }
          if (!(ok = rescale())) break;
          const float msub = (m_used == -CUDART_INF_F) ? 0.f : m_used - kLiftLog2;
          uint32_t packed[32], rest[32];
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            float x0, x1, x2, x3;
            fma2(x0, x1, s[2 * i], s[2 * i + 1], mul, -msub);
            fma2(x2, x3, s[2 * i + 2], s[2 * i + 3], mul, -msub);
            packed[i] = split_p<T>(fast_exp2(x0), fast_exp2(x1), sum0, sum1, rest[i]);
            packed[i + 1] = split_p<T>(fast_exp2(x2), fast_exp2(x3), sum2, sum3, rest[i + 1]);
          }
          tc::st32(lane_base + colS, packed);
          tc::st32(lane_base + colS + 32, rest);
        } else {
          // The K scale of an 8-token group multiplies its scores; its V scale f, in
          // units of vref, multiplies P as 2^(x + log2(f / vref)) and leaves the sum of P
          // by vref / f (both from the producer).
          const int slot = (tile + j) % L::kScaleSlots;
          if (!wait(sc_full + 8 * slot, ((tile + j) / L::kScaleSlots) & 1)) {
            ok = false;
            break;
          }
          tc::fence_after_sync();
          const float4* sc = reinterpret_cast<const float4*>(scales + slot * L::kScaleRow);
          constexpr int kQuads = kGroups8 / 4;
          const float kq = p.scale_log2 * qmul;
          float mx = -CUDART_INF_F;
          uint32_t r[2][32], packed[32], rest[32];
          tc::ld32(lane_base + colS, r[0]);
          tc::ld32(lane_base + colS + 32, r[1]);
          tc::wait_ld();
#pragma unroll
          for (int q4 = 0; q4 < 2; ++q4) {
            const float4 k4 = sc[2 * half + q4];
            const float kg[4] = {k4.x, k4.y, k4.z, k4.w};
#pragma unroll
            for (int g8 = 0; g8 < 4; ++g8) {
              const uint32_t* y = r[q4] + g8 * 8;
              const float m0 = max3(__uint_as_float(y[0]), __uint_as_float(y[1]), __uint_as_float(y[2]));
              const float m1 = max3(__uint_as_float(y[3]), __uint_as_float(y[4]), __uint_as_float(y[5]));
              float m8 = fmaxf(max3(__uint_as_float(y[6]), __uint_as_float(y[7]), m0), m1) * kg[g8];
              if (32 * q4 + 8 * g8 >= lim) m8 = -CUDART_INF_F;
              mx = fmaxf(mx, m8);
            }
          }
          raise_max(mx * kq);
          // O's unit only grows.
          const float unit = scales[slot * L::kScaleRow + 3 * kGroups8];
          if (unit > vref) {
            if (vref > 0.f) {
              factor *= vref / unit;
              grow = true;
            }
            vref = unit;
          }
          if (!(ok = rescale())) break;
          const float msub = (m_used == -CUDART_INF_F) ? 0.f : m_used - kLiftLog2;
#pragma unroll
          for (int q4 = 0; q4 < 2; ++q4) {
            const float4 k4 = sc[2 * half + q4], l4 = sc[kQuads + 2 * half + q4], i4 = sc[2 * kQuads + 2 * half + q4];
            const float kg[4] = {k4.x, k4.y, k4.z, k4.w}, lg[4] = {l4.x, l4.y, l4.z, l4.w};
            const float ig[4] = {i4.x, i4.y, i4.z, i4.w};
#pragma unroll
            for (int g8 = 0; g8 < 4; ++g8) {
              const float kf = kg[g8] * kq;
              float sub = lg[g8] - msub;
              if (32 * q4 + 8 * g8 >= lim) sub = -CUDART_INF_F;  // past the prefix: P = 0
              const uint32_t* y = r[q4] + g8 * 8;
              float e0 = 0.f, e1 = 0.f;
#pragma unroll
              for (int i = 0; i < 8; i += 2) {
                float x0, x1;
                fma2(x0, x1, __uint_as_float(y[i]), __uint_as_float(y[i + 1]), kf, sub);
                const int at = (q4 * 4 + g8) * 4 + i / 2;
                packed[at] = split_p<T>(fast_exp2(x0), fast_exp2(x1), e0, e1, rest[at]);
              }
              sum0 = fmaf(e0, ig[g8], sum0);
              sum1 = fmaf(e1, ig[g8], sum1);
            }
          }
          tc::st32(lane_base + colS, packed);
          tc::st32(lane_base + colS + 32, rest);
        }
        l_sum += (sum0 + sum1) + (sum2 + sum3);
        tc::wait_st();
        tc::fence_before_sync();
        mbar_arrive(pbar + 8 * b);
      }
      tile += n;
      // ---- the partial, once the stream's last P.V completed ----
      if (ok && active) {
        ok = pv_done();
        if (!ok) break;
        tc::fence_after_sync();
      }
      if (!ok) break;
      const int part = kMode == kAlternate ? t : 0;
      const int r_here = kMode == kRowPair ? t * p.tile_rows + row : row;
      const bool store = row < p.tile_rows && r_here < note[3];
      float *o, *ml;
      long long pitch;  // floats between 4-column groups
      if (note[4]) {
        const long long r = (long long)note[0] * p.group + note[2] + r_here;
        const long long u = (long long)part * p.num_kv_heads + note[1];
        o = p.home_o + (u * (p.head_dim / 4) * p.home_rows + r) * 4;
        ml = p.home_ml + (u * p.home_rows + r) * 2;
        pitch = p.home_rows * 4;
      } else {
        const long long u = (long long)cta * 2 + (note[5] ? 0 : 1);
        const int r = NS == 2 ? t * BM + row : row;
        o = p.slot_o + (u * (p.head_dim / 4) * 256 + r) * 4;
        ml = p.slot_ml + (u * 256 + r) * 2;
        pitch = 256 * 4;
      }
      if (store) *reinterpret_cast<float2*>(ml) = make_float2(m_used - kLiftLog2, l_sum);
      if (active) {
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          if (c * 32 >= p.head_dim) break;
          uint32_t r[32];
          tc::ld32(lane_base + colO + 32 * c, r);
          tc::wait_ld();
          if (store) {
            const float f = k8 ? vref : 1.f;
#pragma unroll
            for (int i = 0; i < 8; ++i)
              *reinterpret_cast<float4*>(o + (8 * c + i) * pitch) =
                  make_float4(__uint_as_float(r[4 * i]) * f, __uint_as_float(r[4 * i + 1]) * f,
                              __uint_as_float(r[4 * i + 2]) * f, __uint_as_float(r[4 * i + 3]) * f);
          }
        }
      }
      __syncwarp();  // the note is read: lane 0 may write the next one
    }
  }

  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  if (warp == L::kMmaWarp) tc::tmem_dealloc(tmem, kTmemCols);
  for (int i = tid; i < L::kBars; i += L::kThreads) mbar_inval(bar0 + 8 * i);
}

// Gangs (of per_gang CTAs) that begin with the prefix, in proportion to its share of
// the work a + b.  Whatever the others have left of the own tokens when these are
// done they share, but nobody can help them: so they are rather many.  A line of one
// group is cut at its units where that costs little, since every unit a CTA goes on
// to costs it a query load and a partial more (8 units of 131k tokens: 117 us, 126
// uncut; of 32k, 50 and 58; where it leaves CTAs idle it costs up to 2%).
__device__ __forceinline__ int choose_gangs(long long tiles, int units, int ctas, int per_gang, float a, float b) {
  if (tiles == 0) return 0;
  const int most = int(min(tiles, (long long)max(1, ctas / per_gang)));
  int gangs = min(most, max(1, int(ctas * (a / (a + b)) / per_gang + 0.99f)));
  if (units > 0 && gangs > units) {
    const int whole = gangs / units * units;
    if (whole * 8 >= gangs * 7) gangs = whole;
  }
  return gangs;
}

// TQ: the query type; KVT: the cache type; HD: head_dim.
template <typename TQ, int KVT, int HD>
struct Types {
  static constexpr bool k8 = KVT == FAT_DTYPE_I8 || KVT == FAT_DTYPE_E4M3;
  static constexpr KvType kKv = KVT == FAT_DTYPE_I8 ? kKvI8 : (KVT == FAT_DTYPE_E4M3 ? kKvE4M3 : kKv16);
  static constexpr int D = HD < 64 ? 64 : HD;  // head_dim 32: 64 columns, the copies fill the rest with zeros
  using T = std::conditional_t<k8, __half, TQ>;
};

template <typename TQ, int KVT, int HD, Mode kMode>
__global__ void __launch_bounds__(Layout<Types<TQ, KVT, HD>::D, kMode, Types<TQ, KVT, HD>::k8>::kThreads, 1)
    shared_prefix_kernel(const __grid_constant__ CUtensorMap tp_q, const __grid_constant__ CUtensorMap tp_k,
                         const __grid_constant__ CUtensorMap tp_v,
                         const __grid_constant__ CUtensorMap to_k, const __grid_constant__ CUtensorMap to_v,
                         const __grid_constant__ Params p, const __grid_constant__ own::Params d) {
  using Y = Types<TQ, KVT, HD>;
  using L = Layout<Y::D, kMode, Y::k8>;
  using LO = own::Layout<HD, own::elem_bytes<KVT>()>;
  static_assert(LO::kWarps * 32 <= L::kThreads, "warps for the own tokens");
  // Warps that take no piece give registers back, which 16-bit kernels' have not got.
  static_assert(!L::kSplitRegs || Y::k8 || LO::kWarps * 32 == L::kThreads, "every warp takes pieces");
  static_assert(!L::kSplitRegs || LO::kWarps == 12, "the register split is made for twelve warps");
  extern __shared__ uint8_t smem_raw[];
  grid_allow_dependents();  // the joining kernel may set up beside this one
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (tid == 0) {
    tma_prefetch_desc(&tp_q);
    tma_prefetch_desc(&tp_k);
    tma_prefetch_desc(&tp_v);
    tma_prefetch_desc(&to_k);
    tma_prefetch_desc(&to_v);
  }
  // Every CTA counts the tiles, the groups that have some, and the own tokens.
  long long tiles = 0, tokens = 0;
  int groups = 0;
  for (int g = tid; g < p.groups.count; g += L::kThreads) {
    const int n = Line{p.groups, L::BN, p.num_kv_heads}.tiles(g);
    tiles += n;
    groups += n > 0;
    if (blockIdx.x == 0 && !p.groups.sound(g)) raise_error(p.err, FAT_DEVERR_BAD_GROUP);
  }
  for (int b = tid; b < p.groups.batch; b += L::kThreads) {
    int skip;
    tokens += own::own_tokens(p.groups, d.seq_lens, b, &skip);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    tiles += __shfl_xor_sync(0xffffffffu, tiles, o);
    tokens += __shfl_xor_sync(0xffffffffu, tokens, o);
    groups += __shfl_xor_sync(0xffffffffu, groups, o);
  }
  long long* red = reinterpret_cast<long long*>(smem_raw);
  if (lane == 0) {
    red[3 * warp] = tiles;
    red[3 * warp + 1] = tokens;
    red[3 * warp + 2] = groups;
  }
  __syncthreads();
  tiles = tokens = 0;
  groups = 0;
#pragma unroll
  for (int w = 0; w < L::kThreads / 32; ++w) {
    tiles += red[3 * w];
    tokens += red[3 * w + 1];
    groups += int(red[3 * w + 2]);
  }
  __syncthreads();
  tiles *= p.num_kv_heads;
  if (tiles > kMaxTiles) {
    if (blockIdx.x == 0 && tid == 0) raise_error(p.err, FAT_DEVERR_BAD_LENGTH);
    tiles = 0;
  }
  const int units = p.num_kv_heads * d.head_groups;
  constexpr float kCost = L::kTileCost * (std::is_same<typename Y::T, __nv_bfloat16>::value ? 1.15f : 1.f);
  const float work_p = float(tiles) * p.per_gang * kCost;
  const float work_o = float(tokens) * units * (2.f * LO::kRowBytes / 32768.f);
  const int gangs = choose_gangs(tiles, groups == 1 ? p.num_kv_heads : 0, int(gridDim.x), p.per_gang, work_p, work_o);
  const int piece = own::piece_tokens(tokens, units, d.workers, LO::kTokens);
  if (blockIdx.x == 0 && tid == 0) p.info[0] = gangs;
  if (blockIdx.x == gridDim.x - 1 && warp == L::kThreads / 32 - 1) {
    // The first piece of each sequence, for the joining kernel.
    int before = 0;
    for (int b0 = 0; b0 < p.groups.batch; b0 += 32) {
      int skip, n = 0;
      if (b0 + lane < p.groups.batch)
        n = (own::own_tokens(p.groups, d.seq_lens, b0 + lane, &skip) + piece - 1) / piece * units;
      int incl = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += y;
      }
      if (b0 + lane < p.groups.batch) p.first_piece[b0 + lane] = make_int2(before + incl - n, n / units);
      before += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (lane == 0) d.counter[1] = before + 1;
  }

  const bool prefix = int(blockIdx.x) < gangs * p.per_gang;
  if (prefix) prefix_body<typename Y::T, Y::D, kMode, Y::kKv>(tp_q, tp_k, tp_v, p, int(blockIdx.x), gangs);
  if (tokens == 0) return;
  if (prefix) {
    // Every piece may be taken by now.  Else the shared memory changes hands, to be
    // written by copies again.
    __shared__ int left;
    if (tid == 0) {
      const volatile int* c = d.counter;
      const int total = c[1], taken = c[0];
      left = total == 0 || taken < total - 1;
    }
    fence_proxy_async_smem();
    __syncthreads();
    if (left == 0) return;
  }
  // Registers for the warps that take pieces, from the launch's share or as the
  // prefix body left them.
  if constexpr (L::kSplitRegs) {
    if (warp >= LO::kWarps) {
      regs_dec<L::kRegsIdle>();
      return;
    }
    if (L::kRegsOwn < L::kRegsSoftmax && warp < 8) regs_dec<L::kRegsOwn>();
    else regs_inc<L::kRegsOwn>();
  }
  if (warp < LO::kWarps) own::own_body<TQ, HD, KVT>(to_k, to_v, d, piece);
}

// What a launch is made for (host).
struct Plan {
  Mode mode;
  int tile_rows, cta_rows, bn, per_gang, ctas, parts;
  int head_groups, piece_rows, workers;  // own tokens
};

template <typename TQ, int KVT, int HD, Mode kMode>
int launch_mode(const SharedPrefixArgs& a, const Plan& plan, Params& p, own::Params& o) {
  using Y = Types<TQ, KVT, HD>;
  using L = Layout<Y::D, kMode, Y::k8>;
  using LO = own::Layout<HD, own::elem_bytes<KVT>()>;
  constexpr size_t kSmem = std::max(L::kSmem, LO::kSmem);
  const DecodeArgs& d = a.d;
  auto kern = shared_prefix_kernel<TQ, KVT, HD, kMode>;
  cudaError_t e = ensure_smem_limit(reinterpret_cast<const void*>(kern), int(kSmem), current_device());
  if (e != cudaSuccess) return cuda_failure("cudaFuncSetAttribute(shared prefix)", e);
  if constexpr (L::kSplitRegs) {
    // The register split takes its sum from what the launch allocates.
    static const int regs = [&] {
      cudaFuncAttributes attr;
      return cudaFuncGetAttributes(&attr, reinterpret_cast<const void*>(kern)) == cudaSuccess ? attr.numRegs : 0;
    }();
    if (regs < L::kLaunchRegs) return unsupported("shared_prefix_decode: built with too few registers per thread");
  }
  constexpr uint64_t eb = Y::k8 ? 1 : 2;
  const CUtensorMapDataType dt = Y::k8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_UINT16;
  // A token row narrower than 256 B sits next to another head's row: L2 fills stop at the row.
  const CUtensorMapL2promotion promo =
      LO::kRowBytes >= 256 ? CU_TENSOR_MAP_L2_PROMOTION_L2_256B : CU_TENSOR_MAP_L2_PROMOTION_L2_128B;
  CUtensorMap tq, tk, tv, ok, ov;
  std::string why;
  // Queries: a box is 64 columns of the heads of one KV head of the sequences of a row tile.
  {
    const int group = d.num_heads / d.num_kv_heads;
    const uint64_t dims[3] = {uint64_t(d.head_dim), uint64_t(d.num_heads), uint64_t(d.batch)};
    const uint64_t strides[2] = {uint64_t(d.q_sh) * 2, uint64_t(d.q_sb) * 2};
    const uint32_t box[3] = {64u, uint32_t(group), uint32_t(BM / group)};
    if (!encode_tiled(&tq, CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, d.q, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B,
                      &why))
      return invalid("q: " + why);
  }
  // Prefix: a box is rows of one KV head of one page (16-bit: of one 128-byte column
  // block), as many as divide a page and a tile.
  int box_rows = L::BN;
  while (d.page_size % box_rows) box_rows >>= 1;
  p.box_rows = box_rows;
  {
    const uint64_t dims[4] = {uint64_t(d.head_dim), uint64_t(d.num_kv_heads), uint64_t(d.page_size),
                              uint64_t(d.num_pages)};
    const uint64_t strides[3] = {uint64_t(d.kv_sh) * eb, uint64_t(d.kv_ss) * eb, uint64_t(d.kv_sp) * eb};
    const uint32_t box[4] = {Y::k8 ? uint32_t(d.head_dim) : 64u, 1u, uint32_t(box_rows), 1u};
    const CUtensorMapSwizzle sw = Y::k8 ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B;
    if (!encode_tiled(&tk, dt, 4, d.k_cache, dims, strides, box, sw, &why, promo)) return invalid("k_cache: " + why);
    if (!encode_tiled(&tv, dt, 4, d.v_cache, dims, strides, box, sw, &why, promo)) return invalid("v_cache: " + why);
  }
  // Own tokens: a box is whole token rows, {elements of a column block, column block,
  // KV head, slot, page}, as many as divide a page and a stage.
  box_rows = LO::kTokens;
  while (d.page_size % box_rows) box_rows >>= 1;
  o.box_rows = box_rows;
  {
    const uint64_t dims[5] = {uint64_t(LO::kBoxBytes / eb), uint64_t(LO::kCB), uint64_t(d.num_kv_heads),
                              uint64_t(d.page_size), uint64_t(d.num_pages)};
    const uint64_t strides[4] = {uint64_t(LO::kBoxBytes), uint64_t(d.kv_sh) * eb, uint64_t(d.kv_ss) * eb,
                                 uint64_t(d.kv_sp) * eb};
    const uint32_t box[5] = {uint32_t(LO::kBoxBytes / eb), uint32_t(LO::kCB), 1u, uint32_t(box_rows), 1u};
    const CUtensorMapSwizzle sw = LO::kBoxBytes == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE;
    if (!encode_tiled(&ok, dt, 5, d.k_cache, dims, strides, box, sw, &why, promo)) return invalid("k_cache: " + why);
    if (!encode_tiled(&ov, dt, 5, d.v_cache, dims, strides, box, sw, &why, promo)) return invalid("v_cache: " + why);
  }
  kern<<<plan.ctas, L::kThreads, kSmem, d.stream>>>(tq, tk, tv, ok, ov, p, o);
  e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_failure("shared prefix launch", e);
  return FAT_OK;
}

// Every head_dim and mode of one pair of types.
template <typename TQ, int KVT>
int launch_types(const SharedPrefixArgs& a, const Plan& plan, Params& p, own::Params& o) {
  const bool pair = plan.mode == kRowPair;
  switch (a.d.head_dim) {
    case 32:
      return pair ? launch_mode<TQ, KVT, 32, kRowPair>(a, plan, p, o)
                  : launch_mode<TQ, KVT, 32, kAlternate>(a, plan, p, o);
    case 64:
      return pair ? launch_mode<TQ, KVT, 64, kRowPair>(a, plan, p, o)
                  : launch_mode<TQ, KVT, 64, kAlternate>(a, plan, p, o);
    case 128:
      return pair ? launch_mode<TQ, KVT, 128, kRowPair>(a, plan, p, o)
                  : launch_mode<TQ, KVT, 128, kAlternate>(a, plan, p, o);
    default:
      return launch_mode<TQ, KVT, 256, kSolo>(a, plan, p, o);
  }
}

// One translation unit each.
int launch_f16(const SharedPrefixArgs& a, const Plan& plan, Params& p, own::Params& o);
int launch_bf16(const SharedPrefixArgs& a, const Plan& plan, Params& p, own::Params& o);
int launch_i8(const SharedPrefixArgs& a, const Plan& plan, Params& p, own::Params& o);
int launch_e4m3(const SharedPrefixArgs& a, const Plan& plan, Params& p, own::Params& o);

}  // namespace spx
}  // namespace fat
