// Shared-prefix decode: the kernel that joins the partials, the one that finds a
// shared prefix, and the launches (the kernel over the cache is in
// shared_prefix_kernel.cuh).
#include <algorithm>
#include <mutex>

#include "shared_prefix_kernel.cuh"

namespace fat {
namespace spx {

// ---------------------------------------------------------------------------
// Joining the partials
// ---------------------------------------------------------------------------
struct JoinParams {
  Groups groups;
  const int* seq_lens;
  int bn, num_kv_heads, group, head_dim;
  int per_gang, tile_rows, cta_rows, parts;  // parts: 2 where streams alternate over the tiles of one row tile
  const int* info;       // [0] the number of gangs
  const float* slot_o;
  const float* slot_ml;
  const float* home_o;
  const float* home_ml;
  long long home_rows;
  // The own tokens' pieces: [piece][D / 4][piece_rows][4] and [piece][piece_rows][2].
  const float* part_o;
  const float* part_ml;
  const int2* first_piece;  // [batch] own pieces before a sequence, and its pieces per unit
  int piece_rows, head_groups;
  int* counter;          // pieces claimed: zeroed for the next call
  void* out;
  long long o_sb, o_sh;
  int out_dtype;
  int* err;
};

constexpr int kJoinRows = 8;   // rows of a block: 128-byte segments of the slots
constexpr int kJoinAhead = 4;  // partials whose loads are in flight together, per thread
constexpr int kJoinThreads = 256;

// One thread per (row, 4 columns, way); rows run fastest, so that the slots' rows are
// read in whole segments.  A row has up to some dozen partials (every CTA that held a
// piece of its unit, and its own pieces); each way has four on the way at a time.  The
// kernel is short and begins with a chain of dependent loads of small integers, which
// pass before it waits for the kernel before it.
// kJoinWays threads fold the partials of a row and 4 columns, then together.  Sixteen
// where four would leave SMs without a block (61 sequences, 8 heads of 64: the whole
// decode 20.1 us, 21.7 with four); four elsewhere (64 sequences, 32 heads of 128: 56 us, 78
// with sixteen; 8 sequences, 64 heads of 128: 118, 119).
template <int kJoinWays>
__global__ void __launch_bounds__(kJoinThreads, 4) join_kernel(const JoinParams p) {
  constexpr int kJoinCols = kJoinThreads / kJoinRows / kJoinWays;  // groups of 4 columns of a block
  const int cols = p.head_dim / 4;
  const int tid = threadIdx.x, lane = tid & 31;
  const int row = tid % kJoinRows, col = tid / kJoinRows % kJoinCols, way = tid / (kJoinRows * kJoinCols);
  const int d4 = blockIdx.z * kJoinCols + col;
  const int kvh = blockIdx.y;
  const int R = min(int(blockIdx.x) * kJoinRows + row, int(p.home_rows) - 1);
  const int b = R / p.group, hq = R - b * p.group;
  const int h = kvh * p.group + hq;
  const int len = __ldg(p.seq_lens + b);

  // Tiles on the line in all, and before the row's group.
  const Line line{p.groups, p.bn, p.num_kv_heads};
  const int g = p.groups.count > 0 ? p.groups.near(b) : 0;
  const bool in_group = p.groups.count > 0 && p.groups.has(g, b);
  const int g_first = __shfl_sync(0xffffffffu, g, 0);
  long long all = 0, before = 0;
  for (int i = lane; i < p.groups.count; i += 32) {
    const int n = line.tiles(i);
    all += n;
    if (i < g_first) before += n;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    all += __shfl_xor_sync(0xffffffffu, all, o);
    before += __shfl_xor_sync(0xffffffffu, before, o);
  }
  for (int i = g_first; i < g; ++i) before += line.tiles(i);
  const int n = in_group && all * p.num_kv_heads <= kMaxTiles ? line.tiles(g) : 0;
  const int shared = in_group ? p.groups.tokens(g) : 0;
  const int r = in_group ? R - p.groups.first(g) * p.group : 0;

  // Up to here only inputs were read: this kernel starts beside the one before it.
  grid_dependency_wait();
  const int gangs = __ldcg(p.info);
  const int2 own_pieces = __ldcg(p.first_piece + b);  // pieces before the sequence, per unit
  const bool first_thread = tid == 0 && blockIdx.z == 0 && blockIdx.y == 0 && blockIdx.x == 0;
  if (first_thread) p.counter[0] = p.counter[1] = 0;
  if (d4 == 0 && way == 0 && kvh == 0 && ((len > 0 && len < shared) || len > p.groups.cap_tokens))
    raise_error(p.err, FAT_DEVERR_BAD_LENGTH);

  // Where the row's prefix partials are: the unit's home, or the slots of its CTAs.
  // A gang has at least one tile, so these are gangs ca .. cb, of which only the first may
  // have begun before the unit (its partial is in the CTA's second slot).
  const long long total = all * p.num_kv_heads;
  const long long u = before * p.num_kv_heads + (long long)kvh * n;
  const bool narrow = (total + 1) * (gangs + 1) < (1ll << 32);
  auto owner = [&](long long x) {
    return narrow ? int((uint32_t(x + 1) * uint32_t(gangs) - 1u) / uint32_t(total))
                  : int(((x + 1) * gangs - 1) / total);
  };
  const int ca = n > 0 ? owner(u) : 0, cb = n > 0 ? owner(u + n - 1) : 0;
  const bool home = ca == cb;
  const long long start =
      n == 0 ? 0 : cut(ca, total, gangs);
  const bool began = n > 0 && start < u;
  const int member = r / p.cta_rows, r_cta = r - member * p.cta_rows;
  const int half = p.parts - 1;  // parts is 1 or 2
  const int n_prefix = n > 0 ? (cb - ca + 1) << half : 0;
  const int first_own = own_pieces.x + (kvh * p.head_groups + hq / own::kRows) * own_pieces.y;
  const int pieces = n_prefix + own_pieces.y;

  float M = -CUDART_INF_F, l = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  auto fold = [&](float2 ml, const float4& o) {
    if (ml.x == -CUDART_INF_F && ml.y == 0.f) return;  // no keys: o may hold anything
    const float mn = fmaxf(M, ml.x);
    const float a = M == -CUDART_INF_F ? 0.f : fast_exp2(M - mn);
    const float f = ml.x == -CUDART_INF_F ? 0.f : fast_exp2(ml.x - mn);
    l = l * a + ml.y * f;
    acc.x = acc.x * a + o.x * f;
    acc.y = acc.y * a + o.y * f;
    acc.z = acc.z * a + o.z * f;
    acc.w = acc.w * a + o.w * f;
    M = mn;
  };
  const bool col_in = d4 < cols;
  for (int i0 = way; i0 < pieces; i0 += kJoinWays * kJoinAhead) {
    float2 ml[kJoinAhead];
    float4 o[kJoinAhead];
#pragma unroll
    for (int k = 0; k < kJoinAhead; ++k) {
      ml[k] = make_float2(-CUDART_INF_F, 0.f);
      o[k] = make_float4(0.f, 0.f, 0.f, 0.f);
      const int i = i0 + k * kJoinWays;
      if (i < pieces && col_in) {
        const float *at_ml, *at_o;
        if (i >= n_prefix) {
          const long long x = first_own + (i - n_prefix);
          const int r8 = hq % own::kRows;
          at_ml = p.part_ml + (x * p.piece_rows + r8) * 2;
          at_o = p.part_o + ((x * cols + d4) * p.piece_rows + r8) * 4;
        } else if (home) {
          const long long at = (long long)i * p.num_kv_heads + kvh;
          at_ml = p.home_ml + (at * p.home_rows + R) * 2;
          at_o = p.home_o + ((at * cols + d4) * p.home_rows + R) * 4;
        } else {
          const int j = i >> half, part = i & half;
          const long long at = ((long long)(ca + j) * p.per_gang + member) * 2 + (began && j == 0 ? 1 : 0);
          const int sr = part * BM + r_cta / p.tile_rows * BM + r_cta % p.tile_rows;
          at_ml = p.slot_ml + (at * 256 + sr) * 2;
          at_o = p.slot_o + ((at * cols + d4) * 256 + sr) * 4;
        }
        ml[k] = __ldcg(reinterpret_cast<const float2*>(at_ml));
        o[k] = __ldcg(reinterpret_cast<const float4*>(at_o));
      }
    }
#pragma unroll
    for (int k = 0; k < kJoinAhead; ++k) fold(ml[k], o[k]);
  }

  // The ways of a row together, in their order.
  __shared__ float4 acc_s[kJoinWays][kJoinRows * kJoinCols];
  __shared__ float2 ml_s[kJoinWays][kJoinRows * kJoinCols];
  const int at = tid % (kJoinRows * kJoinCols);
  if (way > 0) {
    acc_s[way][at] = acc;
    ml_s[way][at] = make_float2(M, l);
  }
  __syncthreads();
  if (way > 0 || !col_in || int(blockIdx.x) * kJoinRows + row >= p.home_rows) return;
#pragma unroll
  for (int w = 1; w < kJoinWays; ++w) fold(ml_s[w][at], acc_s[w][at]);

  // A sequence without tokens gives zeros (like the decode kernel), whatever its queries
  // hold; a row whose scores are all -inf has no softmax and gives NaN.
  const float inv = 1.f / l;
  float4 y = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
  if (len <= 0) y = make_float4(0.f, 0.f, 0.f, 0.f);
  const long long out_at = (long long)b * p.o_sb + (long long)h * p.o_sh + d4 * 4;
  if (p.out_dtype == FAT_DTYPE_F32) {
    *reinterpret_cast<float4*>(static_cast<float*>(p.out) + out_at) = y;
  } else {
    uint2 v;
    if (p.out_dtype == FAT_DTYPE_F16) v = make_uint2(pack2<__half>(y.x, y.y), pack2<__half>(y.z, y.w));
    else v = make_uint2(pack2<__nv_bfloat16>(y.x, y.y), pack2<__nv_bfloat16>(y.z, y.w));
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + out_at) = v;
  }
}

// ---------------------------------------------------------------------------
// Finding the shared prefix
// ---------------------------------------------------------------------------
// One block per group: the first column in which a member's table differs from
// the first member's, among the pages that every member fills.
__global__ void __launch_bounds__(256) find_kernel(const Groups groups, const int* table, long long pt_sb,
                                                   int max_pages, const int* seq_lens, int min_sequences,
                                                   int* prefix_out) {
  __shared__ int limit;
  const int g = blockIdx.x;
  const int first = groups.first(g), n = groups.size(g);
  if (threadIdx.x == 0) limit = n >= max(min_sequences, 1) ? max_pages : 0;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += blockDim.x)
    atomicMin(&limit, max(__ldg(seq_lens + first + i), 0) / groups.page_size);
  __syncthreads();
  const int cols = limit;  // read by every thread before it can shrink
  __syncthreads();
  const long long items = (long long)(n - 1) * cols;
  for (long long i = threadIdx.x; i < items; i += blockDim.x) {
    const int m = int(i / cols) + 1, c = int(i % cols);
    if (__ldg(table + (first + m) * pt_sb + c) != __ldg(table + first * pt_sb + c)) atomicMin(&limit, c);
  }
  __syncthreads();
  if (threadIdx.x == 0) prefix_out[g] = limit * groups.page_size;
}

}  // namespace spx

// =============================================================================
// Host side
// =============================================================================
namespace {

size_t align_up(size_t x, size_t a) { return (x + a - 1) / a * a; }

spx::Plan make_plan(int sms, int group, int head_dim, int max_group) {
  spx::Plan p;
  const long long rows = (long long)std::max(max_group, 1) * group;
  p.mode = head_dim > 128 ? spx::kSolo : (max_group > spx::BM / group ? spx::kRowPair : spx::kAlternate);
  p.tile_rows = std::max(1, spx::BM / group) * group;
  p.cta_rows = p.mode == spx::kRowPair ? 2 * p.tile_rows : p.tile_rows;
  p.bn = head_dim > 128 ? 64 : 128;
  p.per_gang = int((rows + p.cta_rows - 1) / p.cta_rows);
  // One CTA per SM; a gang larger than the machine, and a quarter of it for the own tokens.
  p.ctas = std::max(sms, p.per_gang + sms / 4);
  p.parts = p.mode == spx::kAlternate ? 2 : 1;
  p.head_groups = (group + own::kRows - 1) / own::kRows;
  p.piece_rows = std::min(group, own::kRows);
  p.workers = p.ctas * 8;  // pieces are sized for this many warps (head_dim 256: half as many take them)
  return p;
}

struct ScratchLayout {
  size_t info, first_piece, slot_o, slot_ml, home_o, home_ml, part_o, part_ml, total;
};

ScratchLayout scratch_layout(const spx::Plan& p, int batch, int heads, int kv_heads, int head_dim) {
  ScratchLayout s;
  size_t off = 0;
  auto take = [&](size_t floats) {
    const size_t at = off;
    off = align_up(off + floats * sizeof(float), 256);
    return at;
  };
  const size_t ctas = size_t(p.ctas), rows = size_t(batch) * heads;
  s.info = take(64);
  s.first_piece = take(2 * size_t(batch));
  s.slot_o = take(ctas * 2 * 256 * head_dim);
  s.slot_ml = take(ctas * 2 * 256 * 2);
  s.home_o = take(size_t(p.parts) * rows * head_dim);
  s.home_ml = take(size_t(p.parts) * rows * 2);
  const size_t pieces = size_t(batch) * kv_heads * p.head_groups + size_t(p.workers) * own::kPiecesPerWarp;
  s.part_o = take(pieces * p.piece_rows * head_dim);
  s.part_ml = take(pieces * p.piece_rows * 2);
  s.total = off;
  return s;
}

}  // namespace

size_t shared_prefix_scratch_bytes(int device, int batch, int num_heads, int num_kv_heads, int head_dim,
                                   int max_group) {
  if (batch <= 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads || head_dim <= 0) return 0;
  const spx::Plan p = make_plan(sm_count(device), num_heads / num_kv_heads, head_dim, std::min(max_group, batch));
  return scratch_layout(p, batch, num_heads, num_kv_heads, head_dim).total;
}

int check_shared_prefix(const SharedPrefixArgs& a) {
  const DecodeArgs& d = a.d;
  const int rc = check_paged_decode(d);
  if (rc != FAT_OK || d.batch == 0) return rc;
  if (a.num_groups < 0) return invalid("shared_prefix_decode: num_groups must be non-negative");
  if (a.max_group < 0) return invalid("shared_prefix_decode: max_group must be non-negative");
  if (a.cu_groups == nullptr || (a.num_groups > 0 && a.prefix_lens == nullptr))
    return invalid("shared_prefix_decode: null pointer argument");
  if (d.num_heads / d.num_kv_heads > spx::BM)
    return unsupported("shared_prefix_decode: at most " + std::to_string(spx::BM) + " query heads per KV head, got " +
                       std::to_string(d.num_heads / d.num_kv_heads));
  if (d.num_kv_heads > 65535)  // a dimension of the join's grid
    return unsupported("shared_prefix_decode: at most 65535 KV heads, got " + std::to_string(d.num_kv_heads));
  const int ob = d.out_dtype == FAT_DTYPE_F32 ? 4 : 2;
  if ((reinterpret_cast<uintptr_t>(d.out) & 15u) || (d.o_sb * ob) % 16 || (d.o_sh * ob) % 16)
    return unsupported("shared_prefix_decode: out must be 16-byte aligned with 16-byte-multiple strides");
  return FAT_OK;
}

int launch_shared_prefix(const SharedPrefixArgs& a) {
  const DecodeArgs& d = a.d;
  int rc = check_shared_prefix(a);
  if (rc != FAT_OK || d.batch == 0) return rc;
  const int device = current_device();
  if (device < 0) return invalid("shared_prefix_decode: no current CUDA device");
  const int group = d.num_heads / d.num_kv_heads;
  const spx::Plan plan = make_plan(sm_count(device), group, d.head_dim, std::min(a.max_group, d.batch));
  const ScratchLayout lay = scratch_layout(plan, d.batch, d.num_heads, d.num_kv_heads, d.head_dim);
  if (d.workspace_bytes < 2 * sizeof(int)) {
    set_last_error("shared_prefix_decode: workspace too small");
    return FAT_ERR_WORKSPACE;
  }
  if (a.scratch == nullptr) return invalid("shared_prefix_decode: null scratch");
  if (a.scratch_bytes < lay.total) {
    set_last_error("shared_prefix_decode: scratch holds " + std::to_string(a.scratch_bytes) + " bytes, needs " +
                   std::to_string(lay.total));
    return FAT_ERR_WORKSPACE;
  }
  uint8_t* base = static_cast<uint8_t*>(a.scratch);
  auto at = [&](size_t off) { return reinterpret_cast<float*>(base + off); };
  const int cap = int(std::min<long long>((long long)d.max_pages * d.page_size, 1ll << 30));

  spx::Params p{};
  p.tile_rows = plan.tile_rows;
  p.q_bf16 = d.q_dtype == FAT_DTYPE_BF16;
  p.q_negate = d.softmax_scale < 0.f;
  p.scale_log2 = float(std::abs(double(d.softmax_scale)) * 1.4426950408889634);
  p.groups = Groups{a.cu_groups, a.prefix_lens, a.num_groups, d.batch, d.page_size, cap, std::min(a.max_group, d.batch)};
  p.page_table = d.page_table;
  p.pt_sb = d.pt_sb;
  p.seq_lens = d.seq_lens;
  p.max_pages = int(d.max_pages);
  p.num_pages = int(d.num_pages);
  p.page_size = d.page_size;
  p.num_kv_heads = d.num_kv_heads;
  p.group = group;
  p.head_dim = d.head_dim;
  p.k_scale = d.k_scale;
  p.v_scale = d.v_scale;
  p.s_sp = d.scale_sp;
  p.per_gang = plan.per_gang;
  p.info = reinterpret_cast<int*>(base + lay.info);
  p.first_piece = reinterpret_cast<int2*>(base + lay.first_piece);
  p.slot_o = at(lay.slot_o);
  p.slot_ml = at(lay.slot_ml);
  p.home_o = at(lay.home_o);
  p.home_ml = at(lay.home_ml);
  p.home_rows = (long long)d.batch * group;
  p.err = d.error_word;
  p.wait_ns = wait_limit_ns();

  own::Params o{};
  o.q = d.q;
  o.q_sb = d.q_sb;
  o.q_sh = d.q_sh;
  o.page_table = d.page_table;
  o.pt_sb = d.pt_sb;
  o.seq_lens = d.seq_lens;
  o.k_scale = d.k_scale;
  o.v_scale = d.v_scale;
  o.s_sp = d.scale_sp;
  o.groups = p.groups;
  o.num_kv_heads = d.num_kv_heads;
  o.group = group;
  o.head_groups = plan.head_groups;
  o.num_pages = int(d.num_pages);
  o.max_pages = int(d.max_pages);
  o.rows = plan.piece_rows;
  o.workers = plan.workers;
  o.scale_log2 = float(double(d.softmax_scale) * 1.4426950408889634);
  o.part_o = at(lay.part_o);
  o.part_ml = at(lay.part_ml);
  o.counter = static_cast<int*>(d.workspace);
  o.err = d.error_word;
  o.wait_ns = p.wait_ns;
  p.expire = o.expire = take_expire_request() ? 1 : 0;
  // The join reads what the kernel before it on the stream left in the scratch: calls of two
  // threads on one stream go out one after the other.
  static std::mutex order;
  const std::lock_guard<std::mutex> lock(order);
  switch (d.kv_dtype) {
    case FAT_DTYPE_F16:
      rc = spx::launch_f16(a, plan, p, o);
      break;
    case FAT_DTYPE_BF16:
      rc = spx::launch_bf16(a, plan, p, o);
      break;
    case FAT_DTYPE_I8:
      rc = spx::launch_i8(a, plan, p, o);
      break;
    default:
      rc = spx::launch_e4m3(a, plan, p, o);
      break;
  }
  if (rc != FAT_OK) return rc;

  spx::JoinParams j{};
  j.groups = p.groups;
  j.seq_lens = d.seq_lens;
  j.bn = plan.bn;
  j.num_kv_heads = d.num_kv_heads;
  j.group = group;
  j.head_dim = d.head_dim;
  j.info = p.info;
  j.per_gang = plan.per_gang;
  j.tile_rows = plan.tile_rows;
  j.cta_rows = plan.cta_rows;
  j.parts = plan.parts;
  j.slot_o = p.slot_o;
  j.slot_ml = p.slot_ml;
  j.home_o = p.home_o;
  j.home_ml = p.home_ml;
  j.home_rows = p.home_rows;
  j.part_o = o.part_o;
  j.part_ml = o.part_ml;
  j.piece_rows = plan.piece_rows;
  j.head_groups = plan.head_groups;
  j.first_piece = p.first_piece;
  j.counter = o.counter;
  j.out = d.out;
  j.o_sb = d.o_sb;
  j.o_sh = d.o_sh;
  j.out_dtype = d.out_dtype;
  j.err = d.error_word;
  auto join = [&](auto kern, int ways) {
    const int cols = spx::kJoinThreads / spx::kJoinRows / ways * 4;
    const dim3 grid(unsigned((p.home_rows + spx::kJoinRows - 1) / spx::kJoinRows), unsigned(d.num_kv_heads),
                    unsigned((d.head_dim + cols - 1) / cols));
    return launch_dependent(kern, grid, spx::kJoinThreads, 0, d.stream, j);
  };
  // With four ways a block has 8 rows of 32 columns: one per SM from this many values on.
  const bool many = (long long)d.batch * d.num_heads * d.head_dim >= (long long)sm_count(device) * spx::kJoinRows * 32;
  const cudaError_t e = many ? join(spx::join_kernel<4>, 4) : join(spx::join_kernel<16>, 16);
  if (e != cudaSuccess) {
    // Without its join the call leaves pieces counted, and the next call on the workspace
    // would take them as its own.
    cudaMemsetAsync(o.counter, 0, 2 * sizeof(int), d.stream);
    return cuda_failure("shared prefix join launch", e);
  }
  return FAT_OK;
}

int find_shared_prefix(const int32_t* page_table, int64_t pt_sb, int64_t max_pages, const int32_t* seq_lens,
                       int batch, int page_size, const int32_t* cu_groups, int num_groups, int min_sequences,
                       int32_t* prefix_out, cudaStream_t stream) {
  if (batch < 0 || num_groups < 0 || max_pages < 0 || page_size <= 0)
    return invalid("find_shared_prefix: sizes must be non-negative, page_size positive");
  if (num_groups == 0) return FAT_OK;
  if (page_table == nullptr || seq_lens == nullptr || cu_groups == nullptr || prefix_out == nullptr)
    return invalid("find_shared_prefix: null pointer argument");
  const int cap = int(std::min<long long>((long long)max_pages * page_size, 1ll << 30));
  spx::find_kernel<<<num_groups, 256, 0, stream>>>(Groups{cu_groups, nullptr, num_groups, batch, page_size, cap, batch},
                                                   page_table, pt_sb, cap / page_size, seq_lens, min_sequences,
                                                   prefix_out);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_failure("find_shared_prefix launch", e);
  return FAT_OK;
}

}  // namespace fat
