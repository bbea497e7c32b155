// Host-side interface of the page operations (internal to the library).
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace fat {

// The K/V storage of a pool: byte strides, one row = head_dim elements of one (slot, KV head).
struct PageStore {
  void* k{};
  void* v{};
  int64_t sp_bytes{}, ss_bytes{}, sh_bytes{};
  int64_t num_pages{};
  int num_kv_heads{}, page_size{};
  int64_t row_bytes{};
  float* k_scale{};  // optional [num_pages][num_kv_heads], both or neither
  float* v_scale{};
  int64_t scale_sp{};
};

// The rows of a pool: page tables, lengths, owned entries per row, references per page.
struct PageRows {
  int32_t* table{};
  int64_t pt_sb{}, max_pages{};
  int32_t* seq_lens{};
  int32_t* owned{};
  int32_t* refs{};
  int batch{};
  int32_t* released{};  // optional: rows released and not taken up again
  bool skip_released{}; // a reserve of all rows leaves those out
};

size_t page_scratch_bytes(int64_t num_pages, int batch);

int launch_copy_pages(const PageStore& s, const int32_t* src, const int32_t* dst, int n, int32_t* err,
                      cudaStream_t stream);
int launch_fork_rows(const PageStore& s, const PageRows& r, const int32_t* src, const int32_t* dst, int n,
                     void* scratch, size_t scratch_bytes, int32_t* err, cudaStream_t stream);
int launch_release_rows(const PageStore& s, const PageRows& r, const int32_t* rows, int n, int32_t* err,
                        cudaStream_t stream);
int launch_reserve_tokens(const PageStore& s, const PageRows& r, const int32_t* rows, int n, int tokens,
                          void* scratch, size_t scratch_bytes, int32_t* err, cudaStream_t stream);
int launch_compact_pages(const PageStore& s, const PageRows& r, int32_t* table_out, int64_t pt_out_sb,
                         int32_t* refs_out, int32_t* live_out, void* scratch, size_t scratch_bytes, int32_t* err,
                         cudaStream_t stream);

}  // namespace fat
