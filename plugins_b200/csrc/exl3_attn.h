// exl3_attn.h -- a layer's attention side (norms + rotation into a paged cache, tree attention over it, its pages):
// the launch parameters shared by the kernels (exl3_norm_rope.cu, exl3_attn_mma.cu, exl3_attn_tc.cu, exl3_pages.cu) and
// the C entries (exl3_attn.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/exl3_b200.h"

namespace exl3 {

// The device workspace as the attention side uses it: split partials, counters (zero between launches), error word.
struct Workspace {
  float* partials;
  size_t partial_floats;
  uint32_t* counters;
  uint32_t counter_count;
  uint32_t* err;
  int sms;
};
exl3_verdict workspace_create(int device);  // once per device (ensure_device)
bool workspace_get(int device, Workspace& ws);

// One layer of the paged cache and one step's rows, as the kernels read them.
struct PagedBatch {
  uint16_t *k, *v;  // the layer's first slot (16-bit elements)
  int64_t page_stride, head_stride, token_stride;
  int32_t pages, page_shift;  // page_size = 1 << page_shift
  int32_t kv_heads;
  int32_t nseq, rows, max_pages, tree_words;
  const int32_t *row_start, *context, *table;
  const uint32_t* tree;
  const int32_t* position;
  uint32_t* err;
};

struct HeadsView {
  void* data;
  int32_t dtype, heads;
  int64_t row_stride, head_stride;
  int32_t vec;  // vectors of this many times 16 bytes are aligned: 0, 1 or 2
};

struct NormRopeParams {
  PagedBatch b;
  HeadsView q, k, v, out;
  const void *q_weight, *k_weight;
  const double* inv_freq;
  int32_t dim, rot_dims, adjacent, weight_dtype, cache_dtype;
  float eps, weight_offset;
};
cudaError_t launch_norm_rope(const NormRopeParams& p, int sms, cudaStream_t st);

struct AttnParams {
  PagedBatch b;
  HeadsView q, out;
  float* lse;        // [rows][heads], or null
  int32_t group;     // query heads per kv head
  int32_t bf16;      // the element type: bf16, else f16
  int32_t max_rows, max_context;
  float scale_log2;  // scale * log2(e)
  float* partials;   // two slots per CTA
  uint32_t* counters;
};
// Rows per kv head up to which the few-row kernel runs: its one 16-row tile, or half of it with 256-wide heads.  Measured,
// few-row / tensor-core kernel: 32 sequences over 1500-9001 slots, 128-wide heads, 4 rows 121 / 130 us, 16 rows 128 / 136,
// 20 rows (two tiles, K and V read twice) 215 / 141; 64-wide, 8 rows 55 / 63; five sequences over 20-33k slots, 256-wide, 2
// rows 174 / 180, 8 rows 180 / 180, up to 16 rows 192 / 182; one token over 301 slots 14 / 18 (one call between two events;
// the other figures likewise).
constexpr int attn_few_rows(int dim) { return dim == 256 ? 8 : 16; }
// the tensor-core kernel (exl3_attn_tc.cu) and the few-row kernel (exl3_attn_mma.cu)
cudaError_t launch_attn_tc(const AttnParams& p, int dim, int sms, size_t partial_floats, cudaStream_t st);
cudaError_t launch_attn_mma(const AttnParams& p, int dim, int sms, size_t partial_floats, cudaStream_t st);

struct PageParams {
  int32_t pages, page_shift;
  int32_t nseq_in, nseq_out, width_in, width_out;
  const int32_t *refs_in, *table_in, *held_in, *lens_in;
  int32_t *refs, *table, *held, *lens;
  const int32_t *parent, *need;
  int32_t* missing;
  int32_t* moves;    // [1 + 2 * capacity]: count, then (source, destination) pages
  int32_t* scratch;  // grow: [3 * nseq + 2 * pages]
  uint32_t* err;
};
struct PagePool {
  uint16_t *k, *v;
  int64_t layer_stride, page_stride, head_stride, token_stride;
  int32_t layers, kv_heads, page_size, dim;
};
int cache_grow_max_rows();
cudaError_t launch_cache_fork(const PageParams& p, cudaStream_t st);
cudaError_t launch_cache_grow(const PageParams& p, cudaStream_t st);
cudaError_t launch_cache_compact(const PageParams& p, cudaStream_t st);
// copies moves[0] pages, every layer, k and v; max_moves bounds the count
cudaError_t launch_page_copy(const PagePool& pool, const int32_t* moves, int64_t max_moves, int sms, cudaStream_t st);

struct KeepParams {
  PagePool pool;
  PagedBatch b;
  const int32_t *path, *kept;
  int32_t depth;
  int32_t* lens;       // may be b.context, or kept
  uint32_t* counters;  // where it is, one per sequence of a launch; else null
  int32_t seq0;        // the launch's first sequence
};
cudaError_t launch_cache_keep(const KeepParams& p, uint32_t counters, cudaStream_t st);

#if defined(__CUDACC__)
// The sequence that owns `row`: the last s with row_start[s] <= row (empty sequences own none).  Called by a whole warp;
// 32-way search, so two loads deep up to 1024 sequences.
__device__ __forceinline__ int seq_of_row(const int32_t* row_start, int nseq, int row, uint32_t lane) {
  int lo = 0, n = nseq;  // the answer is in [lo, lo + n)
  while (n > 1) {
    const int step = (n + 31) / 32;
    const int at = lo + static_cast<int>(lane) * step;
    const bool le = static_cast<int>(lane) * step < n && row_start[at] <= row;
    const int c = __popc(__ballot_sync(0xFFFFFFFFu, le));  // lane 0's is true: row_start[lo] <= row
    const int first = c > 0 ? (c - 1) * step : 0;
    lo += first;
    n = n - first < step ? n - first : step;
  }
  return lo;
}
#endif

}  // namespace exl3
