// exl3_evict.cu -- of a row's cached tokens those stay that were attended to most, in every layer and kv head for itself
// (exl3_cache_evict, include/exl3_b200.h).  The pages' bookkeeping comes first (evict_pages_kernel, exl3_pages.cu).
//
// One CTA per (row, layer, kv head).  The n-th heaviest weight is found by digits: a histogram of the keys' next 11 bits
// (then 11, then 10) among those that agree with the digits so far, and the digit at which the count from the top reaches n.
// A key is the weight's bits turned so that whole numbers order as weights do, NaN above all; of equal keys the lowest
// slots stay.
// Then the slots in order: a scan of what stays gives each token its new slot, and the tokens move in groups, all of a group
// read before any of it is written.  A token's new slot is never above its old one, and a group's new slots are below every
// later group's old ones: in place, nothing is overwritten before it is read.
//
// What bounds it: HBM while tokens move, every moved byte read and written once (16 rows of 300-1300 slots cut to 400-517 in 36
// layers: 297 us, 1.69 GB, 5.7 TB/s; 20 forked rows in 12 layers: 261 us, 1.53 GB, 5.9 TB/s); with few long rows the chain of
// one CTA (four rows of 30-40k slots cut to 4096 in 6 layers: 195 us, 0.84 GB, 4.3 TB/s).
#include <cuda_runtime.h>

#include "exl3_attn.h"
#include "exl3_common.cuh"
#include "exl3_internal.h"

namespace exl3 {

namespace {

constexpr int kPer = 4;                    // slots of a thread in a run
constexpr int kBins = 2048;
constexpr int kAhead = 4;                  // tokens of a thread in flight (two: 327 us where four take 297)

// Weights as whole numbers of their order: -NaN .. NaN all at the top, -0 as 0.
__device__ __forceinline__ uint32_t key_of(float w) {
  if (w != w) return 0xFFFFFFFFu;
  const uint32_t u = __float_as_uint(w + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Exclusive scan of a pair of 16-bit counts over the CTA; *total receives the sum.
template <int kWarps>
__device__ __forceinline__ uint32_t scan_pair(uint32_t v, uint32_t* s_warp, uint32_t* total) {
  const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
  uint32_t x = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const uint32_t o = __shfl_up_sync(0xFFFFFFFFu, x, d);
    if (static_cast<int>(lane) >= d) x += o;
  }
  if (lane == 31) s_warp[warp] = x;
  __syncthreads();
  uint32_t before = 0, all = 0;
#pragma unroll
  for (uint32_t w = 0; w < kWarps; ++w) {
    const uint32_t o = s_warp[w];
    if (w < warp) before += o;
    all += o;
  }
  *total = all;
  return before + x - v;
}

template <int kThreads>
struct Shared {
  static constexpr int kRing = kThreads * kPer + 512;
  uint32_t hist[kBins];
  uint32_t warp[2][kThreads / 32];
  uint32_t digit, above, inside;
  int slot[kRing], page[kRing];  // tokens that stay and have not moved: old slots and their pages, a ring
};

// The key of the n-th heaviest of the slots [lo, hi) (n of at least 1 and fewer than there are), and how many of its equals
// stay.
template <int kThreads>
__device__ void select_key(const float* w, int lo, int hi, int n, Shared<kThreads>& s, uint32_t& key, int& equals) {
  uint32_t prefix = 0, mask = 0;
  int left = n;
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bins = pass == 2 ? 1024 : kBins;
    for (int i = static_cast<int>(threadIdx.x); i < bins; i += kThreads) s.hist[i] = 0u;
    __syncthreads();
#pragma unroll kThreads / 64  // (512 threads, long rows: 8 at a time 195 us, 4 199, 16 194; 256 threads: 4 297 us, 8 305)
    for (int j = lo + static_cast<int>(threadIdx.x); j < hi; j += kThreads) {
      const uint32_t k = key_of(w[j]);
      if ((k & mask) == prefix) atomicAdd(&s.hist[(k >> shift) & (bins - 1)], 1u);
    }
    __syncthreads();
    // counts from the top: a thread has bins / kThreads neighbours
    const int per = bins / kThreads;
    const int top = bins - 1 - static_cast<int>(threadIdx.x) * per;
    uint32_t mine = 0;
    for (int i = 0; i < per; ++i) mine += s.hist[top - i];
    // (counts may need more than 16 bits here: one at a time)
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    uint32_t upto = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const uint32_t o = __shfl_up_sync(0xFFFFFFFFu, upto, d);
      if (static_cast<int>(lane) >= d) upto += o;
    }
    if (lane == 31) s.warp[0][warp] = upto;
    __syncthreads();
    for (uint32_t v = 0; v < warp; ++v) upto += s.warp[0][v];
    uint32_t before = upto - mine;
    if (before < static_cast<uint32_t>(left) && upto >= static_cast<uint32_t>(left)) {
      int i = 0;
      while (before + s.hist[top - i] < static_cast<uint32_t>(left)) before += s.hist[top - i], ++i;
      s.digit = top - i, s.above = before, s.inside = s.hist[top - i];
    }
    __syncthreads();
    left -= static_cast<int>(s.above);
    prefix |= s.digit << shift;
    mask |= static_cast<uint32_t>(bins - 1) << shift;
    if (static_cast<int>(s.inside) == left && prefix != 0u) {  // the whole digit stays
      key = prefix - 1u, equals = 0;
      return;
    }
  }
  key = prefix;
  equals = left;
}

template <int D, int kThreads>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads) evict_kernel(const EvictParams p) {
  constexpr int kRun = kThreads * kPer, kRing = Shared<kThreads>::kRing;
  __shared__ Shared<kThreads> s;
  pdl_wait();
  const int tid = static_cast<int>(threadIdx.x);
  const int head = static_cast<int>(blockIdx.x) % p.pool.kv_heads;
  const int64_t rest = blockIdx.x / p.pool.kv_heads;
  const int layer = static_cast<int>(rest % p.pool.layers), row = static_cast<int>(rest / p.pool.layers);
  const int len = p.lens_in[row], keep = p.lens[row];
  const float* w = p.w + layer * p.w_layer + row * p.w_row + head * p.w_head;
  float* out = p.w_out + layer * p.out_layer + row * p.out_row + head * p.out_head;
  if (keep >= len) {  // not cut (and perhaps a length past the weights' slots)
    const int all = min(len, p.slots);
    if (w != out)
      for (int j = tid; j < all; j += kThreads) out[j] = w[j];
    return;
  }
  const int lo = p.sink, hi = len - p.recent;  // (sink + recent <= keep < len)
  const int want = keep - p.sink - p.recent;
  uint32_t key = 0xFFFFFFFFu;
  int equals = 0;
  if (want > 0) select_key(w, lo, hi, want, s, key, equals);

  constexpr int kLanes = D / 8, kTokens = kThreads / kLanes, kGroup = kTokens * kAhead;
  static_assert(kGroup <= 512, "what is left in the ring");
  const int c = tid % kLanes, g = tid / kLanes;
  const int64_t base = layer * p.pool.layer_stride + head * p.pool.head_stride + c * 8;
  const int32_t* from = p.table_in + static_cast<int64_t>(row) * p.width;
  const int32_t* to = p.table + static_cast<int64_t>(row) * p.width;
  const int page_mask = (1 << p.page_shift) - 1;
  auto page_of = [&](int id) {  // of a table's entry
    if (id >= 0 && id < p.pages) return id;
    atomicOr(p.err, kErrBadShape);
    return -1;
  };
  int done = 0, found = 0;    // tokens moved, and found
  int ties = 0;               // equals of the key so far
  // tokens done .. done + kGroup - 1 (those found): read, then written
  auto move = [&]() {
    uint4 k[kAhead], v[kAhead];
    int64_t dst[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int d = done + i * kTokens + g;
      dst[i] = -1;
      if (d < found) {
        const int slot = s.slot[d % kRing], page = s.page[d % kRing], page2 = page_of(to[d >> p.page_shift]);
        if (page >= 0 && page2 >= 0 && (slot != d || page != page2)) {
          const int64_t at = base + page * p.pool.page_stride + (slot & page_mask) * p.pool.token_stride;
          k[i] = *reinterpret_cast<const uint4*>(p.pool.k + at);
          v[i] = *reinterpret_cast<const uint4*>(p.pool.v + at);
          dst[i] = base + page2 * p.pool.page_stride + (d & page_mask) * p.pool.token_stride;
        }
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      if (dst[i] >= 0) {
        *reinterpret_cast<uint4*>(p.pool.k + dst[i]) = k[i];
        *reinterpret_cast<uint4*>(p.pool.v + dst[i]) = v[i];
      }
    done += kGroup;
  };
  uint32_t turn = 0;
  // A run's weights and pages, fetched a run ahead (what this run writes lies before the next: 4 rows of 30-40k slots 213 us,
  // 198 so; 16 rows in 36 layers 301 / 292).  A thread's slots lie in one page.
  float next[kPer];
  int next_id;
  auto fetch = [&](int j0) {
    const int j = j0 + tid * kPer;
#pragma unroll
    for (int i = 0; i < kPer; ++i) next[i] = j + i < len ? w[j + i] : 0.f;
    next_id = j < len ? from[j >> p.page_shift] : 0;
  };
  fetch(0);
  for (int j0 = 0; j0 < len; j0 += kRun) {
    float x[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) x[i] = next[i];
    const int id = next_id;
    fetch(j0 + kRun);
    uint32_t pair[kPer], mine = 0;  // low half: stays whatever its equals; high half: equals the key
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int j = j0 + tid * kPer + i;
      pair[i] = 0u;
      if (j < len) {
        if (j < lo || j >= hi) pair[i] = 1u;
        else if (want > 0) {
          const uint32_t u = key_of(x[i]);
          pair[i] = u > key ? 1u : u == key ? 0x10000u : 0u;
        }
      }
      mine += pair[i];
    }
    uint32_t total;
    uint32_t before = scan_pair<kThreads / 32>(mine, s.warp[turn++ & 1u], &total);
    // (its barrier: all of the run's weights are read)
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int j = j0 + tid * kPer + i;
      const int tie = ties + static_cast<int>(before >> 16);
      const bool stays = (pair[i] & 1u) || (pair[i] && tie < equals);
      if (stays) {
        const int d = found + static_cast<int>(before & 0xFFFFu) + min(tie, equals) - min(ties, equals);
        s.slot[d % kRing] = j;
        s.page[d % kRing] = page_of(id);
        if (out != w || d != j) out[d] = x[i];
      }
      before += pair[i];
    }
    const int tied = ties + static_cast<int>(total >> 16);
    found += static_cast<int>(total & 0xFFFFu) + min(tied, equals) - min(ties, equals);
    ties = tied;
    __syncthreads();  // the ring's new entries
    while (found - done >= kGroup) move();
  }
  while (done < found) move();
}

// A thread per layer and kv head of one sequence walks the path, which ascends: a weight is read before its slot is written.
// A few hundred words in all; the launch is what it costs.
__global__ void __launch_bounds__(256) weight_keep_kernel(const WeightKeepParams p) {
  pdl_wait();
  const int s = static_cast<int>(blockIdx.y), item = static_cast<int>(blockIdx.x) * 256 + static_cast<int>(threadIdx.x);
  const int ctx = p.context[s], kept = p.kept[s];
  const int ntok = max(0, min(p.row_start[s + 1], p.rows) - max(p.row_start[s], 0));
  const int32_t* path = p.path + static_cast<int64_t>(s) * p.depth;
  bool ok = ctx >= 0 && kept >= 0 && kept <= min(ntok, p.depth) && static_cast<int64_t>(ctx) + ntok <= p.slots;
  for (int d = 0; ok && d < kept; ++d) ok = path[d] < ntok && path[d] >= (d ? path[d - 1] + 1 : 0);
  if (!ok) {
    if (item == 0) atomicOr(p.err, kErrBadShape);
    return;
  }
  if (item >= p.layers * p.kv_heads) return;
  float* w = p.w + item / p.kv_heads * p.w_layer + s * p.w_row + item % p.kv_heads * p.w_head + ctx;
  for (int d = 0; d < kept; ++d)
    if (path[d] != d) w[d] = w[path[d]];
}

template <int D>
cudaError_t launch_dim(const EvictParams& p, int sms, cudaStream_t st) {
  const int64_t units = static_cast<int64_t>(p.nseq) * p.pool.layers * p.pool.kv_heads;
  // Smaller CTAs where there are many: more of them hide one another's selections (4608 rows of 300-1300 slots: 512 threads
  // 335 us, 256 threads 307); larger ones where a few have to move much each (960 rows of 0.9-4k slots: 262 / 272; 192 rows of
  // 30-40k: 216 / 292).
  const auto grid = dim3(static_cast<unsigned>(units));
  return units >= 16 * static_cast<int64_t>(sms) ? launch_pdl_k(evict_kernel<D, 256>, grid, dim3(256), st, p)
                                                 : launch_pdl_k(evict_kernel<D, 512>, grid, dim3(512), st, p);
}

}  // namespace

cudaError_t launch_weight_keep(const WeightKeepParams& p, cudaStream_t st) {
  const dim3 grid(static_cast<unsigned>((static_cast<int64_t>(p.layers) * p.kv_heads + 255) / 256), static_cast<unsigned>(p.nseq));
  return launch_pdl_k(weight_keep_kernel, grid, dim3(256), st, p);
}

cudaError_t launch_evict_tokens(const EvictParams& p, int sms, cudaStream_t st) {
  switch (p.pool.dim) {
    case 64: return launch_dim<64>(p, sms, st);
    case 128: return launch_dim<128>(p, sms, st);
    default: return launch_dim<256>(p, sms, st);
  }
}

}  // namespace exl3
