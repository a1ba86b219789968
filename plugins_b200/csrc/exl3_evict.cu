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
#include <cuda_runtime.h>

#include "exl3_attn.h"
#include "exl3_common.cuh"
#include "exl3_internal.h"

namespace exl3 {

namespace {

constexpr int kPer = 4;                    // slots of a thread in a run
constexpr int kBins = 2048;
constexpr int kAhead = 4;                  // tokens of a thread in flight

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

constexpr int kHeld = 4096;   // weights that fit in shared memory
constexpr int kFew = 512;     // candidates that are ranked by comparing each with each

template <int kThreads>
struct Shared {
  static constexpr int kRing = kThreads * kPer + 512;
  uint32_t hist[kBins];
  float w[kHeld];
  uint32_t few[kFew];
  uint32_t warp[2][kThreads / 32];
  uint32_t digit, above, inside, count, key;
  int equals;
  int slot[kRing], page[kRing];  // tokens that stay and have not moved: old slots and their pages, a ring
};

// f(key) for every slot of [lo, hi): eight of a thread's weights on their way at once.
template <int kThreads, typename At, typename F>
__device__ __forceinline__ void each_key(At&& at, int lo, int hi, F&& f) {
  constexpr int kBatch = 8;
  int j = lo + static_cast<int>(threadIdx.x);
  for (; j + (kBatch - 1) * kThreads < hi; j += kBatch * kThreads) {
    float x[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) x[i] = at(j + i * kThreads);
#pragma unroll
    for (int i = 0; i < kBatch; ++i) f(key_of(x[i]));
  }
  for (; j < hi; j += kThreads) f(key_of(at(j)));
}

// The n-th heaviest of the slots [lo, hi) (n of at least 1 and fewer than there are): all above `key` stay, and `equals` of
// its equals.  at(j): slot j's weight.
template <int kThreads, typename At>
__device__ void select_key(At&& at, int lo, int hi, int n, Shared<kThreads>& s, uint32_t& key, int& equals) {
  constexpr uint32_t kZero = 0x80000000u;  // the key of 0, which many weights may have: counted apart, not by atomics
  const int tid = static_cast<int>(threadIdx.x);
  const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
  uint32_t prefix = 0, mask = 0;
  int left = n;
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bins = pass == 2 ? 1024 : kBins;
    for (int i = tid; i < bins; i += kThreads) s.hist[i] = 0u;
    if (tid == 0) s.count = 0u;
    __syncthreads();
    uint32_t zeros = 0;
    each_key<kThreads>(at, lo, hi, [&](uint32_t k) {
      if (k == kZero) ++zeros;
      else if ((k & mask) == prefix) atomicAdd(&s.hist[(k >> shift) & (bins - 1)], 1u);
    });
    zeros = __reduce_add_sync(0xFFFFFFFFu, (kZero & mask) == prefix ? zeros : 0u);
    if (lane == 0 && zeros) atomicAdd(&s.hist[(kZero >> shift) & (bins - 1)], zeros);
    __syncthreads();
    // counts from the top: a thread has bins / kThreads neighbours
    const int per = bins / kThreads, top = bins - 1 - tid * per;
    uint32_t mine = 0;
    for (int i = 0; i < per; ++i) mine += s.hist[top - i];
    uint32_t upto = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const uint32_t o = __shfl_up_sync(0xFFFFFFFFu, upto, d);
      if (static_cast<int>(lane) >= d) upto += o;
    }
    if (lane == 31) s.warp[0][warp] = upto;
    __syncthreads();
#pragma unroll
    for (uint32_t v = 0; v < kThreads / 32; ++v)
      if (v < warp) upto += s.warp[0][v];
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
    const int inside = static_cast<int>(s.inside);
    if (inside == left && prefix != 0u) {  // the whole bin stays
      key = prefix - 1u, equals = 0;
      return;
    }
    if (pass < 2 && inside <= kFew && prefix != (kZero & mask)) {
      each_key<kThreads>(at, lo, hi, [&](uint32_t k) {
        if ((k & mask) == prefix) s.few[atomicAdd(&s.count, 1u)] = k;
      });
      __syncthreads();
      for (int i = tid; i < inside; i += kThreads) {
        const uint32_t k = s.few[i];
        int more = 0, same = 0;
        for (int o = 0; o < inside; ++o) more += s.few[o] > k ? 1 : 0, same += s.few[o] == k ? 1 : 0;
        if (more < left && left <= more + same) s.key = k, s.equals = left - more;  // (its equals write the same)
      }
      __syncthreads();
      key = s.key, equals = s.equals;
      return;
    }
  }
  key = prefix, equals = left;
}

template <int D, int kThreads>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads) evict_kernel(const EvictParams p) {
  constexpr int kRun = kThreads * kPer, kRing = Shared<kThreads>::kRing;
  extern __shared__ __align__(16) uint8_t smem[];
  Shared<kThreads>& s = *reinterpret_cast<Shared<kThreads>*>(smem);
  pdl_wait();
  const int tid = static_cast<int>(threadIdx.x);
  const int head = static_cast<int>(blockIdx.x) % p.pool.kv_heads;
  const int64_t rest = blockIdx.x / p.pool.kv_heads;
  const int layer = static_cast<int>(rest % p.pool.layers), row = static_cast<int>(rest / p.pool.layers);
  const int len = p.lens_in[row], keep = p.lens[row];
  const float* w = p.w + layer * p.w_layer + row * p.w_row + head * p.w_head;
  float* out = p.w_out + layer * p.out_layer + row * p.out_row + head * p.out_head;
  if (keep >= len) {  // not cut
    if (w != out)
      for (int j = tid; j < len; j += kThreads) out[j] = w[j];
    return;
  }
  const bool held = len <= kHeld;
  if (held) {
#pragma unroll 4
    for (int j = tid; j < len; j += kThreads) s.w[j] = w[j];
    __syncthreads();
  }
  const int lo = p.sink, hi = len - p.recent;  // (sink + recent <= keep < len)
  const int want = keep - p.sink - p.recent;
  uint32_t key = 0xFFFFFFFFu;
  int equals = 0;
  if (want > 0) {
    if (held) select_key([&](int j) { return s.w[j]; }, lo, hi, want, s, key, equals);
    else select_key([&](int j) { return w[j]; }, lo, hi, want, s, key, equals);
  }

  constexpr int kLanes = D / 8, kTokens = kThreads / kLanes, kGroup = kTokens * kAhead;
  static_assert(kGroup <= 512, "what is left in the ring");
  const int c = tid % kLanes, g = tid / kLanes;
  const int64_t base = layer * p.pool.layer_stride + head * p.pool.head_stride + c * 8;
  const int32_t* from = p.table_in + static_cast<int64_t>(row) * p.width;
  const int32_t* to = p.table + static_cast<int64_t>(row) * p.width;
  const int page_mask = (1 << p.page_shift) - 1;
  int done = 0, found = 0;  // tokens moved, and found
  int ties = 0;             // equals of the key so far
  // tokens done .. done + kGroup - 1 (those found): read, then written
  auto move = [&]() {
    uint4 k[kAhead], v[kAhead];
    int64_t dst[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int d = done + i * kTokens + g;
      dst[i] = -1;
      if (d < found) {
        const int slot = s.slot[d % kRing], page = s.page[d % kRing];
        const int page2 = to[d >> p.page_shift];
        if (page >= 0) {  // (read before it is known whether it stays where it is: the lookup takes as long)
          const int64_t at = base + page * p.pool.page_stride + (slot & page_mask) * p.pool.token_stride;
          k[i] = *reinterpret_cast<const uint4*>(p.pool.k + at);
          v[i] = *reinterpret_cast<const uint4*>(p.pool.v + at);
        }
        if (page2 < 0 || page2 >= p.pages) atomicOr(p.err, kErrBadShape);
        else if (page >= 0 && (slot != d || page != page2))
          dst[i] = base + page2 * p.pool.page_stride + (d & page_mask) * p.pool.token_stride;
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
  // a thread's four slots of a run and their page (pages hold at least 16 slots)
  auto load = [&](int j0, float (&x)[kPer], int& page) {
    const int j = j0 + tid * kPer;
    page = -1;
    if (j < len) page = from[j >> p.page_shift];
#pragma unroll
    for (int i = 0; i < kPer; ++i) x[i] = j + i < len ? (held ? s.w[j + i] : w[j + i]) : 0.f;
  };
  uint32_t turn = 0;
  float next[kPer];
  int next_page;
  load(0, next, next_page);
  for (int j0 = 0; j0 < len; j0 += kRun) {
    float x[kPer];
    int page = next_page;
#pragma unroll
    for (int i = 0; i < kPer; ++i) x[i] = next[i];
    if (j0 + kRun < len) load(j0 + kRun, next, next_page);  // (no token of this run moves there)
    if (j0 + tid * kPer < len && (page < 0 || page >= p.pages)) {
      atomicOr(p.err, kErrBadShape);
      page = -1;
    }
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
      if ((pair[i] & 1u) || (pair[i] && tie < equals)) {
        const int d = found + static_cast<int>(before & 0xFFFFu) + min(tie, equals) - min(ties, equals);
        s.slot[d % kRing] = j;
        s.page[d % kRing] = page;
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

template <int D, int kThreads>
cudaError_t launch_dim(const EvictParams& p, cudaStream_t st) {
  static KernelSetup setup;
  constexpr size_t kSmem = sizeof(Shared<kThreads>);
  cudaError_t e = kernel_setup(setup, evict_kernel<D, kThreads>, kThreads, kSmem);
  if (e != cudaSuccess) return e;
  const int64_t units = static_cast<int64_t>(p.nseq) * p.pool.layers * p.pool.kv_heads;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(units));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, evict_kernel<D, kThreads>, p);
}

}  // namespace

cudaError_t launch_evict_tokens(const EvictParams& p, cudaStream_t st) {
  constexpr int kT = 512;
  switch (p.pool.dim) {
    case 64: return launch_dim<64, kT>(p, st);
    case 128: return launch_dim<128, kT>(p, st);
    default: return launch_dim<256, kT>(p, st);
  }
}

}  // namespace exl3
