// exl3_pages.cu -- the pages of the key/value cache: fork / reorder / free, grow with copy on write, compaction, and
// keeping a drafted tree's accepted path.
//
// The bookkeeping (reference counts, tables) is a few hundred kilobytes of whole numbers with dependent steps -- count,
// scan, assign -- so one thread-block cluster does it in one launch, its CTAs joined by the cluster barrier between the
// steps; a single launch of eight CTAs costs less than the launches a grid would need.  Everything is decided by ranks
// (the n-th lowest free page, the n-th row that asks), never by the order in which threads arrive.  The pages'
// contents then move in a second launch over the whole GPU, bound by HBM: every moved byte read and written once
// (compaction of 2.3 GB in 36 layers: 393 us, 6.0 TB/s; a fork to 48 rows and their growth with copies: 27 us in a graph, 33
// a pair of calls).
#include <cuda_runtime.h>

#include "exl3_attn.h"
#include "exl3_common.cuh"
#include "exl3_internal.h"

namespace exl3 {

namespace {

constexpr int kCluster = 8;
constexpr int kThreads = 1024;
constexpr int kAll = kCluster * kThreads;
constexpr int kMaxGrowRows = 4096;  // rows of a grow call (their asks are scanned in shared memory)

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}

// Shared word w of CTA `rank` of the cluster.
__device__ __forceinline__ int cluster_word(const int* w, int rank) {
  uint32_t a;
  int v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(w)), "r"(rank));
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}

// The cluster's pages cut into one run per CTA, a run into one part per thread: [lo, hi).
struct PageRun {
  int lo, hi;
  __device__ __forceinline__ explicit PageRun(int pages) {
    const int64_t t = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
    lo = static_cast<int>(t * pages / kAll), hi = static_cast<int>((t + 1) * pages / kAll);
  }
};

// Exclusive rank of this thread's `n` in the cluster (CTA by CTA, thread by thread) and the cluster's total.
// s_total: one shared word that nothing else writes until the next cluster_sync.
__device__ __forceinline__ int cluster_scan_excl(int n, int* s_warp, int* s_total, int* total) {
  int mine;
  const int r = cta_scan_excl(n, s_warp, &mine);
  if (threadIdx.x == 0) *s_total = mine;
  cluster_sync();
  int before = 0, all = 0;
  for (int c = 0; c < kCluster; ++c) {
    const int v = cluster_word(s_total, c);
    if (c < static_cast<int>(blockIdx.x)) before += v;
    all += v;
  }
  *total = all;
  return before + r;
}

// A row's pages, held inside the table whatever the device value is.
__device__ __forceinline__ int held_of(const PageParams& p, int r) { return max(0, min(p.held_in[r], p.width_in)); }

// ------------------------------------------------------------------ fork / reorder / free

__global__ void __cluster_dims__(kCluster, 1, 1) __launch_bounds__(kThreads) fork_kernel(const PageParams p) {
  pdl_wait();
  const int t = static_cast<int>(blockIdx.x) * kThreads + static_cast<int>(threadIdx.x);
  const int lane = t & 31, warp = t >> 5;
  for (int i = t; i < p.pages; i += kAll) p.refs[i] = p.refs_in[i];
  for (int r = warp; r < p.nseq_out; r += kAll / 32) {
    int from = p.parent[r];
    if (from < -1 || from >= p.nseq_in) {
      if (lane == 0) atomicOr(p.err, kErrBadShape);
      from = -1;
    }
    const int held = from < 0 ? 0 : max(0, min(p.held_in[from], p.width_in));
    if (lane == 0) p.held[r] = held, p.lens[r] = from < 0 ? 0 : p.lens_in[from];
    const int64_t src = static_cast<int64_t>(from) * p.width_in, dst = static_cast<int64_t>(r) * p.width_out;
    for (int j = lane; j < p.width_out; j += 32) p.table[dst + j] = j < held ? p.table_in[src + j] : -1;
  }
  cluster_sync();  // the copied counts are in place
  for (int r = warp; r < p.nseq_in; r += kAll / 32) {
    int children = 0;
    for (int j = lane; j < p.nseq_out; j += 32) children += p.parent[j] == r ? 1 : 0;
    children = __reduce_add_sync(0xFFFFFFFFu, children);
    if (children == 1) continue;
    const int held = held_of(p, r);
    for (int j = lane; j < held; j += 32) {
      const int id = p.table_in[static_cast<int64_t>(r) * p.width_in + j];
      if (id >= 0 && id < p.pages) atomicAdd(p.refs + id, children - 1);  // (whole numbers: any order)
      else atomicOr(p.err, kErrBadShape);
    }
  }
}

// ------------------------------------------------------------------ grow

// The table places whose pages row r writes: those of the slots len .. need - 1, as far as it holds them.
struct Writes {
  int lo = 0, hi = 0;   // [lo, hi)
  int len, held, want;  // the row's tokens and pages, the pages it needs (at most the table's width)
  int over;             // pages it needs past that
  int id;               // the page at place lo + lane, or -1
  bool shared;          // it has several references
  Writes() = default;
  __device__ __forceinline__ Writes(const PageParams& p, int r, int lane) {
    const int page = 1 << p.page_shift, need = max(p.need[r], 0);
    len = p.lens_in[r], held = held_of(p, r);
    const int all = static_cast<int>((static_cast<int64_t>(need) + page - 1) >> p.page_shift);
    want = min(all, p.width_in), over = all - want;
    if (need > len && len >= 0) lo = min(len >> p.page_shift, held), hi = max(lo, min(want, held));
    place(p, r, lo + lane);
  }
  __device__ __forceinline__ void place(const PageParams& p, int r, int j) {
    id = j < hi ? p.table_in[static_cast<int64_t>(r) * p.width_in + j] : -1;
    if (j < hi && (id < 0 || id >= p.pages)) {
      atomicOr(p.err, kErrBadShape);
      id = -1;
    }
    shared = id >= 0 && p.refs_in[id] > 1;
  }
};

// A page with several references that a row writes is replaced in its table, by a copy where it holds tokens of the row:
// the page of slot len, and pages past it that the row held without needing them (provided for drafts that were rejected)
// when it was forked.  When every reference is a row's that writes the page, the first of these rows keeps it.
__global__ void __cluster_dims__(kCluster, 1, 1) __launch_bounds__(kThreads) grow_kernel(const PageParams p) {
  extern __shared__ int s_row[];  // [nseq + 1] asks before the row, copies before the row
  __shared__ int s_warp[32], s_total;
  int* s_ask = s_row;
  int* s_copy = s_row + p.nseq_in + 1;
  pdl_wait();
  const int tid = static_cast<int>(threadIdx.x);
  const int t = static_cast<int>(blockIdx.x) * kThreads + tid;
  const int lane = t & 31, warp = t >> 5;
  const int n = p.nseq_in, page = 1 << p.page_shift;
  int* asks = p.scratch;         // [nseq] pages each row asks for
  int* copies = asks + n;        // [nseq] of them, copies
  int* overs = copies + n;       // [nseq] pages past the table's width
  int* first = overs + n;        // [pages] of a shared page, the first row that writes it
  int* order = first + p.pages;  // [pages] the free pages in the order they are given
  // a warp takes every 256th row; the first one's places are read once, under the copies
  Writes own;
  if (warp < n) own = Writes(p, warp, lane);
  auto each_row = [&](auto&& f) {
    for (int r = warp; r < n; r += kAll / 32) {
      if (r == warp) {
        f(r, own);
      } else {
        Writes w(p, r, lane);
        f(r, w);
      }
    }
  };
  // f(its place, its 32 places begin at j0) for every place of the row, by lanes
  auto each_place = [&](int r, Writes w, auto&& f) {
    for (int j0 = w.lo; j0 < w.hi; j0 += 32) {
      if (j0 > w.lo) w.place(p, r, j0 + lane);
      f(w, j0);
    }
  };
  // counts and tables as they are, and the free pages ranked
  for (int i = t; i < p.pages; i += kAll) {
    const int refs = p.refs_in[i];
    p.refs[i] = refs;
    if (refs > 1) first[i] = n;
  }
  for (int64_t i = t; i < static_cast<int64_t>(n) * p.width_in; i += kAll) p.table[i] = p.table_in[i];
  const PageRun run(p.pages);
  int mine = 0, free_pages;
  for (int i = run.lo; i < run.hi; ++i) mine += p.refs_in[i] <= 0 ? 1 : 0;
  int rank = cluster_scan_excl(mine, s_warp, &s_total, &free_pages);  // (its barrier: the copies above are in place)
  // a shared page loses the references of the rows that write it (whole numbers: any order)
  each_row([&](int r, const Writes& w) {
    each_place(r, w, [&](const Writes& at, int) {
      if (at.shared) atomicSub(p.refs + at.id, 1), atomicMin(first + at.id, r);
    });
  });
  cluster_sync();
  auto replaced = [&](int r, const Writes& at) {
    return at.shared && (__ldcg(first + at.id) != r || __ldcg(p.refs + at.id) > 0);
  };
  each_row([&](int r, const Writes& w) {
    int ask = max(0, w.want - w.held), copy = 0;
    each_place(r, w, [&](const Writes& at, int j0) {
      const uint32_t which = __ballot_sync(0xFFFFFFFFu, replaced(r, at));
      ask += __popc(which);
      if (j0 == w.lo && (w.len & (page - 1))) copy = which & 1u;
    });
    if (lane == 0) asks[r] = ask, copies[r] = copy, overs[r] = w.over, p.lens[r] = w.len;
  });
  cluster_sync();
  int asked = 0, copied = 0, over = 0;  // every CTA: rows are scanned in runs of kThreads
  for (int base = 0; base < n; base += kThreads) {
    const int r = base + tid;
    int total;
    const int row_asks = r < n ? __ldcg(asks + r) : 0, row_copies = r < n ? __ldcg(copies + r) : 0;
    over |= r < n ? __ldcg(overs + r) : 0;
    const int a = cta_scan_excl(row_asks, s_warp, &total);
    if (r < n) s_ask[r] = asked + a;
    asked += total;
    const int c = cta_scan_excl(row_copies, s_warp, &total);
    if (r < n) s_copy[r] = copied + c;
    copied += total;
  }
  int missing = max(0, asked - free_pages);
  if (__syncthreads_or(over)) {  // (rare) the pages past the width, held below 2^31
    int64_t sum = missing;
    for (int r = 0; r < n; ++r) sum += __ldcg(overs + r);
    missing = static_cast<int>(min(sum, static_cast<int64_t>(0x7FFFFFFF)));
  }
  if (t == 0) {
    p.missing[0] = missing;
    p.moves[0] = missing ? 0 : copied;
  }
  if (missing) {
    for (int i = t; i < p.pages; i += kAll) p.refs[i] = p.refs_in[i];
  } else {
    for (int i = run.lo; i < run.hi && rank < asked; ++i)
      if (p.refs_in[i] <= 0) order[rank++] = i;
  }
  cluster_sync();  // (and no CTA leaves while another may read its shared words)
  each_row([&](int r, const Writes& w) {
    if (lane == 0) p.held[r] = missing ? w.held : max(w.held, w.want);
    if (missing) return;
    int32_t* row = p.table + static_cast<int64_t>(r) * p.width_in;
    int next = s_ask[r];  // the row's next page in `order`
    each_place(r, w, [&](const Writes& at, int j0) {
      const bool goes = replaced(r, at);
      const uint32_t which = __ballot_sync(0xFFFFFFFFu, goes);
      if (goes) {
        const int to = __ldcg(order + next + __popc(which & ((1u << lane) - 1u)));
        row[j0 + lane] = to;
        p.refs[to] = 1;
        if (j0 + lane == w.lo && (w.len & (page - 1)))
          p.moves[1 + 2 * s_copy[r]] = at.id, p.moves[2 + 2 * s_copy[r]] = to;
      } else if (at.shared) {
        p.refs[at.id] = 1;  // kept by the first of its rows (no other row's test reads this count)
      }
      next += __popc(which);
    });
    for (int j = w.held + lane; j < w.want; j += 32) {
      const int to = __ldcg(order + next + j - w.held);
      row[j] = to;
      p.refs[to] = 1;
    }
  });
}

// ------------------------------------------------------------------ compact

// scratch: [2 * pages] after the moves: the live pages by their rank, then the free pages below the live count by theirs
__global__ void __cluster_dims__(kCluster, 1, 1) __launch_bounds__(kThreads) compact_kernel(const PageParams p) {
  __shared__ int s_warp[32], s_total, s_holes;
  pdl_wait();
  int* by_rank = p.moves + 1 + 2 * static_cast<int64_t>(p.pages);
  int* holes = by_rank + p.pages;
  const int t = static_cast<int>(blockIdx.x) * kThreads + static_cast<int>(threadIdx.x);
  const PageRun run(p.pages);
  int mine = 0, live;
  for (int i = run.lo; i < run.hi; ++i) mine += p.refs_in[i] > 0 ? 1 : 0;
  const int before = cluster_scan_excl(mine, s_warp, &s_total, &live);
  // live page of rank k moves to hole k - (live - holes): the last `holes` live pages are the ones at `live` and above
  int rank = before, found = 0;
  for (int i = run.lo; i < run.hi; ++i) {
    if (p.refs_in[i] > 0) by_rank[rank++] = i;
    else if (i < live) holes[i - rank] = i, ++found;
  }
  int holes_mine;
  cta_scan_excl(found, s_warp, &holes_mine);
  if (threadIdx.x == 0) s_holes = holes_mine;
  cluster_sync();
  int moves = 0;
  for (int c = 0; c < kCluster; ++c) moves += cluster_word(&s_holes, c);
  if (t == 0) p.moves[0] = moves;
  for (int i = t; i < moves; i += kAll) {
    p.moves[1 + 2 * i] = __ldcg(by_rank + live - moves + i);
    p.moves[2 + 2 * i] = __ldcg(holes + i);
  }
  for (int i = t; i < p.pages; i += kAll) {
    int v = 0;
    if (i < live) v = p.refs_in[i] > 0 ? p.refs_in[i] : -1;
    if (v >= 0) p.refs[i] = v;
  }
  for (int i = t; i < moves; i += kAll) p.refs[__ldcg(holes + i)] = p.refs_in[__ldcg(by_rank + live - moves + i)];
  for (int r = t; r < p.nseq_in; r += kAll) p.held[r] = p.held_in[r], p.lens[r] = p.lens_in[r];
  for (int64_t i = t; i < static_cast<int64_t>(p.nseq_in) * p.width_in; i += kAll) {
    int id = p.table_in[i];
    if (id >= live && id < p.pages) {
      // its place among the movers: by_rank[live - moves ..] ascends
      int lo = live - moves, hi = live;
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (__ldcg(by_rank + mid) <= id) lo = mid;
        else hi = mid;
      }
      const bool found_it = moves > 0 && __ldcg(by_rank + lo) == id;
      if (!found_it) atomicOr(p.err, kErrBadShape);  // a table names a page with no references
      else id = __ldcg(holes + (lo - (live - moves)));
    } else if (id >= p.pages) {
      atomicOr(p.err, kErrBadShape);
    }
    p.table[i] = id < 0 ? -1 : id;
  }
  cluster_sync();  // no CTA leaves while another may read its shared words
}

// ------------------------------------------------------------------ page contents

constexpr int kCopyThreads = 256;
constexpr int kCopyPer = 8;  // 16-byte chunks a thread has in flight
constexpr int kCopyUnit = kCopyThreads * kCopyPer;

__global__ void __launch_bounds__(kCopyThreads) page_copy_kernel(const PagePool pool, const int32_t* moves) {
  pdl_wait();
  const int count = moves[0];
  const int dshift = 31 - __clz(pool.dim / 8), pshift = 31 - __clz(pool.page_size);
  const int chunks = pool.kv_heads << (pshift + dshift);  // of one page, one layer, k or v
  const int units = (chunks + kCopyUnit - 1) / kCopyUnit;
  const int64_t total = static_cast<int64_t>(count) * pool.layers * 2 * units;
  for (int64_t u = blockIdx.x; u < total; u += gridDim.x) {
    const int part = static_cast<int>(u % units);
    int64_t rest = u / units;
    uint16_t* base = (rest & 1) ? pool.v : pool.k;
    rest >>= 1;
    base += (rest % pool.layers) * pool.layer_stride;
    const int64_t m = rest / pool.layers;
    const uint16_t* src = base + moves[1 + 2 * m] * pool.page_stride;
    uint16_t* dst = base + moves[2 + 2 * m] * pool.page_stride;
    uint4 v[kCopyPer];
    int64_t off[kCopyPer];
#pragma unroll
    for (int i = 0; i < kCopyPer; ++i) {
      const int c = part * kCopyUnit + i * kCopyThreads + static_cast<int>(threadIdx.x);
      const int row = c >> dshift;
      off[i] = c < chunks ? (row >> pshift) * pool.head_stride + (row & (pool.page_size - 1)) * pool.token_stride +
                                (c & ((1 << dshift) - 1)) * 8
                          : -1;
      if (off[i] >= 0) v[i] = *reinterpret_cast<const uint4*>(src + off[i]);
    }
#pragma unroll
    for (int i = 0; i < kCopyPer; ++i)
      if (off[i] >= 0) *reinterpret_cast<uint4*>(dst + off[i]) = v[i];
  }
}

// ------------------------------------------------------------------ keep a path

constexpr int kKeepThreads = 256;
constexpr int kKeepBatch = 8;  // tokens read before any of them is written

// One thread per (16-byte chunk of a head, kv head, k or v, layer) of one sequence (blockIdx.y): it walks the path.  The
// path ascends, so path[d] >= d, and a slot is never read after a later token was written to it.  lens may be context or kept
// (a loop's lengths kept in place): lens[s] is then written by the sequence's last block to have read them.  The count takes
// 2 us of 16 (32 trees, 36 layers); lengths apart from both are written at once.
__global__ void __launch_bounds__(kKeepThreads) keep_kernel(const KeepParams p) {
  pdl_wait();
  const int s = p.seq0 + static_cast<int>(blockIdx.y);
  const int ctx = p.b.context[s];
  const int ntok = max(0, min(p.b.row_start[s + 1], p.b.rows) - max(p.b.row_start[s], 0));
  int kept = p.kept[s];
  bool ok = ctx >= 0 && kept >= 0 && kept <= ntok && (!p.path || kept <= p.depth);
  const int64_t room = static_cast<int64_t>(p.b.max_pages) << p.b.page_shift;
  if (ok && static_cast<int64_t>(ctx) + ntok > room) ok = false;
  const int32_t* path = p.path ? p.path + static_cast<int64_t>(s) * p.depth : nullptr;
  if (ok && path) {
    for (int d = 0; d < kept; ++d) {
      const int a = path[d];
      if (a >= ntok || a < (d ? path[d - 1] + 1 : 0)) ok = false;
    }
  }
  const int64_t item = static_cast<int64_t>(blockIdx.x) * kKeepThreads + threadIdx.x;
  if (!ok) kept = 0;
  bool last = item == 0;
  if (p.counters) {
    __syncthreads();  // the block's reads of context and kept are done
    last = false;
    if (threadIdx.x == 0) {
      __threadfence();
      last = atomicAdd(p.counters + blockIdx.y, 1u) + 1u == gridDim.x;
      __threadfence();
      if (last) p.counters[blockIdx.y] = 0u;
    }
  }
  if (last) {
    p.lens[s] = max(ctx, 0) + kept;
    if (!ok) atomicOr(p.b.err, kErrBadShape);
  }
  if (!path) return;
  const int per = p.pool.dim / 8;
  const int c = static_cast<int>(item % per);
  int64_t rest = item / per;
  const int h = static_cast<int>(rest % p.pool.kv_heads);
  rest /= p.pool.kv_heads;
  const bool is_v = (rest & 1) != 0;
  const int64_t layer = rest >> 1;
  if (layer >= p.pool.layers) return;
  uint16_t* base = (is_v ? p.pool.v : p.pool.k) + layer * p.pool.layer_stride + h * p.pool.head_stride + c * 8;
  const int32_t* tab = p.b.table + static_cast<int64_t>(s) * p.b.max_pages;
  const int mask = (1 << p.b.page_shift) - 1;
  auto slot = [&](int at) -> int64_t {
    const int id = tab[at >> p.b.page_shift];
    if (id < 0 || id >= p.b.pages) {
      atomicOr(p.b.err, kErrBadShape);
      return -1;
    }
    return id * p.b.page_stride + (at & mask) * p.b.token_stride;
  };
  for (int d0 = 0; d0 < kept; d0 += kKeepBatch) {
    uint4 v[kKeepBatch];
    int64_t to[kKeepBatch];
#pragma unroll
    for (int i = 0; i < kKeepBatch; ++i) {
      const int d = d0 + i;
      to[i] = -1;
      if (d < kept && path[d] != d) {
        const int64_t from = slot(ctx + path[d]);
        to[i] = slot(ctx + d);
        if (from < 0) to[i] = -1;
        if (to[i] >= 0) v[i] = *reinterpret_cast<const uint4*>(base + from);
      }
    }
#pragma unroll
    for (int i = 0; i < kKeepBatch; ++i)
      if (to[i] >= 0) *reinterpret_cast<uint4*>(base + to[i]) = v[i];
  }
}

template <typename Kern>
cudaError_t launch_cluster(Kern kern, size_t smem, cudaStream_t st, const PageParams& p) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(kCluster);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, p);
}

}  // namespace

int cache_grow_max_rows() { return kMaxGrowRows; }

cudaError_t launch_cache_fork(const PageParams& p, cudaStream_t st) { return launch_cluster(fork_kernel, 0, st, p); }

cudaError_t launch_cache_grow(const PageParams& p, cudaStream_t st) {
  static KernelSetup setup;
  const size_t smem = (static_cast<size_t>(p.nseq_in) + 1) * 2 * sizeof(int);
  cudaError_t e = kernel_setup(setup, grow_kernel, kThreads, (static_cast<size_t>(kMaxGrowRows) + 1) * 2 * sizeof(int));
  if (e != cudaSuccess) return e;
  return launch_cluster(grow_kernel, smem, st, p);
}

cudaError_t launch_cache_compact(const PageParams& p, cudaStream_t st) {
  return launch_cluster(compact_kernel, 0, st, p);
}

cudaError_t launch_page_copy(const PagePool& pool, const int32_t* moves, int64_t max_moves, int sms, cudaStream_t st) {
  const int64_t units = (static_cast<int64_t>(pool.kv_heads) * pool.page_size * pool.dim / 8 + kCopyUnit - 1) / kCopyUnit;
  int64_t grid = max_moves * pool.layers * 2 * units;
  if (grid > static_cast<int64_t>(sms) * 8) grid = static_cast<int64_t>(sms) * 8;
  if (grid < 1) return cudaSuccess;
  return launch_pdl_k(page_copy_kernel, dim3(static_cast<unsigned>(grid)), dim3(kCopyThreads), st, pool, moves);
}

cudaError_t launch_cache_keep(const KeepParams& p, uint32_t counters, cudaStream_t st) {
  const int64_t items = p.path ? static_cast<int64_t>(p.pool.layers) * 2 * p.pool.kv_heads * (p.pool.dim / 8) : 1;
  KeepParams part = p;
  const int most = p.counters ? static_cast<int>(counters) : p.b.nseq;  // sequences of a launch
  for (part.seq0 = 0; part.seq0 < p.b.nseq; part.seq0 += most) {
    const int left = p.b.nseq - part.seq0;
    const dim3 grid(static_cast<unsigned>((items + kKeepThreads - 1) / kKeepThreads), static_cast<unsigned>(left < most ? left : most));
    cudaError_t e = launch_pdl_k(keep_kernel, grid, dim3(kKeepThreads), st, part);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

}  // namespace exl3
