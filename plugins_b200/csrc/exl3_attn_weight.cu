// exl3_attn_weight.cu -- how much every cached token was attended to: the column sums of the attention's probabilities,
// accumulated over steps (exl3_attention_weight, include/exl3_b200.h), on the 5th-generation tensor cores.
//
//   w[s][g][j] = (j < context ? decay w[s][g][j] : 0) + sum_i sum_{h in g} exp(scale q_ih . k_j - lse_ih)
//
// over the rows i of sequence s that see slot j.  The log-sum-exps are given, so a slot's sum needs nothing of the other
// slots: S^T = K Q^T with the keys as the MMA's M dimension puts a key on a TMEM lane and hence in one thread, which sums its
// probabilities over the columns (rows of Q) with no exchange; each thread's own f32 sum runs over its columns in order.
//
// The work: (sequence, kv head, block of keys) items, an item's tiles its query row tiles, all items' tiles on one line cut
// into equal parts, one per CTA.  An item's keys stay in shared memory while the row tiles stream by; where a sequence has
// one row tile (decoding, small trees) that stays, and the keys stream.  An item cut between CTAs is joined by the last of
// them to finish, its partial sums added in the line's order: the bits do not depend on which CTA that is.
//
// Roles: four groups of four warps for the exponentials and sums (a thread per key), then one warp each for the MMAs and the
// copies of K (TMA, one box per page and 64 columns, 128-byte swizzle) and of the query rows (row t * group + g is token t's
// query head g: a box of the kv head's query heads by tokens).  Queries whose addresses TMA does not take, or with more heads
// per kv head than a tile has rows, are brought by two warps instead.  Heads up to 128 wide: an item is 256 keys, two groups per half
// that take its row tiles by turns.  256 wide: 128 keys, all four by turns.
//
// A quarter of the exponentials are polynomials on the FMA pipe, beside the special-function unit (4096 rows on 4096 slots, an
// eighth / a quarter / half of them: 245 / 235 / 271 us; a step earlier none took 265 where a quarter took 256).
//
// What bounds it: few rows, HBM (32 sequences' tokens over 1.5-9k slots 65 us in a graph, 5.4 TB/s; nine trees of 5-17 rows over
// 6-16k 256-wide slots 72 us, 5.8 TB/s), the rest being the start and the line's cut.  Many rows, no one unit: a 4096-row chunk
// on 4096 slots takes 238 us at 1965 MHz (0.87 PFLOP/s, against 127 us of products), its schedulers issue in 62 % of the active
// cycles, the special-function unit is busy for 64 % and the tensor pipe for 43 %, and of a warp's 8.1 cycles an instruction
// 2.0 are on the long scoreboard, 1.3 a fixed latency, 0.9 another warp's issue and 0.8 at barriers; the SMs are active for
// 88 % of it.  Called for longer than a few hundred milliseconds it draws the card's 1000 W, which clocks it
// at about 1790 MHz: 263 us.  Two groups of summing warps took 256 us (of 232 then) where four took 253; fetching the
// log-sum-exps a tile ahead then brought 233; passing every tile's publication (lfull), which order needs, costs 2 %.
//
// Every mbarrier wait is bounded (wait_bar): one that gives up raises an abort flag that all roles poll.  A weight is then
// written whole or not at all, and the counters of the items that the CTA shares return to zero (exl3_parts.h).
#include <cuda.h>
#include <cuda_runtime.h>

#include "exl3_attn.h"
#include "exl3_attn_dev.cuh"
#include "exl3_attn_tc.cuh"
#include "exl3_common.cuh"
#include "exl3_internal.h"
#include "exl3_parts.h"

namespace exl3 {

using namespace tc;

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kPolyEvery = 8;  // one pair of this many numbers takes the FMA pipe

template <int D, bool FEW>
struct WtShape {
  static constexpr int HB = D == 256 ? 1 : 2;       // 128-key halves of an item
  static constexpr int KB = HB * 128;               // keys of an item
  static constexpr int RT = FEW ? 32 : D == 256 ? 64 : 128;  // query rows of a tile
  static constexpr int kBufs = D == 256 ? 4 : 2;    // accumulators of a half
  static constexpr int kKTile = 128 * D * 2;
  static constexpr int kQTile = RT * D * 2;
  static constexpr int QS = FEW && D == 256 ? 1 : D == 64 ? 3 : 2;                         // query tiles in flight
  static constexpr int KS = FEW ? (D == 256 ? 3 : D == 128 ? 6 : 12) : D == 256 ? 2 : D == 128 ? 4 : 6;  // K halves
  static constexpr int LS = 4;                      // log-sum-exps of query tiles: used later than the tiles themselves
  static constexpr int kEpi = 512;                  // threads of the sums: four groups of four warps
  static constexpr int GH = 4 / HB;                 // groups of a half, which take its tiles by turns
  static constexpr int kLoad = 64;                  // threads that bring the queries
  static constexpr int kThreads = kEpi + 64 + kLoad;
  static constexpr int kTmem = D == 256 ? 256 : 512;
  static constexpr int kBars = 2 * KS + 2 * QS + 2 * LS + 2 * HB * kBufs + 2;
  static constexpr int kSmem = KS * kKTile + QS * kQTile + LS * RT * 4 + 2 * 3 * 128 * 4 + kBars * 8 + 64;
  static_assert(HB * kBufs * RT <= kTmem && kSmem <= 232448 - 2048, "shared memory or TMEM");
};

// A block of keys of one sequence and kv head, with the row tiles that see any of it.
struct WtItem {
  Item s;                  // the sequence (item_seq) and kv head
  int block, nblocks;
  int row_tiles;           // of the sequence
  int first_tile, tiles;   // the block's: first_tile .. row_tiles - 1
  int64_t first;           // its first tile on the line
};

template <int D, bool FEW>
struct WtLine : WorkLine {
  using S = WtShape<D, FEW>;
  __device__ __forceinline__ static void set_seq(const WeightParams& p, WtItem& it) {
    if (it.s.total_keys > p.slots) atomicOr(p.a.b.err, kErrBadShape);
    it.s.total_keys = min(it.s.total_keys, p.slots);
    it.s.context = min(it.s.context, it.s.total_keys);
    it.nblocks = it.s.nrows ? (it.s.total_keys + S::KB - 1) / S::KB : 0;
    it.row_tiles = (it.s.nrows + p.row_tile - 1) / p.row_tile;
  }
  // The first row tile that sees any key of the block: without a tree, slot context + d is seen from token d on.
  __device__ __forceinline__ static int first_of(const WeightParams& p, const WtItem& it, int block) {
    const int d = block * S::KB - it.s.context;
    return p.a.b.tree || d <= 0 ? 0 : static_cast<int>(divide(static_cast<int64_t>(d) * p.a.group, p.row_tile));
  }
  __device__ __forceinline__ static void set_block(const WeightParams& p, WtItem& it) {
    it.first_tile = it.row_tiles == 1 ? 0 : first_of(p, it, it.block);
    it.tiles = it.row_tiles - it.first_tile;
  }
  __device__ __forceinline__ static int64_t tiles_of_head(const WeightParams& p, const WtItem& it) {
    int64_t t = static_cast<int64_t>(it.nblocks) * it.row_tiles;
    if (p.a.b.tree || it.row_tiles == 1) return t;
    // first_of for the blocks past the context, kept as quotient and remainder
    int b = it.s.context / S::KB + 1;
    const int64_t x = (static_cast<int64_t>(b) * S::KB - it.s.context) * p.a.group;
    int64_t q = divide(x, p.row_tile);
    int r = static_cast<int>(x - q * p.row_tile);
    const int dq = S::KB * p.a.group / p.row_tile, dr = S::KB * p.a.group % p.row_tile;
    for (; b < it.nblocks; ++b) {
      t -= q;
      q += dq, r += dr;
      if (r >= p.row_tile) ++q, r -= p.row_tile;
    }
    return t;
  }
  __device__ __forceinline__ int64_t seq_tiles(const WeightParams& p, int s) const {
    if (s >= p.a.b.nseq) return 0;
    WtItem it;
    item_seq(p.a, s, it.s);
    set_seq(p, it);
    return tiles_of_head(p, it) * p.a.b.kv_heads;
  }
  // Cuts the line and finds the item that holds this CTA's first tile (if it has any).  scratch: 36 words.
  __device__ void begin_line(const WeightParams& p, int64_t* scratch, WtItem& it) {
    int64_t sum = 0, mine = 0, upto = 0;
    for (int base = 0; base < p.a.b.nseq; base += blockDim.x) {
      mine = seq_tiles(p, base + static_cast<int>(threadIdx.x));
      upto = sum + scan(mine, scratch);
      if (threadIdx.x == blockDim.x - 1) scratch[33] = upto;
      __syncthreads();
      sum = scratch[33];
      __syncthreads();
    }
    total = sum;
    parts = static_cast<int>(min(static_cast<int64_t>(gridDim.x), total));
    begin = end = 0;
    if (static_cast<int>(blockIdx.x) >= parts) return;
    share = divide(total, parts);
    extra = static_cast<int>(total - share * parts);
    const int c = static_cast<int>(blockIdx.x);
    begin = share * c + min(c, extra);
    end = begin + share + (c < extra ? 1 : 0);
    const bool one = p.a.b.nseq <= static_cast<int>(blockDim.x);  // the scan above is the whole
    sum = 0;
    for (int base = 0; base < p.a.b.nseq; base += blockDim.x) {
      const int s = base + static_cast<int>(threadIdx.x);
      if (!one) {
        mine = seq_tiles(p, s);
        upto = sum + scan(mine, scratch);
      }
      if (threadIdx.x == blockDim.x - 1) scratch[33] = upto;
      if (begin < upto && begin >= upto - mine) scratch[34] = s, scratch[35] = upto - mine;
      __syncthreads();
      sum = scratch[33];
      if (begin < sum) break;
      __syncthreads();
    }
    const int s = static_cast<int>(scratch[34]);
    const int64_t first = scratch[35];
    __syncthreads();
    item_seq(p.a, s, it.s);
    set_seq(p, it);
    const int64_t per_head = tiles_of_head(p, it);
    it.s.kv_head = static_cast<int>(divide(begin - first, per_head));
    it.first = first + it.s.kv_head * per_head;
    // the blocks that begin in the context have all row tiles
    const int whole = p.a.b.tree ? it.nblocks : min(it.nblocks, it.s.context / S::KB + 1);
    it.block = static_cast<int>(min(divide(begin - it.first, it.row_tiles), static_cast<int64_t>(whole - 1)));
    it.first += static_cast<int64_t>(it.block) * it.row_tiles;
    set_block(p, it);
    while (begin >= it.first + it.tiles) {
      it.first += it.tiles;
      ++it.block;
      set_block(p, it);
    }
  }
  // The item after `it` (there is one).
  __device__ __forceinline__ static void step(const WeightParams& p, WtItem& it) {
    it.first += it.tiles;
    if (++it.block < it.nblocks && it.row_tiles == 1) return;  // (its one tile)
    if (it.block == it.nblocks) {
      it.block = 0;
      if (++it.s.kv_head == p.a.b.kv_heads) {
        it.s.kv_head = 0;
        int s = it.s.seq;
        do item_seq(p.a, ++s, it.s);
        while (it.s.ntok == 0 && s + 1 < p.a.b.nseq);
        set_seq(p, it);
      }
    }
    set_block(p, it);
  }
};

// Which of the rows row0 .. row0 + 31 of the sequence (row t * group + g: token t) see slot context + d (d >= 0).
__device__ __forceinline__ uint32_t seeing32(const WeightParams& p, const Item& it, int row0, int d) {
  if (!p.a.b.tree) {
    const int64_t n = static_cast<int64_t>(d) * p.a.group - row0;  // the first that does
    return n <= 0 ? ~0u : n >= 32 ? 0u : ~0u << n;
  }
  const int word = d >> 5;
  if (word >= p.a.b.tree_words) return 0u;
  uint32_t m = 0;
  int t = row0 / p.a.group, next = (t + 1) * p.a.group - row0;
  for (int i = 0; i < 32; ++t) {
    const uint32_t bit = t < it.ntok ? (p.a.b.tree[static_cast<int64_t>(it.row0 + t) * p.a.b.tree_words + word] >> (d & 31)) & 1u : 0u;
    const int to = min(next, 32);
    if (bit) m |= (to == 32 ? ~0u : (1u << to) - 1u) & ~((1u << i) - 1u);
    i = to;
    next += p.a.group;
  }
  return m;
}

// 2^x of two numbers at most about 0 on the FMA pipe: x = n + f with |f| <= 1/2, a polynomial of degree 5 for 2^f (the
// minimax of its relative error, 7.5e-8, by Remez' exchange), times 2^n.  Below -125 exactly zero, NaN stays.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ uint64_t exp2_fma(float a, float b) {
  constexpr float kRound = 12582912.f;  // 1.5 x 2^23: what is added to it loses its fraction
  const uint64_t x = f2(max_nan(a, -125.f), max_nan(b, -125.f));
  const uint64_t t = add2(x, f2(kRound, kRound));
  const uint64_t f = fma2(add2(t, f2(-kRound, -kRound)), f2(-1.f, -1.f), x);
  uint64_t y = fma2(f2(0.0013276472f, 0.0013276472f), f, f2(0.00967554133f, 0.00967554133f));
  y = fma2(y, f, f2(0.0555071327f, 0.0555071327f));
  y = fma2(y, f, f2(0.240221197f, 0.240221197f));
  y = fma2(y, f, f2(0.693146967f, 0.693146967f));
  y = fma2(y, f, f2(1.00000007f, 1.00000007f));
  float t0, t1;
  f2_split(t, t0, t1);
  const float n0 = __uint_as_float((__float_as_uint(t0) << 23) + 0x3F800000u);  // 2^n (a NaN's is whatever it is)
  const float n1 = __uint_as_float((__float_as_uint(t1) << 23) + 0x3F800000u);
  constexpr float kLeast = 0x1p-125f * 1.00000007f;  // what x = -125 comes to
  return fma2(y, f2(n0, n1), f2(-kLeast, -kLeast));
}

// The sum of 2^(scale x - lse) over 32 accumulators; lse in shared memory, in units of log 2.
__device__ __forceinline__ void add32(const uint32_t (&x)[32], const float* lse, uint64_t scale2, uint64_t (&sum)[2]) {
#pragma unroll
  for (int i = 0; i < 32; i += 4) {
    const float4 l = *reinterpret_cast<const float4*>(lse + i);
    float a, b, c, d;
    f2_split(fma2(f2(__uint_as_float(x[i]), __uint_as_float(x[i + 1])), scale2, f2(l.x, l.y)), a, b);
    f2_split(fma2(f2(__uint_as_float(x[i + 2]), __uint_as_float(x[i + 3])), scale2, f2(l.z, l.w)), c, d);
    sum[0] = add2(sum[0], f2(ex2(a), ex2(b)));
    sum[1] = add2(sum[1], i % kPolyEvery == 0 ? exp2_fma(c, d) : f2(ex2(c), ex2(d)));
  }
}

// Counts a part of an item that is cut between CTAs c0 .. c1 -> whether it is the item's last and all have brought theirs.
__device__ __forceinline__ bool arrive_part(const WeightParams& p, int c0, int c1, bool brought) {
  const uint32_t n = atomicAdd(p.a.counters + c0, part_arrival(brought)) + part_arrival(brought);
  if (!parts_arrived(n, c1 - c0 + 1)) return false;
  p.a.counters[c0] = 0u;
  return parts_whole(n);
}

// A CTA that gave up still counts itself into the items it shares from tile `at` on, as one that brings nothing: their counters
// return to zero, and none of them is written.
template <int D, bool FEW>
__device__ __noinline__ void give_up(const WeightParams& p, const WtLine<D, FEW>& line, WtItem& it, int64_t at) {
  while (at < line.end) {
    while (at >= it.first + it.tiles) WtLine<D, FEW>::step(p, it);
    const int64_t to = min(line.end, it.first + it.tiles);
    if (to - at != it.tiles) arrive_part(p, line.part_of(it.first), line.part_of(it.first + it.tiles - 1), false);
    at = to;
  }
}

template <int D, bool FEW, bool BF16>
__global__ void __launch_bounds__(WtShape<D, FEW>::kThreads, 1)
    weight_kernel(const __grid_constant__ WeightParams p, const __grid_constant__ CUtensorMap kmap,
                  const __grid_constant__ CUtensorMap qmap) {
  using S = WtShape<D, FEW>;
  constexpr int HB = S::HB, KS = S::KS, QS = S::QS, LS = S::LS, RT = S::RT, kBufs = S::kBufs;
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ WtLine<D, FEW> line;
  __shared__ WtItem s_items[S::kThreads / 32];
  uint8_t* s_k = smem;                           // [slot][64-column block][128 keys][128 bytes], swizzled
  uint8_t* s_q = s_k + KS * S::kKTile;           // [slot][64-column block][RT rows][128 bytes], swizzled
  float* s_lse = reinterpret_cast<float*>(s_q + QS * S::kQTile);  // [slot][RT], negated, in units of log 2
  float* s_sums = s_lse + LS * RT;               // [2][3][128]: the other groups' sums, by turns
  uint64_t* bars = reinterpret_cast<uint64_t*>(s_sums + 768);
  uint64_t *kfull = bars, *kempty = kfull + KS, *qfull = kempty + KS, *qempty = qfull + QS, *lfull = qempty + QS;
  uint64_t *lempty = lfull + LS, *afull = lempty + LS, *aempty = afull + HB * kBufs, *xsync = aempty + HB * kBufs, *fin = xsync + 1;
  uint32_t* words = reinterpret_cast<uint32_t*>(bars + S::kBars);
  uint32_t* s_tmem = words;
  volatile uint32_t* abort_flag = words + 1;
  int* s_last = reinterpret_cast<int*>(words + 2);
  int64_t* s_counted = reinterpret_cast<int64_t*>(words + 4);  // the end of the last item this CTA has counted itself into
  const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
  const PagedBatch& b = p.a.b;

  if (smem_u32(smem) & 1023u) {  // the swizzle goes by address bits: not served
    if (tid == 0) atomicOr(b.err, kErrBadShape);
    return;
  }
  if (warp == 16) {
    tmem_alloc(smem_u32(s_tmem), S::kTmem);
    tmem_relinquish();
  }
  if (tid == 0) {
    for (int i = 0; i < KS; ++i) mbar_init(&kfull[i], 1), mbar_init(&kempty[i], 1);
    for (int i = 0; i < QS; ++i) mbar_init(&qfull[i], p.box_tokens ? 1 + 32 : S::kLoad), mbar_init(&qempty[i], 1);
    // The log-sum-exps' ring: every summing warp has seen a tile published before it releases it (lempty), by lfull, or by the
    // accumulators of a tile that it reads itself (their MMA waits for the same loader).  So a warp arrives once in a phase:
    // it cannot release tile n + LS before that is published, which the loader does not do before all sixteen have released
    // tile n; and neither side can be two phases ahead of the other, which a parity does not tell apart.
    for (int i = 0; i < LS; ++i) mbar_init(&lfull[i], p.box_tokens ? 32 : S::kLoad), mbar_init(&lempty[i], 16);
    for (int i = 0; i < HB * kBufs; ++i) mbar_init(&afull[i], 1), mbar_init(&aempty[i], 4);
    mbar_init(xsync, 16), mbar_init(fin, 1);
    fence_barrier_init();
    *abort_flag = 0u;
    *s_counted = 0;
  }
  if (tid == 32) asm volatile("prefetch.tensormap [%0];" ::"l"(&kmap) : "memory");
  if (tid == 64 && p.box_tokens) asm volatile("prefetch.tensormap [%0];" ::"l"(&qmap) : "memory");
  pdl_wait();
  {
    WtLine<D, FEW> own;
    WtItem first;
    own.begin_line(p, reinterpret_cast<int64_t*>(s_sums), first);  // (no place that TMA writes: that is another proxy)
    if (tid == 0) line = own;
    if (lane == 0) s_items[warp] = first;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *s_tmem;
  WtItem& it = s_items[warp];
  int64_t at = line.begin;
  const int64_t end = line.end;
  auto advance = [&](int tiles) {
    at += tiles;
    if (at < end) {
      __syncwarp();
      if (lane == 0) WtLine<D, FEW>::step(p, it);
      __syncwarp();
    }
  };
  // Whether the tile needs its queries brought: not where the sequence's one tile is there already.
  int held_seq = -1, held_head = -1;
  auto brings = [&]() {
    const bool there = it.row_tiles == 1 && it.s.seq == held_seq && it.s.kv_head == held_head;
    held_seq = it.s.seq, held_head = it.s.kv_head;
    return !there;
  };
  auto tiles_here = [&]() { return static_cast<int>(min(end - at, it.tiles - (at - it.first))); };
  auto first_here = [&]() { return it.first_tile + static_cast<int>(at - it.first); };
  auto halves_here = [&]() { return min(HB, (it.s.total_keys - it.block * S::KB + 127) / 128); };
  auto rows_of = [&](int tile) { return min(p.row_tile, it.s.nrows - tile * p.row_tile); };

  if (warp < 16) {
    // ---------------------------------------------------------------- exponentials and sums: a thread per key
    constexpr uint32_t GH = S::GH;
    const uint32_t g = warp >> 2, wq = warp & 3u, r128 = wq * 32 + lane;  // key of the half = TMEM lane
    const uint32_t lane_off = (wq * 32u) << 16;
    const int half = static_cast<int>(g / GH);
    const uint64_t scale2 = f2(p.a.scale_log2, p.a.scale_log2);
    uint32_t brought = 0, served = 0, x_phase = 0, turn = 0;  // query tiles so far; the half's tiles so far
    bool ok = true;
    auto group_sync = [&]() {  // all groups, none of which has given up
      __syncwarp();
      if (ok && lane == 0) mbar_arrive(xsync);
      ok = __all_sync(0xFFFFFFFFu, ok && wait_bar(xsync, x_phase, abort_flag, b.err));
      x_phase ^= 1u;
    };
    while (ok && at < end) {
      const int tiles = tiles_here(), tile0 = first_here(), halves = halves_here();
      const int key = it.block * S::KB + half * 128 + static_cast<int>(r128);
      const bool mine = half < halves;
      const bool solo = it.row_tiles == 1;  // its one tile's group has nobody to wait for
      const uint32_t writer = half * GH + (solo ? served % GH : 0u);
      const bool writes = mine && key < it.s.total_keys && g == writer;
      float* w = p.w + it.s.seq * p.row_stride + it.s.kv_head * p.head_stride + key;
      const bool keeps = writes && key < it.s.context && p.decay != 0.f;
      const float old = keeps ? __ldcg(w) : 0.f;
      const int d = key - it.s.context, d_last = d + 31 - static_cast<int>(lane);  // place among the new tokens; the warp's last
      const int nrows = it.s.nrows;
      const bool all = d_last < 0, by_place = !b.tree;
      // a sequence of one query tile may have it here already; those of more bring each
      bool bring = brings();
      int row0 = tile0 * p.row_tile;
      // The rows from `full` on see every key of the warp, those before `some` none, counted from the tile's first row.
      // (A call has at most 2^30 query vectors: a key's place times the group stays below 2^31.)
      int full = all ? -(1 << 30) : by_place ? d_last * p.a.group - row0 : 1 << 30;
      int some = all || !by_place ? -(1 << 30) : max(d_last - 31, 0) * p.a.group - row0;
      float total = 0.f;
      for (int i = 0; ok && i < tiles; ++i) {
        const int rows = min(p.row_tile, nrows - row0);
        if (bring) {
          if (brought && lane == 0) mbar_arrive(&lempty[(brought - 1) % LS]);
          // (a tile of its own: its accumulators say so.  With the whole wait there too 240 us for the 4096-row chunk, 237 so)
          if (!(mine && served % GH == g % GH) && !__all_sync(0xFFFFFFFFu, mbar_try_wait(&lfull[brought % LS], brought / LS & 1u)))
            ok = __all_sync(0xFFFFFFFFu, ok && wait_bar(&lfull[brought % LS], brought / LS & 1u, abort_flag, b.err));
          ++brought;
        }
        bring = true;
        const uint32_t use = served;
        if (mine) ++served;
        if (mine && use % GH == g % GH) {
          const uint32_t ab = half * kBufs + use % kBufs;
          ok = __all_sync(0xFFFFFFFFu, ok && wait_bar(&afull[ab], use / kBufs & 1u, abort_flag, b.err));
          tc_fence_after();
          const float* lse = s_lse + (brought - 1) % LS * RT;
          const uint32_t acc = tmem + lane_off + ab * RT;
          uint64_t sum[2] = {0, 0};
          float odd = 0.f;
          if (full <= 0 && rows == RT) {  // the loads of 32 columns under the exponentials of the 32 before
            uint32_t x[2][32];
            tmem_ld32(acc, x[0]);
#pragma unroll
            for (int c = 0; c < RT; c += 32) {
              tmem_wait_ld(x[c / 32 & 1]);
              if (c + 32 < RT) tmem_ld32(acc + c + 32, x[~(c / 32) & 1]);
              add32(x[c / 32 & 1], lse + c, scale2, sum);
            }
          } else {
#pragma unroll 1
            for (int c = 0; c < rows; c += 32) {
              if (c + 31 < some) continue;
              uint32_t x[32];
              tmem_ld32(acc + c, x);
              if (c >= full && c + 32 <= rows) {
                tmem_wait_ld(x);
                add32(x, lse + c, scale2, sum);
                continue;
              }
              uint32_t see = d >= 0 ? seeing32(p, it.s, row0 + c, d) : ~0u;
              if (rows - c < 32) see &= (1u << (rows - c)) - 1u;
              tmem_wait_ld(x);
#pragma unroll
              for (int j = 0; j < 32; ++j) {
                const float e = ex2(fmaf(__uint_as_float(x[j]), p.a.scale_log2, lse[c + j]));
                if (see & (1u << j)) odd += e;
              }
            }
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&aempty[ab]);
          float s0, s1;
          f2_split(add2(sum[0], sum[1]), s0, s1);
          total += (s0 + s1) + odd;
        }
        row0 += p.row_tile;
        if (!all && by_place) full -= p.row_tile, some -= p.row_tile;
      }
      if (!solo) {  // the groups' sums together, in their order
        float* there = s_sums + (turn++ & 1u) * 384;
        if (g % GH != 0) there[(g - 1) * 128 + r128] = total;
        group_sync();
        if (g % GH == 0)
#pragma unroll
          for (uint32_t o = 1; o < GH; ++o) total += there[(g + o - 1) * 128 + r128];
      }
      if (!ok) break;
      if (tiles == it.tiles) {
        if (writes) *w = keeps ? fmaf(p.decay, old, total) : total;
      } else {
        // a part of the item: the last of its CTAs adds them up, in the line's order
        if (writes) line.slot(p.a, S::KB, at != it.first)[half * 128 + r128] = total;
        const int c0 = line.part_of(it.first), c1 = line.part_of(it.first + it.tiles - 1);
        __threadfence();
        group_sync();
        if (!ok) break;
        if (tid == 0) *s_last = arrive_part(p, c0, c1, true), *s_counted = at + tiles;
        group_sync();
        if (ok && *s_last) {
          __threadfence();
          if (writes) {
            float all = 0.f;
#pragma unroll 4
            for (int c = c0; c <= c1; ++c)
              all += __ldcg(p.a.partials + (static_cast<int64_t>(c) * 2 + (c == c0 ? 0 : 1)) * S::KB + half * 128 + r128);
            *w = keeps ? fmaf(p.decay, old, all) : all;
          }
        }
        group_sync();  // s_last is read
      }
      advance(tiles);
    }
    if (tid == 0 && at < end) give_up(p, line, it, max(at, *s_counted));
  } else if (warp == 16) {
    // ---------------------------------------------------------------- MMA issuer: converged, one elected lane issues
    const uint32_t on = elect_one();
    const uint32_t tm = __shfl_sync(0xFFFFFFFFu, tmem, 0);
    const uint64_t qdesc = sw128_desc(smem_u32(s_q)), kdesc = sw128_desc(smem_u32(s_k));
    constexpr uint32_t kIdesc = attn_idesc<BF16>(128, 0, false);
    uint32_t k_slot = 0, k_phase = 0, q_slot = QS - 1, q_phase = 1;
    uint32_t used[HB] = {};  // tiles a half's accumulators have served
    bool ok = true, any_q = false;
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      if (__all_sync(0xFFFFFFFFu, mbar_try_wait(bar, parity))) return;
      ok = __all_sync(0xFFFFFFFFu, ok && wait_bar(bar, parity, abort_flag, b.err));
    };
    while (ok && at < end) {
      const int tiles = tiles_here(), halves = halves_here();
      int left = it.s.nrows - first_here() * p.row_tile;  // rows from the tile on
      bool bring = brings();
      uint32_t ks[HB] = {};
#pragma unroll
      for (int h = 0; h < HB; ++h) {
        if (h >= halves) break;
        ks[h] = uniform(k_slot * (S::kKTile >> 4));
        wait(&kfull[k_slot], k_phase);
        if (++k_slot == KS) k_slot = 0, k_phase ^= 1u;
      }
      for (int i = 0; ok && i < tiles; ++i, left -= p.row_tile) {
        if (bring) {
          if (any_q) commit(on, &qempty[q_slot]);
          any_q = true;
          if (++q_slot == QS) q_slot = 0, q_phase ^= 1u;
          wait(&qfull[q_slot], q_phase);
        }
        bring = true;
        // as many columns as the tile has rows, in whole chunks of 32
        const uint32_t idesc = uniform(kIdesc | static_cast<uint32_t>((min(left, p.row_tile) + 31) >> 5) << 19);
        const uint32_t qo = uniform(q_slot * (S::kQTile >> 4));
#pragma unroll
        for (int h = 0; h < HB; ++h) {
          if (h >= halves) break;
          const uint32_t ab = uniform(h * kBufs + used[h] % kBufs);
          if (used[h] >= kBufs) wait(&aempty[ab], (used[h] / kBufs - 1) & 1u);
          ++used[h];
          if (!ok) break;
          tc_fence_after();
          const uint32_t ad = tm + ab * RT;
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk)
            mma_ss(on, ad, desc_at(kdesc, ks[h] + (((kk >> 2) * (128 * 128) + (kk & 3) * 32) >> 4)),
                   desc_at(qdesc, qo + (((kk >> 2) * (RT * 128) + (kk & 3) * 32) >> 4)), idesc, kk != 0 ? 1u : 0u);
          commit(on, &afull[ab]);
        }
      }
#pragma unroll
      for (int h = 0; h < HB; ++h)
        if (h < halves) commit(on, &kempty[(k_slot + KS - halves + h) % KS]);
      advance(tiles);
    }
    commit(on, fin);  // every MMA has finished before TMEM is released
    if (lane == 0 && !mbar_wait_bounded(fin, 0)) atomicOr(b.err, kErrWaitTimeout);
    __syncwarp();
  } else if (warp == 17) {
    // ---------------------------------------------------------------- K copies
    const uint32_t base = smem_u32(s_k);
    const int box_rows = min(1 << b.page_shift, 128);
    const int parts = 128 / box_rows, boxes = parts * (D / 64);  // at most 32: a lane each
    const int blk = static_cast<int>(lane) % (D / 64), part = static_cast<int>(lane) / (D / 64);
    uint32_t n = 0;
    bool ok = true;
    while (ok && at < end) {
      const int32_t* tab = b.table + static_cast<int64_t>(it.s.seq) * b.max_pages;
      const int halves = halves_here(), tiles = tiles_here();
      for (int h = 0; ok && h < halves; ++h, ++n) {
        const uint32_t slot = n % KS;
        const int key = it.block * S::KB + h * 128 + part * box_rows;
        int id = -1;
        if (static_cast<int>(lane) < boxes && key < it.s.total_keys) {
          id = tab[key >> b.page_shift];
          if (id < 0 || id >= b.pages) {
            atomicOr(b.err, kErrBadShape);
            id = b.pages;  // past the map: the box arrives as zeros
          }
        }
        const uint32_t loads = __popc(__ballot_sync(0xFFFFFFFFu, id >= 0));
        if (n >= KS) ok = wait_bar(&kempty[slot], (n / KS - 1) & 1u, abort_flag, b.err);
        ok = __all_sync(0xFFFFFFFFu, ok);
        if (!ok) break;
        if (lane == 0) mbar_arrive_expect_tx(&kfull[slot], loads * box_rows * 128);
        if (id >= 0)
          tma_box(base + slot * S::kKTile + blk * (128 * 128) + part * box_rows * 128, &kmap, blk * 64,
                  key & ((1 << b.page_shift) - 1), it.s.kv_head, id, &kfull[slot]);
      }
      advance(tiles);
    }
    // no copy may outlive the CTA: wait (bounded) for the last fill of every slot
    const uint32_t last = min(n, static_cast<uint32_t>(KS));
    for (uint32_t i = 1; i <= last; ++i) {
      const uint32_t f = n - i;
      if (!mbar_wait_bounded(&kfull[f % KS], (f / KS) & 1u)) atomicOr(b.err, kErrWaitTimeout);
    }
    __syncwarp();
  } else if (p.box_tokens) {
    // ---------------------------------------------------------------- queries (TMA) and their log-sum-exps: one warp
    if (warp == 18) {
      const int tokens = p.row_tile / p.a.group;  // of a tile
      int64_t off[RT / 32];                       // a lane's rows lie at the same places of every tile
#pragma unroll
      for (int j = 0; j < RT / 32; ++j) {
        const int r = j * 32 + static_cast<int>(lane);
        off[j] = static_cast<int64_t>(r / p.a.group) * p.a.q.heads + r % p.a.group;
      }
      uint32_t n = 0;
      bool ok = true;
      while (ok && at < end) {
        const int tiles = tiles_here();
        bool bring = brings();
        if (!bring) {
          advance(tiles);
          continue;
        }
        const int tile0 = first_here(), kv_head = it.s.kv_head;
        int left = it.s.nrows - tile0 * p.row_tile, token = it.s.row0 + tile0 * tokens;  // the tile's rows, its first token
        const float* lse = p.lse + static_cast<int64_t>(token) * p.a.q.heads + kv_head * p.a.group;
        float l[RT / 32], next[RT / 32];
        auto fetch = [&]() {
#pragma unroll
          for (int j = 0; j < RT / 32; ++j)
            next[j] = j * 32 + static_cast<int>(lane) < min(left, p.row_tile) ? lse[off[j]] : -INFINITY;
        };
        fetch();
        for (int i = 0; ok && i < tiles; ++i, token += tokens) {
          const uint32_t slot = n % QS;
          if (n >= QS) ok = __all_sync(0xFFFFFFFFu, wait_bar(&qempty[slot], (n / QS - 1) & 1u, abort_flag, b.err));
          if (!ok) break;
          if (lane == 0) {
            mbar_arrive_expect_tx(&qfull[slot], p.box_tokens * p.a.group * D * 2);
            for (int c = 0; c < D / 64; ++c)
              tma_box(smem_u32(s_q) + slot * S::kQTile + c * (RT * 128), &qmap, c * 64, 0, kv_head, token, &qfull[slot]);
          }
#pragma unroll
          for (int j = 0; j < RT / 32; ++j) l[j] = next[j];
          left -= p.row_tile, lse += static_cast<int64_t>(tokens) * p.a.q.heads;
          if (i + 1 < tiles) fetch();  // (a tile ahead)
          if (n >= LS) ok = __all_sync(0xFFFFFFFFu, wait_bar(&lempty[n % LS], (n / LS - 1) & 1u, abort_flag, b.err));
          // a row that saw nothing (or is not there) adds nothing: 2^(x - inf)
#pragma unroll
          for (int j = 0; j < RT / 32; ++j) s_lse[n % LS * RT + j * 32 + lane] = l[j] == -INFINITY ? -INFINITY : -l[j] * kLog2e;
          mbar_arrive(&qfull[slot]), mbar_arrive(&lfull[n % LS]);
          ++n;
        }
        advance(tiles);
      }
      // no copy may outlive the CTA
      const uint32_t last = min(n, static_cast<uint32_t>(QS));
      for (uint32_t i = 1; i <= last; ++i) {
        const uint32_t f = n - i;
        if (!mbar_wait_bounded(&qfull[f % QS], (f / QS) & 1u)) atomicOr(b.err, kErrWaitTimeout);
      }
      __syncwarp();
    }
  } else {
    // ---------------------------------------------------------------- queries that TMA cannot fetch, likewise: two warps
    const uint32_t t = tid - (S::kEpi + 64);
    constexpr int kChunks = D / 8, kPerPass = S::kLoad / kChunks;  // a row's 16-byte chunks lie on neighbouring lanes
    const int c = static_cast<int>(t) % kChunks, r_first = static_cast<int>(t) / kChunks;
    uint32_t n = 0;        // tiles brought
    bool ok = true, pending = false;  // the last one's copies are on their way: not published yet
    auto publish = [&](uint32_t which) {
      fence_proxy_async_smem();
      mbar_arrive(&qfull[which % QS]), mbar_arrive(&lfull[which % LS]);
    };
    auto flush = [&]() {
      if (!pending) return;
      cp_async_wait<0>();
      publish(n - 1);
      pending = false;
    };
    while (ok && at < end) {
      const int tiles = tiles_here(), tile0 = first_here();
      for (int i = 0; ok && i < tiles; ++i) {
        if (!brings()) {
          flush();
          continue;
        }
        const uint32_t slot = n % QS;
        if (n >= QS && !__all_sync(0xFFFFFFFFu, mbar_try_wait(&qempty[slot], (n / QS - 1) & 1u))) {
          flush();
          ok = __all_sync(0xFFFFFFFFu, wait_bar(&qempty[slot], (n / QS - 1) & 1u, abort_flag, b.err));
          if (!ok) break;
        }
        if (n >= LS && !__all_sync(0xFFFFFFFFu, mbar_try_wait(&lempty[n % LS], (n / LS - 1) & 1u))) {
          flush();
          ok = __all_sync(0xFFFFFFFFu, wait_bar(&lempty[n % LS], (n / LS - 1) & 1u, abort_flag, b.err));
          if (!ok) break;
        }
        const int rows = rows_of(tile0 + i), wide = (rows + 31) & ~31, row0 = (tile0 + i) * p.row_tile;
        uint8_t* dst = s_q + slot * S::kQTile + (c >> 3) * (RT * 128);
        for (int r = r_first; r < wide; r += kPerPass) {
          const int rr = row0 + r, tok = rr / p.a.group, h = it.s.kv_head * p.a.group + rr % p.a.group;
          const uint32_t to = smem_u32(dst + image_offset(static_cast<uint32_t>(r), static_cast<uint32_t>((c & 7) * 8)));
          const bool in = r < rows;
          if (p.a.q.vec) {
            const uint16_t* src = static_cast<const uint16_t*>(p.a.q.data);
            if (in) src += static_cast<int64_t>(it.s.row0 + tok) * p.a.q.row_stride + static_cast<int64_t>(h) * p.a.q.head_stride + c * 8;
            cp_async16(to, src, in);
          } else {
            const uint4 u = in ? load_q8(p.a.q, it.s.row0 + tok, h, c * 8) : make_uint4(0u, 0u, 0u, 0u);
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to), "r"(u.x), "r"(u.y), "r"(u.z), "r"(u.w) : "memory");
          }
        }
        cp_async_commit();
        for (int r = static_cast<int>(t); r < RT; r += S::kLoad) {
          const int rr = row0 + r;
          float l = -INFINITY;
          if (r < rows)
            l = p.lse[static_cast<int64_t>(it.s.row0 + rr / p.a.group) * p.a.q.heads + it.s.kv_head * p.a.group + rr % p.a.group];
          // a row that saw nothing (or is not there) adds nothing: 2^(x - inf)
          s_lse[n % LS * RT + r] = l == -INFINITY ? -INFINITY : -l * kLog2e;
        }
        if (pending) {
          cp_async_wait<1>();
          publish(n - 1);
        }
        pending = true;
        ++n;
      }
      advance(tiles);
    }
    flush();
    cp_async_wait<0>();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 16) {
    tc_fence_after();
    tmem_dealloc(tmem, S::kTmem);
  }
}

template <int D, bool FEW>
cudaError_t launch_dim(const WeightParams& params, int sms, size_t partial_floats, cudaStream_t st) {
  using S = WtShape<D, FEW>;
  static KernelSetup setup[2];
  WeightParams p = params;
  auto kern = p.a.bf16 ? weight_kernel<D, FEW, true> : weight_kernel<D, FEW, false>;
  cudaError_t e = kernel_setup(setup[p.a.bf16 ? 1 : 0], kern, S::kThreads, S::kSmem);
  if (e != cudaSuccess) return e;
  CUtensorMap kmap;
  if (!kv_tensor_map(kmap, p.a.b.k, p.a, D, 128)) return cudaErrorInvalidValue;
  // whole tokens to a tile where they fit: then a tile of queries is a box
  p.row_tile = p.a.group <= S::RT ? S::RT / p.a.group * p.a.group : S::RT;
  CUtensorMap qmap = kmap;
  if (p.a.q.vec && p.a.group <= S::RT) {
    const int tokens = S::RT / p.a.group;
    if (q_tensor_map(qmap, p.a, D, tokens)) p.box_tokens = tokens;
  }
  const int64_t tiles = static_cast<int64_t>(p.a.b.nseq) * p.a.b.kv_heads * ((p.a.max_context + S::KB - 1) / S::KB) *
                        ((static_cast<int64_t>(p.a.max_rows) * p.a.group + p.row_tile - 1) / p.row_tile);
  int64_t grid = sms;
  if (grid > tiles) grid = tiles;
  const int64_t fit = static_cast<int64_t>(partial_floats / (2 * S::KB));
  if (grid > fit) grid = fit;
  if (grid > kMaxParts) grid = kMaxParts;
  if (grid < 1) grid = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(S::kThreads);
  cfg.dynamicSmemBytes = S::kSmem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, p, kmap, qmap);
}

}  // namespace

cudaError_t launch_attn_weight(const WeightParams& p, int dim, int sms, size_t partial_floats, cudaStream_t st) {
  // blocks with room for 32 query rows leave the rest to the keys (32 sequences' tokens: 66.3 us with room for 128, 64.5 us)
  const bool few = static_cast<int64_t>(p.a.max_rows) * p.a.group <= 32;
  switch (dim) {
    case 64: return (few ? launch_dim<64, true> : launch_dim<64, false>)(p, sms, partial_floats, st);
    case 128: return (few ? launch_dim<128, true> : launch_dim<128, false>)(p, sms, partial_floats, st);
    default: return (few ? launch_dim<256, true> : launch_dim<256, false>)(p, sms, partial_floats, st);
  }
}

}  // namespace exl3
