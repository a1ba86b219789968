// exl3_attn_tc.cu -- attention of many rows per kv head over the paged cache (drafted trees, prompt chunks) on the
// 5th-generation tensor cores.
//
// The same one-pass softmax as exl3_attn_mma.cu.  A row block is up to 256 rows (kv head's query heads x new tokens) in
// one or two 128-row tiles; scores S = Q K^T and outputs O += P V are tcgen05.mma products with the accumulators in
// TMEM.  P, the probabilities in 16 bits, overwrites its own scores' columns in TMEM and is the A operand of the second
// product from there.
//
// Two S/P buffers keep the tensor pipe and the exponentials busy at once.  With two row tiles, each buffer belongs to
// one of them (the events of a block: (tile 0, rows 0), (tile 0, rows 1), (tile 1, rows 0), ...); with one, the key
// tiles alternate between the buffers, for heads up to 128 wide each with its own O and running maximum, joined at the
// end -- so a small block also has two chains in flight.  256-wide heads (whose O takes half of TMEM) have one O, and
// 64-key tiles.
//
// Roles: NG groups of four softmax warps (a thread per row: tcgen05.ld of its scores, maximum, exponentials, P back by
// tcgen05.st), then one warp each for the MMAs, K copies, V copies (TMA, one box per page and 64 columns, 128-byte
// swizzle) and the V tiles' cleaning.  O is rescaled only when a row's maximum has grown by more than a factor (2^8; 2^4
// for f16, whose probabilities have less room); the old maximum is kept otherwise, and the f32 sums and the final division
// take out the difference.
//
// Keys that some row of the block does not see (stale slots, other branches) are masked in S by index; their V rows
// cannot be masked there (0 x inf = NaN), so in the tiles that hold such keys the cleaning warp zeroes slots past the
// sequence and infinities and NaN; the latter are added back in the epilogue to the rows that see them.
//
// What bounds it: up to 128 rows HBM (32 sequences' 16-token trees over 4-8k slots: 148 us, 5.5 TB/s; 154 us, 5.2 TB/s back
// to back); with 256 rows the softmax warps, whose chain with the products of their buffer is 3.4k clocks per 256 x 128
// scores against 2.0k of either the exponentials or the products alone (a 4096-row chunk on 4096 slots: 386 us, 1.07 PFLOP/s;
// back to back, where power limits the clock, 420 us, 0.98 PFLOP/s).
//
// Every mbarrier wait is bounded (wait_bar): one that gives up raises an abort flag that all roles poll.
#include <cuda.h>
#include <cuda_runtime.h>

#include "exl3_attn.h"
#include "exl3_attn_dev.cuh"
#include "exl3_common.cuh"
#include "exl3_internal.h"
#include "exl3_tc.cuh"

namespace exl3 {

using namespace tc;

namespace {

template <int D, int ROWS>
struct TcShape {
  static constexpr int NG = D == 256 ? 1 : 2;             // softmax groups (and O accumulators)
  static constexpr int KT = D == 256 ? 64 : 128;          // keys per tile
  static constexpr int kRows = ROWS;                      // rows per block: 128, or 256 in two row tiles
  static constexpr int kThreads = NG * 128 + 128;
  static constexpr int kSoft = NG * 128;                  // softmax threads
  static constexpr int kTile = KT * D * 2;                // bytes of a K or V tile
  static constexpr int kQBytes = kRows * D * 2;
  static constexpr int kSlots = (229376 - kQBytes) / kTile > 10 ? 10 : (229376 - kQBytes) / kTile;
  static constexpr int VS = kSlots / 2, KS = kSlots - VS; // V and K tiles in flight
  static constexpr int kOCol = 256;                       // TMEM: S buffers at columns 0 and KT, O of group g at 256 + g * D
  static constexpr int kTmem = 512;
  static constexpr int kParts = KT / 64;                  // P comes in parts of 64 keys, each a product of its own
  static constexpr int kBars = 2 * KS + 3 * VS + 2 + 2 * kParts + 2 + 5;
  static constexpr int kSmem = kQBytes + kSlots * kTile + 2 * 128 * 8 + kBars * 8 + 48 + sizeof(WorkLine) + kThreads / 32 * sizeof(Item);
  static_assert(KS * kTile + VS * kTile + kQBytes <= 229376 && kSmem <= 232448, "shared memory");
  static_assert(VS <= 8, "the odd flags cover eight items");
};

// Two f32 in one 64-bit register pair: one issue slot for both.
__device__ __forceinline__ uint64_t f2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void f2_split(uint64_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// the largest of three (NaN is passed over: it shows in its own probability)
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// Bounded wait (about two seconds) that also gives up when another role has.  The abort flag and the clock are read once
// in many polls: a read of the global timer between polls held each wait up, and every tile's chain has three of them
// (32 x 16-token trees 207 us with it, 192 without).
__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity, volatile uint32_t* abort_flag, uint32_t* err) {
  uint64_t t0 = 0;
  for (uint32_t i = 1;; ++i) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((i & 63u) != 0u) continue;
    if (*abort_flag) return false;
    if ((i & 1023u) != 0u) continue;
    const uint64_t now = global_timer_ns();
    if (t0 == 0) t0 = now;
    else if (now - t0 > 2000000000ull) {
      *abort_flag = 1u;
      atomicOr(err, kErrWaitTimeout);
      return false;
    }
  }
}

// A box of the cache: 64 columns from x, the rows from `tok` of one page and head.
__device__ __forceinline__ void tma_box(uint32_t dst, const CUtensorMap* map, int x, int tok, int head, int page,
                                        uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::
          "r"(dst),
      "l"(map), "r"(x), "r"(tok), "r"(head), "r"(page), "r"(smem_u32(bar))
      : "memory");
}

// Shared-memory descriptor of an operand whose rows are k (keys) and whose contiguous direction is M or N: 64-element
// blocks of 128-byte swizzled rows, `block_bytes` apart; 8-key groups 1024 bytes apart.
__device__ __forceinline__ uint64_t sw128_mn_desc(uint32_t saddr, uint32_t block_bytes) {
  return static_cast<uint64_t>((saddr >> 4) & 0x3FFFu) | (static_cast<uint64_t>((block_bytes >> 4) & 0x3FFFu) << 16) |
         (static_cast<uint64_t>(1024 >> 4) << 32) | (static_cast<uint64_t>(1) << 46) | (static_cast<uint64_t>(2) << 61);
}

// Instruction descriptor of kind::f16 with f32 accumulators; b_mn: B's contiguous direction is N.
template <bool BF16>
constexpr uint32_t attn_idesc(int m, int n, bool b_mn) {
  return umma_idesc(m, n) | (BF16 ? (1u << 7) | (1u << 10) : 0u) | (b_mn ? 1u << 16 : 0u);
}

// The MMA warp runs converged and one elected lane issues: its operands then stay in uniform registers.  (Issued inside
// a one-lane branch, each MMA took some 100 clocks to issue, against the 64 it runs for: 4.1k clocks per 256 x 128 tile.)
__device__ __forceinline__ uint32_t elect_one() {
  uint32_t e;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xFFFFFFFF;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(e));
  return e;
}
// The same value, known to the compiler to be one for the whole warp.
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return __shfl_sync(0xFFFFFFFFu, v, 0); }
// A descriptor `bytes` further on (its address field counts 16 bytes in the low word).
__device__ __forceinline__ uint64_t desc_at(uint64_t desc, uint32_t lo_add) {
  return (desc & 0xFFFFFFFF00000000ull) | (static_cast<uint32_t>(desc) + lo_add);
}
// D[tmem] (+)= A[smem] * B[smem]^T, where `on`
__device__ __forceinline__ void mma_ss(uint32_t on, uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                       uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(on)
      : "memory");
}
// D[tmem] (+)= A[tmem] * B[smem], where `on`
__device__ __forceinline__ void mma_ts(uint32_t on, uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc,
                                       uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(on)
      : "memory");
}
// Arrives on `bar` when every tcgen05 operation the elected lane issued before has completed.
__device__ __forceinline__ void commit(uint32_t on, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar)),
      "r"(on)
      : "memory");
}

// Orders uses of registers loaded by tmem_ld32 after an earlier wait (tmem_wait_ld of another load).
__device__ __forceinline__ void after_wait(uint32_t (&r)[32]) {
#pragma unroll
  for (int i = 0; i < 32; ++i) asm volatile("" : "+r"(r[i])::"memory");
}

// Moves registers from the copy and MMA warps to the softmax warps: a row's 128 scores stay in registers.  The shares
// (8 x 32 x 200 + 4 x 32 x 104 = 64512) are what 384 threads were launched with (168 each).
template <int R>
__device__ __forceinline__ void regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(R)); }
template <int R>
__device__ __forceinline__ void regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(R)); }

// The block as the roles walk it: its key tiles [tile0, tile0 + tiles), one or two row tiles, and its events.
struct Block {
  int tile0, tiles, rows, qt, events, full_keys;
};
template <int D, int ROWS>
__device__ __forceinline__ Block block_of(const AttnParams& p, const WorkLine& line, const Item& it, int64_t at) {
  using S = TcShape<D, ROWS>;
  Block b;
  b.tile0 = static_cast<int>(at - it.first);
  b.tiles = static_cast<int>(min(line.end - at, static_cast<int64_t>(it.tiles - b.tile0)));
  b.rows = min(S::kRows, it.nrows - it.row_block * S::kRows);
  b.qt = b.rows > 128 ? 2 : 1;
  b.events = b.qt * b.tiles;
  // the leading keys that every row sees
  const int own = p.b.tree ? 0 : it.row_block * S::kRows / p.group + 1;
  b.full_keys = it.context + min(own, it.total_keys - it.context);
  return b;
}

// Which of the slots key0 .. key0 + 31 new token tok sees.
__device__ __forceinline__ uint32_t seen32(const PagedBatch& b, const Item& it, int tok, int key0) {
  if (tok >= it.ntok) return 0u;
  uint32_t m;
  const int d = key0 - it.context;  // the first slot's place among the new tokens
  if (!b.tree) {
    const int n = tok + 1 - d;
    m = n >= 32 ? ~0u : (n <= 0 ? 0u : (1u << n) - 1u);
  } else if (d <= -32) {
    m = ~0u;
  } else {
    const uint32_t* t = b.tree + static_cast<int64_t>(it.row0 + tok) * b.tree_words;
    if (d < 0) {
      m = (t[0] << (-d)) | ((1u << (-d)) - 1u);
    } else {
      const int w = d >> 5;
      const uint32_t lo = w < b.tree_words ? t[w] : 0u, hi = w + 1 < b.tree_words ? t[w + 1] : 0u;
      m = __funnelshift_r(lo, hi, d & 31);
    }
  }
  const int left = it.total_keys - key0;
  if (left < 32) m &= left <= 0 ? 0u : (1u << left) - 1u;
  return m;
}

// The infinities and NaN of V among keys [key_lo, key_hi) that row token `tok` of head `h` sees, which the cleaning
// warp took out of the product: o[i] += e^(s - m) v for columns d0 .. d0 + 31.  Rare, so plain loads and one thread.
template <int D, bool BF16>
__device__ __noinline__ void add_odd(const AttnParams& p, const Item& it, int tok, int h, int key_lo, int key_hi,
                                     int full_keys, float m, int d0, float* o) {
  if (tok >= it.ntok) return;
  const uint16_t* q = static_cast<const uint16_t*>(p.q.data) + static_cast<int64_t>(it.row0 + tok) * p.q.row_stride +
                      h * p.q.head_stride;
  for (int key = max(key_lo, full_keys); key < min(key_hi, it.total_keys); ++key) {
    if (!sees(p.b, it, tok, key)) continue;
    const int id = p.b.table[static_cast<int64_t>(it.seq) * p.b.max_pages + (key >> p.b.page_shift)];
    if (id < 0 || id >= p.b.pages) continue;
    const int64_t off = id * p.b.page_stride + (key & ((1 << p.b.page_shift) - 1)) * p.b.token_stride +
                        it.kv_head * p.b.head_stride;
    bool any = false;
    for (int i = 0; i < 32; ++i) any |= !isfinite(unpack1<BF16>(p.b.v[off + d0 + i], 0));
    if (!any) continue;
    float s = 0.f;
    for (int d = 0; d < D; ++d) s += unpack1<BF16>(q[d], 0) * unpack1<BF16>(p.b.k[off + d], 0);
    const float w = ex2(s * p.scale_log2 - (m == -INFINITY ? 0.f : m));
    for (int i = 0; i < 32; ++i) {
      const float v = unpack1<BF16>(p.b.v[off + d0 + i], 0);
      if (!isfinite(v)) o[i] += w * v;
    }
  }
}

// The last of the CTAs that an item was cut between joins their slots, in key order: o as [D / 4][ROWS] float4, then
// (m, l) per row.  A thread takes one row and every n-th pair of column quads, four pairs in flight.
template <int D, int ROWS, bool BF16, typename Sync>
__device__ void join_block(const AttnParams& p, const WorkLine& line, const Item& it, int rows, int* s_word, Sync&& sync) {
  constexpr int kThreads = TcShape<D, ROWS>::kSoft;
  constexpr int64_t kFloats = static_cast<int64_t>(ROWS) * (D + 2);
  const int c0 = line.part_of(it.first), c1 = line.part_of(it.first + it.tiles - 1);
  __threadfence();
  sync();
  if (threadIdx.x == 0) {
    const bool last = atomicAdd(p.counters + c0, 1u) + 1u == static_cast<uint32_t>(c1 - c0 + 1);
    if (last) p.counters[c0] = 0u;
    *s_word = last;
  }
  sync();
  if (*s_word) {
    __threadfence();
    int pad = 32;
    while (pad < rows) pad <<= 1;
    const int r = static_cast<int>(threadIdx.x) & (pad - 1), first = static_cast<int>(threadIdx.x) / pad, step = kThreads / pad;
    if (r < rows) {
      auto slot = [&](int c) { return p.partials + (static_cast<int64_t>(c) * 2 + (c == c0 ? 0 : 1)) * kFloats; };
      float m = -INFINITY, l = 0.f;
#pragma unroll 4
      for (int c = c0; c <= c1; ++c) {
        const float2 ml = __ldcg(reinterpret_cast<const float2*>(slot(c) + ROWS * D) + r);
        const float top = fmaxf(m, ml.x), base = top == -INFINITY ? 0.f : top;
        l = l * ex2(m - base) + ml.y * ex2(ml.x - base);
        m = top;
      }
      const float base = m == -INFINITY ? 0.f : m, inv = l == 0.f ? 0.f : 1.f / l;
      const int rr = it.row_block * ROWS + r, h = it.kv_head * p.group + rr % p.group;
      const int64_t row = it.row0 + rr / p.group;
      uint16_t* dst = static_cast<uint16_t*>(p.out.data) + row * p.out.row_stride + h * p.out.head_stride;
      constexpr int kBatch = 4;
      for (int j0 = first; j0 < D / 8; j0 += step * kBatch) {
        float4 a[kBatch][2];
#pragma unroll
        for (int u = 0; u < kBatch; ++u) a[u][0] = a[u][1] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 2
        for (int c = c0; c <= c1; ++c) {
          const float* s = slot(c);
          const float f = ex2(__ldcg(reinterpret_cast<const float2*>(s + ROWS * D) + r).x - base);
          float4 v[kBatch][2];
#pragma unroll
          for (int u = 0; u < kBatch; ++u) {
            const int j = min(j0 + u * step, D / 8 - 1);
#pragma unroll
            for (int e = 0; e < 2; ++e) v[u][e] = __ldcg(reinterpret_cast<const float4*>(s) + (2 * j + e) * ROWS + r);
          }
#pragma unroll
          for (int u = 0; u < kBatch; ++u)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              a[u][e].x += v[u][e].x * f, a[u][e].y += v[u][e].y * f;
              a[u][e].z += v[u][e].z * f, a[u][e].w += v[u][e].w * f;
            }
        }
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          const int j = j0 + u * step;
          if (j >= D / 8) continue;
          uint32_t w[4];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            w[2 * e] = l == 0.f ? 0u : pack2<BF16>(a[u][e].x * inv, a[u][e].y * inv);
            w[2 * e + 1] = l == 0.f ? 0u : pack2<BF16>(a[u][e].z * inv, a[u][e].w * inv);
          }
          if (p.out.vec) {
            *reinterpret_cast<uint4*>(dst + j * 8) = make_uint4(w[0], w[1], w[2], w[3]);
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              dst[j * 8 + 2 * i] = static_cast<uint16_t>(w[i]), dst[j * 8 + 2 * i + 1] = static_cast<uint16_t>(w[i] >> 16);
          }
        }
      }
      if (p.lse && first == 0) p.lse[row * p.out.heads + h] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
    }
  }
  sync();
}

template <int D, int ROWS, bool BF16>
__global__ void __launch_bounds__(TcShape<D, ROWS>::kThreads, 1)
    attn_tc_kernel(const __grid_constant__ AttnParams p, const __grid_constant__ CUtensorMap kmap,
                   const __grid_constant__ CUtensorMap vmap) {
  using S = TcShape<D, ROWS>;
  constexpr int NG = S::NG, KT = S::KT, KS = S::KS, VS = S::VS;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* s_q = smem;                       // [row tile][64-column block][128 rows][128 bytes], swizzled
  uint8_t* s_k = s_q + S::kQBytes;           // [slot][64-column block][KT rows][128 bytes]
  uint8_t* s_v = s_k + KS * S::kTile;
  float2* s_ml = reinterpret_cast<float2*>(s_v + VS * S::kTile);  // [2][128]
  uint64_t* bars = reinterpret_cast<uint64_t*>(s_ml + 256);
  uint64_t *kfull = bars, *kempty = kfull + KS, *vfull = kempty + KS, *vclean = vfull + VS, *vempty = vclean + VS;
  uint64_t *sfull = vempty + VS, *pready = sfull + 2, *ofull = pready + 2 * S::kParts;
  uint64_t *qfull = ofull + 2, *ofree = qfull + 1, *xsync = ofree + 1, *pvdone = xsync + 1, *fin = pvdone + 1;
  uint32_t* words = reinterpret_cast<uint32_t*>(bars + S::kBars);
  uint32_t* s_tmem = words;
  volatile uint32_t* abort_flag = words + 1;
  int* s_last = reinterpret_cast<int*>(words + 2);
  volatile uint32_t* s_odd = words + 4;  // [8]: serial + 1 of an item whose V held infinities or NaN
  WorkLine* s_line = reinterpret_cast<WorkLine*>(words + 12);
  Item* s_items = reinterpret_cast<Item*>(s_line + 1);  // one per warp
  const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;

  if (smem_u32(smem) & 1023u) {  // the swizzle goes by address bits: not served
    if (tid == 0) atomicOr(p.b.err, kErrBadShape);
    return;
  }
  if (warp == NG * 4) {
    tmem_alloc(smem_u32(s_tmem), S::kTmem);
    tmem_relinquish();
  }
  if (tid == 0) {
    for (int i = 0; i < KS; ++i) mbar_init(&kfull[i], 1), mbar_init(&kempty[i], 1);
    for (int i = 0; i < VS; ++i) mbar_init(&vfull[i], 1), mbar_init(&vclean[i], 1), mbar_init(&vempty[i], 1);
    for (int i = 0; i < 2; ++i) mbar_init(&sfull[i], 1), mbar_init(&ofull[i], 1);
    for (int i = 0; i < 2 * S::kParts; ++i) mbar_init(&pready[i], 128);
    mbar_init(qfull, S::kSoft), mbar_init(ofree, S::kSoft), mbar_init(xsync, S::kSoft);
    mbar_init(pvdone, 1), mbar_init(fin, 1);
    fence_barrier_init();
    *abort_flag = 0u;
    for (int i = 0; i < 8; ++i) s_odd[i] = 0u;
  }
  if (tid == 32) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&kmap) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&vmap) : "memory");
  }
  pdl_wait();
  {
    WorkLine own;
    Item first;
    own.start(p, S::kRows, KT, reinterpret_cast<int64_t*>(s_ml), first);  // (not where TMA will write: that is another proxy)
    if (tid == 0) *s_line = own;
    if (lane == 0) s_items[warp] = first;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *s_tmem;
  // The line, and each warp's item on it, stay in shared memory: what did not fit in registers went to local memory,
  // which the shared memory leaves next to no L1 for, and a block's end took as long as eight tiles.
  const WorkLine& line = *s_line;
  Item& it = s_items[warp];
  if constexpr (NG == 2) {
    if (warp < NG * 4) regs_up<200>();
    else regs_down<104>();
  }
  int64_t at = line.begin;
  auto advance = [&](int tiles) {
    at += tiles;
    if (at < line.end) {
      __syncwarp();
      if (lane == 0) line.next(p, it);
      __syncwarp();
    }
  };

  if (warp < NG * 4) {
    // ---------------------------------------------------------------- softmax groups
    const uint32_t g = warp >> 2, wq = warp & 3u, r128 = wq * 32 + lane;  // row of the 128-row tile = TMEM lane
    const uint32_t lane_off = (wq * 32u) << 16;
    uint32_t sphase = 0, ophase = 0, xphase = 0, pvphase = 0;  // sphase: a bit per buffer; ophase: per group
    bool ok = true;
    auto group_sync = [&]() {  // all softmax threads
      mbar_arrive(xsync);
      ok = __all_sync(0xFFFFFFFFu, ok && wait_bar(xsync, xphase, abort_flag, p.b.err));
      xphase ^= 1u;
    };
    for (uint32_t serial = 0; ok && at < line.end; ++serial) {
      const Block b = block_of<D, ROWS>(p, line, it, at);
      // the query rows into their swizzled tiles: with two row tiles a group loads its own, else both share the one
      {
        const uint32_t tile = b.qt == 2 ? g : 0u;
        const int cols0 = b.qt == 2 || NG == 1 ? 0 : static_cast<int>(g) * (D / 2);
        const int ncols = b.qt == 2 || NG == 1 ? D : D / 2;
        const int r = static_cast<int>(tile * 128u + r128);
        const int rr = it.row_block * S::kRows + r, t = rr / p.group, h = it.kv_head * p.group + rr % p.group;
        const int64_t q_row = it.row0 + t;
        for (int c0 = 0; c0 < ncols; c0 += 64) {  // eight loads in flight
          uint4 u[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) u[i] = make_uint4(0u, 0u, 0u, 0u);
          if (r < b.rows) {
            if (p.q.vec) {
              const uint4* src = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.q.data) +
                                                                q_row * p.q.row_stride + h * p.q.head_stride + cols0 + c0);
#pragma unroll
              for (int i = 0; i < 8; ++i)
                if (c0 + i * 8 < ncols) u[i] = src[i];
            } else {
#pragma unroll
              for (int i = 0; i < 8; ++i)
                if (c0 + i * 8 < ncols) u[i] = load_q8(p.q, q_row, h, cols0 + c0 + i * 8);
            }
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int col = cols0 + c0 + i * 8;
            if (c0 + i * 8 < ncols)
              *reinterpret_cast<uint4*>(s_q + tile * (128 * D * 2) + (col >> 6) * (128 * 128) +
                                        image_offset(r128, static_cast<uint32_t>(col & 63))) = u[i];
          }
        }
      }
      fence_proxy_async_smem();
      mbar_arrive(qfull);

      const int row = (b.qt == 2 ? static_cast<int>(g) * 128 : 0) + static_cast<int>(r128);
      const int tok = (it.row_block * S::kRows + row) / p.group;
      const bool idle = row - static_cast<int>(lane) >= b.rows;
      float m = -INFINITY, l = 0.f;  // m in units of log2
      for (int e = static_cast<int>(g); e < b.events; e += NG) {
        const uint32_t buf = e & 1;
        const int tile = b.qt == 2 ? e >> 1 : e;
        const int key0 = (b.tile0 + tile) * KT;
        const uint32_t pv_parity = pvphase ^ 1u;  // the product of the event before (NG = 1)
        pvphase ^= 1u;
        const uint32_t s_addr = tmem + lane_off + buf * KT;
        ok = __all_sync(0xFFFFFFFFu, ok && wait_bar(&sfull[buf], (sphase >> buf) & 1u, abort_flag, p.b.err));
        sphase ^= 1u << buf;
        if (idle) {  // none of the warp's rows is in the block: whatever P holds there is never read back
          for (int c = 0; c < S::kParts; ++c) mbar_arrive(&pready[buf * S::kParts + c]);
          continue;
        }
        tc_fence_after();
        uint32_t x[KT / 32][32];
#pragma unroll
        for (int c = 0; c < KT / 32; ++c) tmem_ld32(s_addr + c * 32, x[c]);
        tmem_wait_ld(x[0]);
#pragma unroll
        for (int c = 1; c < KT / 32; ++c) after_wait(x[c]);
        if (key0 + KT > b.full_keys) {
#pragma unroll
          for (int c = 0; c < KT / 32; ++c) {
            const uint32_t mask = seen32(p.b, it, tok, key0 + c * 32);
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (!(mask & (1u << i))) x[c][i] = 0xFF800000u;  // -inf
          }
        }
        float mx[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) mx[i] = __uint_as_float(x[0][i]);
#pragma unroll
        for (int i = 4; i < KT; i += 8) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int u = i + 2 * j < KT ? i + 2 * j : KT - 2;  // (the last step sees its neighbours again)
            mx[j] = max3(mx[j], __uint_as_float(x[u >> 5][u & 31]), __uint_as_float(x[(u + 1) >> 5][(u + 1) & 31]));
          }
        }
        const float top = max3(max3(mx[0], mx[1], mx[2]), mx[3], mx[3]) * p.scale_log2;
        const bool grow = top > m + kSlack<BF16>;  // (m = -inf: as soon as anything is seen)
        if (e < NG) {
          m = top;
        } else if (__any_sync(0xFFFFFFFFu, grow)) {
          if constexpr (NG == 1) ok = __all_sync(0xFFFFFFFFu, ok && wait_bar(pvdone, pv_parity, abort_flag, p.b.err));
          tc_fence_after();
          const float f = grow ? ex2(m - top) : 1.f;
          if (grow) m = top, l *= f;
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            uint32_t o[32];
            const uint32_t o_addr = tmem + lane_off + S::kOCol + g * D + c * 32;
            tmem_ld32(o_addr, o);
            tmem_wait_ld(o);
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
            tmem_st32(o_addr, o);
          }
          tmem_wait_st();
        }
        const float base = (m == -INFINITY ? 0.f : m) - kLift<BF16>;
        const uint64_t scale2 = f2(p.scale_log2, p.scale_log2), base2 = f2(-base, -base);
        uint64_t sum[2] = {0, 0};
#pragma unroll
        for (int c = 0; c < KT / 64; ++c) {
          uint32_t pk[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const int u = (2 * i) & 31;
            float y0, y1;
            f2_split(fma2(f2(__uint_as_float(x[2 * c + (i >> 4)][u]), __uint_as_float(x[2 * c + (i >> 4)][u + 1])), scale2, base2),
                     y0, y1);
            y0 = ex2(y0), y1 = ex2(y1);
            sum[i & 1] = add2(sum[i & 1], f2(y0, y1));
            pk[i] = pack2<BF16>(y0, y1);  // (l keeps the f32 values)
          }
          tmem_st32(s_addr + c * 32, pk);
          tmem_wait_st();
          tc_fence_before();
          mbar_arrive(&pready[buf * S::kParts + c]);
        }
        float s0, s1;
        f2_split(add2(sum[0], sum[1]), s0, s1);
        l += s0 + s1;
      }

      // ---- the block's end: o / l, or a partial for the join
      m -= kLift<BF16>;
      const bool whole = b.tiles == it.tiles;
      const bool two = b.qt == 1 && NG == 2;  // two key halves of the same rows
      const int mine = two ? (b.events > static_cast<int>(g) ? 1 : 0) : 1;  // this group had a tile
      if (mine) {
        ok = __all_sync(0xFFFFFFFFu, ok && wait_bar(&ofull[g], ophase, abort_flag, p.b.err));
        ophase ^= 1u;
      }
      float f0 = 1.f, f1 = 0.f;
      if (two) {
        s_ml[g * 128 + r128] = make_float2(m, l);
        group_sync();
        const float2 a = s_ml[r128], c = s_ml[128 + r128];
        m = fmaxf(a.x, c.x);
        const float base = m == -INFINITY ? 0.f : m;
        f0 = ex2(a.x - base), f1 = ex2(c.x - base);
        l = a.y * f0 + c.y * f1;
      }
      tc_fence_after();
      const bool second = two && b.events > 1;
      const bool odd = s_odd[serial & 7u] == serial + 1u;
      const int cols0 = two ? static_cast<int>(g) * (D / 2) : 0, ncols = two ? D / 2 : D;
      const uint32_t o0 = tmem + lane_off + S::kOCol + (two ? 0u : g * D), o1 = tmem + lane_off + S::kOCol + D;
      const bool live = row < b.rows;
      const int rr = it.row_block * S::kRows + row;
      const int h = it.kv_head * p.group + rr % p.group;
      const int64_t out_row = it.row0 + tok;
      float* slot = whole ? nullptr : line.slot(p, S::kRows * (D + 2), at != it.first);
      const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll 1
      for (int c = cols0; c < cols0 + ncols; c += 32) {
        uint32_t v[32];
        float o[32];
        tmem_ld32(o0 + c, v);
        tmem_wait_ld(v);
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] = __uint_as_float(v[i]);
        if (second) {
          tmem_ld32(o1 + c, v);
          tmem_wait_ld(v);
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = o[i] * f0 + __uint_as_float(v[i]) * f1;
        }
        if (!live) continue;
        if (odd) {
          float t[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) t[i] = o[i];
          add_odd<D, BF16>(p, it, tok, h, b.tile0 * KT, (b.tile0 + b.tiles) * KT, b.full_keys, m, c, t);
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = t[i];
        }
        if (whole) {
          uint16_t* dst = static_cast<uint16_t*>(p.out.data) + out_row * p.out.row_stride + h * p.out.head_stride + c;
          uint32_t w[16];
#pragma unroll
          for (int i = 0; i < 16; ++i)
            w[i] = l == 0.f ? 0u : pack2<BF16>(o[2 * i] * inv, o[2 * i + 1] * inv);
          if (p.out.vec == 2) {  // a whole sector per lane and store
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const uint32_t w8[8] = {w[8 * i],     w[8 * i + 1], w[8 * i + 2], w[8 * i + 3],
                                      w[8 * i + 4], w[8 * i + 5], w[8 * i + 6], w[8 * i + 7]};
              st_global_v8(dst + 16 * i, w8);
            }
          } else if (p.out.vec) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              reinterpret_cast<uint4*>(dst)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
          } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) dst[2 * i] = static_cast<uint16_t>(w[i]), dst[2 * i + 1] = static_cast<uint16_t>(w[i] >> 16);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i)  // [D / 4][rows] float4: a warp's rows are neighbours
            reinterpret_cast<float4*>(slot)[(c / 4 + i) * S::kRows + row] =
                make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
        }
      }
      if (live && cols0 == 0) {
        if (whole) {
          if (p.lse) p.lse[out_row * p.out.heads + h] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
        } else {
          *reinterpret_cast<float2*>(slot + S::kRows * D + 2 * row) = make_float2(m, l);
        }
      }
      tc_fence_before();
      mbar_arrive(ofree);
      if (!whole) join_block<D, ROWS, BF16>(p, line, it, b.rows, s_last, group_sync);
      group_sync();  // every MMA of the block has finished, and its rows are read: Q may be replaced
      advance(b.tiles);
    }
  } else if (warp == NG * 4) {
    // ---------------------------------------------------------------- MMA issuer
    constexpr uint32_t idesc_s = attn_idesc<BF16>(128, KT, false), idesc_o = attn_idesc<BF16>(128, D, true);
    const uint32_t on = elect_one();
    const uint32_t tm = __shfl_sync(0xFFFFFFFFu, tmem, 0);
    const uint64_t qdesc = sw128_desc(smem_u32(s_q)), kdesc = sw128_desc(smem_u32(s_k));
    const uint64_t vdesc = sw128_mn_desc(smem_u32(s_v), KT * 128);
    uint32_t kslot = 0, kphase = 0, vslot = 0, vphase = 0;  // the next K and V tile to come
    uint32_t pphase = 0;
    bool ok = true;
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      if (__all_sync(0xFFFFFFFFu, mbar_try_wait(bar, parity))) return;
      ok = __all_sync(0xFFFFFFFFu, ok && wait_bar(bar, parity, abort_flag, p.b.err));
    };
    for (uint32_t serial = 0; ok && at < line.end; ++serial) {
      const Block b = block_of<D, ROWS>(p, line, it, at);
      const bool both = b.qt == 2;  // a key tile serves two events
      wait(qfull, serial & 1u);
      auto scores_wait = [&](int e) {
        if (!both || !(e & 1)) wait(&kfull[kslot], kphase);
      };
      auto scores = [&](int e) {
        const uint32_t buf = e & 1;
        const uint32_t qo = uniform(both && buf ? (128 * D * 2) >> 4 : 0), ko = uniform(kslot * (S::kTile >> 4));
        const uint32_t sd = uniform(tm + buf * KT);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
          mma_ss(on, sd, desc_at(qdesc, qo + (((kk >> 2) * (128 * 128) + (kk & 3) * 32) >> 4)),
                 desc_at(kdesc, ko + (((kk >> 2) * (KT * 128) + (kk & 3) * 32) >> 4)), idesc_s, kk != 0 ? 1u : 0u);
        commit(on, &sfull[buf]);
        if (!both || buf) {
          commit(on, &kempty[kslot]);
          if (++kslot == KS) kslot = 0, kphase ^= 1u;
        }
      };
      for (int e = 0; e < 2 && e < b.events; ++e) {
        scores_wait(e);
        if (!ok) break;
        tc_fence_after();
        scores(e);
      }
      if (serial) wait(ofree, (serial - 1) & 1u);
      for (int e = 0; ok && e < b.events; ++e) {
        const uint32_t buf = e & 1;
        // everything the event needs but P first: the products then follow one another
        if (!both || buf == 0) wait(&vclean[vslot], vphase);
        if (e + 2 < b.events) scores_wait(e + 2);
        const uint32_t vo = uniform(vslot * (S::kTile >> 4)), sd = uniform(tm + buf * KT);
        const uint32_t od = uniform(tm + S::kOCol + (NG == 2 ? buf * D : 0)), more = uniform(e >= NG ? 1u : 0u);
        const uint32_t pp = (pphase >> buf) & 1u;
        pphase ^= 1u << buf;
#pragma unroll
        for (int c = 0; c < S::kParts; ++c) {
          wait(&pready[buf * S::kParts + c], pp);
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int kk = c * 4; kk < c * 4 + 4; ++kk)
            mma_ts(on, od, sd + kk * 8, desc_at(vdesc, vo + ((kk * 2048) >> 4)), idesc_o, kk != 0 ? 1u : more);
        }
        if (!ok) break;
        if (e + 2 < b.events) scores(e + 2);
        if constexpr (NG == 1) commit(on, pvdone);
        if (!both || buf) {
          commit(on, &vempty[vslot]);
          if (++vslot == VS) vslot = 0, vphase ^= 1u;
        }
        if (e + NG >= b.events) commit(on, &ofull[NG == 2 ? buf : 0]);
      }
      advance(b.tiles);
    }
    commit(on, fin);  // every MMA has finished before TMEM is released
    if (lane == 0 && !mbar_wait_bounded(fin, 0)) atomicOr(p.b.err, kErrWaitTimeout);
    __syncwarp();
  } else if (warp <= NG * 4 + 2) {
    // ---------------------------------------------------------------- K copies, V copies
    const bool is_v = warp == NG * 4 + 2;
    const int slots = is_v ? VS : KS;
    uint64_t *full = is_v ? vfull : kfull, *empty = is_v ? vempty : kempty;
    const uint32_t base = smem_u32(is_v ? s_v : s_k);
    const CUtensorMap* map = is_v ? &vmap : &kmap;
    const int box_rows = min(1 << p.b.page_shift, KT);
    const int boxes = KT / box_rows * (D / 64);  // at most 16: a lane each
    const int blk = static_cast<int>(lane) % (D / 64), part = static_cast<int>(lane) / (D / 64);
    uint32_t n = 0;
    bool ok = true;
    while (ok && at < line.end) {
      const Block b = block_of<D, ROWS>(p, line, it, at);
      const int32_t* tab = p.b.table + static_cast<int64_t>(it.seq) * p.b.max_pages;
      for (int t = 0; ok && t < b.tiles; ++t, ++n) {
        const uint32_t slot = n % slots;
        const int key = (b.tile0 + t) * KT + part * box_rows;
        int id = -1;
        if (static_cast<int>(lane) < boxes && key < it.total_keys) {
          id = tab[key >> p.b.page_shift];
          if (id < 0 || id >= p.b.pages) {
            atomicOr(p.b.err, kErrBadShape);
            id = p.b.pages;  // past the map: the box arrives as zeros, as in the few-row kernel
          }
        }
        const uint32_t loads = __popc(__ballot_sync(0xFFFFFFFFu, id >= 0));
        if (n >= static_cast<uint32_t>(slots))
          ok = wait_bar(&empty[slot], (n / slots - 1) & 1u, abort_flag, p.b.err);
        ok = __all_sync(0xFFFFFFFFu, ok);
        if (!ok) break;
        if (lane == 0) mbar_arrive_expect_tx(&full[slot], loads * box_rows * 128);
        if (id >= 0)
          tma_box(base + slot * S::kTile + blk * (KT * 128) + part * box_rows * 128, map, blk * 64,
                  key & ((1 << p.b.page_shift) - 1), it.kv_head, id, &full[slot]);
      }
      advance(b.tiles);
    }
    // no copy may outlive the CTA: wait (bounded) for the last fill of every slot
    const uint32_t last = min(n, static_cast<uint32_t>(slots));
    for (uint32_t i = 1; i <= last; ++i) {
      const uint32_t f = n - i;
      if (!mbar_wait_bounded(&full[f % slots], (f / slots) & 1u)) atomicOr(p.b.err, kErrWaitTimeout);
    }
    __syncwarp();
  } else {
    // ---------------------------------------------------------------- V cleaning
    uint32_t n = 0;
    bool ok = true;
    for (uint32_t serial = 0; ok && at < line.end; ++serial) {
      const Block b = block_of<D, ROWS>(p, line, it, at);
      for (int t = 0; ok && t < b.tiles; ++t, ++n) {
        const uint32_t slot = n % VS;
        ok = wait_bar(&vfull[slot], (n / VS) & 1u, abort_flag, p.b.err);
        ok = __all_sync(0xFFFFFFFFu, ok);
        if (!ok) break;
        const int key0 = (b.tile0 + t) * KT;
        if (key0 + KT > b.full_keys) {
          // only the slots that some row does not see: a lane takes a 16-byte chunk of every fourth of them, in all
          // 64-column blocks, kAhead slots in flight (one at a time, the last tile of a block waited 7k clocks on this)
          constexpr int kAhead = 4, kBlocks = D / 64;
          uint8_t* tile = s_v + slot * S::kTile + (lane & 7u) * 16;
          const int r0 = max(0, b.full_keys - key0) + static_cast<int>(lane >> 3), end = min(KT, it.total_keys - key0);
          bool odd = false;
          for (int r = r0; r < end; r += 4 * kAhead) {
            uint4 u[kAhead][kBlocks];
#pragma unroll
            for (int i = 0; i < kAhead; ++i)
#pragma unroll
              for (int c = 0; c < kBlocks; ++c) {
                u[i][c] = make_uint4(0u, 0u, 0u, 0u);
                if (r + 4 * i < end) u[i][c] = *reinterpret_cast<const uint4*>(tile + (c * KT + r + 4 * i) * 128);
              }
#pragma unroll
            for (int i = 0; i < kAhead; ++i)
#pragma unroll
              for (int c = 0; c < kBlocks; ++c)
                if (odd2<BF16>(u[i][c].x) || odd2<BF16>(u[i][c].y) || odd2<BF16>(u[i][c].z) || odd2<BF16>(u[i][c].w)) {
                  odd = true;
                  *reinterpret_cast<uint4*>(tile + (c * KT + r + 4 * i) * 128) =
                      make_uint4(zero_odd2<BF16>(u[i][c].x), zero_odd2<BF16>(u[i][c].y), zero_odd2<BF16>(u[i][c].z),
                                 zero_odd2<BF16>(u[i][c].w));
                }
          }
          for (int r = max(end, 0) + static_cast<int>(lane >> 3); r < KT; r += 4)  // past the sequence
#pragma unroll
            for (int c = 0; c < kBlocks; ++c) *reinterpret_cast<uint4*>(tile + (c * KT + r) * 128) = make_uint4(0u, 0u, 0u, 0u);
          if (odd) s_odd[serial & 7u] = serial + 1u;
          fence_proxy_async_smem();
          __syncwarp();
        }
        if (lane == 0) mbar_arrive(&vclean[slot]);
      }
      advance(b.tiles);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == NG * 4) {
    tc_fence_after();
    tmem_dealloc(tmem, S::kTmem);
  }
}

// ------------------------------------------------------------------ host

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeFn encode_fn() {
  static const EncodeFn fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &found) != cudaSuccess ||
        found != cudaDriverEntryPointSuccess)
      f = nullptr;
    return reinterpret_cast<EncodeFn>(f);
  }();
  return fn;
}

// The layer's K or V as [pages][kv_heads][page_size][dim], in boxes of 64 columns by min(page_size, key tile) rows.
bool encode(CUtensorMap& map, void* base, const AttnParams& p, int dim, int tile_keys) {
  const EncodeFn fn = encode_fn();
  if (!fn) return false;
  const cuuint64_t page = 1ull << p.b.page_shift;
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(dim), page, static_cast<cuuint64_t>(p.b.kv_heads),
                              static_cast<cuuint64_t>(p.b.pages)};
  // (a dimension of one takes no steps: its stride need not mean anything)
  const cuuint64_t row = static_cast<cuuint64_t>(p.b.token_stride) * 2;
  const cuuint64_t strides[3] = {row, p.b.kv_heads > 1 ? static_cast<cuuint64_t>(p.b.head_stride) * 2 : row,
                                 p.b.pages > 1 ? static_cast<cuuint64_t>(p.b.page_stride) * 2 : row};
  const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(page < static_cast<cuuint64_t>(tile_keys) ? page : tile_keys), 1, 1};
  const cuuint32_t step[4] = {1, 1, 1, 1};
  return fn(&map, p.bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, base, dims, strides, box,
            step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, int ROWS>
cudaError_t launch_dim(const AttnParams& p, int sms, size_t partial_floats, cudaStream_t st) {
  using S = TcShape<D, ROWS>;
  static KernelSetup setup[2];
  auto kern = p.bf16 ? attn_tc_kernel<D, ROWS, true> : attn_tc_kernel<D, ROWS, false>;
  cudaError_t e = kernel_setup(setup[p.bf16 ? 1 : 0], kern, S::kThreads, S::kSmem);
  if (e != cudaSuccess) return e;
  CUtensorMap kmap, vmap;
  if (!encode(kmap, p.b.k, p, D, S::KT) || !encode(vmap, p.b.v, p, D, S::KT)) return cudaErrorInvalidValue;
  const int64_t blocks = (static_cast<int64_t>(p.max_rows) * p.group + S::kRows - 1) / S::kRows;
  const int64_t tiles = static_cast<int64_t>(p.b.nseq) * p.b.kv_heads * blocks * ((p.max_context + S::KT - 1) / S::KT);
  int64_t grid = sms;
  if (grid > tiles) grid = tiles;
  const int64_t fit = static_cast<int64_t>(partial_floats / (2 * S::kRows * (D + 2)));
  if (grid > fit) grid = fit;
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
  return cudaLaunchKernelEx(&cfg, kern, p, kmap, vmap);
}

}  // namespace

cudaError_t launch_attn_tc(const AttnParams& p, int dim, int sms, size_t partial_floats, cudaStream_t st) {
  // blocks of one row tile where no sequence needs two: a slot more for K and V in the second tile's place (32 sequences' 8,
  // 16 and 32-token trees over 4-8k slots: 143 / 148 / 158 us, with room for two tiles 145 / 148 / 161)
  const bool one = static_cast<int64_t>(p.max_rows) * p.group <= 128;
  switch (dim) {
    case 64: return (one ? launch_dim<64, 128> : launch_dim<64, 256>)(p, sms, partial_floats, st);
    case 128: return (one ? launch_dim<128, 128> : launch_dim<128, 256>)(p, sms, partial_floats, st);
    default: return launch_dim<256, 128>(p, sms, partial_floats, st);
  }
}

}  // namespace exl3
