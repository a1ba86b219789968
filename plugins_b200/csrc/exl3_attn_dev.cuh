// exl3_attn_dev.cuh -- what the paged attention kernels share: the line of work and its division over the CTAs, which
// keys a row sees, the join of an item cut between CTAs, and the 16-bit element pieces.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "exl3_attn.h"
#include "exl3_common.cuh"

namespace exl3 {

__device__ __forceinline__ float ex2(float x) {  // 2^x
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

constexpr float kLn2 = 0.6931471805599453f;

// The probabilities e^(s - m) are rounded to the element type for the product with V.  f16 has full precision down to 2^-14
// only, and thousands of keys that far below the largest can weigh as much as it does: f16's are held 2^kLift higher, which
// leaves 2^kSlack below its largest value for a running maximum that is behind (the many-row kernel's rescales O only when
// the maximum has grown by more than that).  bf16 has f32's range.  Both kernels subtract kLift from m at an item's end:
// l and o then refer to it.
template <bool BF16>
constexpr float kSlack = BF16 ? 8.f : 4.f;
template <bool BF16>
constexpr float kLift = BF16 ? 0.f : 11.f;

// ------------------------------------------------------------------ the work

// A row block of one sequence and kv head.  Its rows are (new token t, query head g) pairs, row = t * group + g.
struct Item {
  int seq, kv_head, row_block, nblocks;
  int row0, ntok;    // the sequence's first batch row and its new tokens
  int nrows;         // ntok * group
  int context, total_keys;
  int keys;          // slots any row of this block can see
  int tiles;         // of them, in tiles of the kernel's width
  int64_t first;     // the item's first tile on the line
};

// Sequence s's rows and keys, held inside the batch's arrays whatever the device values are.
__device__ __forceinline__ void item_seq(const AttnParams& p, int s, Item& it) {
  const int r0 = p.b.row_start[s], r1 = p.b.row_start[s + 1], ctx = p.b.context[s];
  it.seq = s;
  it.row0 = max(0, min(r0, p.b.rows));
  it.ntok = max(0, min(r1, p.b.rows) - it.row0);
  const int64_t room = static_cast<int64_t>(p.b.max_pages) << p.b.page_shift;
  const int64_t keys = static_cast<int64_t>(max(0, ctx)) + it.ntok;
  it.total_keys = static_cast<int>(min(keys, min(room, static_cast<int64_t>(0x7FFFFFFF))));
  it.context = max(0, min(ctx, it.total_keys));  // (keys up to here fit 32 bits; context + a row's place need not)
  it.nrows = it.ntok * p.group;
  if ((ctx < 0 || keys > room || r0 < 0 || r1 < r0 || r1 > p.b.rows) && threadIdx.x == 0) atomicOr(p.b.err, kErrBadShape);
}
// The keys a row block can see: all with a tree, up to its last token without.
__device__ __forceinline__ int block_keys(const AttnParams& p, const Item& it, int rb, int rows_per_block) {
  if (p.b.tree) return it.total_keys;
  // (rb + 1) rows_per_block is below nrows + a block: under 2^31
  const int last = min(it.ntok - 1, static_cast<int>(((rb + 1u) * rows_per_block - 1u) / static_cast<uint32_t>(p.group)));
  return it.context + min(it.total_keys - it.context, last + 1);
}

// a / b for a >= 0, b > 0: nearly always in 32 bits
__device__ __forceinline__ int64_t divide(int64_t a, int64_t b) {
  if (static_cast<uint64_t>(a | b) >> 32 == 0) return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
  return a / b;
}

// All items' tiles on one line, (sequence, kv head, row block)-major, cut into equal parts, one per CTA.
struct WorkLine {
  int64_t total, begin, end;
  int64_t share;  // tiles of a part; the first `extra` parts have one more
  int extra;
  int parts, rows_per_block, tile_keys, tile_shift;

  // the tiles of one kv head of sequence s
  __device__ __forceinline__ int64_t head_tiles(const AttnParams& p, const Item& it) const {
    const int nb = (it.nrows + rows_per_block - 1) / rows_per_block;
    if (p.b.tree) return static_cast<int64_t>(nb) * ((it.total_keys + tile_keys - 1) >> tile_shift);
    // block_keys for every block, the last token (rows_per_block (rb + 1) - 1) / group kept as quotient and remainder
    int q = (rows_per_block - 1) / p.group, r = (rows_per_block - 1) % p.group;
    const int dq = rows_per_block / p.group, dr = rows_per_block % p.group;
    int64_t t = 0;
    for (int rb = 0; rb < nb; ++rb) {
      t += (it.context + min(it.total_keys - it.context, min(it.ntok - 1, q) + 1) + tile_keys - 1) >> tile_shift;
      q += dq, r += dr;
      if (r >= p.group) ++q, r -= p.group;
    }
    return t;
  }

  // Inclusive scan of v over the CTA; scratch: 33 words.
  __device__ __forceinline__ int64_t scan(int64_t v, int64_t* scratch) const {
    const int lane = static_cast<int>(threadIdx.x & 31u), warp = static_cast<int>(threadIdx.x >> 5);
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t y = __shfl_up_sync(0xFFFFFFFFu, v, d);
      if (lane >= d) v += y;
    }
    if (lane == 31) scratch[warp] = v;
    __syncthreads();
    for (int w = 0; w < warp; ++w) v += scratch[w];
    __syncthreads();
    return v;
  }

  // Cuts the line and finds the item that holds this CTA's first tile (if it has any).
  __device__ void start(const AttnParams& p, int rows_per_block_, int tile_keys_, int64_t* scratch, Item& it) {
    int64_t mine, upto;  // this thread's sequence of the last scanned chunk
    init(p, rows_per_block_, tile_keys_, scratch, mine, upto);
    if (begin < end) locate(p, begin, it, scratch, mine, upto);
  }

  __device__ void init(const AttnParams& p, int rows_per_block_, int tile_keys_, int64_t* scratch, int64_t& mine_,
                       int64_t& upto_) {
    rows_per_block = rows_per_block_, tile_keys = tile_keys_, tile_shift = 31 - __clz(tile_keys_);
    int64_t sum = 0;
    for (int base = 0; base < p.b.nseq; base += blockDim.x) {
      const int s = base + static_cast<int>(threadIdx.x);
      mine_ = 0;
      if (s < p.b.nseq) {
        Item it;
        item_seq(p, s, it);
        mine_ = head_tiles(p, it) * p.b.kv_heads;
      }
      upto_ = sum + scan(mine_, scratch);
      if (threadIdx.x == blockDim.x - 1) scratch[32] = upto_;
      __syncthreads();
      sum = scratch[32];
      __syncthreads();
    }
    total = sum;
    parts = static_cast<int>(min(static_cast<int64_t>(gridDim.x), total));
    begin = end = 0;
    if (static_cast<int>(blockIdx.x) < parts) {
      share = divide(total, parts);
      extra = static_cast<int>(total - share * parts);
      const int c = static_cast<int>(blockIdx.x);
      begin = share * c + min(c, extra);
      end = begin + share + (c < extra ? 1 : 0);
    }
  }

  // The item that holds tile `at` of the line.
  __device__ void locate(const AttnParams& p, int64_t at, Item& it, int64_t* scratch, int64_t mine, int64_t upto) const {
    const bool one = p.b.nseq <= static_cast<int>(blockDim.x);  // init's scan is the whole
    int64_t sum = 0;
    for (int base = 0; base < p.b.nseq; base += blockDim.x) {
      const int s = base + static_cast<int>(threadIdx.x);
      if (!one) {
        mine = 0;
        if (s < p.b.nseq) {
          Item o;
          item_seq(p, s, o);
          mine = head_tiles(p, o) * p.b.kv_heads;
        }
        upto = sum + scan(mine, scratch);
      }
      if (threadIdx.x == blockDim.x - 1) scratch[32] = upto;
      if (at < upto && at >= upto - mine) scratch[33] = s, scratch[34] = upto - mine;
      __syncthreads();
      sum = scratch[32];
      if (at < sum) break;
      __syncthreads();
    }
    const int s = static_cast<int>(scratch[33]);
    const int64_t first = scratch[34];
    __syncthreads();
    item_seq(p, s, it);
    it.nblocks = (it.nrows + rows_per_block - 1) / rows_per_block;
    const int64_t per_head = head_tiles(p, it);
    it.kv_head = static_cast<int>(divide(at - first, per_head));
    it.first = first + it.kv_head * per_head;
    it.row_block = 0;
    set_block(p, it);
    if (p.b.tree) {  // blocks of one length
      it.row_block = static_cast<int>(divide(at - it.first, it.tiles));
      it.first += static_cast<int64_t>(it.row_block) * it.tiles;
      set_block(p, it);
    }
    while (at >= it.first + it.tiles) {
      it.first += it.tiles;
      ++it.row_block;
      set_block(p, it);
    }
  }
  __device__ __forceinline__ void set_block(const AttnParams& p, Item& it) const {
    it.keys = block_keys(p, it, it.row_block, rows_per_block);
    it.tiles = (it.keys + tile_keys - 1) >> tile_shift;
  }
  // The item after `it` (there is one).
  __device__ __forceinline__ void next(const AttnParams& p, Item& it) const {
    it.first += it.tiles;
    if (++it.row_block == it.nblocks) {
      it.row_block = 0;
      if (++it.kv_head == p.b.kv_heads) {
        it.kv_head = 0;
        int s = it.seq;
        do item_seq(p, ++s, it);
        while (it.ntok == 0 && s + 1 < p.b.nseq);
        it.nblocks = (it.nrows + rows_per_block - 1) / rows_per_block;
      }
    }
    set_block(p, it);
  }

  // The CTA whose part holds tile t.
  __device__ __forceinline__ int part_of(int64_t t) const {
    const int64_t longer = (share + 1) * extra;  // tiles of the parts with one more
    return t < longer ? static_cast<int>(divide(t, share + 1)) : extra + static_cast<int>(divide(t - longer, share));
  }

  // This CTA's partial of an item it does not hold whole: slot 1 when the item began in an earlier part, else slot 0.
  // A slot is [rows][D] o, then [rows] (m, l).
  __device__ __forceinline__ float* slot(const AttnParams& p, int floats, bool began_before) const {
    return p.partials + (static_cast<int64_t>(blockIdx.x) * 2 + (began_before ? 1 : 0)) * floats;
  }

  // After this CTA wrote its slot: the last of the item's CTAs joins them all, in key order.  Called by the CTA's first
  // `threads` threads; sync() joins them.
  template <int D, bool BF16, typename Sync>
  __device__ void join(const AttnParams& p, const Item& it, int slot_rows, int rows, int* s_word, int threads,
                       Sync&& sync) const;
};

// Whether new token `tok` of the item's sequence sees slot `key`.
__device__ __forceinline__ bool sees(const PagedBatch& b, const Item& it, int tok, int key) {
  if (tok >= it.ntok || key >= it.total_keys) return false;
  const int d = key - it.context;
  if (d < 0) return true;
  if (!b.tree) return d <= tok;
  if ((d >> 5) >= b.tree_words) return false;
  return (b.tree[static_cast<int64_t>(it.row0 + tok) * b.tree_words + (d >> 5)] >> (d & 31)) & 1u;
}

// ------------------------------------------------------------------ 16-bit elements

template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (BF16) {
    const __nv_bfloat162 t = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&t);
  } else {
    const __half2 t = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&t);
  }
}
template <bool BF16>
__device__ __forceinline__ float unpack1(uint32_t w, int hi) {
  const uint16_t h = static_cast<uint16_t>(hi ? w >> 16 : w);
  if constexpr (BF16) return __uint_as_float(static_cast<uint32_t>(h) << 16);
  else return __half2float(__ushort_as_half(h));
}
// whether either half of w is an infinity or NaN
template <bool BF16>
__device__ __forceinline__ bool odd2(uint32_t w) {
  constexpr uint32_t e = BF16 ? 0x7F80u : 0x7C00u;
  return (w & e) == e || (w & (e << 16)) == (e << 16);
}
template <bool BF16>
__device__ __forceinline__ uint32_t zero_odd2(uint32_t w) {
  constexpr uint32_t e = BF16 ? 0x7F80u : 0x7C00u;
  if ((w & e) == e) w &= 0xFFFF0000u;
  if ((w & (e << 16)) == (e << 16)) w &= 0xFFFFu;
  return w;
}

template <bool BF16>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (BF16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    mma_16816(d, a, b0, b1);
}

__device__ __forceinline__ void ldmatrix_x4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

// 16 bytes global -> shared, or zeros where !in (nothing is read then)
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool in) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// A warp over a [16][D] shared tile: whether this lane's share holds an infinity or NaN / those set to zero.
template <int D, bool BF16>
__device__ __forceinline__ uint32_t odd_values(uint32_t tile, uint32_t lane) {
  uint32_t any = 0;
#pragma unroll
  for (int i = 0; i < 16 * D / 64; ++i) any |= odd2<BF16>(lds32(tile + (i * 32 + lane) * 4u)) ? 1u : 0u;
  return any;
}
template <int D, bool BF16>
__device__ __forceinline__ void zero_odd_values(uint32_t tile, uint32_t lane) {
#pragma unroll 1
  for (int i = 0; i < 16 * D / 64; ++i) {
    const uint32_t a = tile + (i * 32 + lane) * 4u;
    asm volatile("st.shared.b32 [%0], %1;" ::"r"(a), "r"(zero_odd2<BF16>(lds32(a))) : "memory");
  }
}

// Eight elements of a query head, 16-bit.
__device__ __forceinline__ uint4 load_q8(const HeadsView& q, int64_t row, int64_t head, int col) {
  const uint16_t* s = static_cast<const uint16_t*>(q.data) + row * q.row_stride + head * q.head_stride + col;
  if (q.vec) return *reinterpret_cast<const uint4*>(s);
  uint4 u;
  u.x = s[0] | (static_cast<uint32_t>(s[1]) << 16), u.y = s[2] | (static_cast<uint32_t>(s[3]) << 16);
  u.z = s[4] | (static_cast<uint32_t>(s[5]) << 16), u.w = s[6] | (static_cast<uint32_t>(s[7]) << 16);
  return u;
}

// Row r of the item's block, elements d0 .. d0 + 3: o / l rounded once (zeros where the row saw nothing), and once per
// row its log-sum-exp.
template <bool BF16>
__device__ __forceinline__ void store_out4(const AttnParams& p, const Item& it, int rows_per_block, int r, int d0,
                                           const float (&acc)[4], float mx, float sum) {
  const int rr = it.row_block * rows_per_block + r, row = it.row0 + rr / p.group;
  const int h = it.kv_head * p.group + rr % p.group;
  const float f = sum == 0.f ? 0.f : 1.f / sum;
  const uint32_t w0 = pack2<BF16>(sum == 0.f ? 0.f : acc[0] * f, sum == 0.f ? 0.f : acc[1] * f);
  const uint32_t w1 = pack2<BF16>(sum == 0.f ? 0.f : acc[2] * f, sum == 0.f ? 0.f : acc[3] * f);
  uint16_t* dst = static_cast<uint16_t*>(p.out.data) + row * p.out.row_stride + h * p.out.head_stride + d0;
  if (p.out.vec) {
    *reinterpret_cast<uint2*>(dst) = make_uint2(w0, w1);
  } else {
    dst[0] = static_cast<uint16_t>(w0), dst[1] = static_cast<uint16_t>(w0 >> 16);
    dst[2] = static_cast<uint16_t>(w1), dst[3] = static_cast<uint16_t>(w1 >> 16);
  }
  if (p.lse && d0 == 0)
    p.lse[static_cast<int64_t>(row) * p.out.heads + h] = sum == 0.f ? -INFINITY : (mx + log2f(sum)) * kLn2;
}

template <int D, bool BF16, typename Sync>
__device__ void WorkLine::join(const AttnParams& p, const Item& it, int slot_rows, int rows, int* s_word, int threads,
                               Sync&& sync) const {
  const int c0 = part_of(it.first), c1 = part_of(it.first + it.tiles - 1), n = c1 - c0 + 1;
  __threadfence();
  sync();
  if (threadIdx.x == 0) {
    const uint32_t before = atomicAdd(p.counters + c0, 1u);
    const bool last = before + 1u == static_cast<uint32_t>(n);
    if (last) p.counters[c0] = 0u;
    *s_word = last;
  }
  sync();
  if (*s_word) {
    __threadfence();
    const int floats = slot_rows * (D + 2);
    for (int i = static_cast<int>(threadIdx.x); i < rows * (D / 4); i += threads) {
      const int r = i / (D / 4), d0 = (i % (D / 4)) * 4;
      float mx = -INFINITY, sum = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
      for (int c = c0; c <= c1; ++c) {  // unrolled: the loads of several slots are in flight
        const float* s = p.partials + (static_cast<int64_t>(c) * 2 + (c == c0 ? 0 : 1)) * floats;
        const float2 ml = __ldcg(reinterpret_cast<const float2*>(s + slot_rows * D + 2 * r));
        const float4 v = __ldcg(reinterpret_cast<const float4*>(s + r * D + d0));
        const float m2 = fmaxf(mx, ml.x), base = m2 == -INFINITY ? 0.f : m2;
        const float fa = ex2(mx - base), fb = ex2(ml.x - base);
        acc[0] = acc[0] * fa + v.x * fb, acc[1] = acc[1] * fa + v.y * fb;
        acc[2] = acc[2] * fa + v.z * fb, acc[3] = acc[3] * fa + v.w * fb;
        sum = sum * fa + ml.y * fb;
        mx = m2;
      }
      store_out4<BF16>(p, it, slot_rows, r, d0, acc, mx, sum);
    }
  }
  sync();
}

}  // namespace exl3
