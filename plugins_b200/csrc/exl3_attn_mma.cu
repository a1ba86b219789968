// exl3_attn_mma.cu -- attention of a few rows per kv head over the paged cache (decode steps, small drafted trees).
//
// One pass over the keys with the running maximum m and sum l of a softmax (all in f32):
//   s = scale q . k,  m' = max(m, s),  l = l e^(m - m') + e^(s - m'),  o = o e^(m - m') + e^(s - m') v;   out = o / l.
// The rows that share a kv head (its query heads x the sequence's new tokens) are packed into one m16n8k16 row tile,
// so a key is read once for all of them.  Bound by HBM: K and V once, 16 x rows / 16-bit element operations against them.
//
// Work: the (sequence, kv head, row block) items' keys, in tiles of 64, form one line that the CTAs cut into equal
// parts, whatever the sequences' lengths.  A CTA's four warps take 16 keys of each tile, every warp with its own ring of
// cp.async stages (no barrier in the loop) and its own m, l, o; they are joined through shared memory at the end of an
// item, and an item cut between CTAs through the workspace, by the CTA that finishes last, in key order: the result
// does not depend on which that is.
//
// Measured: 32 sequences' single tokens over 1500-9001 slots, 32 / 8 heads of 128: 117 us in a graph (5.9 TB/s); eight of
// them 42 us, of which some 11 are the start and the join; one token over 301 slots 9 us in a graph, 12 us a call.
#include <cuda_runtime.h>

#include "exl3_attn.h"
#include "exl3_attn_dev.cuh"
#include "exl3_common.cuh"
#include "exl3_internal.h"

namespace exl3 {

namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kGroupKeys = 16;                   // keys a warp takes per step: inside one page
constexpr int kTileKeys = kWarps * kGroupKeys;

template <int D>
struct MmaShape {
  static constexpr int kRows = 16;
  static constexpr int kGroupBytes = kGroupKeys * D * 2;       // K or V of one warp step
  static constexpr int kStages = D == 64 ? 6 : 3;
  static constexpr int kRing = kStages * 2 * kGroupBytes;      // per warp
  static constexpr int kQBytes = kRows * D * 2;
  static constexpr int kSmem = kWarps * kRing + kQBytes + kRows * kWarps * 8 + 64;
  static_assert(kWarps * kRing >= kWarps * kRows * D * 4, "the join of the warps' o reuses the ring");
};

// Byte offset of 16-byte chunk c of row r in a [rows][D] 16-bit tile: chunks rotated by the row, so eight rows' same
// chunk lie in eight different bank groups.
template <int D>
__device__ __forceinline__ uint32_t tile_off(uint32_t r, uint32_t c) {
  return r * (D * 2) + ((c ^ (r & 7u)) << 4);
}

template <int D, bool BF16>
__global__ void __launch_bounds__(kThreads) attn_mma_kernel(const AttnParams p) {
  using S = MmaShape<D>;
  extern __shared__ __align__(128) uint8_t smem[];
  uint8_t* s_q = smem + kWarps * S::kRing;
  float2* s_ml = reinterpret_cast<float2*>(s_q + S::kQBytes);  // [rows][warps]
  int* s_word = reinterpret_cast<int*>(s_ml + S::kRows * kWarps);
  const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
  const uint32_t g = lane >> 2, q4 = lane & 3u;
  pdl_wait();

  WorkLine line;
  Item it;
  line.start(p, S::kRows, kTileKeys, reinterpret_cast<int64_t*>(smem), it);
  int64_t at = line.begin, end = line.end;
  if (at >= end) return;

  const uint32_t ring = smem_u32(smem + warp * S::kRing);
  while (at < end) {
    const int tile0 = static_cast<int>(at - it.first);
    const int tiles = static_cast<int>(min(end - at, static_cast<int64_t>(it.tiles - tile0)));
    const int rows = min(S::kRows, it.nrows - it.row_block * S::kRows);
    // the item's query rows, [rows][D], into shared memory
    __syncthreads();
    for (int i = static_cast<int>(tid); i < S::kRows * (D / 8); i += kThreads) {
      const int r = i / (D / 8), c = i % (D / 8);
      uint4 u = make_uint4(0u, 0u, 0u, 0u);
      if (r < rows) {
        const int rr = it.row_block * S::kRows + r, t = rr / p.group, h = it.kv_head * p.group + rr % p.group;
        u = load_q8(p.q, it.row0 + t, h, c * 8);
      }
      *reinterpret_cast<uint4*>(s_q + tile_off<D>(static_cast<uint32_t>(r), static_cast<uint32_t>(c))) = u;
    }
    __syncthreads();

    // the query fragments stay in registers where they fit beside o
    constexpr bool kQRegs = D <= 128;
    uint32_t qa[kQRegs ? D / 16 : 1][4];
    if constexpr (kQRegs) {
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) ldmatrix_x4(smem_u32(s_q) + tile_off<D>(lane & 15u, 2u * kk + (lane >> 4)), qa[kk]);
    }

    float o[D / 8][4];
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};  // rows g and g + 8
#pragma unroll
    for (int j = 0; j < D / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;

    const int32_t* tab = p.b.table + static_cast<int64_t>(it.seq) * p.b.max_pages;
    const int page_mask = (1 << p.b.page_shift) - 1;
    auto page_at = [&](int t) {
      const int key0 = (tile0 + t) * kTileKeys + static_cast<int>(warp) * kGroupKeys;
      return t < tiles && key0 < it.keys ? tab[key0 >> p.b.page_shift] : -1;
    };
    int page = page_at(0);  // of the next tile to issue, looked up one tile ahead of its copies
    // this warp's 16 keys of tile t into ring stage st: rows past the sequence's last key are zeros
    auto issue = [&](int t, int st) {
      const int key0 = (tile0 + t) * kTileKeys + static_cast<int>(warp) * kGroupKeys;
      int id = page;
      page = page_at(t + 1);
      if (t < tiles && key0 < it.keys) {
        const bool ok = id >= 0 && id < p.b.pages;
        if (!ok) {
          if (lane == 0) atomicOr(p.b.err, kErrBadShape);
          id = 0;
        }
        const int64_t base = id * p.b.page_stride + (key0 & page_mask) * p.b.token_stride +
                             it.kv_head * p.b.head_stride;
        const uint32_t dst = ring + st * 2 * S::kGroupBytes;
        constexpr int kPer = kGroupKeys * (D / 8) / 32;  // chunks per lane, K and V each
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          const uint32_t c = (i * 32 + lane) % (D / 8), r = (i * 32 + lane) / (D / 8);
          const int64_t off = base + r * p.b.token_stride + c * 8;
          const bool in = ok && key0 + static_cast<int>(r) < it.keys;
          cp_async16(dst + tile_off<D>(r, c), p.b.k + off, in);
          cp_async16(dst + S::kGroupBytes + tile_off<D>(r, c), p.b.v + off, in);
        }
      }
      cp_async_commit();
    };
#pragma unroll
    for (int st = 0; st < S::kStages - 1; ++st) issue(st, st);

    for (int t = 0; t < tiles; ++t) {
      issue(t + S::kStages - 1, (t + S::kStages - 1) % S::kStages);
      cp_async_wait<S::kStages - 1>();
      __syncwarp();
      const int key0 = (tile0 + t) * kTileKeys + static_cast<int>(warp) * kGroupKeys;
      if (key0 < it.keys) {
        const uint32_t sk = ring + (t % S::kStages) * 2 * S::kGroupBytes, sv = sk + S::kGroupBytes;
        float s[2][4] = {};
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          uint32_t b[4];  // keys 0..7 (k low, high), keys 8..15 (k low, high)
          ldmatrix_x4(sk + tile_off<D>((lane & 7u) + ((lane >> 4) << 3), 2u * kk + ((lane >> 3) & 1u)), b);
          if constexpr (!kQRegs) ldmatrix_x4(smem_u32(s_q) + tile_off<D>(lane & 15u, 2u * kk + (lane >> 4)), qa[0]);
          mma16816<BF16>(s[0], qa[kQRegs ? kk : 0], b[0], b[1]);
          mma16816<BF16>(s[1], qa[kQRegs ? kk : 0], b[2], b[3]);
        }
        const bool tail = key0 + kGroupKeys > it.context;  // some key is not in the context: rows see it or not
        uint32_t odd = 0;                                  // a tail key's V holds an infinity or NaN
        if (tail) odd = odd_values<D, BF16>(sv, lane);
        uint32_t pa[4];
#pragma unroll
        for (int hh = 0; hh < 2; ++hh) {  // rows g and g + 8 of the row tile
          float x[4] = {s[0][2 * hh], s[0][2 * hh + 1], s[1][2 * hh], s[1][2 * hh + 1]};
#pragma unroll
          for (int j = 0; j < 4; ++j) x[j] *= p.scale_log2;
          if (tail) {
            const int r = it.row_block * S::kRows + 8 * hh + static_cast<int>(g);
            const int tok = r / p.group;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int key = key0 + (j >> 1) * 8 + static_cast<int>(q4) * 2 + (j & 1);
              if (!sees(p.b, it, tok, key)) x[j] = -INFINITY;
            }
          }
          float mx = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
          mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, 2));
          mx = fmaxf(mx, m[hh]);
          const float top = mx == -INFINITY ? 0.f : mx;  // nothing seen so far: every term below is 0
          const float base = top - kLift<BF16>;
          const float f = ex2(m[hh] - top);
          m[hh] = mx;
          float sum = 0.f;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            x[j] = ex2(x[j] - base);
            sum += x[j];
          }
          l[hh] = l[hh] * f + sum;
#pragma unroll
          for (int j = 0; j < D / 8; ++j) o[j][2 * hh] *= f, o[j][2 * hh + 1] *= f;
          // 2^kLift e^(s - m), rounded to the element type for the product with V (l keeps the f32 values)
          pa[hh] = pack2<BF16>(x[0], x[1]);
          pa[2 + hh] = pack2<BF16>(x[2], x[3]);
        }
        if (__any_sync(0xFFFFFFFFu, odd != 0u)) {
          // rare: an infinity or NaN in V reaches the rows that see its key and no others, so it cannot go through
          // the product (0 x inf = NaN); add it by hand, then zero it in shared memory
#pragma unroll 1
          for (int key = 0; key < kGroupKeys; ++key) {
            const int src = static_cast<int>((lane & ~3u) | ((key & 7u) >> 1));
#pragma unroll
            for (int hh = 0; hh < 2; ++hh) {
              const uint32_t w = __shfl_sync(0xFFFFFFFFu, key < 8 ? pa[hh] : pa[2 + hh], src);
              const float pv = unpack1<BF16>(w, key & 1);
              const int r = it.row_block * S::kRows + 8 * hh + static_cast<int>(g);
              const bool see = key0 + key < it.keys && sees(p.b, it, r / p.group, key0 + key);
#pragma unroll
              for (int j = 0; j < D / 8; ++j) {
                const uint32_t v2 = lds32(sv + tile_off<D>(static_cast<uint32_t>(key), static_cast<uint32_t>(j)) + q4 * 4u);
                const float v0 = unpack1<BF16>(v2, 0), v1 = unpack1<BF16>(v2, 1);
                if (see && !isfinite(v0)) o[j][2 * hh] += pv * v0;
                if (see && !isfinite(v1)) o[j][2 * hh + 1] += pv * v1;
              }
            }
          }
          __syncwarp();
          zero_odd_values<D, BF16>(sv, lane);
          __syncwarp();
        }
#pragma unroll
        for (int jj = 0; jj < D / 16; ++jj) {
          uint32_t b[4];  // d 16 jj .. + 7 (keys low, high), d 16 jj + 8 .. (keys low, high)
          ldmatrix_x4_trans(sv + tile_off<D>(lane & 15u, 2u * jj + (lane >> 4)), b);
          mma16816<BF16>(o[2 * jj], pa, b[0], b[1]);
          mma16816<BF16>(o[2 * jj + 1], pa, b[2], b[3]);
        }
      }
      __syncwarp();  // the stage may be refilled
    }
    cp_async_wait<0>();
    __syncthreads();

    // ---- join the four warps: m and l per row, then o scaled to the common maximum, summed in warp order
    float* s_o = reinterpret_cast<float*>(smem);  // [warps][rows][D]
#pragma unroll
    for (int hh = 0; hh < 2; ++hh) {
      float sum = l[hh];
      sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 1);
      sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 2);
      const uint32_t r = 8u * hh + g;
      if (q4 == 0) s_ml[r * kWarps + warp] = make_float2(m[hh] - kLift<BF16>, sum);
#pragma unroll
      for (int j = 0; j < D / 8; ++j)
        *reinterpret_cast<float2*>(s_o + (warp * S::kRows + r) * D + j * 8 + q4 * 2) =
            make_float2(o[j][2 * hh], o[j][2 * hh + 1]);
    }
    __syncthreads();
    const bool whole = tiles == it.tiles;
    float* slot = nullptr;
    if (!whole) slot = line.slot(p, S::kRows * (D + 2), at != it.first);  // head: began in an earlier CTA
    for (int i = static_cast<int>(tid); i < rows * (D / 4); i += kThreads) {
      const int r = i / (D / 4), d0 = (i % (D / 4)) * 4;
      float mx = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, s_ml[r * kWarps + w].x);
      const float base = mx == -INFINITY ? 0.f : mx;
      float sum = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float2 ml = s_ml[r * kWarps + w];
        const float f = ex2(ml.x - base);
        const float4 v = *reinterpret_cast<const float4*>(s_o + (w * S::kRows + r) * D + d0);
        sum += ml.y * f;
        acc[0] += v.x * f, acc[1] += v.y * f, acc[2] += v.z * f, acc[3] += v.w * f;
      }
      if (whole) {
        store_out4<BF16>(p, it, S::kRows, r, d0, acc, mx, sum);
      } else {
        *reinterpret_cast<float4*>(slot + r * D + d0) = make_float4(acc[0], acc[1], acc[2], acc[3]);
        if (d0 == 0) *reinterpret_cast<float2*>(slot + S::kRows * D + 2 * r) = make_float2(mx, sum);
      }
    }
    if (!whole) line.template join<D, BF16>(p, it, S::kRows, rows, s_word, kThreads, [] { __syncthreads(); });
    at += tiles;
    if (at < end) line.next(p, it);
  }
}

template <int D>
cudaError_t launch_dim(const AttnParams& p, int sms, size_t partial_floats, cudaStream_t st) {
  using S = MmaShape<D>;
  static KernelSetup setup[2];
  auto kern = p.bf16 ? attn_mma_kernel<D, true> : attn_mma_kernel<D, false>;
  int per_sm = 1;
  cudaError_t e = kernel_setup(setup[p.bf16 ? 1 : 0], kern, kThreads, S::kSmem, false, &per_sm, 4);
  if (e != cudaSuccess) return e;
  // as many CTAs as fit the GPU, the keys' tiles and the workspace
  const int64_t blocks = (static_cast<int64_t>(p.max_rows) * p.group + S::kRows - 1) / S::kRows;
  int64_t tiles = static_cast<int64_t>(p.b.nseq) * p.b.kv_heads * blocks * ((p.max_context + kTileKeys - 1) / kTileKeys);
  int64_t grid = static_cast<int64_t>(sms) * per_sm;
  if (grid > tiles) grid = tiles;
  const int64_t fit = static_cast<int64_t>(partial_floats / (2 * S::kRows * (D + 2)));
  if (grid > fit) grid = fit;
  if (grid < 1) grid = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = S::kSmem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, p);
}

}  // namespace

cudaError_t launch_attn_mma(const AttnParams& p, int dim, int sms, size_t partial_floats, cudaStream_t st) {
  switch (dim) {
    case 64: return launch_dim<64>(p, sms, partial_floats, st);
    case 128: return launch_dim<128>(p, sms, partial_floats, st);
    default: return launch_dim<256>(p, sms, partial_floats, st);
  }
}

}  // namespace exl3
