// exl3_norm_rope.cu -- per-head norms of queries and keys, the position rotation, and the cache append, in one pass.
//
//   y = x / sqrt(mean(x^2) + eps) * (w + w0);   (a, b) -> (a cos t - b sin t, b cos t + a sin t),  t = position * f_i
// over q (into q_out) and k (into its cache slot); v goes to its slot as it is.  Bound by HBM: every element is read
// and written once, the arithmetic is f32 in registers and each output is rounded once.
//
// Eight elements (16 bytes of f16 / bf16) per thread, so dim / 8 neighbouring lanes hold one head: the sum of squares
// and the rotation's partner element are shuffles inside them; the row's sines and cosines stay in registers over its
// heads.  The angle is reduced to turns in f64 (its error is the
// product's rounding, also at long positions) and its sine and cosine are shared through shared memory by all heads of
// the row.
#include <cuda_runtime.h>

#include "exl3_attn.h"
#include "exl3_common.cuh"
#include "exl3_internal.h"

namespace exl3 {

namespace {

constexpr int kThreads = 256;
constexpr int kMaxRowsPerCta = 4;
constexpr int kBatch = 3;  // head vectors a thread has in flight
constexpr int64_t kOutside = -1;  // the row's slot is not in the table
constexpr int64_t kPadding = -2;  // no sequence owns the row
constexpr double kInvTwoPi = 0.15915494309189533576888;

// Eight elements as they lie in memory: 16 bytes, or 32 of f32 (WIDE).
template <bool WIDE>
struct Raw {
  uint4 u[WIDE ? 2 : 1];
};

template <bool WIDE>
__device__ __forceinline__ Raw<WIDE> load8(const void* p, int64_t at, bool vec) {
  Raw<WIDE> r;
  if (vec) {
    const uint4* s = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(p) + at * (WIDE ? 4 : 2));
#pragma unroll
    for (int i = 0; i < (WIDE ? 2 : 1); ++i) r.u[i] = s[i];
  } else if constexpr (WIDE) {
    const uint32_t* f = static_cast<const uint32_t*>(p) + at;
    r.u[0] = make_uint4(f[0], f[1], f[2], f[3]), r.u[1] = make_uint4(f[4], f[5], f[6], f[7]);
  } else {
    const uint16_t* h = static_cast<const uint16_t*>(p) + at;
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = h[2 * i] | (static_cast<uint32_t>(h[2 * i + 1]) << 16);
    r.u[0] = make_uint4(w[0], w[1], w[2], w[3]);
  }
  return r;
}

template <bool WIDE>
__device__ __forceinline__ void widen(const Raw<WIDE>& r, int32_t dt, float (&x)[8]) {
  const uint32_t w[4] = {r.u[0].x, r.u[0].y, r.u[0].z, r.u[0].w};
  if constexpr (WIDE) {
    const uint32_t v[4] = {r.u[1].x, r.u[1].y, r.u[1].z, r.u[1].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(w[i]), x[4 + i] = __uint_as_float(v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = dt == kF16 ? __half22float2(*reinterpret_cast<const __half2*>(&w[i]))
                                  : __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[i]));
      x[2 * i] = f.x, x[2 * i + 1] = f.y;
    }
  }
}

__device__ __forceinline__ void store8(void* p, int64_t at, int32_t dt, bool vec, const float (&x)[8]) {
  if (dt == kF32) {
    float* f = static_cast<float*>(p) + at;
    if (vec) {
      reinterpret_cast<float4*>(f)[0] = make_float4(x[0], x[1], x[2], x[3]);
      reinterpret_cast<float4*>(f)[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = x[i];
    }
    return;
  }
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (dt == kF16) {
      const __half2 t = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&t);
    } else {
      const __nv_bfloat162 t = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&t);
    }
  }
  uint16_t* h = static_cast<uint16_t*>(p) + at;
  if (vec) {
    *reinterpret_cast<uint4*>(h) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) h[2 * i] = static_cast<uint16_t>(w[i]), h[2 * i + 1] = static_cast<uint16_t>(w[i] >> 16);
  }
}

// One CTA per rows_per_cta rows; its threads walk a row's head vectors -- the heads of q, then of k, then of v -- kBatch
// of them in flight per thread, the first ones already under the search for the rows' slots.
template <int D, bool WIDE>
__global__ void __launch_bounds__(kThreads) norm_rope_kernel(const NormRopeParams p, int rows_per_cta) {
  constexpr int kLanes = D / 8;                    // lanes per head vector
  constexpr int kVecs = kThreads / kLanes;         // head vectors per pass of the CTA
  __shared__ float2 s_turn[kMaxRowsPerCta][D / 2]; // (cos, sin) of the row's pairs
  __shared__ __align__(16) float s_weight[2][D];   // of q and k
  __shared__ int64_t s_slot[kMaxRowsPerCta];       // the row's first cache element (or below 0)
  const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
  const int row0 = blockIdx.x * rows_per_cta;
  const int nrow = min(rows_per_cta, p.b.rows - row0);
  const int sub = static_cast<int>(threadIdx.x) % kLanes, e0 = sub * 8;  // this thread's elements e0 .. e0 + 7
  const int vecs = p.q.heads + 2 * p.b.kv_heads, passes = (vecs + kVecs - 1) / kVecs;
  const int first = static_cast<int>(threadIdx.x) / kLanes;
  const int half = p.rot_dims / 2;
  pdl_wait();

  Raw<WIDE> raw[kBatch];
  auto fetch = [&](int row, int k0) {
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int c = (k0 + u) * kVecs + first;
      if (c < vecs) {
        const bool is_q = c < p.q.heads, is_v = c >= p.q.heads + p.b.kv_heads;
        const HeadsView& in = is_q ? p.q : (is_v ? p.v : p.k);
        const int head = is_q ? c : c - p.q.heads - (is_v ? p.b.kv_heads : 0);
        raw[u] = load8<WIDE>(in.data, row * in.row_stride + head * in.head_stride + e0, in.vec != 0);
      }
    }
  };
  fetch(row0, 0);
  for (int i = static_cast<int>(threadIdx.x); i < 2 * D; i += kThreads) {
    const void* w = i < D ? p.q_weight : p.k_weight;
    if (w) s_weight[i / D][i % D] = load_act(w, i % D, p.weight_dtype) + p.weight_offset;
  }
  for (int i = static_cast<int>(warp); i < nrow; i += kThreads / 32) {
    const int row = row0 + i;
    if (row < p.b.row_start[0] || row >= p.b.row_start[p.b.nseq]) {  // padding: nothing is written for it
      if (lane == 0) s_slot[i] = kPadding;
      continue;
    }
    const int s = seq_of_row(p.b.row_start, p.b.nseq, row, lane);
    const int at = p.b.context[s] + row - p.b.row_start[s];
    const int pg = at >> p.b.page_shift;
    int id = -1;
    if (at >= 0 && pg < p.b.max_pages) id = p.b.table[static_cast<int64_t>(s) * p.b.max_pages + pg];
    const bool ok = id >= 0 && id < p.b.pages;
    if (lane == 0) {
      if (!ok) atomicOr(p.b.err, kErrBadShape);
      s_slot[i] = ok ? id * p.b.page_stride + (at & ((1 << p.b.page_shift) - 1)) * p.b.token_stride : kOutside;
    }
    const double pos = p.b.position ? p.b.position[row] : at;
    for (int f = static_cast<int>(lane); f < half; f += 32) {
      double t = pos * p.inv_freq[f] * kInvTwoPi;
      t -= rint(t);
      float2 cs;
      sincospif(2.f * static_cast<float>(t), &cs.y, &cs.x);
      s_turn[i][f] = cs;
    }
  }
  __syncthreads();

  // with split halves (half a multiple of 8) the partners of this thread's elements are all in one lane
  const int hl = half / 8;
  const bool low = sub < hl;
  const int partner = static_cast<int>(lane) - sub + (low ? sub + hl : (sub < 2 * hl ? sub - hl : sub));
  for (int i = 0; i < nrow; ++i) {
    const int row = row0 + i;
    const int64_t slot = s_slot[i];
    float2 turn[8];  // of this thread's elements (adjacent: of its four pairs)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int f = p.adjacent ? e0 / 2 + j : (low ? e0 + j : e0 + j - half);
      turn[j] = f >= 0 && f < half && (!p.adjacent || j < 4) ? s_turn[i][f] : make_float2(1.f, 0.f);
    }
    for (int k0 = 0; k0 < passes; k0 += kBatch) {
      if (i > 0 || k0 > 0) fetch(row, k0);
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        if (k0 + u >= passes) break;
        const int c = (k0 + u) * kVecs + first;
        const bool on = c < vecs, is_q = c < p.q.heads, is_v = c >= p.q.heads + p.b.kv_heads;
        float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (on) widen<WIDE>(raw[u], p.q.dtype, x);
        float ss = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) ss += x[j] * x[j];
#pragma unroll
        for (int d = 1; d < kLanes; d <<= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, d);
        if (!is_v && (is_q ? p.q_weight : p.k_weight)) {
          const float r = 1.f / sqrtf(ss * (1.f / D) + p.eps);
          const float4* w = reinterpret_cast<const float4*>(&s_weight[is_q ? 0 : 1][e0]);
          const float4 w0 = w[0], w1 = w[1];
          x[0] *= r * w0.x, x[1] *= r * w0.y, x[2] *= r * w0.z, x[3] *= r * w0.w;
          x[4] *= r * w1.x, x[5] *= r * w1.y, x[6] *= r * w1.z, x[7] *= r * w1.w;
        }
        if (p.adjacent) {
          if (!is_v) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float a = x[2 * j], b = x[2 * j + 1];
              x[2 * j] = a * turn[j].x - b * turn[j].y, x[2 * j + 1] = b * turn[j].x + a * turn[j].y;
            }
          }
        } else if (half) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float o = __shfl_sync(0xFFFFFFFFu, x[j], partner);
            if (!is_v && sub < 2 * hl) x[j] = low ? x[j] * turn[j].x - o * turn[j].y : x[j] * turn[j].x + o * turn[j].y;
          }
        }
        if (!on || slot == kPadding) continue;
        if (is_q) {
          store8(p.out.data, row * p.out.row_stride + c * p.out.head_stride + e0, p.out.dtype, p.out.vec != 0, x);
        } else if (slot >= 0) {
          const int head = c - p.q.heads - (is_v ? p.b.kv_heads : 0);
          store8(is_v ? p.b.v : p.b.k, slot + head * p.b.head_stride + e0, p.cache_dtype, true, x);
        }
      }
    }
  }
}

}  // namespace

cudaError_t launch_norm_rope(const NormRopeParams& p, int sms, cudaStream_t st) {
  if (p.b.rows <= 0) return cudaSuccess;
  const int rpc = p.b.rows >= kMaxRowsPerCta * 4 * sms ? kMaxRowsPerCta : 1;
  const dim3 grid((p.b.rows + rpc - 1) / rpc), block(kThreads);
  const bool wide = p.q.dtype == kF32;
  switch (p.dim) {
    case 64: return launch_pdl_k(wide ? norm_rope_kernel<64, true> : norm_rope_kernel<64, false>, grid, block, st, p, rpc);
    case 128: return launch_pdl_k(wide ? norm_rope_kernel<128, true> : norm_rope_kernel<128, false>, grid, block, st, p, rpc);
    default: return launch_pdl_k(wide ? norm_rope_kernel<256, true> : norm_rope_kernel<256, false>, grid, block, st, p, rpc);
  }
}

}  // namespace exl3
