// exl3_norm_rope.cu -- per-head norms of queries and keys, the position rotation, and the cache append, in one pass.
//
//   y = x / sqrt(mean(x^2) + eps) * (w + w0);   (a, b) -> (a cos t - b sin t, b cos t + a sin t),  t = position * f_i
// over q (into q_out) and k (into its cache slot); v goes to its slot as it is.  Bound by HBM: every element is read
// and written once, the arithmetic is f32 in registers and each output is rounded once.
//
// Eight elements (16 bytes of f16 / bf16) per thread, so dim / 8 neighbouring lanes hold one head: the sum of squares
// and the rotation's partner element are shuffles inside them.  The angle is reduced to turns in f64 (its error is the
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
constexpr int64_t kOutside = -1;  // the row's slot is not in the table
constexpr int64_t kPadding = -2;  // no sequence owns the row
constexpr double kInvTwoPi = 0.15915494309189533576888;

__device__ __forceinline__ void load8(const void* p, int64_t at, int32_t dt, bool vec, float (&x)[8]) {
  if (dt == kF32) {
    const float* f = static_cast<const float*>(p) + at;
    if (vec) {
      const float4 a = reinterpret_cast<const float4*>(f)[0], b = reinterpret_cast<const float4*>(f)[1];
      x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = f[i];
    }
    return;
  }
  uint32_t w[4];
  const uint16_t* h = static_cast<const uint16_t*>(p) + at;
  if (vec) {
    const uint4 u = *reinterpret_cast<const uint4*>(h);
    w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = h[2 * i] | (static_cast<uint32_t>(h[2 * i + 1]) << 16);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = dt == kF16 ? __half22float2(*reinterpret_cast<const __half2*>(&w[i]))
                                : __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[i]));
    x[2 * i] = f.x, x[2 * i + 1] = f.y;
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

// One CTA per rows_per_cta rows; its threads walk the rows' (row, head) vectors: the heads of q, then of k, then of v.
template <int D>
__global__ void __launch_bounds__(kThreads) norm_rope_kernel(const NormRopeParams p, int rows_per_cta) {
  constexpr int kLanes = D / 8;                    // lanes per head vector
  constexpr int kVecs = kThreads / kLanes;         // head vectors per pass of the CTA
  __shared__ float2 s_turn[kMaxRowsPerCta][D / 2]; // (cos, sin) of the row's pairs
  __shared__ int64_t s_slot[kMaxRowsPerCta];       // the row's first cache element (or below 0)
  const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
  const int row0 = blockIdx.x * rows_per_cta;
  const int nrow = min(rows_per_cta, p.b.rows - row0);
  pdl_wait();
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
    for (int f = static_cast<int>(lane); f < p.rot_dims / 2; f += 32) {
      double t = pos * p.inv_freq[f] * kInvTwoPi;
      t -= rint(t);
      float2 cs;
      sincospif(2.f * static_cast<float>(t), &cs.y, &cs.x);
      s_turn[i][f] = cs;
    }
  }
  __syncthreads();
  const int sub = static_cast<int>(threadIdx.x) % kLanes, e0 = sub * 8;  // this thread's elements e0 .. e0 + 7
  const int vecs = p.q.heads + 2 * p.b.kv_heads;
  const int half = p.rot_dims / 2;
  for (int base = 0; base < nrow * vecs; base += kVecs) {
    const int item = base + static_cast<int>(threadIdx.x) / kLanes;
    const bool on = item < nrow * vecs;
    const int i = on ? item / vecs : 0, c = on ? item % vecs : 0;
    const int row = row0 + i;
    const bool is_q = c < p.q.heads, is_v = c >= p.q.heads + p.b.kv_heads;
    const int head = is_q ? c : (is_v ? c - p.q.heads - p.b.kv_heads : c - p.q.heads);
    const HeadsView& in = is_q ? p.q : (is_v ? p.v : p.k);
    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (on) load8(in.data, row * in.row_stride + head * in.head_stride + e0, in.dtype, in.vec != 0, x);
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) ss += x[j] * x[j];
#pragma unroll
    for (int d = 1; d < kLanes; d <<= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, d);
    const void* weight = is_q ? p.q_weight : p.k_weight;
    if (!is_v && weight) {
      const float r = 1.f / sqrtf(ss * (1.f / D) + p.eps);
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] *= r * (load_act(weight, e0 + j, p.weight_dtype) + p.weight_offset);
    }
    if (p.adjacent) {
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        const int f = (e0 + j) >> 1;
        if (!is_v && f < half) {
          const float2 cs = s_turn[i][f];
          const float a = x[j], b = x[j + 1];
          x[j] = a * cs.x - b * cs.y, x[j + 1] = b * cs.x + a * cs.y;
        }
      }
    } else {
      // half is a multiple of 8: the partners of this lane's elements are all in one lane
      const int hl = half / 8, first = static_cast<int>(lane) - sub;
      const bool low = sub < hl;
      const int src = first + (low ? sub + hl : (sub < 2 * hl ? sub - hl : sub));
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float o = __shfl_sync(0xFFFFFFFFu, x[j], src);
        if (!is_v && sub < 2 * hl) {
          const float2 cs = s_turn[i][low ? e0 + j : e0 + j - half];
          x[j] = low ? x[j] * cs.x - o * cs.y : x[j] * cs.x + o * cs.y;
        }
      }
    }
    if (!on || s_slot[i] == kPadding) continue;
    if (is_q) {
      store8(p.out.data, row * p.out.row_stride + head * p.out.head_stride + e0, p.out.dtype, p.out.vec != 0, x);
    } else if (s_slot[i] >= 0) {
      store8(is_v ? p.b.v : p.b.k, s_slot[i] + head * p.b.head_stride + e0, p.cache_dtype, true, x);
    }
  }
}

}  // namespace

cudaError_t launch_norm_rope(const NormRopeParams& p, int sms, cudaStream_t st) {
  if (p.b.rows <= 0) return cudaSuccess;
  const int rpc = p.b.rows >= kMaxRowsPerCta * 4 * sms ? kMaxRowsPerCta : 1;
  const dim3 grid((p.b.rows + rpc - 1) / rpc), block(kThreads);
  switch (p.dim) {
    case 64: return launch_pdl_k(norm_rope_kernel<64>, grid, block, st, p, rpc);
    case 128: return launch_pdl_k(norm_rope_kernel<128>, grid, block, st, p, rpc);
    default: return launch_pdl_k(norm_rope_kernel<256>, grid, block, st, p, rpc);
  }
}

}  // namespace exl3
