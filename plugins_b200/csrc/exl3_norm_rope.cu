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
// the row.  Measured: 8192 rows of 48 128-wide heads, bf16: 56 us in a graph (3.6 TB/s; the same path as a bare copy 45 us,
// one call between events 63).
#include <cuda_runtime.h>

#include "exl3_attn.h"
#include "exl3_common.cuh"
#include "exl3_internal.h"

namespace exl3 {

namespace {

constexpr int kThreads = 256;
// Measured at 8192 rows of 48 heads: 2 / 4 / 6 / 8 / 16 rows 74 / 64 / 68 / 63 / 72 us.  The steps are those of the waves (9.2,
// 4.6, 3.1, 2.3, 1.2): no number is best for every count of rows; 8 pays the search and the fill once for enough of them.
constexpr int kMaxRowsPerCta = 8;
constexpr int kCtasPerSm = 3;
constexpr int kDepth = 2;  // rows a thread has in flight
// Head vectors a thread has in flight.  Measured at 8190 rows, 2 / 3 / 4 of them: 48 vectors of 128, bf16, which are three
// passes, 70 / 63 / 74 us; 32 of them 47 / 51 / 61; 64 of them 80 / 90 / 88; 32 f32 vectors of 256, four passes, 121 / 155 /
// 172.  So 3 where it divides the passes, else 2 would be the better: one number serves all as yet.
constexpr int kBatch = 3;
constexpr int64_t kOutside = -1;  // the row's slot is not in the table
constexpr int64_t kPadding = -2;  // no sequence owns the row
constexpr double kInvTwoPi = 0.15915494309189533576888;

// Eight elements as they lie in memory: 16 bytes, or 32 of f32 (WIDE).
template <bool WIDE>
struct Raw {
  uint4 u[WIDE ? 2 : 1];
};

template <bool WIDE>
__device__ __forceinline__ Raw<WIDE> load8(const void* p) {  // element by element: any alignment
  Raw<WIDE> r;
  if constexpr (WIDE) {
    const uint32_t* f = static_cast<const uint32_t*>(p);
    r.u[0] = make_uint4(f[0], f[1], f[2], f[3]), r.u[1] = make_uint4(f[4], f[5], f[6], f[7]);
  } else {
    const uint16_t* h = static_cast<const uint16_t*>(p);
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = h[2 * i] | (static_cast<uint32_t>(h[2 * i + 1]) << 16);
    r.u[0] = make_uint4(w[0], w[1], w[2], w[3]);
  }
  return r;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

// Two f32 in a register pair: one instruction for both (the kernel is near its issue rate).
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
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

template <bool WIDE>
__device__ __forceinline__ void widen(const Raw<WIDE>& r, int32_t dt, uint64_t (&x)[4]) {
  const uint32_t w[4] = {r.u[0].x, r.u[0].y, r.u[0].z, r.u[0].w};
  if constexpr (WIDE) {
    const uint32_t v[4] = {r.u[1].x, r.u[1].y, r.u[1].z, r.u[1].w};
    x[0] = f2(__uint_as_float(w[0]), __uint_as_float(w[1])), x[1] = f2(__uint_as_float(w[2]), __uint_as_float(w[3]));
    x[2] = f2(__uint_as_float(v[0]), __uint_as_float(v[1])), x[3] = f2(__uint_as_float(v[2]), __uint_as_float(v[3]));
  } else if (dt == kF16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      x[i] = f2(f.x, f.y);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = f2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xFFFF0000u));
  }
}

__device__ __forceinline__ void store8(void* p, int32_t dt, bool vec, const uint64_t (&x)[4]) {
  float a[4], b[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) f2_split(x[i], a[i], b[i]);
  if (dt == kF32) {
    float* f = static_cast<float*>(p);
    if (vec) {
      reinterpret_cast<float4*>(f)[0] = make_float4(a[0], b[0], a[1], b[1]);
      reinterpret_cast<float4*>(f)[1] = make_float4(a[2], b[2], a[3], b[3]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) f[2 * i] = a[i], f[2 * i + 1] = b[i];
    }
    return;
  }
  uint32_t w[4];
  if (dt == kF16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 t = __floats2half2_rn(a[i], b[i]);
      w[i] = *reinterpret_cast<const uint32_t*>(&t);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 t = __floats2bfloat162_rn(a[i], b[i]);
      w[i] = *reinterpret_cast<const uint32_t*>(&t);
    }
  }
  uint16_t* h = static_cast<uint16_t*>(p);
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
__global__ void __launch_bounds__(kThreads, kCtasPerSm) norm_rope_kernel(const NormRopeParams p, int rows_per_cta) {
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

  // this thread's head vectors of a batch of passes: where a row's elements are, and go (k and v: in the row's slot)
  enum : uint32_t { kOff = 0, kQ = 1, kK = 2, kV = 3 };
  uint32_t kind[kBatch];
  const uint8_t* src[kBatch];
  int64_t src_row[kBatch];  // bytes
  uint8_t* dst[kBatch];
  constexpr int kIn = WIDE ? 4 : 2;
  auto place = [&](int k0) {
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int c = (k0 + u) * kVecs + first;
      kind[u] = c >= vecs ? kOff : (c < p.q.heads ? kQ : (c < p.q.heads + p.b.kv_heads ? kK : kV));
      const HeadsView& in = kind[u] == kV ? p.v : (kind[u] == kK ? p.k : p.q);
      const int head = kind[u] == kV ? c - p.q.heads - p.b.kv_heads : (kind[u] == kK ? c - p.q.heads : c);
      src[u] = static_cast<const uint8_t*>(in.data) + (row0 * in.row_stride + head * in.head_stride + e0) * kIn;
      src_row[u] = in.row_stride * kIn;
      if (kind[u] == kQ)
        dst[u] = static_cast<uint8_t*>(p.out.data) +
                 (row0 * p.out.row_stride + head * p.out.head_stride + e0) * (p.out.dtype == kF32 ? 4 : 2);
      else
        dst[u] = reinterpret_cast<uint8_t*>((kind[u] == kV ? p.b.v : p.b.k) + head * p.b.head_stride + e0);
    }
  };
  // a thread's elements of the next kDepth rows, in shared memory that no other thread touches: registers for them
  // would halve the CTAs on an SM
  extern __shared__ __align__(16) uint8_t s_ahead[];
  constexpr int kRaw = sizeof(Raw<WIDE>);
  const bool vec = p.q.vec && p.k.vec && p.v.vec;
  auto ahead = [&](int stage, int u) { return s_ahead + ((stage * kBatch + u) * kThreads + threadIdx.x) * kRaw; };
  auto fetch = [&](int i) {
    if (vec && i < nrow) {
#pragma unroll
      for (int u = 0; u < kBatch; ++u)
        if (kind[u] != kOff) {
          const uint32_t to = smem_u32(ahead(i % kDepth, u));
          cp_async16(to, src[u]);
          if constexpr (WIDE) cp_async16(to + 16, src[u] + 16);
          src[u] += src_row[u];
        }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  auto start = [&](int k0) {
    place(k0);
#pragma unroll
    for (int d = 0; d < kDepth; ++d) fetch(d);
  };
  start(0);
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
    const int64_t at = static_cast<int64_t>(p.b.context[s]) + row - p.b.row_start[s];
    const int64_t pg = at >> p.b.page_shift;
    int id = -1;
    if (at >= 0 && pg < p.b.max_pages) id = p.b.table[static_cast<int64_t>(s) * p.b.max_pages + pg];
    const bool ok = id >= 0 && id < p.b.pages;
    if (lane == 0) {
      if (!ok) atomicOr(p.b.err, kErrBadShape);
      s_slot[i] = ok ? id * p.b.page_stride + (at & ((1 << p.b.page_shift) - 1)) * p.b.token_stride : kOutside;
    }
    const double pos = p.b.position ? p.b.position[row] : static_cast<double>(at);
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
  const uint32_t head_mask = (kLanes == 32 ? 0xFFFFFFFFu : (1u << (kLanes % 32)) - 1u) << (lane & ~static_cast<uint32_t>(kLanes - 1));
  const int partner = static_cast<int>(lane) - sub + (low ? sub + hl : (sub < 2 * hl ? sub - hl : sub));
  const int64_t out_row = p.out.row_stride * (p.out.dtype == kF32 ? 4 : 2);
  for (int k0 = 0; k0 < passes; k0 += kBatch) {
    if (k0 > 0) start(k0);
    for (int i = 0; i < nrow; ++i) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kDepth - 1) : "memory");
      Raw<WIDE> raw[kBatch];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        if (vec) raw[u] = *reinterpret_cast<const Raw<WIDE>*>(ahead(i % kDepth, u));
        else if (kind[u] != kOff) raw[u] = load8<WIDE>(src[u] + i * src_row[u]);
      }
      fetch(i + kDepth);
      const int64_t slot = s_slot[i];
      // the sines and cosines of this thread's elements, as the packed products take them
      uint64_t tc[4], ts[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int f = e0 / 2 + j, h = low ? e0 + 2 * j : e0 + 2 * j - half;
        float2 a = make_float2(1.f, 0.f), b = a;
        if (p.adjacent) {
          if (f < half) a = b = s_turn[i][f];
          tc[j] = f2(a.x, a.x), ts[j] = f2(-a.y, a.y);
        } else {
          if (h >= 0 && h < half) a = s_turn[i][h], b = s_turn[i][h + 1];
          tc[j] = f2(a.x, b.x), ts[j] = low ? f2(-a.y, -b.y) : f2(a.y, b.y);
        }
      }
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        if (k0 + u >= passes) break;
        const bool is_q = kind[u] == kQ, qk = is_q || kind[u] == kK;
        uint64_t x[4];  // pairs
        widen<WIDE>(raw[u], p.q.dtype, x);
        if (__any_sync(0xFFFFFFFFu, qk)) {
          if (is_q ? p.q_weight != nullptr : p.k_weight != nullptr) {
            uint64_t s2 = mul2(x[0], x[0]);
#pragma unroll
            for (int j = 1; j < 4; ++j) s2 = fma2(x[j], x[j], s2);
            float ss, sb;
            f2_split(s2, ss, sb);
            ss += sb;
            const uint32_t mask = head_mask;
#pragma unroll
            for (int d = 1; d < kLanes; d <<= 1) ss += __shfl_xor_sync(mask, ss, d);
            if (qk) {
              const float r = rsqrtf(ss * (1.f / D) + p.eps);
              const ulonglong2* w = reinterpret_cast<const ulonglong2*>(&s_weight[is_q ? 0 : 1][e0]);
              const ulonglong2 w0 = w[0], w1 = w[1];
              const uint64_t r2 = f2(r, r);
              x[0] = mul2(x[0], mul2(r2, w0.x)), x[1] = mul2(x[1], mul2(r2, w0.y));
              x[2] = mul2(x[2], mul2(r2, w1.x)), x[3] = mul2(x[3], mul2(r2, w1.y));
            }
          }
          if (p.adjacent) {
            if (qk) {
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                float a, b;
                f2_split(x[j], a, b);
                x[j] = fma2(x[j], tc[j], mul2(f2(b, a), ts[j]));
              }
            }
          } else if (half) {
            __syncwarp();
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const uint64_t o = __shfl_sync(0xFFFFFFFFu, x[j], partner);
              if (qk && sub < 2 * hl) x[j] = fma2(x[j], tc[j], mul2(o, ts[j]));
            }
          }
        }
        if (kind[u] == kOff || slot == kPadding) continue;
        if (is_q) store8(dst[u], p.out.dtype, p.out.vec != 0, x);
        else if (slot >= 0) store8(dst[u] + slot * 2, p.cache_dtype, true, x);
      }
#pragma unroll
      for (int u = 0; u < kBatch; ++u)
        if (kind[u] == kQ) dst[u] += out_row;
    }
  }
}

}  // namespace

namespace {

template <int D, bool WIDE>
cudaError_t launch_as(const NormRopeParams& p, int sms, cudaStream_t st) {
  static KernelSetup setup;
  auto kern = norm_rope_kernel<D, WIDE>;
  constexpr size_t kSmem = static_cast<size_t>(kDepth) * kBatch * kThreads * sizeof(Raw<WIDE>);
  cudaError_t e = kernel_setup(setup, kern, kThreads, kSmem);
  if (e != cudaSuccess) return e;
  // one wave of CTAs, each with as many rows as that takes, up to kMaxRowsPerCta: a CTA's search for its rows' slots, and
  // the fill of its ring, are paid once for them
  int rpc = (p.b.rows + kCtasPerSm * sms - 1) / (kCtasPerSm * sms);
  if (rpc > kMaxRowsPerCta) rpc = kMaxRowsPerCta;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((p.b.rows + rpc - 1) / rpc);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, p, rpc);
}

}  // namespace

cudaError_t launch_norm_rope(const NormRopeParams& p, int sms, cudaStream_t st) {
  if (p.b.rows <= 0) return cudaSuccess;
  const bool wide = p.q.dtype == kF32;
  switch (p.dim) {
    case 64: return (wide ? launch_as<64, true> : launch_as<64, false>)(p, sms, st);
    case 128: return (wide ? launch_as<128, true> : launch_as<128, false>)(p, sms, st);
    default: return (wide ? launch_as<256, true> : launch_as<256, false>)(p, sms, st);
  }
}

}  // namespace exl3
