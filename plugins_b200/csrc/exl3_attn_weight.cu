// exl3_attn_weight.cu -- how much every cached token was attended to: the column sums of the attention's probabilities,
// accumulated over steps (exl3_attention_weight, include/exl3_b200.h).
//
// w[s][g][j] = (j < context ? decay w[s][g][j] : 0) + sum_i sum_{h in g} exp(scale q_ih . k_j - lse_ih) over the rows i of
// sequence s that see slot j.  A thread per slot; a block of 128 slots takes the rows sixteen at a time.
#include <cuda_runtime.h>

#include "exl3_attn.h"
#include "exl3_attn_dev.cuh"
#include "exl3_common.cuh"
#include "exl3_internal.h"

namespace exl3 {

namespace {

constexpr int kThreads = 128;
constexpr int kRows = 16;

template <int D, bool BF16>
__global__ void __launch_bounds__(kThreads) weight_kernel(const WeightParams p) {
  __shared__ float s_q[kRows][D];
  __shared__ float s_lse[kRows];
  __shared__ int s_tok[kRows];
  pdl_wait();
  Item it;
  item_seq(p.a, static_cast<int>(blockIdx.y), it);
  it.kv_head = static_cast<int>(blockIdx.z);
  const PagedBatch& b = p.a.b;
  if (it.ntok == 0) return;
  for (int key0 = static_cast<int>(blockIdx.x) * kThreads; key0 < min(it.total_keys, p.slots); key0 += gridDim.x * kThreads) {
    const int key = key0 + static_cast<int>(threadIdx.x);
    int id = -1;
    if (key < it.total_keys) {
      id = b.table[static_cast<int64_t>(it.seq) * b.max_pages + (key >> b.page_shift)];
      if (id < 0 || id >= b.pages) {
        atomicOr(b.err, kErrBadShape);
        id = -1;
      }
    }
    const uint16_t* k = b.k + id * b.page_stride + (key & ((1 << b.page_shift) - 1)) * b.token_stride + it.kv_head * b.head_stride;
    float sum = 0.f;
    for (int r0 = 0; r0 < it.nrows; r0 += kRows) {
      __syncthreads();
      for (int i = static_cast<int>(threadIdx.x); i < kRows * D; i += kThreads) {
        const int r = r0 + i / D, t = r / p.a.group, h = it.kv_head * p.a.group + r % p.a.group;
        float v = 0.f;
        if (r < it.nrows)
          v = unpack1<BF16>(static_cast<const uint16_t*>(p.a.q.data)[(it.row0 + t) * p.a.q.row_stride + h * p.a.q.head_stride + i % D], 0);
        s_q[i / D][i % D] = v;
        if (i % D == 0) {
          s_tok[i / D] = r < it.nrows ? t : it.ntok;
          const float l = r < it.nrows ? p.lse[static_cast<int64_t>(it.row0 + t) * p.a.q.heads + h] : 0.f;
          s_lse[i / D] = l == -INFINITY ? INFINITY : l * 1.4426950408889634f;
        }
      }
      __syncthreads();
      float dot[kRows];
#pragma unroll
      for (int r = 0; r < kRows; ++r) dot[r] = 0.f;
      if (id >= 0) {
        for (int d = 0; d < D; d += 2) {
          const uint32_t u = *reinterpret_cast<const uint32_t*>(k + d);
          const float x = unpack1<BF16>(u, 0), y = unpack1<BF16>(u, 1);
#pragma unroll
          for (int r = 0; r < kRows; ++r) dot[r] = fmaf(s_q[r][d + 1], y, fmaf(s_q[r][d], x, dot[r]));
        }
      }
#pragma unroll
      for (int r = 0; r < kRows; ++r)
        if (sees(b, it, s_tok[r], key)) sum += ex2(fmaf(dot[r], p.a.scale_log2, -s_lse[r]));
    }
    if (key < it.total_keys && key < p.slots) {
      float* w = p.w + it.seq * p.row_stride + it.kv_head * p.head_stride + key;
      *w = key < it.context && p.decay != 0.f ? fmaf(p.decay, *w, sum) : sum;
    }
  }
  if (it.total_keys > p.slots && threadIdx.x == 0) atomicOr(b.err, kErrBadShape);
}

template <int D>
cudaError_t launch_dim(const WeightParams& p, cudaStream_t st) {
  const int tiles = (p.a.max_context + kThreads - 1) / kThreads;
  const dim3 grid(static_cast<unsigned>(tiles < 1 ? 1 : tiles > 65535 ? 65535 : tiles), static_cast<unsigned>(p.a.b.nseq),
                  static_cast<unsigned>(p.a.b.kv_heads));
  return p.a.bf16 ? launch_pdl_k(weight_kernel<D, true>, grid, dim3(kThreads), st, p)
                  : launch_pdl_k(weight_kernel<D, false>, grid, dim3(kThreads), st, p);
}

}  // namespace

cudaError_t launch_attn_weight(const WeightParams& p, int dim, int sms, size_t partial_floats, cudaStream_t st) {
  switch (dim) {
    case 64: return launch_dim<64>(p, st);
    case 128: return launch_dim<128>(p, st);
    default: return launch_dim<256>(p, st);
  }
}

}  // namespace exl3
