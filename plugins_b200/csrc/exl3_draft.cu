// exl3_draft.cu -- which drafted tokens of each sequence's tree stay, by the target's probabilities and given random
// numbers, and the token that follows them (exl3_draft_verify, include/exl3_b200.h).
//
// At a node of the path, p = softmax(logits / T) and q the drafter's probabilities.  The children are tried in turn, the
// k-th (token x) against r_k = max(p - A_k q, 0) with A_0 = 0, A_k+1 = A_k + Z_k and Z_k = sum r_k: accepted where
// u q(x) Z_k < r_k(x).  (That r_k is what the repeated r <- max(r - Z q, 0) comes to: what is cut to zero stays there.)
// Without q a rejected token simply leaves p.  The path ends at the node none of whose children is accepted; its last r
// gives the next token by its cumulative sums.
//
// One cluster per sequence walks its path, a slice of the vocabulary per CTA: the row's exponentials e^((x - m) / T), m the
// slice's own maximum, stay in shared memory as f32; the sums over them are f64, so that r, which can be a small rest of p,
// keeps what the exponentials have (an f32 sum would leave 2^-24 of all of p in it).  Each CTA sends its slice's (m, sum)
// to all others, and every CTA then takes the same decisions from the same numbers.  Only rows on the path are read.
#include <cuda_runtime.h>
#include <float.h>

#include "exl3_attn.h"
#include "exl3_common.cuh"
#include "exl3_internal.h"

namespace exl3 {

namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kCluster = 8;
constexpr double kLog2e = 1.4426950408889634;
constexpr double kNone = 0x1p-100;  // a token this far below the likeliest has no probability

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_store(void* p, int rank, double a, double b) {
  uint32_t at;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("st.shared::cluster.v2.f64 [%0], {%1, %2};" ::"r"(at), "d"(a), "d"(b) : "memory");
}

template <int DT>
struct Elem {
  using type = uint16_t;
  static constexpr int kVec = 8;  // elements of 16 bytes
};
template <>
struct Elem<EXL3_F32> {
  using type = float;
  static constexpr int kVec = 4;
};
template <int DT>
__device__ __forceinline__ float widen(typename Elem<DT>::type v) {
  if constexpr (DT == EXL3_F16) return __half2float(__ushort_as_half(v));
  else if constexpr (DT == EXL3_BF16) return __uint_as_float(static_cast<uint32_t>(v) << 16);
  else return v;
}
// A logit as it counts: NaN as -inf, +inf as the largest finite number.
__device__ __forceinline__ float logit(float x) { return x == x ? fminf(x, FLT_MAX) : -INFINITY; }
// A drafter's probability: NaN and negative numbers as 0.
template <int DT>
__device__ __forceinline__ float draft_p(const void* row, int64_t i) {
  return fmaxf(widen<DT>(static_cast<const typename Elem<DT>::type*>(row)[i]), 0.f);
}
__device__ __forceinline__ float draft_at(const void* row, int dtype, int64_t i) {
  return dtype == EXL3_F32 ? draft_p<EXL3_F32>(row, i) : dtype == EXL3_F16 ? draft_p<EXL3_F16>(row, i) : draft_p<EXL3_BF16>(row, i);
}

// 2^((x - m) c), c = c1 + c2 = log2(e) / T.  The rounding of the difference and of the product, up to 2^-24 of an
// exponent of 100, is carried along: what is left is the exponential's own.
struct Scale {
  float c1, c2;
};
__device__ __forceinline__ float power(float x, float m, Scale c) {
  if (x == -INFINITY) return 0.f;
  const float d = x - m, b = d - x, d2 = (x - (d - b)) + (-m - b);
  const float z = d * c.c1;
  if (!(z > -150.f)) return 0.f;
  const float z2 = fmaf(d, c.c1, -z) + fmaf(d, c.c2, d2 * c.c1);
  return exp2f(z) * fmaf(z2, 0.6931472f, 1.f);
}

// The elements of a slice [0, n) at `src`, by 16-byte chunks where the address allows: f(index, values, count).
template <int DT>
__device__ __forceinline__ int head_of(const typename Elem<DT>::type* src, int n) {
  constexpr int kVec = Elem<DT>::kVec;
  const int off = static_cast<int>(reinterpret_cast<uintptr_t>(src) % 16 / sizeof(typename Elem<DT>::type));
  return min(n, (kVec - off) % kVec);
}
template <int DT, typename F>
__device__ __forceinline__ void each_chunk(const typename Elem<DT>::type* src, int n, F&& f) {
  using E = Elem<DT>;
  constexpr int kVec = E::kVec;
  const int head = head_of<DT>(src, n), chunks = (n - head) / kVec, tail = head + chunks * kVec;
  const int t = static_cast<int>(threadIdx.x);
  constexpr int kAhead = 4;
  for (int i0 = t; i0 < chunks; i0 += kThreads * kAhead) {
    uint4 u[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j)
      if (i0 + j * kThreads < chunks) u[j] = *(reinterpret_cast<const uint4*>(src + head) + i0 + j * kThreads);
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      if (i0 + j * kThreads >= chunks) break;
      float v[kVec];
      const uint32_t w[4] = {u[j].x, u[j].y, u[j].z, u[j].w};
#pragma unroll
      for (int k = 0; k < kVec; ++k) {
        if constexpr (DT == EXL3_F32) v[k] = __uint_as_float(w[k]);
        else v[k] = widen<DT>(static_cast<uint16_t>(w[k / 2] >> (16 * (k & 1))));
      }
      f(head + (i0 + j * kThreads) * kVec, v, kVec);
    }
  }
  for (int i = t; i < head + (n - tail); i += kThreads) {
    const int at = i < head ? i : tail + i - head;
    float v[kVec];
    v[0] = widen<DT>(src[at]);
    f(at, v, 1);
  }
}

// The drafter's probabilities of a slice: f(index, q).
template <int DT, typename F>
__device__ __forceinline__ void each_draft_of(const DraftParams& p, int64_t row, int v0, int n, F&& f) {
  const void* q = p.draft;
  const int64_t base = row * p.draft_stride + v0;
#pragma unroll 8
  for (int i = static_cast<int>(threadIdx.x); i < n; i += kThreads) f(i, draft_p<DT>(q, base + i));
}
template <typename F>
__device__ __forceinline__ void each_draft(const DraftParams& p, int64_t row, int v0, int n, F&& f) {
  if (p.draft_dtype == EXL3_F32) each_draft_of<EXL3_F32>(p, row, v0, n, f);
  else if (p.draft_dtype == EXL3_F16) each_draft_of<EXL3_F16>(p, row, v0, n, f);
  else each_draft_of<EXL3_BF16>(p, row, v0, n, f);
}

struct Block {
  double sum[kWarps];
  double2 slice[2][kCluster];  // (maximum, sum) of every CTA's slice, sent by its owner; two, by turns
  float top[kWarps];
  int at[kWarps];
  // the walk, as warp 0 leaves it
  int command, node, owner, token, found, last;
  double a, lift, unit, target;  // A; e^((m_slice - m) / T) of this CTA's slice; 1 / the row's sum; what is left to pass
};
enum : int { kNext = 0, kStop = 1, kCut = 2 };  // on to a child; the path ends; r has to be summed

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, d);
  return v;
}

template <int DT>
__global__ void __cluster_dims__(kCluster, 1, 1) __launch_bounds__(kThreads) verify_kernel(const DraftParams p) {
  using T = typename Elem<DT>::type;
  constexpr int kVec = Elem<DT>::kVec;
  extern __shared__ __align__(16) float s_e[];  // [slice + 8]
  __shared__ Block b;
  __shared__ int s_out[kDraftMaxRows];  // the node's rejected tokens, where there is no q
  pdl_wait();
  const int tid = static_cast<int>(threadIdx.x), lane = tid & 31, warp = tid >> 5;
  const int rank = static_cast<int>(blockIdx.x) % kCluster, s = static_cast<int>(blockIdx.x) / kCluster;
  const int r0 = p.row_start[s], r1 = p.row_start[s + 1];
  const int row0 = max(0, min(r0, p.rows)), all = max(0, min(r1, p.rows) - row0), ntok = min(all, p.max_rows);
  const float temp = p.temperature ? p.temperature[s] : 1.f;
  const bool warm = temp > 0.f && temp <= FLT_MAX;
  if (tid == 0 && rank == 0 && (r0 < 0 || r1 < r0 || r1 > p.rows || all > ntok || (!warm && temp != 0.f)))
    atomicOr(p.err, kErrBadShape);
  int32_t* path = p.path + static_cast<int64_t>(s) * p.depth;
  if (ntok == 0) {  // (the whole cluster)
    if (rank == 0) {
      for (int d = tid; d < p.depth; d += kThreads) path[d] = -1;
      if (tid == 0) p.kept[s] = 0, p.token[s] = -1;
    }
    return;
  }
  Scale c{0.f, 0.f};
  if (warm) {
    const double cd = kLog2e / static_cast<double>(temp);
    c.c1 = static_cast<float>(fmin(cd, static_cast<double>(FLT_MAX)));
    c.c2 = cd < 1e30 ? static_cast<float>(cd - static_cast<double>(c.c1)) : 0.f;
  }
  const int v0 = min(rank * p.slice, p.vocab), n = min(p.vocab - v0, p.slice);
  const bool has_q = p.draft != nullptr && warm;
  int node = 0, kept = 0;
  uint32_t turn = 0;

  // This CTA's pair to all, and theirs into b.slice[the returned turn].
  auto exchange = [&](double x, double y) {
    const uint32_t which = turn++ & 1u;
    if (tid < kCluster) cluster_store(&b.slice[which][rank], tid, x, y);
    cluster_sync();
    return which;
  };
  auto block_sum = [&](double v) {  // in every thread
    v = warp_sum(v);
    if (lane == 0) b.sum[warp] = v;
    __syncthreads();
    double t = 0.0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) t += b.sum[w];
    return t;
  };

  for (;;) {
    // ---- the node's row: its maximum, its exponentials and their sum
    const int64_t row = row0 + node;
    const T* logits = static_cast<const T*>(p.logits) + row * p.logits_stride;
    const int pad = (4 - (head_of<DT>(logits + v0, n) & 3)) & 3;  // whole chunks lie on multiples of four in s_e
    const int end = pad + n;
    if (tid < pad) s_e[tid] = -INFINITY;
    if (tid < 4 && end + tid < ((end + 3) & ~3)) s_e[end + tid] = -INFINITY;
    float top = -INFINITY;
    int at = 0x7FFFFFFF;
    each_chunk<DT>(logits + v0, n, [&](int i, const float (&v)[kVec], int count) {
      float x[kVec];
#pragma unroll
      for (int k = 0; k < kVec; ++k) {
        x[k] = k < count ? logit(v[k]) : -INFINITY;
        // (a thread meets its places in ascending order, but for the few outside whole chunks, which come last)
        if (x[k] > top || (x[k] == top && i + k < at && x[k] != -INFINITY)) top = x[k], at = i + k;
      }
      if (count == 1) {
        s_e[pad + i] = x[0];
      } else {
#pragma unroll
        for (int k = 0; k < kVec; k += 4)
          *reinterpret_cast<float4*>(s_e + pad + i + k) = make_float4(x[k], x[k + 1], x[k + 2], x[k + 3]);
      }
    });
#pragma unroll
    for (int d = 16; d; d >>= 1) {
      const float o = __shfl_xor_sync(0xFFFFFFFFu, top, d);
      const int oat = __shfl_xor_sync(0xFFFFFFFFu, at, d);
      if (o > top || (o == top && oat < at)) top = o, at = oat;
    }
    if (lane == 0) b.top[warp] = top, b.at[warp] = at;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWarps; ++w)
      if (b.top[w] > top || (b.top[w] == top && b.at[w] < at)) top = b.top[w], at = b.at[w];
    double sum = 0.0;
    if (warm) {
      for (int i = tid * 4; i < end; i += kThreads * 4) {
        float4 e = *reinterpret_cast<const float4*>(s_e + i);
        e.x = power(e.x, top, c), e.y = power(e.y, top, c), e.z = power(e.z, top, c), e.w = power(e.w, top, c);
        *reinterpret_cast<float4*>(s_e + i) = e;
        sum += (static_cast<double>(e.x) + static_cast<double>(e.y)) + (static_cast<double>(e.z) + static_cast<double>(e.w));
      }
      sum = block_sum(sum);
    } else {
      sum = static_cast<double>(v0) + static_cast<double>(at);  // a greedy sequence's slice: where its maximum is
    }
    uint32_t which = exchange(static_cast<double>(top), sum);

    // ---- the children in turn: warp 0 of every CTA decides the same from the same numbers
    if (rank == 0 && tid == 0) path[kept] = node;
    ++kept;
    // warp 0: lane r holds slice r's (maximum, sum of what is left), its e^((m_r - m) / T), and r's sum over it
    double2 mine = make_double2(-INFINITY, 0.0);
    double lift = 0.0, unit = 0.0, rest = 0.0, a = 0.0, z = 1.0;
    int best = -1, tried = node + 1, rejected = 0;
    if (warp == 0) {
      if (lane < kCluster) mine = b.slice[which][lane];
      double m = mine.x;
#pragma unroll
      for (int d = 4; d; d >>= 1) m = fmax(m, __shfl_xor_sync(0xFFFFFFFFu, m, d));
      m = __shfl_sync(0xFFFFFFFFu, m, 0);
      if (warm) {
        lift = static_cast<double>(power(static_cast<float>(mine.x), static_cast<float>(m), c));
        if (lift < kNone) lift = 0.0;  // no token of the slice has a probability
        unit = 1.0 / warp_sum(mine.y * lift);
        rest = mine.y * lift * unit;
      }
      const uint32_t has = __ballot_sync(0xFFFFFFFFu, mine.x == m && m != -INFINITY);
      const double where = __shfl_sync(0xFFFFFFFFu, mine.y, __ffs(has) - 1);
      best = has ? (warm ? 0 : static_cast<int>(where)) : -1;  // -1: the row has no finite logit
      tried = best < 0 || kept >= p.depth ? ntok : tried;
    }
    for (;;) {
      if (warp == 0) {
        int command = kStop, child = 0;
        for (; command == kStop && tried < ntok; tried += 32) {
          const int i = tried + lane;
          const bool is = i < ntok && (p.parent ? p.parent[row0 + i] == node : i == node + 1);
          uint32_t left = __ballot_sync(0xFFFFFFFFu, is);
          int tok = -1;
          float x = 0.f, u = 0.f, q = 1.f;
          if (is) {
            tok = p.tokens[row0 + i];
            if (tok >= 0 && tok < p.vocab) {
              x = logit(widen<DT>(logits[tok]));
              u = p.uniform[2 * (row0 + static_cast<int64_t>(i))];
              if (has_q) q = draft_at(p.draft, p.draft_dtype, row * p.draft_stride + tok);
            } else {
              tok = -1;
            }
          }
          while (left && command == kStop) {
            const int l = __ffs(left) - 1;
            left &= left - 1;
            const int t = __shfl_sync(0xFFFFFFFFu, tok, l);
            if (t < 0) continue;  // (a token outside the vocabulary is not tried)
            child = tried + l;
            if (!warm) {
              if (t == best) command = kNext;
              continue;
            }
            const int owner = t / p.slice;
            const float e = power(__shfl_sync(0xFFFFFFFFu, x, l), static_cast<float>(__shfl_sync(0xFFFFFFFFu, mine.x, owner)), c);
            const double le = static_cast<double>(e) * __shfl_sync(0xFFFFFFFFu, lift, owner);
            const double qt = static_cast<double>(__shfl_sync(0xFFFFFFFFu, q, l));
            double rt = le < kNone ? 0.0 : le * unit;
            if (has_q) {
              if (a > 0.0) rt = fmax(rt - a * qt, 0.0);
            } else {
              bool gone = false;
              for (int j = lane; j < rejected; j += 32) gone |= s_out[j] == t;
              if (__any_sync(0xFFFFFFFFu, gone)) continue;  // its sibling took it out of p
            }
            if (static_cast<double>(__shfl_sync(0xFFFFFFFFu, u, l)) * qt * z < rt) {
              command = kNext;
            } else if (has_q) {
              a += z;
              command = kCut;
            } else {
              if (lane == 0) {
                s_out[rejected] = t;
                if (owner == rank) s_e[pad + t - v0] = 0.f;
              }
              if (lane == owner) mine.y -= static_cast<double>(e), rest = fmax(mine.y, 0.0) * lift * unit;
              ++rejected;
              __syncwarp();
              z = warp_sum(rest);
              if (!(z > 0.0)) {  // nothing is left: p again
                for (int j = 0; j < rejected; ++j) {
                  const int g = s_out[j];
                  const float ge = power(logit(widen<DT>(logits[g])), static_cast<float>(__shfl_sync(0xFFFFFFFFu, mine.x, g / p.slice)), c);
                  if (lane == 0 && g / p.slice == rank) s_e[pad + g - v0] = ge;
                }
                if (lane < kCluster) mine.y = b.slice[which][lane].y;
                rest = mine.y * lift * unit;
                rejected = 0, z = 1.0;
                __syncwarp();
              }
            }
          }
          if (command == kCut) {
            tried = child + 1;
            break;
          }
        }
        if (command == kStop) {  // the slice that holds the next token, and what is left to pass in it
          const float u = p.uniform[2 * row + 1];
          const double goal = static_cast<double>(u) * z;
          double upto = rest;
#pragma unroll
          for (int d = 1; d < kCluster; d <<= 1) {
            const double o = __shfl_up_sync(0xFFFFFFFFu, upto, d);
            if (lane >= d) upto += o;
          }
          const double before = __shfl_up_sync(0xFFFFFFFFu, upto, 1);
          const uint32_t over = __ballot_sync(0xFFFFFFFFu, lane < kCluster && upto > goal && rest > 0.0);
          const uint32_t some = __ballot_sync(0xFFFFFFFFu, lane < kCluster && rest > 0.0);
          const int owner = over ? __ffs(over) - 1 : (some ? 31 - __clz(some) : 0);
          if (lane == owner) b.target = goal - (lane ? before : 0.0);
          if (lane == 0) b.owner = owner, b.token = best, b.found = b.last = -1;
        }
        if (lane == rank) b.lift = lift;
        if (lane == 0) b.command = command, b.node = child, b.a = a, b.unit = unit;
      }
      __syncthreads();
      if (b.command != kCut) break;
      double part = 0.0;  // r over this slice
      const double la = b.a, lu = b.unit, ll = b.lift;
      each_draft(p, row, v0, n, [&](int i, float q) {
        const double e = static_cast<double>(s_e[pad + i]) * ll;
        if (e >= kNone) part += fmax(e * lu - la * static_cast<double>(q), 0.0);
      });
      part = block_sum(part);
      const uint32_t to = exchange(part, 0.0);
      if (warp == 0) {
        const double got = lane < kCluster ? b.slice[to][lane].x : 0.0;
        z = warp_sum(got);
        if (z > 0.0) {
          rest = got;
        } else {  // nothing is left: p again
          a = 0.0, z = 1.0;
          rest = mine.y * lift * unit;
        }
      }
    }
    if (b.command == kStop) break;
    node = b.node;
    __syncthreads();  // the walk's words are read
  }

  if (rank == 0) {
    for (int d = kept + tid; d < p.depth; d += kThreads) path[d] = -1;
    if (tid == 0) p.kept[s] = kept;
  }
  if (!warm || b.token < 0) {
    if (rank == 0 && tid == 0) p.token[s] = b.token;
    return;
  }
  // ---- the next token: the first of the slice whose cumulative sum passes the target
  if (rank != b.owner) return;
  const int64_t row = row0 + node;
  const int pad = (4 - (head_of<DT>(static_cast<const T*>(p.logits) + row * p.logits_stride + v0, n) & 3)) & 3;
  const double la = b.a, lu = b.unit, ll = b.lift, target = b.target;
  auto at = [&](int i) {
    const double e = static_cast<double>(s_e[pad + i]) * ll;
    if (e < kNone) return 0.0;
    if (!(has_q && la > 0.0)) return e * lu;
    return fmax(e * lu - la * static_cast<double>(draft_at(p.draft, p.draft_dtype, row * p.draft_stride + v0 + i)), 0.0);
  };
  const int len = ((n + kThreads - 1) / kThreads) | 1;  // a run per thread; odd: no two lanes on one bank
  const int lo = min(n, tid * len), hi = min(n, lo + len);
  double own = 0.0;
  int last = -1;
  for (int i = lo; i < hi; ++i) {
    const double r = at(i);
    if (r > 0.0) last = i;
    own += r;
  }
  double upto = own;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const double o = __shfl_up_sync(0xFFFFFFFFu, upto, d);
    if (lane >= d) upto += o;
  }
  if (lane == 31) b.sum[warp] = upto;
  const int top_last = __reduce_max_sync(0xFFFFFFFFu, last);
  if (lane == 0) atomicMax(&b.last, top_last);
  __syncthreads();
  double off = 0.0;
  for (int w = 0; w < warp; ++w) off += b.sum[w];
  double before = __shfl_up_sync(0xFFFFFFFFu, upto, 1);
  before = off + (lane ? before : 0.0);
  upto += off;
  if (before <= target && upto > target) {  // (one thread at most: before is the last one's upto)
    double acc = before;
    int found = last;  // rounding may leave none
    for (int i = lo; i < hi; ++i) {
      const double r = at(i);
      acc += r;
      if (r > 0.0 && acc > target) {
        found = i;
        break;
      }
    }
    b.found = found;
  }
  __syncthreads();
  if (tid == 0) {
    int t = b.found;
    if (t < 0) {  // before the first (a negative number) or past the last
      t = target < 0.0 ? -1 : b.last;
      if (t < 0)
        for (t = 0; t < n - 1 && !(s_e[pad + t] > 0.f);) ++t;
    }
    p.token[s] = v0 + t;
  }
}

template <int DT>
cudaError_t launch_dtype(const DraftParams& p, int nseq, cudaStream_t st) {
  static KernelSetup setup;
  const size_t smem = (static_cast<size_t>(p.slice) + 8) * sizeof(float);
  cudaError_t e = kernel_setup(setup, verify_kernel<DT>, kThreads, smem);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(nseq) * kCluster);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, verify_kernel<DT>, p);
}

}  // namespace

cudaError_t launch_draft_verify(const DraftParams& params, int nseq, cudaStream_t st) {
  DraftParams p = params;
  p.slice = ((p.vocab + kCluster - 1) / kCluster + 7) & ~7;
  switch (p.logits_dtype) {
    case EXL3_F16: return launch_dtype<EXL3_F16>(p, nseq, st);
    case EXL3_BF16: return launch_dtype<EXL3_BF16>(p, nseq, st);
    default: return launch_dtype<EXL3_F32>(p, nseq, st);
  }
}

}  // namespace exl3
