// exl3_draft.cu -- which drafted tokens of each sequence's tree stay, by the target's probabilities and given random
// numbers, and the token that follows them (exl3_draft_verify, include/exl3_b200.h).
//
// At a node of the path, p = softmax(logits / T) and q the drafter's probabilities.  The children are tried in turn, the
// k-th (token x) against r_k = max(p - A_k q, 0) with A_0 = 0, A_k+1 = A_k + Z_k and Z_k = sum r_k: accepted where
// u q(x) Z_k < r_k(x).  (That r_k is what the repeated r <- max(r - Z q, 0) comes to: what is cut to zero stays there.)
// Without q a rejected token simply leaves p.  The path ends at the node none of whose children is accepted; its last r
// gives the next token by its cumulative sums.
//
// One cluster per sequence walks its path; each of sixteen warps per CTA has a slice of the vocabulary.  A node costs one
// pass over its row and one cluster barrier: a warp takes its slice's maximum m_w and the exponentials e^((x - m_w) / T) (kept
// in shared memory as f32) by itself, sends (m_w, their sum) to every CTA, and each CTA's seventeenth warp then takes the same
// decisions from the same numbers.  Sums carry their additions' roundings along and the slices' are joined in f64, so that r,
// which can be a small rest of p, keeps what the exponentials have (an f32 sum would leave 2^-24 of all of p in it).  Only rows
// on the path are read, and each node's first child, whose slice is on its way to registers while the node is decided.
//
// What bounds it is this walk, a row at a time: in a 17-token tree of 128000 a node takes about 0.9k clocks for its row, 2.4k
// for the exponentials, 0.7k to start the next row, 1.5k for the barrier, 1.9k for the decision, and 5k more where a child is
// rejected against q.  (A row's maxima and sums depend on the row alone: taken for all rows at once they would not wait.)  In
// a graph: one token of 32000 5.9 us, 8 chains of 65537 21 us, 32 16-token trees of 131072 28 us, 64 17-token trees of 128000
// with the drafter's probabilities 85 us.  Eight CTAs to a cluster: four take 36 us for the 32 trees, sixteen 50 (fewer clusters
// fit).  Sixteen warps with a slice each: eight took 122 us for the 64 trees where sixteen took 96.
#include <cuda_runtime.h>
#include <float.h>

#include <type_traits>

#include "exl3_attn.h"
#include "exl3_common.cuh"
#include "exl3_internal.h"

namespace exl3 {

namespace {

constexpr int kWarps = 16;                   // with a slice each
constexpr int kThreads = (kWarps + 1) * 32;  // and one that decides
constexpr int kCluster = 8;
constexpr int kSlices = kCluster * kWarps;
constexpr int kOwn = kSlices / 32;  // slices that a lane of a deciding warp looks after, neighbours
constexpr int kChunks = 8;          // 16-byte chunks of a lane's slice in registers
constexpr double kLog2e = 1.4426950408889634;
constexpr double kNone = 0x1p-100;  // a token this far below the likeliest has no probability

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}
// The first barrier in two halves: a CTA's shared memory may be written by others once it is known to have started.
__device__ __forceinline__ void cluster_started() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); }
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
// Element k of a chunk.
template <int DT>
__device__ __forceinline__ float element(const uint4& u, int k) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  if constexpr (DT == EXL3_F32) return __uint_as_float(w[k]);
  else return widen<DT>(static_cast<uint16_t>(w[k / 2] >> (16 * (k & 1))));
}
// A drafter's probability: NaN and negative numbers as 0.
template <int DT>
__device__ __forceinline__ float draft_p(const void* row, int64_t i) {
  return fmaxf(widen<DT>(static_cast<const typename Elem<DT>::type*>(row)[i]), 0.f);
}
__device__ __forceinline__ float draft_at(const void* row, int dtype, int64_t i) {
  return dtype == EXL3_F32 ? draft_p<EXL3_F32>(row, i) : dtype == EXL3_F16 ? draft_p<EXL3_F16>(row, i) : draft_p<EXL3_BF16>(row, i);
}

// Two f32 in one 64-bit register pair: one issue slot for both.
struct Two {
  uint64_t v;
  __device__ __forceinline__ Two() : v(0) {}
  __device__ __forceinline__ Two(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b)); }
  __device__ __forceinline__ void split(float& a, float& b) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
};
__device__ __forceinline__ Two operator+(Two a, Two b) {
  Two r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Two operator*(Two a, Two b) {
  Two r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Two fma(Two a, Two b, Two c) {
  Two r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ Two operator-(Two a, Two b) { return fma(b, Two(-1.f, -1.f), a); }
__device__ __forceinline__ float ex2(float x) {  // 2^x
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 2^(d c), d = min(x - m, 0) and c = c1 + c2 = log2(e) / T.  What the product and c's first part leave out, up to 2^-24 of an
// exponent of 100, is carried along: left are the exponential's own 2^-22 and the difference's rounding, 2^-24 |d| / T (none
// for 16-bit logits near one another).  Nothing below 2^-200, which is zero: so x of -inf and NaN, and m of -inf; x of +inf
// is m.
struct Scale {
  float c1, c2, least;
};
__device__ __forceinline__ Two power2(float x0, float x1, float m, Scale c) {
  float d0, d1;
  (Two(x0, x1) + Two(-m, -m)).split(d0, d1);
  const Two d(fminf(fmaxf(d0, c.least), 0.f), fminf(fmaxf(d1, c.least), 0.f));
  const Two c1(c.c1, c.c1), z = d * c1, none;
  const Two z2 = fma(d, Two(c.c2, c.c2), fma(d, c1, none - z));
  float z0, z1;
  z.split(z0, z1);
  const Two e(ex2(z0), ex2(z1));
  return fma(e * Two(0.6931472f, 0.6931472f), z2, e);
}
__device__ __forceinline__ float power(float x, float m, Scale c) {  // (the same steps)
  float a, b;
  power2(x, x, m, c).split(a, b);
  return a;
}

// A sum of f32 numbers with the rounding of every addition kept apart (Knuth's two-sum): good to 2^-48 of itself.  Of f64
// arithmetic, the conversions alone would take as long as the exponentials.
struct Sum {
  Two s, c;
  __device__ __forceinline__ void add(Two e) {
    const Two t = s + e, b = t - s;
    c = c + ((s - (t - b)) + (e - b));
    s = t;
  }
  __device__ __forceinline__ double total() const {
    float a, b, x, y;
    s.split(a, b), c.split(x, y);
    return (static_cast<double>(a) + static_cast<double>(b)) + (static_cast<double>(x) + static_cast<double>(y));
  }
};

// Whether x counts as the maximum `top`.
__device__ __forceinline__ bool is_top(float x, float top) { return x == x && fminf(x, FLT_MAX) == top; }

__device__ __forceinline__ uint32_t ordered(float x) {  // whole numbers in the order of the floats
  const uint32_t u = __float_as_uint(x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t u) { return __uint_as_float(u & 0x80000000u ? u & 0x7FFFFFFFu : ~u); }

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, d);
  return v;
}

struct Block {
  double2 slice[2][kSlices];  // every slice's (maximum, sum), sent by its warp; two, by turns
  float top[kSlices];         // their maxima and e^((m_w - m) / T)
  double lift[kSlices];
  // the walk, as the deciding warp leaves it
  int command, node, owner, token;
  float a;                    // A, in units of the exponentials (as all of r)
  double target;              // what is left to pass in the owner's slice
  // the sequence's rows
  int parent[kDraftMaxRows], tokens[kDraftMaxRows], first[kDraftMaxRows];  // first: a row's first child, or none
  int out[kDraftMaxRows];     // the node's rejected tokens, where there is no q
};
enum : int { kNext = 0, kStop = 1, kCut = 2 };  // on to a child; the path ends; r has to be summed

// r of an element after rejections: e its exponential in its slice, lift the slice's.
__device__ __forceinline__ float rest_of(float e, float lift, float a, float q) {
  const float v = e * lift;
  return v < static_cast<float>(kNone) ? 0.f : fmaxf(fmaf(-a, q, v), 0.f);
}

// Where elements of a row lie in s_e: whole 16-byte chunks of the row on multiples of four.
template <int DT>
__device__ __forceinline__ int chunks_begin(const typename Elem<DT>::type* src) {
  constexpr int kVec = Elem<DT>::kVec;
  return (kVec - static_cast<int>(reinterpret_cast<uintptr_t>(src) % 16 / sizeof(typename Elem<DT>::type))) % kVec;
}
template <int DT>
__device__ __forceinline__ int pad_of(const typename Elem<DT>::type* src) { return (4 - (chunks_begin<DT>(src) & 3)) & 3; }

// A lane's part of a slice of n elements: `head` and tail elements outside of whole 16-byte chunks, one a lane.
template <int DT>
struct Part {
  using T = typename Elem<DT>::type;
  static constexpr int kVec = Elem<DT>::kVec;
  const T* src;
  int n, head, chunks, lane;
  int odd;  // this lane's single element, or -1
  __device__ __forceinline__ Part(const T* s, int n_, int lane_) : src(s), n(n_), lane(lane_) {
    head = min(n, chunks_begin<DT>(s));
    chunks = (n - head) / kVec;
    const int tail = n - head - chunks * kVec;
    odd = lane < head ? lane : lane < head + tail ? chunks * kVec + lane : -1;
  }
  __device__ __forceinline__ void load(int from, uint4 (&u)[kChunks]) const {
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      u[i] = make_uint4(0u, 0u, 0u, 0u);
      if (from + i * 32 + lane < chunks) u[i] = reinterpret_cast<const uint4*>(src + head)[from + i * 32 + lane];
    }
  }
};

__device__ __forceinline__ uint4 four(uint4 v) { return v; }
__device__ __forceinline__ uint4 four(uint2 v) { return make_uint4(v.x, v.y, 0u, 0u); }

// f(e, q, e', q') for the elements of a warp's slice, four neighbours a lane (an element alone: beside zeros).
template <int DT, typename F>
__device__ __forceinline__ void each_draft_of(const void* draft, int64_t at, const float* own, int pad, int n, int lane, F&& f) {
  using T = typename Elem<DT>::type;
  const T* q = static_cast<const T*>(draft) + at - pad;
  const bool vec = reinterpret_cast<uintptr_t>(q) % (4 * sizeof(T)) == 0;
  constexpr int kBatch = 2;
  using V = typename std::conditional<DT == EXL3_F32, uint4, uint2>::type;  // four elements
  for (int t0 = lane * 4; t0 < pad + n; t0 += 128 * kBatch) {
    V v[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int t = t0 + i * 128;
      if (vec && t >= pad && t + 4 <= pad + n) v[i] = *reinterpret_cast<const V*>(q + t);
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int t = t0 + i * 128;
      if (t >= pad + n) break;
      const float4 e = *reinterpret_cast<const float4*>(own + t);
      if (vec && t >= pad && t + 4 <= pad + n) {
        const uint4 u = four(v[i]);
        f(e.x, fmaxf(element<DT>(u, 0), 0.f), e.y, fmaxf(element<DT>(u, 1), 0.f));
        f(e.z, fmaxf(element<DT>(u, 2), 0.f), e.w, fmaxf(element<DT>(u, 3), 0.f));
      } else {
        const float es[4] = {e.x, e.y, e.z, e.w};
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (t + k >= pad && t + k < pad + n) f(es[k], fmaxf(widen<DT>(q[t + k]), 0.f), 0.f, 0.f);
      }
    }
  }
}
template <typename F>
__device__ __forceinline__ void each_draft(const DraftParams& p, int64_t at, const float* own, int pad, int n, int lane, F&& f) {
  if (p.draft_dtype == EXL3_F32) each_draft_of<EXL3_F32>(p.draft, at, own, pad, n, lane, f);
  else if (p.draft_dtype == EXL3_F16) each_draft_of<EXL3_F16>(p.draft, at, own, pad, n, lane, f);
  else each_draft_of<EXL3_BF16>(p.draft, at, own, pad, n, lane, f);
}

template <int DT>
__global__ void __cluster_dims__(kCluster, 1, 1) __launch_bounds__(kThreads, 1) verify_kernel(const DraftParams p) {
  using T = typename Elem<DT>::type;
  constexpr int kVec = Elem<DT>::kVec;
  extern __shared__ __align__(16) float s_e[];  // [slice + 8]
  __shared__ Block b;
  cluster_started();
  pdl_wait();
  const int tid = static_cast<int>(threadIdx.x), lane = tid & 31, warp = tid >> 5;
  const int rank = static_cast<int>(blockIdx.x) % kCluster, s = static_cast<int>(blockIdx.x) / kCluster;
  const int r0 = p.row_start[s], r1 = p.row_start[s + 1];
  const float temp = p.temperature ? p.temperature[s] : 1.f;
  const int row0 = max(0, min(r0, p.rows)), all = max(0, min(r1, p.rows) - row0), ntok = min(all, p.max_rows);
  const bool warm = temp >= 0x1p-100f && temp <= 0x1p100f;
  if (tid == 0 && rank == 0 && (r0 < 0 || r1 < r0 || r1 > p.rows || all > ntok || (!warm && temp != 0.f)))
    atomicOr(p.err, kErrBadShape);
  int32_t* path = p.path + static_cast<int64_t>(s) * p.depth;
  if (ntok == 0) {  // (the whole cluster)
    if (rank == 0) {
      for (int d = tid; d < p.depth; d += kThreads) path[d] = -1;
      if (tid == 0) p.kept[s] = 0, p.token[s] = -1;
    }
    cluster_wait();
    return;
  }
  const bool decides = warp == kWarps;
  // this warp's slice, of p.slice elements but for the last
  const int mine = rank * kWarps + warp;
  const int v0 = min(mine * p.slice, p.vocab), n = decides ? 0 : min(p.vocab - v0, p.slice);
  auto row_of = [&](int i) { return static_cast<const T*>(p.logits) + (row0 + static_cast<int64_t>(i)) * p.logits_stride; };
  uint4 raw[kChunks];
  T odd = {};  // the lane's single element
  auto fetch = [&](int i) {
    const Part<DT> part(row_of(i) + v0, n, lane);
    if (part.chunks <= kChunks * 32) part.load(0, raw);  // (else they are loaded as they are used)
    if (part.odd >= 0) odd = part.src[part.odd];
  };
  if (!decides) fetch(0);
  for (int i = tid; i < ntok; i += kThreads) {
    b.parent[i] = p.parent ? p.parent[row0 + i] : i - 1;
    b.tokens[i] = p.tokens[row0 + i];
    b.first[i] = kDraftMaxRows;
  }
  Scale c{0.f, 0.f, 0.f};
  if (warm) {
    const double cd = kLog2e / static_cast<double>(temp);
    c.c1 = static_cast<float>(fmin(cd, static_cast<double>(FLT_MAX)));
    c.c2 = cd < 1e30 ? static_cast<float>(cd - static_cast<double>(c.c1)) : 0.f;
    c.least = fmaxf(-200.f / c.c1, -FLT_MAX);
  }
  __syncthreads();
  for (int i = tid; i < ntok; i += kThreads) {
    const int a = b.parent[i];
    if (a >= 0 && a < i) atomicMin(&b.first[a], i);
  }
  __syncthreads();
  const bool has_q = p.draft != nullptr && warm;
  int node = 0, kept = 0;
  uint32_t turn = 0;

  if (!decides) {
    // ---------------------------------------------------------------- a slice of every row on the path
    float* own = s_e + warp * p.slice;
    auto send = [&](double x, double y) {
      if (turn == 0) cluster_wait();  // every CTA of the cluster has started
      if (lane < kCluster) cluster_store(&b.slice[turn & 1u][mine], lane, x, y);
      ++turn;
      cluster_sync();
    };
    for (;;) {
      const Part<DT> part(row_of(node) + v0, n, lane);
      const int pad = pad_of<DT>(part.src);
      const bool whole = part.chunks <= kChunks * 32;
      const float single = part.odd >= 0 ? widen<DT>(odd) : -INFINITY;
      float top = fmaxf(single, -INFINITY);  // (NaN is passed over)
      for (int from = 0; from < part.chunks; from += kChunks * 32) {
        if (!whole) part.load(from, raw);
#pragma unroll
        for (int i = 0; i < kChunks; ++i)
          if (from + i * 32 + lane < part.chunks)
#pragma unroll
            for (int k = 0; k < kVec; ++k) top = fmaxf(top, element<DT>(raw[i], k));
      }
      top = fminf(unordered(__reduce_max_sync(0xFFFFFFFFu, ordered(top))), FLT_MAX);  // (+inf counts as the largest number)
      double sum = 0.0;
      if (warm) {
        Sum parts;
        if (part.odd >= 0) {
          const float e = power(single, top, c);
          own[pad + part.odd] = e;
          parts.s = Two(e, 0.f);
        }
        for (int from = 0; from < part.chunks; from += kChunks * 32) {
          if (!whole) part.load(from, raw);
#pragma unroll
          for (int i = 0; i < kChunks; ++i) {
            const int at = from + i * 32 + lane;
            if (at >= part.chunks) continue;
#pragma unroll
            for (int k = 0; k < kVec; k += 4) {
              const Two lo = power2(element<DT>(raw[i], k), element<DT>(raw[i], k + 1), top, c);
              const Two hi = power2(element<DT>(raw[i], k + 2), element<DT>(raw[i], k + 3), top, c);
              float4 e;
              lo.split(e.x, e.y), hi.split(e.z, e.w);
              *reinterpret_cast<float4*>(own + pad + part.head + at * kVec + k) = e;
              parts.add(lo), parts.add(hi);
            }
          }
        }
        sum = warp_sum(parts.total());
      } else {  // a greedy sequence's slice: where its maximum is first
        uint32_t at = part.odd >= 0 && is_top(single, top) ? part.odd : 0x7FFFFFFFu;
        for (int from = 0; from < part.chunks; from += kChunks * 32) {
          if (!whole) part.load(from, raw);
#pragma unroll
          for (int i = 0; i < kChunks; ++i)
            if (from + i * 32 + lane < part.chunks)
#pragma unroll
              for (int k = 0; k < kVec; ++k)
                if (is_top(element<DT>(raw[i], k), top)) at = min(at, static_cast<uint32_t>(part.head + (from + i * 32 + lane) * kVec + k));
        }
        sum = static_cast<double>(v0) + static_cast<double>(__reduce_min_sync(0xFFFFFFFFu, at));
      }
      // the first child's row, should it be the next
      const int guess = kept + 1 < p.depth ? b.first[node] : kDraftMaxRows;
      if (guess < kDraftMaxRows) fetch(guess);
      ++kept;
      send(static_cast<double>(top), sum);
      __syncthreads();  // the decision
      if (b.command == kCut) {  // (the first child is rejected: what was fetched for it is not needed)
        do {
          const float la = b.a, lu = static_cast<float>(b.lift[mine]);
          Sum r;
          each_draft(p, (row0 + static_cast<int64_t>(node)) * p.draft_stride + v0, own, pad, n, lane,
                     [&](float e0, float q0, float e1, float q1) { r.add(Two(rest_of(e0, lu, la, q0), rest_of(e1, lu, la, q1))); });
          send(warp_sum(r.total()), 0.0);
          __syncthreads();
        } while (b.command == kCut);
        if (b.command == kStop) break;
        node = b.node;
        fetch(node);
      } else {
        if (b.command == kStop) break;
        node = b.node;
        if (node != guess) fetch(node);
      }
    }
    if (!warm || b.token < 0 || mine != b.owner) return;
    // ---- the next token: the first of the owner's slice whose cumulative sum passes the target, a run of places per lane
    const int64_t q_at = (row0 + static_cast<int64_t>(node)) * p.draft_stride + v0;
    const int pad = pad_of<DT>(row_of(node) + v0);
    const double target = b.target, lift = b.lift[mine];
    const float la = b.a, lu = static_cast<float>(lift);
    const float least = static_cast<float>(fmin(kNone / lift, 2.0));  // (lift is at least kNone)
    const double scale = has_q && la > 0.f ? 1.0 : lift;              // of the numbers that at() gives
    auto at = [&](int i) {
      const float e = own[pad + i];
      if (has_q && la > 0.f) return rest_of(e, lu, la, draft_at(p.draft, p.draft_dtype, q_at + i));
      return e < least ? 0.f : e;
    };
    const double goal = target / scale;
    const int len = ((n + 31) / 32) | 1;  // odd: no two lanes on one bank
    const int lo = min(n, lane * len), hi = min(n, lo + len);
    Sum parts;
    int last = -1;
    for (int i = lo; i < hi; i += 2) {
      const float x = at(i), y = i + 1 < hi ? at(i + 1) : 0.f;
      if (x > 0.f) last = i;
      if (y > 0.f) last = i + 1;
      parts.add(Two(x, y));
    }
    auto scan = [&](double v) {  // inclusive
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const double o = __shfl_up_sync(0xFFFFFFFFu, v, d);
        if (lane >= d) v += o;
      }
      return v;
    };
    const double upto = scan(parts.total());
    const uint32_t over = __ballot_sync(0xFFFFFFFFu, upto > goal && last >= 0);
    int found = -1;
    if (over) {  // the run, a place per lane
      const int l = __ffs(over) - 1;
      double acc = __shfl_sync(0xFFFFFFFFu, upto, l > 0 ? l - 1 : 0);
      if (l == 0) acc = 0.0;
      const int end = min(n, (l + 1) * len);
      for (int i0 = l * len; i0 < end && found < 0; i0 += 32) {
        const float x = i0 + lane < end ? at(i0 + lane) : 0.f;
        const double sum = acc + scan(static_cast<double>(x));
        const uint32_t here = __ballot_sync(0xFFFFFFFFu, sum > goal && x > 0.f);
        if (here) found = i0 + __ffs(here) - 1;
        acc = __shfl_sync(0xFFFFFFFFu, sum, 31);
      }
      if (found < 0) found = __shfl_sync(0xFFFFFFFFu, last, l);  // rounding has left none
    }
    last = __reduce_max_sync(0xFFFFFFFFu, last);
    if (lane == 0) {
      if (found < 0) found = last;  // past the last
      if (found < 0)                // (what is left of the slice is none, token by token)
        for (found = 0; found < n - 1 && !(own[pad + found] > 0.f);) ++found;
      p.token[s] = v0 + found;
    }
    return;
  }

  // ---------------------------------------------------------------- the decisions: the same in every CTA
  for (;;) {
    const int64_t row = row0 + static_cast<int64_t>(node);
    const T* logits = row_of(node);
    const int pad = pad_of<DT>(logits), base = rank * kWarps * p.slice;
    // the children's numbers, of 32 rows at a time, one a lane
    int tok = -1;
    float x = 0.f, u = 0.f, q = 1.f;
    auto look = [&](int i) {
      tok = -1;
      if (i >= ntok || b.parent[i] != node) return;
      tok = b.tokens[i];
      if (tok < 0 || tok >= p.vocab) {
        tok = -1;  // (a token outside the vocabulary is not tried)
        return;
      }
      x = widen<DT>(logits[tok]);
      u = p.uniform[2 * (row0 + static_cast<int64_t>(i))];
      if (has_q) q = draft_at(p.draft, p.draft_dtype, row * p.draft_stride + tok);
    };
    const int guess = kept + 1 < p.depth ? b.first[node] : kDraftMaxRows;
    if (guess < kDraftMaxRows) look(guess + lane);
    const float u_next = p.uniform[2 * row + 1];
    if (rank == 0 && lane == 0) path[kept] = node;
    ++kept;
    if (turn == 0) cluster_wait();  // (the first of two)
    const double2* sent = b.slice[turn++ & 1u];
    cluster_sync();

    // a lane's slices: their sums of exponentials (of what is left of them) and e^((m_w - m) / T); r's sums
    double sums[kOwn], rest[kOwn];
    double a = 0.0, z = 0.0;
    int best = -1, tried = guess, rejected = 0;
    {
      float m = -INFINITY, m_own[kOwn];
#pragma unroll
      for (int j = 0; j < kOwn; ++j) {
        const double2 v = sent[lane * kOwn + j];
        m_own[j] = static_cast<float>(v.x), sums[j] = v.y;
        m = fmaxf(m, m_own[j]);
      }
      const float m_lane = m;
      m = unordered(__reduce_max_sync(0xFFFFFFFFu, ordered(m)));
      const uint32_t has = __ballot_sync(0xFFFFFFFFu, m_lane == m && m != -INFINITY);
      if (warm) {
        z = 0.0;
#pragma unroll
        for (int j = 0; j < kOwn; ++j) {
          double lift = static_cast<double>(power(m_own[j], m, c));
          if (lift < kNone) lift = 0.0;  // no token of the slice has a probability
          rest[j] = sums[j] * lift;
          z += rest[j];
          b.top[lane * kOwn + j] = m_own[j], b.lift[lane * kOwn + j] = lift;
        }
        z = warp_sum(z);
        best = has ? 0 : -1;
        __syncwarp();
      } else if (has) {  // the first slice with the maximum
        double where = 0.0;
#pragma unroll
        for (int j = kOwn - 1; j >= 0; --j)
          if (m_own[j] == m) where = sums[j];
        best = static_cast<int>(__shfl_sync(0xFFFFFFFFu, where, __ffs(has) - 1));
      }
      if (best < 0) tried = kDraftMaxRows;  // the row has no finite logit
    }
    int command, child = 0;
    for (;;) {
      command = kStop;
      for (; command == kStop && tried < ntok; tried += 32) {
        if (tried != guess) look(tried + lane);
        // every lane's token: its exponential and p, as the warp whose slice it is in computed them
        float e = 0.f;
        double le = 0.0;
        if (tok >= 0 && warm) {
          e = power(x, b.top[tok / p.slice], c);
          le = static_cast<double>(e) * b.lift[tok / p.slice];
          if (le < kNone) le = 0.0;
        }
        uint32_t left = __ballot_sync(0xFFFFFFFFu, tok >= 0);
        while (left && command == kStop) {
          const int l = __ffs(left) - 1;
          left &= left - 1;
          const int t = __shfl_sync(0xFFFFFFFFu, tok, l);
          child = tried + l;
          if (!warm) {
            if (t == best) command = kNext;
            continue;
          }
          const double qt = static_cast<double>(__shfl_sync(0xFFFFFFFFu, q, l));
          double rt = __shfl_sync(0xFFFFFFFFu, le, l);
          if (has_q) {
            if (a > 0.0) rt = fmax(rt - a * qt, 0.0);
          } else {
            bool gone = false;
            for (int j = lane; j < rejected; j += 32) gone |= b.out[j] == t;
            if (__any_sync(0xFFFFFFFFu, gone)) continue;  // its sibling took it out of p
          }
          if (static_cast<double>(__shfl_sync(0xFFFFFFFFu, u, l)) * qt * z < rt) {
            command = kNext;
          } else if (has_q) {
            a += z;
            command = kCut;
          } else {
            const int slice = t / p.slice;
            const double et = static_cast<double>(__shfl_sync(0xFFFFFFFFu, e, l));
            if (lane == 0) {
              b.out[rejected] = t;
              if (slice / kWarps == rank) s_e[pad + t - base] = 0.f;
            }
            ++rejected;
            z = 0.0;
#pragma unroll
            for (int j = 0; j < kOwn; ++j) {
              if (slice == lane * kOwn + j) sums[j] = fmax(sums[j] - et, 0.0), rest[j] = sums[j] * b.lift[slice];
              z += rest[j];
            }
            __syncwarp();
            z = warp_sum(z);
            if (!(z > 0.0)) {  // nothing is left: p again
              for (int j = lane; j < rejected; j += 32) {
                const int g = b.out[j];
                if (g / p.slice / kWarps == rank) s_e[pad + g - base] = power(widen<DT>(logits[g]), b.top[g / p.slice], c);
              }
              z = 0.0;
#pragma unroll
              for (int j = 0; j < kOwn; ++j)
                sums[j] = sent[lane * kOwn + j].y, rest[j] = sums[j] * b.lift[lane * kOwn + j], z += rest[j];
              z = warp_sum(z);
              rejected = 0;
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
        const double goal = static_cast<double>(u_next) * z;
        double upto = 0.0;
#pragma unroll
        for (int j = 0; j < kOwn; ++j) upto += rest[j];
        const bool some = upto > 0.0;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
          const double o = __shfl_up_sync(0xFFFFFFFFu, upto, d);
          if (lane >= d) upto += o;
        }
        const double before = __shfl_up_sync(0xFFFFFFFFu, upto, 1);
        const uint32_t over = __ballot_sync(0xFFFFFFFFu, upto > goal && some);
        const uint32_t any = __ballot_sync(0xFFFFFFFFu, some);
        if (lane == (over ? __ffs(over) - 1 : (any ? 31 - __clz(any) : 0))) {
          double acc = lane ? before : 0.0, target = 0.0;
          int slice = -1;  // the last that begins at or before the goal
#pragma unroll
          for (int j = 0; j < kOwn; ++j) {
            if (rest[j] > 0.0 && (slice < 0 || !(acc > goal))) slice = lane * kOwn + j, target = goal - acc;
            acc += rest[j];
          }
          b.owner = slice, b.target = target, b.token = best;
        }
      }
      if (lane == 0) {
        b.command = command, b.node = child;
        b.a = static_cast<float>(a);
      }
      __syncthreads();
      if (command != kCut) break;
      const double2* got = b.slice[turn++ & 1u];
      cluster_sync();  // the slices' sums of r
      z = 0.0;
#pragma unroll
      for (int j = 0; j < kOwn; ++j) rest[j] = got[lane * kOwn + j].x, z += rest[j];
      z = warp_sum(z);
      if (!(z > 0.0)) {  // nothing is left: p again
        a = z = 0.0;
#pragma unroll
        for (int j = 0; j < kOwn; ++j) rest[j] = sums[j] * b.lift[lane * kOwn + j], z += rest[j];
        z = warp_sum(z);
      }
    }
    if (command == kStop) break;
    node = child;
  }
  if (rank == 0) {
    for (int d = kept + lane; d < p.depth; d += 32) path[d] = -1;
    if (lane == 0) {
      p.kept[s] = kept;
      if (!warm || b.token < 0) p.token[s] = b.token;
    }
  }
}

template <int DT>
cudaError_t launch_dtype(const DraftParams& p, int nseq, cudaStream_t st) {
  static KernelSetup setup;
  const size_t smem = (static_cast<size_t>(p.slice) * kWarps + 8) * sizeof(float);
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
  p.slice = ((p.vocab + kSlices - 1) / kSlices + 7) & ~7;
  switch (p.logits_dtype) {
    case EXL3_F16: return launch_dtype<EXL3_F16>(p, nseq, st);
    case EXL3_BF16: return launch_dtype<EXL3_BF16>(p, nseq, st);
    default: return launch_dtype<EXL3_F32>(p, nseq, st);
  }
}

}  // namespace exl3
