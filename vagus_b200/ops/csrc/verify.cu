// Verification of drafted tokens against the target's probabilities, from given
// random numbers.  Per row: drafted token i is accepted while
// u_i q_i(d_i) < p_i(d_i) (q = 1 without draft probabilities); at the first
// rejected place n the next token comes from w = max(p_n - q_n, 0) (without
// draft probabilities: p_n with d_n struck out; p_n itself where that leaves
// nothing), after the last accepted one from w = p_n: the first v with
// w_0 + .. + w_v > u sum(w).
//
// The sums are held in 64 bits: with 10^5 candidates the 32-bit rounding of a
// running sum moves a border past u once in a few hundred draws, and the token
// would depend on the order of summation.  That order follows from the batch, the
// vocabulary and the alignment (they set the pieces and the width of the loads), so a
// call repeats itself; a row alone and the same row in a batch may differ where u lies
// within those sums' rounding of a border.
//
// What bounds it is one row of p and of q a request, or latency for few
// requests: two dependent reads (the drafted tokens, their probabilities) before
// the row is known.  A cluster of CTAs takes a row, each warp one contiguous
// piece of it: one pass for the pieces' sums, which meet through distributed
// shared memory, then the CTA whose piece holds the border goes over that piece again
// (it is in L2), a part a warp, and the warp whose part holds it finds the token.  64 rows
// of 131072 candidates, fp32 with draft probabilities, take 18.5 us from HBM (their 67 MB
// alone 10.4), one row of 32000 takes 6.2.
#include "common.cuh"
#include "kernels.h"

namespace vagus {
namespace {

constexpr int kWarps = 8, kThreads = 32 * kWarps, kMaxCluster = 8;

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f(float v) { return v; }
template <> __device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }

__device__ __forceinline__ double ld_cluster_f64(const double* p, uint32_t rank) {
  double v;
  asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(mapa_shared(smem_u32(p), rank)) : "memory");
  return v;
}

__device__ __forceinline__ double warp_sum_f64(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// The weights of the row the next token is drawn from.
template <typename T>
struct Row {
  const T* p;
  const T* q;          // subtracted, or null
  long long struck;    // index that counts nothing, or -1
  __device__ __forceinline__ float weight(long long v, float pv, float qv) const {
    const float w = v == struck ? 0.f : pv - qv;
    return w > 0.f ? w : 0.f;        // negative and NaN weights count nothing
  }
  __device__ __forceinline__ float at(long long v) const { return weight(v, to_f(p[v]), q ? to_f(q[v]) : 0.f); }
};

template <typename T>
struct alignas(4 * sizeof(T)) Quad { T v[4]; };

// weights v .. v + 3 (those >= hi are zero)
template <typename T, bool VEC>
__device__ __forceinline__ void four(const Row<T>& r, long long v, long long hi, float (&w)[4]) {
  if (VEC) {
    if (v < hi) {
      const Quad<T> a = *reinterpret_cast<const Quad<T>*>(r.p + v);
      Quad<T> b;
      if (r.q) b = *reinterpret_cast<const Quad<T>*>(r.q + v);
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = r.weight(v + j, to_f(a.v[j]), r.q ? to_f(b.v[j]) : 0.f);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = 0.f;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = v + j < hi ? r.at(v + j) : 0.f;
  }
}

// Sum of the weights lo .. hi - 1 over a warp: whole stretches with kAhead vectors of each
// row under way (their loads in front of everything that branches), then the rest.
constexpr int kAhead = 4;
template <typename T, bool HAS_Q>
__device__ __forceinline__ double sum_whole(const Row<T>& r, long long& v, long long hi) {
  double s = 0;
  for (; v - 4 * (threadIdx.x % 32) + 128 * kAhead <= hi; v += 128 * kAhead) {
    Quad<T> p[kAhead], q[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      p[j] = *reinterpret_cast<const Quad<T>*>(r.p + v + 128 * j);
      if (HAS_Q) q[j] = *reinterpret_cast<const Quad<T>*>(r.q + v + 128 * j);
    }
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      float w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = r.weight(v + 128 * j + e, to_f(p[j].v[e]), HAS_Q ? to_f(q[j].v[e]) : 0.f);
      s += (static_cast<double>(w[0]) + w[1]) + (static_cast<double>(w[2]) + w[3]);
    }
  }
  return s;
}

template <typename T, bool VEC>
__device__ __forceinline__ double sum_of(const Row<T>& r, long long lo, long long hi, int lane) {
  double s = 0;
  long long v = lo + 4 * lane;
  if (VEC) s = r.q ? sum_whole<T, true>(r, v, hi) : sum_whole<T, false>(r, v, hi);
  for (; v < hi; v += 128) {
    float w[4];
    four<T, VEC>(r, v, hi, w);
    s += (static_cast<double>(w[0]) + w[1]) + (static_cast<double>(w[2]) + w[3]);
  }
  return warp_sum_f64(s);
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(kThreads, 4) verify_k(const VerifyArgs a) {
  __shared__ double warp_total[kWarps], part_total[kWarps];
  __shared__ double cta_total;
  __shared__ int s_acc;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int C = a.cluster;                             // CTAs of a row, which are a cluster
  const long long b = blockIdx.x / C;
  const int rank = static_cast<int>(blockIdx.x - b * C);
  const T* target = static_cast<const T*>(a.target) + b * a.st_b;
  const T* draft = a.draft ? static_cast<const T*>(a.draft) + b * a.sd_b : nullptr;
  const long long* tok = a.tokens + b * a.stok_b;

  int K = a.K;
  if (a.lengths) {
    const long long n = a.len_i64 ? static_cast<const long long*>(a.lengths)[b] : static_cast<const int*>(a.lengths)[b];
    K = static_cast<int>(n < 0 ? 0 : n < a.K ? n : a.K);
  }
  if (warp == 0) {
    int acc = K;
    for (int i0 = 0; i0 < K; i0 += 32) {
      const int i = i0 + lane;
      bool ok = true;
      if (i < K) {
        const long long d = tok[i];
        ok = d >= 0 && d < a.V;                        // a token outside the vocabulary is rejected
        if (ok) {
          const float p = to_f(target[i * a.st_k + d]), q = draft ? to_f(draft[i * a.sd_k + d]) : 1.f;
          ok = __fmul_rn(a.u_accept[b * a.su_b + i], q) < p;
        }
      }
      const unsigned bad = __ballot_sync(0xffffffffu, !ok);
      if (bad) { acc = i0 + __ffs(bad) - 1; break; }
    }
    if (lane == 0) s_acc = acc;
  }
  __syncthreads();
  const int acc = s_acc;

  Row<T> row;
  row.p = target + acc * a.st_k;
  row.q = acc < K && draft ? draft + acc * a.sd_k : nullptr;
  row.struck = acc < K && !draft ? tok[acc] : -1;
  // contiguous pieces, a multiple of 128 so that a warp reads whole vectors
  const long long piece = ((a.V + C * kWarps - 1) / (C * kWarps) + 127) / 128 * 128;
  const long long lo = min(a.V, (static_cast<long long>(rank) * kWarps + warp) * piece), hi = min(a.V, lo + piece);

  double before = 0, total = 0, totals[kMaxCluster];
  for (int pass = 0; pass < 2; ++pass) {
    const double s = sum_of<T, VEC>(row, lo, hi, lane);
    if (lane == 0) warp_total[warp] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
      double t = 0;
      for (int w = 0; w < kWarps; ++w) t += warp_total[w];
      cta_total = t;
    }
    cluster_sync();
    before = total = 0;
#pragma unroll
    for (int c = 0; c < kMaxCluster; ++c) {
      if (c >= C) break;
      totals[c] = ld_cluster_f64(&cta_total, c);
      if (c == rank) before = total;
      total += totals[c];
    }
    cluster_sync();            // nobody leaves, or writes its total again, while it is read
    if (total > 0 || acc == K) break;
    row.q = nullptr;           // nothing is left of the difference: draw from the target
    row.struck = -1;
  }

  // The piece that holds the border: the last one with any weight whose sum of
  // everything before it does not exceed u sum(w).  (Where rounding, or u = 1,
  // leaves no border above, that is the last token with any weight.)
  const double t = static_cast<double>(a.u_sample[b]) * total;
  int owner = -1;
  double at = 0;
#pragma unroll
  for (int c = 0; c < kMaxCluster; ++c) {
    if (c >= C) break;
    const double mine = totals[c];
    if (mine > 0 && !(at > t)) owner = c;
    at += mine;
  }
  if (rank != (owner < 0 ? 0 : owner)) return;
  // The same again for the pieces of this CTA's warps, then for the parts of that piece, one a warp.
  auto last_below = [&](const double* sums, double& base) {
    int found = -1;
    double run = base;
    for (int w = 0; w < kWarps; ++w) {
      const double mine = sums[w];
      if (mine > 0 && !(run > t)) { found = w; base = run; }
      run += mine;
    }
    return found;
  };
  double base = before;
  const int piece_at = last_below(warp_total, base);
  long long token = 0;                 // a row without any weight gives token 0
  if (piece_at >= 0) {
    const long long plo = min(a.V, (static_cast<long long>(rank) * kWarps + piece_at) * piece), phi = min(a.V, plo + piece);
    const long long part = (piece / 128 + kWarps - 1) / kWarps * 128;
    const long long qlo = min(phi, plo + warp * part), qhi = min(phi, qlo + part);
    const double s = sum_of<T, VEC>(row, qlo, qhi, lane);
    if (lane == 0) part_total[warp] = s;
    __syncthreads();
    int mine = last_below(part_total, base);
    if (mine < 0) mine = 0;            // rounding left the piece nothing below: its first part
    if (warp != mine) return;
    long long found = -1, last = -1;
    for (long long v0 = qlo; v0 < qhi && found < 0; v0 += 128) {
      const long long v = v0 + 4 * lane;
      float w[4];
      four<T, VEC>(row, v, qhi, w);
      double in[4];                    // running sums of this lane's four, the lane's first included
      in[0] = w[0];
#pragma unroll
      for (int j = 1; j < 4; ++j) in[j] = in[j - 1] + w[j];
      double scan = in[3];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double up = __shfl_up_sync(0xffffffffu, scan, o);
        if (lane >= o) scan += up;
      }
      const double off = base + (scan - in[3]);
      int first = 4, some = -1;
#pragma unroll
      for (int j = 3; j >= 0; --j) {
        if (off + in[j] > t && w[j] > 0.f) first = j;
        if (w[j] > 0.f && some < 0) some = j;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, first < 4), any = __ballot_sync(0xffffffffu, some >= 0);
      if (hit) {
        const int src = __ffs(hit) - 1;
        found = v0 + 4 * src + __shfl_sync(0xffffffffu, first, src);
      } else if (any) {
        const int src = 31 - __clz(any);
        last = v0 + 4 * src + __shfl_sync(0xffffffffu, some, src);
      }
      base += __shfl_sync(0xffffffffu, scan, 31);
    }
    token = found >= 0 ? found : last;
  } else if (warp != 0) {
    return;
  }
  for (int i = lane; i <= a.K; i += 32)
    a.out[b * (a.K + 1) + i] = i < acc ? tok[i] : i == acc ? token : -1;
  if (lane == 0) a.accepted[b] = acc;
}

template <typename T>
int launch(VerifyArgs a, cudaStream_t st) {
  // CTAs a row: enough to fill the GPU, each with 1024 candidates at least (1 row of 32000: 5.8 us, 9.2 with one CTA;
  // 64 of 131072, read from L2: 12.5 and 29.3)
  int C = 1;
  while (C < kMaxCluster && a.B * C < 148 * 2 && a.V > static_cast<long long>(C) * 1024) C *= 2;
  auto al = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % (4 * sizeof(T)) == 0; };
  const bool vec = al(a.target) && a.V % 4 == 0 && a.st_b % 4 == 0 && a.st_k % 4 == 0 &&
                   (!a.draft || (al(a.draft) && a.sd_b % 4 == 0 && a.sd_k % 4 == 0));
  cudaLaunchConfig_t cfg = {};
  a.cluster = C;
  cfg.gridDim = dim3(static_cast<unsigned>(a.B * C));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = C;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t rc = vec ? cudaLaunchKernelEx(&cfg, verify_k<T, true>, a) : cudaLaunchKernelEx(&cfg, verify_k<T, false>, a);
  return rc == cudaSuccess ? 0 : 3;
}

}  // namespace

int verify_draft(const VerifyArgs& a, int type, cudaStream_t st) {
  if (a.V < 1 || a.K < 0) return 1;
  if (a.B > 0x0fffffffLL) return 2;
  if (a.B == 0) return 0;
  if (type == 0) return launch<float>(a, st);
  if (type == 1) return launch<__half>(a, st);
  return launch<__nv_bfloat16>(a, st);
}

}  // namespace vagus
