// Rotary positions of queries and keys, one launch for both, forward and (with
// the angles negated) backward:
//
//   y_a = m (x_a cos t - x_b sin t),  y_b = m (x_a sin t + x_b cos t),
//   t = position * inv_freq[i],  i = 0 .. R / 2 - 1,
//
// over the channel pairs (a, b) = (2 i, 2 i + 1) (interleaved) or
// (i, i + R / 2) (half); channels R .. D - 1 pass through.
//
// The angle of a far position needs more than 32 bits (a position of 2^20 times
// a frequency of 1 leaves a float 0.06 rad of step), so it is formed in 64 bits
// and reduced to a fraction of a turn before the 32-bit sine and cosine; the
// products are 32-bit, rounded once to the output type.  A CTA takes a few
// tokens: its threads first form the tokens' R / 2 angles, one each, in shared
// memory, then stream every head of q and k past them with 16-byte accesses, so
// an angle is computed once per token and not once per head.  What bounds it is
// the HBM traffic of q and k, read once and written once.
#include "common.cuh"
#include "kernels.h"

namespace vagus {
namespace {

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f(float v) { return v; }
template <> __device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f(float v) { return v; }
template <> __device__ __forceinline__ __half from_f(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }

template <typename T>
struct alignas(16) Vec {
  static constexpr int N = 16 / sizeof(T);
  T v[N];
};

// two values, neighbours in a vector
__device__ __forceinline__ void put2(float* d, float a, float b) { d[0] = a; d[1] = b; }
__device__ __forceinline__ void put2(__half* d, float a, float b) { *reinterpret_cast<__half2*>(d) = __floats2half2_rn(a, b); }
__device__ __forceinline__ void put2(__nv_bfloat16* d, float a, float b) {
  *reinterpret_cast<__nv_bfloat162*>(d) = __floats2bfloat162_rn(a, b);
}

// two channel pairs by their angles, w = (cos, cos, sin, sin)
__device__ __forceinline__ void turn2(F2& xa, F2& xb, float4 w) {
  const F2 c = pair2(w.x, w.y), s = pair2(w.z, w.w), a = xa;
  xa = fma2(a, c, mul2(xb, pair2(-w.z, -w.w)));
  xb = fma2(a, s, mul2(xb, c));
}

constexpr int kThreads = 256;
constexpr int kMaxAngles = 4096;     // pairs of angles of a CTA's tokens in shared memory

__device__ __forceinline__ long long position_of(const RotaryArgs& a, long long b, long long l) {
  if (a.pos == nullptr) return a.offset + l;
  const long long i = b * a.pos_sb + l * a.pos_sl;
  return a.pos_i64 ? static_cast<const long long*>(a.pos)[i] : static_cast<const int*>(a.pos)[i];
}

__device__ __forceinline__ float2 angle_of(double pos, double inv, float m, float sign) {
  const double turns = pos * inv * 0.15915494309189533577;      // 1 / (2 pi)
  const float f = static_cast<float>(turns - rint(turns));
  float s, c;
  sincospif(2.f * f, &s, &c);
  return make_float2(c * m, s * m * sign);
}

// one row (token, head) of either tensor
template <typename T>
__device__ __forceinline__ void row_of(const RotaryArgs& a, long long b, long long l, int h, const T*& src, T*& dst) {
  if (h < a.H) {
    src = static_cast<const T*>(a.q) + b * a.sq_b + l * a.sq_l + h * a.sq_h;
    dst = static_cast<T*>(a.yq) + ((b * a.L + l) * a.H + h) * a.D;
  } else {
    h -= a.H;
    src = static_cast<const T*>(a.k) + b * a.sk_b + l * a.sk_l + h * a.sk_h;
    dst = static_cast<T*>(a.yk) + ((b * a.L + l) * a.Hk + h) * a.D;
  }
}

constexpr int ctas_per_sm(bool inter, int size) { return inter ? 8 : size == 4 ? 6 : 5; }

// blockDim = (items of a head, rows); the rows are `across` heads of one token or, where the
// heads are few, of several; an item is one 16-byte vector, or for the half
// layout's rotated channels the two vectors that pair up.  The angles of an item's P pairs
// are read as float4s of two; those lie [which of the P / 2][item], so that neighbouring
// threads read neighbouring 16 bytes (item-major, 8 threads met in 2 of 8 bank groups).
// A head's address is worked out once and its tokens follow.  Many resident threads matter
// more than loads held ahead in registers (rows' loads taken two to four at a time: 146 to
// 187 us for both directions of 4 x 4096 tokens of 32 heads of 128 in bf16), and in 16 bits
// so does the arithmetic a byte: two pairs an operation take 93 us where one takes 105 (5.6
// TB/s; fp32 6.3 TB/s).
template <typename T, bool INTER>
__global__ void __launch_bounds__(kThreads, ctas_per_sm(INTER, sizeof(T))) rotary_vec_k(const RotaryArgs a, int tokens, int across) {
  constexpr int N = Vec<T>::N, P = INTER ? N / 2 : N;
  extern __shared__ __align__(16) float2 cs[];                    // [tokens][R / 2]
  __shared__ long long q_at[kThreads], k_at[kThreads];            // where a token's heads begin
  const int half = a.R / 2, tid = threadIdx.y * blockDim.x + threadIdx.x, nthr = blockDim.x * blockDim.y;
  const unsigned t0 = blockIdx.x * tokens, L = static_cast<unsigned>(a.L);
  const int nt = min(tokens, static_cast<int>(static_cast<unsigned>(a.B) * L - t0));
  for (int i = tid; i < nt * half; i += nthr) {
    const int k = i / half, p = i - k * half;
    const unsigned t = t0 + k, b = t / L, l = t - b * L;
    const int it = p / P, e = p - it * P;
    const float2 w = angle_of(static_cast<double>(position_of(a, b, l)), a.inv[p], a.scale, a.sign);
    float* to = reinterpret_cast<float*>(cs + k * half + (e / 2 * (half / P) + it) * 2) + e % 2;
    to[0] = w.x;
    to[2] = w.y;
    if (p == 0) {
      q_at[k] = b * a.sq_b + l * a.sq_l;
      k_at[k] = b * a.sk_b + l * a.sk_l;
    }
  }
  __syncthreads();
  const int heads = a.H + a.Hk, item = threadIdx.x;
  const int rot = INTER ? a.R / N : half / N;                     // items that rotate
  const bool pair = !INTER && item < rot;
  const int c0 = INTER || pair ? item * N : a.R + (item - rot) * N;
  const int ty = threadIdx.y / across, tstep = blockDim.y / across;
  for (int h = threadIdx.y - ty * across; h < heads; h += across) {
    const bool is_q = h < a.H;
    const T* in = is_q ? static_cast<const T*>(a.q) + h * a.sq_h : static_cast<const T*>(a.k) + (h - a.H) * a.sk_h;
    const long long* at = is_q ? q_at : k_at;
    const long long pitch = static_cast<long long>(is_q ? a.H : a.Hk) * a.D;
    T* out = (is_q ? static_cast<T*>(a.yq) + h * a.D : static_cast<T*>(a.yk) + (h - a.H) * a.D) + t0 * pitch;
#pragma unroll 1
    for (int tk = ty; tk < nt; tk += tstep) {
      const float4* c = reinterpret_cast<const float4*>(cs + tk * half) + item;
      const T* src = in + at[tk] + c0;
      T* dst = out + tk * pitch + c0;
      Vec<T> x = *reinterpret_cast<const Vec<T>*>(src);
      if (INTER) {
        if (item < rot) {
#pragma unroll
          for (int e = 0; e < N; e += 4) {
            F2 xa = pair2(to_f(x.v[e]), to_f(x.v[e + 2])), xb = pair2(to_f(x.v[e + 1]), to_f(x.v[e + 3]));
            turn2(xa, xb, c[e / 4 * rot]);
            float a0, a1, b0, b1;
            halves(xa, a0, a1);
            halves(xb, b0, b1);
            put2(x.v + e, a0, b0);
            put2(x.v + e + 2, a1, b1);
          }
        }
      } else if (pair) {
        Vec<T> y = *reinterpret_cast<const Vec<T>*>(src + half);
#pragma unroll
        for (int e = 0; e < N; e += 2) {
          F2 xa = pair2(to_f(x.v[e]), to_f(x.v[e + 1])), xb = pair2(to_f(y.v[e]), to_f(y.v[e + 1]));
          turn2(xa, xb, c[e / 2 * rot]);
          float a0, a1, b0, b1;
          halves(xa, a0, a1);
          halves(xb, b0, b1);
          put2(x.v + e, a0, a1);
          put2(y.v + e, b0, b1);
        }
        *reinterpret_cast<Vec<T>*>(dst + half) = y;
      }
      *reinterpret_cast<Vec<T>*>(dst) = x;
    }
  }
}

// any D, even R, any alignment: one channel pair (or one passed channel) a thread (4 x 4096
// tokens of 32 heads of 128 in bf16, two bytes off: 206 us; a copy and the kernel above 188,
// with that much memory more)
template <typename T>
__global__ void __launch_bounds__(kThreads) rotary_any_k(const RotaryArgs a, int tokens) {
  extern __shared__ __align__(16) float2 cs[];
  const int half = a.R / 2;
  const long long t0 = static_cast<long long>(blockIdx.x) * tokens, total = a.B * a.L;
  const int nt = static_cast<int>(min(static_cast<long long>(tokens), total - t0));
  for (int i = threadIdx.x; i < nt * half; i += blockDim.x) {
    const int tk = i / half, p = i - tk * half;
    const long long t = t0 + tk, b = t / a.L, l = t - b * a.L;
    cs[i] = angle_of(static_cast<double>(position_of(a, b, l)), a.inv[p], a.scale, a.sign);
  }
  __syncthreads();
  const int items = half + a.D - a.R, heads = a.H + a.Hk;
  for (int i = threadIdx.x; i < nt * heads * items; i += blockDim.x) {
    const int r = i / items, it = i - r * items, tk = r / heads;
    const long long t = t0 + tk, b = t / a.L, l = t - b * a.L;
    const T* src;
    T* dst;
    row_of<T>(a, b, l, r - tk * heads, src, dst);
    if (it < half) {
      const int ca = a.interleaved ? 2 * it : it, cb = a.interleaved ? 2 * it + 1 : it + half;
      const float2 w = cs[tk * half + it];
      const float xa = to_f(src[ca]), xb = to_f(src[cb]);
      dst[ca] = from_f<T>(xa * w.x - xb * w.y);
      dst[cb] = from_f<T>(xa * w.y + xb * w.x);
    } else {
      dst[it + half] = src[it + half];
    }
  }
}

template <typename T>
int launch(const RotaryArgs& a, cudaStream_t st) {
  constexpr int N = Vec<T>::N;
  const int half = a.R / 2;
  // tokens a CTA: up to as many as its threads have angles for at once, the share whose waves over the GPU end first
  // (a CTA's start counts for two tokens).  4610 tokens of 40 heads of 128, 64 channels rotated, bf16: half 7 a CTA 19.4
  // us, 2 a CTA 22.7; interleaved 4 a CTA 16.1, 2 a CTA 17.1
  const long long slots = 148LL * ctas_per_sm(a.interleaved, sizeof(T));
  auto length = [&](int t) { return ((a.B * a.L + t - 1) / t + slots - 1) / slots * (t + 2); };
  int tokens = half >= kThreads ? 1 : half <= 8 ? 32 : kThreads / half;
  for (int t = tokens - 1; t > 0; --t)
    if (length(t) < length(tokens)) tokens = t;
  while (tokens > 1 && static_cast<long long>(tokens) * (a.H + a.Hk) * a.D > 1 << 30) --tokens;
  const long long grid = (a.B * a.L + tokens - 1) / tokens;
  if (a.B * a.L > 0x7fff0000LL) return 2;                // tokens are counted in 32 bits, and so is what one of them holds
  if (static_cast<long long>(a.H + a.Hk) * a.D > 1 << 30) return 2;
  const size_t smem = static_cast<size_t>(tokens) * half * sizeof(float2);
  auto al = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
  auto mul = [](long long s) { return s % N == 0; };
  const bool vec = al(a.q) && al(a.yq) && mul(a.sq_b) && mul(a.sq_l) && mul(a.sq_h) &&
                   (a.Hk == 0 || (al(a.k) && al(a.yk) && mul(a.sk_b) && mul(a.sk_l) && mul(a.sk_h))) &&
                   a.D % N == 0 && (a.interleaved ? a.R % N == 0 : half % N == 0);
  const int items = vec ? (a.interleaved ? a.D / N : half / N + (a.D - a.R) / N) : 0;
  if (vec && items <= kThreads) {
    // rows: all heads of as many tokens as fit, or an even share of the heads of one
    const int room = kThreads / items, heads = a.H + a.Hk, turns = (heads + room - 1) / room;
    const int across = (heads + turns - 1) / turns, each = turns > 1 ? 1 : room / heads;
    const dim3 block(items, across * (each < tokens ? each : tokens));
    if (a.interleaved) rotary_vec_k<T, true><<<static_cast<unsigned>(grid), block, smem, st>>>(a, tokens, across);
    else rotary_vec_k<T, false><<<static_cast<unsigned>(grid), block, smem, st>>>(a, tokens, across);
  } else {
    rotary_any_k<T><<<static_cast<unsigned>(grid), kThreads, smem, st>>>(a, tokens);
  }
  return cudaGetLastError() == cudaSuccess ? 0 : 3;
}

}  // namespace

int rotary(const RotaryArgs& a, int type, cudaStream_t st) {
  if (a.R < 2 || a.R % 2 || a.R > a.D || a.R / 2 > kMaxAngles) return 1;
  if (a.B * a.L == 0 || a.H + a.Hk == 0) return 0;
  if (type == 0) return launch<float>(a, st);
  if (type == 1) return launch<__half>(a, st);
  return launch<__nv_bfloat16>(a, st);
}

}  // namespace vagus
