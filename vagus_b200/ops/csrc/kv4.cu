// A key / value cache held in 4 bits: writing it, reading it back, and softmax
// attention over it.
//
// Format.  For each (sequence, KV head, token) one 4-bit code c a channel,
// channel 2 j in the low half of byte j, and for each group of 32 channels a
// step s and an offset b in bf16.  A code stands for bf16((128 + c) s + b).
// 0.5 + 4 / 32 = 0.625 bytes a value, against 2 of a bf16 cache.  Why 128 + c
// and not c: bf16 has 7 mantissa bits, so the bit pattern 0x4300 | c IS the
// number 128 + c, and a pair of codes becomes a pair of values with one bitwise
// operation and one bf16 fused multiply-add, exactly as the format defines them.
// b is rounded to bf16 near -128 s, by at most 0.53 s; the codes are computed
// from the rounded b, so this shifts the group's grid of 16 levels and adds no
// error to a value inside it.
#include "common.cuh"
#include "kernels.h"
#include "mma.cuh"

namespace vagus {
namespace {

constexpr int kGroup = 32;

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f(float v) { return v; }
template <> __device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }

// NaN in any operand gives NaN
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ long long index_at(const void* p, int i64, long long i) {
  return i64 ? static_cast<const long long*>(p)[i] : static_cast<const int*>(p)[i];
}

// ---------------------------------------------------------------- append --

// (x - b) / s rounded to the nearest whole number (ties to even).  The product
// with the reciprocal is within 2^-22 of the quotient's value (at most 143 and a
// bit), so it rounds alike unless it lies near a half: then, and where the
// reciprocal is not finite, the quotient is taken.
__device__ __forceinline__ int code_of(float x, float s, float inv, float b) {
  const float d = __fsub_rn(x, b), r = d * inv;
  float k = rintf(r);
  if (!(fabsf(r - k) < 0.499f)) k = rintf(__fdiv_rn(d, s));
  const int c = __float2int_rn(fminf(fmaxf(k, 128.f), 143.f)) - 128;
  return s > 0.f ? c : 0;
}

// 8 channels a thread, 4 threads a group of 32; rows (b, l, h) in the order the
// projections leave them, so the reads are contiguous.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) kv4_append_k(const Kv4AppendArgs a) {
  const int which = blockIdx.y;                       // 0: keys, 1: values
  const int D = which ? a.Dv : a.D, per = D / 8;
  const T* x = static_cast<const T*>(which ? a.v : a.k);
  const long long sb = which ? a.sv_b : a.sk_b, sh = which ? a.sv_h : a.sk_h, sl = which ? a.sv_l : a.sk_l;
  const long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x;
  const long long row = i / per, total = a.B * a.L * a.Hk;
  const bool live = row < total;                      // whole groups of 4 threads are live or not
  const int c0 = static_cast<int>(i - row * per) * 8;
  const long long bl = row / a.Hk, b = bl / a.L;
  const long long l = bl - b * a.L, h = row - bl * a.Hk;
  float v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = 0.f;
  if (live) {
    const T* p = x + b * sb + h * sh + l * sl + c0;
    if (VEC) {
      constexpr int N = 16 / sizeof(T);
#pragma unroll
      for (int j = 0; j < 8; j += N) {
        const uint4 u = *reinterpret_cast<const uint4*>(p + j);
        const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
        for (int k = 0; k < N; ++k) v[j + k] = to_f(e[k]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = to_f(p[j]);
    }
  }
  float lo = v[0], hi = v[0];
#pragma unroll
  for (int j = 1; j < 8; ++j) { lo = min_nan(lo, v[j]); hi = max_nan(hi, v[j]); }
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
  if (!live) return;
  const long long t = l + (a.start ? index_at(a.start, a.start_i64, b) : a.offset);
  if (t < 0 || t >= a.cap) {                          // a start given on the device that leaves the cache
    record_error(a.err, kErrBadArgument);
    return;
  }
  const __nv_bfloat16 s16 = __float2bfloat16_rn(__fdiv_rn(__fsub_rn(hi, lo), 15.f));
  const float s = __bfloat162float(s16);
  const __nv_bfloat16 b16 = __float2bfloat16_rn(__fsub_rn(lo, __fmul_rn(128.f, s)));
  const float off = __bfloat162float(b16), inv = __frcp_rn(s);
  uint32_t w = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) w |= static_cast<uint32_t>(code_of(v[j], s, inv, off)) << (4 * j);
  const long long out = (b * a.Hk + h) * a.cap + t;
  uint32_t* codes = reinterpret_cast<uint32_t*>(which ? a.v_codes : a.k_codes);
  codes[out * per + c0 / 8] = w;
  if ((c0 & (kGroup - 1)) == 0) {
    const __nv_bfloat162 pr = __halves2bfloat162(s16, b16);
    uint32_t* params = reinterpret_cast<uint32_t*>(which ? a.v_params : a.k_params);
    params[out * (D / kGroup) + c0 / kGroup] = *reinterpret_cast<const uint32_t*>(&pr);
  }
}

// ------------------------------------------------------------------ read --

__device__ __forceinline__ uint32_t fma_bf16x2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
// nibbles i and i + 4 of w (i = 0 .. 3) as the pair of values they stand for
template <int I>
__device__ __forceinline__ uint32_t pair_of(uint32_t w, uint32_t ss, uint32_t bb) {
  return fma_bf16x2(((w >> (4 * I)) & 0x000F000Fu) | 0x43004300u, ss, bb);
}
__device__ __forceinline__ uint32_t low2(uint32_t a, uint32_t b) { return __byte_perm(a, b, 0x5410); }
__device__ __forceinline__ uint32_t high2(uint32_t a, uint32_t b) { return __byte_perm(a, b, 0x7632); }

// 8 channels a thread: 4 bytes of codes in, 16 bytes of values out
__global__ void __launch_bounds__(256) kv4_read_k(const Kv4ReadArgs a) {
  const int which = blockIdx.y;
  const int D = which ? a.Dv : a.D, per = D / 8;
  const uint32_t* codes = reinterpret_cast<const uint32_t*>(which ? a.v_codes : a.k_codes);
  const uint32_t* params = reinterpret_cast<const uint32_t*>(which ? a.v_params : a.k_params);
  uint4* out = reinterpret_cast<uint4*>(which ? a.v : a.k);
  const long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x;
  const long long row = i / per;
  if (row >= a.B * a.Hk * a.L) return;
  const int cw = static_cast<int>(i - row * per);
  const long long bh = row / a.L, l = row - bh * a.L, b = bh / a.Hk;
  const long long t = l + (a.start ? index_at(a.start, a.start_i64, b) : a.offset);
  if (t < 0 || t >= a.cap) {
    record_error(a.err, kErrBadArgument);
    out[i] = make_uint4(0, 0, 0, 0);
    return;
  }
  const long long at = bh * a.cap + t;
  const uint32_t w = codes[at * per + cw], p = params[at * (D / kGroup) + cw / 4];
  const uint32_t ss = low2(p, p), bb = high2(p, p);
  const uint32_t p0 = pair_of<0>(w, ss, bb), p1 = pair_of<1>(w, ss, bb), p2 = pair_of<2>(w, ss, bb),
                 p3 = pair_of<3>(w, ss, bb);
  out[i] = make_uint4(low2(p0, p1), low2(p2, p3), high2(p0, p1), high2(p2, p3));
}

// ------------------------------------------------------------- attention --
//
// One CTA of four warps per (split of the tokens, KV head and tile of query
// rows, sequence).  The rows of a KV head are its Lq queries times the H / Hk
// heads that share it; a tile has 8 NT of them, so one pass over the cache
// serves them all.  Everything stays in registers:
//
//   S^T (16 tokens x 8 rows)    += K (16 x 16 channels) q^T      mma m16n8k16
//   O^T (16 channels x 8 rows)  += V^T (16 x 16 tokens) P^T
//
// The order of the channels inside a product is free, so a lane takes the
// codes as they lie: for K the D / 4 adjacent channels of its token (lane t of
// a quad), whose nibble pairs are A fragments as they are; for V the words g of
// two neighbouring tokens, whose halves one byte permute brings together.  S^T
// leaves the product with a token a row; transposing the 8 x 8 tile of the
// rounded probabilities (movmatrix) makes it the B operand of the second.
//
// Each warp has its own running maximum and sum over every fourth block of 32
// tokens; the four meet in shared memory, the splits in a second kernel.
// Probabilities are rounded to bf16 for the second product (2^-9 relative, the
// size of the output's own rounding); scores, sums and accumulators are fp32.

constexpr int kAttnWarps = 4;
constexpr int kBlock = 32;            // tokens a warp takes at once

__device__ __forceinline__ uint32_t transpose8(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}

template <int W>
__device__ __forceinline__ void load_words(uint32_t (&r)[W], const uint8_t* p) {
  if constexpr (W == 4) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    r[0] = u.x; r[1] = u.y; r[2] = u.z; r[3] = u.w;
  } else if constexpr (W == 2) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    r[0] = u.x; r[1] = u.y;
  } else {
    r[0] = *reinterpret_cast<const uint32_t*>(p);
  }
}

// the codes and parameters of 16 tokens that one lane works on
template <int D, int DV>
struct Frag {
  static constexpr int KW = D / 32, VW = DV / 64;
  uint32_t k[2][KW], kp[2], v[4][VW], vp[4];

  // t0: first token (a multiple of 16); the cache holds whole blocks of 16
  __device__ __forceinline__ void load(const Kv4AttnArgs& a, long long bh, int t0, int g, int t) {
    const long long at = bh * a.cap + t0;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const long long row = at + g + 8 * r;
      load_words<KW>(k[r], a.k_codes + row * (D / 2) + t * (4 * KW));
      kp[r] = reinterpret_cast<const uint32_t*>(a.k_params)[row * (D / kGroup) + t * KW / 4];
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const long long row = at + 2 * t + (r & 1) + 8 * (r >> 1);
      load_words<VW>(v[r], a.v_codes + row * (DV / 2) + g * (4 * VW));
      vp[r] = reinterpret_cast<const uint32_t*>(a.v_params)[row * (DV / kGroup) + g * VW / 4];
    }
  }
  // tokens >= n stand for zero whatever the cache holds there
  __device__ __forceinline__ void cut(int t0, int n, int t) {
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (t0 + 2 * t + (r & 1) + 8 * (r >> 1) >= n) vp[r] = 0u;
  }
};

template <int D, int NT>
struct Query {
  uint32_t b[NT][D / 16][2];
};

template <int D, int DV, int NT>
__device__ __forceinline__ void scores_of(const Frag<D, DV>& f, const Query<D, NT>& q, float (&s)[NT][4]) {
#pragma unroll
  for (int n = 0; n < NT; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
  const uint32_t s0 = low2(f.kp[0], f.kp[0]), b0 = high2(f.kp[0], f.kp[0]);
  const uint32_t s1 = low2(f.kp[1], f.kp[1]), b1 = high2(f.kp[1], f.kp[1]);
#pragma unroll
  for (int w = 0; w < D / 32; ++w) {
    const uint32_t x = f.k[0][w], y = f.k[1][w];
    const uint32_t a0[4] = {pair_of<0>(x, s0, b0), pair_of<0>(y, s1, b1), pair_of<1>(x, s0, b0), pair_of<1>(y, s1, b1)};
    const uint32_t a1[4] = {pair_of<2>(x, s0, b0), pair_of<2>(y, s1, b1), pair_of<3>(x, s0, b0), pair_of<3>(y, s1, b1)};
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      mma::mma16816(s[n], a0, q.b[n][2 * w][0], q.b[n][2 * w][1]);
      mma::mma16816(s[n], a1, q.b[n][2 * w + 1][0], q.b[n][2 * w + 1][1]);
    }
  }
}

template <int D, int DV, int NT>
__device__ __forceinline__ void add_values(const Frag<D, DV>& f, const uint32_t (&p)[NT][2], float (&o)[DV / 16][NT][4]) {
  const uint32_t sl = low2(f.vp[0], f.vp[1]), bl = high2(f.vp[0], f.vp[1]);
  const uint32_t sh = low2(f.vp[2], f.vp[3]), bh = high2(f.vp[2], f.vp[3]);
  uint32_t xl[Frag<D, DV>::VW], yl[Frag<D, DV>::VW], xh[Frag<D, DV>::VW], yh[Frag<D, DV>::VW];
#pragma unroll
  for (int w = 0; w < Frag<D, DV>::VW; ++w) {
    xl[w] = low2(f.v[0][w], f.v[1][w]); yl[w] = high2(f.v[0][w], f.v[1][w]);
    xh[w] = low2(f.v[2][w], f.v[3][w]); yh[w] = high2(f.v[2][w], f.v[3][w]);
  }
  auto product = [&](int i, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
    const uint32_t a[4] = {a0, a1, a2, a3};
#pragma unroll
    for (int n = 0; n < NT; ++n) mma::mma16816(o[i][n], a, p[n][0], p[n][1]);
  };
  if constexpr (DV == 128) {
    // product i: rows g are nibble i of word 2 g, rows g + 8 nibble i of word 2 g + 1
#define VAGUS_KV4_V(I)                                                                                     \
  product(I, pair_of<I>(xl[0], sl, bl), pair_of<I>(xl[1], sl, bl), pair_of<I>(xh[0], sh, bh),              \
          pair_of<I>(xh[1], sh, bh));                                                                      \
  product(I + 4, pair_of<I>(yl[0], sl, bl), pair_of<I>(yl[1], sl, bl), pair_of<I>(yh[0], sh, bh),          \
          pair_of<I>(yh[1], sh, bh));
    VAGUS_KV4_V(0) VAGUS_KV4_V(1) VAGUS_KV4_V(2) VAGUS_KV4_V(3)
#undef VAGUS_KV4_V
  } else {
    // product i: rows g are nibble i of word g, rows g + 8 nibble i + 4
#define VAGUS_KV4_V(I) \
  product(I, pair_of<I>(xl[0], sl, bl), pair_of<I>(yl[0], sl, bl), pair_of<I>(xh[0], sh, bh), pair_of<I>(yh[0], sh, bh));
    VAGUS_KV4_V(0) VAGUS_KV4_V(1) VAGUS_KV4_V(2) VAGUS_KV4_V(3)
#undef VAGUS_KV4_V
  }
}

// channel of accumulator row (product i, row g or g + 8)
template <int DV>
__device__ __forceinline__ int channel_of(int i, int g, int upper) {
  return DV == 128 ? 16 * g + 8 * upper + i : 8 * g + 4 * upper + i;
}

template <int D, int DV, int NT>
__global__ void __launch_bounds__(32 * kAttnWarps) kv4_attn_k(const Kv4AttnArgs a) {
  constexpr int ROWS = 8 * NT;
  __shared__ float sm[kAttnWarps][ROWS], sl[kAttnWarps][ROWS];
  __shared__ float so[ROWS][DV + 4];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane >> 2, t = lane & 3;
  const int split = blockIdx.x, hk = blockIdx.y % a.Hk, tile = blockIdx.y / a.Hk, G = a.H / a.Hk;
  const long long b = blockIdx.z, bh = b * a.Hk + hk;
  const int R = G * a.Lq, r0 = tile * ROWS;

  long long len = a.lengths ? index_at(a.lengths, a.len_i64, b) : a.length;
  if (len > a.cap) {
    if (threadIdx.x == 0) record_error(a.err, kErrBadArgument);
    len = a.cap;
  }
  const int n = len < 0 ? 0 : static_cast<int>(len);

  // rows are numbered query-major; a row sees the first `vis` tokens, the tile
  // between `least` and `most`
  const int first = r0 / G, last = (min(r0 + ROWS, R) - 1) / G;
  const int least = a.causal ? max(0, n - a.Lq + 1 + first) : n;
  const int most = a.causal ? max(0, n - a.Lq + 1 + last) : n;
  int vis[NT][2];
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = r0 + 8 * j + 2 * t + e;
      vis[j][e] = r < R && a.causal ? max(0, n - a.Lq + 1 + r / G) : most;
    }

  Query<D, NT> q;
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int r = r0 + 8 * j + g;
    const __nv_bfloat16* src =
        static_cast<const __nv_bfloat16*>(a.q) + b * a.sq_b + (hk * G + r % G) * a.sq_h + (r / G) * a.sq_l;
#pragma unroll
    for (int w = 0; w < D / 32; ++w) {
      uint4 u = make_uint4(0, 0, 0, 0);
      if (r < R) u = *reinterpret_cast<const uint4*>(src + 8 * (t * (D / 32) + w));
      q.b[j][2 * w][0] = low2(u.x, u.z);          // channels (0, 4)
      q.b[j][2 * w][1] = high2(u.x, u.z);         // (1, 5)
      q.b[j][2 * w + 1][0] = low2(u.y, u.w);      // (2, 6)
      q.b[j][2 * w + 1][1] = high2(u.y, u.w);     // (3, 7)
    }
  }

  float o[DV / 16][NT][4], m[NT][2], l[NT][2];
#pragma unroll
  for (int i = 0; i < DV / 16; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) o[i][j][0] = o[i][j][1] = o[i][j][2] = o[i][j][3] = 0.f;
#pragma unroll
  for (int j = 0; j < NT; ++j) { m[j][0] = m[j][1] = -INFINITY; l[j][0] = l[j][1] = 0.f; }

  const int blocks = (most + kBlock - 1) / kBlock, per = (blocks + a.splits - 1) / a.splits;
  const int end = min(blocks, (split + 1) * per);
  for (int blk = split * per + warp; blk < end; blk += kAttnWarps) {
    const int t0 = blk * kBlock;
    Frag<D, DV> f[2];
    float s[2][NT][4];
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (h == 0 || t0 + 16 < most) f[h].load(a, bh, t0 + 16 * h, g, t);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int th = t0 + 16 * h;
      if (h == 0 || th < most) scores_of<D, DV, NT>(f[h], q, s[h]);
      if (th + 16 > least) {
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (th + g + 8 * (e >> 1) >= vis[j][e & 1]) s[h][j][e] = -INFINITY;
        f[h].cut(th, most, t);
      }
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      float mx[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        mx[e] = fmaxf(fmaxf(s[0][j][e], s[0][j][e + 2]), fmaxf(s[1][j][e], s[1][j][e + 2]));
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], off));
        mx[e] = fmaxf(mx[e] * a.scale_log2, m[j][e]);
      }
      const float ref0 = mx[0] == -INFINITY ? 0.f : mx[0], ref1 = mx[1] == -INFINITY ? 0.f : mx[1];
      if (__any_sync(0xffffffffu, mx[0] != m[j][0] || mx[1] != m[j][1])) {
        const float c0 = ex2_approx(m[j][0] - ref0), c1 = ex2_approx(m[j][1] - ref1);
        l[j][0] *= c0;
        l[j][1] *= c1;
#pragma unroll
        for (int i = 0; i < DV / 16; ++i) {
          o[i][j][0] *= c0; o[i][j][1] *= c1; o[i][j][2] *= c0; o[i][j][3] *= c1;
        }
        m[j][0] = mx[0];
        m[j][1] = mx[1];
      }
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[h][j][e] = ex2_approx(fmaf(s[h][j][e], a.scale_log2, -((e & 1) ? ref1 : ref0)));
          l[j][e & 1] += s[h][j][e];
        }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (h == 1 && t0 + 16 >= most) break;
      uint32_t p[NT][2];
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        p[j][0] = transpose8(pack_bf16x2(s[h][j][0], s[h][j][1]));
        p[j][1] = transpose8(pack_bf16x2(s[h][j][2], s[h][j][3]));
      }
      add_values<D, DV, NT>(f[h], p, o);
    }
  }

  // the four warps meet
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) l[j][e] += __shfl_xor_sync(0xffffffffu, l[j][e], off);
      if (g == 0) {
        sm[warp][8 * j + 2 * t + e] = m[j][e];
        sl[warp][8 * j + 2 * t + e] = l[j][e];
      }
    }
  for (int i = threadIdx.x; i < ROWS * DV; i += blockDim.x) so[i / DV][i % DV] = 0.f;
  __syncthreads();
  for (int w = 0; w < kAttnWarps; ++w) {
    if (warp == w) {
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = 8 * j + 2 * t + e;
          float all = -INFINITY;
#pragma unroll
          for (int x = 0; x < kAttnWarps; ++x) all = fmaxf(all, sm[x][r]);
          const float c = m[j][e] == -INFINITY ? 0.f : ex2_approx(m[j][e] - all);
#pragma unroll
          for (int i = 0; i < DV / 16; ++i) {
            so[r][channel_of<DV>(i, g, 0)] += c * o[i][j][e];
            so[r][channel_of<DV>(i, g, 1)] += c * o[i][j][e + 2];
          }
        }
    }
    __syncthreads();
  }
  for (int i = threadIdx.x; i < ROWS * (DV / 2); i += blockDim.x) {
    const int rr = i / (DV / 2), c = 2 * (i - rr * (DV / 2)), r = r0 + rr;
    if (r >= R) continue;
    float all = -INFINITY, sum = 0.f;
#pragma unroll
    for (int x = 0; x < kAttnWarps; ++x) all = fmaxf(all, sm[x][rr]);
#pragma unroll
    for (int x = 0; x < kAttnWarps; ++x)
      sum += sm[x][rr] == -INFINITY ? 0.f : sl[x][rr] * ex2_approx(sm[x][rr] - all);
    const int head = hk * G + r % G, qi = r / G;
    const long long orow = (b * a.Lq + qi) * a.H + head;         // o is token-major
    if (a.splits == 1) {
      const float inv = sum == 0.f ? 0.f : 1.f / sum;            // a row that sees nothing gives zeros
      *reinterpret_cast<uint32_t*>(static_cast<__nv_bfloat16*>(a.o) + orow * DV + c) =
          pack_bf16x2(so[rr][c] * inv, so[rr][c + 1] * inv);
    } else {
      const long long part = orow * a.splits + split;
      *reinterpret_cast<float2*>(a.part_o + part * DV + c) = make_float2(so[rr][c], so[rr][c + 1]);
      if (c == 0) *reinterpret_cast<float2*>(a.part_ml + 2 * part) = make_float2(all, sum);
    }
  }
}

// joins the splits of one row: a warp a row
template <int DV>
__global__ void __launch_bounds__(128) kv4_join_k(const Kv4AttnArgs a) {
  const long long row = static_cast<long long>(blockIdx.x) * 4 + threadIdx.x / 32;
  if (row >= a.B * a.Lq * a.H) return;
  const int lane = threadIdx.x % 32;
  const float* ml = a.part_ml + 2 * row * a.splits;
  const float* po = a.part_o + row * a.splits * DV;
  float all = -INFINITY;
  for (int s = lane; s < a.splits; s += 32) all = fmaxf(all, ml[2 * s]);
  all = warp_max(all);
  constexpr int N = DV / 32;
  float acc[N], sum = 0.f;
#pragma unroll
  for (int j = 0; j < N; ++j) acc[j] = 0.f;
  for (int s = 0; s < a.splits; ++s) {
    const float ms = ml[2 * s];
    if (ms == -INFINITY) continue;
    const float c = ex2_approx(ms - all);
    sum += c * ml[2 * s + 1];
#pragma unroll
    for (int j = 0; j < N; ++j) acc[j] += c * po[static_cast<long long>(s) * DV + N * lane + j];
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  __nv_bfloat16* o = static_cast<__nv_bfloat16*>(a.o) + row * DV + N * lane;
#pragma unroll
  for (int j = 0; j < N; j += 2) *reinterpret_cast<uint32_t*>(o + j) = pack_bf16x2(acc[j] * inv, acc[j + 1] * inv);
}

template <int D, int DV>
int attn_launch(const Kv4AttnArgs& a, cudaStream_t st) {
  const int R = a.H / a.Hk * a.Lq, NT = kv4_attn_tiles(a);
  const dim3 grid(a.splits, a.Hk * ((R + 8 * NT - 1) / (8 * NT)), static_cast<unsigned>(a.B));
  if (grid.y > 65535 || a.B > 65535) return 2;
  if (NT == 1) kv4_attn_k<D, DV, 1><<<grid, 32 * kAttnWarps, 0, st>>>(a);
  else kv4_attn_k<D, DV, 2><<<grid, 32 * kAttnWarps, 0, st>>>(a);
  if (cudaGetLastError() != cudaSuccess) return 3;
  if (a.splits > 1) {
    const long long rows = a.B * a.Lq * a.H;
    kv4_join_k<DV><<<static_cast<unsigned>((rows + 3) / 4), 128, 0, st>>>(a);
    if (cudaGetLastError() != cudaSuccess) return 3;
  }
  return 0;
}

}  // namespace

int kv4_append(const Kv4AppendArgs& a, int type, cudaStream_t st) {
  if (a.D % kGroup || a.Dv % kGroup || a.D < kGroup || a.Dv < kGroup) return 1;
  if (a.B * a.L * a.Hk == 0) return 0;
  const long long most = a.B * a.L * a.Hk * ((a.D > a.Dv ? a.D : a.Dv) / 8), blocks = (most + 255) / 256;
  if (blocks > 0x7fffffffLL) return 2;
  const dim3 grid(static_cast<unsigned>(blocks), 2);
  const int es = type == 0 ? 4 : 2;
  auto al = [es](const void* p, long long x, long long y, long long z) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && x * es % 16 == 0 && y * es % 16 == 0 && z * es % 16 == 0;
  };
  const bool vec = al(a.k, a.sk_b, a.sk_h, a.sk_l) && al(a.v, a.sv_b, a.sv_h, a.sv_l);
#define VAGUS_KV4_APPEND(T) \
  if (vec) kv4_append_k<T, true><<<grid, 256, 0, st>>>(a); else kv4_append_k<T, false><<<grid, 256, 0, st>>>(a)
  if (type == 0) { VAGUS_KV4_APPEND(float); }
  else if (type == 1) { VAGUS_KV4_APPEND(__half); }
  else { VAGUS_KV4_APPEND(__nv_bfloat16); }
#undef VAGUS_KV4_APPEND
  return cudaGetLastError() == cudaSuccess ? 0 : 3;
}

int kv4_read(const Kv4ReadArgs& a, cudaStream_t st) {
  if (a.D % kGroup || a.Dv % kGroup || a.D < kGroup || a.Dv < kGroup) return 1;
  if (a.B * a.L * a.Hk == 0) return 0;
  const long long most = a.B * a.L * a.Hk * ((a.D > a.Dv ? a.D : a.Dv) / 8), blocks = (most + 255) / 256;
  if (blocks > 0x7fffffffLL) return 2;
  kv4_read_k<<<dim3(static_cast<unsigned>(blocks), 2), 256, 0, st>>>(a);
  return cudaGetLastError() == cudaSuccess ? 0 : 3;
}

int kv4_attn_tiles(const Kv4AttnArgs& a) { return a.H / a.Hk * a.Lq <= 8 ? 1 : 2; }

// Splits of the tokens: enough CTAs for three a SM, each warp of a split with
// one block of 32 tokens at least.
int kv4_attn_splits(const Kv4AttnArgs& a, long long most_tokens) {
  const int NT = kv4_attn_tiles(a);
  const long long tiles = (static_cast<long long>(a.H / a.Hk) * a.Lq + 8 * NT - 1) / (8 * NT);
  const long long ctas = a.B * a.Hk * tiles, blocks = (most_tokens + kBlock - 1) / kBlock;
  long long s = (148 * 3 + ctas - 1) / ctas, most = (blocks + kAttnWarps - 1) / kAttnWarps;
  if (s > most) s = most;
  return static_cast<int>(s < 1 ? 1 : s);
}

int kv4_attn(const Kv4AttnArgs& a, cudaStream_t st) {
  if (a.Hk < 1 || a.H % a.Hk || a.splits < 1 || a.cap % 16) return 1;
  if (a.B * a.H * a.Lq == 0) return 0;
  if (a.D == 64 && a.Dv == 64) return attn_launch<64, 64>(a, st);
  if (a.D == 64 && a.Dv == 128) return attn_launch<64, 128>(a, st);
  if (a.D == 128 && a.Dv == 64) return attn_launch<128, 64>(a, st);
  if (a.D == 128 && a.Dv == 128) return attn_launch<128, 128>(a, st);
  return 1;
}

}  // namespace vagus
