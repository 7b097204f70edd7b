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
// The codes are computed from the rounded b, so its rounding, e <= 2^-8 |min - 128 s|,
// shifts the group's grid of 16 levels: a value inside the grid is off by s / 2 at most,
// one at the group's edge by at most e + 0.06 s (the rounding of s over 15 of them), and
// then the value itself rounds to bf16.  Groups near zero lose nothing by it (0.55 s at
// worst in 40000 groups of unit variance), far ones do: 0.64 s at a mean of 5 times their
// deviation, 0.93 s at 20, 1.7 s at 60, where a bf16 value's own rounding is 0.9 s.
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

__device__ __forceinline__ uint32_t low2(uint32_t a, uint32_t b) { return __byte_perm(a, b, 0x5410); }
__device__ __forceinline__ uint32_t high2(uint32_t a, uint32_t b) { return __byte_perm(a, b, 0x7632); }

// ---------------------------------------------------------------- append --

// The codes of 16 channels by their definition: (x - b) / s rounded to the nearest whole
// number (ties to even), less 128.
__device__ __noinline__ uint2 codes_by_division(const float* x, float s, float b) {
  uint32_t w[2] = {0u, 0u};
#pragma unroll 1
  for (int j = 15; j >= 0; --j) {
    const float k = rintf(__fdiv_rn(__fsub_rn(x[j], b), s));
    const uint32_t c = s > 0.f ? static_cast<uint32_t>(__float2int_rn(fminf(fmaxf(k, 128.f), 143.f)) - 128) : 0u;
    w[j / 8] = w[j / 8] * 16u + c;
  }
  return make_uint2(w[0], w[1]);
}

// The same in operations on two channels at once where there is one (the scalar ones made
// the append 107 us instead of 91).  q0 = d r with the correctly rounded reciprocal r of s,
// corrected once by its exact remainder, is the correctly rounded d / s (Markstein); outside
// the range of s where neither over- nor underflows, by division.  (Checking d r for being
// near to a half and dividing only then took a branch in two warps out of three, since a
// bf16 x lies exactly half way in one case of 500: 254 us against 115.)  Adding and
// subtracting 1.5 * 2^23 rounds to a whole number, ties to even; four codes are gathered as
// one float, whose low 16 bits they are once 2^23 is added.
__device__ __forceinline__ uint2 codes_of(const float* x, float s, float b) {
  constexpr float kRound = 12582912.f, kGather = 8388608.f - 128.f * 4369.f;      // 4369 = 1 + 16 + 256 + 4096
  if (!(s > 1e-30f && s < 1e36f)) {
    float y[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) y[j] = x[j];
    return codes_by_division(y, s, b);
  }
  const float r = __frcp_rn(s);
  const F2 r2 = pair2(r, r), ns = pair2(-s, -s), nb = pair2(-b, -b);
  const F2 up = pair2(kRound, kRound), down = pair2(-kRound, -kRound), k256 = pair2(256.f, 256.f);
  auto codes2 = [&](float x0, float x1) {
    const F2 d = add2(pair2(x0, x1), nb), q0 = mul2(d, r2);
    float t0, t1;
    halves(fma2(fma2(q0, ns, d), r2, q0), t0, t1);
    return add2(add2(pair2(fminf(fmaxf(t0, 128.f), 143.f), fminf(fmaxf(t1, 128.f), 143.f)), up), down);
  };
  uint32_t four[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    float even, odd;
    halves(fma2(codes2(x[4 * q + 2], x[4 * q + 3]), k256, codes2(x[4 * q], x[4 * q + 1])), even, odd);
    four[q] = __float_as_uint(fmaf(odd, 16.f, even) + kGather);
  }
  return make_uint2(low2(four[0], four[1]), low2(four[2], four[3]));
}

// x / 15 correctly rounded: the product with 1 / 15, corrected once by its exact remainder
// (by division outside the range where that holds).
__device__ __forceinline__ float fifteenth(float x) {
  if (!(x > 1e-30f && x < 1e37f)) return __fdiv_rn(x, 15.f);
  constexpr float c = 1.f / 15.f;
  const float q = x * c;
  return fmaf(fmaf(-15.f, q, x), c, q);
}

// the range of 16 channels held as pairs (a NaN among them gives NaN)
template <typename T> struct TwoOf;
template <> struct TwoOf<__half> { using type = __half2; };
template <> struct TwoOf<__nv_bfloat16> { using type = __nv_bfloat162; };
template <typename T> using Two = typename TwoOf<T>::type;
template <int N, typename P>
__device__ __forceinline__ void two_range(const P* w, float& lo, float& hi) {
  P a = w[0], b = w[0];
#pragma unroll
  for (int j = 1; j < N; ++j) {
    a = __hmin2_nan(a, w[j]);
    b = __hmax2_nan(b, w[j]);
  }
  lo = min_nan(to_f(a.x), to_f(a.y));
  hi = max_nan(to_f(b.x), to_f(b.y));
}

// A group of 32 channels a thread, ROWS rows a thread.  Rows go in the order (token, head) in
// which the projections leave them, so the reads are contiguous.  Bound by the arithmetic of
// the codes, some 14 operations a channel: 4.5 TB/s for 4 x 8191 tokens of 16 heads of 128
// (78 us; its reads and writes alone would take 54).  With 16 channels a thread, what a row
// costs once was paid twice: 91 us, though a call of a few tokens took 2.1 us instead of 2.3.
template <typename T, bool VEC, int ROWS>
__global__ void __launch_bounds__(256, ROWS == 1 ? 4 : sizeof(T) == 4 ? 2 : 3) kv4_append_k(const Kv4AppendArgs a) {
  const int which = blockIdx.y;                       // 0: keys, 1: values
  const int D = which ? a.Dv : a.D, per = D / kGroup, rows = 256 / per;
  const int ty = threadIdx.x / per, part = threadIdx.x - ty * per;
  const unsigned seq = blockIdx.x / a.blocks, block = blockIdx.x - seq * a.blocks;
  const long long b = seq;
  const T* x = static_cast<const T*>(which ? a.v : a.k) + b * (which ? a.sv_b : a.sk_b) + kGroup * part;
  const long long sh = which ? a.sv_h : a.sk_h, sl = which ? a.sv_l : a.sk_l;
  const unsigned total = static_cast<unsigned>(a.L) * a.Hk, Hk = a.Hk;
  const unsigned long long begin = static_cast<unsigned long long>(block) * (rows * ROWS);
  if (begin >= total) return;                         // the narrower of keys and values takes fewer blocks
  const unsigned r0 = static_cast<unsigned>(begin) + ty;
  const long long start = a.start ? index_at(a.start, a.start_i64, b) : a.offset;
  const bool idle = ty >= rows;                       // threads past the last whole row of threads

  // token and head of each row, by one division
  unsigned ls[ROWS], hs[ROWS];
  const unsigned dl = rows / Hk, dh = rows - dl * Hk;
  ls[0] = r0 / Hk;
  hs[0] = r0 - ls[0] * Hk;
#pragma unroll
  for (int i = 1; i < ROWS; ++i) {
    ls[i] = ls[i - 1] + dl;
    hs[i] = hs[i - 1] + dh;
    if (hs[i] >= Hk) {
      hs[i] -= Hk;
      ++ls[i];
    }
  }
  constexpr int N = 16 / sizeof(T);                   // elements a 16-byte load
  uint4 raw[VEC ? ROWS : 1][kGroup / N];
  if (VEC) {
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      if (!idle && r0 + i * rows < total) {
#pragma unroll
        for (int j = 0; j < kGroup / N; ++j) raw[i][j] = *reinterpret_cast<const uint4*>(x + hs[i] * sh + ls[i] * sl + j * N);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    if (idle || r0 + i * rows >= total) break;
    const unsigned l = ls[i], h = hs[i];
    float v[kGroup];
    if (VEC) {
#pragma unroll
      for (int j = 0; j < kGroup / N; ++j) {
        const T* e = reinterpret_cast<const T*>(&raw[i][j]);
#pragma unroll
        for (int k = 0; k < N; ++k) v[j * N + k] = to_f(e[k]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < kGroup; ++j) v[j] = to_f(x[h * sh + l * sl + j]);
    }
    float lo, hi;
    if constexpr (VEC && sizeof(T) == 2) {
      two_range<kGroup / 2>(reinterpret_cast<const Two<T>*>(raw[i]), lo, hi);
    } else {
      lo = hi = v[0];
#pragma unroll
      for (int j = 1; j < kGroup; ++j) { lo = min_nan(lo, v[j]); hi = max_nan(hi, v[j]); }
    }
    const unsigned long long t = static_cast<unsigned long long>(start) + l;
    if (t >= static_cast<unsigned long long>(a.cap)) {        // a start given on the device that leaves the cache
      record_error(a.err, kErrBadArgument);
      continue;
    }
    const __nv_bfloat16 s16 = __float2bfloat16_rn(fifteenth(__fsub_rn(hi, lo)));
    const float s = __bfloat162float(s16);
    const __nv_bfloat16 b16 = __float2bfloat16_rn(__fsub_rn(lo, __fmul_rn(128.f, s)));
    const float b32 = __bfloat162float(b16);
    const long long out = (b * a.Hk + h) * a.cap + static_cast<long long>(t);
    const uint2 w = codes_of(v, s, b32), u = codes_of(v + 16, s, b32);
    reinterpret_cast<uint4*>(which ? a.v_codes : a.k_codes)[out * per + part] = make_uint4(w.x, w.y, u.x, u.y);
    const __nv_bfloat162 pr = __halves2bfloat162(s16, b16);
    reinterpret_cast<uint32_t*>(which ? a.v_params : a.k_params)[out * per + part] = *reinterpret_cast<const uint32_t*>(&pr);
  }
}

// ------------------------------------------------------------------ read --

__device__ __forceinline__ uint32_t fma_bf16x2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
// Nibbles i and i + 4 of w (i = 0 .. 3) as the pair of values they stand for.  magic is 0x43004300, from the
// kernel's arguments: the logic operation takes one immediate at most, and with both constants known to the
// compiler each unpacking cost two operations (attention over 2 x 131067 tokens 90 us instead of 76).
template <int I>
__device__ __forceinline__ uint32_t pair_of(uint32_t w, uint32_t ss, uint32_t bb, uint32_t magic) {
  uint32_t x;
  asm("lop3.b32 %0, %1, 0x000F000F, %2, 0xEA;" : "=r"(x) : "r"(w >> (4 * I)), "r"(magic));   // (w & mask) | magic
  return fma_bf16x2(x, ss, bb);
}
__device__ __forceinline__ uint4 unpack(uint32_t w, uint32_t p, uint32_t magic) {
  const uint32_t ss = low2(p, p), bb = high2(p, p);
  const uint32_t p0 = pair_of<0>(w, ss, bb, magic), p1 = pair_of<1>(w, ss, bb, magic), p2 = pair_of<2>(w, ss, bb, magic),
                 p3 = pair_of<3>(w, ss, bb, magic);
  return make_uint4(low2(p0, p1), low2(p2, p3), high2(p0, p1), high2(p2, p3));
}

// A head's tokens lie one after the other in the codes, the parameters and the result, so
// word i of its codes goes with parameter i / 4 and becomes 16-byte vector i of the result.
// 8 words a thread, loaded at once; bound by its reads and writes (4 x 8191 tokens of 16
// heads of 128: 55 us, 6.4 TB/s).
constexpr int kReadWords = 8;
__global__ void __launch_bounds__(256) kv4_read_k(const Kv4ReadArgs a, unsigned blocks_k) {
  // the first blocks take the keys, the others the values
  const int which = blockIdx.x >= blocks_k;
  const unsigned block = which ? blockIdx.x - blocks_k : blockIdx.x;
  const int D = which ? a.Dv : a.D;
  const long long words = a.L * (D / 8);
  const unsigned per_head = static_cast<unsigned>((words + 256 * kReadWords - 1) / (256 * kReadWords));
  const unsigned bh = block / per_head;
  const long long i0 = static_cast<long long>(block - bh * per_head) * (256 * kReadWords) + threadIdx.x;
  // any start given on the device, brought to where nothing below overflows
  const long long given = a.start ? index_at(a.start, a.start_i64, bh / a.Hk) : a.offset;
  const long long start = given < -a.L ? -a.L : given > a.cap ? a.cap : given;
  const long long at = static_cast<long long>(bh) * a.cap + start;
  const uint32_t* codes = reinterpret_cast<const uint32_t*>(which ? a.v_codes : a.k_codes) + at * (D / 8);
  const uint32_t* params = reinterpret_cast<const uint32_t*>(which ? a.v_params : a.k_params) + at * (D / kGroup);
  uint4* out = reinterpret_cast<uint4*>(which ? a.v : a.k) + bh * words;
  // a start given on the device may leave the cache: tokens outside read as zeros
  long long lo = 0, hi = words;
  if (start < 0 || start + a.L > a.cap) {
    if (threadIdx.x == 0) record_error(a.err, kErrBadArgument);
    lo = start < 0 ? -start * (D / 8) : 0;
    hi = (a.cap - start) * (D / 8);
  }
  uint32_t w[kReadWords], p[kReadWords];
#pragma unroll
  for (int j = 0; j < kReadWords; ++j) {
    const long long i = i0 + 256 * j;
    w[j] = p[j] = 0u;
    if (i < words && i >= lo && i < hi) { w[j] = codes[i]; p[j] = params[i / 4]; }
  }
#pragma unroll
  for (int j = 0; j < kReadWords; ++j)
    if (i0 + 256 * j < words) out[i0 + 256 * j] = unpack(w[j], p[j], a.magic);
}

// Few tokens: a word a thread, over the heads of all sequences.
__global__ void __launch_bounds__(256) kv4_read_few_k(const Kv4ReadArgs a) {
  const int which = blockIdx.y, D = which ? a.Dv : a.D;
  const unsigned words = static_cast<unsigned>(a.L) * (D / 8), i = blockIdx.x * 256 + threadIdx.x, bh = i / words;
  if (bh >= a.B * a.Hk) return;
  const unsigned iw = i - bh * words, l = iw / (D / 8);
  const unsigned long long t = l + static_cast<unsigned long long>(a.start ? index_at(a.start, a.start_i64, bh / a.Hk) : a.offset);
  uint4 x = make_uint4(0, 0, 0, 0);
  if (t >= static_cast<unsigned long long>(a.cap)) {
    record_error(a.err, kErrBadArgument);
  } else {
    const long long at = (bh * a.cap + static_cast<long long>(t)) * (D / 8) + (iw - l * (D / 8));
    x = unpack(reinterpret_cast<const uint32_t*>(which ? a.v_codes : a.k_codes)[at],
               reinterpret_cast<const uint32_t*>(which ? a.v_params : a.k_params)[at / 4], a.magic);
  }
  reinterpret_cast<uint4*>(which ? a.v : a.k)[i] = x;
}

// ------------------------------------------------------------- attention --
//
// The rows of a KV head are its Lq queries times the H / Hk heads that share it,
// numbered query-major; a tile of 8 NT of them goes over the head's tokens once,
// so one pass over the cache serves them all.  Everything stays in registers:
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
// The softmax's reference is raised only when a score exceeds it by 2^8: until
// then probabilities above 1 do no harm (they keep their relative precision), and
// a 16-token tile needs no reduction over its tokens.  Probabilities are rounded
// to bf16 for the second product (2^-8 relative at most, the size of the output's own
// rounding); scores, sums and accumulators are fp32.
//
// Work.  An item is a row tile of one KV head of one sequence; its tokens are cut
// into units of 128 (each of a CTA's four warps takes 32 of them).  There are two ways
// to deal them out, and kv4_attn_plan picks the one that should end first:
//
// - by clusters: equal lengths known to the host, an item to a cluster of up to 8 CTAs
//   whose parts meet in distributed shared memory.  One launch.
// - flat: all items' units, laid end to end with two blank ones ahead of each item (what
//   starting and ending it costs), go to the CTAs in equal contiguous shares, so ragged
//   batches and few long sequences fill the GPU alike.  A CTA writes the items it has
//   whole; of the first and last item of its share it may have a part, which it leaves in
//   slot 0 or 1 of its scratch, and a second kernel adds the parts of an item in order.
//
// What bounds it: latency.  Of 16 tokens x 128 channels of K and V a warp does 64 shift /
// mask-or / fma triples, 16 products and 12 permutes in one chain from scores to products,
// at 11 warps an SM; in the ragged batch of 32 single tokens over up to 8192 tokens the ALU
// pipe (where the logic operations issue at half rate), DRAM and the issue slots are each
// half busy, and the waits are fixed latencies and loads about equally.  2 x 131067 tokens
// of 8 KV heads of 128 take 72 us (4.7 TB/s; their bytes alone 52), and about the same with
// the loads served by L2.  A ring of bulk copies into shared memory with 8, 12 or 16 warps
// an SM, and scores formed one block ahead, all measured the same within 4 percent; 4 or 5
// CTAs an SM at head dim 64 too.  Loads two tiles ahead into registers are the simplest of
// them.

constexpr int kAttnWarps = 4;
constexpr int kUnit = 32 * kAttnWarps;      // tokens
constexpr int kMaxCluster = 8;
constexpr int kHead = 2;                    // what starting and ending an item costs, in units
constexpr float kUnset = 3e38f;             // minus the softmax reference before the first score: above any score's
constexpr float kLazy = 8.f;                // raise the reference when a score exceeds it by so many powers of 2

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

// A lane's places in the tensors of one item, and the codes and parameters of the
// 16 tokens that start `token` tokens further on.
template <int D, int DV>
struct Keys {
  static constexpr int W = D / 32;
  const uint8_t *codes, *params;
  __device__ __forceinline__ void at(const Kv4AttnArgs& a, long long row, int g, int t) {
    codes = a.k_codes + (row + g) * (D / 2) + t * (4 * W);
    params = static_cast<const uint8_t*>(a.k_params) + ((row + g) * (D / kGroup) + t * W / 4) * 4;
  }
  __device__ __forceinline__ void skip(int tokens) { codes += tokens * (D / 2); params += tokens * (D / kGroup * 4); }
};
template <int D, int DV>
struct KeyFrag {
  static constexpr int W = D / 32;
  uint32_t w[2][W], p[2];
  __device__ __forceinline__ void load(const Keys<D, DV>& k, int token) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      load_words<W>(w[r], k.codes + (token + 8 * r) * (D / 2));
      p[r] = *reinterpret_cast<const uint32_t*>(k.params + (token + 8 * r) * (D / kGroup * 4));
    }
  }
};
template <int D, int DV>
struct Values {
  static constexpr int W = DV / 64;
  const uint8_t *codes, *params;
  __device__ __forceinline__ void at(const Kv4AttnArgs& a, long long row, int g, int t) {
    codes = a.v_codes + (row + 2 * t) * (DV / 2) + g * (4 * W);
    params = static_cast<const uint8_t*>(a.v_params) + ((row + 2 * t) * (DV / kGroup) + g * W / 4) * 4;
  }
  __device__ __forceinline__ void skip(int tokens) { codes += tokens * (DV / 2); params += tokens * (DV / kGroup * 4); }
};
template <int D, int DV>
struct ValueFrag {
  static constexpr int W = DV / 64;
  uint32_t w[4][W], p[4];                  // tokens 2 t, 2 t + 1, 2 t + 8, 2 t + 9
  __device__ __forceinline__ void load(const Values<D, DV>& v, int token) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int at = token + (r & 1) + 8 * (r >> 1);
      load_words<W>(w[r], v.codes + at * (DV / 2));
      p[r] = *reinterpret_cast<const uint32_t*>(v.params + at * (DV / kGroup * 4));
    }
  }
  // of 16 tokens the first n stand for what they hold, the others for zero
  __device__ __forceinline__ void cut(int n, int t) {
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (2 * t + (r & 1) + 8 * (r >> 1) >= n) p[r] = 0u;
  }
};

template <int D, int NT>
struct Query {
  uint32_t b[NT][D / 16][2];
};

template <int D, int DV, int NT>
__device__ __forceinline__ void scores_of(const KeyFrag<D, DV>& f, const Query<D, NT>& q, float (&s)[NT][4], uint32_t un) {
#pragma unroll
  for (int n = 0; n < NT; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
  const uint32_t s0 = low2(f.p[0], f.p[0]), b0 = high2(f.p[0], f.p[0]);
  const uint32_t s1 = low2(f.p[1], f.p[1]), b1 = high2(f.p[1], f.p[1]);
#pragma unroll
  for (int w = 0; w < D / 32; ++w) {
    const uint32_t x = f.w[0][w], y = f.w[1][w];
    const uint32_t a0[4] = {pair_of<0>(x, s0, b0, un), pair_of<0>(y, s1, b1, un), pair_of<1>(x, s0, b0, un),
                            pair_of<1>(y, s1, b1, un)};
    const uint32_t a1[4] = {pair_of<2>(x, s0, b0, un), pair_of<2>(y, s1, b1, un), pair_of<3>(x, s0, b0, un),
                            pair_of<3>(y, s1, b1, un)};
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      mma::mma16816(s[n], a0, q.b[n][2 * w][0], q.b[n][2 * w][1]);
      mma::mma16816(s[n], a1, q.b[n][2 * w + 1][0], q.b[n][2 * w + 1][1]);
    }
  }
}

template <int D, int DV, int NT>
__device__ __forceinline__ void add_values(const ValueFrag<D, DV>& f, const uint32_t (&p)[NT][2],
                                           float (&o)[DV / 16][NT][4], uint32_t un) {
  constexpr int W = DV / 64;
  const uint32_t sl = low2(f.p[0], f.p[1]), bl = high2(f.p[0], f.p[1]);
  const uint32_t sh = low2(f.p[2], f.p[3]), bh = high2(f.p[2], f.p[3]);
  uint32_t xl[W], yl[W], xh[W], yh[W];
#pragma unroll
  for (int w = 0; w < W; ++w) {
    xl[w] = low2(f.w[0][w], f.w[1][w]); yl[w] = high2(f.w[0][w], f.w[1][w]);
    xh[w] = low2(f.w[2][w], f.w[3][w]); yh[w] = high2(f.w[2][w], f.w[3][w]);
  }
  auto product = [&](int i, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
    const uint32_t a[4] = {a0, a1, a2, a3};
#pragma unroll
    for (int n = 0; n < NT; ++n) mma::mma16816(o[i][n], a, p[n][0], p[n][1]);
  };
  if constexpr (DV == 128) {
    // product i: rows g are nibble i of word 2 g, rows g + 8 nibble i of word 2 g + 1
#define VAGUS_KV4_V(I)                                                                                     \
  product(I, pair_of<I>(xl[0], sl, bl, un), pair_of<I>(xl[1], sl, bl, un), pair_of<I>(xh[0], sh, bh, un),              \
          pair_of<I>(xh[1], sh, bh, un));                                                                      \
  product(I + 4, pair_of<I>(yl[0], sl, bl, un), pair_of<I>(yl[1], sl, bl, un), pair_of<I>(yh[0], sh, bh, un),          \
          pair_of<I>(yh[1], sh, bh, un));
    VAGUS_KV4_V(0) VAGUS_KV4_V(1) VAGUS_KV4_V(2) VAGUS_KV4_V(3)
#undef VAGUS_KV4_V
  } else {
    // product i: rows g are nibble i of word g, rows g + 8 nibble i + 4
#define VAGUS_KV4_V(I) \
  product(I, pair_of<I>(xl[0], sl, bl, un), pair_of<I>(yl[0], sl, bl, un), pair_of<I>(xh[0], sh, bh, un), pair_of<I>(yh[0], sh, bh, un));
    VAGUS_KV4_V(0) VAGUS_KV4_V(1) VAGUS_KV4_V(2) VAGUS_KV4_V(3)
#undef VAGUS_KV4_V
  }
}

// channel of accumulator row (product i, row g or g + 8)
template <int DV>
__device__ __forceinline__ int channel_of(int i, int g, int upper) {
  return DV == 128 ? 16 * g + 8 * upper + i : 8 * g + 4 * upper + i;
}

// The running softmax of a warp over the tokens it has seen, for its 8 NT rows.
template <int D, int DV, int NT>
struct Running {
  float o[DV / 16][NT][4], l[NT][2], nref[NT][2];      // nref: minus the reference, in powers of 2

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      nref[j][0] = nref[j][1] = kUnset;
      l[j][0] = l[j][1] = 0.f;
#pragma unroll
      for (int i = 0; i < DV / 16; ++i) o[i][j][0] = o[i][j][1] = o[i][j][2] = o[i][j][3] = 0.f;
    }
  }

  // raises the references to the largest scores of this tile where those are above
  __device__ __forceinline__ void raise(const float (&s)[NT][4]) {
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float mx = fmaxf(s[j][e], s[j][e + 2]);
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
        const float to = fminf(nref[j][e], -mx), c = ex2_approx(to - nref[j][e]);
        nref[j][e] = to;
        l[j][e] *= c;
#pragma unroll
        for (int i = 0; i < DV / 16; ++i) {
          o[i][j][e] *= c;
          o[i][j][e + 2] *= c;
        }
      }
  }

  // scores -> probabilities against the references, added to the sums; as B operands in p.  A score is scaled
  // and rounded before the reference comes off, so that the largest one's power is exactly 0: one fma would
  // leave the reference's own rounding, which is past 2^127 for scores of 2^31.
  __device__ __forceinline__ void weigh(float (&s)[NT][4], float scale, uint32_t (&p)[NT][2]) {
    float above = -INFINITY;
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[j][e] = __fmul_rn(s[j][e], scale);
        above = fmaxf(above, s[j][e] + nref[j][e & 1]);
      }
    if (__any_sync(0xffffffffu, above > kLazy)) raise(s);
#pragma unroll
    for (int j = 0; j < NT; ++j) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[j][e] = ex2_approx(s[j][e] + nref[j][e & 1]);
        l[j][e & 1] += s[j][e];
      }
      p[j][0] = transpose8(pack_bf16x2(s[j][0], s[j][1]));
      p[j][1] = transpose8(pack_bf16x2(s[j][2], s[j][3]));
    }
  }
};

__device__ __forceinline__ int length_of(const Kv4AttnArgs& a, long long b) {
  long long n = a.lengths ? index_at(a.lengths, a.len_i64, b) : a.length;
  if (n > a.cap) {
    record_error(a.err, kErrBadArgument);
    n = a.cap;
  }
  return n < 0 ? 0 : static_cast<int>(n);
}
// an empty sequence has one unit too: somebody writes its zeros
__device__ __forceinline__ int units_of(int n) { return n <= kUnit ? 1 : (n + kUnit - 1) / kUnit; }

// One warp: units (blank ones included) of all sequences (times `per` items each), and with
// `flat` >= 0 the sequence that holds unit `flat` and the units before it.  The host has
// checked that the units fit 31 bits.
__device__ int scan_units(const Kv4AttnArgs& a, int per, int flat, int& seq, int& before) {
  const int lane = threadIdx.x % 32;
  if (a.lengths == nullptr) {
    const int u = (kHead + units_of(static_cast<int>(a.length))) * per;
    if (flat >= 0) { seq = flat / u; before = seq * u; }
    return u * static_cast<int>(a.B);
  }
  int run = 0;
  for (int b0 = 0; b0 < a.B; b0 += 32) {
    const int b = b0 + lane, u = b < a.B ? (kHead + units_of(length_of(a, b))) * per : 0;
    int in = u;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, in, o);
      if (lane >= o) in += up;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, flat >= 0 && run + in > flat);
    if (hit) {
      const int src = __ffs(hit) - 1;
      seq = b0 + src;
      before = run + __shfl_sync(0xffffffffu, in - u, src);
      return 0;
    }
    run += __shfl_sync(0xffffffffu, in, 31);
  }
  return run;
}

// What the four warps of a CTA have of one part of an item.
template <int DV, int NT>
struct Part {
  static constexpr int ROWS = 8 * NT;
  float m[kAttnWarps][ROWS], l[kAttnWarps][ROWS];       // softmax reference and sum
  float o[kAttnWarps][ROWS][DV + 4];
  // row rr, channels c and c + 1, over the warps
  __device__ __forceinline__ void join(int rr, int c, float& top, float& sum, float& x, float& y) const {
    top = m[0][rr];
    sum = x = y = 0.f;
#pragma unroll
    for (int w = 1; w < kAttnWarps; ++w) top = fmaxf(top, m[w][rr]);
#pragma unroll
    for (int w = 0; w < kAttnWarps; ++w) {
      const float f = ex2_approx(m[w][rr] - top);
      sum += f * l[w][rr];
      x += f * o[w][rr][c];
      y += f * o[w][rr][c + 1];
    }
  }
};

// Units [ua, ub) of an item (sequence seq of n tokens) into part; ends with a barrier.
template <int D, int DV, int NT>
__device__ __forceinline__ void attend(const Kv4AttnArgs& a, int seq, int n, int hk, int r0, int ua, int ub,
                                       Part<DV, NT>& part) {
  constexpr int ROWS = 8 * NT;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane >> 2, t = lane & 3;
  const int G = a.H / a.Hk, R = G * a.Lq;
  const uint32_t un = a.magic;
  // a row sees the first `vis` tokens; the tile between `least` and `most`
  const int first = r0 / G, last = (min(r0 + ROWS, R) - 1) / G;
  const int least = a.causal ? max(0, n - a.Lq + 1 + first) : n;
  const int most = a.causal ? max(0, n - a.Lq + 1 + last) : n;

  // this warp's tiles of 16 tokens: two neighbouring ones of every unit, up to `most`
  const int tile0 = 8 * ua + 2 * warp, tiles16 = min((most + 15) / 16, 8 * ub);
  const int left = tiles16 - tile0, count = left > 0 ? left / 8 * 2 + min(left % 8, 2) : 0;
  Keys<D, DV> kp;
  Values<D, DV> vp;
  const long long row = (static_cast<long long>(seq) * a.Hk + hk) * a.cap + 16LL * tile0;
  kp.at(a, row, g, t);
  vp.at(a, row, g, t);
  KeyFrag<D, DV> kf[2];
  ValueFrag<D, DV> vf[2];
  if (count > 0) { kf[0].load(kp, 0); vf[0].load(vp, 0); }
  if (count > 1) { kf[1].load(kp, 16); vf[1].load(vp, 16); }

  Query<D, NT> q;
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    const int r = r0 + 8 * j + g;
    const __nv_bfloat16* src = static_cast<const __nv_bfloat16*>(a.q) + seq * a.sq_b + (hk * G + r % G) * a.sq_h +
                               static_cast<long long>(r / G) * a.sq_l;
#pragma unroll
    for (int w = 0; w < D / 32; ++w) {
      uint4 x = make_uint4(0, 0, 0, 0);
      if (r < R) x = *reinterpret_cast<const uint4*>(src + 8 * (t * (D / 32) + w));
      q.b[j][2 * w][0] = low2(x.x, x.z);          // channels (0, 4)
      q.b[j][2 * w][1] = high2(x.x, x.z);         // (1, 5)
      q.b[j][2 * w + 1][0] = low2(x.y, x.w);      // (2, 6)
      q.b[j][2 * w + 1][1] = high2(x.y, x.w);     // (3, 7)
    }
  }

  Running<D, DV, NT> run;
  run.clear();
  // a tile's own registers are loaded again, for the tile two on, as soon as they are used
  auto step = [&](KeyFrag<D, DV>& k, ValueFrag<D, DV>& v, int ahead, int token, bool more) {
    float s[NT][4];
    uint32_t p[NT][2];
    scores_of<D, DV, NT>(k, q, s, un);
    if (more) k.load(kp, ahead);
    if (token + 16 > least) {
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = r0 + 8 * j + 2 * t + (e & 1);
          const int vis = r < R && a.causal ? max(0, n - a.Lq + 1 + r / G) : most;
          if (token + g + 8 * (e >> 1) >= vis) s[j][e] = -INFINITY;
        }
      v.cut(most - token, t);
    }
    run.weigh(s, a.scale_log2, p);
    add_values<D, DV, NT>(v, p, run.o, un);
    if (more) v.load(vp, ahead);
  };
  for (int i = 0, token = 16 * tile0; i < count; i += 2, token += kUnit) {
    step(kf[0], vf[0], kUnit, token, i + 2 < count);
    if (i + 1 < count) step(kf[1], vf[1], kUnit + 16, token + 16, i + 3 < count);
    kp.skip(kUnit);
    vp.skip(kUnit);
  }

#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = 8 * j + 2 * t + e;
      float l = run.l[j][e];
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
      if (g == 0) {
        part.m[warp][r] = -run.nref[j][e];
        part.l[warp][r] = l;
      }
#pragma unroll
      for (int i = 0; i < DV / 16; ++i) {
        part.o[warp][r][channel_of<DV>(i, g, 0)] = run.o[i][j][e];
        part.o[warp][r][channel_of<DV>(i, g, 1)] = run.o[i][j][e + 2];
      }
    }
  __syncthreads();
}

// row r of KV head hk, channels c and c + 1; o is token-major.  A row that sees nothing gives zeros.
template <int DV>
__device__ __forceinline__ void store_row(const Kv4AttnArgs& a, int seq, int hk, int r, int c, float sum, float x, float y) {
  const int G = a.H / a.Hk;
  const long long row = (static_cast<long long>(seq) * a.Lq + r / G) * a.H + hk * G + r % G;
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  *reinterpret_cast<uint32_t*>(static_cast<__nv_bfloat16*>(a.o) + row * DV + c) = pack_bf16x2(x * inv, y * inv);
}

constexpr int ctas_per_sm(int NT) { return NT == 1 ? 3 : 2; }

template <int D, int DV, int NT>
__global__ void __launch_bounds__(32 * kAttnWarps, ctas_per_sm(NT)) kv4_attn_k(const Kv4AttnArgs a) {
  constexpr int ROWS = 8 * NT;
  __shared__ Part<DV, NT> part;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int R = a.H / a.Hk * a.Lq, tiles = (R + ROWS - 1) / ROWS, per = a.Hk * tiles;
  int seq = 0, before = 0;
  const int total = scan_units(a, per, -1, seq, before);
  const int share = (total + gridDim.x - 1) / gridDim.x;
  int u = min(total, static_cast<int>(blockIdx.x) * share);
  const int end = min(total, u + share);
  if (u >= end) return;
  scan_units(a, per, u, seq, before);
  bool first_of_share = true;

  while (u < end) {
    // the item that holds unit u, and the part of it that is this CTA's
    const int n = length_of(a, seq), units = units_of(n);
    const int item = (u - before) / (kHead + units), item0 = before + item * (kHead + units) + kHead;
    const int ua = max(0, u - item0), ub = min(end - item0, units);
    if (ub <= 0) break;                       // only blank units of it: the next CTA starts it
    const int hk = item / tiles, r0 = (item - hk * tiles) * ROWS;
    attend<D, DV, NT>(a, seq, n, hk, r0, ua, ub, part);

    const bool alone = ua == 0 && ub == units;
    const long long slot = 2LL * blockIdx.x + (first_of_share ? 0 : 1);
    for (int i = threadIdx.x; i < ROWS * (DV / 2); i += blockDim.x) {
      const int rr = i / (DV / 2), c = 2 * (i - rr * (DV / 2));
      if (r0 + rr >= R) break;
      float top, sum, x, y;
      part.join(rr, c, top, sum, x, y);
      if (alone) {
        store_row<DV>(a, seq, hk, r0 + rr, c, sum, x, y);
      } else {
        *reinterpret_cast<float2*>(a.part_o + (slot * ROWS + rr) * DV + c) = make_float2(x, y);
        if (c == 0) *reinterpret_cast<float2*>(a.part_ml + 2 * (slot * ROWS + rr)) = make_float2(top, sum);
      }
    }
    __syncthreads();
    u = item0 + ub;
    first_of_share = false;
    if (item + 1 == per && ub == units) {
      before = u;
      ++seq;
    }
  }
}

// One CTA a row of an item whose units several CTAs of the first kernel shared: the largest
// reference of its parts, then their weighted sum, a fixed set of parts a warp, then the warps.
template <int DV, int NT, int kJoinWarps>
__global__ void __launch_bounds__(32 * kJoinWarps) kv4_join_k(const Kv4AttnArgs a) {
  constexpr int ROWS = 8 * NT, N = DV / 32;
  __shared__ float sm[kJoinWarps], sl[kJoinWarps], so[kJoinWarps][DV];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int R = a.H / a.Hk * a.Lq, tiles = (R + ROWS - 1) / ROWS, per = a.Hk * tiles;
  const int item = blockIdx.x % per, hk = item / tiles, rr = blockIdx.y, r = (item - hk * tiles) * ROWS + rr;
  const int seq = blockIdx.x / per;
  int before = 0, total, none;
  if (a.lengths == nullptr) {
    total = scan_units(a, per, -1, none, none);
    before = seq * (total / static_cast<int>(a.B));
  } else {
    total = 0;
    for (int b = lane; b < a.B; b += 32) {
      const int x = (kHead + units_of(length_of(a, b))) * per;
      total += x;
      if (b < seq) before += x;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      total += __shfl_xor_sync(0xffffffffu, total, o);
      before += __shfl_xor_sync(0xffffffffu, before, o);
    }
  }
  const int share = (total + a.ctas - 1) / a.ctas, units = units_of(length_of(a, seq));
  const int u0 = before + item * (kHead + units) + kHead, c0 = u0 / share, c1 = (u0 + units - 1) / share;
  asm volatile("griddepcontrol.wait;" ::: "memory");   // the first kernel is done and its writes are here
  if (r >= R || c0 == c1) return;                      // one CTA had it whole and has written it
  // where CTA c left it: slot 0, the first item of its share, but for a CTA c0 whose share begins before it (and its
  // blank units)
  const int late = c0 * share < u0 - kHead;
  auto place = [&](int c) { return (2LL * c + (c == c0 ? late : 0)) * ROWS + rr; };
  float top = -kUnset;
  for (int c = c0 + threadIdx.x; c <= c1; c += 32 * kJoinWarps) top = fmaxf(top, a.part_ml[2 * place(c)]);
  top = warp_max(top);
  if (lane == 0) sm[warp] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kJoinWarps; ++w) top = fmaxf(top, sm[w]);
  float acc[N], l = 0.f;
#pragma unroll
  for (int j = 0; j < N; ++j) acc[j] = 0.f;
#pragma unroll 4
  for (int c = c0 + warp; c <= c1; c += kJoinWarps) {
    const long long at = place(c);
    const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + 2 * at);
    const float f = ex2_approx(ml.x - top);
    const float* po = a.part_o + at * DV + N * lane;
    l += f * ml.y;
#pragma unroll
    for (int j = 0; j < N; ++j) acc[j] += f * po[j];
  }
  if (lane == 0) sl[warp] = l;
#pragma unroll
  for (int j = 0; j < N; ++j) so[warp][N * lane + j] = acc[j];
  __syncthreads();
  if (threadIdx.x >= DV / 2) return;
  float sum = 0.f, x = 0.f, y = 0.f;
#pragma unroll
  for (int w = 0; w < kJoinWarps; ++w) {
    sum += sl[w];
    x += so[w][2 * threadIdx.x];
    y += so[w][2 * threadIdx.x + 1];
  }
  store_row<DV>(a, seq, hk, r, 2 * threadIdx.x, sum, x, y);
}

__device__ __forceinline__ float ld_cluster_f32(const float* p, int rank) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(mapa_shared(smem_u32(p), rank)) : "memory");
  return v;
}

// An item a cluster: CTA `rank` of `a.cluster` has an equal share of its units.
template <int D, int DV, int NT>
__global__ void __launch_bounds__(32 * kAttnWarps, ctas_per_sm(NT)) kv4_attn_cluster_k(const Kv4AttnArgs a) {
  constexpr int ROWS = 8 * NT;
  __shared__ Part<DV, NT> part;
  __shared__ float top_of[ROWS], sum_of[ROWS];
  const int R = a.H / a.Hk * a.Lq, tiles = (R + ROWS - 1) / ROWS, per = a.Hk * tiles, C = a.cluster;
  const int flat = blockIdx.x / C, rank = blockIdx.x - flat * C, seq = flat / per, item = flat - seq * per;
  const int hk = item / tiles, r0 = (item - hk * tiles) * ROWS;
  const int n = static_cast<int>(a.length), units = units_of(n), share = (units + C - 1) / C;
  attend<D, DV, NT>(a, seq, n, hk, r0, min(units, rank * share), min(units, (rank + 1) * share), part);

  const int rows = min(ROWS, R - r0);
  for (int i = threadIdx.x; i < rows * (DV / 2); i += blockDim.x) {
    const int rr = i / (DV / 2), c = 2 * (i - rr * (DV / 2));
    float top, sum, x, y;
    part.join(rr, c, top, sum, x, y);
    if (C == 1) {
      store_row<DV>(a, seq, hk, r0 + rr, c, sum, x, y);
    } else {                                  // this thread alone reads these places of the warps' parts
      part.o[0][rr][c] = x;
      part.o[0][rr][c + 1] = y;
      if (c == 0) {
        top_of[rr] = top;
        sum_of[rr] = sum;
      }
    }
  }
  if (C == 1) return;
  cluster_sync();
  for (int i = rank * blockDim.x + threadIdx.x; i < rows * (DV / 2); i += C * blockDim.x) {
    const int rr = i / (DV / 2), c = 2 * (i - rr * (DV / 2));
    float top = -kUnset, sum = 0.f, x = 0.f, y = 0.f, tops[kMaxCluster];
#pragma unroll
    for (int k = 0; k < kMaxCluster; ++k) {
      tops[k] = k < C ? ld_cluster_f32(&top_of[rr], k) : -kUnset;
      top = fmaxf(top, tops[k]);
    }
#pragma unroll
    for (int k = 0; k < kMaxCluster; ++k) {
      if (k >= C) break;
      const float f = ex2_approx(tops[k] - top);
      sum += f * ld_cluster_f32(&sum_of[rr], k);
      x += f * ld_cluster_f32(&part.o[0][rr][c], k);
      y += f * ld_cluster_f32(&part.o[0][rr][c + 1], k);
    }
    store_row<DV>(a, seq, hk, r0 + rr, c, sum, x, y);
  }
  cluster_sync();                              // nobody leaves while it is read
}

int tiles_of(const Kv4AttnArgs& a) { return a.H / a.Hk * a.Lq <= 8 ? 1 : 2; }

template <typename... Args>
int launch_with(void (*kernel)(Args...), dim3 grid, int threads, cudaStream_t st, cudaLaunchAttribute attr, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.stream = st;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...) == cudaSuccess ? 0 : 3;
}

template <int D, int DV, int NT>
int attn_launch(const Kv4AttnArgs& a, cudaStream_t st) {
  const int R = a.H / a.Hk * a.Lq;
  const unsigned items = static_cast<unsigned>(a.B * a.Hk * ((R + 8 * NT - 1) / (8 * NT)));
  cudaLaunchAttribute attr = {};
  if (a.cluster > 0) {
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = a.cluster;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    return launch_with(kv4_attn_cluster_k<D, DV, NT>, dim3(items * a.cluster), 32 * kAttnWarps, st, attr, a);
  }
  kv4_attn_k<D, DV, NT><<<a.ctas, 32 * kAttnWarps, 0, st>>>(a);
  if (cudaGetLastError() != cudaSuccess) return 3;
  // launched while the first kernel runs; it waits for that one's writes itself
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  const dim3 rows(items, R < 8 * NT ? R : 8 * NT);
  // eight warps where an item has many parts (131072 tokens of one head: 20 us against 37), four where most have one
  // or two (1024 items of 300 tokens: 28 us against 33)
  if (a.ctas > 16LL * items) return launch_with(kv4_join_k<DV, NT, 8>, rows, 256, st, attr, a);
  return launch_with(kv4_join_k<DV, NT, 4>, rows, 128, st, attr, a);
}

}  // namespace

int kv4_append(Kv4AppendArgs a, int type, cudaStream_t st) {
  if (a.D % kGroup || a.Dv % kGroup || a.D < kGroup || a.Dv < kGroup || a.D > 4096 || a.Dv > 4096) return 1;
  if (a.B * a.L * a.Hk == 0) return 0;
  if (a.L * a.Hk > 0x7fffffffLL - 65536) return 2;
  const int widest = a.D > a.Dv ? a.D : a.Dv;
  // two rows a thread, whose loads overlap, once that still makes 16 blocks an SM (4 x 8191 tokens of 16 heads of 128:
  // 78 us against 84); one row below (2 x 4096 tokens of 16 heads of 64: 11 us against 16)
  const int each = a.B * a.L * a.Hk * (widest / kGroup) >= 2LL * 256 * 148 * 16 ? 2 : 1;
  const int rows = each * (256 / (widest / kGroup));       // rows a block takes
  a.blocks = static_cast<unsigned>((a.L * a.Hk + rows - 1) / rows);
  if (a.B * a.blocks > 0x7fffffffLL) return 2;
  const dim3 grid(static_cast<unsigned>(a.B * a.blocks), 2);
  const int es = type == 0 ? 4 : 2;
  auto al = [es](const void* p, long long x, long long y, long long z) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && x * es % 16 == 0 && y * es % 16 == 0 && z * es % 16 == 0;
  };
  const bool vec = al(a.k, a.sk_b, a.sk_h, a.sk_l) && al(a.v, a.sv_b, a.sv_h, a.sv_l);
#define VAGUS_KV4_APPEND(T)                                              \
  if (vec && each == 2) kv4_append_k<T, true, 2><<<grid, 256, 0, st>>>(a); \
  else if (vec) kv4_append_k<T, true, 1><<<grid, 256, 0, st>>>(a);        \
  else if (each == 2) kv4_append_k<T, false, 2><<<grid, 256, 0, st>>>(a); \
  else kv4_append_k<T, false, 1><<<grid, 256, 0, st>>>(a)
  if (type == 0) { VAGUS_KV4_APPEND(float); }
  else if (type == 1) { VAGUS_KV4_APPEND(__half); }
  else { VAGUS_KV4_APPEND(__nv_bfloat16); }
#undef VAGUS_KV4_APPEND
  return cudaGetLastError() == cudaSuccess ? 0 : 3;
}

int kv4_read(Kv4ReadArgs a, cudaStream_t st) {
  if (a.D % kGroup || a.Dv % kGroup || a.D < kGroup || a.Dv < kGroup) return 1;
  if (a.B * a.L * a.Hk == 0) return 0;
  a.magic = 0x43004300u;
  // fewer words a head than a block of the first kernel takes (one token of 64 sequences of 8 heads: 1.9 us
  // against 4.6 with a block a head)
  const long long widest = a.L * ((a.D > a.Dv ? a.D : a.Dv) / 8), flat = a.B * a.Hk * widest;
  if (widest < 256 * kReadWords && flat < 0x7fffff00LL) {
    kv4_read_few_k<<<dim3(static_cast<unsigned>((flat + 255) / 256), 2), 256, 0, st>>>(a);
    return cudaGetLastError() == cudaSuccess ? 0 : 3;
  }
  auto blocks = [&](int D) { return a.B * a.Hk * ((a.L * (D / 8) + 256 * kReadWords - 1) / (256 * kReadWords)); };
  const long long k = blocks(a.D), v = blocks(a.Dv);
  if (k + v > 0x7fffffffLL) return 2;
  kv4_read_k<<<static_cast<unsigned>(k + v), 256, 0, st>>>(a, static_cast<unsigned>(k));
  return cudaGetLastError() == cudaSuccess ? 0 : 3;
}

// How the units are dealt out (see above).  A way's length is the units of its longest CTA; the flat one's
// second kernel costs as much as some five units more (3 us against 0.6 to 0.7 us a unit).
int kv4_attn_plan(Kv4AttnArgs& a, long long most_tokens) {
  const int NT = tiles_of(a);
  const long long tiles = (static_cast<long long>(a.H / a.Hk) * a.Lq + 8 * NT - 1) / (8 * NT);
  const long long items = a.B * a.Hk * tiles, per_item = most_tokens <= kUnit ? 1 : (most_tokens + kUnit - 1) / kUnit;
  const long long units = items * (kHead + per_item), slots = 148LL * ctas_per_sm(NT);
  if (units > 0x3fffffffLL || items > 0x0fffffffLL) return 2;
  a.magic = 0x43004300u;
  a.ctas = static_cast<int>(units < slots ? units : slots);
  a.part_rows = 2LL * a.ctas * 8 * NT;
  a.cluster = 0;
  if (a.lengths == nullptr && items <= slots) {
    long long c = slots / items;
    if (c > kMaxCluster) c = kMaxCluster;
    if (c > per_item) c = per_item;
    const long long by_cluster = (per_item + c - 1) / c, by_flat = (units + slots - 1) / slots + 5;
    if (by_cluster <= by_flat) {
      a.cluster = static_cast<int>(c);
      a.part_rows = 0;
    }
  }
  return 0;
}

// Whether many query rows over equal lengths are better served by unpacking the values once and running the
// tcgen05 attention on them.  At head dim 128 the kernels above take 5.2 ns a unit and tile of 16 rows, on the whole
// GPU; the other way takes the read, some 12 us of launches and, a wave of 128-row CTAs, 1.5 us per 128 tokens.
// Measured, codes against unpacked.  16 heads of 128 over 8192 tokens: 62 / 103 / 124 / 146 / 187 / 351 us against 114
// to 118 at 128 / 256 / 320 / 384 / 512 / 1024 rows; the rule changes sides between 320 and 384.  16 heads of 64 over
// 32768 tokens: 122 / 218 / 269 / 306 / 361 / 396 / 765 against 386 to 392 at 128 / 256 / 320 / 384 / 448 / 512 / 1024.
// There a tile takes about 2.9 ns, which the one constant does not know: the rule changes sides between 256 and 320
// rows, and from there to 512 it takes the slower way.
bool kv4_attn_unpack_first(const Kv4AttnArgs& a) {
  if (a.lengths || a.Lq < 128 || a.length < 128 || a.Lq > a.length || a.D != a.Dv || a.B * a.H == 0) return false;
  if (a.B * a.H > 65535) return false;       // that attention's grid holds batch times heads in its second dimension
  const double tiles = (static_cast<double>(a.H / a.Hk) * a.Lq + 15) / 16, units = (a.length + kUnit - 1) / kUnit;
  const double here = 0.0052 * a.B * a.Hk * tiles * units;
  const long long ctas = a.B * a.H * ((a.Lq + 127) / 128), wave = a.D == 64 ? 296 : 148;
  const double there = 12 + 5e-7 * a.B * a.Hk * a.length * (a.D + a.Dv) + 1.5 * ((ctas + wave - 1) / wave) * units;
  return there < here;
}

int kv4_attn(const Kv4AttnArgs& a, cudaStream_t st) {
  if (a.Hk < 1 || a.H % a.Hk || (a.cluster < 1 && a.ctas < 1) || a.cap % 16) return 1;
  if (a.B * a.H * a.Lq == 0) return 0;
#define VAGUS_KV4_ATTN(D_, DV_) \
  if (a.D == D_ && a.Dv == DV_) return tiles_of(a) == 1 ? attn_launch<D_, DV_, 1>(a, st) : attn_launch<D_, DV_, 2>(a, st)
  VAGUS_KV4_ATTN(64, 64);
  VAGUS_KV4_ATTN(64, 128);
  VAGUS_KV4_ATTN(128, 64);
  VAGUS_KV4_ATTN(128, 128);
#undef VAGUS_KV4_ATTN
  return 1;
}

}  // namespace vagus
