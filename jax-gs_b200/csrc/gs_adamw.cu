// AdamW over many tensors at once, with the moments in 32 bits or in 8, the
// global gradient norm that clips it, and the conversions of the 8-bit
// moments.
//
// For element e of a tensor, c steps taken before this one, t = c + 1:
//   g  = s grad                        (s: device scalar, or 1)
//   m' = b1 m + (1 - b1) g,   v' = b2 v + (1 - b2) g^2
//   p' = p - lr (m' / (1 - b1^t) / (sqrt(v' / (1 - b2^t)) + eps) + wd p)
// in fp32 throughout; m' and v' are sums of two rounded products (no FMA), so
// that the 8-bit codes are a function of the inputs that any fp32
// implementation reproduces bit for bit (but the sign of a zero). p' takes a
// root and a quotient that are rounded to nearest; only the kernel for many
// elements with 8-bit moments takes the approximate ones (adamw_param4_fast).
//
// 8-bit moments. A block is 128 elements, counted from the tensor's start.
// Each moment has one exponent byte a block,
//   F = (bits(max |x|) + 0xfffff) >> 23,
// the smallest biased power of two under which the maximum, rounded up to 3
// mantissa bits, still has the top code. Scaling by a power of two is exact,
// so nothing but the code's own rounding is lost and no division is needed.
// m: sign, 4 exponent and 3 mantissa bits; v >= 0 needs no sign: 5 exponent
// and 3 mantissa bits, 32 octaves, so that sqrt(v) has the 16 octaves of m.
// y = |x| 2^(127 - F) 2^-112 (m) or 2^-96 (v) has the code's exponent field
// in place and its underflow in fp32's own subnormals; code = (bits(y) +
// noise) >> 20. noise is 16 random bits << 4: a step changes v by about 1 - b2
// of itself, far below half a step of any 8-bit float, so rounding to nearest
// would freeze v where it stands; rounding up with the probability of the
// remainder keeps its mean. A v > 0 is never stored as 0 (the update of a
// nonzero m over sqrt(0) + eps would be unbounded). F = 255 marks a block
// with a value that is not finite: all of it reads as NaN.
//
// Bytes an element with fp32 gradients: 28 with 32-bit moments, 16 with 8-bit
// ones. Measured on a B200 whose copies run at 6.45 TB/s: the 32-bit step on
// 59M elements 260 us (28 B: 6.35 TB/s, bound by HBM); the 8-bit step on 236M
// elements, a quarter of them in rows that are off, 576 us (13.5 B moved:
// 5.5 TB/s), bound by HBM and by the issue of 62 instructions an element
// (2.7 of 4 a cycle); the norm of 236M fp32 gradients 141 us (6.7 TB/s, some
// of it from L2).
#include <algorithm>
#include <cmath>

#include "gs_kernels.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace gs {

constexpr int kAdamwBlock = GS_ADAMW_BLOCK;  // elements of a block of 8-bit moments, and what a warp does at least
constexpr int kAdamwWarps = 8;
constexpr int kAdamwUnroll = 2;  // blocks of a chunk, what a warp takes at a time (32-bit moments)
constexpr int kAdamwChunk = kAdamwBlock * kAdamwUnroll;
constexpr int kAdamwTile = kAdamwChunk * kAdamwWarps;  // elements a CTA takes at a time
static_assert(kAdamwBlock == 128, "a warp holds a block, four elements a lane");
// CTAs an SM, which bound the registers. 32-bit moments, 59M elements: 2 or 3
// CTAs of 256 262 us, 4 276, 5 291 (and 1 block a chunk 278, 4 blocks 264).
#ifndef GS_ADAMW_CTAS
#define GS_ADAMW_CTAS 3
#endif
// 8-bit moments, 236M elements: 5 CTAs of 128 (as many as the shared memory
// holds) 567 us, 4 596.
#ifndef GS_ADAMW8_CTAS
#define GS_ADAMW8_CTAS 5
#endif
// Blocks per SM up to which every warp takes one (k_adamw_small). 32-bit
// moments: 118k elements 4.3 us so and 4.6 in chunks, 177k 4.4 and 4.0, 590k
// 5.5 and 4.3. 8-bit: 59k 4.8 and 7.1, 590k 6.9 and 7.4, 885k 8.2 and 7.5.
#ifndef GS_ADAMW_SMALL
#define GS_ADAMW_SMALL 8
#endif
#ifndef GS_ADAMW8_SMALL
#define GS_ADAMW8_SMALL 32
#endif
// Gradient norm: 16-byte loads a thread has in flight, and CTAs of 256 an SM.
// 236M fp32 gradients: 2 x 8 and 4 x 4 141 us (the rate of a copy), 2 x 4 173.
#ifndef GS_NORM_VECS
#define GS_NORM_VECS 2
#endif
#ifndef GS_NORM_CTAS
#define GS_NORM_CTAS 8
#endif
// Decoding: groups of 8 codes of each moment a thread has in flight. 236M
// elements to bf16: 1 252 us, 2 244, 4 251.
#ifndef GS_DECODE_UNROLL
#define GS_DECODE_UNROLL 2
#endif

// One tensor as the kernels see it.
struct AdamwDesc {
  float* param;
  const void* grad;
  void* mu;
  void* nu;
  uint8_t* mu_exp;
  uint8_t* nu_exp;
  void* copy;
  const uint8_t* active;
  long long count;
  float lr_init, ln_decay, weight_decay;  // lr = lr_init exp(c ln_decay)
  unsigned width;                         // elements per active flag
  unsigned long long magic;               // ceil(2^64 / width)
  uint8_t grad_type, copy_type, vec;
  uint8_t skip;  // elements of the first row that lie before the first element (below 4)
  int index;     // place in the caller's list (the noise key)
};
// AdamwDesc::vec: accesses of one element, of four, and (8-bit moments, fp32
// gradients) of four but for the parameter and the gradient, which are not
// 16-byte aligned: they pass through shared memory word by word (59M elements:
// 201 us, aligned 161). 8-bit moments with 16-bit gradients off the alignment
// are kScalar, element by element (59M: 777 us, aligned 158), as are 32-bit
// ones whose arrays lie differently far behind it (275 us, aligned 258).
constexpr int kScalar = 0, kVec = 1, kLoose = 2;

// Tables travel as kernel parameters (no device copy, nothing to keep alive,
// and a captured graph holds its own); N is a size class.
template <int N>
struct AdamwTable {
  AdamwDesc t[N];
  int first[N + 1];  // first tile of each tensor; first[n] = tiles
  int n;
};

// The tensor of a tile, the last whose first tile is not behind it, by a whole
// warp, 32 entries at a time. first[n] is behind every tile.
template <int N>
__device__ __forceinline__ int tensor_after(const int (&first)[N], int n, int tile, int k) {
  const int lane = threadIdx.x & 31;
  for (int hits = 32; hits == 32; k += hits)
    hits = __popc(__ballot_sync(0xffffffffu, first[min(k + 1 + lane, n)] <= tile));
  return k;
}
template <int N>
__device__ __forceinline__ int tensor_of(const int (&first)[N], int n, int tile) {
  const int lane = threadIdx.x & 31, stride = (n + 31) / 32;
  const int hits = __popc(__ballot_sync(0xffffffffu, first[min(lane * stride, n)] <= tile));
  return tensor_after(first, n, tile, max(hits - 1, 0) * stride);
}

struct AdamwParams {
  float b1, omb1, b2, omb2, eps, ln_b1, ln_b2;
  unsigned seed;
  bool fine_root;  // eps is so small that the root of a subnormal v counts beside it
  const float* scale;
  int* state;    // [count, ticket, skipped, 0]
  bool advance;  // this launch is the step's last
};

__device__ __forceinline__ unsigned mix32(unsigned x) {
  // an integer hash from C. Wellons, "Prospecting for Hash Functions" (2018)
  x ^= x >> 16;
  x *= 0x7feb352du;
  x ^= x >> 15;
  x *= 0x846ca68bu;
  return x ^ (x >> 16);
}
constexpr unsigned kGolden = 0x9E3779B9u;

// 2^(field - 127), field 0 .. 254
__device__ __forceinline__ float pow2_biased(int field) {
  return __int_as_float(field > 0 ? field << 23 : 0x00400000);
}

// Exponent byte of a block from the largest bit pattern of its magnitudes.
__device__ __forceinline__ int block_field(unsigned top) {
  return min((int)((top + 0xFFFFFu) >> 23), 255);
}

template <bool SIGNED>
__device__ __forceinline__ float decode8(unsigned code, float up) {
  const float y = __uint_as_float((SIGNED ? (code & 127u) : code) << 20) * (SIGNED ? 0x1p112f : 0x1p96f) * up;
  return (SIGNED && code > 127u) ? -y : y;
}

// noise in [0, 2^20); down = 2^(127 - F)
template <bool SIGNED>
__device__ __forceinline__ unsigned encode8(float x, float down, unsigned noise) {
  const float y = fabsf(x) * down * (SIGNED ? 0x1p-112f : 0x1p-96f);
  unsigned c = min((__float_as_uint(y) + noise) >> 20, SIGNED ? 127u : 255u);
  if (SIGNED) return c | ((__float_as_uint(x) >> 31) << 7);
  return (c == 0u && x > 0.f) ? 1u : c;
}

__device__ __forceinline__ float load_as_float(const void* p, long long i, int type) {
  if (type == GS_TYPE_F32) return static_cast<const float*>(p)[i];
  if (type == GS_TYPE_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(static_cast<const __half*>(p)[i]);
}

__device__ __forceinline__ void store_as(void* p, long long i, int type, float x) {
  if (type == GS_TYPE_BF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(x);
  else static_cast<__half*>(p)[i] = __float2half_rn(x);
}

struct AdamwStep {
  float inv1, inv2;   // 1 / (1 - b^t)
  float rate, decay;  // lr inv1 and -lr wd of the tensor
};

// p - lr (m inv1 / (sqrt(v inv2) + eps) + wd p) for four elements, with one
// rounding of p's own size: the decay joins the update, not p. Root and quotient
// are to nearest but for a few near ties: the approximations and one Newton step
// each. x = v inv2 that overflowed stays an infinite denominator (x 2^-126 is
// below 2^-62 of the root of any other x), clamped to a number whose
// approximate reciprocal is 0; NaN passes. The root of a subnormal x is below
// 2^-63 and comes out anywhere below that, which changes a denominator by less
// than a rounding unless eps < 2^-39: then the compiler's root and quotient.
// 32-bit moments, bound by memory: 59M elements 260 us, 259 with the
// approximations alone, 273 with the compiler's; 12M, half of them off: 45.5,
// 45.2, 60.
__device__ __forceinline__ void adamw_param4(const float p[4], const float m[4], const float v[4], const AdamwStep& h,
                                             const AdamwParams& a, float out[4]) {
  constexpr float kMost = 3.402823466e38f, kLeast = 0x1p-126f;
  if (a.fine_root) {
#pragma unroll
    for (int q = 0; q < 4; ++q)
      out[q] = p[q] + fmaf(h.decay, p[q], -__fdiv_rn(m[q] * h.rate, __fsqrt_rn(v[q] * h.inv2) + a.eps));
    return;
  }
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const float x = v[q] * h.inv2, n = m[q] * h.rate;
    float xc, y, den, r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(xc) : "f"(x), "f"(kMost));
    asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(fmaxf(xc, kLeast)));
    const float s = xc * y;
    const float root = fmaf(fmaf(-s, s, xc), 0.5f * y, s);
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(den) : "f"(root + fmaf(x, kLeast, a.eps)), "f"(kMost));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(den));
    const float t = n * r;
    out[q] = p[q] + fmaf(h.decay, p[q], -fmaf(fmaf(-t, den, n), r, t));
  }
}

// The same with the approximate root and reciprocal (2^-23 of each at most):
// the update is off by up to 4 units of 2^-24 instead of 2, below its own
// uncertainty from moments of 4 significant bits. For k_adamw8, which is bound
// by the issue of instructions: 236M elements 575 us so, 626 with the Newton
// steps, 955 with the compiler's root and quotient. eps is a normal float, so
// the denominator is one too and lies far below 2^126: the approximate
// reciprocal needs no care for subnormals.
__device__ __forceinline__ void adamw_param4_fast(const float p[4], const float m[4], const float v[4],
                                                  const AdamwStep& h, const AdamwParams& a, float out[4]) {
  float root[4];
  if (a.fine_root) {
#pragma unroll
    for (int q = 0; q < 4; ++q) asm("sqrt.approx.f32 %0, %1;" : "=f"(root[q]) : "f"(v[q] * h.inv2));
  } else {
#pragma unroll
    for (int q = 0; q < 4; ++q) asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(root[q]) : "f"(v[q] * h.inv2));
  }
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    float inv;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(root[q] + a.eps));
    out[q] = p[q] + fmaf(-(m[q] * h.rate), inv, h.decay * p[q]);
  }
}

// Largest magnitude of four, NaN if one is.
__device__ __forceinline__ float max_abs4(const float x[4]) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x[0]), "f"(x[1]), "f"(x[2]));
  asm("max.NaN.abs.f32 %0, %1, %2, %2;" : "=f"(r) : "f"(r), "f"(x[3]));
  return r;
}

__device__ __forceinline__ float max_abs8(const float x[8]) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x[0]), "f"(x[1]), "f"(x[2]));
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(r), "f"(x[3]), "f"(x[4]));
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(r), "f"(x[5]), "f"(x[6]));
  asm("max.NaN.abs.f32 %0, %1, %2, %2;" : "=f"(r) : "f"(r), "f"(x[7]));
  return r;
}

// Element q of a lane in a block: four consecutive elements a lane (16-byte
// accesses), or, where a pointer is not aligned for that, every 32nd.
template <bool VEC>
__device__ __forceinline__ int block_element(int lane, int q) {
  return VEC ? 4 * lane + q : lane + 32 * q;
}

// Four elements of a lane, the first at p[i].
template <bool VEC>
__device__ __forceinline__ void load4(const float* p, unsigned i, float x[4]) {
  if (VEC) {
    const float4 t = *reinterpret_cast<const float4*>(p + i);
    x[0] = t.x; x[1] = t.y; x[2] = t.z; x[3] = t.w;
  } else {
#pragma unroll
    for (int q = 0; q < 4; ++q) x[q] = p[i + 32 * q];
  }
}

template <bool VEC>
__device__ __forceinline__ void store4(float* p, unsigned i, const float x[4]) {
  if (VEC) {
    *reinterpret_cast<float4*>(p + i) = make_float4(x[0], x[1], x[2], x[3]);
  } else {
#pragma unroll
    for (int q = 0; q < 4; ++q) p[i + 32 * q] = x[q];
  }
}

__device__ __forceinline__ unsigned differ4(const float x[4], const float y[4]) {
  unsigned d = 0u;
#pragma unroll
  for (int q = 0; q < 4; ++q) d |= __float_as_uint(x[q]) ^ __float_as_uint(y[q]);
  return d;
}
__device__ __forceinline__ unsigned any_bits4(const float x[4]) {
  return __float_as_uint(x[0]) | __float_as_uint(x[1]) | __float_as_uint(x[2]) | __float_as_uint(x[3]);
}

// The two 16-bit values of a word.
template <int GT>
__device__ __forceinline__ void two_floats(unsigned w, float& lo, float& hi) {
  if (GT == GS_TYPE_BF16) {
    lo = __uint_as_float(w << 16);
    hi = __uint_as_float(w & 0xFFFF0000u);
  } else {
    const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w));
    lo = t.x;
    hi = t.y;
  }
}

// Four gradients as loaded (16-bit ones two to a register where VEC).
template <int GT, bool VEC>
struct Grad4 {
  uint32_t w[(GT == GS_TYPE_F32 || !VEC) ? 4 : 2];
  __device__ __forceinline__ void load(const void* g, unsigned i) {
    if (GT == GS_TYPE_F32) {
      float x[4];
      load4<VEC>(static_cast<const float*>(g), i, x);
#pragma unroll
      for (int q = 0; q < 4; ++q) w[q] = __float_as_uint(x[q]);
    } else if (VEC) {
      const uint2 t = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(g) + i);
      w[0] = t.x;
      w[1] = t.y;
    } else {
#pragma unroll
      for (int q = 0; q < 4; ++q) w[q] = static_cast<const uint16_t*>(g)[i + 32 * q];
    }
  }
  __device__ __forceinline__ void get(float g[4]) const {
    if (GT == GS_TYPE_F32) {
#pragma unroll
      for (int q = 0; q < 4; ++q) g[q] = __uint_as_float(w[q]);
    } else {
      two_floats<GT>(VEC ? w[0] : w[0] | w[1] << 16, g[0], g[1]);
      two_floats<GT>(VEC ? w[1] : w[2] | w[3] << 16, g[2], g[3]);
    }
  }
};

// Two floats rounded to the 16-bit type, the first in the low half.
__device__ __forceinline__ unsigned round2(int type, float lo, float hi) {
  if (type == GS_TYPE_BF16) {
    const __nv_bfloat162 t = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const unsigned*>(&t);
  }
  const __half2 t = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const unsigned*>(&t);
}

template <bool VEC>
__device__ __forceinline__ void store_copy4(void* p, unsigned i, int type, const float x[4]) {
  const unsigned a = round2(type, x[0], x[1]), b = round2(type, x[2], x[3]);
  uint16_t* c = static_cast<uint16_t*>(p) + i;
  if (VEC) {
    *reinterpret_cast<uint2*>(c) = make_uint2(a, b);
  } else {
    c[0] = (uint16_t)a;
    c[32] = (uint16_t)(a >> 16);
    c[64] = (uint16_t)b;
    c[96] = (uint16_t)(b >> 16);
  }
}

// Place of an element in the rows of an active mask: row and rest. Divisions
// by the width are multiplications with its rounded-up reciprocal, exact
// because the numerator times the reciprocal's excess (below the width, at
// most 2^15) stays below the reciprocal's scale: elements < 2^37 under 2^64,
// and a rest plus a chunk, below 2^16, under 2^32.
struct RowPlace {
  const uint8_t* flags;  // of the row
  unsigned rest;

  static __device__ __forceinline__ unsigned rows(const AdamwDesc& d, unsigned x) {
    return d.width == 1 ? x : __umulhi(x, (unsigned)(d.magic >> 32) + 1u);
  }
  __device__ __forceinline__ void start(const AdamwDesc& d, unsigned long long e) {
    e += d.skip;
    const unsigned long long row = d.width == 1 ? e : __umul64hi(e, d.magic);
    flags = d.active + row;
    rest = (unsigned)(e - row * d.width);
  }
};

// Flags of a lane's four elements from `off` elements on, one bit each.
template <bool VEC>
__device__ __forceinline__ unsigned active4(const AdamwDesc& d, const RowPlace& at, unsigned off) {
  if (VEC && d.width >= 4) {  // at most two rows in four elements
    const unsigned x = at.rest + off;
    const unsigned r = RowPlace::rows(d, x);
    const unsigned left = (r + 1) * d.width - x;  // elements up to the next row
    const unsigned head = left >= 4 ? 15u : (1u << left) - 1u;
    unsigned bits = at.flags[r] != 0 ? head : 0u;
    if (left < 4 && at.flags[r + 1] != 0) bits |= 15u & ~head;
    return bits;
  }
  unsigned bits = 0u;
#pragma unroll
  for (int q = 0; q < 4; ++q)
    bits |= (at.flags[RowPlace::rows(d, at.rest + off + (VEC ? q : 32 * q))] != 0 ? 1u : 0u) << q;
  return bits;
}

// b times the four moments that a word of codes stands for, k = b 2^(F - 127)
// 2^112 or 2^96: with b folded into the scale, the same single rounding of the
// same product as long as the code's value is exact and k a normal float,
// F <= 142 (mu) and 11 <= F <= 158 (nu).
template <bool SIGNED>
__device__ __forceinline__ void decayed4(unsigned w, float k, float x[4]) {
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    unsigned y;
    if (SIGNED) y = (unsigned)((int)__byte_perm(w, 0u, 0x0444 | (q << 12)) >> 4) & 0x87F00000u;
    else y = (q < 3 ? w << (20 - 8 * q) : w >> 4) & 0x0FF00000u;
    x[q] = mul_rn(__uint_as_float(y), k);
  }
}
__device__ __forceinline__ bool foldable(int fm, int fv) {
  return fm <= 142 && (unsigned)(fv - 11) <= 147u;
}
template <bool SIGNED>
__device__ __forceinline__ float folded(int field, float b) {
  return __int_as_float((field + (SIGNED ? 112 : 96)) << 23) * b;
}

// The same for any block, in steps.
template <bool SIGNED>
__device__ __noinline__ float4 decayed4_any(unsigned w, int field, float b) {
  const float up = field == 255 ? NAN : pow2_biased(field);
  float x[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) x[q] = mul_rn(decode8<SIGNED>((w >> (8 * q)) & 255u, up), b);
  return make_float4(x[0], x[1], x[2], x[3]);
}

// encode8 of four values that `scale` takes to their block's format, one code
// a byte, with 16 bits of r as noise: (bits >> 4) + noise has the code in its
// third byte. No code exceeds the largest: F leaves the largest magnitude at
// most at the top code, and noise is less than the next code away.
template <bool SIGNED>
__device__ __forceinline__ unsigned encode4(const float x[4], float scale, const unsigned r[4]) {
  unsigned t[4];
#pragma unroll
  for (int q = 0; q < 4; ++q)
    t[q] = (__float_as_uint((SIGNED ? fabsf(x[q]) : x[q]) * scale) >> 4) + (SIGNED ? r[q] & 0xFFFFu : r[q] >> 16);
  unsigned w = __byte_perm(__byte_perm(t[0], t[1], 0x0062), __byte_perm(t[2], t[3], 0x0062), 0x5410);
  if (SIGNED) {
    const unsigned lo = __byte_perm(__float_as_uint(x[0]), __float_as_uint(x[1]), 0x0073);
    const unsigned hi = __byte_perm(__float_as_uint(x[2]), __float_as_uint(x[3]), 0x0073);
    w |= __byte_perm(lo, hi, 0x5410) & 0x80808080u;
  } else if ((w - 0x01010101u) & ~w & 0x80808080u) {  // a code is 0: not if its value is above
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (x[q] > 0.f && ((w >> (8 * q)) & 255u) == 0u) w |= 1u << (8 * q);
  }
  return w;
}

// Scales of a block's new moments, 2^(127 - F) 2^-112 and 2^-96, powers of two
// as long as those are normal floats; beyond, the values are scaled in two steps.
template <int K>
__device__ __forceinline__ void block_scales(float (&m)[K], float (&v)[K], int fm, int fv, float& sm, float& sv) {
  sm = __int_as_float((142 - fm) << 23);
  sv = __int_as_float((158 - fv) << 23);
  if (fm > 141 || fv > 157) {
    const float dm = pow2_biased(max(254 - fm, 0)), dv = pow2_biased(max(254 - fv, 0));
#pragma unroll
    for (int q = 0; q < K; ++q) {
      m[q] = fm == 255 ? 0.f : m[q] * dm;
      // a v > 0 stays above 0
      v[q] = fv == 255 ? 0.f : (v[q] > 0.f ? fmaxf(v[q] * dv, __int_as_float(1)) : 0.f);
    }
    sm = 0x1p-112f;
    sv = 0x1p-96f;
  }
}

// Whole blocks with 32-bit moments from element `base` by one warp, all loads
// issued before the first use.
template <int GT, bool VEC>
__device__ __forceinline__ void adamw32_chunk(const AdamwDesc& d, long long base, const AdamwParams& a,
                                              const AdamwStep& h, float s) {
  constexpr int U = kAdamwUnroll;
  const int lane = threadIdx.x & 31;
  float p[U][4], m[U][4], v[U][4];
  Grad4<GT, VEC> g[U];
  float* const param = d.param + base;
  float* const mu = static_cast<float*>(d.mu) + base;
  float* const nu = static_cast<float*>(d.nu) + base;
  const unsigned i0 = block_element<VEC>(lane, 0);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const unsigned i = i0 + u * kAdamwBlock;
    load4<VEC>(param, i, p[u]);
    g[u].load(static_cast<const char*>(d.grad) + base * (GT == GS_TYPE_F32 ? 4 : 2), i);
    load4<VEC>(mu, i, m[u]);
    load4<VEC>(nu, i, v[u]);
  }
  unsigned act = 0xFFFFFFFFu;
  if (d.active) {
    RowPlace rows;
    rows.start(d, (unsigned long long)base);
    act = 0u;
#pragma unroll
    for (int u = 0; u < U; ++u) act |= active4<VEC>(d, rows, u * kAdamwBlock + block_element<VEC>(lane, 0)) << (4 * u);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const unsigned i = i0 + u * kAdamwBlock;
    float g1[4], m1[4], v1[4], p1[4];
    g[u].get(g1);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float gq = g1[q] * s;
      m1[q] = add_rn(mul_rn(m[u][q], a.b1), mul_rn(gq, a.omb1));
      v1[q] = add_rn(mul_rn(v[u][q], a.b2), mul_rn(mul_rn(gq, gq), a.omb2));
    }
    adamw_param4(p[u], m1, v1, h, a, p1);
    const unsigned bits = (act >> (4 * u)) & 15u;
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (!((bits >> q) & 1u)) p1[q] = p[u][q];
    if (d.copy) store_copy4<VEC>(static_cast<char*>(d.copy) + base * 2, i, d.copy_type, p1);
    // the parameters of rows that are not active, and moments that were and
    // stay zero (slots that never had a gradient), are not stored again
    if (bits != 0u) store4<VEC>(param, i, p1);
    if (differ4(m1, m[u]) | differ4(v1, v[u]) | ((any_bits4(m[u]) | any_bits4(v[u])) << 1)) {
      store4<VEC>(mu, i, m1);
      store4<VEC>(nu, i, v1);
    }
  }
}

// Up to one block by one warp, `rem` elements of it in range, element by
// element: the ends of tensors, few elements in all, and, with 8-bit moments,
// tensors that are kScalar.
template <int BITS>
struct AdamwBlock {
  long long base;
  int rem;
  float p[4], g[4], m[4], v[4];
  unsigned cm, cv, act;
  int fm, fv;

  __device__ __forceinline__ void load(const AdamwDesc& d, long long from, int in_range) {
    const int lane = threadIdx.x & 31;
    base = from;
    rem = in_range;
    RowPlace rows;
    if (d.active) rows.start(d, (unsigned long long)base);
    cm = cv = act = 0u;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      p[q] = g[q] = m[q] = v[q] = 0.f;
      const int e = lane + 32 * q;
      const long long i = base + e;
      if (e >= rem) continue;
      p[q] = d.param[i];
      g[q] = load_as_float(d.grad, i, d.grad_type);
      if (BITS == 8) {
        cm |= (unsigned)static_cast<const uint8_t*>(d.mu)[i] << (8 * q);
        cv |= (unsigned)static_cast<const uint8_t*>(d.nu)[i] << (8 * q);
      } else {
        m[q] = static_cast<const float*>(d.mu)[i];
        v[q] = static_cast<const float*>(d.nu)[i];
      }
      if (!d.active || rows.flags[RowPlace::rows(d, rows.rest + e)] != 0) act |= 1u << q;
    }
    if (BITS == 8) {
      fm = d.mu_exp[base / kAdamwBlock];
      fv = d.nu_exp[base / kAdamwBlock];
    }
  }

  __device__ __forceinline__ void step(const AdamwDesc& d, const AdamwParams& a, const AdamwStep& h, float s,
                                       unsigned key) {
    const int lane = threadIdx.x & 31;
    const long long blk = base / kAdamwBlock;
    if (BITS == 8) {
      const float4 x = decayed4_any<true>(cm, fm, a.b1), y = decayed4_any<false>(cv, fv, a.b2);
      m[0] = x.x; m[1] = x.y; m[2] = x.z; m[3] = x.w;
      v[0] = y.x; v[1] = y.y; v[2] = y.z; v[3] = y.w;
    }
    float fresh[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const bool in = lane + 32 * q < rem;  // else zeros, which leave no trace in the block
      const float gq = g[q] * s;
      if (BITS == 32) {
        m[q] = mul_rn(m[q], a.b1);
        v[q] = mul_rn(v[q], a.b2);
      }
      m[q] = in ? add_rn(m[q], mul_rn(gq, a.omb1)) : 0.f;
      v[q] = in ? add_rn(v[q], mul_rn(mul_rn(gq, gq), a.omb2)) : 0.f;
    }
    adamw_param4(p, m, v, h, a, fresh);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const long long i = base + lane + 32 * q;
      if (lane + 32 * q >= rem) continue;
      if ((act >> q) & 1u) d.param[i] = p[q] = fresh[q];
      if (d.copy) store_as(d.copy, i, d.copy_type, p[q]);
      if (BITS == 32) {
        static_cast<float*>(d.mu)[i] = m[q];
        static_cast<float*>(d.nu)[i] = v[q];
      }
    }
    if (BITS == 32) return;
    fm = block_field(__reduce_max_sync(0xffffffffu, __float_as_uint(max_abs4(m))));
    fv = block_field(__reduce_max_sync(0xffffffffu, __float_as_uint(max_abs4(v))));
    const unsigned bkey = mix32(key ^ (unsigned)blk);
    unsigned r[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) r[q] = mix32(bkey + kGolden * (unsigned)(lane + 32 * q));
    float sm, sv;
    block_scales(m, v, fm, fv, sm, sv);
    cm = encode4<true>(m, sm, r);
    cv = encode4<false>(v, sv, r);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int e = lane + 32 * q;
      if (e >= rem) continue;
      static_cast<uint8_t*>(d.mu)[base + e] = (uint8_t)(cm >> (8 * q));
      static_cast<uint8_t*>(d.nu)[base + e] = (uint8_t)(cv >> (8 * q));
    }
    if (lane == 0) {
      d.mu_exp[blk] = (uint8_t)fm;
      d.nu_exp[blk] = (uint8_t)fv;
    }
  }
};

// A tile's elements behind its `full` whole chunks, which are the first
// warps', block by block, the warps without a chunk first.
template <int BITS, int WARPS>
__device__ __forceinline__ void adamw_blocks(const AdamwDesc& d, long long tile, int full, const AdamwParams& a,
                                             const AdamwStep& h, float s, unsigned key) {
  static_assert((WARPS & (WARPS - 1)) == 0, "");
  const int end = (int)min(d.count - tile, (long long)kAdamwTile);
  int e = full * (kAdamwTile / WARPS) + (((int)(threadIdx.x >> 5) - full) & (WARPS - 1)) * kAdamwBlock;
#pragma unroll 1
  for (; e < end; e += WARPS * kAdamwBlock) {
    AdamwBlock<BITS> b;
    b.load(d, tile + e, min(end - e, kAdamwBlock));
    b.step(d, a, h, s, key);
  }
}

// What a step takes from the device: count, scale, bias corrections (1 - b^t
// as -expm1(t ln b): no cancellation at small t), read by one thread of the
// CTA. Its ticket is drawn after the read (an acquire) and looked at when the
// CTA's work is done: the CTA with the last ticket knows that every CTA has
// read the count, and advances it. Nothing waits for another CTA.
struct AdamwHead {
  int c;
  float s, inv1, inv2;
  bool go;
};

__device__ __forceinline__ unsigned adamw_head(const AdamwParams& a, AdamwHead& head) {
  unsigned ticket = 0u;
  if (threadIdx.x == 0) {
    int c;
    asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(c) : "l"(a.state) : "memory");
    const float s = a.scale ? *(volatile const float*)a.scale : 1.f;
    if (a.advance) ticket = atomicAdd(reinterpret_cast<unsigned*>(a.state + 1), 1u);
    const float t = (float)c + 1.f;
    head.c = c;
    head.s = s;
    head.go = fabsf(s) <= 3.402823466e38f;
    head.inv1 = 1.f / -expm1f(t * a.ln_b1);
    head.inv2 = 1.f / -expm1f(t * a.ln_b2);
  }
  __syncthreads();
  return ticket;
}

__device__ __forceinline__ void adamw_finish(const AdamwParams& a, const AdamwHead& head, unsigned ticket) {
  if (threadIdx.x == 0 && a.advance && ticket == gridDim.x - 1) {
    if (head.go) a.state[0] = head.c + 1;
    else a.state[2] = a.state[2] + 1;
    a.state[1] = 0;
  }
}

// A CTA's walk over the tiles of a table, every gridDim.x-th.
template <int N>
struct TileWalk {
  const AdamwTable<N>& tab;
  int tile, k;

  __device__ __forceinline__ TileWalk(const AdamwTable<N>& t) : tab(t), tile(blockIdx.x), k(0) {
    if (valid()) k = tensor_of(tab.first, tab.n, tile);
  }
  __device__ __forceinline__ bool valid() const { return tile < tab.first[tab.n]; }
  __device__ __forceinline__ void next() {
    tile += gridDim.x;
    if (valid() && tab.first[k + 1] <= tile) k = tensor_after(tab.first, tab.n, tile, k);
  }
  // first element of the tile in its tensor
  __device__ __forceinline__ long long base() const { return (long long)(tile - tab.first[k]) * kAdamwTile; }
};

// Step values of a tensor.
__device__ __forceinline__ void adamw_rates(AdamwStep& h, const AdamwDesc& d, float cf) {
  const float lr = d.lr_init * expf(cf * d.ln_decay);
  h.rate = lr * h.inv1;
  h.decay = -lr * d.weight_decay;
}

template <int N>
__global__ void __launch_bounds__(32 * kAdamwWarps, GS_ADAMW_CTAS)
k_adamw32(const __grid_constant__ AdamwTable<N> tab, const __grid_constant__ AdamwParams a) {
  GS_PDL_ENTRY_PLAIN();
  __shared__ AdamwHead head;
  const unsigned ticket = adamw_head(a, head);
  if (head.go) {
    const float s = head.s, cf = (float)head.c;
    AdamwStep h;
    h.inv1 = head.inv1;
    h.inv2 = head.inv2;
    int last = -1;
    for (TileWalk<N> w(tab); w.valid(); w.next()) {
      const AdamwDesc& d = tab.t[w.k];
      if (w.k != last) adamw_rates(h, d, cf);
      last = w.k;
      const long long base = w.base() + (threadIdx.x >> 5) * kAdamwChunk;
      if (d.count - base >= kAdamwChunk) {
        switch (d.grad_type * 2 + (d.vec == kVec)) {
          case 0: adamw32_chunk<GS_TYPE_F32, false>(d, base, a, h, s); break;
          case 1: adamw32_chunk<GS_TYPE_F32, true>(d, base, a, h, s); break;
          case 2: adamw32_chunk<GS_TYPE_BF16, false>(d, base, a, h, s); break;
          case 3: adamw32_chunk<GS_TYPE_BF16, true>(d, base, a, h, s); break;
          case 4: adamw32_chunk<GS_TYPE_F16, false>(d, base, a, h, s); break;
          default: adamw32_chunk<GS_TYPE_F16, true>(d, base, a, h, s); break;
        }
      }
      if (d.count - w.base() < kAdamwTile) {
        // what is left of the tensor behind its chunks, at most a block a warp
        adamw_blocks<32, kAdamwWarps>(d, w.base(), (int)(d.count - w.base()) / kAdamwChunk, a, h, s, 0u);
      }
    }
  }
  adamw_finish(a, head, ticket);
}

// Few elements: the time is latency, so every warp has one block, loads its
// data before it knows the step's values, and runs little code.
constexpr int kSmallWarps = 4;
template <int BITS, int N>
__global__ void __launch_bounds__(32 * kSmallWarps)
k_adamw_small(const __grid_constant__ AdamwTable<N> tab, const __grid_constant__ AdamwParams a) {
  GS_PDL_ENTRY_PLAIN();
  __shared__ AdamwHead head;
  const TileWalk<N> w(tab);  // here a tile is kSmallWarps blocks
  const AdamwDesc& d = tab.t[w.k];
  AdamwBlock<BITS> b;
  b.rem = 0;
  if (w.valid()) {
    const long long base = ((long long)(w.tile - tab.first[w.k]) * kSmallWarps + (threadIdx.x >> 5)) * kAdamwBlock;
    if (base < d.count) b.load(d, base, (int)(d.count - base < kAdamwBlock ? d.count - base : kAdamwBlock));
  }
  const unsigned ticket = adamw_head(a, head);
  if (head.go && b.rem > 0) {
    AdamwStep h;
    h.inv1 = head.inv1;
    h.inv2 = head.inv2;
    adamw_rates(h, d, (float)head.c);
    const unsigned key = mix32(a.seed + kGolden * (unsigned)head.c);
    b.step(d, a, h, head.s, mix32(key + kGolden * (unsigned)d.index));
  }
  adamw_finish(a, head, ticket);
}

// 8-bit moments. The step's instructions take the SMs about as long as its
// bytes take the memory (the same step with a block a warp and every test at
// each element: 98 instructions, 765 us at 236M elements, now 62 and 576), so
//  - no warp waits for memory: each copies its next chunk into shared memory
//    (cp.async, 16 bytes a lane) before it works on the current one;
//  - half a warp holds a block, eight elements a lane in two groups of four,
//    so that what is done once a block is done for two blocks at a time;
//  - what differs between tensors (gradient type) and chunks (rows that are
//    not active) is decided once a chunk, not once an element.
constexpr int kChunk8 = 4 * kAdamwBlock;
constexpr int kWarps8 = 4;
static_assert(kChunk8 * kWarps8 == kAdamwTile, "both kernels share the tables' tiles");

struct __align__(16) Adamw8Stage {
  float p[kChunk8];
  unsigned g[kChunk8];
  uint8_t mu[kChunk8], nu[kChunk8];
};

__device__ __forceinline__ void cp_async4(void* dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"((unsigned)__cvta_generic_to_shared(dst)), "l"(src)
               : "memory");
}
__device__ __forceinline__ void cp_async16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((unsigned)__cvta_generic_to_shared(dst)), "l"(src)
               : "memory");
}

// A chunk on its way: what the copies do not carry.
struct Adamw8Chunk {
  long long tile;  // first element of the CTA's tile
  int k;
  int kind;       // copied to shared memory, with no / some / all rows active; or kDirect
  unsigned act;   // flags of the lane's elements, group by group (some)
  unsigned exps;  // exponent byte of mu (lanes 0 .. 3) or nu (4 .. 7) of block lane & 3
};
constexpr int kNone = 0, kSome = 1, kAll = 2, kDirect = 3;

// Place in the chunk of group (j, i) of a lane: block 2 j + lane / 16, then
// elements 64 i + 4 (lane % 16) and on.
__device__ __forceinline__ int group8(int j, int i, int lane) {
  return 256 * j + 128 * (lane >> 4) + 64 * i + 4 * (lane & 15);
}

// Rows of the warp's chunk: none, some or all active, from one flag a lane and row.
__device__ __forceinline__ int chunk_rows(const AdamwDesc& d, const RowPlace& at, int lane) {
  const unsigned rows = RowPlace::rows(d, at.rest + kChunk8 - 1) + 1;
  bool all = true, any = false;
  for (unsigned r = lane; r < rows; r += 32) {
    const bool f = at.flags[r] != 0;
    all &= f;
    any |= f;
  }
  return __all_sync(0xffffffffu, all) ? kAll : (__any_sync(0xffffffffu, any) ? kSome : kNone);
}

template <bool LOOSE>
__device__ __forceinline__ void adamw8_issue(const AdamwDesc& d, Adamw8Chunk& c, Adamw8Stage& st, int lane) {
  const int chunk = (threadIdx.x >> 5) * kChunk8;
  c.kind = kDirect;
  if (d.vec != kScalar && d.count - c.tile >= chunk + kChunk8) {
    const int two = d.grad_type == GS_TYPE_F32 ? 2 : 1;
    if (!LOOSE || d.vec == kVec) {
      const char* g = static_cast<const char*>(d.grad) + (c.tile << two) + (unsigned)((chunk << two) + 16 * lane);
      char* sg = reinterpret_cast<char*>(st.g) + 16 * lane;
      cp_async16(sg, g);
      cp_async16(sg + 512, g + 512);
      if (two == 2) {
        cp_async16(sg + 1024, g + 1024);
        cp_async16(sg + 1536, g + 1536);
      }
    } else {
      const float* g = static_cast<const float*>(d.grad) + c.tile + (unsigned)(chunk + lane);
#pragma unroll
      for (int n = 0; n < kChunk8 / 32; ++n) cp_async4(st.g + lane + 32 * n, g + 32 * n);
    }
    cp_async16(st.mu + 16 * lane, static_cast<const uint8_t*>(d.mu) + c.tile + (unsigned)(chunk + 16 * lane));
    cp_async16(st.nu + 16 * lane, static_cast<const uint8_t*>(d.nu) + c.tile + (unsigned)(chunk + 16 * lane));
    if (lane < 8)
      c.exps = ((lane < 4 ? d.mu_exp : d.nu_exp) + c.tile / kAdamwBlock)[(unsigned)(chunk / kAdamwBlock + (lane & 3))];
    c.kind = kAll;
    if (d.active) {
      RowPlace rows;
      rows.start(d, (unsigned long long)(c.tile + chunk));
      c.kind = chunk_rows(d, rows, lane);
      if (c.kind == kSome) {
        c.act = 0u;
#pragma unroll
        for (int n = 0; n < 4; ++n) c.act |= active4<true>(d, rows, group8(n >> 1, n & 1, lane)) << (4 * n);
      }
    }
    if (c.kind != kNone || d.copy) {
      const float* p = d.param + c.tile + (unsigned)chunk;
      if (!LOOSE || d.vec == kVec) {
#pragma unroll
        for (int n = 0; n < 4; ++n) cp_async16(st.p + 4 * lane + 128 * n, p + 4 * lane + 128 * n);
      } else {
#pragma unroll
        for (int n = 0; n < kChunk8 / 32; ++n) cp_async4(st.p + lane + 32 * n, p + lane + 32 * n);
      }
    }
  }
  asm volatile("cp.async.commit_group;" ::: "memory");
}

template <int GT>
__device__ __forceinline__ void grads4(const unsigned* st, int e, float g[4]) {
  if (GT == GS_TYPE_F32) {
    load4<true>(reinterpret_cast<const float*>(st), e, g);
  } else {
    const uint2 w = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(st) + e);
    two_floats<GT>(w.x, g[0], g[1]);
    two_floats<GT>(w.y, g[2], g[3]);
  }
}

// Largest of a half warp's exponent bytes, two 16-bit values at a time.
__device__ __forceinline__ unsigned half_max2(unsigned x) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) x = __vmaxu2(x, __shfl_xor_sync(0xffffffffu, x, o));
  return x;
}

// Blocks 2 j and 2 j + 1 of a chunk. ALL: every row active; COPY: a copy is
// written; LOOSE: the parameter is not 16-byte aligned.
template <int GT, bool ALL, bool COPY, bool LOOSE>
__device__ __forceinline__ void adamw8_blocks(const AdamwDesc& d, const Adamw8Chunk& c, Adamw8Stage& st, int j,
                                              unsigned& exps, const AdamwParams& a, const AdamwStep& h, float s,
                                              unsigned key, int lane) {
  const int src = 2 * j + (lane >> 4);  // the half's block
  int fm = (int)__shfl_sync(0xffffffffu, c.exps, src), fv = (int)__shfl_sync(0xffffffffu, c.exps, 4 + src);
  float m[8], v[8];
  {
    const unsigned w[4] = {*reinterpret_cast<const unsigned*>(st.mu + group8(j, 0, lane)),
                           *reinterpret_cast<const unsigned*>(st.mu + group8(j, 1, lane)),
                           *reinterpret_cast<const unsigned*>(st.nu + group8(j, 0, lane)),
                           *reinterpret_cast<const unsigned*>(st.nu + group8(j, 1, lane))};
    if (foldable(fm, fv)) {
      const float km = folded<true>(fm, a.b1), kv = folded<false>(fv, a.b2);
      decayed4<true>(w[0], km, m);
      decayed4<true>(w[1], km, m + 4);
      decayed4<false>(w[2], kv, v);
      decayed4<false>(w[3], kv, v + 4);
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float4 x = decayed4_any<true>(w[i], fm, a.b1), y = decayed4_any<false>(w[2 + i], fv, a.b2);
        m[4 * i] = x.x; m[4 * i + 1] = x.y; m[4 * i + 2] = x.z; m[4 * i + 3] = x.w;
        v[4 * i] = y.x; v[4 * i + 1] = y.y; v[4 * i + 2] = y.z; v[4 * i + 3] = y.w;
      }
    }
  }
  const unsigned chunk = (threadIdx.x >> 5) * kChunk8;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int e = group8(j, i, lane);
    float g[4], p[4], fresh[4];
    grads4<GT>(st.g, e, g);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float gq = g[q] * s;
      m[4 * i + q] = add_rn(m[4 * i + q], mul_rn(gq, a.omb1));
      v[4 * i + q] = add_rn(v[4 * i + q], mul_rn(mul_rn(gq, gq), a.omb2));
    }
    if (ALL || COPY || c.kind != kNone) {
      load4<true>(st.p, e, p);
      adamw_param4_fast(p, m + 4 * i, v + 4 * i, h, a, fresh);
      if (!ALL) {
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (c.kind == kNone || !((c.act >> (8 * j + 4 * i + q)) & 1u)) fresh[q] = p[q];
      }
      if (ALL || c.kind != kNone) {
        if (LOOSE) store4<true>(st.p, e, fresh);  // stored from there when the chunk is done
        else store4<true>(d.param + c.tile, chunk + e, fresh);
      }
      if (COPY)
        store_copy4<true>(static_cast<char*>(d.copy) + c.tile * 2, chunk + e, d.copy_type, fresh);
    }
  }
  const unsigned top = half_max2((unsigned)block_field(__float_as_uint(max_abs8(m))) |
                                 (unsigned)block_field(__float_as_uint(max_abs8(v))) << 16);
  fm = (int)(top & 0xFFFFu);
  fv = (int)(top >> 16);
  float sm, sv;
  block_scales(m, v, fm, fv, sm, sv);
  const unsigned bkey = mix32(key ^ ((unsigned)(c.tile / kAdamwBlock) + chunk / kAdamwBlock + (unsigned)src)) +
                        kGolden * (unsigned)(4 * (lane & 15));
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    unsigned r[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) r[q] = mix32(bkey + kGolden * (unsigned)(64 * i + q));
    const unsigned at = chunk + (unsigned)group8(j, i, lane);
    *reinterpret_cast<unsigned*>(static_cast<uint8_t*>(d.mu) + c.tile + at) = encode4<true>(m + 4 * i, sm, r);
    *reinterpret_cast<unsigned*>(static_cast<uint8_t*>(d.nu) + c.tile + at) = encode4<false>(v + 4 * i, sv, r);
  }
  // lane b collects the byte of mu of block b, lane 4 + b that of nu
  const unsigned both = __shfl_sync(0xffffffffu, top, (lane & 1) << 4);
  if ((lane & 3) >> 1 == j) exps = lane < 4 ? both & 0xFFFFu : both >> 16;
}

template <int GT, bool ALL, bool COPY, bool LOOSE>
__device__ __forceinline__ void adamw8_chunk(const AdamwDesc& d, const Adamw8Chunk& c, Adamw8Stage& st,
                                             const AdamwParams& a, const AdamwStep& h, float s, unsigned key, int lane) {
  unsigned exps = 0u;
  if (!ALL && !COPY && c.kind == kNone) {
    // moments and gradients all zero in rows that are not active: nothing
    // changes but for the sign of a zero. (An exponent byte of 0 alone may be
    // a block of subnormals.)
    unsigned any = lane < 8 ? c.exps : 0u;
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const int e = group8(n >> 1, n & 1, lane);
      any |= (*reinterpret_cast<const unsigned*>(st.mu + e) & 0x7F7F7F7Fu) |
             *reinterpret_cast<const unsigned*>(st.nu + e);
      float g[4];
      grads4<GT>(st.g, e, g);
#pragma unroll
      for (int q = 0; q < 4; ++q) any |= __float_as_uint(g[q]) << 1;
    }
    if (__all_sync(0xffffffffu, any == 0u)) return;
  }
#pragma unroll 1
  for (int j = 0; j < 2; ++j) adamw8_blocks<GT, ALL, COPY, LOOSE>(d, c, st, j, exps, a, h, s, key, lane);
  if (lane < 8)
    ((lane < 4 ? d.mu_exp : d.nu_exp) + c.tile / kAdamwBlock)[(threadIdx.x >> 5) * 4 + (lane & 3)] = (uint8_t)exps;
  if (LOOSE && (ALL || c.kind != kNone)) {
    __syncwarp();
    float* const param = d.param + c.tile + (threadIdx.x >> 5) * kChunk8 + lane;
#pragma unroll
    for (int n = 0; n < kChunk8 / 32; ++n) param[32 * n] = st.p[lane + 32 * n];
  }
}

template <int GT, bool LOOSE>
__device__ __forceinline__ void adamw8_typed(const AdamwDesc& d, const Adamw8Chunk& c, Adamw8Stage& st,
                                             const AdamwParams& a, const AdamwStep& h, float s, unsigned key, int lane) {
  if (c.kind == kAll) {
    if (d.copy) adamw8_chunk<GT, true, true, LOOSE>(d, c, st, a, h, s, key, lane);
    else adamw8_chunk<GT, true, false, LOOSE>(d, c, st, a, h, s, key, lane);
  } else {
    if (d.copy) adamw8_chunk<GT, false, true, LOOSE>(d, c, st, a, h, s, key, lane);
    else adamw8_chunk<GT, false, false, LOOSE>(d, c, st, a, h, s, key, lane);
  }
}

// LOOSE: tensors with kLoose are among the table's (a kernel of its own: the
// code for them costs the others 3 %).
template <int N, bool LOOSE>
__global__ void __launch_bounds__(32 * kWarps8, GS_ADAMW8_CTAS)
k_adamw8(const __grid_constant__ AdamwTable<N> tab, const __grid_constant__ AdamwParams a) {
  GS_PDL_ENTRY_PLAIN();
  __shared__ Adamw8Stage stages[kWarps8][2];
  __shared__ AdamwHead head;
  const int lane = threadIdx.x & 31;
  TileWalk<N> w(tab);
  Adamw8Chunk now = {}, next = {};
  Adamw8Stage* st = stages[threadIdx.x >> 5];
  bool more = w.valid();
  if (more) {
    now.k = w.k;
    now.tile = w.base();
    adamw8_issue<LOOSE>(tab.t[now.k], now, st[0], lane);
  }
  const unsigned ticket = adamw_head(a, head);
  if (head.go) {
    const float s = head.s;
    AdamwStep h;
    h.inv1 = head.inv1;
    h.inv2 = head.inv2;
    unsigned tkey = 0u;
    int at = 0, last = -1;
    while (more) {
      w.next();
      more = w.valid();
      if (more) {
        next.k = w.k;
        next.tile = w.base();
        adamw8_issue<LOOSE>(tab.t[next.k], next, st[at ^ 1], lane);
        asm volatile("cp.async.wait_group 1;" ::: "memory");
      } else {
        asm volatile("cp.async.wait_group 0;" ::: "memory");
      }
      __syncwarp();
      const AdamwDesc& d = tab.t[now.k];
      if (now.k != last) {
        adamw_rates(h, d, (float)head.c);
        tkey = mix32(mix32(a.seed + kGolden * (unsigned)head.c) + kGolden * (unsigned)d.index);
        last = now.k;
      }
      if (now.kind != kDirect) {
        if (LOOSE && d.vec == kLoose) adamw8_typed<GS_TYPE_F32, true>(d, now, st[at], a, h, s, tkey, lane);
        else if (d.grad_type == GS_TYPE_F32) adamw8_typed<GS_TYPE_F32, false>(d, now, st[at], a, h, s, tkey, lane);
        else if (d.grad_type == GS_TYPE_BF16) adamw8_typed<GS_TYPE_BF16, false>(d, now, st[at], a, h, s, tkey, lane);
        else adamw8_typed<GS_TYPE_F16, false>(d, now, st[at], a, h, s, tkey, lane);
      }
      if (d.vec == kScalar) {
        adamw_blocks<8, kWarps8>(d, now.tile, 0, a, h, s, tkey);
      } else if (d.count - now.tile < kAdamwTile) {
        // what is left of the tensor behind its chunks, at most a block a warp
        adamw_blocks<8, kWarps8>(d, now.tile, (int)(d.count - now.tile) / kChunk8, a, h, s, tkey);
      }
      __syncwarp();  // the stage has been read before it is copied into again
      now = next;
      at ^= 1;
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");  // of a step that is skipped
  adamw_finish(a, head, ticket);
}

// With 32-bit moments, how many elements all arrays of a tensor lie behind a
// 16-byte boundary (8 bytes for 16-bit values); -1 where they differ.
static int elements_behind(const GsAdamwTensor& t) {
  const uintptr_t p = (uintptr_t)t.param, g = (uintptr_t)t.grad, m = (uintptr_t)t.mu, v = (uintptr_t)t.nu,
                  c = (uintptr_t)t.copy;
  const uintptr_t behind = p / 4 & 3;
  const bool same = (m / 4 & 3) == behind && (v / 4 & 3) == behind &&
                    ((t.grad_type == GS_TYPE_F32 ? g / 4 : g / 2) & 3) == behind &&
                    (!t.copy || (c / 2 & 3) == behind);
  return same ? (int)behind : -1;
}

// Entries of a tensor in the table: one, or two with 32-bit moments where all
// arrays lie the same 1 to 3 elements behind a boundary (the groups of a flat
// buffer of odd capacity): the elements up to the next boundary, and the rest,
// which is accessed four elements at a time (333331 slots: 67 us element by
// element, 63 us so).
static int entries_of(const GsAdamwTensor& t, int bits) {
  const int behind = bits == 32 ? elements_behind(t) : 0;
  return behind > 0 && t.count > 4 - behind ? 2 : 1;
}

static int describe(const GsAdamwTensor& t, int index, int bits, AdamwDesc out[2]) {
  AdamwDesc d;
  d.param = t.param;
  d.grad = t.grad;
  d.mu = t.mu;
  d.nu = t.nu;
  d.mu_exp = t.mu_exp;
  d.nu_exp = t.nu_exp;
  d.copy = t.copy;
  d.active = t.active;
  d.count = t.count;
  d.lr_init = t.lr_init;
  d.ln_decay = t.decay_rate == 1.f ? 0.f : (float)(std::log((double)t.decay_rate) / (double)t.transition_steps);
  d.weight_decay = t.weight_decay;
  d.width = (unsigned)t.width;
  d.magic = t.width > 1 ? ~0ull / (unsigned)t.width + 1ull : 0ull;
  d.grad_type = (uint8_t)t.grad_type;
  d.copy_type = (uint8_t)t.copy_type;
  d.skip = 0;
  d.index = index;
  const bool f32 = t.grad_type == GS_TYPE_F32;
  d.vec = kScalar;
  if (bits == 8) {
    const uintptr_t pg = (uintptr_t)t.param | (uintptr_t)t.grad;
    if ((((uintptr_t)t.mu | (uintptr_t)t.nu) & 15) == 0 && ((uintptr_t)t.copy & 7) == 0)
      d.vec = (pg & 15) == 0 ? kVec : (f32 ? kLoose : kScalar);
    out[0] = d;
    return 1;
  }
  const int behind = elements_behind(t);
  if (behind == 0) d.vec = kVec;
  out[0] = d;
  if (entries_of(t, bits) == 1) return 1;
  const int64_t head = 4 - behind;
  out[0].count = head;
  d.param += head;
  d.grad = static_cast<const char*>(d.grad) + head * (f32 ? 4 : 2);
  d.mu = static_cast<float*>(d.mu) + head;
  d.nu = static_cast<float*>(d.nu) + head;
  if (d.copy) d.copy = static_cast<char*>(d.copy) + head * 2;
  d.count -= head;
  d.skip = (uint8_t)head;
  d.vec = kVec;
  out[1] = d;
  return 2;
}

// Tensors t[0 .. n), the caller's index0-th and on, in at most N entries.
template <int BITS, int N>
static void launch_adamw_class(const GsAdamwTensor* t, int n, int index0, const AdamwParams& a, cudaStream_t st) {
  static thread_local AdamwTable<N> tab;
  long long blocks = 0;
  for (int i = 0; i < n; ++i) blocks += (t[i].count + kAdamwBlock - 1) / kAdamwBlock;
  const bool small = blocks <= (long long)device_sms() * (BITS == 8 ? GS_ADAMW8_SMALL : GS_ADAMW_SMALL);
  const int tile = small ? kSmallWarps * kAdamwBlock : kAdamwTile;
  int tiles = 0, entries = 0;
  bool loose = false;
  for (int i = 0; i < n; ++i) {
    AdamwDesc d[2];
    const int k = describe(t[i], index0 + i, BITS, d);
    if (small && k == 2) d[0].count = t[i].count;  // element by element all the same
    for (int j = 0; j < (small ? 1 : k); ++j) {
      tab.t[entries] = d[j];
      loose |= d[j].vec == kLoose;
      tab.first[entries++] = tiles;
      tiles += (int)((d[j].count + tile - 1) / tile);
    }
  }
  tab.first[entries] = tiles;
  tab.n = entries;
  GS_TIMED(BITS == 8 ? "adamw8" : "adamw", st);
  if (small) {
    launch_kernel_plain(k_adamw_small<BITS, N>, std::max(1, tiles), 32 * kSmallWarps, 0, st, tab, a);
  } else if (BITS == 8) {
    launch_kernel_plain(loose ? k_adamw8<N, true> : k_adamw8<N, false>, std::min(tiles, device_sms() * GS_ADAMW8_CTAS),
                        32 * kWarps8, 0, st, tab, a);
  } else {
    launch_kernel_plain(k_adamw32<N>, std::min(tiles, device_sms() * 8), 32 * kAdamwWarps, 0, st, tab, a);
  }
}

constexpr int kAdamwSmall = 12, kAdamwMost = 256;  // entries of a table

template <int BITS>
static void launch_adamw_bits(const GsAdamwTensor* tensors, int n, AdamwParams& a, cudaStream_t st) {
  int at = 0;
  do {
    // as many tensors as have entries
    int entries = 0, take = 0;
    for (; at + take < n; ++take) {
      const int k = entries_of(tensors[at + take], BITS);
      if (entries + k > kAdamwMost) break;
      entries += k;
    }
    a.advance = at + take >= n;
    if (entries <= kAdamwSmall) launch_adamw_class<BITS, kAdamwSmall>(tensors + at, take, at, a, st);
    else launch_adamw_class<BITS, kAdamwMost>(tensors + at, take, at, a, st);
    at += take;
  } while (at < n);
}

void launch_adamw(const GsAdamwTensor* tensors, int n, const GsAdamwConfig& cfg, const float* scale, int* state,
                  cudaStream_t st) {
  AdamwParams a;
  a.b1 = (float)cfg.b1;
  a.b2 = (float)cfg.b2;
  a.omb1 = (float)(1.0 - cfg.b1);
  a.omb2 = (float)(1.0 - cfg.b2);
  a.eps = (float)cfg.eps;
  a.ln_b1 = (float)std::log(cfg.b1);
  a.ln_b2 = (float)std::log(cfg.b2);
  a.seed = cfg.seed;
  a.fine_root = a.eps < 0x1p-39f;
  a.scale = scale;
  a.state = state;
  if (cfg.moment_bits == 8) launch_adamw_bits<8>(tensors, n, a, st);
  else launch_adamw_bits<32>(tensors, n, a, st);
}

// ---------------------------------------------------------------------------
// Global gradient norm: u sqrt(sum of squares) over every tensor, and the
// factor that clips it. The squares are summed in fp64: no gradient of fp32
// range overflows or underflows, and the sum is not finite exactly when a
// gradient is not. Fixed order: per-thread sums over a fixed grid, per-CTA
// partials, summed by the last CTA (atomic ticket, no waiting).
struct GradDesc {
  const void* grad;
  long long count;
  int type;
};

template <int N>
struct GradTable {
  GradDesc t[N];
  int first[N + 1];
  int n;
};

// A tile is 8 KB of a tensor counted from the 16-byte boundary at or before
// its first element, 32 bytes a thread in 16-byte loads; only the vectors
// that hold both the tensor's elements and others are read one by one.
constexpr int kNormSmall = 8, kNormMost = 1024, kNormGrid = 1184;  // 8 CTAs an SM
constexpr int kNormVecs = GS_NORM_VECS;
constexpr int kNormTileBytes = 256 * 16 * kNormVecs;

__host__ __device__ __forceinline__ long long norm_tiles(const void* grad, long long count, int type) {
  const long long bytes = (long long)((uintptr_t)grad & 15) + count * (type == GS_TYPE_F32 ? 4 : 2);
  return count > 0 ? (bytes + kNormTileBytes - 1) / kNormTileBytes : 0;
}

template <int GT>
__device__ __forceinline__ void norm_add(const uint4& w, double acc[4]) {
  const unsigned b[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    if (GT == GS_TYPE_F32) {
      const double x = (double)__uint_as_float(b[q]);
      acc[q] = fma(x, x, acc[q]);
    } else {
      float lo, hi;
      two_floats<GT>(b[q], lo, hi);
      const double x = (double)lo, y = (double)hi;
      acc[q] = fma(x, x, acc[q]);
      acc[q] = fma(y, y, acc[q]);
    }
  }
}

template <int GT>
__device__ __forceinline__ void norm_tile(const GradDesc& d, long long tile, double acc[4]) {
  constexpr int PER = GT == GS_TYPE_F32 ? 4 : 8;  // elements of a vector
  const unsigned shift = (unsigned)((uintptr_t)d.grad & 15) / (16 / PER);
  const long long v0 = tile * (256 * kNormVecs);  // the tile's first vector; its first element is v0 PER - shift
  const uint4* vecs = reinterpret_cast<const uint4*>((uintptr_t)d.grad & ~(uintptr_t)15) + v0;
  if (v0 * PER >= shift && (v0 + 256 * kNormVecs) * PER - shift <= d.count) {  // all of it in the tensor
    uint4 w[kNormVecs];
#pragma unroll
    for (int j = 0; j < kNormVecs; ++j) w[j] = __ldg(vecs + threadIdx.x + 256 * j);
#pragma unroll
    for (int j = 0; j < kNormVecs; ++j) norm_add<GT>(w[j], acc);
    return;
  }
  for (int j = 0; j < kNormVecs; ++j) {
    const unsigned k = threadIdx.x + 256 * j;
    const long long e = (v0 + k) * PER - shift;
    if (e >= 0 && e + PER <= d.count) {
      norm_add<GT>(__ldg(vecs + k), acc);
    } else if (e + PER > 0 && e < d.count) {
      for (int q = 0; q < PER; ++q)
        if (e + q >= 0 && e + q < d.count) {
          const double x = (double)load_as_float(d.grad, e + q, GT);
          acc[0] = fma(x, x, acc[0]);
        }
    }
  }
}

template <int N>
__global__ void __launch_bounds__(256, GS_NORM_CTAS)
k_grad_norm(const __grid_constant__ GradTable<N> tab, double* __restrict__ partials, int part0, int parts,
            float max_norm, const float* __restrict__ unscale, GsGradNorm* __restrict__ out) {
  GS_PDL_ENTRY_PLAIN();
  __shared__ double s_red[8];
  __shared__ bool s_last;
  double sums[4] = {0.0, 0.0, 0.0, 0.0};
  const int tiles = tab.first[tab.n];
  // Many tensors: consecutive tiles, so that a CTA reads few entries of the
  // table (each new one is a miss of the constant cache: 197 tensors of 100 MB
  // took 39 us in strides and 28 us so). Few: strides, which end more evenly.
  constexpr bool kRange = N > kNormSmall;
  const int t0 = kRange ? (int)((long long)tiles * blockIdx.x / gridDim.x) : (int)blockIdx.x;
  const int t1 = kRange ? (int)((long long)tiles * (blockIdx.x + 1) / gridDim.x) : tiles;
  const int step = kRange ? 1 : (int)gridDim.x;
  int k = t0 < t1 ? tensor_of(tab.first, tab.n, t0) : 0;
  for (int tile = t0; tile < t1; tile += step) {
    if (tab.first[k + 1] <= tile) k = tensor_after(tab.first, tab.n, tile, k);
    const GradDesc& d = tab.t[k];
    const long long t = tile - tab.first[k];
    if (d.type == GS_TYPE_F32) norm_tile<GS_TYPE_F32>(d, t, sums);
    else if (d.type == GS_TYPE_BF16) norm_tile<GS_TYPE_BF16>(d, t, sums);
    else norm_tile<GS_TYPE_F16>(d, t, sums);
  }
  double acc = (sums[0] + sums[1]) + (sums[2] + sums[3]);
  acc = block_sum_d256(acc, s_red);
  if (threadIdx.x == 0) {
    partials[part0 + blockIdx.x] = acc;
    __threadfence();
    const unsigned t = atomicAdd(&out->ticket, 1u);
    s_last = t == (unsigned)(parts - 1);
  }
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  double sum = 0.0;
  for (int b = threadIdx.x; b < parts; b += 256) sum += ((volatile double*)partials)[b];
  __syncthreads();
  sum = block_sum_d256(sum, s_red);
  if (threadIdx.x == 0) {
    const double norm = sqrt(sum) * (unscale ? (double)*unscale : 1.0);
    const float nf = (float)norm;
    const bool finite = fabsf(nf) <= 3.402823466e38f;
    double scale = norm < (double)max_norm ? 1.0 : (double)max_norm / norm;
    if (unscale) scale *= (double)*unscale;
    out->norm = nf;
    out->scale = finite ? (float)scale : NAN;
    out->ticket = 0u;
  }
}

template <int N>
static int fill_grad_table(const GsGradTensor* t, int n, GradTable<N>& tab) {
  int tiles = 0;
  for (int i = 0; i < n; ++i) {
    tab.t[i].grad = t[i].grad;
    tab.t[i].count = t[i].count;
    tab.t[i].type = t[i].type;
    tab.first[i] = tiles;
    tiles += (int)norm_tiles(t[i].grad, t[i].count, t[i].type);
  }
  tab.first[n] = tiles;
  tab.n = n;
  return tiles;
}

size_t grad_norm_workspace_bytes(int n) {
  const size_t launches = n > 0 ? ((size_t)n + kNormMost - 1) / kNormMost : 1;
  return launches * kNormGrid * sizeof(double);
}

static int norm_grid(const GsGradTensor* t, int n) {
  long long tiles = 0;
  for (int i = 0; i < n; ++i) tiles += norm_tiles(t[i].grad, t[i].count, t[i].type);
  return (int)std::max(1ll, std::min(tiles, (long long)kNormGrid));
}

template <int N>
static void launch_norm_class(const GsGradTensor* t, int n, double* partials, int part0, int parts, float max_norm,
                              const float* unscale, GsGradNorm* out, cudaStream_t st) {
  static thread_local GradTable<N> tab;
  fill_grad_table(t, n, tab);
  GS_TIMED("grad_norm", st);
  launch_kernel_plain(k_grad_norm<N>, norm_grid(t, n), 256, 0, st, tab, partials, part0, parts, max_norm, unscale,
                      out);
}

void launch_grad_norm(const GsGradTensor* tensors, int n, float max_norm, const float* unscale, GsGradNorm* out,
                      void* ws, cudaStream_t st) {
  int parts = 0;
  for (int at = 0; at == 0 || at < n; at += kNormMost) parts += norm_grid(tensors + at, std::min(n - at, kNormMost));
  int part0 = 0;
  for (int at = 0; at == 0 || at < n; at += kNormMost) {
    const int take = std::min(n - at, kNormMost);
    double* partials = static_cast<double*>(ws);
    if (take <= kNormSmall)
      launch_norm_class<kNormSmall>(tensors + at, take, partials, part0, parts, max_norm, unscale, out, st);
    else
      launch_norm_class<kNormMost>(tensors + at, take, partials, part0, parts, max_norm, unscale, out, st);
    part0 += norm_grid(tensors + at, take);
  }
}

// ---------------------------------------------------------------------------
// 8-bit moments to and from values. Encoding rounds to nearest (halves up):
// the values of a block's codes are kept exactly. Decoding 236M elements to
// bf16: 245 us (6 B an element: 5.8 TB/s); encoding them from fp32: 521 us
// (10 B: 4.5 TB/s, a byte a lane).
__device__ __forceinline__ void store_value(float* p, float x) { *p = x; }
__device__ __forceinline__ void store_value(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }

__device__ __forceinline__ void store_values8(float* p, const float x[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
}
__device__ __forceinline__ void store_values8(__nv_bfloat16* p, const float x[8]) {
  unsigned w[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(x[2 * q], x[2 * q + 1]);
    w[q] = *reinterpret_cast<const unsigned*>(&a);
  }
  *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}

template <bool SIGNED>
__device__ __forceinline__ void values4(unsigned w, int field, float x[4]) {
  if (SIGNED ? field <= 142 : (unsigned)(field - 11) <= 147u) {
    decayed4<SIGNED>(w, folded<SIGNED>(field, 1.f), x);
  } else {
    const float4 y = decayed4_any<SIGNED>(w, field, 1.f);
    x[0] = y.x; x[1] = y.y; x[2] = y.z; x[3] = y.w;
  }
}

// VEC: eight codes of each moment a thread, U times in flight; else one.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256)
k_moments8_decode(const uint8_t* __restrict__ mu, const uint8_t* __restrict__ nu, const uint8_t* __restrict__ mu_exp,
                  const uint8_t* __restrict__ nu_exp, long long count, T* __restrict__ mu_out,
                  T* __restrict__ nu_out) {
  GS_PDL_ENTRY_PLAIN();
  const long long stride = (long long)gridDim.x * 256;
  long long i = blockIdx.x * 256ll + threadIdx.x;
  if (VEC) {
    constexpr int U = GS_DECODE_UNROLL;
    const long long n8 = count / 8;
    for (; i < n8; i += U * stride) {
      uint2 wm[U], wv[U];
      int fm[U], fv[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const long long k = i + u * stride;
        if (k < n8) {
          wm[u] = reinterpret_cast<const uint2*>(mu)[k];
          wv[u] = reinterpret_cast<const uint2*>(nu)[k];
          fm[u] = mu_exp[k / (kAdamwBlock / 8)];
          fv[u] = nu_exp[k / (kAdamwBlock / 8)];
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const long long k = i + u * stride;
        if (k < n8) {
          float x[8];
          values4<true>(wm[u].x, fm[u], x);
          values4<true>(wm[u].y, fm[u], x + 4);
          store_values8(mu_out + 8 * k, x);
          values4<false>(wv[u].x, fv[u], x);
          values4<false>(wv[u].y, fv[u], x + 4);
          store_values8(nu_out + 8 * k, x);
        }
      }
    }
    i = 8 * n8 + blockIdx.x * 256ll + threadIdx.x;  // the last few
  }
  for (; i < count; i += stride) {
    const int fm = mu_exp[i / kAdamwBlock], fv = nu_exp[i / kAdamwBlock];
    const float m = decode8<true>(mu[i], pow2_biased(min(fm, 254)));
    const float v = decode8<false>(nu[i], pow2_biased(min(fv, 254)));
    store_value(mu_out + i, fm == 255 ? NAN : m);
    store_value(nu_out + i, fv == 255 ? NAN : v);
  }
}

__global__ void __launch_bounds__(256)
k_moments8_encode(const float* __restrict__ mu, const float* __restrict__ nu, long long count,
                  uint8_t* __restrict__ mu8, uint8_t* __restrict__ nu8, uint8_t* __restrict__ mu_exp,
                  uint8_t* __restrict__ nu_exp) {
  GS_PDL_ENTRY_PLAIN();
  const int lane = threadIdx.x & 31;
  const long long blocks = (count + kAdamwBlock - 1) / kAdamwBlock;
  for (long long blk = blockIdx.x * 8ll + (threadIdx.x >> 5); blk < blocks; blk += (long long)gridDim.x * 8) {
    float m[4], v[4];
    unsigned top_m = 0u, top_v = 0u;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const long long i = blk * kAdamwBlock + lane + 32 * q;
      m[q] = i < count ? mu[i] : 0.f;
      v[q] = i < count ? nu[i] : 0.f;
      top_m = max(top_m, __float_as_uint(fabsf(m[q])));
      top_v = max(top_v, __float_as_uint(fabsf(v[q])));
    }
    const int fm = block_field(__reduce_max_sync(0xffffffffu, top_m));
    const int fv = block_field(__reduce_max_sync(0xffffffffu, top_v));
    const float down_m = pow2_biased(max(254 - fm, 0)), down_v = pow2_biased(max(254 - fv, 0));
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const long long i = blk * kAdamwBlock + lane + 32 * q;
      if (i >= count) continue;
      mu8[i] = (uint8_t)(fm == 255 ? 0u : encode8<true>(m[q], down_m, 1u << 19));
      nu8[i] = (uint8_t)(fv == 255 ? 0u : encode8<false>(v[q], down_v, 1u << 19));
    }
    if (lane == 0) {
      mu_exp[blk] = (uint8_t)fm;
      nu_exp[blk] = (uint8_t)fv;
    }
  }
}

void launch_moments8_decode(const uint8_t* mu, const uint8_t* nu, const uint8_t* mu_exp, const uint8_t* nu_exp,
                            long long count, int type, void* mu_out, void* nu_out, cudaStream_t st) {
  const bool vec = (((uintptr_t)mu_out | (uintptr_t)nu_out) & 15) == 0 && (((uintptr_t)mu | (uintptr_t)nu) & 7) == 0;
  const long long items = vec ? count / 8 + 7 : count;
  const int grid = (int)std::min((items + 255) / 256, (long long)device_sms() * 8);
  GS_TIMED("moments8_decode", st);
  auto launch = [&](auto kernel, auto* m, auto* v) {
    launch_kernel_plain(kernel, grid, 256, 0, st, mu, nu, mu_exp, nu_exp, count, m, v);
  };
  if (type == GS_TYPE_F32) {
    float *m = static_cast<float*>(mu_out), *v = static_cast<float*>(nu_out);
    if (vec) launch(k_moments8_decode<float, true>, m, v);
    else launch(k_moments8_decode<float, false>, m, v);
  } else {
    __nv_bfloat16 *m = static_cast<__nv_bfloat16*>(mu_out), *v = static_cast<__nv_bfloat16*>(nu_out);
    if (vec) launch(k_moments8_decode<__nv_bfloat16, true>, m, v);
    else launch(k_moments8_decode<__nv_bfloat16, false>, m, v);
  }
}

void launch_moments8_encode(const float* mu, const float* nu, long long count, uint8_t* mu8, uint8_t* nu8,
                            uint8_t* mu_exp, uint8_t* nu_exp, cudaStream_t st) {
  const long long blocks = (count + kAdamwBlock - 1) / kAdamwBlock;
  const int grid = (int)std::min((blocks + 7) / 8, (long long)device_sms() * 8);
  GS_TIMED("moments8_encode", st);
  launch_kernel_plain(k_moments8_encode, grid, 256, 0, st, mu, nu, count, mu8, nu8, mu_exp, nu_exp);
}

// Rows of the five groups that move to other slots (density control), one
// moment. A row's new block has another exponent, so a block that receives
// rows is encoded again as a whole, to nearest; the others are not touched.
// Values are read from a copy of the codes: a source may lie in a block that
// is encoded again. 240k of 4M rows moved (236M elements): both moments 1.35 ms,
// 0.15 of it the copies at the rate of a copy, the rest the tests of every
// element's row and the blocks encoded again. A training runs it once in a
// hundred steps.
struct Moments8Groups {
  int first[6];    // first block of each group
  unsigned width[5];
  unsigned count[5];  // elements
};

template <bool SIGNED>
__global__ void __launch_bounds__(256)
k_moments8_move(const uint8_t* __restrict__ from, const uint8_t* __restrict__ from_exp, uint8_t* __restrict__ codes,
                uint8_t* __restrict__ exps, Moments8Groups g, const int* __restrict__ source) {
  GS_PDL_ENTRY_PLAIN();
  const int lane = threadIdx.x & 31;
  for (int blk = blockIdx.x * 8 + (threadIdx.x >> 5); blk < g.first[5]; blk += gridDim.x * 8) {
    int k = 0;
#pragma unroll
    for (int q = 1; q < 5; ++q)
      if (blk >= g.first[q]) k = q;
    const unsigned w = g.width[k], count = g.count[k], e0 = (unsigned)(blk - g.first[k]) * kAdamwBlock;
    const size_t base = (size_t)g.first[k] * kAdamwBlock;
    unsigned at[4];  // element of the group that each one takes its value from
    bool moved = false;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const unsigned e = e0 + lane + 32 * q, row = e / w;
      at[q] = e;
      if (e >= count) continue;
      const int src = source[row];
      if (src < 0) continue;
      at[q] = (unsigned)src * w + (e - row * w);
      moved = true;
    }
    if (!__any_sync(0xffffffffu, moved)) continue;
    float x[4];
    unsigned top = 0u;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      x[q] = 0.f;
      if (e0 + lane + 32 * q < count) {
        const size_t i = base + at[q];
        const int f = from_exp[i / kAdamwBlock];
        x[q] = f == 255 ? NAN : decode8<SIGNED>(from[i], pow2_biased(f));
      }
      top = max(top, __float_as_uint(fabsf(x[q])));
    }
    const int f = block_field(__reduce_max_sync(0xffffffffu, top));
    const float down = pow2_biased(max(254 - f, 0));
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const unsigned e = e0 + lane + 32 * q;
      if (e < count) codes[base + e] = (uint8_t)(f == 255 ? 0u : encode8<SIGNED>(x[q], down, 1u << 19));
    }
    if (lane == 0) exps[blk] = (uint8_t)f;
  }
}

static Moments8Groups moments8_groups(int n, int sh_k) {
  const unsigned widths[5] = {3u, 3u, 4u, 1u, 3u * (unsigned)sh_k};
  Moments8Groups g;
  g.first[0] = 0;
  for (int k = 0; k < 5; ++k) {
    g.width[k] = widths[k];
    g.count[k] = widths[k] * (unsigned)n;
    g.first[k + 1] = g.first[k] + (int)((g.count[k] + kAdamwBlock - 1) / kAdamwBlock);
  }
  return g;
}

// A copy of one moment's codes and exponent bytes.
size_t moments8_move_bytes(int n, int sh_k) { return (size_t)moments8_groups(n, sh_k).first[5] * (kAdamwBlock + 1); }

void launch_moments8_move(uint8_t* mu, uint8_t* nu, uint8_t* mu_exp, uint8_t* nu_exp, int n, int sh_k,
                          const int* source, void* ws, cudaStream_t st) {
  const Moments8Groups g = moments8_groups(n, sh_k);
  const size_t blocks = (size_t)g.first[5], codes = blocks * kAdamwBlock;
  if (blocks == 0) return;
  uint8_t *from = static_cast<uint8_t*>(ws), *from_exp = from + codes;
  const int grid = (int)std::min<long long>(((long long)blocks + 7) / 8, (long long)device_sms() * 8);
  GS_TIMED("moments8_move", st);
  for (int moment = 0; moment < 2; ++moment) {
    uint8_t *x = moment ? nu : mu, *f = moment ? nu_exp : mu_exp;
    cudaMemcpyAsync(from, x, codes, cudaMemcpyDeviceToDevice, st);
    cudaMemcpyAsync(from_exp, f, blocks, cudaMemcpyDeviceToDevice, st);
    launch_kernel_plain(moment ? k_moments8_move<false> : k_moments8_move<true>, grid, 256, 0, st, from, from_exp, x,
                        f, g, source);
  }
}

}  // namespace gs
