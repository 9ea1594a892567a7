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
// implementation reproduces bit for bit. p' needs no such care: its divide
// and square root are the approximate ones (a few ulps of the update).
//
// 8-bit moments. A block is 128 elements from the tensor's start: one warp,
// four elements a lane. Each moment has one exponent byte a block,
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
// The kernels are bound by HBM: 28 B an element with 32-bit moments and fp32
// gradients, 16 B with 8-bit ones.
#include <algorithm>
#include <cmath>

#include "gs_kernels.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace gs {

constexpr int kAdamwBlock = GS_ADAMW_BLOCK;  // elements of a quantisation block and of a warp's unit of work
constexpr int kAdamwWarps = 8;
#ifndef GS_ADAMW_UNROLL
#define GS_ADAMW_UNROLL 2
#endif
constexpr int kAdamwUnroll = GS_ADAMW_UNROLL;  // blocks a warp has in flight
constexpr int kAdamwChunk = kAdamwBlock * kAdamwUnroll;
constexpr int kAdamwTile = kAdamwChunk * kAdamwWarps;  // elements a CTA takes at a time
static_assert(kAdamwBlock == 128, "a warp holds a block, four elements a lane");

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
  uint8_t grad_type, copy_type, vec, pad[5];
};

// Tables travel as kernel parameters (no device copy, nothing to keep alive,
// and a captured graph holds its own); N is a size class.
template <int N>
struct AdamwTable {
  AdamwDesc t[N];
  int first[N + 1];  // first tile of each tensor; first[n] = tiles
  int n;
  int index0;  // place of t[0] in the caller's list (the noise key)
};

struct AdamwParams {
  float b1, omb1, b2, omb2, eps, ln_b1, ln_b2;
  unsigned seed;
  const float* scale;
  int* state;    // [count, ticket, skipped, 0]
  bool advance;  // this launch is the step's last
};

__device__ __forceinline__ unsigned mix32(unsigned x) {
  // lowbias32, C. Wellons, "Prospecting for Hash Functions" (2018)
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
  float lr, wd, inv1, inv2;
};

__device__ __forceinline__ float adamw_param(float p, float m, float v, const AdamwStep& h, float eps) {
  float root;
  asm("sqrt.approx.f32 %0, %1;" : "=f"(root) : "f"(v * h.inv2));
  const float d = root + eps;
  return p - h.lr * (__fdividef(m * h.inv1, d) + h.wd * p);
}

// Element q of a lane in a block: four consecutive elements a lane (16-byte
// accesses), or, where a pointer is not aligned for that, every 32nd.
template <bool VEC>
__device__ __forceinline__ int block_element(int lane, int q) {
  return VEC ? 4 * lane + q : lane + 32 * q;
}

template <bool VEC>
__device__ __forceinline__ void load4(const float* __restrict__ p, int lane, float x[4]) {
  if (VEC) {
    const float4 t = reinterpret_cast<const float4*>(p)[lane];
    x[0] = t.x; x[1] = t.y; x[2] = t.z; x[3] = t.w;
  } else {
#pragma unroll
    for (int q = 0; q < 4; ++q) x[q] = p[lane + 32 * q];
  }
}

template <bool VEC>
__device__ __forceinline__ void store4(float* __restrict__ p, int lane, const float x[4]) {
  if (VEC) {
    reinterpret_cast<float4*>(p)[lane] = make_float4(x[0], x[1], x[2], x[3]);
  } else {
#pragma unroll
    for (int q = 0; q < 4; ++q) p[lane + 32 * q] = x[q];
  }
}

// Four gradients as loaded (16-bit ones two to a register where VEC).
template <int GT, bool VEC>
struct Grad4 {
  uint32_t w[(GT == GS_TYPE_F32 || !VEC) ? 4 : 2];
  __device__ __forceinline__ void load(const void* g, long long base, int lane) {
    if (GT == GS_TYPE_F32) {
      float x[4];
      load4<VEC>(static_cast<const float*>(g) + base, lane, x);
#pragma unroll
      for (int q = 0; q < 4; ++q) w[q] = __float_as_uint(x[q]);
    } else if (VEC) {
      const uint2 t = reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(g) + base)[lane];
      w[0] = t.x;
      w[1] = t.y;
    } else {
#pragma unroll
      for (int q = 0; q < 4; ++q) w[q] = (static_cast<const uint16_t*>(g) + base)[lane + 32 * q];
    }
  }
  __device__ __forceinline__ float get(int q) const {
    if (GT == GS_TYPE_F32) return __uint_as_float(w[q]);
    const unsigned h = VEC ? (q & 1 ? w[q >> 1] >> 16 : w[q >> 1] & 0xFFFFu) : w[q];
    if (GT == GS_TYPE_BF16) return __uint_as_float(h << 16);
    return __half2float(__ushort_as_half((unsigned short)h));
  }
};

template <bool VEC>
__device__ __forceinline__ void store_copy4(void* p, long long base, int lane, int type, const float x[4]) {
  unsigned h[4];
#pragma unroll
  for (int q = 0; q < 4; ++q)
    h[q] = type == GS_TYPE_BF16 ? __bfloat16_as_ushort(__float2bfloat16_rn(x[q]))
                                : __half_as_ushort(__float2half_rn(x[q]));
  uint16_t* c = static_cast<uint16_t*>(p) + base;
  if (VEC) {
    reinterpret_cast<uint2*>(c)[lane] = make_uint2(h[0] | (h[1] << 16), h[2] | (h[3] << 16));
  } else {
#pragma unroll
    for (int q = 0; q < 4; ++q) c[lane + 32 * q] = (uint16_t)h[q];
  }
}

// Four codes, one to a byte.
template <bool VEC>
__device__ __forceinline__ unsigned load_codes(const void* p, long long base, int lane) {
  const uint8_t* c = static_cast<const uint8_t*>(p) + base;
  if (VEC) return reinterpret_cast<const unsigned*>(c)[lane];
  unsigned w = 0u;
#pragma unroll
  for (int q = 0; q < 4; ++q) w |= (unsigned)c[lane + 32 * q] << (8 * q);
  return w;
}

template <bool VEC>
__device__ __forceinline__ void store_codes(void* p, long long base, int lane, unsigned w) {
  uint8_t* c = static_cast<uint8_t*>(p) + base;
  if (VEC) {
    reinterpret_cast<unsigned*>(c)[lane] = w;
  } else {
#pragma unroll
    for (int q = 0; q < 4; ++q) c[lane + 32 * q] = (uint8_t)(w >> (8 * q));
  }
}

// Whole blocks of a tensor by one warp, all loads issued before the first use.
template <int BITS, int GT, bool VEC>
__device__ __forceinline__ void adamw_chunk(const AdamwDesc& d, long long base, const AdamwParams& a,
                                            const AdamwStep& h, float s, unsigned key) {
  constexpr int U = kAdamwUnroll;
  const int lane = threadIdx.x & 31;
  float p[U][4], m[U][4], v[U][4];
  Grad4<GT, VEC> g[U];
  unsigned cm[U], cv[U];
  int fm[U], fv[U];
  const long long blk0 = base / kAdamwBlock;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const long long b = base + u * kAdamwBlock;
    load4<VEC>(d.param + b, lane, p[u]);
    g[u].load(d.grad, b, lane);
    if (BITS == 8) {
      cm[u] = load_codes<VEC>(d.mu, b, lane);
      cv[u] = load_codes<VEC>(d.nu, b, lane);
      fm[u] = d.mu_exp[blk0 + u];
      fv[u] = d.nu_exp[blk0 + u];
    } else {
      load4<VEC>(static_cast<const float*>(d.mu) + b, lane, m[u]);
      load4<VEC>(static_cast<const float*>(d.nu) + b, lane, v[u]);
    }
  }
  unsigned act = 0xFFFFFFFFu;
  if (d.active) {
    // row of element e: (base + e) / width, by multiplications with the
    // rounded-up reciprocal (exact: base < 2^37 and width <= 2^15, so that
    // their product with the reciprocal's excess stays below its scale)
    const unsigned w = d.width;
    const unsigned long long row0 = w == 1 ? (unsigned long long)base : __umul64hi((unsigned long long)base, d.magic);
    const unsigned rem0 = (unsigned)((unsigned long long)base - row0 * w);
    const unsigned magic = (unsigned)(d.magic >> 32) + 1u;  // > 2^32 / width
    const uint8_t* flags = d.active + row0;
    act = 0u;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const unsigned x = rem0 + u * kAdamwBlock + block_element<VEC>(lane, q);
        const unsigned r = w == 1 ? x : __umulhi(x, magic);
        act |= (flags[r] != 0 ? 1u : 0u) << (4 * u + q);
      }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const long long b = base + u * kAdamwBlock;
    float up_m = 0.f, up_v = 0.f;
    if (BITS == 8) {
      up_m = pow2_biased(min(fm[u], 254));
      up_v = pow2_biased(min(fv[u], 254));
      if (fm[u] == 255) up_m = NAN;
      if (fv[u] == 255) up_v = NAN;
    }
    unsigned top_m = 0u, top_v = 0u;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if (BITS == 8) {
        m[u][q] = decode8<true>((cm[u] >> (8 * q)) & 255u, up_m);
        v[u][q] = decode8<false>((cv[u] >> (8 * q)) & 255u, up_v);
      }
      const float gq = g[u].get(q) * s;
      m[u][q] = add_rn(mul_rn(m[u][q], a.b1), mul_rn(gq, a.omb1));
      v[u][q] = add_rn(mul_rn(v[u][q], a.b2), mul_rn(mul_rn(gq, gq), a.omb2));
      const float fresh = adamw_param(p[u][q], m[u][q], v[u][q], h, a.eps);
      if ((act >> (4 * u + q)) & 1u) p[u][q] = fresh;
      if (BITS == 8) {
        top_m = max(top_m, __float_as_uint(fabsf(m[u][q])));
        top_v = max(top_v, __float_as_uint(v[u][q]) & 0x7FFFFFFFu);
      }
    }
    store4<VEC>(d.param + b, lane, p[u]);
    if (d.copy) store_copy4<VEC>(d.copy, b, lane, d.copy_type, p[u]);
    if (BITS == 32) {
      store4<VEC>(static_cast<float*>(d.mu) + b, lane, m[u]);
      store4<VEC>(static_cast<float*>(d.nu) + b, lane, v[u]);
    } else {
      const int nm = block_field(__reduce_max_sync(0xffffffffu, top_m));
      const int nv = block_field(__reduce_max_sync(0xffffffffu, top_v));
      const float down_m = pow2_biased(max(254 - nm, 0)), down_v = pow2_biased(max(254 - nv, 0));
      const unsigned bkey = mix32(key ^ (unsigned)(blk0 + u));
      unsigned wm = 0u, wv = 0u;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const unsigned r = mix32(bkey + kGolden * (unsigned)block_element<VEC>(lane, q));
        wm |= encode8<true>(m[u][q], down_m, (r & 0xFFFFu) << 4) << (8 * q);
        wv |= encode8<false>(v[u][q], down_v, (r >> 16) << 4) << (8 * q);
      }
      store_codes<VEC>(d.mu, b, lane, nm == 255 ? 0u : wm);
      store_codes<VEC>(d.nu, b, lane, nv == 255 ? 0u : wv);
      if (lane == 0) {
        d.mu_exp[blk0 + u] = (uint8_t)nm;
        d.nu_exp[blk0 + u] = (uint8_t)nv;
      }
    }
  }
}

// One block of a tensor by one warp, `rem` elements of it in range.
template <int BITS>
__device__ __forceinline__ void adamw_block(const AdamwDesc& d, long long base, int rem, const AdamwParams& a,
                                            const AdamwStep& h, float s, unsigned key) {
  const int lane = threadIdx.x & 31;
  const long long blk = base / kAdamwBlock;
  float p[4], m[4], v[4];
  float up_m = 0.f, up_v = 0.f;
  bool nan_m = false, nan_v = false;
  if (BITS == 8) {
    const int fm = d.mu_exp[blk], fv = d.nu_exp[blk];
    nan_m = fm == 255;
    nan_v = fv == 255;
    up_m = pow2_biased(min(fm, 254));
    up_v = pow2_biased(min(fv, 254));
  }
  unsigned top_m = 0u, top_v = 0u;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int e = lane + 32 * q;
    const long long i = base + e;
    p[q] = m[q] = v[q] = 0.f;
    if (e >= rem) continue;
    float g = load_as_float(d.grad, i, d.grad_type) * s;
    p[q] = d.param[i];
    if (BITS == 8) {
      m[q] = decode8<true>(static_cast<const uint8_t*>(d.mu)[i], up_m);
      v[q] = decode8<false>(static_cast<const uint8_t*>(d.nu)[i], up_v);
      if (nan_m) m[q] = NAN;
      if (nan_v) v[q] = NAN;
    } else {
      m[q] = static_cast<const float*>(d.mu)[i];
      v[q] = static_cast<const float*>(d.nu)[i];
    }
    m[q] = add_rn(mul_rn(m[q], a.b1), mul_rn(g, a.omb1));
    v[q] = add_rn(mul_rn(v[q], a.b2), mul_rn(mul_rn(g, g), a.omb2));
    const float fresh = adamw_param(p[q], m[q], v[q], h, a.eps);
    if (!d.active || d.active[i / d.width] != 0) {
      p[q] = fresh;
      d.param[i] = fresh;
    }
    if (d.copy) store_as(d.copy, i, d.copy_type, p[q]);
    if (BITS == 32) {
      static_cast<float*>(d.mu)[i] = m[q];
      static_cast<float*>(d.nu)[i] = v[q];
    }
    top_m = max(top_m, __float_as_uint(fabsf(m[q])));
    top_v = max(top_v, __float_as_uint(fabsf(v[q])));
  }
  if (BITS == 8) {
    const int fm = block_field(__reduce_max_sync(0xffffffffu, top_m));
    const int fv = block_field(__reduce_max_sync(0xffffffffu, top_v));
    const float down_m = pow2_biased(max(254 - fm, 0)), down_v = pow2_biased(max(254 - fv, 0));
    const unsigned bkey = mix32(key ^ (unsigned)blk);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int e = lane + 32 * q;
      if (e >= rem) continue;
      const unsigned r = mix32(bkey + kGolden * (unsigned)e);
      unsigned cm = encode8<true>(m[q], down_m, (r & 0xFFFFu) << 4);
      unsigned cv = encode8<false>(v[q], down_v, (r >> 16) << 4);
      if (fm == 255) cm = 0u;
      if (fv == 255) cv = 0u;
      static_cast<uint8_t*>(d.mu)[base + e] = (uint8_t)cm;
      static_cast<uint8_t*>(d.nu)[base + e] = (uint8_t)cv;
    }
    if (lane == 0) {
      d.mu_exp[blk] = (uint8_t)fm;
      d.nu_exp[blk] = (uint8_t)fv;
    }
  }
}

template <int BITS, int N>
__global__ void __launch_bounds__(32 * kAdamwWarps)
k_adamw(const __grid_constant__ AdamwTable<N> tab, const __grid_constant__ AdamwParams a) {
  GS_PDL_ENTRY_PLAIN();
  const int c = *(volatile int*)a.state;
  const float s = a.scale ? *(volatile const float*)a.scale : 1.f;
  const bool go = fabsf(s) <= 3.402823466e38f;
  if (go) {
    const float cf = (float)c;
    AdamwStep h;
    // 1 - b^t as -expm1(t ln b): no cancellation at small t
    h.inv1 = 1.f / -expm1f((cf + 1.f) * a.ln_b1);
    h.inv2 = 1.f / -expm1f((cf + 1.f) * a.ln_b2);
    const unsigned key = mix32(a.seed + kGolden * (unsigned)c);
    const int tiles = tab.first[tab.n];
    int k = 0;
    for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
      // the last tensor whose first tile is not behind this one
      int hi = tab.n;
      while (hi - k > 1) {
        const int mid = (k + hi) >> 1;
        if (tab.first[mid] <= tile) k = mid;
        else hi = mid;
      }
      const AdamwDesc& d = tab.t[k];
      h.lr = d.lr_init * expf(cf * d.ln_decay);
      h.wd = d.weight_decay;
      const long long base = (long long)(tile - tab.first[k]) * kAdamwTile + (threadIdx.x >> 5) * kAdamwChunk;
      const long long left = d.count - base;
      if (left <= 0) continue;
      const unsigned tkey = mix32(key + kGolden * (unsigned)(tab.index0 + k));
      if (left >= kAdamwChunk) {
        switch (d.grad_type * 2 + d.vec) {
          case 0: adamw_chunk<BITS, GS_TYPE_F32, false>(d, base, a, h, s, tkey); break;
          case 1: adamw_chunk<BITS, GS_TYPE_F32, true>(d, base, a, h, s, tkey); break;
          case 2: adamw_chunk<BITS, GS_TYPE_BF16, false>(d, base, a, h, s, tkey); break;
          case 3: adamw_chunk<BITS, GS_TYPE_BF16, true>(d, base, a, h, s, tkey); break;
          case 4: adamw_chunk<BITS, GS_TYPE_F16, false>(d, base, a, h, s, tkey); break;
          default: adamw_chunk<BITS, GS_TYPE_F16, true>(d, base, a, h, s, tkey); break;
        }
      } else {
        for (int e = 0; e < left; e += kAdamwBlock)
          adamw_block<BITS>(d, base + e, (int)(left - e < kAdamwBlock ? left - e : kAdamwBlock), a, h, s, tkey);
      }
    }
  }
  if (!a.advance) return;
  // the last CTA to finish (atomic ticket, no waiting) advances the count
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    const unsigned t = atomicAdd(reinterpret_cast<unsigned*>(a.state + 1), 1u);
    if (t == gridDim.x - 1) {
      if (go) a.state[0] = c + 1;
      else a.state[2] = a.state[2] + 1;
      a.state[1] = 0;
    }
  }
}

template <int BITS, int N>
static void launch_adamw_class(const GsAdamwTensor* t, int n, int index0, const AdamwParams& a, cudaStream_t st) {
  static thread_local AdamwTable<N> tab;
  int tiles = 0;
  for (int i = 0; i < n; ++i) {
    AdamwDesc& d = tab.t[i];
    d.param = t[i].param;
    d.grad = t[i].grad;
    d.mu = t[i].mu;
    d.nu = t[i].nu;
    d.mu_exp = t[i].mu_exp;
    d.nu_exp = t[i].nu_exp;
    d.copy = t[i].copy;
    d.active = t[i].active;
    d.count = t[i].count;
    d.lr_init = t[i].lr_init;
    d.ln_decay = (float)(std::log((double)t[i].decay_rate) / (double)t[i].transition_steps);
    d.weight_decay = t[i].weight_decay;
    d.width = (unsigned)t[i].width;
    d.grad_type = (uint8_t)t[i].grad_type;
    d.copy_type = (uint8_t)t[i].copy_type;
    d.magic = t[i].width > 1 ? ~0ull / (unsigned)t[i].width + 1ull : 0ull;
    const size_t g4 = t[i].grad_type == GS_TYPE_F32 ? 16 : 8;
    uintptr_t bits = (uintptr_t)t[i].param | ((uintptr_t)t[i].copy * 2) | ((uintptr_t)t[i].grad * (16 / g4));
    if (BITS == 32) bits |= (uintptr_t)t[i].mu | (uintptr_t)t[i].nu;
    d.vec = (bits & 15) == 0;
    tab.first[i] = tiles;
    tiles += (int)((t[i].count + kAdamwTile - 1) / kAdamwTile);
  }
  tab.first[n] = tiles;
  tab.n = n;
  tab.index0 = index0;
  const int grid = std::max(1, std::min(tiles, device_sms() * 8));
  GS_TIMED(BITS == 8 ? "adamw8" : "adamw", st);
  launch_kernel_plain(k_adamw<BITS, N>, grid, 32 * kAdamwWarps, 0, st, tab, a);
}

constexpr int kAdamwSmall = 8, kAdamwMost = 256;

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
  a.scale = scale;
  a.state = state;
  int at = 0;
  do {
    const int take = std::min(n - at, kAdamwMost);
    a.advance = at + take >= n;
    if (cfg.moment_bits == 8) {
      if (take <= kAdamwSmall) launch_adamw_class<8, kAdamwSmall>(tensors + at, take, at, a, st);
      else launch_adamw_class<8, kAdamwMost>(tensors + at, take, at, a, st);
    } else {
      if (take <= kAdamwSmall) launch_adamw_class<32, kAdamwSmall>(tensors + at, take, at, a, st);
      else launch_adamw_class<32, kAdamwMost>(tensors + at, take, at, a, st);
    }
    at += take;
  } while (at < n);
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

// A tile is 16 KB of a tensor counted from the 16-byte boundary at or before
// its first element, 64 bytes a thread in 16-byte loads; only the vectors
// that hold both the tensor's elements and others are read one by one.
constexpr int kNormVecs = 4;
constexpr int kNormTileBytes = 256 * 16 * kNormVecs;

__host__ __device__ __forceinline__ long long norm_tiles(const void* grad, long long count, int type) {
  const long long bytes = (long long)((uintptr_t)grad & 15) + count * (type == GS_TYPE_F32 ? 4 : 2);
  return count > 0 ? (bytes + kNormTileBytes - 1) / kNormTileBytes : 0;
}

template <int GT>
__device__ __forceinline__ void norm_tile(const GradDesc& d, long long tile, double acc[4]) {
  constexpr int PER = GT == GS_TYPE_F32 ? 4 : 8;  // elements of a vector
  const unsigned shift = (unsigned)((uintptr_t)d.grad & 15) / (16 / PER);
  const uint4* vecs = reinterpret_cast<const uint4*>((uintptr_t)d.grad & ~(uintptr_t)15);
  const long long v0 = tile * (256 * kNormVecs) + threadIdx.x;
  uint4 w[kNormVecs];
#pragma unroll
  for (int j = 0; j < kNormVecs; ++j) {
    const long long e = (v0 + 256 * j) * PER - shift;  // the vector's first element
    w[j] = make_uint4(0u, 0u, 0u, 0u);
    if (e >= 0 && e + PER <= d.count) {
      w[j] = __ldg(vecs + v0 + 256 * j);
    } else if (e + PER > 0 && e < d.count) {
      for (int q = 0; q < PER; ++q)
        if (e + q >= 0 && e + q < d.count) {
          const double x = (double)load_as_float(d.grad, e + q, GT);
          acc[0] += x * x;
        }
    }
  }
#pragma unroll
  for (int j = 0; j < kNormVecs; ++j) {
    const unsigned b[4] = {w[j].x, w[j].y, w[j].z, w[j].w};
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if (GT == GS_TYPE_F32) {
        const double x = (double)__uint_as_float(b[q]);
        acc[q] = fma(x, x, acc[q]);
      } else {
        float lo, hi;
        if (GT == GS_TYPE_BF16) {
          lo = __uint_as_float(b[q] << 16);
          hi = __uint_as_float(b[q] & 0xFFFF0000u);
        } else {
          lo = __half2float(__ushort_as_half((unsigned short)(b[q] & 0xFFFFu)));
          hi = __half2float(__ushort_as_half((unsigned short)(b[q] >> 16)));
        }
        const double x = (double)lo, y = (double)hi;
        acc[q] = fma(x, x, acc[q]);
        acc[q] = fma(y, y, acc[q]);
      }
    }
  }
}

template <int N>
__global__ void __launch_bounds__(256)
k_grad_norm(const __grid_constant__ GradTable<N> tab, double* __restrict__ partials, int part0, int parts,
            float max_norm, const float* __restrict__ unscale, GsGradNorm* __restrict__ out) {
  GS_PDL_ENTRY_PLAIN();
  __shared__ double s_red[8];
  __shared__ bool s_last;
  double sums[4] = {0.0, 0.0, 0.0, 0.0};
  const int tiles = tab.first[tab.n];
  int k = 0;
  for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    int hi = tab.n;
    while (hi - k > 1) {
      const int mid = (k + hi) >> 1;
      if (tab.first[mid] <= tile) k = mid;
      else hi = mid;
    }
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

constexpr int kNormSmall = 8, kNormMost = 1024, kNormGrid = 1184;

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
// 8-bit moments to and from values, one warp a block. Encoding rounds to
// nearest (halves up): values that came from codes are kept exactly.
template <typename T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ float from_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

template <typename T>
__global__ void __launch_bounds__(256)
k_moments8_decode(const uint8_t* __restrict__ mu, const uint8_t* __restrict__ nu, const uint8_t* __restrict__ mu_exp,
                  const uint8_t* __restrict__ nu_exp, long long count, T* __restrict__ mu_out,
                  T* __restrict__ nu_out) {
  GS_PDL_ENTRY_PLAIN();
  const long long stride = (long long)gridDim.x * 256;
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < count; i += stride) {
    const long long blk = i / kAdamwBlock;
    const int fm = mu_exp[blk], fv = nu_exp[blk];
    const float m = decode8<true>(mu[i], pow2_biased(min(fm, 254)));
    const float v = decode8<false>(nu[i], pow2_biased(min(fv, 254)));
    mu_out[i] = from_float<T>(fm == 255 ? NAN : m);
    nu_out[i] = from_float<T>(fv == 255 ? NAN : v);
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
  const int grid = (int)std::min((count + 255) / 256, (long long)device_sms() * 8);
  GS_TIMED("moments8_decode", st);
  if (type == GS_TYPE_F32)
    launch_kernel_plain(k_moments8_decode<float>, grid, 256, 0, st, mu, nu, mu_exp, nu_exp, count,
                        static_cast<float*>(mu_out), static_cast<float*>(nu_out));
  else
    launch_kernel_plain(k_moments8_decode<__nv_bfloat16>, grid, 256, 0, st, mu, nu, mu_exp, nu_exp, count,
                        static_cast<__nv_bfloat16*>(mu_out), static_cast<__nv_bfloat16*>(nu_out));
}

void launch_moments8_encode(const float* mu, const float* nu, long long count, uint8_t* mu8, uint8_t* nu8,
                            uint8_t* mu_exp, uint8_t* nu_exp, cudaStream_t st) {
  const long long blocks = (count + kAdamwBlock - 1) / kAdamwBlock;
  const int grid = (int)std::min((blocks + 7) / 8, (long long)device_sms() * 8);
  GS_TIMED("moments8_encode", st);
  launch_kernel_plain(k_moments8_encode, grid, 256, 0, st, mu, nu, count, mu8, nu8, mu_exp, nu_exp);
}

}  // namespace gs
