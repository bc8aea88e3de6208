// AdamW over a list of tensors in one launch, with the moments in fp32 or in 8 bits.
//
//   m <- b1 m + (1 - b1) g,   v <- b2 v + (1 - b2) g^2
//   p <- p - lr wd p - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// All arithmetic is fp32.  Products and sums that reach a stored moment are rounded one by one (no fused multiply-add), so that the same
// inputs give the same codes wherever the formula is evaluated in IEEE fp32.
//
// 8-bit moments.  ADAMW_BLOCK consecutive elements of a tensor share a scale.  m is held with a sign, 4 exponent and 3 mantissa bits;
// of v its root r is held, with 4 exponent and 4 mantissa bits (the root halves the range in octaves, and r has no sign to store):
//   value(c) = (1 + mantissa / 2^MB) 2^exponent, value(0) = 0, the largest code stands for NaN; element = value(c) * scale,
//   scale = the smallest power of two with which the block's largest finite magnitude does not exceed the largest finite code.
// Rounding is stochastic.  To nearest, a moment whose change per step is below half a step of its code would never move: r changes by at most
// 0.05 % a step while v decays (b2 = 0.999) and a step is 3 to 6 %, so a v that was large once would stay large.  Rounded
// up with a probability equal to the fraction, the stored moment follows the fp32 one on average.  A power of two as scale keeps that noise
// small: a moment that has not changed has the same code in every step, whatever the largest element does.  The 16 random bits of an
// element come from a hash of (seed, step, tensor, element): the result is a function of the inputs alone.
// An r above zero takes code 1 at least: with r = 0 beside an m that is not, the next update would be unbounded.
// B200K_ADAMW_PEAK_SCALES: the older rule, for states that were begun with it: scale = the block's peak / the largest finite code's value, and an r
// below code 1 is rounded like an m there, up to code 1 with a probability equal to the fraction, else to zero.
// A non-finite moment takes the NaN code and does not enter the scale, so that it stays with its element.
//
// Bound: HBM with fp32 moments (184 M fp32 parameters, 28 bytes each: 800 us, 6.4 TB/s, all of the copy rate); with 8 bits the instructions, about 90 an
// element (87 M bf16 parameters, 10 bytes each: 278 us, 3.2 TB/s, 83 % of the issue slots).

#include <math.h>

#include "dtypes.cuh"
#include "launch.h"
#include "ptx.cuh"

namespace b200k {

constexpr int ADAMW_BLOCK = 256;                      // elements that share a scale: one warp, 8 elements a lane
constexpr int ADAMW_THREADS = 256;
constexpr int ADAMW_CHUNK = 64 * ADAMW_BLOCK;         // elements of one CTA
// Tensors of a launch: the table is a kernel parameter, which the host copies whole.  40 tensors take 13.1 us a step (host) with the small table and 16.7 with the
// large one, the kernel 5.0 us with either; a small table of 120 costs 0.6 us with up to 40 tensors and saves 3 with more.
constexpr int ADAMW_SMALL_TABLE = 40, ADAMW_LARGE_TABLE = 400;

// What the kernels read of the step number; one per optimiser, in device memory.
struct AdamwState {
  double b1_pow, b2_pow;   // b1^t, b2^t after t steps
  int64_t step;            // t
  double inv_bc1;          // 1 / (1 - b1^(t+1))
  float inv_sqrt_bc2;      // 1 / sqrt(1 - b2^(t+1))
  unsigned ticket;         // CTAs of the running launch that are done
};
static_assert(sizeof(AdamwState) == 40, "layout shared with the host");

template <int CAP>
struct AdamwTable {
  b200k_adamw_tensor t[CAP];
  int first_chunk[CAP + 1];
};

struct AdamwParams {
  AdamwState* state;
  const float* lr_dev;           // overrides lr when not null
  const float* grad_scale_dev;   // overrides grad_scale when not null
  double lr, weight_decay;
  double b1d, b2d;
  float b1, one_minus_b1, b2, one_minus_b2, eps, grad_scale;
  uint32_t seed;
  // Powers of two that come as parameters: a shift and add by a constant would run on the ALU pipe, which the byte and bit work of the 8-bit moments
  // fills before anything else; a multiply-add by a number the compiler does not know runs on the FMA pipe.
  uint32_t two4, two5, two16, two19, two20;
  int n;                         // tensors in the table
  int advance;                   // this launch ends the step
};

// 32-bit hash: two rounds of xor-shift and an odd multiplier (the leading bits of sqrt(3)/2 and sqrt(2)/2).
__device__ __forceinline__ uint32_t mix32(uint32_t x, uint32_t two16) {
  x ^= __umulhi(x, two16);           // x >> 16
  x *= 0xDDB3D743u;
  x ^= x >> 15;
  x *= 0xB504F335u;
  return x ^ __umulhi(x, two16);
}

// Exponent field E of the block's scale 2^(E - 142): the largest finite code has the value (2 - 2^(1 - MB)) 2^15, and adding what a mantissa may
// lack of that carries a peak beyond it into the next octave.  E >= 16 keeps the scale and its inverse normal numbers.
template <int MB>
__device__ __forceinline__ uint32_t scale_exponent(float peak) {
  const uint32_t e = (__float_as_uint(peak) + ((1u << (24 - MB)) - 1)) >> 23;
  return e < 16 ? 16 : e;
}
template <int MB>
__device__ __forceinline__ constexpr float top_value() { return (2.f - 2.f / (1 << MB)) * 32768.f; }
// Scale and inverse of a block by its peak: two divisions, so that each is the formula's.  Where the inverse would overflow (peaks below 2^-112, and zero, whose
// scale is zero) it is the other rule's for the smallest peaks.
template <int MB>
__device__ __forceinline__ void peak_scale(float peak, float& scale, float& inverse) {
  scale = __fdiv_rn(peak, top_value<MB>());
  inverse = __fdiv_rn(top_value<MB>(), peak);
  if (!(inverse <= 3.4028234663852886e38f)) {
    scale = peak == 0.f ? 0.f : 0x1p-126f;
    inverse = 0x1p126f;
  }
}
__device__ __forceinline__ float scale_of(uint32_t e) { return __uint_as_float((e - 15) << 23); }
__device__ __forceinline__ float inverse_scale_of(uint32_t e) { return __uint_as_float((269 - e) << 23); }

// prmt with the top bit of the selected bytes spread over them (selector nibbles 8..15, which __byte_perm does not pass on).
__device__ __forceinline__ uint32_t spread_top(uint32_t x, uint32_t selector) {
  uint32_t d;
  asm("prmt.b32 %0, %1, %1, %2;" : "=r"(d) : "r"(x), "r"(selector));
  return d;
}

// The values of a word's four codes (to be multiplied by their block's scale); up = 2^(23 - MB).
template <int MB>
__device__ __forceinline__ void decode4(uint32_t word, uint32_t up, float (&f)[4]) {
  constexpr uint32_t MASK = MB == 3 ? 0x7F7F7F7Fu : 0xFFFFFFFFu;
  const uint32_t mag = word & MASK;
  uint32_t bits[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) bits[j] = __byte_perm(mag, 0, 0x4440 + j) * up + (127u << 23);
  if (MB == 3) {
    // zeros are common among first moments: a mask per element, and the sign with the same instruction
    const uint32_t some = mag + 0x7F7F7F7Fu, sign = word & 0x80808080u;      // some: top bit of each byte that is not 0
#pragma unroll
    for (int j = 0; j < 4; ++j) bits[j] = (bits[j] & spread_top(some, 0x8888 + 0x1111 * j)) | __byte_perm(sign, 0, (j << 12) | 0x0444);
  }
  // rare: the NaN code, and a zero root.  All four bytes at once, by carries; a false alarm only costs time.
  const uint32_t rare = MB == 3 ? (mag + 0x01010101u) & 0x80808080u : ((mag - 0x01010101u) & ~mag & 0x80808080u) | ((~mag - 0x01010101u) & mag & 0x80808080u);
  if (rare != 0) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t c = (mag >> (8 * j)) & 0xFFu;
      if (c == (1u << (4 + MB)) - 1) bits[j] = 0x7FC00000u;
      if (MB == 4 && c == 0) bits[j] = 0;
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) f[j] = __uint_as_float(bits[j]);
}

__device__ __forceinline__ bool is_finite(float x) { return fabsf(x) <= 3.4028234663852886e38f; }

__device__ __forceinline__ float min3(float a, float b, float c) {
  float d;
  asm("min.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// The codes of four elements, m's with their signs, given 16 random bits of each hash.  up = 2^(1 + MB).  `finite`: none of the block's elements is infinite or NaN.
//
// A normal code is the exponent and the MB first mantissa bits of |x| * inverse (in [1, 2^16), so that exponent 127 is 0), after the random bits were
// added just below them.  Multiplied by 2^(1 + MB) those 4 + MB bits are the top byte of the word (m's with a zero above them), the random bits
// are bytes 1 and 2 of what is added, and the exponent's offset is a constant in byte 3: a byte permutation and a multiply-add.
// PEAK: by the older rule; a product with the inverse may then pass the largest code's value by a rounding.
template <int MB, bool PEAK>
__device__ __forceinline__ uint32_t encode4(const float (&x)[4], float inverse, const uint32_t (&hash)[4], uint32_t up, bool finite) {
  constexpr float LEAST = 1.f + 1.f / (1 << MB);       // value of code 1
  uint32_t c[4];
  float y[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    y[j] = __fmul_rn(fabsf(x[j]), inverse);
    if (PEAK) y[j] = fminf(y[j], top_value<MB>());
    // -(127 << 23) * up is 8 << 24 and 16 << 24 modulo 2^32
    const uint32_t add = __byte_perm(hash[j], MB == 3 ? 0x08u : 0x10u, MB == 3 ? 0x4105 : 0x4325);
    c[j] = __float_as_uint(y[j]) * up + add;
  }
  if (min3(min3(y[0], y[1], y[2]), y[3], y[3]) < LEAST) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      // below code 1: an m up to it with probability y / value(1), an r above zero always (by the older rule like an m).  u = 1 + (2 r + 1) / 2^17 for the 16 bits r.
      const float u = __uint_as_float((MB == 3 ? hash[j] & 0xFFFFu : hash[j] >> 16) * 128u + 0x3F800040u);
      const uint32_t small = (MB == 3 || PEAK ? fmaf(u, LEAST, -LEAST) : 0.f) < y[j] ? 1u << 24 : 0u;
      c[j] = y[j] < LEAST ? small : c[j];
    }
  }
  if (!finite) {
#pragma unroll
    for (int j = 0; j < 4; ++j) c[j] = is_finite(x[j]) ? c[j] : MB == 3 ? 0x7F000000u : 0xFF000000u;
  }
  if (MB == 3) {
#pragma unroll
    for (int j = 0; j < 4; ++j) c[j] = (c[j] & 0x7FFFFFFFu) | (__float_as_uint(x[j]) & 0x80000000u);
  }
  return __byte_perm(__byte_perm(c[0], c[1], 0x0073), __byte_perm(c[2], c[3], 0x0073), 0x5410);
}

// Maximum that lets NaN through.
__device__ __forceinline__ float max_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float warp_max_nonneg(float v) {   // floats >= 0 order like their bits, infinity and NaN above them
  return __uint_as_float(__reduce_max_sync(0xFFFFFFFFu, __float_as_uint(v)));
}

// 4 consecutive elements at p[0..4), of which the first `left` exist, as the words that they take in memory.
template <typename T>
struct Four {
  uint32_t w[sizeof(T)];
};
template <typename T>
__device__ __forceinline__ Four<T> fetch4(const T* p, bool vec, int left) {
  Four<T> v;
  if (vec) {
    if constexpr (sizeof(T) == 4) {
      const uint4 u = *reinterpret_cast<const uint4*>(p);
      v.w[0] = u.x; v.w[1] = u.y; v.w[2] = u.z; v.w[3] = u.w;
    } else {
      const uint2 u = *reinterpret_cast<const uint2*>(p);
      v.w[0] = u.x; v.w[1] = u.y;
    }
  } else {
    float f[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = i < left ? to_f32<T>(p[i]) : 0.f;
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)); ++i) {
      if constexpr (sizeof(T) == 4) v.w[i] = __float_as_uint(f[i]); else v.w[i] = pack_word<T>(f[2 * i], f[2 * i + 1]);
    }
  }
  return v;
}
template <typename T>
__device__ __forceinline__ void values4(const Four<T>& v, float (&f)[4]) {
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(T)); ++i) {
    if constexpr (sizeof(T) == 4) f[i] = __uint_as_float(v.w[i]); else unpack_word<T>(v.w[i], f[2 * i], f[2 * i + 1]);
  }
}
template <typename T>
__device__ __forceinline__ void store4(T* p, bool vec, int left, const float (&f)[4]) {
  if (vec) {
    store_vec<T, 4>(p, f);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < left) p[i] = from_f32<T>(f[i]);
  }
}

// sqrt(x), correctly rounded, of two numbers in [2^-60, 2^120]: Goldschmidt's iteration from an approximate 1 / sqrt(x), and a last step on the exact
// residual, which by Markstein's theorem rounds correctly (P. Markstein, IA-64 and Elementary Functions, ch. 9).  Without the range test of
// the general function it takes no branch and runs on packed numbers.  Half the reciprocal root and the residual are held negated.
__device__ __forceinline__ uint64_t sqrt_in_range(uint64_t x) {
  float x0, x1, y0, y1;
  unpack_f32x2(x, x0, x1);
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(y0) : "f"(x0));
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(y1) : "f"(x1));
  const uint64_t y = pack_f32x2(y0, y1);
  uint64_t g = mul_f32x2(x, y), h = mul_f32x2(pack_f32x2(-0.5f, -0.5f), y);
  const uint64_t r = fma_f32x2(g, h, pack_f32x2(0.5f, 0.5f));
  g = fma_f32x2(g, r, g);
  h = fma_f32x2(h, r, h);
  return fma_f32x2(fma_f32x2(g, g, mul_f32x2(x, pack_f32x2(-1.f, -1.f))), h, g);
}
__device__ __forceinline__ void sqrt4(const float (&f)[4], float (&root)[4]) {
  const float lo = min3(min3(f[0], f[1], f[2]), f[3], f[3]);
  const float hi = max_nan(max_nan(f[0], f[1], f[2]), f[3], f[3]);
  if (lo >= 0x1p-60f && hi <= 0x1p120f) {
#pragma unroll
    for (int j = 0; j < 2; ++j) unpack_f32x2(sqrt_in_range(pack_f32x2(f[2 * j], f[2 * j + 1])), root[2 * j], root[2 * j + 1]);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) root[j] = __fsqrt_rn(f[j]);
  }
}

// What a lane reads of a block: twice four elements, 128 apart.
template <typename P, typename G, bool MASTER, int BITS>
struct AdamwBlock {
  Four<P> p[MASTER ? 1 : 2];
  Four<float> master[MASTER ? 2 : 1];
  Four<G> g[2];
  uint32_t cm[2], cr[2];                           // 8-bit moments
  Four<float> m[BITS == 32 ? 2 : 1], v[BITS == 32 ? 2 : 1];
  float scale_m, scale_r;
};
__device__ __forceinline__ int left_of(int64_t i, int64_t end) { return i >= end ? 0 : (end - i < 4 ? static_cast<int>(end - i) : 4); }

// `full`: the block is whole and everything is aligned (the same for all lanes).
template <typename P, typename G, bool MASTER, int BITS>
__device__ __forceinline__ void adamw_read(AdamwBlock<P, G, MASTER, BITS>& k, const b200k_adamw_tensor& t, int64_t base, int64_t end, bool full) {
  const int64_t i0 = base + (threadIdx.x & 31) * 4;
  if constexpr (BITS == 8) {
    k.scale_m = t.m_scale[base / ADAMW_BLOCK];
    k.scale_r = t.v_scale[base / ADAMW_BLOCK];
#pragma unroll
    for (int h = 0; h < 2; ++h) {                  // the code buffers are padded to whole blocks
      k.cm[h] = reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(t.m) + i0)[32 * h];
      k.cr[h] = reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(t.v) + i0)[32 * h];
    }
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int64_t i = i0 + h * 128;
    const int left = full ? 4 : left_of(i, end);
    if constexpr (MASTER) k.master[h] = fetch4<float>(t.master + i, full, left); else k.p[h] = fetch4<P>(static_cast<const P*>(t.p) + i, full, left);
    k.g[h] = fetch4<G>(static_cast<const G*>(t.g) + i, full, left);
    if constexpr (BITS == 32) {
      k.m[h] = fetch4<float>(static_cast<const float*>(t.m) + i, full, left);
      k.v[h] = fetch4<float>(static_cast<const float*>(t.v) + i, full, left);
    }
  }
}

// KIND: 32, 8, or 8 + B200K_ADAMW_PEAK_SCALES.
template <typename P, typename G, bool MASTER, int KIND, int CAP>
__global__ void __launch_bounds__(ADAMW_THREADS) adamw_kernel(const __grid_constant__ AdamwTable<CAP> table, const AdamwParams q) {
  constexpr int BITS = KIND % B200K_ADAMW_PEAK_SCALES;
  constexpr bool PEAK = KIND >= B200K_ADAMW_PEAK_SCALES;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const double lr = q.lr_dev != nullptr ? static_cast<double>(*q.lr_dev) : q.lr;
  const float step_size = static_cast<float>(lr * q.state->inv_bc1);
  const float decay = static_cast<float>(1.0 - lr * q.weight_decay);
  const float inv_sqrt_bc2 = q.state->inv_sqrt_bc2;
  const float grad_scale = q.grad_scale_dev != nullptr ? *q.grad_scale_dev : q.grad_scale;
  const uint32_t step = static_cast<uint32_t>(q.state->step + 1);

  // the tensor of this CTA's chunk: the last one whose first chunk is not beyond it
  const int chunk = blockIdx.x;
  int lo = 0, hi = q.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (table.first_chunk[mid] <= chunk) lo = mid; else hi = mid - 1;
  }
  const b200k_adamw_tensor& t = table.t[lo];
  const int64_t begin = static_cast<int64_t>(chunk - table.first_chunk[lo]) * ADAMW_CHUNK;
  const int64_t end = begin + ADAMW_CHUNK < t.n ? begin + ADAMW_CHUNK : t.n;
  const uint32_t salt = BITS == 8 ? mix32(mix32(q.seed + step * 0x9E3779B9u, q.two16) + static_cast<uint32_t>(t.index), q.two16) : 0u;
  P* const tp = static_cast<P*>(t.p);
  const bool aligned = ((reinterpret_cast<uintptr_t>(tp) & (4 * sizeof(P) - 1)) | (reinterpret_cast<uintptr_t>(t.g) & (4 * sizeof(G) - 1))) == 0;

  // the next block's loads are under way while this one is worked on
  AdamwBlock<P, G, MASTER, BITS> next;
  int64_t base = begin + warp * ADAMW_BLOCK;
  if (base < end) adamw_read<P, G, MASTER, BITS>(next, t, base, end, aligned && base + ADAMW_BLOCK <= end);
  for (; base < end; base += (ADAMW_THREADS / 32) * ADAMW_BLOCK) {
    const int64_t block = base / ADAMW_BLOCK;
    const AdamwBlock<P, G, MASTER, BITS> now = next;
    const int64_t following = base + (ADAMW_THREADS / 32) * ADAMW_BLOCK;
    if (following < end) adamw_read<P, G, MASTER, BITS>(next, t, following, end, aligned && following + ADAMW_BLOCK <= end);
    const bool full = aligned && base + ADAMW_BLOCK <= end;
    float m1[2][4], root[2][4];
    float peak_m = 0.f, peak_r = 0.f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int64_t i = base + h * 128 + lane * 4;
      const int left = full ? 4 : left_of(i, end);
      float p[4], g[4], m[4], v[4];
      if constexpr (MASTER) values4<float>(now.master[h], p); else values4<P>(now.p[h], p);
      values4<G>(now.g[h], g);
      if constexpr (BITS == 8) {
        decode4<3>(now.cm[h], q.two20, m);
        decode4<4>(now.cr[h], q.two19, v);
      } else {
        values4<float>(now.m[h], m);
        values4<float>(now.v[h], v);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (BITS == 8) {
          m[j] = __fmul_rn(m[j], now.scale_m);
          v[j] = __fmul_rn(v[j], now.scale_r);
          v[j] = __fmul_rn(v[j], v[j]);
        }
        g[j] = __fmul_rn(g[j], grad_scale);
        m[j] = __fadd_rn(__fmul_rn(m[j], q.b1), __fmul_rn(g[j], q.one_minus_b1));
        v[j] = __fadd_rn(__fmul_rn(v[j], q.b2), __fmul_rn(__fmul_rn(g[j], g[j]), q.one_minus_b2));
        m1[h][j] = m[j];
      }
      sqrt4(v, root[h]);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        // p alone may round otherwise than the plain formula: the quotient takes an approximate reciprocal (1 unit in the last place), of an
        // update that is itself a small part of p.  The divisor is zero or a normal number: sqrt of the smallest fp32 is 2^-74.5, eps is 0 or normal.
        float inverse;
        asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inverse) : "f"(fmaf(root[h][j], inv_sqrt_bc2, q.eps)));
        p[j] = p[j] * decay - m[j] * inverse * step_size;
      }
      if (BITS == 8) {                     // behind the tensor's end all of it is zero
        peak_m = max_nan(max_nan(peak_m, fabsf(m[0]), fabsf(m[1])), fabsf(m[2]), fabsf(m[3]));
        peak_r = max_nan(max_nan(peak_r, root[h][0], root[h][1]), root[h][2], root[h][3]);
      }
      if (MASTER) store4<float>(t.master + i, full, left, p);
      store4<P>(tp + i, full, left, p);
      if (BITS == 32) {
        store4<float>(static_cast<float*>(t.m) + i, full, left, m);
        store4<float>(static_cast<float*>(t.v) + i, full, left, v);
      }
    }
    if (BITS == 8) {
      peak_m = warp_max_nonneg(peak_m);
      peak_r = warp_max_nonneg(peak_r);
      const bool finite_m = is_finite(peak_m), finite_r = is_finite(peak_r);
      if (!(finite_m && finite_r)) {         // the largest finite magnitudes
        peak_m = peak_r = 0.f;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (is_finite(m1[h][j])) peak_m = fmaxf(peak_m, fabsf(m1[h][j]));
            if (is_finite(root[h][j])) peak_r = fmaxf(peak_r, root[h][j]);
          }
        peak_m = warp_max_nonneg(peak_m);
        peak_r = warp_max_nonneg(peak_r);
      }
      float scale_m, scale_r, inv_m, inv_r;
      if constexpr (PEAK) {
        peak_scale<3>(peak_m, scale_m, inv_m);
        peak_scale<4>(peak_r, scale_r, inv_r);
      } else {
        const uint32_t exp_m = scale_exponent<3>(peak_m), exp_r = scale_exponent<4>(peak_r);
        scale_m = scale_of(exp_m);
        scale_r = scale_of(exp_r);
        inv_m = inverse_scale_of(exp_m);
        inv_r = inverse_scale_of(exp_r);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int64_t i = base + h * 128 + lane * 4;
        uint32_t hash[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) hash[j] = mix32(static_cast<uint32_t>(i) + j + salt, q.two16);
        // behind the tensor's end the codes are those of zero
        *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(t.m) + i) =
            peak_m == 0.f && finite_m ? 0u : encode4<3, PEAK>(m1[h], inv_m, hash, q.two4, finite_m);
        *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(t.v) + i) = peak_r == 0.f && finite_r ? 0u : encode4<4, PEAK>(root[h], inv_r, hash, q.two5, finite_r);
      }
      if (lane == 0) {
        t.m_scale[block] = scale_m;
        t.v_scale[block] = scale_r;
      }
    }
  }

  // the last CTA to finish moves the step on: by then every CTA has read the old one
  if (q.advance) {
    __syncthreads();
    if (threadIdx.x == 0) {
      __threadfence();
      if (atomicAdd(&q.state->ticket, 1u) == gridDim.x - 1) {
        AdamwState s = *q.state;
        s.b1_pow *= q.b1d;
        s.b2_pow *= q.b2d;
        s.step += 1;
        s.inv_bc1 = 1.0 / (1.0 - s.b1_pow * q.b1d);
        s.inv_sqrt_bc2 = static_cast<float>(1.0 / sqrt(1.0 - s.b2_pow * q.b2d));
        s.ticket = 0;
        *q.state = s;
      }
    }
  }
}

// The values that 8-bit moments stand for: m, and v = r^2.  One warp per block of ADAMW_BLOCK elements.
__global__ void __launch_bounds__(256) adamw_moments_kernel(const uint8_t* __restrict__ m, const float* __restrict__ m_scale,
                                                            const uint8_t* __restrict__ r, const float* __restrict__ r_scale,
                                                            float* __restrict__ m_out, float* __restrict__ v_out, int64_t n4) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= n4) return;
  const int64_t block = i / (ADAMW_BLOCK / 4);
  float fm[4], fr[4];
  decode4<3>(reinterpret_cast<const uint32_t*>(m)[i], 1u << 20, fm);
  decode4<4>(reinterpret_cast<const uint32_t*>(r)[i], 1u << 19, fr);
  const float sm = m_scale[block], sr = r_scale[block];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    fm[j] = __fmul_rn(fm[j], sm);
    fr[j] = __fmul_rn(fr[j], sr);
  }
  const float4 a = make_float4(fm[0], fm[1], fm[2], fm[3]);
  const float4 b = make_float4(__fmul_rn(fr[0], fr[0]), __fmul_rn(fr[1], fr[1]), __fmul_rn(fr[2], fr[2]), __fmul_rn(fr[3], fr[3]));
  reinterpret_cast<float4*>(m_out)[i] = a;
  reinterpret_cast<float4*>(v_out)[i] = b;
}

// ---------------------------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------------------------
template <typename P, typename G, bool MASTER, int KIND, int CAP>
static int adamw_launch(const b200k_adamw_tensor* tensors, int n, AdamwParams q, cudaStream_t stream) {
  AdamwTable<CAP> table;
  int used = 0;
  int64_t chunks = 0;
  const int advance = q.advance;
  for (int i = 0; i <= n; ++i) {
    const int64_t more = i < n ? (tensors[i].n + ADAMW_CHUNK - 1) / ADAMW_CHUNK : 0;
    if (i == n || used == CAP || chunks + more > 0x7FFFFFFF) {   // the table is full, or the list ends
      for (int k = used; k <= CAP; ++k) table.first_chunk[k] = static_cast<int>(chunks);
      q.n = used;
      q.advance = i == n ? advance : 0;
      adamw_kernel<P, G, MASTER, KIND, CAP><<<static_cast<unsigned>(chunks), ADAMW_THREADS, 0, stream>>>(table, q);
      count_launch();
      B200K_CHECK_LAUNCH("adamw_kernel");
      if (i == n) break;
      used = 0;
      chunks = 0;
    }
    table.t[used] = tensors[i];
    table.first_chunk[used] = static_cast<int>(chunks);
    chunks += more;
    ++used;
  }
  return B200K_OK;
}

template <typename P, typename G, bool MASTER, int KIND>
static int adamw_table(const b200k_adamw_tensor* t, int n, const AdamwParams& q, cudaStream_t s) {
  return n <= ADAMW_SMALL_TABLE ? adamw_launch<P, G, MASTER, KIND, ADAMW_SMALL_TABLE>(t, n, q, s) : adamw_launch<P, G, MASTER, KIND, ADAMW_LARGE_TABLE>(t, n, q, s);
}
template <typename P, typename G, bool MASTER>
static int adamw_bits(const b200k_adamw_tensor* t, int n, int bits, const AdamwParams& q, cudaStream_t s) {
  if (bits == 32) return adamw_table<P, G, MASTER, 32>(t, n, q, s);
  return bits == 8 ? adamw_table<P, G, MASTER, 8>(t, n, q, s) : adamw_table<P, G, MASTER, 8 + B200K_ADAMW_PEAK_SCALES>(t, n, q, s);
}

template <typename P>
static int adamw_16bit(const b200k_adamw_tensor* t, int n, int gdtype, bool master, int bits, const AdamwParams& q, cudaStream_t s) {
  if (gdtype == B200K_DTYPE_F32) return master ? adamw_bits<P, float, true>(t, n, bits, q, s) : adamw_bits<P, float, false>(t, n, bits, q, s);
  return master ? adamw_bits<P, P, true>(t, n, bits, q, s) : adamw_bits<P, P, false>(t, n, bits, q, s);
}

int adamw(const AdamwArgs& a, cudaStream_t stream) {
  if (a.n <= 0 || a.tensors == nullptr) return set_error(B200K_ERR_INVALID_ARG, "adamw: at least one tensor expected (got %d)", a.n);
  if (a.dtype < B200K_DTYPE_F32 || a.dtype > B200K_DTYPE_F16) return set_error(B200K_ERR_INVALID_ARG, "adamw: bad parameter type %d", a.dtype);
  if (a.gdtype != a.dtype && a.gdtype != B200K_DTYPE_F32)
    return set_error(B200K_ERR_INVALID_ARG, "adamw: gradients have the parameters' type or fp32 (got %d for parameters of type %d)", a.gdtype, a.dtype);
  if (a.state_bits != 8 && a.state_bits != 32 && a.state_bits != 8 + B200K_ADAMW_PEAK_SCALES)
    return set_error(B200K_ERR_INVALID_ARG, "adamw: state_bits must be 8 (+ B200K_ADAMW_PEAK_SCALES) or 32 (got %d)", a.state_bits);
  if (a.state == nullptr || (reinterpret_cast<uintptr_t>(a.state) & 7u)) return set_error(B200K_ERR_INVALID_ARG, "adamw: null or misaligned state");
  if (!(a.beta1 >= 0.0 && a.beta1 < 1.0 && a.beta2 >= 0.0 && a.beta2 < 1.0))
    return set_error(B200K_ERR_INVALID_ARG, "adamw: betas must be in [0, 1) (got %g, %g)", a.beta1, a.beta2);
  if (!(a.eps >= 0.0) || !(a.weight_decay >= 0.0) || (a.lr_dev == nullptr && !(a.lr >= 0.0)))
    return set_error(B200K_ERR_INVALID_ARG, "adamw: lr, eps and weight_decay must be >= 0 (got %g, %g, %g)", a.lr, a.eps, a.weight_decay);
  // the reciprocal takes a subnormal divisor for zero, and eps is all there is of it where v is 0
  if (a.eps > 0.0 && a.eps < 0x1p-126) return set_error(B200K_ERR_INVALID_ARG, "adamw: eps must be 0 or at least 2^-126 (got %g)", a.eps);
  const bool master = a.tensors[0].master != nullptr;
  if (master && a.dtype == B200K_DTYPE_F32) return set_error(B200K_ERR_INVALID_ARG, "adamw: fp32 parameters take no master copy");
  const size_t psize = a.dtype == B200K_DTYPE_F32 ? 4 : 2, gsize = a.gdtype == B200K_DTYPE_F32 ? 4 : 2;
  for (int i = 0; i < a.n; ++i) {
    const b200k_adamw_tensor& t = a.tensors[i];
    if (t.n <= 0 || t.n > (int64_t(1) << 40)) return set_error(B200K_ERR_INVALID_ARG, "adamw: tensor %d has %lld elements", i, (long long)t.n);
    if (t.p == nullptr || t.g == nullptr || t.m == nullptr || t.v == nullptr || (a.state_bits != 32 && (t.m_scale == nullptr || t.v_scale == nullptr)))
      return set_error(B200K_ERR_INVALID_ARG, "adamw: tensor %d has a null pointer", i);
    if ((t.master != nullptr) != master) return set_error(B200K_ERR_INVALID_ARG, "adamw: tensor %d differs in having a master copy", i);
    if ((reinterpret_cast<uintptr_t>(t.p) & (psize - 1)) || (reinterpret_cast<uintptr_t>(t.g) & (gsize - 1)))
      return set_error(B200K_ERR_INVALID_ARG, "adamw: tensor %d is not aligned to its element size", i);
    if ((reinterpret_cast<uintptr_t>(t.m) | reinterpret_cast<uintptr_t>(t.v) | reinterpret_cast<uintptr_t>(t.master)) & 15u)
      return set_error(B200K_ERR_INVALID_ARG, "adamw: moments and master copy of tensor %d must be 16-byte aligned", i);
    if ((reinterpret_cast<uintptr_t>(t.m_scale) | reinterpret_cast<uintptr_t>(t.v_scale)) & 3u)
      return set_error(B200K_ERR_INVALID_ARG, "adamw: scales of tensor %d must be 4-byte aligned", i);
  }
  const DeviceInfo* dev = current_device_info();
  if (dev == nullptr) return B200K_ERR_NO_DEVICE;
  AdamwParams q{};
  q.state = static_cast<AdamwState*>(a.state);
  q.lr_dev = a.lr_dev;
  q.grad_scale_dev = a.grad_scale_dev;
  q.lr = a.lr;
  q.weight_decay = a.weight_decay;
  q.b1d = a.beta1;
  q.b2d = a.beta2;
  q.b1 = static_cast<float>(a.beta1);
  q.one_minus_b1 = static_cast<float>(1.0 - a.beta1);
  q.b2 = static_cast<float>(a.beta2);
  q.one_minus_b2 = static_cast<float>(1.0 - a.beta2);
  q.eps = static_cast<float>(a.eps);
  q.grad_scale = a.grad_scale;
  q.seed = a.seed;
  q.two4 = 1u << 4;
  q.two5 = 1u << 5;
  q.two16 = 1u << 16;
  q.two19 = 1u << 19;
  q.two20 = 1u << 20;
  q.advance = a.advance;
  if (a.dtype == B200K_DTYPE_F32) return adamw_bits<float, float, false>(a.tensors, a.n, a.state_bits, q, stream);
  if (a.dtype == B200K_DTYPE_BF16) return adamw_16bit<__nv_bfloat16>(a.tensors, a.n, a.gdtype, master, a.state_bits, q, stream);
  return adamw_16bit<__half>(a.tensors, a.n, a.gdtype, master, a.state_bits, q, stream);
}

int adamw_moments(const uint8_t* m, const float* m_scale, const uint8_t* r, const float* r_scale, float* m_out, float* v_out, int64_t blocks,
                  cudaStream_t stream) {
  if (blocks < 0 || blocks > (int64_t(1) << 32)) return set_error(B200K_ERR_INVALID_ARG, "adamw_moments: %lld blocks", (long long)blocks);
  if (blocks == 0) return B200K_OK;
  if (m == nullptr || m_scale == nullptr || r == nullptr || r_scale == nullptr || m_out == nullptr || v_out == nullptr)
    return set_error(B200K_ERR_INVALID_ARG, "adamw_moments: null pointer");
  if ((reinterpret_cast<uintptr_t>(m) | reinterpret_cast<uintptr_t>(r)) & 3u || (reinterpret_cast<uintptr_t>(m_out) | reinterpret_cast<uintptr_t>(v_out)) & 15u)
    return set_error(B200K_ERR_INVALID_ARG, "adamw_moments: codes must be 4-byte and outputs 16-byte aligned");
  const DeviceInfo* dev = current_device_info();
  if (dev == nullptr) return B200K_ERR_NO_DEVICE;
  const int64_t n4 = blocks * (ADAMW_BLOCK / 4);
  adamw_moments_kernel<<<static_cast<unsigned>((n4 + 255) / 256), 256, 0, stream>>>(m, m_scale, r, r_scale, m_out, v_out, n4);
  count_launch();
  B200K_CHECK_LAUNCH("adamw_moments_kernel");
  return B200K_OK;
}

}  // namespace b200k
