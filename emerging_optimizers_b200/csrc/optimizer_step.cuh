// Elementwise optimizer operators over lists of tensors: the AdamW step with fp32 or 8-bit states, the global gradient
// norm with clipping, and the block quantiser of the 8-bit states.
//
// A list travels as a table in the kernel parameters (no device-side table, no copy, safe under stream capture).  The
// elements of all tensors are cut into chunks, one CTA per chunk; a CTA finds its tensor by bisection over the first
// chunk of every tensor.  A warp takes 256 consecutive elements at a time, eight per lane:
//   - aligned, whole runs: lane l holds elements 8 l .. 8 l + 7 and moves them with 32-byte accesses (fp32), 16-byte
//     (16-bit types) or 8-byte ones (codes);
//   - otherwise (unaligned pointers, the end of a tensor): lane l holds elements l, l + 32, ... with guarded scalar
//     accesses, still coalesced.
// 256 elements are also one block of an 8-bit state, so a block's largest magnitude is one warp reduction.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

namespace eo {

constexpr int kOptThreads = 256;
constexpr int kOptRun = 256;                                  // elements a warp takes at a time; block of an 8-bit state
constexpr int kOptTrip = kOptThreads / 32 * kOptRun;          // elements a CTA takes per trip
// Tensors per launch: the large table fills the 32 KB that a launch may carry, and carrying it costs the host 4 us more
// than the 2 KB of the small one (24 tensors 8.8 us a call, 25 tensors 12.7 us).
constexpr int kOptSmallTable = 24, kOptLargeTable = 384;

// ---- memory access ---------------------------------------------------------------------------------------------------
// A lane's eight elements of a run as they lie in memory.  get / put: elements 8 l .. 8 l + 7 from their own address (plus
// kOffset elements, an immediate), one wide access; get_some / put_some: elements l, l + 32, ... of the run at `p`, guarded by
// `left` (elements beyond the end read as zero and are not written).

template <int kBytes>
__device__ __forceinline__ uint4 load_16(const void* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4+%5];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p), "n"(kBytes));
  return v;
}
template <int kBytes>
__device__ __forceinline__ uint2 load_8(const void* p) {
  uint2 v;
  asm volatile("ld.global.L1::no_allocate.v2.u32 {%0,%1}, [%2+%3];" : "=r"(v.x), "=r"(v.y) : "l"(p), "n"(kBytes));
  return v;
}

template <typename T>
struct Run;

template <>
struct __align__(16) Run<float> {
  float x[8];
  template <int kOffset = 0>
  __device__ __forceinline__ void get(const float* p) {
    asm volatile("ld.global.L1::no_allocate.v8.f32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8+%9];"
                 : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3]), "=f"(x[4]), "=f"(x[5]), "=f"(x[6]), "=f"(x[7])
                 : "l"(p), "n"(4 * kOffset));
  }
  __device__ __forceinline__ void put(float* p) const {
    asm volatile("st.global.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "f"(x[0]), "f"(x[1]), "f"(x[2]), "f"(x[3]),
                 "f"(x[4]), "f"(x[5]), "f"(x[6]), "f"(x[7])
                 : "memory");
  }
  // as put, for addresses aligned to 16 bytes only
  __device__ __forceinline__ void put_halves(float* p) const {
    reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
  }
  __device__ __forceinline__ void get_some(const float* p, long long left, int lane) {
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = (32 * k + lane < left) ? p[32 * k + lane] : 0.0f;
  }
  __device__ __forceinline__ void put_some(float* p, long long left, int lane) const {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (32 * k + lane < left) p[32 * k + lane] = x[k];
  }
  __device__ __forceinline__ void unpack(float2 (&out)[4]) const {
#pragma unroll
    for (int k = 0; k < 4; ++k) out[k] = make_float2(x[2 * k], x[2 * k + 1]);
  }
  __device__ __forceinline__ void pack(const float2 (&in)[4]) {
#pragma unroll
    for (int k = 0; k < 4; ++k) x[2 * k] = in[k].x, x[2 * k + 1] = in[k].y;
  }
};

template <typename T>
struct __align__(16) Run16 {  // eight 16-bit elements, element k in half k % 2 of word k / 2
  uint32_t w[4];
  template <int kOffset = 0>
  __device__ __forceinline__ void get(const T* p) {
    const uint4 v = load_16<2 * kOffset>(p);
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
  }
  __device__ __forceinline__ void put(T* p) const { *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]); }
  __device__ __forceinline__ void get_some(const T* base, long long left, int lane) {
    const uint16_t* p = reinterpret_cast<const uint16_t*>(base);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const uint32_t h = (32 * k + lane < left) ? p[32 * k + lane] : 0u;
      w[k / 2] = k % 2 == 0 ? h : w[k / 2] | (h << 16);
    }
  }
  __device__ __forceinline__ void put_some(T* base, long long left, int lane) const {
    uint16_t* p = reinterpret_cast<uint16_t*>(base);
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (32 * k + lane < left) p[32 * k + lane] = static_cast<uint16_t>(w[k / 2] >> (16 * (k % 2)));
  }
};

template <>
struct Run<int16_t> : Run16<int16_t> {};

template <>
struct Run<__nv_bfloat16> : Run16<__nv_bfloat16> {
  __device__ __forceinline__ void unpack(float2 (&out)[4]) const {
#pragma unroll
    for (int k = 0; k < 4; ++k) out[k] = make_float2(__uint_as_float(w[k] << 16), __uint_as_float(w[k] & 0xffff0000u));
  }
  __device__ __forceinline__ void pack(const float2 (&in)[4]) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const __nv_bfloat162 h = __float22bfloat162_rn(in[k]);
      w[k] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
};

template <>
struct __align__(8) Run<uint8_t> {  // element k in byte k % 4 of word k / 4
  uint32_t w[2];
  template <int kOffset = 0>
  __device__ __forceinline__ void get(const uint8_t* p) {
    const uint2 v = load_8<kOffset>(p);
    w[0] = v.x, w[1] = v.y;
  }
  __device__ __forceinline__ void put(uint8_t* p) const { *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]); }
  __device__ __forceinline__ void get_some(const uint8_t* p, long long left, int lane) {
    w[0] = w[1] = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (32 * k + lane < left) w[k / 4] |= static_cast<uint32_t>(p[32 * k + lane]) << (8 * (k % 4));
  }
  __device__ __forceinline__ void put_some(uint8_t* p, long long left, int lane) const {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (32 * k + lane < left) p[32 * k + lane] = static_cast<uint8_t>(w[k / 4] >> (8 * (k % 4)));
  }
};

// Two fp32 operations in one instruction, each rounded to nearest.
#define EO_PAIR_2(name, op)                                                                                               \
  __device__ __forceinline__ float2 name(float2 a, float2 b) {                                                             \
    float2 d;                                                                                                              \
    asm("{.reg .b64 a, b, d; mov.b64 a, {%2, %3}; mov.b64 b, {%4, %5}; " op ".rn.f32x2 d, a, b; mov.b64 {%0, %1}, d;}"      \
        : "=f"(d.x), "=f"(d.y)                                                                                             \
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));                                                                         \
    return d;                                                                                                              \
  }
EO_PAIR_2(mul2, "mul")
EO_PAIR_2(add2, "add")
#undef EO_PAIR_2
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{.reg .b64 a, b, c, d; mov.b64 a, {%2, %3}; mov.b64 b, {%4, %5}; mov.b64 c, {%6, %7}; "
      "fma.rn.f32x2 d, a, b, c; mov.b64 {%0, %1}, d;}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }
// a * b, rounded before anything is done with it: the assembler fuses a paired multiplication with a following addition, but not
// a fused one whose addend it does not know.  minus_zero: -0, from a kernel parameter.
__device__ __forceinline__ float2 product(float2 a, float2 b, float2 minus_zero) { return fma2(a, b, minus_zero); }

// bf16 weights whose fp32 master is kept as bf16 plus a signed 16-bit remainder: master bits = (bf16 bits << 16) +
// remainder.  Written back as the nearest bf16 (halves away from zero, so that the remainder fits 16 bits); a NaN
// becomes the quiet NaN with remainder zero, as adding to its payload could wrap.
// A weight that somebody set to zero since (a mask, a padding row) may still have a negative remainder, which no split leaves beside
// a zero and which would borrow from the sign: it is zero then.
__device__ __forceinline__ void join_masters(const Run<__nv_bfloat16>& hi, const Run<int16_t>& lo, float2 (&out)[4]) {
  uint32_t zeros = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    zeros |= ((hi.w[k] & 0x7fff7fffu) - 0x00010001u) & 0x80008000u;
    out[k].x = __uint_as_float((hi.w[k] << 16) + static_cast<uint32_t>(static_cast<int32_t>(lo.w[k] << 16) >> 16));
    out[k].y = __uint_as_float((hi.w[k] & 0xffff0000u) + static_cast<uint32_t>(static_cast<int32_t>(lo.w[k]) >> 16));
  }
  if (zeros != 0) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if ((hi.w[k] & 0x7fffu) == 0 && (lo.w[k] & 0x8000u)) out[k].x = 0.0f;
      if ((hi.w[k] & 0x7fff0000u) == 0 && (lo.w[k] & 0x80000000u)) out[k].y = 0.0f;
    }
  }
}
__device__ __forceinline__ void split_masters(const float2 (&x)[4], Run<__nv_bfloat16>& hi, Run<int16_t>& lo) {
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    // a NaN as 0x7fc00000: rounding leaves it, its low half is zero
    const uint32_t a = x[k].x != x[k].x ? 0x7fc00000u : __float_as_uint(x[k].x);
    const uint32_t b = x[k].y != x[k].y ? 0x7fc00000u : __float_as_uint(x[k].y);
    hi.w[k] = __byte_perm(a + 0x8000u, b + 0x8000u, 0x7632);
    lo.w[k] = __byte_perm(a, b, 0x5410);  // bits - (hi << 16), modulo 2^16
  }
}

// ---- 8-bit block-scaled numbers ---------------------------------------------------------------------------------------
// A block of 256 elements shares one byte, the exponent field E of its largest finite magnitude (at least 1).  A code is
// a small float, its bits those of an fp32 number shifted right by 20:
//   signed   (first moments):  sign, 4 exponent bits, 3 mantissa bits; down to 2^-16 of the block's power of two
//   unsigned (second moments):       5 exponent bits, 3 mantissa bits; down to 2^-32
//   value = f32(code << 20) * 2^kShift * 2^(E - 127),    code = (bits(|x| * 2^(127 - E) * 2^-kShift) + d) >> 20,
//   kShift = 113 and 97,
// so the block's largest magnitude has exponent field 14 (of 15) or 30 (of 31): rounding up never leaves the format, and
// values lie exactly in bf16 and fp32 because the scale is a power of two.  The second moment itself is stored, not its
// root: decoding needs no multiplication and rounding is unbiased in what the moving average averages.
// d = 16 r + 8 with 16 random bits r rounds up with the probability of the part cut off; d = 2^19 rounds to nearest.
// Blocks that reach 2^127 are rounded towards zero (d = 0): above them fp32 has only infinity.
// Why random: a moving average in a format with 3 mantissa bits stands still under rounding to nearest as soon as one
// step moves it by less than half a unit.  Simulated with Gaussian gradients that fall tenfold, the root of the second
// moment stays 10 (beta2 = 0.95 and 0.99) or 4.6 (0.999) times too large with rounding to nearest; with random rounding
// its mean is within 1 % and its spread 7 - 13 %.
// An unsigned value above zero never becomes code 0: it divides.  What is not finite (unsigned: or is negative) becomes
// the code with all exponent and mantissa bits set, which no finite value reaches, and reads as NaN.
//
// What this costs decides the speed of the 8-bit step, and the integer pipe has half the rate of the floating-point one:
// everything an element needs is a multiplication or an add, except the byte moves.  What is not finite is looked for
// once per block, in the maximum that the exponent needs anyway, and dealt with off the common path.
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
template <bool kSigned>
struct Code8 {
  static constexpr int kTop = kSigned ? 14 : 30;
  static constexpr uint32_t kNan = kSigned ? 0x7f : 0xff;
  static __device__ __forceinline__ float down() { return __uint_as_float(static_cast<uint32_t>(kTop) << 23); }  // 2^-kShift

  static __device__ __forceinline__ void decode(const Run<uint8_t>& codes, uint32_t exponent, float2 (&out)[4]) {
    if constexpr (kSigned) {
      // The bits are those of e4m3 (sign, 4 exponent, 3 mantissa bits, 0x7f NaN), 2^7 times as large.
      const float2 scale = both(__uint_as_float(exponent << 23) * 0x1p-7f);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        uint32_t h2;
        const uint16_t two = static_cast<uint16_t>(codes.w[k / 2] >> (16 * (k % 2)));
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"(two));
        out[k] = mul2(__half22float2(*reinterpret_cast<const __half2*>(&h2)), scale);
      }
    } else {
      // 2^97 * 2^(E - 127), in two steps where it leaves the fp32 range
      const float2 scale = both(__uint_as_float((min(exponent, 157u) + 97u) << 23));
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t w = codes.w[k / 2];
        // the byte at bit 16, times 2^4
        const uint32_t a = __byte_perm(w, 0, 0x4044 | (2 * (k % 2)) << 8) * 16u;
        const uint32_t b = __byte_perm(w, 0, 0x4044 | (2 * (k % 2) + 1) << 8) * 16u;
        out[k] = mul2(make_float2(__uint_as_float(a), __uint_as_float(b)), scale);
      }
      if (exponent > 157u) {
#pragma unroll
        for (int k = 0; k < 4; ++k) out[k] = mul2(out[k], both(__uint_as_float((exponent - 30u) << 23)));
      }
      const uint32_t nans = ((~codes.w[0] - 0x01010101u) & codes.w[0]) | ((~codes.w[1] - 0x01010101u) & codes.w[1]);
      if (nans & 0x80808080u) {  // a byte is 0xff
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t two = codes.w[k / 2] >> (16 * (k % 2));
          if ((two & 0xffu) == kNan) out[k].x = __uint_as_float(0x7fc00000u);
          if (((two >> 8) & 0xffu) == kNan) out[k].y = __uint_as_float(0x7fc00000u);
        }
      }
    }
  }

  // Largest magnitude of the block as fp32 bits; at least those of infinity where something is not a number to be kept.
  static __device__ __forceinline__ uint32_t block_top(const float2 (&in)[4]) {
    const float x[8] = {in[0].x, in[0].y, in[1].x, in[1].y, in[2].x, in[2].y, in[3].x, in[3].y};
    uint32_t top;
    if constexpr (kSigned) {
      const float a = max3_nan(fabsf(x[0]), fabsf(x[1]), fabsf(x[2])), b = max3_nan(fabsf(x[3]), fabsf(x[4]), fabsf(x[5]));
      top = __float_as_uint(max3_nan(max3_nan(a, fabsf(x[6]), fabsf(x[7])), b, b));
    } else {
      const uint32_t a = __vimax3_u32(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]));
      const uint32_t b = __vimax3_u32(__float_as_uint(x[3]), __float_as_uint(x[4]), __float_as_uint(x[5]));
      top = max(__vimax3_u32(a, __float_as_uint(x[6]), __float_as_uint(x[7])), b);
    }
    return __reduce_max_sync(0xffffffffu, top);
  }
  static __device__ __forceinline__ bool is_kept(float x) {
    const uint32_t b = __float_as_uint(x);
    return (kSigned ? (b & 0x7fffffffu) : b) < 0x7f800000u;
  }

  // Whether a block with this top takes the rare path: beyond what one factor reaches (2^14 for first, 2^30 for second moments),
  // infinity, NaN; unsigned: a negative number.
  static __device__ __forceinline__ bool is_rare(uint32_t top) { return top >= static_cast<uint32_t>(127 + kTop) << 23; }

  // Exponent byte and codes of a block; d16[k]: 16 d of each element; top: of block_top.  kRare is right for every block, the other
  // one where is_rare(top) is false.
  template <bool kRare>
  static __device__ __forceinline__ uint32_t encode(const float2 (&in)[4], uint32_t top, const uint32_t (&d16)[8],
                                                    Run<uint8_t>& codes) {
    const float x[8] = {in[0].x, in[0].y, in[1].x, in[1].y, in[2].x, in[2].y, in[3].x, in[3].y};
    if constexpr (kRare) {
      uint32_t mine = 0;
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (is_kept(x[k])) mine = max(mine, __float_as_uint(x[k]) & 0x7fffffffu);
      top = __reduce_max_sync(0xffffffffu, mine);
    }
    const uint32_t e = max(top >> 23, 1u);
    uint32_t t[8];  // 16 (bits + d) has the code in its top byte; the sign, if any, is shifted out
    if constexpr (kRare) {
      const float inv = __uint_as_float(max((254u - e) << 23, 0x00400000u));  // 2^(127 - e); subnormal for e = 254
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float y = __fmul_rn(__fmul_rn(x[k], inv), down());
        t[k] = __float_as_uint(y) * 16u + (e == 254u ? 0u : d16[k]);  // towards zero in the last binade
        if (!kSigned && x[k] > 0.0f) t[k] = max(t[k], 1u << 24);
        if (!is_kept(x[k])) t[k] = (!kSigned && __float_as_uint(x[k]) == 0x80000000u) ? 0u : kNan << 24;  // -0 is kept as 0
      }
    } else {
      const float2 factor = both(__uint_as_float((127u + kTop - e) << 23));  // 2^(127 - E) * 2^-kShift
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 y = mul2(in[k], factor);
        t[2 * k] = __float_as_uint(y.x) * 16u + d16[2 * k];
        t[2 * k + 1] = __float_as_uint(y.y) * 16u + d16[2 * k + 1];
        if constexpr (!kSigned) {
          if (in[k].x > 0.0f) t[2 * k] = max(t[2 * k], 1u << 24);
          if (in[k].y > 0.0f) t[2 * k + 1] = max(t[2 * k + 1], 1u << 24);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      uint32_t w = __byte_perm(__byte_perm(t[4 * j], t[4 * j + 1], 0x0073),
                               __byte_perm(t[4 * j + 2], t[4 * j + 3], 0x0073), 0x5410);
      if constexpr (kSigned) {
        const uint32_t signs = __byte_perm(
            __byte_perm(__float_as_uint(x[4 * j]), __float_as_uint(x[4 * j + 1]), 0x0073),
            __byte_perm(__float_as_uint(x[4 * j + 2]), __float_as_uint(x[4 * j + 3]), 0x0073), 0x5410);
        w = (w & 0x7f7f7f7fu) | (signs & 0x80808080u);
      }
      codes.w[j] = w;
    }
    return e;
  }
};

// The finaliser of MurmurHash3: 32 random bits of an element from mix(key ^ element), key from (seed, tensor, step).
__host__ __device__ __forceinline__ uint32_t mix32(uint32_t x) {
  x = (x ^ (x >> 16)) * 0x85ebca6bu;
  x = (x ^ (x >> 13)) * 0xc2b2ae35u;
  return x ^ (x >> 16);
}
__host__ __device__ __forceinline__ uint32_t rounding_key(uint32_t seed, uint32_t tensor, uint32_t step) {
  return mix32(mix32(mix32(seed) ^ tensor) ^ step);
}
// 16 d = 256 r + 128 of a lane's eight elements, r the low (first moments) and the high half (second moments) of
// mix32(key ^ element); `first`: the lane's first element.  Elements of a lane differ in bits below 16 only, which the first
// step of the mixer leaves alone, so that step is done once; its last one is the exclusive or of the halves.
template <bool kVec>
__device__ __forceinline__ void random_dither(uint32_t key, uint32_t first, uint32_t (&low)[8], uint32_t (&high)[8]) {
  first ^= key;
  first ^= first >> 16;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    uint32_t x = (first ^ static_cast<uint32_t>(kVec ? k : 32 * k)) * 0x85ebca6bu;
    x = (x ^ (x >> 13)) * 0xc2b2ae35u;
    high[k] = __byte_perm(x, 0x80u, 0x5324);                // 0, the high half, 0x80
    low[k] = __byte_perm(x, 0x80u, 0x5105) ^ high[k];       // 0, the halves' exclusive or, 0x80
  }
}

// ---- tables -----------------------------------------------------------------------------------------------------------

template <typename Entry, int kCapacity>
struct TensorTable {
  int n;
  int trips;  // trips of kOptTrip elements per chunk
  uint32_t first[kCapacity];  // first chunk of each tensor
  Entry t[kCapacity];
};

template <typename Table>
__device__ __forceinline__ int find_tensor(const Table& table, uint32_t chunk) {
  int lo = 0, hi = table.n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (table.first[mid] <= chunk) lo = mid; else hi = mid;
  }
  return lo;
}

// ---- AdamW ------------------------------------------------------------------------------------------------------------

struct AdamWEntry {
  void* p;
  const void* g;
  void* m;
  void* v;
  uint8_t* me;  // exponent bytes of 8-bit states
  uint8_t* ve;
  int16_t* r;   // remainders of bf16 weights, or nullptr
  const long long* step;  // step counter in device memory, or nullptr
  long long numel;
  uint32_t index;  // place in the caller's list (random rounding)
  uint32_t vec;    // every pointer is aligned for the wide accesses
};

struct AdamWFactors {
  float decay, step_size, inv_root_bc2;
  uint32_t step;
};

struct AdamWScalars {
  float beta1, one_minus_beta1, beta2, one_minus_beta2, eps, l2, minus_zero;
  float root_scale, root_unscale;  // the root is taken of -root_scale v and multiplied by root_unscale
  uint32_t seed;
  AdamWFactors f;             // used when dev_factors is nullptr
  const AdamWFactors* dev_factors;  // per tensor of this launch, from adamw_factors_kernel
  const float* grad_scale;    // device scalar, or nullptr
};

enum { kDecayDecoupled = 0, kDecayIndependent = 1, kDecayPalm = 2, kDecayL2 = 3 };

// Factors of step t in float64: 1 - beta^t loses its digits in fp32.
__host__ __device__ inline AdamWFactors adamw_factors(double lr, double beta1, double beta2, double weight_decay, int method,
                                                      long long t) {
  AdamWFactors f;
  f.decay = static_cast<float>(method == kDecayDecoupled    ? 1.0 - lr * weight_decay
                               : method == kDecayIndependent ? 1.0 - weight_decay
                               : method == kDecayPalm        ? 1.0 - lr * lr * weight_decay
                                                             : 1.0);
  f.step_size = static_cast<float>(lr / (1.0 - pow(beta1, static_cast<double>(t))));
  f.inv_root_bc2 = static_cast<float>(1.0 / sqrt(1.0 - pow(beta2, static_cast<double>(t))));
  f.step = static_cast<uint32_t>(t);
  return f;
}

template <int kCapacity>
__global__ void __launch_bounds__(128)
    adamw_factors_kernel(const __grid_constant__ TensorTable<AdamWEntry, kCapacity> table, double lr, const float* dev_lr,
                         double beta1, double beta2, double weight_decay, int method, long long step,
                         AdamWFactors* __restrict__ out) {
  if (dev_lr != nullptr) lr = static_cast<double>(*dev_lr);
  for (int i = threadIdx.x; i < table.n; i += blockDim.x)
    out[i] = adamw_factors(lr, beta1, beta2, weight_decay, method, table.t[i].step != nullptr ? *table.t[i].step : step);
}

__device__ __forceinline__ float rsqrt_approx(float x) {
  float y;
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// g, p, m, v of one lane, two elements to an instruction.  Every operation is rounded once, in this order, so that the result
// does not depend on how the compiler would contract it (the 8-bit codes of a run must not depend on the build).
//
// Root and quotient are rounded to nearest too, without the branches and the range checks of the compiler's, which run the
// eight elements of a lane one after the other: one Newton step each on the hardware's approximations, its residual exact
// through the fused multiply-add (Markstein, IBM J. Res. Dev. 34, 1990).  Compared with __fsqrt_rn on every positive float: the
// same where the operand is at least 2^-102; with __fdiv_rn on 3.4e10 pairs of mantissas: the same, and the reciprocal inside is
// the nearest for every mantissa.  Below 2^-102 a root does not count beside an eps of 1e-10 and more.  Where eps is smaller the
// root is taken of 2^36 v: right within three roundings down to the smallest subnormal v (the 2^-126 that keeps the
// approximation of zero finite is 2^-13 of it then, and the Newton step squares that).  Zero gives zero.  Negated operands (-v,
// -root, -denominator) save the sign changes that the paired instructions do not have.
__device__ __forceinline__ float2 adamw_quotient(float2 m, float2 v, float root_scale, float2 inv, float2 minus_eps, float2 mz) {
  const float2 nv = mul2(v, both(root_scale));
  const float2 above_zero = add2(nv, both(-0x1p-126f));
  const float2 y = make_float2(rsqrt_approx(-above_zero.x), rsqrt_approx(-above_zero.y));
  float2 nroot = product(nv, y, mz);
  nroot = fma2(fma2(nroot, nroot, nv), mul2(y, both(0.5f)), nroot);
  const float2 nd = add2(product(nroot, inv, mz), minus_eps);
  float2 z = make_float2(rcp_approx(-nd.x), rcp_approx(-nd.y));
  z = fma2(z, fma2(nd, z, both(1.0f)), z);
  const float2 q = product(m, z, mz);
  return fma2(fma2(nd, q, m), z, q);
}

__device__ __forceinline__ void adamw_moments(const float2 (&p)[4], const float2 (&g_in)[4], float2 (&m)[4], float2 (&v)[4],
                                              const AdamWScalars& c, float grad_scale) {
  const float2 scale = both(grad_scale), b1 = both(c.beta1), ob1 = both(c.one_minus_beta1), b2 = both(c.beta2);
  const float2 ob2 = both(c.one_minus_beta2), l2 = both(c.l2), mz = both(c.minus_zero);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    float2 g = product(g_in[k], scale, mz);
    if (c.l2 != 0.0f) g = add2(g, product(p[k], l2, mz));
    m[k] = add2(product(m[k], b1, mz), product(g, ob1, mz));
    v[k] = add2(product(v[k], b2, mz), product(product(g, g, mz), ob2, mz));
  }
}

// The Newton steps make NaN of an infinite operand.  kLarge: one of the lane's second moments may be infinite, or its 2^36-fold where
// that is what the root is taken of.  The latter are taken as they are then, and an infinite one gives the quotient zero (NaN
// with an infinite first moment), as dividing by its root does.  Which of the two it is is decided for all of a lane at once, from
// the largest of its second moments; with 8-bit states from the block's maximum, which the rounding needs anyway.
template <bool kLarge>
__device__ __forceinline__ void adamw_apply(float2 (&p)[4], const float2 (&m)[4], const float2 (&v)[4], const AdamWScalars& c,
                                            const AdamWFactors& f) {
  const float2 eps = both(-c.eps), decay = both(f.decay), size = both(-f.step_size), mz = both(c.minus_zero);
  const float2 inv = both(f.inv_root_bc2 * c.root_unscale);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    float2 q = adamw_quotient(m[k], v[k], c.root_scale, inv, eps, mz);
    if constexpr (kLarge) {
      const float infinity = __uint_as_float(0x7f800000u), up = -c.root_scale;
      const float2 plain = adamw_quotient(m[k], v[k], -1.0f, both(f.inv_root_bc2), eps, mz);
      if (!(v[k].x * up < infinity)) q.x = v[k].x == infinity ? __fmul_rn(m[k].x, 0.0f) : plain.x;
      if (!(v[k].y * up < infinity)) q.y = v[k].y == infinity ? __fmul_rn(m[k].y, 0.0f) : plain.y;
    }
    p[k] = add2(product(p[k], decay, mz), product(q, size, mz));
  }
}

// Largest of a lane's second moments; NaN where one of them is.
__device__ __forceinline__ float largest(const float2 (&v)[4]) {
  return max3_nan(max3_nan(v[0].x, v[0].y, v[1].x), max3_nan(v[1].y, v[2].x, v[2].y), max3_nan(v[3].x, v[3].y, v[3].y));
}

// The eight elements of a lane: parameters, gradients, moments as they lie in memory.
template <typename P, typename G, bool kRemainder, bool k8>
struct AdamWRun {
  using Moment = typename std::conditional<k8, uint8_t, float>::type;
  Run<P> p;
  Run<G> g;
  Run<Moment> m, v;
  Run<int16_t> r;
  uint32_t me, ve;

  // kVec, first: as the lane's elements lie, and the index of its first one (random rounding).
  template <bool kVec>
  __device__ __forceinline__ void step(const AdamWScalars& c, const AdamWFactors& f, float grad_scale, uint32_t key,
                                       uint32_t first) {
    float2 xp[4], xg[4], xm[4], xv[4];
    g.unpack(xg);
    if constexpr (kRemainder) join_masters(p, r, xp); else p.unpack(xp);
    if constexpr (k8) {
      Code8<true>::decode(m, me, xm);
      Code8<false>::decode(v, ve, xv);
    } else {
      m.unpack(xm);
      v.unpack(xv);
    }
    adamw_moments(xp, xg, xm, xv, c, grad_scale);
    if constexpr (k8) {
      // One branch for both blocks and for the quotient: a block with a large second moment is a rare one too.
      using First = Code8<true>;
      using Second = Code8<false>;
      uint32_t low[8], high[8];
      random_dither<kVec>(key, first, low, high);
      const uint32_t m_top = First::block_top(xm), v_top = Second::block_top(xv);
      if (!(First::is_rare(m_top) || Second::is_rare(v_top))) {
        adamw_apply<false>(xp, xm, xv, c, f);
        me = First::template encode<false>(xm, m_top, low, m);
        ve = Second::template encode<false>(xv, v_top, high, v);
      } else {
        adamw_apply<true>(xp, xm, xv, c, f);
        me = First::template encode<true>(xm, m_top, low, m);
        ve = Second::template encode<true>(xv, v_top, high, v);
      }
    } else {
      if (largest(xv) * -c.root_scale < __uint_as_float(0x7f800000u)) adamw_apply<false>(xp, xm, xv, c, f);
      else adamw_apply<true>(xp, xm, xv, c, f);
      m.pack(xm);
      v.pack(xv);
    }
    if constexpr (kRemainder) split_masters(xp, p, r); else p.pack(xp);
  }
};

// Addresses of a lane's elements in whole, aligned runs; they move on by one trip.
template <typename P, typename G, bool kRemainder>
struct AdamWCursor {
  using Data = AdamWRun<P, G, kRemainder, false>;
  P* p;
  const G* g;
  float *m, *v;
  int16_t* r;
  __device__ __forceinline__ AdamWCursor(const AdamWEntry& t, long long at, int lane)
      : p(static_cast<P*>(t.p) + at + 8 * lane),
        g(static_cast<const G*>(t.g) + at + 8 * lane),
        m(static_cast<float*>(t.m) + at + 8 * lane),
        v(static_cast<float*>(t.v) + at + 8 * lane),
        r(t.r + at + 8 * lane) {}
  __device__ __forceinline__ void get(Data& d) const {
    d.g.get(g);
    d.p.get(p);
    d.m.get(m);
    d.v.get(v);
    if constexpr (kRemainder) d.r.get(r);
  }
  __device__ __forceinline__ void put(const Data& d) const {
    d.p.put(p);
    if constexpr (kRemainder) d.r.put(r);
    d.m.put(m);
    d.v.put(v);
  }
  __device__ __forceinline__ void next() {
    p += kOptTrip, g += kOptTrip, m += kOptTrip, v += kOptTrip;
    if constexpr (kRemainder) r += kOptTrip;
  }
};

// Runs of the 8-bit step on their way through shared memory: a warp's own ring of kRingStages runs, filled by asynchronous
// copies two trips ahead.  Without it the loads wait for the 60 instructions an element that lie between a load and its
// store, and prefetching into registers costs the occupancy it should replace: 268 M fp32 elements 1028 us without, 650 us
// with the ring.  Three stages leave room for three CTAs an SM with fp32 types; four (two CTAs) are 4 % slower under a
// sustained load, two 3 % slower with bf16 gradients.
constexpr int kRingStages = 3;
template <typename P, typename G, bool kRemainder>
struct AdamWRing {
  static constexpr int kP = 0, kG = kP + kOptRun * sizeof(P), kM = kG + kOptRun * sizeof(G), kV = kM + kOptRun,
                       kR = kV + kOptRun, kBytes = kR + (kRemainder ? 2 * kOptRun : 0);
  static constexpr int kWarpBytes = kBytes * kRingStages, kCtaBytes = kWarpBytes * (kOptThreads / 32);
  static constexpr int kAhead = (kRingStages - 1) * kOptTrip;  // elements between the run fetched and the run worked on

  // A lane's addresses in the run to be fetched: it copies other elements than it works on where its eight take 32 bytes.
  const char *p, *g;
  uint8_t *m, *v;
  int16_t* r;
  __device__ __forceinline__ AdamWRing(const AdamWEntry& t, long long at, int lane)
      : p(reinterpret_cast<const char*>(static_cast<const P*>(t.p) + at) + 16 * lane),
        g(reinterpret_cast<const char*>(static_cast<const G*>(t.g) + at) + 16 * lane),
        m(static_cast<uint8_t*>(t.m) + at + 8 * lane),
        v(static_cast<uint8_t*>(t.v) + at + 8 * lane),
        r(t.r + at + 8 * lane) {}

  template <int kRunBytes>
  static __device__ __forceinline__ void copy(uint32_t to, const void* from) {
    if constexpr (kRunBytes == 256) {
      asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(to), "l"(from) : "memory");
    } else {
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
      if constexpr (kRunBytes == 1024)
        asm volatile("cp.async.cg.shared.global [%0+512], [%1+512], 16;" ::"r"(to), "l"(from) : "memory");
    }
  }
  // stage: shared address of the stage, plus 8 lane
  __device__ __forceinline__ void fetch(uint32_t stage, int lane) const {
    copy<kOptRun * sizeof(P)>(stage + 8 * lane + kP, p);
    copy<kOptRun * sizeof(G)>(stage + 8 * lane + kG, g);
    copy<kOptRun>(stage + kM, m);
    copy<kOptRun>(stage + kV, v);
    if constexpr (kRemainder) copy<kOptRun * 2>(stage + 8 * lane + kR, r);
  }
  __device__ __forceinline__ void next() {
    p += kOptTrip * sizeof(P), g += kOptTrip * sizeof(G), m += kOptTrip, v += kOptTrip;
    if constexpr (kRemainder) r += kOptTrip;
  }
  static __device__ __forceinline__ void read(const char* stage, int lane, AdamWRun<P, G, kRemainder, true>& d) {
    d.p = reinterpret_cast<const Run<P>*>(stage + kP)[lane];
    d.g = reinterpret_cast<const Run<G>*>(stage + kG)[lane];
    d.m = reinterpret_cast<const Run<uint8_t>*>(stage + kM)[lane];
    d.v = reinterpret_cast<const Run<uint8_t>*>(stage + kV)[lane];
    if constexpr (kRemainder) d.r = reinterpret_cast<const Run<int16_t>*>(stage + kR)[lane];
  }
  // The run worked on lies kAhead elements before the one to be fetched.
  __device__ __forceinline__ void put(const AdamWRun<P, G, kRemainder, true>& d, int lane) const {
    if constexpr (sizeof(P) == 4)
      d.p.put_halves(reinterpret_cast<P*>(const_cast<char*>(p) + 16 * lane) - kAhead);
    else
      d.p.put(reinterpret_cast<P*>(const_cast<char*>(p)) - kAhead);
    if constexpr (kRemainder) d.r.put(r - kAhead);
    d.m.put(m - kAhead);
    d.v.put(v - kAhead);
  }
};

// kRemainder: p is bf16 with remainders.  k8: m and v are codes with exponent bytes.
// fp32 moments: bound by HBM.  268 M elements: fp32 types 1.13 ms (28 bytes an element, 6.65 TB/s), bf16 gradients 1.06 ms
// (6.6), bf16 weights 0.98 ms (6.6), both bf16 0.91 ms (6.5), with remainders 1.08 ms (6.4).
// 8-bit moments: 58 to 60 instructions an element for its 10 to 16 bytes.  fp32 types 0.65 ms (6.6 TB/s), bf16 gradients 0.58 ms (6.5),
// bf16 weights 0.54 ms (6.0), both bf16 0.54 ms (4.9), with remainders 0.61 ms (6.1): bf16 is bound by the issue slots (79 % used,
// the pipe of the integer multiplications 74 %).  These are bursts; run without a pause the 8-bit step reaches the GPU's power limit
// and its clock falls from 1.97 to 1.6 GHz (fp32 types 0.70 ms, bf16 0.59), while the step with fp32 moments does not slow down.
// Three CTAs an SM (80 registers): two are 6 - 12 % slower with bf16 types, four spill.
template <typename P, typename G, bool kRemainder, bool k8, int kCapacity>
__global__ void __launch_bounds__(kOptThreads, 3)
    adamw_kernel(const __grid_constant__ TensorTable<AdamWEntry, kCapacity> table, const __grid_constant__ AdamWScalars c) {
  using Data = AdamWRun<P, G, kRemainder, k8>;
  using Moment = typename Data::Moment;
  const int which = find_tensor(table, blockIdx.x);
  const AdamWEntry& t = table.t[which];
  const AdamWFactors f = c.dev_factors != nullptr ? c.dev_factors[which] : c.f;
  const float grad_scale = c.grad_scale != nullptr ? *c.grad_scale : 1.0f;
  const uint32_t key = k8 ? rounding_key(c.seed, t.index, f.step) : 0u;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long begin = static_cast<long long>(blockIdx.x - table.first[which]) * table.trips * kOptTrip;
  const long long end = min(begin + static_cast<long long>(table.trips) * kOptTrip, t.numel);
  long long at = begin + warp * kOptRun;
  if (t.vec) {
    const int whole = end - at >= kOptRun ? static_cast<int>((end - at - kOptRun) / kOptTrip) + 1 : 0;
    Data data;
    if constexpr (k8) {
      using Ring = AdamWRing<P, G, kRemainder>;
      extern __shared__ __align__(16) char ring_bytes[];
      const char* const stages = ring_bytes + warp * Ring::kWarpBytes;
      const uint32_t stages_at = static_cast<uint32_t>(__cvta_generic_to_shared(stages)) + 8 * lane;
      Ring ring(t, at, lane);
      uint8_t *me = t.me + at / kOptRun, *ve = t.ve + at / kOptRun;
      uint32_t mes = 0, ves = 0;  // lane l: the exponents of the warp's run l, of 32 at a time
#pragma unroll
      for (int i = 0; i < kRingStages - 1; ++i) {
        if (i < whole) ring.fetch(stages_at + i * Ring::kBytes, lane);
        asm volatile("cp.async.commit_group;" ::: "memory");
        ring.next();
      }
      int stage = 0;  // byte offset of the run worked on
      uint32_t first = static_cast<uint32_t>(at) + 8 * lane;
      for (int i = 0; i < whole; ++i) {
        if ((i & 31) == 0 && i + lane < whole) {
          mes = me[(i + lane) * (kOptTrip / kOptRun)];
          ves = ve[(i + lane) * (kOptTrip / kOptRun)];
        }
        asm volatile("cp.async.wait_group %0;" ::"n"(kRingStages - 2) : "memory");
        __syncwarp();  // the run is there for all lanes, and all of them have read the one whose place is filled next
        Ring::read(stages + stage, lane, data);
        if (i + kRingStages - 1 < whole) ring.fetch(stages_at + (stage == 0 ? Ring::kWarpBytes : stage) - Ring::kBytes, lane);
        asm volatile("cp.async.commit_group;" ::: "memory");
        stage = stage == Ring::kWarpBytes - Ring::kBytes ? 0 : stage + Ring::kBytes;
        data.me = __shfl_sync(0xffffffffu, mes, i & 31);
        data.ve = __shfl_sync(0xffffffffu, ves, i & 31);
        data.template step<true>(c, f, grad_scale, key, first);
        ring.put(data, lane);
        if (lane == 0) {
          me[i * (kOptTrip / kOptRun)] = static_cast<uint8_t>(data.me);
          ve[i * (kOptTrip / kOptRun)] = static_cast<uint8_t>(data.ve);
        }
        ring.next();
        first += kOptTrip;
      }
    } else {
      AdamWCursor<P, G, kRemainder> cursor(t, at, lane);
      for (int i = 0; i < whole; ++i, cursor.next()) {
        cursor.get(data);
        data.template step<true>(c, f, grad_scale, key, 0u);
        cursor.put(data);
      }
    }
    at += static_cast<long long>(whole) * kOptTrip;
  }
  for (; at < end; at += kOptTrip) {
    const long long left = end - at;
    Data data;
    data.g.get_some(static_cast<const G*>(t.g) + at, left, lane);
    data.p.get_some(static_cast<const P*>(t.p) + at, left, lane);
    data.m.get_some(static_cast<const Moment*>(t.m) + at, left, lane);
    data.v.get_some(static_cast<const Moment*>(t.v) + at, left, lane);
    if constexpr (kRemainder) data.r.get_some(t.r + at, left, lane);
    if constexpr (k8) {
      data.me = t.me[at / kOptRun];
      data.ve = t.ve[at / kOptRun];
    }
    data.template step<false>(c, f, grad_scale, key, static_cast<uint32_t>(at) + lane);
    data.p.put_some(static_cast<P*>(t.p) + at, left, lane);
    if constexpr (kRemainder) data.r.put_some(t.r + at, left, lane);
    data.m.put_some(static_cast<Moment*>(t.m) + at, left, lane);
    data.v.put_some(static_cast<Moment*>(t.v) + at, left, lane);
    if constexpr (k8) {
      __syncwarp();  // every lane has read the exponents
      if (lane == 0) {
        t.me[at / kOptRun] = static_cast<uint8_t>(data.me);
        t.ve[at / kOptRun] = static_cast<uint8_t>(data.ve);
      }
    }
  }
}

// ---- global norm and clipping -----------------------------------------------------------------------------------------

struct GradEntry {
  void* g;
  long long numel;
  uint32_t vec;
};

// Sum of squares of a lane's eight elements.  Squares of fp32 gradients leave the fp32 range, so fp32 may be used only where they
// stay well inside it: there squares and their sums in pairs are rounded to fp32 (2^-24 of the sum each, so 2^-24 of the norm
// together) and half the conversions to float64 are saved, which run at an eighth of the rate of the additions and bound the sum
// of bf16 gradients.
__device__ __forceinline__ double sum_of_squares(const float2 (&g)[4]) {
  float2 s[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) s[k] = mul2(g[k], g[k]);
  const float2 a = add2(s[0], s[1]), b = add2(s[2], s[3]);
  const float top = fmaxf(fmaxf(a.x, a.y), fmaxf(b.x, b.y));
  if (top > 0x1p-80f && top < 0x1p120f)
    return (static_cast<double>(a.x) + static_cast<double>(a.y)) + (static_cast<double>(b.x) + static_cast<double>(b.y));
  double sum = 0.0;
#pragma unroll
  for (int k = 0; k < 4; ++k)
    sum += static_cast<double>(g[k].x) * g[k].x + static_cast<double>(g[k].y) * g[k].y;
  return sum;
}

// partial[chunk] = sum of squares of the chunk, in a fixed order.
template <typename G, int kCapacity>
__global__ void __launch_bounds__(kOptThreads)
    grad_sumsq_kernel(const __grid_constant__ TensorTable<GradEntry, kCapacity> table, double* __restrict__ partial) {
  const int which = find_tensor(table, blockIdx.x);
  const GradEntry& t = table.t[which];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long begin = static_cast<long long>(blockIdx.x - table.first[which]) * table.trips * kOptTrip;
  const long long end = min(begin + static_cast<long long>(table.trips) * kOptTrip, t.numel);
  long long at = begin + warp * kOptRun;
  const G* const tg = static_cast<const G*>(t.g);
  double acc = 0.0;
  float2 g[4];
  if (t.vec) {
    constexpr int kDeep = 16 / sizeof(G);  // loads in flight: 128 bytes a lane
    const G* p = tg + at + 8 * lane;
    for (; at + (kDeep - 1) * kOptTrip + kOptRun <= end; at += kDeep * kOptTrip, p += kDeep * kOptTrip) {
      Run<G> run[kDeep];
#pragma unroll
      for (int i = 0; i < kDeep; ++i) run[i].get(p + i * kOptTrip);
#pragma unroll
      for (int i = 0; i < kDeep; ++i) {
        run[i].unpack(g);
        acc += sum_of_squares(g);
      }
    }
    for (; at + kOptRun <= end; at += kOptTrip, p += kOptTrip) {
      Run<G> run;
      run.get(p);
      run.unpack(g);
      acc += sum_of_squares(g);
    }
  }
  for (; at < end; at += kOptTrip) {
    Run<G> run;
    run.get_some(tg + at, end - at, lane);
    run.unpack(g);
    acc += sum_of_squares(g);
  }
  const double total = block_reduce_sum(acc);
  if (threadIdx.x == 0) partial[blockIdx.x] = total;
}

// out[0] = norm, out[1] = min(1, max_norm / (norm + 1e-6)); NaN stays NaN.  Launched ahead of the end of the kernels before it
// and waits for them here, so that its launch costs nothing.
constexpr int kNormThreads = 1024;
__global__ void __launch_bounds__(kNormThreads)
    grad_norm_final_kernel(const double* __restrict__ partial, long long n, float max_norm, float* __restrict__ out) {
  __shared__ double warp_sums[kNormThreads / 32];
  cudaGridDependencySynchronize();
  double acc = 0.0;
  for (long long i = threadIdx.x; i < n; i += 4 * kNormThreads) {
    double x[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = i + k * kNormThreads < n ? __ldcg(partial + i + k * kNormThreads) : 0.0;
    acc += (x[0] + x[1]) + (x[2] + x[3]);
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, off);
  if ((threadIdx.x & 31) == 0) warp_sums[threadIdx.x >> 5] = acc;
  __syncthreads();
  if (threadIdx.x < 32) {
    double total = warp_sums[threadIdx.x];
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) total += __shfl_xor_sync(0xffffffffu, total, off);
    if (threadIdx.x == 0) {
      const float norm = static_cast<float>(sqrt(total));
      const float coef = __fdiv_rn(max_norm, __fadd_rn(norm, 1e-6f));
      out[0] = norm;
      out[1] = coef > 1.0f ? 1.0f : coef;
    }
  }
}

// g <- g * coef; nothing to do when coef is 1.  Chunks are taken from the last to the first: the end of the gradients is still in
// L2 from the sum of squares.
template <typename G, int kCapacity>
__global__ void __launch_bounds__(kOptThreads)
    grad_scale_kernel(const __grid_constant__ TensorTable<GradEntry, kCapacity> table, const float* __restrict__ coef_ptr) {
  const float coef = *coef_ptr;
  if (coef == 1.0f) return;
  const uint32_t chunk = gridDim.x - 1 - blockIdx.x;
  const int which = find_tensor(table, chunk);
  const GradEntry& t = table.t[which];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long begin = static_cast<long long>(chunk - table.first[which]) * table.trips * kOptTrip;
  const long long end = min(begin + static_cast<long long>(table.trips) * kOptTrip, t.numel);
  long long at = begin + warp * kOptRun;
  G* const tg = static_cast<G*>(t.g);
  auto scale = [coef](Run<G>& run) {
    float2 g[4];
    run.unpack(g);
#pragma unroll
    for (int k = 0; k < 4; ++k) g[k] = mul2(g[k], both(coef));
    run.pack(g);
  };
  if (t.vec) {
    G* p = tg + at + 8 * lane;
    for (; at + kOptTrip + kOptRun <= end; at += 2 * kOptTrip, p += 2 * kOptTrip) {  // two loads in flight
      Run<G> a, b;
      a.get(p);
      b.template get<kOptTrip>(p);
      scale(a);
      a.put(p);
      scale(b);
      b.put(p + kOptTrip);
    }
    for (; at + kOptRun <= end; at += kOptTrip, p += kOptTrip) {
      Run<G> run;
      run.get(p);
      scale(run);
      run.put(p);
    }
  }
  for (; at < end; at += kOptTrip) {
    Run<G> run;
    run.get_some(tg + at, end - at, lane);
    scale(run);
    run.put_some(tg + at, end - at, lane);
  }
}

// ---- block quantiser --------------------------------------------------------------------------------------------------
// A warp takes kQuantRuns blocks, all of them read before the first is worked on.

constexpr int kQuantRuns = 4;
constexpr int kQuantChunk = kQuantRuns * kOptTrip;  // elements of a CTA

// kRandom: rounded at random with `key`, else to nearest (halves away from zero).
template <bool kVec, bool kSigned, bool kRandom, typename T>
__device__ __forceinline__ uint32_t quantize_run(const Run<T>& run, uint32_t key, uint32_t first, Run<uint8_t>& out) {
  float2 v[4];
  run.unpack(v);
  uint32_t low[8], high[8];
  if constexpr (kRandom) {
    random_dither<kVec>(key, first, low, high);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) low[k] = high[k] = 0x800000u;
  }
  using Code = Code8<kSigned>;
  const uint32_t top = Code::block_top(v);
  return Code::is_rare(top) ? Code::template encode<true>(v, top, kSigned ? low : high, out)
                            : Code::template encode<false>(v, top, kSigned ? low : high, out);
}
template <typename T, bool kSigned, bool kRandom>
__global__ void __launch_bounds__(kOptThreads)
    quantize_kernel(const T* __restrict__ x, long long numel, int aligned, uint32_t key, uint8_t* __restrict__ codes,
                    uint8_t* __restrict__ exponents) {
  const int lane = threadIdx.x & 31;
  const long long begin = static_cast<long long>(blockIdx.x) * kQuantChunk + (threadIdx.x >> 5) * kOptRun;
  Run<uint8_t> out;
  if (aligned && begin + (kQuantRuns - 1) * kOptTrip + kOptRun <= numel) {
    Run<T> run[kQuantRuns];
    const T* p = x + begin + 8 * lane;
    uint8_t *to = codes + begin + 8 * lane, *e_to = exponents + begin / kOptRun;
    run[0].get(p);
    run[1].template get<kOptTrip>(p);
    run[2].template get<2 * kOptTrip>(p);
    run[3].template get<3 * kOptTrip>(p);
#pragma unroll
    for (int i = 0; i < kQuantRuns; ++i) {
      const uint32_t first = static_cast<uint32_t>(begin) + i * kOptTrip + 8 * lane;
      const uint32_t e = quantize_run<true, kSigned, kRandom>(run[i], key, first, out);
      out.put(to + i * kOptTrip);
      if (lane == 0) e_to[i * (kOptTrip / kOptRun)] = static_cast<uint8_t>(e);
    }
    return;
  }
  for (long long at = begin; at < numel && at < begin + kQuantChunk; at += kOptTrip) {
    Run<T> run;
    run.get_some(x + at, numel - at, lane);
    const uint32_t e = quantize_run<false, kSigned, kRandom>(run, key, static_cast<uint32_t>(at) + lane, out);
    out.put_some(codes + at, numel - at, lane);
    if (lane == 0) exponents[at / kOptRun] = static_cast<uint8_t>(e);
  }
}

template <typename T, bool kSigned>
__global__ void __launch_bounds__(kOptThreads)
    dequantize_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ exponents, long long numel, int aligned,
                      T* __restrict__ out) {
  const int lane = threadIdx.x & 31;
  const long long begin = static_cast<long long>(blockIdx.x) * kQuantChunk + (threadIdx.x >> 5) * kOptRun;
  float2 v[4];
  Run<T> run;
  if (aligned && begin + (kQuantRuns - 1) * kOptTrip + kOptRun <= numel) {
    Run<uint8_t> in[kQuantRuns];
    uint32_t e[kQuantRuns];
    const uint8_t* p = codes + begin + 8 * lane;
    in[0].get(p);
    in[1].template get<kOptTrip>(p);
    in[2].template get<2 * kOptTrip>(p);
    in[3].template get<3 * kOptTrip>(p);
#pragma unroll
    for (int i = 0; i < kQuantRuns; ++i) e[i] = exponents[(begin + i * kOptTrip) / kOptRun];
#pragma unroll
    for (int i = 0; i < kQuantRuns; ++i) {
      Code8<kSigned>::decode(in[i], e[i], v);
      run.pack(v);
      run.put(out + begin + i * kOptTrip + 8 * lane);
    }
    return;
  }
  for (long long at = begin; at < numel && at < begin + kQuantChunk; at += kOptTrip) {
    Run<uint8_t> in;
    in.get_some(codes + at, numel - at, lane);
    Code8<kSigned>::decode(in, exponents[at / kOptRun], v);
    run.pack(v);
    run.put_some(out + at, numel - at, lane);
  }
}

}  // namespace eo
