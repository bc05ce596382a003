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
#include <cuda_runtime.h>
#include <stdint.h>

namespace eo {

constexpr int kOptThreads = 256;
constexpr int kOptRun = 256;                                  // elements a warp takes at a time; block of an 8-bit state
constexpr int kOptTrip = kOptThreads / 32 * kOptRun;          // elements a CTA takes per trip
constexpr int kOptSmallTable = 24, kOptLargeTable = 384;      // tensors per launch

// ---- memory access ---------------------------------------------------------------------------------------------------

__device__ __forceinline__ void load_run(const float* p, float (&x)[8]) {
  asm volatile("ld.global.L1::no_allocate.v8.f32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3]), "=f"(x[4]), "=f"(x[5]), "=f"(x[6]), "=f"(x[7])
               : "l"(p));
}
__device__ __forceinline__ void store_run(float* p, const float (&x)[8]) {
  asm volatile("st.global.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "f"(x[0]), "f"(x[1]), "f"(x[2]), "f"(x[3]),
               "f"(x[4]), "f"(x[5]), "f"(x[6]), "f"(x[7])
               : "memory");
}
__device__ __forceinline__ uint4 load_16(const void* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ uint2 load_8(const void* p) {
  uint2 v;
  asm volatile("ld.global.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
  return v;
}
__device__ __forceinline__ void store_16(void* p, uint4 v) { *reinterpret_cast<uint4*>(p) = v; }
__device__ __forceinline__ void store_8(void* p, uint2 v) { *reinterpret_cast<uint2*>(p) = v; }

__device__ __forceinline__ float bf16_bits_to_f32(uint32_t h) { return __uint_as_float(h << 16); }
__device__ __forceinline__ uint32_t f32_to_bf16_bits(float x) { return __bfloat16_as_ushort(__float2bfloat16_rn(x)); }

__device__ __forceinline__ void load_run(const __nv_bfloat16* p, float (&x)[8]) {
  const uint4 v = load_16(p);
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    x[2 * k] = __uint_as_float(w[k] << 16);
    x[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
  }
}
__device__ __forceinline__ void store_run(__nv_bfloat16* p, const float (&x)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * k], x[2 * k + 1]);
    w[k] = *reinterpret_cast<const uint32_t*>(&h);
  }
  store_16(p, make_uint4(w[0], w[1], w[2], w[3]));
}
__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void from_f32(float* p, float x) { *p = x; }
__device__ __forceinline__ void from_f32(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }

// The run of `left` elements (from `x`) as eight values per lane; elements beyond the end read as zero.
template <typename T>
__device__ __forceinline__ void load_lane(const T* x, long long left, int lane, bool vec, float (&out)[8]) {
  if (vec) {
    load_run(x + 8 * lane, out);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) out[k] = (32 * k + lane < left) ? to_f32(x[32 * k + lane]) : 0.0f;
  }
}
template <typename T>
__device__ __forceinline__ void store_lane(T* x, long long left, int lane, bool vec, const float (&v)[8]) {
  if (vec) {
    store_run(x + 8 * lane, v);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (32 * k + lane < left) from_f32(x + 32 * k + lane, v[k]);
  }
}
// Bytes: packed little-endian, element k of the lane in byte k % 4 of word k / 4.
__device__ __forceinline__ void load_codes(const uint8_t* x, long long left, int lane, bool vec, uint32_t (&w)[2]) {
  if (vec) {
    const uint2 v = load_8(x + 8 * lane);
    w[0] = v.x;
    w[1] = v.y;
  } else {
    w[0] = w[1] = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (32 * k + lane < left) w[k / 4] |= static_cast<uint32_t>(x[32 * k + lane]) << (8 * (k % 4));
  }
}
__device__ __forceinline__ void store_codes(uint8_t* x, long long left, int lane, bool vec, const uint32_t (&w)[2]) {
  if (vec) {
    store_8(x + 8 * lane, make_uint2(w[0], w[1]));
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (32 * k + lane < left) x[32 * k + lane] = static_cast<uint8_t>(w[k / 4] >> (8 * (k % 4)));
  }
}
// Place, within its run, of element k of a lane.
__device__ __forceinline__ int place_of(int k, int lane, bool vec) { return vec ? 8 * lane + k : 32 * k + lane; }

// bf16 weights whose fp32 master is kept as bf16 plus a signed 16-bit remainder: master bits = (bf16 bits << 16) +
// remainder.  Written back as the nearest bf16 (halves away from zero, so that the remainder fits 16 bits); a NaN
// becomes the quiet NaN with remainder zero, as adding to its payload could wrap.
__device__ __forceinline__ void load_master(const __nv_bfloat16* p, const int16_t* r, long long left, int lane, bool vec,
                                            float (&out)[8]) {
  if (vec) {
    const uint4 hi = load_16(p + 8 * lane), lo = load_16(r + 8 * lane);
    const uint32_t h[4] = {hi.x, hi.y, hi.z, hi.w}, l[4] = {lo.x, lo.y, lo.z, lo.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      out[2 * k] = __uint_as_float((h[k] << 16) + static_cast<uint32_t>(static_cast<int32_t>(l[k] << 16) >> 16));
      out[2 * k + 1] = __uint_as_float((h[k] & 0xffff0000u) + static_cast<uint32_t>(static_cast<int32_t>(l[k]) >> 16));
    }
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int i = 32 * k + lane;
      out[k] = (i < left) ? __uint_as_float((static_cast<uint32_t>(__bfloat16_as_ushort(p[i])) << 16) +
                                            static_cast<uint32_t>(static_cast<int32_t>(r[i])))
                          : 0.0f;
    }
  }
}
__device__ __forceinline__ void split_master(float x, uint32_t& hi, uint32_t& lo) {
  const uint32_t bits = __float_as_uint(x);
  hi = (bits + 0x8000u) >> 16;
  lo = bits & 0xffffu;  // bits - (hi << 16), modulo 2^16
  if (x != x) hi = 0x7fc0u, lo = 0;
}
__device__ __forceinline__ void store_master(__nv_bfloat16* p, int16_t* r, long long left, int lane, bool vec,
                                             const float (&x)[8]) {
  uint32_t hi[8], lo[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) split_master(x[k], hi[k], lo[k]);
  if (vec) {
    uint32_t h[4], l[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      h[k] = hi[2 * k] | (hi[2 * k + 1] << 16);
      l[k] = lo[2 * k] | (lo[2 * k + 1] << 16);
    }
    store_16(p + 8 * lane, make_uint4(h[0], h[1], h[2], h[3]));
    store_16(r + 8 * lane, make_uint4(l[0], l[1], l[2], l[3]));
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int i = 32 * k + lane;
      if (i < left) {
        p[i] = __ushort_as_bfloat16(static_cast<unsigned short>(hi[k]));
        r[i] = static_cast<int16_t>(static_cast<uint16_t>(lo[k]));
      }
    }
  }
}

// ---- 8-bit block-scaled numbers ---------------------------------------------------------------------------------------
// A block of 256 elements shares one byte, the exponent field E of its largest finite magnitude (at least 1).  A code is
// a small float, its bits those of an fp32 number shifted right by 20:
//   signed   (first moments):  sign, 4 exponent bits, 3 mantissa bits; down to 2^-16 of the block's power of two
//   unsigned (second moments):       5 exponent bits, 3 mantissa bits; down to 2^-32
//   value = f32(code << 20) * 2^kShift * 2^(E - 127),    code = (bits(|x| * 2^(127 - E) * 2^-kShift) + d) >> 20
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
template <bool kSigned>
struct Code8 {
  static constexpr int kTop = kSigned ? 14 : 30;
  static constexpr uint32_t kNan = kSigned ? 0x7f : 0xff;
  // 2^kShift and 2^-kShift with kShift = 127 - kTop
  static __device__ __forceinline__ float up() { return __uint_as_float(static_cast<uint32_t>(254 - kTop) << 23); }
  static __device__ __forceinline__ float down() { return __uint_as_float(static_cast<uint32_t>(kTop) << 23); }

  // value of code k of a lane; scale = 2^(E - 127)
  static __device__ __forceinline__ float decode(uint32_t word, int byte, float scale) {
    uint32_t bits;
    if (kSigned) {
      bits = static_cast<uint32_t>(static_cast<int32_t>(word << (24 - 8 * byte)) >> 4) & 0x87f00000u;
    } else {
      bits = (byte == 3 ? word >> 4 : word << (20 - 8 * byte)) & 0x0ff00000u;
    }
    const float x = __fmul_rn(__fmul_rn(__uint_as_float(bits), up()), scale);
    return ((bits & 0x0ff00000u) == (kNan << 20)) ? __uint_as_float(0x7fc00000u) : x;
  }
  static __device__ __forceinline__ uint32_t magnitude(float x) {  // for the block's maximum; 0 if it does not count
    const uint32_t b = kSigned ? (__float_as_uint(x) & 0x7fffffffu) : __float_as_uint(x);
    return b >= 0x7f800000u ? 0u : b;
  }
  // inv_scale = 2^(127 - E)
  static __device__ __forceinline__ uint32_t encode(float x, float inv_scale, uint32_t d) {
    const uint32_t b = __float_as_uint(x);
    const float y = __fmul_rn(__fmul_rn(kSigned ? fabsf(x) : x, inv_scale), down());
    uint32_t c = (__float_as_uint(y) + d) >> 20;
    if (kSigned) {
      c = ((b & 0x7fffffffu) >= 0x7f800000u) ? kNan : c;
      return c | ((b >> 24) & 0x80u);
    }
    if (c == 0 && x > 0.0f) c = 1;
    if (b == 0x80000000u) return 0;  // -0
    return b >= 0x7f800000u ? kNan : c;
  }
};
__device__ __forceinline__ float scale_of(uint32_t e) { return __uint_as_float((e == 0 ? 1u : e) << 23); }
__device__ __forceinline__ float inv_scale_of(uint32_t e) {
  return __uint_as_float(e >= 254u ? 0x00400000u : (254u - e) << 23);
}
// d = r * mul + add for a block with exponent byte e.
struct Dither {
  uint32_t mul, add;
  __device__ __forceinline__ Dither(uint32_t e, bool random) {
    mul = (random && e < 254u) ? 16u : 0u;
    add = e >= 254u ? 0u : random ? 8u : 0x80000u;
  }
  __device__ __forceinline__ uint32_t operator()(uint32_t r) const { return r * mul + add; }
};
template <bool kSigned>
__device__ __forceinline__ uint32_t block_exponent(const float (&x)[8]) {
  uint32_t top = 0;
#pragma unroll
  for (int k = 0; k < 8; ++k) top = max(top, Code8<kSigned>::magnitude(x[k]));
  const uint32_t e = __reduce_max_sync(0xffffffffu, top) >> 23;
  return e < 1u ? 1u : e;
}
// The finaliser of MurmurHash3: 32 random bits of an element from mix(key ^ element), key from (seed, tensor, step).
__host__ __device__ __forceinline__ uint32_t mix32(uint32_t x) {
  x = (x ^ (x >> 16)) * 0x85ebca6bu;
  x = (x ^ (x >> 13)) * 0xc2b2ae35u;
  return x ^ (x >> 16);
}
__host__ __device__ __forceinline__ uint32_t rounding_key(uint32_t seed, uint32_t tensor, uint32_t step) {
  return mix32(mix32(mix32(seed) ^ tensor) ^ step);
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
  float beta1, one_minus_beta1, beta2, one_minus_beta2, eps, l2;
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

// g, p, m, v of one lane; every operation rounded once, in this order, so that the result does not depend on how the
// compiler would contract it (the 8-bit codes of a run must not depend on the build).
__device__ __forceinline__ void adamw_update(float (&p)[8], const float (&g_in)[8], float (&m)[8], float (&v)[8],
                                             const AdamWScalars& c, const AdamWFactors& f, float grad_scale) {
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    float g = __fmul_rn(g_in[k], grad_scale);
    if (c.l2 != 0.0f) g = __fadd_rn(g, __fmul_rn(p[k], c.l2));
    m[k] = __fadd_rn(__fmul_rn(m[k], c.beta1), __fmul_rn(g, c.one_minus_beta1));
    v[k] = __fadd_rn(__fmul_rn(v[k], c.beta2), __fmul_rn(__fmul_rn(g, g), c.one_minus_beta2));
    const float denom = __fadd_rn(__fmul_rn(__fsqrt_rn(v[k]), f.inv_root_bc2), c.eps);
    p[k] = __fsub_rn(__fmul_rn(p[k], f.decay), __fmul_rn(__fdiv_rn(m[k], denom), f.step_size));
  }
}

// kRemainder: p is bf16 with remainders.  k8: m and v are codes with exponent bytes.
template <typename P, typename G, bool kRemainder, bool k8, int kCapacity>
__global__ void __launch_bounds__(kOptThreads)
    adamw_kernel(const __grid_constant__ TensorTable<AdamWEntry, kCapacity> table, const __grid_constant__ AdamWScalars c) {
  const int which = find_tensor(table, blockIdx.x);
  const AdamWEntry& t = table.t[which];
  const AdamWFactors f = c.dev_factors != nullptr ? c.dev_factors[which] : c.f;
  const float grad_scale = c.grad_scale != nullptr ? *c.grad_scale : 1.0f;
  const uint32_t key = k8 ? rounding_key(c.seed, t.index, f.step) : 0u;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long numel = t.numel;
  long long at = (static_cast<long long>(blockIdx.x - table.first[which]) * table.trips) * kOptTrip + warp * kOptRun;
  P* const tp = static_cast<P*>(t.p);
  const G* const tg = static_cast<const G*>(t.g);
  for (int trip = 0; trip < table.trips && at < numel; ++trip, at += kOptTrip) {
    const long long left = numel - at;
    const bool vec = t.vec != 0 && left >= kOptRun;
    float p[8], g[8], m[8], v[8];
    load_lane(tg + at, left, lane, vec, g);
    if constexpr (kRemainder) {
      load_master(tp + at, t.r + at, left, lane, vec, p);
    } else {
      load_lane(tp + at, left, lane, vec, p);
    }
    if constexpr (k8) {
      uint32_t cm[2], cv[2];
      load_codes(static_cast<uint8_t*>(t.m) + at, left, lane, vec, cm);
      load_codes(static_cast<uint8_t*>(t.v) + at, left, lane, vec, cv);
      const float sm = scale_of(t.me[at / kOptRun]), sv = scale_of(t.ve[at / kOptRun]);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        m[k] = Code8<true>::decode(cm[k / 4], k % 4, sm);
        v[k] = Code8<false>::decode(cv[k / 4], k % 4, sv);
      }
    } else {
      load_lane(static_cast<const float*>(t.m) + at, left, lane, vec, m);
      load_lane(static_cast<const float*>(t.v) + at, left, lane, vec, v);
    }
    adamw_update(p, g, m, v, c, f, grad_scale);
    if constexpr (kRemainder) {
      store_master(tp + at, t.r + at, left, lane, vec, p);
    } else {
      store_lane(tp + at, left, lane, vec, p);
    }
    if constexpr (k8) {
      const uint32_t em = block_exponent<true>(m), ev = block_exponent<false>(v);
      const float im = inv_scale_of(em), iv = inv_scale_of(ev);
      const Dither dm(em, true), dv(ev, true);
      uint32_t cm[2] = {0, 0}, cv[2] = {0, 0};
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const uint32_t r = mix32(key ^ static_cast<uint32_t>(at + place_of(k, lane, vec)));
        cm[k / 4] |= Code8<true>::encode(m[k], im, dm(r & 0xffffu)) << (8 * (k % 4));
        cv[k / 4] |= Code8<false>::encode(v[k], iv, dv(r >> 16)) << (8 * (k % 4));
      }
      store_codes(static_cast<uint8_t*>(t.m) + at, left, lane, vec, cm);
      store_codes(static_cast<uint8_t*>(t.v) + at, left, lane, vec, cv);
      if (lane == 0) {
        t.me[at / kOptRun] = static_cast<uint8_t>(em);
        t.ve[at / kOptRun] = static_cast<uint8_t>(ev);
      }
    } else {
      store_lane(static_cast<float*>(t.m) + at, left, lane, vec, m);
      store_lane(static_cast<float*>(t.v) + at, left, lane, vec, v);
    }
  }
}

// ---- global norm and clipping -----------------------------------------------------------------------------------------

struct GradEntry {
  void* g;
  long long numel;
  uint32_t vec;
};

// partial[chunk] = sum of squares of the chunk, in float64 (the squares of fp32 gradients leave the fp32 range) and in a
// fixed order.
template <typename G, int kCapacity>
__global__ void __launch_bounds__(kOptThreads)
    grad_sumsq_kernel(const __grid_constant__ TensorTable<GradEntry, kCapacity> table, double* __restrict__ partial) {
  const int which = find_tensor(table, blockIdx.x);
  const GradEntry& t = table.t[which];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long numel = t.numel;
  long long at = (static_cast<long long>(blockIdx.x - table.first[which]) * table.trips) * kOptTrip + warp * kOptRun;
  const G* const tg = static_cast<const G*>(t.g);
  double acc = 0.0;
  for (int trip = 0; trip < table.trips && at < numel; ++trip, at += kOptTrip) {
    float g[8];
    load_lane(tg + at, numel - at, lane, t.vec != 0 && numel - at >= kOptRun, g);
#pragma unroll
    for (int k = 0; k < 8; ++k) acc += static_cast<double>(g[k]) * g[k];
  }
  const double total = block_reduce_sum(acc);
  if (threadIdx.x == 0) partial[blockIdx.x] = total;
}

// out[0] = norm, out[1] = min(1, max_norm / (norm + 1e-6)); NaN stays NaN.
__global__ void __launch_bounds__(kEwThreads)
    grad_norm_final_kernel(const double* __restrict__ partial, long long n, float max_norm, float* __restrict__ out) {
  double acc = 0.0;
  for (long long i = threadIdx.x; i < n; i += kEwThreads) acc += partial[i];
  const double total = block_reduce_sum(acc);
  if (threadIdx.x == 0) {
    const float norm = static_cast<float>(sqrt(total));
    const float coef = __fdiv_rn(max_norm, __fadd_rn(norm, 1e-6f));
    out[0] = norm;
    out[1] = coef > 1.0f ? 1.0f : coef;
  }
}

// g <- g * coef; nothing to do when coef is 1.
template <typename G, int kCapacity>
__global__ void __launch_bounds__(kOptThreads)
    grad_scale_kernel(const __grid_constant__ TensorTable<GradEntry, kCapacity> table, const float* __restrict__ coef_ptr) {
  const float coef = *coef_ptr;
  if (coef == 1.0f) return;
  const int which = find_tensor(table, blockIdx.x);
  const GradEntry& t = table.t[which];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long numel = t.numel;
  long long at = (static_cast<long long>(blockIdx.x - table.first[which]) * table.trips) * kOptTrip + warp * kOptRun;
  G* const tg = static_cast<G*>(t.g);
  for (int trip = 0; trip < table.trips && at < numel; ++trip, at += kOptTrip) {
    const long long left = numel - at;
    const bool vec = t.vec != 0 && left >= kOptRun;
    float g[8];
    load_lane(static_cast<const G*>(tg) + at, left, lane, vec, g);
#pragma unroll
    for (int k = 0; k < 8; ++k) g[k] = __fmul_rn(g[k], coef);
    store_lane(tg + at, left, lane, vec, g);
  }
}

// ---- block quantiser --------------------------------------------------------------------------------------------------

// One warp per block of 256.  `random`: stochastic rounding with `key`, else to nearest (halves away from zero).
template <typename T, bool kSigned>
__global__ void __launch_bounds__(kOptThreads)
    quantize_kernel(const T* __restrict__ x, long long numel, int aligned, int random, uint32_t key,
                    uint8_t* __restrict__ codes, uint8_t* __restrict__ exponents) {
  const int lane = threadIdx.x & 31;
  const long long block = static_cast<long long>(blockIdx.x) * (kOptThreads / 32) + (threadIdx.x >> 5);
  const long long at = block * kOptRun, left = numel - at;
  if (left <= 0) return;
  const bool vec = aligned && left >= kOptRun;
  float v[8];
  load_lane(x + at, left, lane, vec, v);
  const uint32_t e = block_exponent<kSigned>(v);
  const float inv = inv_scale_of(e);
  const Dither d(e, random != 0);
  uint32_t w[2] = {0, 0};
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const uint32_t r = mix32(key ^ static_cast<uint32_t>(at + place_of(k, lane, vec)));
    w[k / 4] |= Code8<kSigned>::encode(v[k], inv, d(kSigned ? (r & 0xffffu) : (r >> 16))) << (8 * (k % 4));
  }
  store_codes(codes + at, left, lane, vec, w);
  if (lane == 0) exponents[block] = static_cast<uint8_t>(e);
}

template <typename T, bool kSigned>
__global__ void __launch_bounds__(kOptThreads)
    dequantize_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ exponents, long long numel, int aligned,
                      T* __restrict__ out) {
  const int lane = threadIdx.x & 31;
  const long long block = static_cast<long long>(blockIdx.x) * (kOptThreads / 32) + (threadIdx.x >> 5);
  const long long at = block * kOptRun, left = numel - at;
  if (left <= 0) return;
  const bool vec = aligned && left >= kOptRun;
  uint32_t w[2];
  load_codes(codes + at, left, lane, vec, w);
  const float scale = scale_of(exponents[block]);
  float v[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = Code8<kSigned>::decode(w[k / 4], k % 4, scale);
  store_lane(out + at, left, lane, vec, v);
}

}  // namespace eo
