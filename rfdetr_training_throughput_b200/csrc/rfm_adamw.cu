// AdamW over many tensors in one launch, moments in 32 bits or in 8.
//
//   g  = grad * grad_scale
//   m' = b1 m + (1 - b1) g,   v' = b2 v + (1 - b2) g^2
//   p' = p (1 - lr wd) - lr / (1 - b1^t) * m' / (sqrt(v') / sqrt(1 - b2^t) + eps)
//
// fp32 arithmetic for every parameter type; a 16-bit parameter is rounded once,
// at its store.
//
// 8-bit moments.  256 consecutive elements of a tensor share one fp32 scale per
// moment, the block's largest value, and each element one byte c:
//   m = scale c|c| / 127^2  (c in -127..127),   v = scale (c / 255)^4  (c in 0..255).
// The powers spend the codes where the values are small: |m| spans 1 : 16129
// and sqrt(v), which the update divides by, 1 : 65025 within a block.  A nonzero
// v keeps a code of at least 1, so the update never divides by eps alone.  Codes
// are rounded at random, down or up in proportion to the distance (in code
// units): with b2 = 0.999 one step moves v by a thousandth of itself, far less
// than half a code, and rounding to nearest would never let it move.  The random
// bits are a hash of the step, the tensor's number and the element's index, so
// a step is reproducible and a replayed graph whose step counter advances
// rounds anew.  Every operation on the way to a code is an explicitly rounded
// fp32 one (no contraction), so the codes are defined bit for bit.
//
// HBM-bound: 28 bytes a parameter in fp32 with 32-bit moments, 16 with 8-bit
// ones.  The tensors' table travels in the kernel's parameters (64 bytes a
// tensor), so no upload precedes the launch.  One CTA takes 1024 consecutive
// elements of one tensor, a warp a block of 256, a lane two quads of it, so that
// every access of a warp is contiguous; small CTAs, nine of them an SM, keep
// loads in flight while others compute.  100 M fp32 parameters: 406 us with
// 32-bit moments (6.9 TB/s); 299 us with 8-bit ones (5.4 TB/s; 83 instructions a parameter,
// most of them for the codes, keep the issue slots two thirds busy; four CTAs of
// 256 threads took 326, several blocks a warp 344 and more).
#include <math.h>

#include <type_traits>

#include "rfm_types.cuh"

namespace rfm {
namespace {

constexpr int kThreads = 128;
constexpr int kBlock = RFM_MOMENT_BLOCK;          // elements that share a scale
constexpr int kChunk = 1024;                      // elements of one CTA
static_assert(kBlock == 32 * 8 && kChunk == kThreads / 32 * kBlock, "a warp holds one block, eight elements a lane");
static_assert(sizeof(rfm_adamw_tensor) == 64, "tensor entries are 64 bytes");

struct AdamScalars {
  float keep;         // 1 - lr wd
  float step_size;    // lr / (1 - b1^t)
  float inv_sqrt_bc2; // 1 / sqrt(1 - b2^t)
  uint32_t seed;      // t's share of the random key
};

struct AdamTensor {
  void* param;
  const void* grad;
  void* m;
  void* v;
  float* m_scale;
  float* v_scale;
  int64_t numel;
  int32_t first_chunk;  // its first CTA of the launch
  uint32_t ordinal;     // its number in the call
};
static_assert(sizeof(AdamTensor) == 64, "table entries are 64 bytes");

struct AdamCommon {
  float b1, b2, one_b1, one_b2, eps;
  AdamScalars s;
  const AdamScalars* device_s;  // instead of s, when not null
  const float* grad_scale;      // may be null
  int32_t count;
};

template <int N>
struct AdamArgs {
  AdamCommon c;
  AdamTensor t[N];
};

// Table sizes: most calls fit the small one (a short parameter copy); the large
// one fills the 32,764 bytes that a kernel's parameters may have.
constexpr int kSmallTable = 60;
constexpr int kLargeTable = 508;
static_assert(sizeof(AdamArgs<kLargeTable>) <= 32764, "kernel parameter space");

__host__ __device__ __forceinline__ uint32_t mix(uint32_t h) {
  h *= 0x9E3779B1u;
  h ^= h >> 15;
  h *= 0x85C1E8B7u;
  return h ^ (h >> 13);
}

__host__ __device__ inline AdamScalars adam_scalars(double lr, double b1, double b2, double wd, int64_t t) {
  AdamScalars s;
  s.keep = static_cast<float>(1.0 - lr * wd);
  s.step_size = static_cast<float>(lr / (1.0 - pow(b1, static_cast<double>(t))));
  s.inv_sqrt_bc2 = static_cast<float>(1.0 / sqrt(1.0 - pow(b2, static_cast<double>(t))));
  s.seed = static_cast<uint32_t>(t) * 0xC2B2AE35u;
  return s;
}

__global__ void adam_scalars_kernel(const float* device_lr, const int64_t* device_step, double lr, double b1,
                                    double b2, double wd, int64_t step, AdamScalars* out) {
  chain_start();
  *out = adam_scalars(device_lr != nullptr ? static_cast<double>(*device_lr) : lr, b1, b2, wd,
                      device_step != nullptr ? *device_step : step);
}

// Four elements of a lane: those from `i` on, of `left` that the tensor has there.
// WHOLE: all of the warp's block lies in the tensor, aligned.
template <bool WHOLE, typename T>
__device__ __forceinline__ void load_quad(Pair (&r)[2], const T* p, int64_t left) {
  if (WHOLE) {
    const Pack<T, 4> q = *reinterpret_cast<const Pack<T, 4>*>(p);
    r[0] = load_pair(q, 0);
    r[1] = load_pair(q, 1);
  } else {
    float f[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = j < left ? to_float(p[j]) : 0.f;
    r[0] = pair(f[0], f[1]);
    r[1] = pair(f[2], f[3]);
  }
}

template <bool WHOLE, typename T>
__device__ __forceinline__ void store_quad(const Pair (&r)[2], T* p, int64_t left) {
  const float2 a = split(r[0]), b = split(r[1]);
  const float f[4] = {a.x, a.y, b.x, b.y};
  if (WHOLE) {
    Pack<T, 4> q;
#pragma unroll
    for (int j = 0; j < 4; ++j) q.v[j] = from_float<T>(f[j]);
    *reinterpret_cast<Pack<T, 4>*>(p) = q;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < left) p[j] = from_float<T>(f[j]);
  }
}

// Four codes as one word, element j in byte j.
template <bool WHOLE>
__device__ __forceinline__ uint32_t load_codes(const uint8_t* p, int64_t left) {
  if (WHOLE) return *reinterpret_cast<const uint32_t*>(p);
  uint32_t w = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (j < left) w |= static_cast<uint32_t>(p[j]) << (8 * j);
  return w;
}

template <bool WHOLE>
__device__ __forceinline__ void store_codes(uint32_t w, uint8_t* p, int64_t left) {
  if constexpr (WHOLE) {
    *reinterpret_cast<uint32_t*>(p) = w;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < left) p[j] = static_cast<uint8_t>(w >> (8 * j));
  }
}

constexpr float kInv127 = static_cast<float>(1.0 / 127.0);
constexpr float kInv255 = static_cast<float>(1.0 / 255.0);

// a + b where both are products: ptxas contracts a packed product and a packed
// sum into a multiply-add even with explicit rounding, which the codes'
// definition does not have; scalar sums stay as they are.
__device__ __forceinline__ Pair sum_of_products(Pair a, Pair b) {
  const float2 x = split(a), y = split(b);
  return pair(__fadd_rn(x.x, y.x), __fadd_rn(x.y, y.y));
}

// 2^23 + byte j of a word, as a float: conversions of integers run at an eighth
// of the rate of additions, a byte moved under 2^23's mantissa at half of it.
__device__ __forceinline__ float byte_float(uint32_t w, int j) {
  return __uint_as_float(__byte_perm(w, 0x4B000000u, 0x7440u + j));
}

// Codes j, j + 1 of a word; `flipped`: with every byte's top bit inverted (c + 128).
__device__ __forceinline__ Pair decode_m(uint32_t flipped, int j, float scale) {
  const Pair a = (pair(byte_float(flipped, j), byte_float(flipped, j + 1)) + both(-8388736.f)) * both(kInv127);
  const float2 f = split(a);
  return both(scale) * pair(__fmul_rn(f.x, fabsf(f.x)), __fmul_rn(f.y, fabsf(f.y)));
}

__device__ __forceinline__ Pair decode_v(uint32_t codes, int j, float scale) {
  Pair b = (pair(byte_float(codes, j), byte_float(codes, j + 1)) + both(-8388608.f)) * both(kInv255);
  b = b * b;
  return both(scale) * (b * b);
}

// The codes by definition.  A NaN quotient (a block of infinities) converts to
// code 0, as does a block of zeros.
__device__ __noinline__ uint32_t exact_code_m(float m, float scale, uint32_t h) {
  const float u = __fmul_rn(static_cast<float>(h & 0xffffu), 1.f / 65536.f);
  const float x = __fadd_rn(__fmul_rn(__fsqrt_rn(__fdiv_rn(fabsf(m), scale)), 127.f), u);
  return static_cast<uint32_t>(min(__float2int_rz(x), 127));
}

__device__ __noinline__ uint32_t exact_code_v(float v, float scale, uint32_t h) {
  const float u = __fmul_rn(static_cast<float>(h >> 16), 1.f / 65536.f);
  const float x = __fadd_rn(__fmul_rn(__fsqrt_rn(__fsqrt_rn(__fdiv_rn(v, scale))), 255.f), u);
  return static_cast<uint32_t>(min(__float2int_rz(x), 255));
}

__device__ __forceinline__ float sqrt_fast(float x) {
  float r;
  asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Codes the quick way: with the scale's reciprocal and the approximate root the
// value x is off by at most 255 * 2^-21 = 1.2e-4 from the definition's (the root
// and the reciprocal 2^-22 of themselves each, the roundings of both ways 2^-23
// and less).  Where x lies further than kNear from a whole number both have the
// same floor; `sure` says so, and false also for a NaN or an infinity.  About
// one code in 2500 is computed again.
constexpr float kNear = 2e-4f;

// Two floors of root * top + u, each in the low byte of a word.  The random
// fraction u is 16 bits at the top of the mantissa of 1 + u.
__device__ __forceinline__ void quick_floor(Pair root, float top, uint32_t bits_a, uint32_t bits_b, uint32_t& a,
                                            uint32_t& b, bool& sure) {
  const Pair one_u = pair(__uint_as_float(0x3F800000u | (bits_a & 0x7fff80u)),
                          __uint_as_float(0x3F800000u | (bits_b & 0x7fff80u)));
  const Pair x1 = fma(root, both(top), one_u);  // x + 1
  Pair low;                                     // 2^23 + floor(x)
  asm("add.rm.f32x2 %0, %1, %2;" : "=l"(low.v) : "l"(x1.v), "l"(both(8388607.f).v));
  // x - floor(x) - 1/2, exactly: floor(x) + 1.5 first
  const Pair floor15 = low + both(-8388606.5f);
  const float2 f = split(floor15), x = split(x1), l = split(low);
  sure = sure && fabsf(x.x - f.x) < 0.5f - kNear && fabsf(x.y - f.y) < 0.5f - kNear;
  a = __float_as_uint(l.x);
  b = __float_as_uint(l.y);
}

// The low bytes of four words, in order.
__device__ __forceinline__ uint32_t pack_bytes(const uint32_t (&q)[4]) {
  return __byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410);
}

// The codes of four elements, element j in byte j; `inv`: the scale's reciprocal.
__device__ __forceinline__ uint32_t encode_m(const float (&m)[4], float scale, float inv, const uint32_t (&h)[4]) {
  uint32_t q[4];
  bool sure = true;
#pragma unroll
  for (int j = 0; j < 4; j += 2) {
    quick_floor(pair(sqrt_fast(fabsf(m[j]) * inv), sqrt_fast(fabsf(m[j + 1]) * inv)), 127.f, h[j] << 7, h[j + 1] << 7,
                q[j], q[j + 1], sure);
  }
  if (!sure) {  // a scale of 0 ends here too
#pragma unroll
    for (int j = 0; j < 4; ++j) q[j] = scale == 0.f ? 0u : exact_code_m(m[j], scale, h[j]);
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) q[j] = m[j] < 0.f ? 0u - q[j] : q[j];  // 2^23 leaves the low byte as it is
  return pack_bytes(q);
}

__device__ __forceinline__ uint32_t encode_v(const float (&v)[4], float scale, float inv, const uint32_t (&h)[4]) {
  uint32_t q[4];
  bool sure = true;
#pragma unroll
  for (int j = 0; j < 4; j += 2) {
    const float2 t = split(pair(v[j], v[j + 1]) * both(inv));
    quick_floor(pair(sqrt_fast(sqrt_fast(t.x)), sqrt_fast(sqrt_fast(t.y))), 255.f, h[j] >> 9, h[j + 1] >> 9, q[j],
                q[j + 1], sure);
  }
  if (!sure) {
#pragma unroll
    for (int j = 0; j < 4; ++j) q[j] = 0x4B000000u | (scale == 0.f ? 0u : exact_code_v(v[j], scale, h[j]));
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) q[j] = v[j] > 0.f ? max(q[j], 0x4B000001u) : q[j];  // code 1 at least
  return pack_bytes(q);
}

// Largest of a warp's non-negative values (their bit patterns order as the
// values do, and a NaN's is above infinity's, so a NaN is kept).
__device__ __forceinline__ float warp_max_bits(uint32_t bits) {
  return __uint_as_float(__reduce_max_sync(kFullMask, bits));
}

// One warp's block of 256 elements from `first` on: lane l holds the quads at 4 l
// and 128 + 4 l.
template <typename T, bool EIGHT, bool WHOLE>
__device__ __forceinline__ void adam_block(const AdamTensor& t, const AdamCommon& c, const AdamScalars& s,
                                           float grad_scale, int64_t first) {
  const int lane = threadIdx.x & 31;
  const int64_t place = first + lane * 4;
  const int64_t left = WHOLE ? 256 : t.numel - place;  // elements from this lane's first on
  T* param = static_cast<T*>(t.param) + place;
  const T* grad = static_cast<const T*>(t.grad) + place;
  using Moment = typename std::conditional<EIGHT, uint8_t, float>::type;
  Moment* avg = static_cast<Moment*>(t.m) + place;
  Moment* avg_sq = static_cast<Moment*>(t.v) + place;

  Pair p[2][2], g[2][2], m[2][2], v[2][2];
  uint32_t cm[2], cv[2];
  float sm = 0.f, sv = 0.f;
  if constexpr (EIGHT) {
    sm = t.m_scale[first / kBlock];
    sv = t.v_scale[first / kBlock];
  }
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    load_quad<WHOLE>(g[q], grad + q * 128, left - q * 128);
    load_quad<WHOLE>(p[q], param + q * 128, left - q * 128);
    if constexpr (EIGHT) {
      cm[q] = load_codes<WHOLE>(avg + q * 128, left - q * 128) ^ 0x80808080u;
      cv[q] = load_codes<WHOLE>(avg_sq + q * 128, left - q * 128);
    } else {
      load_quad<WHOLE>(m[q], avg + q * 128, left - q * 128);
      load_quad<WHOLE>(v[q], avg_sq + q * 128, left - q * 128);
    }
  }

  float top_m = 0.f, top_v = 0.f;
#pragma unroll
  for (int q = 0; q < 2; ++q) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if constexpr (EIGHT) {
        m[q][i] = decode_m(cm[q], 2 * i, sm);
        v[q][i] = decode_v(cv[q], 2 * i, sv);
      }
      const Pair gi = g[q][i] * both(grad_scale);
      m[q][i] = sum_of_products(m[q][i] * both(c.b1), gi * both(c.one_b1));
      v[q][i] = sum_of_products(v[q][i] * both(c.b2), (gi * gi) * both(c.one_b2));
      // Approximate root and reciprocal: 2^-21 of an update that is a small part
      // of the parameter.  The root takes subnormal values too: with eps 0 one of
      // 0 would be divided by.
      const float2 fv = split(v[q][i]), fm = split(m[q][i]);
      float r0, r1;
      asm("sqrt.approx.f32 %0, %1;" : "=f"(r0) : "f"(fv.x));
      asm("sqrt.approx.f32 %0, %1;" : "=f"(r1) : "f"(fv.y));
      const float2 denom = split(fma(pair(r0, r1), both(s.inv_sqrt_bc2), both(c.eps)));
      asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r0) : "f"(denom.x));
      asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r1) : "f"(denom.y));
      p[q][i] = fma(m[q][i] * pair(r0, r1), both(-s.step_size), p[q][i] * both(s.keep));
      if constexpr (EIGHT) {
        // elements past the tensor's end count as zeros whatever their block's scale is
        const bool in0 = WHOLE || q * 128 + 2 * i < left, in1 = WHOLE || q * 128 + 2 * i + 1 < left;
        const auto raise = [](float& top, float x) {  // a NaN is kept
          asm("max.NaN.f32 %0, %0, %1;" : "+f"(top) : "f"(x));
        };
        raise(top_m, in0 ? fabsf(fm.x) : 0.f);
        raise(top_m, in1 ? fabsf(fm.y) : 0.f);
        raise(top_v, in0 ? fv.x : 0.f);
        raise(top_v, in1 ? fv.y : 0.f);
      }
    }
    store_quad<WHOLE>(p[q], param + q * 128, left - q * 128);
    if constexpr (!EIGHT) {
      store_quad<WHOLE>(m[q], avg + q * 128, left - q * 128);
      store_quad<WHOLE>(v[q], avg_sq + q * 128, left - q * 128);
    }
  }
  if constexpr (EIGHT) {
    const uint32_t key = mix(t.ordinal * 0x632BE5ABu + s.seed) + static_cast<uint32_t>(place);
    const float new_sm = warp_max_bits(__float_as_uint(top_m) & 0x7fffffffu);
    const float new_sv = warp_max_bits(__float_as_uint(top_v) & 0x7fffffffu);
    const float inv_m = __frcp_rn(new_sm), inv_v = __frcp_rn(new_sv);
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      uint32_t h[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) h[j] = mix(key + (q * 128 + j));
      const float2 m0 = split(m[q][0]), m1 = split(m[q][1]), v0 = split(v[q][0]), v1 = split(v[q][1]);
      const float fm[4] = {m0.x, m0.y, m1.x, m1.y}, fv[4] = {v0.x, v0.y, v1.x, v1.y};
      store_codes<WHOLE>(encode_m(fm, new_sm, inv_m, h), avg + q * 128, left - q * 128);
      store_codes<WHOLE>(encode_v(fv, new_sv, inv_v, h), avg_sq + q * 128, left - q * 128);
    }
    if (lane == 0) {
      t.m_scale[first / kBlock] = new_sm;
      t.v_scale[first / kBlock] = new_sv;
    }
  }
}

template <typename T, bool EIGHT, int N>
__global__ void __launch_bounds__(kThreads, 9) adamw_kernel(const __grid_constant__ AdamArgs<N> a) {
  chain_start();
  // the tensor of this CTA: the last whose first chunk is not after it
  int lo = 0, hi = a.c.count - 1;
  const int chunk = static_cast<int>(blockIdx.x);
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (a.t[mid].first_chunk <= chunk) {
      lo = mid;
    } else {
      hi = mid - 1;
    }
  }
  const AdamTensor& t = a.t[lo];
  const AdamScalars s = a.c.device_s != nullptr ? *a.c.device_s : a.c.s;
  const float grad_scale = a.c.grad_scale != nullptr ? *a.c.grad_scale : 1.f;
  const int64_t first = static_cast<int64_t>(chunk - t.first_chunk) * kChunk + (threadIdx.x >> 5) * kBlock;
  if (first >= t.numel) return;
  const uintptr_t wide = reinterpret_cast<uintptr_t>(t.param) | reinterpret_cast<uintptr_t>(t.grad);
  const uintptr_t state = reinterpret_cast<uintptr_t>(t.m) | reinterpret_cast<uintptr_t>(t.v);
  const bool aligned = (wide & (4 * sizeof(T) - 1)) == 0 && (state & (EIGHT ? 3 : 15)) == 0;
  if (aligned && first + kBlock <= t.numel) {
    adam_block<T, EIGHT, true>(t, a.c, s, grad_scale, first);
  } else {
    adam_block<T, EIGHT, false>(t, a.c, s, grad_scale, first);
  }
}

// The values that 8-bit moments stand for; a warp decodes one block.
template <bool WHOLE>
__device__ __forceinline__ void decode_block(const uint8_t* m, const uint8_t* v, float sm, float sv, int64_t left,
                                             float* out_m, float* out_v) {
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const uint32_t cm = load_codes<WHOLE>(m + q * 128, left - q * 128) ^ 0x80808080u;
    const uint32_t cv = load_codes<WHOLE>(v + q * 128, left - q * 128);
    const Pair dm[2] = {decode_m(cm, 0, sm), decode_m(cm, 2, sm)};
    const Pair dv[2] = {decode_v(cv, 0, sv), decode_v(cv, 2, sv)};
    store_quad<WHOLE>(dm, out_m + q * 128, left - q * 128);
    store_quad<WHOLE>(dv, out_v + q * 128, left - q * 128);
  }
}

__global__ void __launch_bounds__(kThreads) adam_moments_kernel(const uint8_t* m, const uint8_t* v,
                                                               const float* m_scale, const float* v_scale, int64_t n,
                                                               float* out_m, float* out_v) {
  chain_start();
  const int64_t block = static_cast<int64_t>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5);
  if (block * kBlock >= n) return;
  const uintptr_t at = reinterpret_cast<uintptr_t>(m) | reinterpret_cast<uintptr_t>(v);
  const bool aligned = (at & 3) == 0 && aligned16(out_m) && aligned16(out_v);
  const float sm = m_scale[block], sv = v_scale[block];
  const int64_t place = block * kBlock + (threadIdx.x & 31) * 4;
  if (aligned && (block + 1) * kBlock <= n) {
    decode_block<true>(m + place, v + place, sm, sv, 0, out_m + place, out_v + place);
  } else {
    decode_block<false>(m + place, v + place, sm, sv, n - place, out_m + place, out_v + place);
  }
}

template <typename T, bool EIGHT, int N>
int launch_adamw(const AdamCommon& common, const rfm_adamw_tensor* tensors, int first, int last, bool& started,
                 cudaStream_t s) {
  AdamArgs<N> a;
  a.c = common;
  int64_t chunks = 0;
  int k = 0;
  for (int i = first; i < last; ++i) {
    const rfm_adamw_tensor& t = tensors[i];
    if (t.numel == 0) continue;
    a.t[k++] = AdamTensor{t.param,           t.grad,
                          t.exp_avg,         t.exp_avg_sq,
                          t.exp_avg_scale,   t.exp_avg_sq_scale,
                          t.numel,           static_cast<int32_t>(chunks),
                          static_cast<uint32_t>(i)};
    chunks += (t.numel + kChunk - 1) / kChunk;
    if (chunks > 0x7fffffff) return RFM_ERR_UNSUPPORTED;
  }
  if (k == 0) return RFM_OK;
  a.c.count = k;
  const Chain chain = started ? Chain::kNext : Chain::kFirst;
  started = true;
  return launch_chained(chain, adamw_kernel<T, EIGHT, N>, dim3(static_cast<unsigned>(chunks)), kThreads, 0, 1,
                        s, a);
}

template <typename T, bool EIGHT>
int run_adamw(const AdamCommon& c, const rfm_adamw_tensor* tensors, int count, cudaStream_t s) {
  bool started = c.device_s != nullptr;  // one of the call's kernels has been launched
  if (count <= kSmallTable) return launch_adamw<T, EIGHT, kSmallTable>(c, tensors, 0, count, started, s);
  for (int first = 0; first < count; first += kLargeTable) {
    const int last = count - first < kLargeTable ? count : first + kLargeTable;
    const int rc = launch_adamw<T, EIGHT, kLargeTable>(c, tensors, first, last, started, s);
    if (rc != RFM_OK) return rc;
  }
  return RFM_OK;
}

}  // namespace
}  // namespace rfm

extern "C" int rfm_adamw(const rfm_adamw_tensor* tensors, int count, int dtype, int moment_bits, double lr,
                         double beta1, double beta2, double eps, double weight_decay, int64_t step,
                         const float* device_lr, const int64_t* device_step, const float* grad_scale,
                         void* workspace, void* stream) {
  using namespace rfm;
  if (count < 0 || (count > 0 && tensors == nullptr) || !dtype_known(dtype) ||
      (moment_bits != 8 && moment_bits != 32)) {
    return RFM_ERR_INVALID_ARGUMENT;
  }
  if (!(beta1 >= 0.0 && beta1 < 1.0) || !(beta2 >= 0.0 && beta2 < 1.0) || !(eps >= 0.0) || !(lr >= 0.0) ||
      !(weight_decay >= 0.0) || (device_step == nullptr && step < 1)) {
    return RFM_ERR_INVALID_ARGUMENT;
  }
  const bool on_device = device_lr != nullptr || device_step != nullptr;
  if (on_device && (workspace == nullptr || !aligned16(workspace))) return RFM_ERR_INVALID_ARGUMENT;
  const uintptr_t elem = static_cast<uintptr_t>(dtype_bytes(dtype)) - 1;
  bool any = false;
  for (int i = 0; i < count; ++i) {
    const rfm_adamw_tensor& t = tensors[i];
    if (t.numel < 0 || t.reserved != 0) return RFM_ERR_INVALID_ARGUMENT;
    if (t.numel == 0) continue;
    any = true;
    if (t.numel > (int64_t(1) << 42)) return RFM_ERR_UNSUPPORTED;
    if (t.param == nullptr || t.grad == nullptr || t.exp_avg == nullptr || t.exp_avg_sq == nullptr) {
      return RFM_ERR_INVALID_ARGUMENT;
    }
    if (((reinterpret_cast<uintptr_t>(t.param) | reinterpret_cast<uintptr_t>(t.grad)) & elem) != 0) {
      return RFM_ERR_INVALID_ARGUMENT;
    }
    const uintptr_t state = moment_bits == 32 ? reinterpret_cast<uintptr_t>(t.exp_avg) |
                                                    reinterpret_cast<uintptr_t>(t.exp_avg_sq)
                                              : reinterpret_cast<uintptr_t>(t.exp_avg_scale) |
                                                    reinterpret_cast<uintptr_t>(t.exp_avg_sq_scale);
    if ((state & 3) != 0) return RFM_ERR_INVALID_ARGUMENT;
    if (moment_bits == 8 && (t.exp_avg_scale == nullptr || t.exp_avg_sq_scale == nullptr)) {
      return RFM_ERR_INVALID_ARGUMENT;
    }
  }
  if (!any) return RFM_OK;
  AdamCommon c{};
  c.b1 = static_cast<float>(beta1);
  c.b2 = static_cast<float>(beta2);
  c.one_b1 = static_cast<float>(1.0 - beta1);
  c.one_b2 = static_cast<float>(1.0 - beta2);
  c.eps = static_cast<float>(eps);
  c.grad_scale = grad_scale;
  cudaStream_t s = as_stream(stream);
  if (on_device) {
    AdamScalars* out = static_cast<AdamScalars*>(workspace);
    const int rc = launch_chained(Chain::kFirst, adam_scalars_kernel, dim3(1), 1, 0, 1, s, device_lr, device_step, lr,
                                  beta1, beta2, weight_decay, step, out);
    if (rc != RFM_OK) return rc;
    c.device_s = out;
  } else {
    c.s = adam_scalars(lr, beta1, beta2, weight_decay, step);
  }
  if (moment_bits == 8) {
    if (dtype == RFM_DTYPE_F32) return run_adamw<float, true>(c, tensors, count, s);
    if (dtype == RFM_DTYPE_BF16) return run_adamw<__nv_bfloat16, true>(c, tensors, count, s);
    return run_adamw<__half, true>(c, tensors, count, s);
  }
  if (dtype == RFM_DTYPE_F32) return run_adamw<float, false>(c, tensors, count, s);
  if (dtype == RFM_DTYPE_BF16) return run_adamw<__nv_bfloat16, false>(c, tensors, count, s);
  return run_adamw<__half, false>(c, tensors, count, s);
}

extern "C" int rfm_adamw_moments(const void* exp_avg, const void* exp_avg_sq, const float* exp_avg_scale,
                                 const float* exp_avg_sq_scale, int64_t numel, float* out_avg, float* out_avg_sq,
                                 void* stream) {
  using namespace rfm;
  if (numel < 0) return RFM_ERR_INVALID_ARGUMENT;
  if (numel == 0) return RFM_OK;
  if (numel > (int64_t(1) << 41)) return RFM_ERR_UNSUPPORTED;
  if (exp_avg == nullptr || exp_avg_sq == nullptr || exp_avg_scale == nullptr || exp_avg_sq_scale == nullptr ||
      out_avg == nullptr || out_avg_sq == nullptr) {
    return RFM_ERR_INVALID_ARGUMENT;
  }
  const int64_t per = static_cast<int64_t>(kThreads / 32) * kBlock;
  const dim3 grid(static_cast<unsigned>((numel + per - 1) / per));
  return launch_chained(Chain::kFirst, adam_moments_kernel, grid, kThreads, 0, 1, as_stream(stream),
                        static_cast<const uint8_t*>(exp_avg), static_cast<const uint8_t*>(exp_avg_sq), exp_avg_scale,
                        exp_avg_sq_scale, numel, out_avg, out_avg_sq);
}
