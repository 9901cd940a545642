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
// tensor), so no upload precedes the launch.  One CTA takes 2048 consecutive
// elements of one tensor, a warp a block of 256, a lane two quads of it, so that
// every access of a warp is contiguous.
#include <math.h>

#include "rfm_types.cuh"

namespace rfm {
namespace {

constexpr int kThreads = 256;
constexpr int kBlock = RFM_MOMENT_BLOCK;          // elements that share a scale
constexpr int kChunk = 2048;                      // elements of one CTA
constexpr int kWarpBlocks = kChunk / kBlock / 8;  // blocks of one warp
static_assert(kBlock == 32 * 8, "a warp holds one block, eight elements a lane");
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
  *out = adam_scalars(device_lr != nullptr ? static_cast<double>(*device_lr) : lr, b1, b2, wd,
                      device_step != nullptr ? *device_step : step);
}

template <typename T>
__device__ __forceinline__ void load_quad(float (&r)[4], const T* p, int64_t i, int64_t n, bool vec) {
  if (vec && i + 4 <= n) {
    const Pack<T, 4> q = *reinterpret_cast<const Pack<T, 4>*>(p + i);
#pragma unroll
    for (int j = 0; j < 4; ++j) r[j] = to_float(q.v[j]);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) r[j] = i + j < n ? to_float(p[i + j]) : 0.f;
  }
}

template <typename T>
__device__ __forceinline__ void store_quad(const float (&r)[4], T* p, int64_t i, int64_t n, bool vec) {
  if (vec && i + 4 <= n) {
    Pack<T, 4> q;
#pragma unroll
    for (int j = 0; j < 4; ++j) q.v[j] = from_float<T>(r[j]);
    *reinterpret_cast<Pack<T, 4>*>(p + i) = q;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (i + j < n) p[i + j] = from_float<T>(r[j]);
  }
}

// Four codes as one word, element j in byte j.
__device__ __forceinline__ uint32_t load_codes(const void* base, int64_t i, int64_t n, bool vec) {
  const uint8_t* p = static_cast<const uint8_t*>(base) + i;
  if (vec && i + 4 <= n) return *reinterpret_cast<const uint32_t*>(p);
  uint32_t w = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (i + j < n) w |= static_cast<uint32_t>(p[j]) << (8 * j);
  return w;
}

__device__ __forceinline__ void store_codes(uint32_t w, void* base, int64_t i, int64_t n, bool vec) {
  uint8_t* p = static_cast<uint8_t*>(base) + i;
  if (vec && i + 4 <= n) {
    *reinterpret_cast<uint32_t*>(p) = w;
    return;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (i + j < n) p[j] = static_cast<uint8_t>(w >> (8 * j));
}

constexpr float kInv127 = static_cast<float>(1.0 / 127.0);
constexpr float kInv255 = static_cast<float>(1.0 / 255.0);

// Byte j of a word as a float, through the mantissa of 2^23 (conversions run at
// an eighth of the rate of additions).
__device__ __forceinline__ float byte_float(uint32_t w, int j) {
  return __uint_as_float(__byte_perm(w, 0x4B000000u, 0x7440u + j)) - 8388608.f;
}

// `flipped`: the word of codes with every byte's top bit inverted (c + 128).
__device__ __forceinline__ float decode_m(uint32_t flipped, int j, float scale) {
  const float a = __fmul_rn(byte_float(flipped, j) - 128.f, kInv127);
  return __fmul_rn(scale, __fmul_rn(a, fabsf(a)));
}

__device__ __forceinline__ float decode_v(uint32_t codes, int j, float scale) {
  float b = __fmul_rn(byte_float(codes, j), kInv255);
  b = __fmul_rn(b, b);
  return __fmul_rn(scale, __fmul_rn(b, b));
}

// The codes by definition.  A NaN quotient (a block of zeros, or of infinities)
// converts to code 0.
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

__device__ __forceinline__ uint32_t quick_floor(float root, float top, uint32_t bits16, bool& sure) {
  // 1 + the random fraction, exactly: its 16 bits at the top of the mantissa
  const float one_u = __uint_as_float(0x3F800000u | (bits16 & 0x7fff80u));
  const float x1 = fmaf(root, top, one_u);           // x + 1
  const float low = __fadd_rd(x1, 8388607.f);        // 2^23 + floor(x)
  const float part = x1 - (low - 8388607.f);         // x - floor(x)
  sure = sure && fabsf(part - 0.5f) < 0.5f - kNear;
  return __float_as_uint(low) & 0xffu;
}

// The codes of four elements, element j in byte j; `inv`: the scale's reciprocal
//.
__device__ __forceinline__ uint32_t encode_m(const float (&m)[4], float scale, float inv, const uint32_t (&h)[4]) {
  uint32_t q[4];
  bool sure = true;
#pragma unroll
  for (int j = 0; j < 4; ++j) q[j] = quick_floor(sqrt_fast(fabsf(m[j]) * inv), 127.f, h[j] << 7, sure);
  if (!sure) {  // a scale of 0 ends here too: its block is all zeros
#pragma unroll
    for (int j = 0; j < 4; ++j) q[j] = scale == 0.f ? 0u : exact_code_m(m[j], scale, h[j]);
  }
  uint32_t w = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) w |= ((m[j] < 0.f ? 0u - q[j] : q[j]) & 0xffu) << (8 * j);
  return w;
}

__device__ __forceinline__ uint32_t encode_v(const float (&v)[4], float scale, float inv, const uint32_t (&h)[4]) {
  uint32_t q[4];
  bool sure = true;
#pragma unroll
  for (int j = 0; j < 4; ++j) q[j] = quick_floor(sqrt_fast(sqrt_fast(v[j] * inv)), 255.f, h[j] >> 9, sure);
  if (!sure) {
#pragma unroll
    for (int j = 0; j < 4; ++j) q[j] = scale == 0.f ? 0u : exact_code_v(v[j], scale, h[j]);
  }
  uint32_t w = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) w |= (v[j] > 0.f ? max(q[j], 1u) : q[j]) << (8 * j);
  return w;
}

// Largest of a warp's non-negative values (their bit patterns order as the
// values do, and a NaN's is above infinity's, so a NaN is kept).
__device__ __forceinline__ float warp_max_bits(uint32_t bits) {
  return __uint_as_float(__reduce_max_sync(kFullMask, bits));
}

template <typename T, bool EIGHT, int N>
__global__ void __launch_bounds__(kThreads, 4) adamw_kernel(const __grid_constant__ AdamArgs<N> a) {
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
  const int64_t n = t.numel;
  T* param = static_cast<T*>(t.param);
  const T* grad = static_cast<const T*>(t.grad);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t base = static_cast<int64_t>(chunk - t.first_chunk) * kChunk + warp * (kWarpBlocks * kBlock);
  const uintptr_t wide = reinterpret_cast<uintptr_t>(t.param) | reinterpret_cast<uintptr_t>(t.grad);
  const uintptr_t state = reinterpret_cast<uintptr_t>(t.m) | reinterpret_cast<uintptr_t>(t.v);
  const bool vec = (wide & (4 * sizeof(T) - 1)) == 0 && (state & (EIGHT ? 3 : 15)) == 0;

  float p[kWarpBlocks][2][4], g[kWarpBlocks][2][4], m[kWarpBlocks][2][4], v[kWarpBlocks][2][4];
  uint32_t cm[kWarpBlocks][2], cv[kWarpBlocks][2];
  float sm[kWarpBlocks], sv[kWarpBlocks];
#pragma unroll
  for (int b = 0; b < kWarpBlocks; ++b) {
    const int64_t first = base + b * kBlock;
    if (EIGHT) {
      sm[b] = first < n ? t.m_scale[first / kBlock] : 0.f;
      sv[b] = first < n ? t.v_scale[first / kBlock] : 0.f;
    }
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const int64_t i = first + q * 128 + lane * 4;
      load_quad<T>(g[b][q], grad, i, n, vec);
      load_quad<T>(p[b][q], param, i, n, vec);
      if (EIGHT) {
        cm[b][q] = load_codes(t.m, i, n, vec);
        cv[b][q] = load_codes(t.v, i, n, vec);
      } else {
        load_quad<float>(m[b][q], static_cast<const float*>(t.m), i, n, vec);
        load_quad<float>(v[b][q], static_cast<const float*>(t.v), i, n, vec);
      }
    }
  }

#pragma unroll
  for (int b = 0; b < kWarpBlocks; ++b) {
    uint32_t top_m = 0, top_v = 0;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float& pj = p[b][q][j];
        float& mj = m[b][q][j];
        float& vj = v[b][q][j];
        if (EIGHT) {
          mj = decode_m(cm[b][q] ^ 0x80808080u, j, sm[b]);
          vj = decode_v(cv[b][q], j, sv[b]);
        }
        const float gj = __fmul_rn(g[b][q][j], grad_scale);
        mj = __fadd_rn(__fmul_rn(mj, a.c.b1), __fmul_rn(gj, a.c.one_b1));
        vj = __fadd_rn(__fmul_rn(vj, a.c.b2), __fmul_rn(__fmul_rn(gj, gj), a.c.one_b2));
        // approximate root and quotient: 2^-22 of an update that is a small part of the parameter
        float root;  // of subnormal values too: with eps 0 a root of 0 would be divided by
        asm("sqrt.approx.f32 %0, %1;" : "=f"(root) : "f"(vj));
        const float denom = fmaf(root, s.inv_sqrt_bc2, a.c.eps);
        pj = fmaf(pj, s.keep, -s.step_size * __fdividef(mj, denom));
        if (EIGHT) {
          // elements past the tensor's end count as zeros whatever their block's scale is
          const bool in = base + b * kBlock + q * 128 + lane * 4 + j < n;
          top_m = max(top_m, in ? __float_as_uint(mj) & 0x7fffffffu : 0u);
          top_v = max(top_v, in ? __float_as_uint(vj) & 0x7fffffffu : 0u);
        }
      }
      const int64_t i = base + b * kBlock + q * 128 + lane * 4;
      store_quad<T>(p[b][q], param, i, n, vec);
      if (!EIGHT) {
        store_quad<float>(m[b][q], static_cast<float*>(t.m), i, n, vec);
        store_quad<float>(v[b][q], static_cast<float*>(t.v), i, n, vec);
      }
    }
    if (EIGHT) {
      const uint32_t key = mix(t.ordinal * 0x632BE5ABu + s.seed);
      const float new_sm = warp_max_bits(top_m), new_sv = warp_max_bits(top_v);
      const float inv_m = __frcp_rn(new_sm), inv_v = __frcp_rn(new_sv);
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const int64_t i = base + b * kBlock + q * 128 + lane * 4;
        uint32_t h[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) h[j] = mix(static_cast<uint32_t>(i + j) + key);
        store_codes(encode_m(m[b][q], new_sm, inv_m, h), t.m, i, n, vec);
        store_codes(encode_v(v[b][q], new_sv, inv_v, h), t.v, i, n, vec);
      }
      const int64_t first = base + b * kBlock;
      if (lane == 0 && first < n) {
        t.m_scale[first / kBlock] = new_sm;
        t.v_scale[first / kBlock] = new_sv;
      }
    }
  }
}

// The values that 8-bit moments stand for; a warp decodes one block.
__global__ void __launch_bounds__(kThreads) adam_moments_kernel(const void* m, const void* v, const float* m_scale,
                                                               const float* v_scale, int64_t n, float* out_m,
                                                               float* out_v) {
  const int lane = threadIdx.x & 31;
  const int64_t block = static_cast<int64_t>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5);
  if (block * kBlock >= n) return;
  const uintptr_t at = reinterpret_cast<uintptr_t>(m) | reinterpret_cast<uintptr_t>(v);
  const bool vec = (at & 3) == 0 && aligned16(out_m) && aligned16(out_v);
  const float sm = m_scale[block], sv = v_scale[block];
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const int64_t i = block * kBlock + q * 128 + lane * 4;
    const uint32_t cm = load_codes(m, i, n, vec), cv = load_codes(v, i, n, vec);
    float dm[4], dv[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      dm[j] = decode_m(cm ^ 0x80808080u, j, sm);
      dv[j] = decode_v(cv, j, sv);
    }
    store_quad<float>(dm, out_m, i, n, vec);
    store_quad<float>(dv, out_v, i, n, vec);
  }
}

template <typename T, bool EIGHT, int N>
int launch_adamw(const AdamCommon& common, const rfm_adamw_tensor* tensors, int first, int last, cudaStream_t s) {
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
  adamw_kernel<T, EIGHT, N><<<static_cast<unsigned>(chunks), kThreads, 0, s>>>(a);
  return launch_status();
}

template <typename T, bool EIGHT>
int run_adamw(const AdamCommon& c, const rfm_adamw_tensor* tensors, int count, cudaStream_t s) {
  if (count <= kSmallTable) return launch_adamw<T, EIGHT, kSmallTable>(c, tensors, 0, count, s);
  for (int first = 0; first < count; first += kLargeTable) {
    const int last = count - first < kLargeTable ? count : first + kLargeTable;
    const int rc = launch_adamw<T, EIGHT, kLargeTable>(c, tensors, first, last, s);
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
    adam_scalars_kernel<<<1, 1, 0, s>>>(device_lr, device_step, lr, beta1, beta2, weight_decay, step, out);
    const int rc = launch_status();
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
  adam_moments_kernel<<<static_cast<unsigned>((numel + per - 1) / per), kThreads, 0, as_stream(stream)>>>(
      exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale, numel, out_avg, out_avg_sq);
  return launch_status();
}
