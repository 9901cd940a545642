// The layers' matrix products on the 5th-generation tensor cores, bf16 and fp16.
//
//   forward     out = act(x W^T + bias) + residual        [rows, out]
//   backward    dP = dY act'(pre),  dX = dP W,  dW = dP^T X,  dbias = sum_rows dP
//
// One kernel computes D[M, N] = sum_k A[m, k] B[n, k] for all three products;
// they differ in which dimension of an operand is contiguous in memory: k for
// both (forward), k for A and n for B (dX), m and n (dW).  TMA reads all of them
// as stored, so nothing is transposed.
//
// Structure.  A persistent CTA walks 128 x BN tiles: one thread issues the TMA
// loads of 64-deep operand slices into a ring of stages, one issues tcgen05.mma
// (fp32 accumulators in tensor memory, two of them, so that a tile's products
// overlap the previous tile's epilogue), and 16 warps (8 for the narrow tile) read
// the accumulators back, apply bias, activation and residual in fp32, round once
// and store boxes of 32 rows through shared memory by TMA.  A warp can only read
// its own quarter of the lanes; the four warps of a quarter share the columns, one
// box a warp: shallow products are bound by the epilogue's latencies (tensor
// memory, the proxy fence, the store's read), which more warps overlap.  The
// residual is fetched by TMA into the box it is added in, while the products run.
//
// Few tiles leave SMs idle while the contraction is long (dW: a layer's weight
// is a handful of tiles over tens of thousands of rows; one row against a wide
// layer): the contraction is then split, each part leaves fp32 sums in the
// workspace, and a second kernel adds the parts in their order and applies the
// epilogue.  No atomics: the same bits on every run.
//
// The gradient of an activation and dX come from one kernel where a row of dX is
// short (grad_x_kernel); else dP has a pass of its own.
//
// Every wait on a barrier is bounded.  One that runs out marks the call as
// failed (rfm_linear_faults) and every role leaves its loop.
#include <math.h>

#include <type_traits>

#include "rfm_tcgen05.cuh"
#include "rfm_types.cuh"

namespace rfm {
namespace {

constexpr int kBM = 128;
constexpr int kBK = 64;  // one 128-byte row of 16-bit elements
constexpr int kMaxSplits = 32;
constexpr uint32_t kWaitTries = 1u << 22;       // of a wait for what is in flight after a failure
constexpr long long kWaitCycles = 1ll << 35;    // of any other wait: some 18 s, the deepest product takes less than 10

__device__ int g_linear_faults = 0;

// Shared memory of one CTA.  CG 2: two CTAs share a tile of 256 rows; each holds
// its own 128 rows of A and half of B's.
template <int BN, int CG>
struct Shape {
  static constexpr int kBRows = BN / CG;
  static constexpr int kABytes = kBM * kBK * 2;
  static constexpr int kBBytes = kBRows * kBK * 2;
  static constexpr int kStageBytes = kABytes + kBBytes;
  // four warps a quarter of the lanes (two for 64 columns), each with one box of 32 rows
  static constexpr int kEpiWarps = BN == 64 ? 8 : 16;
  static constexpr int kLoadWarp = kEpiWarps;
  static constexpr int kMmaWarp = kEpiWarps + 1;
  static constexpr int kThreads = 32 * (kEpiWarps + 2);
  static constexpr int kBoxCols = BN / (kEpiWarps / 4);  // 64, 32, 32
  static constexpr int kBoxBytes = 32 * kBoxCols * 2;
  static constexpr int kBoxesBytes = kEpiWarps * kBoxBytes;
  static constexpr int kBiasBytes = kEpiWarps * 32 * 4;  // 32 columns a warp
  static constexpr int kSmem = 232448;                   // of one CTA
  static constexpr int kStages = (kSmem - kBoxesBytes - kBiasBytes - 512) / kStageBytes;  // pair: 5; 3, 6, 8
  static constexpr int kBoxes = kStages * kStageBytes;
  static constexpr int kBias = kBoxes + kBoxesBytes;
  static constexpr int kBars = kBias + kBiasBytes;
  // full and empty per stage, full and empty per accumulator, residual per warp
  static constexpr int kNumBars = 2 * kStages + 4 + kEpiWarps;
  static constexpr int kFlags = kBars + kNumBars * 8;
  static constexpr int kBytes = kFlags + 16;
  static_assert(kBytes <= kSmem, "shared memory of one CTA");
};

struct GemmArgs {
  int64_t m;
  int32_t n;
  int32_t tiles_m, tiles_n;
  int32_t k_blocks;       // of the whole contraction
  int32_t splits;
  int32_t activation;     // of the second kernel; the product's own is a template argument
  int32_t bias_dtype;
  int32_t tma_out, tma_res;
  const void* bias;
  const void* residual;   // null: none
  int64_t ld_res;
  void* out;              // [m, n], contiguous
  void* pre;              // null: not kept
  float* partial;         // splits > 1: [splits][m][n]
};

struct GemmMaps {
  CUtensorMap a, b, out, pre, res;
};

__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// The normal distribution's cdf at two values: its tail q(|v|) as 2 to a polynomial.
// log2 q is smooth where q itself falls over many orders; the coefficients are a
// least-maximum fit of degree 8 on [0, 6]: q is off by at most 2.5e-6 of itself
// up to 3 and 1.2e-5 up to 6 (below 2^-30 there), |v| q by 3e-7: far under half a
// step of fp16 anywhere, and of bf16 down to v = -6.9.  Below that, where |v| q is
// 1.4e-11 and less, bf16 still has steps: there q is off by more than half of one
// (2.6 % of itself at -8, 45 % at -10), in values that 1 + erf in fp32 gives as 0
// from -5.6 on.  Beyond 6 the polynomial keeps falling and q underflows to 0 (at an
// infinity too; a NaN stays one).  Seven instructions a value and one of the
// special-function unit, against some 25 of erff.
__device__ __forceinline__ Pair normal_cdf(Pair v) {
  const float2 f = split(v);
  const Pair z = pair(fabsf(f.x), fabsf(f.y));
  Pair p = fma(both(-1.2245089919815655e-07f), z, both(8.983980137600156e-07f));
  p = fma(p, z, both(3.7126268580323085e-05f));
  p = fma(p, z, both(-8.181885350495577e-04f));
  p = fma(p, z, both(8.22749175131321e-03f));
  p = fma(p, z, both(-5.3588107228279114e-02f));
  p = fma(p, z, both(-4.587007761001587e-01f));
  p = fma(p, z, both(-1.1511954069137573f));
  p = fma(p, z, both(-9.999973773956299e-01f));
  const float2 e = split(p);
  const float qx = exp2_fast(e.x), qy = exp2_fast(e.y);
  return pair(f.x > 0.f ? 1.f - qx : qx, f.y > 0.f ? 1.f - qy : qy);
}

__device__ __forceinline__ float relu(float v) {  // a NaN stays one
  float r;
  asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(r) : "f"(v));
  return r;
}

__device__ __forceinline__ Pair activate(Pair v, int act) {
  if (act == RFM_ACT_RELU) {
    const float2 f = split(v);
    return pair(relu(f.x), relu(f.y));
  }
  return act == RFM_ACT_GELU ? v * normal_cdf(v) : v;
}

__device__ __forceinline__ float activate(float v, int act) { return split(activate(both(v), act)).x; }

// dy act'(v): act' is 0 at relu's border, and cdf(v) + v pdf(v) for gelu.  What
// relu cut leaves a 0 whatever dy is there (an infinity times 0 would be NaN), and
// a NaN that it kept passes dy on.
__device__ __forceinline__ Pair times_activate_grad(Pair dy, Pair v, int act) {
  const float2 f = split(v);
  if (act == RFM_ACT_RELU) {
    const float2 d = split(dy);
    return pair(f.x <= 0.f ? 0.f : d.x, f.y <= 0.f ? 0.f : d.y);
  }
  if (act == RFM_ACT_GELU) {
    // pdf(v) = 2^(-v^2 log2(e) / 2) / sqrt(2 pi)
    const float2 e = split(v * v * both(-0.72134752044448170f));
    const Pair pdf = pair(exp2_fast(e.x), exp2_fast(e.y));
    return dy * fma(v * both(0.39894228040143268f), pdf, normal_cdf(v));
  }
  return dy;
}

// `pre` is kept in the operands' 16 bits, half the bytes of fp32 both ways: the
// derivative of gelu is then taken at a value half a step off (as where a product
// and a gelu are two 16-bit operations).  With dP's rounding this puts the gradients
// of 13608 x 384 -> 1536 fp16 3.0e-4 from 64 bits, 2.1e-4 with both in fp32.
// It is kept finite where it is: a value beyond the type's range would come back
// as an infinity, whose gelu gradient is NaN, where the value's is 0 or 1.  An
// infinity stays one.
template <typename T>
__device__ __forceinline__ float keep_finite(float v) {
  const float most = std::is_same<T, __half>::value ? 65504.f : 3.3895313892515355e38f;
  return fabsf(v) > most && !isinf(v) ? copysignf(most, v) : v;
}

// Adds two values to two registers that hold floats.
__device__ __forceinline__ void add2(uint32_t& a, uint32_t& b, float x, float y) {
  const float2 s = split(pair(__uint_as_float(a), __uint_as_float(b)) + pair(x, y));
  a = __float_as_uint(s.x);
  b = __float_as_uint(s.y);
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return reinterpret_cast<const uint32_t&>(v);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 v = __floats2half2_rn(a, b);
  return reinterpret_cast<const uint32_t&>(v);
}
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t v);
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t v) {
  return __bfloat1622float2(reinterpret_cast<const __nv_bfloat162&>(v));
}
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t v) {
  return __half22float2(reinterpret_cast<const __half2&>(v));
}

// A wait that gives up after kWaitCycles, or as soon as another role has given up.
__device__ __forceinline__ bool bounded_wait(uint32_t bar, uint32_t parity, volatile int* dead) {
  if (mbar_try(bar, parity)) return true;
  const long long start = clock64();
  do {
#pragma unroll 1
    for (int i = 0; i < 64; ++i)
      if (mbar_try(bar, parity)) return true;
    if (*dead) return false;
  } while (clock64() - start < kWaitCycles);
  *dead = 1;
  atomicExch(&g_linear_faults, 1);
  return false;
}

// Work item `w` of the grid: a part of the contraction of one tile.  Tiles run
// down 16 rows of tiles before the next column, so that a wave's operands
// overlap in L2.
struct Work {
  int tile_m, tile_n, split, k0, k1;
};

__device__ __forceinline__ Work work_item(const GemmArgs& a, uint32_t w) {
  Work r;
  uint32_t tile = w;
  r.split = 0;
  r.k0 = 0;
  r.k1 = a.k_blocks;
  if (a.splits > 1) {
    const uint32_t splits = static_cast<uint32_t>(a.splits);
    tile = w / splits;
    r.split = static_cast<int>(w - tile * splits);
    // whole slices to every part, one more to the first ones
    const int each = a.k_blocks / a.splits, more = a.k_blocks - each * a.splits;
    r.k0 = each * r.split + min(r.split, more);
    r.k1 = r.k0 + each + (r.split < more ? 1 : 0);
  }
  constexpr uint32_t kGroup = 16;
  const uint32_t per_group = kGroup * static_cast<uint32_t>(a.tiles_n);
  const uint32_t group = tile / per_group, inside = tile - group * per_group;
  const uint32_t height = min(kGroup, static_cast<uint32_t>(a.tiles_m) - group * kGroup);
  const uint32_t column = height == kGroup ? inside / kGroup : inside / height;
  r.tile_m = static_cast<int>(group * kGroup + inside - column * height);
  r.tile_n = static_cast<int>(column);
  return r;
}

template <typename T, int BN, int CG, bool A_MN, bool B_MN, int ACT>
__global__ void __launch_bounds__(Shape<BN, CG>::kThreads, 1)
    gemm_kernel(const __grid_constant__ GemmMaps maps, const __grid_constant__ GemmArgs a) {
  using S = Shape<BN, CG>;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t base = smem_u32(smem);
  const uint32_t bars = base + S::kBars;
  const uint32_t full = bars, empty = bars + 8 * S::kStages;
  const uint32_t acc_full = empty + 8 * S::kStages, acc_empty = acc_full + 16, res_full = acc_empty + 16;
  volatile int* dead = reinterpret_cast<volatile int*>(smem + S::kFlags);
  const int warp = static_cast<int>(threadIdx.x) >> 5, lane = static_cast<int>(threadIdx.x) & 31;
  constexpr uint32_t kTmemColumns = 2 * BN;
  // of a pair, CTA 0 issues the products and counts both CTAs' loads
  const uint32_t rank = CG == 2 ? cluster_rank() : 0u;

  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (threadIdx.x == 0) {
    *dead = 0;
    if ((base & 1023u) != 0) {  // the swizzles count on it; never expected
      *dead = 1;
      atomicExch(&g_linear_faults, 1);
    }
    for (int i = 0; i < S::kStages; ++i) {
      mbar_init(full + 8 * i, 1);
      mbar_init(empty + 8 * i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(acc_full + 8 * i, 1);
      mbar_init(acc_empty + 8 * i, S::kEpiWarps * CG);
    }
    for (int i = 0; i < S::kEpiWarps; ++i) mbar_init(res_full + 8 * i, 1);
    mbar_init_fence();
    tma_prefetch_map(&maps.a);
    tma_prefetch_map(&maps.b);
  }
  if (warp == S::kMmaWarp) tmem_alloc<CG>(base + S::kFlags + 4, kTmemColumns);
  tc_fence_before();
  if (CG == 2) {
    cluster_sync();
  } else {
    __syncthreads();
  }
  tc_fence_after();
  grid_dependency_wait();  // the set-up above touches nothing that the kernel before writes
  const uint32_t tmem = *reinterpret_cast<const volatile uint32_t*>(smem + S::kFlags + 4);
  const uint32_t items = static_cast<uint32_t>(a.tiles_m) * a.tiles_n * a.splits;  // below 2^31
  const uint32_t first = blockIdx.x / CG, stride = gridDim.x / CG;

  if (warp == S::kLoadWarp) {
    if (lane == 0) {
      uint32_t stage = 0, phase = 0, issued = 0;
      bool ok = true;
      for (uint32_t w = first; ok && w < items; w += stride) {
        const Work t = work_item(a, w);
        const int m0 = (t.tile_m * CG + static_cast<int>(rank)) * kBM;
        const int n0 = t.tile_n * BN + static_cast<int>(rank) * S::kBRows;
        for (int kb = t.k0; kb < t.k1; ++kb) {
          if (!bounded_wait(empty + 8 * stage, phase ^ 1u, dead)) {
            ok = false;
            break;
          }
          uint32_t bar = full + 8 * stage;
          const uint32_t sa = base + stage * S::kStageBytes, sb = sa + S::kABytes;
          if (rank == 0) mbar_expect(bar, CG * S::kStageBytes);
          if (CG == 2) bar = map_rank(bar, 0);
          const auto load = [&](uint32_t dst, const CUtensorMap* map, int x, int y) {
            if (CG == 2) {
              tma_load_2d_pair(dst, map, x, y, bar);
            } else {
              tma_load_2d(dst, map, x, y, bar);
            }
          };
          if (A_MN) {
#pragma unroll
            for (int j = 0; j < kBM / 64; ++j) load(sa + j * 8192, &maps.a, m0 + j * 64, kb * kBK);
          } else {
            load(sa, &maps.a, kb * kBK, m0);
          }
          if (B_MN) {
#pragma unroll
            for (int j = 0; j < S::kBRows / 64; ++j) load(sb + j * 8192, &maps.b, n0 + j * 64, kb * kBK);
          } else {
            load(sb, &maps.b, kb * kBK, n0);
          }
          if (issued < S::kStages) ++issued;
          if (++stage == S::kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      // Every arrival on this CTA's `empty` barriers has come before it leaves: of a
      // pair, CTA 0's products signal CTA 1's too, and nothing else waits for the
      // last of them there.
      for (int i = 0; ok && i < S::kStages; ++i) {
        ok = bounded_wait(empty + 8 * stage, phase ^ 1u, dead);
        if (ok && ++stage == S::kStages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      if (!ok && rank == 0) {
        // the copies in flight (a pair's: of both) land before the shared memory is given up
        for (uint32_t i = 0; i < issued; ++i) {
          if (stage == 0) {
            stage = S::kStages;
            phase ^= 1u;
          }
          --stage;
          for (uint32_t k = 0; k < kWaitTries && !mbar_try(full + 8 * stage, phase); ++k) {
          }
        }
      }
    }
  } else if (warp == S::kMmaWarp) {
    if (lane == 0 && rank == 0) {
      constexpr int kType = std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
      constexpr uint32_t kInstr = mma_instr(kType, A_MN, B_MN, kBM * CG, BN);
      constexpr uint32_t kAStep = A_MN ? 2048 : 32, kBStep = B_MN ? 2048 : 32;  // bytes of 16 along k
      uint32_t stage = 0, phase = 0, acc = 0, acc_phase = 0;
      bool ok = true;
      for (uint32_t w = first; ok && w < items; w += stride) {
        const Work t = work_item(a, w);
        if (!bounded_wait(acc_empty + 8 * acc, acc_phase ^ 1u, dead)) break;
        tc_fence_after();
        const uint32_t d = tmem + acc * BN;
        for (int kb = t.k0; kb < t.k1; ++kb) {
          if (!bounded_wait(full + 8 * stage, phase, dead)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t sa = base + stage * S::kStageBytes, sb = sa + S::kABytes;
#pragma unroll
          for (int k = 0; k < kBK / 16; ++k) {
            tc_mma_f16<CG>(d, operand_desc(sa + k * kAStep, A_MN ? 8192 : 16, 1024),
                           operand_desc(sb + k * kBStep, B_MN ? 8192 : 16, 1024), kInstr, kb > t.k0 || k > 0);
          }
          tc_commit<CG>(empty + 8 * stage);
          if (++stage == S::kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (!ok) break;
        tc_commit<CG>(acc_full + 8 * acc);
        acc ^= 1u;
        if (acc == 0) acc_phase ^= 1u;
      }
      // The products in flight end before the tensor memory is given up: the
      // epilogue waits for the last accumulator's barrier, and a role that gave
      // up waits here.
      if (*dead) {
        tc_commit<CG>(acc_full + 8 * acc);
        for (uint32_t k = 0; k < kWaitTries && !mbar_try(acc_full + 8 * acc, acc_phase); ++k) {
        }
      }
    }
  } else {
    constexpr int kCols = S::kBoxCols;
    constexpr int kTurns = kCols / 32;  // 32 columns at a time in registers
    const int quarter = warp & 3, part = warp >> 2;
    const uint32_t box = base + S::kBoxes + warp * S::kBoxBytes;
    uint8_t* box_ptr = smem + S::kBoxes + warp * S::kBoxBytes;
    float* bias_smem = reinterpret_cast<float*>(smem + S::kBias) + warp * 32;
    const uint32_t res_bar = res_full + 8 * warp;
    const uint32_t released = CG == 2 ? map_rank(acc_empty, 0) : acc_empty;
    const bool whole = a.splits == 1;
    const bool has_bias = whole && a.bias != nullptr;
    const bool has_res = whole && a.residual != nullptr, has_pre = whole && a.pre != nullptr;
    // the box can only wait for the residual where `pre` does not pass through it first
    const bool tma_res = has_res && a.tma_res && !has_pre;
    // beside `pre`, the aligned residual comes straight from memory, 8 columns at a time
    const bool straight = has_res && a.tma_res && has_pre && (a.n & 7) == 0;
    uint32_t acc = 0, acc_phase = 0, res_phase = 0;
    // where a lane's 16-byte pieces of its row go in the box: the TMA swizzle of
    // its row length, which also spreads the lanes' accesses over the banks
    const int row_off = lane * kCols * 2, swz = kCols == 64 ? lane & 7 : (lane >> 1) & 3;
    const auto piece = [&](int j) { return reinterpret_cast<uint4*>(box_ptr + row_off + ((j ^ swz) << 4)); };
    // element (r, c) of the box
    const auto cell = [&](int r, int c) {
      return reinterpret_cast<T*>(box_ptr) + r * kCols +
             (((c >> 3) ^ (kCols == 64 ? r & 7 : (r >> 1) & 3)) << 3) + (c & 7);
    };

    // lane l holds the bias of its box's columns l and l + 32, read a tile ahead
    float bias[kTurns];
    const auto read_bias = [&](int tile_n) {
#pragma unroll
      for (int s = 0; s < kTurns; ++s) {
        const int col = tile_n * BN + part * kCols + s * 32 + lane;
        bias[s] = col < a.n ? load_param(a.bias, a.bias_dtype, col) : 0.f;
      }
    };
    Work next = work_item(a, min(first, items - 1));
    if (has_bias) read_bias(next.tile_n);

    for (uint32_t w = first; w < items; w += stride) {
      const Work t = next;
      const int64_t row0 = (static_cast<int64_t>(t.tile_m) * CG + rank) * kBM + quarter * 32;
      const int col0 = t.tile_n * BN + part * kCols;
      const bool inside = row0 < a.m && col0 < a.n;
      if (w + stride < items) next = work_item(a, w + stride);
      if (inside && tma_res) {
        if (lane == 0) {
          tma_wait_read<0>();
          proxy_fence();
          mbar_expect(res_bar, S::kBoxBytes);
          tma_load_2d(box, &maps.res, col0, static_cast<int>(row0), res_bar);
        }
        __syncwarp();
      }
      bool live = __all_sync(kFullMask, bounded_wait(acc_full + 8 * acc, acc_phase, dead));
      tc_fence_after();
      const uint32_t from =
          tmem + (static_cast<uint32_t>(quarter * 32) << 16) + acc * BN + part * kCols;
      const auto release = [&] {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (CG == 2) {
            mbar_arrive_cluster(released + 8 * acc);
          } else {
            mbar_arrive(released + 8 * acc);
          }
        }
      };
      // columns s * 32 .. of this lane's row, with the bias
      const auto take = [&](uint32_t(&v)[32], int s) {
        tmem_load_32(v, from + s * 32);
        if (has_bias) {
          __syncwarp();
          bias_smem[lane] = bias[s];
          __syncwarp();
        }
        tmem_wait_load(v);
        if (has_bias) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float4 q = reinterpret_cast<const float4*>(bias_smem)[j];
            add2(v[4 * j], v[4 * j + 1], q.x, q.y);
            add2(v[4 * j + 2], v[4 * j + 3], q.z, q.w);
          }
        }
      };
      // the box's last store has been read before anything is written to it
      const auto box_free = [&] {
        if (lane == 0) tma_wait_read<0>();
        __syncwarp();
      };
      const auto put = [&](const uint32_t(&v)[32], int s) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t p[4];
#pragma unroll
          for (int i = 0; i < 4; ++i)
            p[i] = pack2<T>(__uint_as_float(v[8 * j + 2 * i]), __uint_as_float(v[8 * j + 2 * i + 1]));
          *piece(s * 4 + j) = make_uint4(p[0], p[1], p[2], p[3]);
        }
      };
      // the filled box goes out: by TMA, or a lane a column where rows do not start on 16 bytes
      const auto send = [&](const CUtensorMap* map, void* to) {
        if (a.tma_out) {
          proxy_fence();
          __syncwarp();
          if (lane == 0 && live) {
            tma_store_2d(map, col0, static_cast<int>(row0), box);
            tma_commit();
          }
        } else {
          __syncwarp();
          const int rows = live ? static_cast<int>(min(a.m - row0, static_cast<int64_t>(32))) : 0;
          T* dst = static_cast<T*>(to) + row0 * a.n + col0;
#pragma unroll 8
          for (int r = 0; r < rows; ++r) {
#pragma unroll
            for (int c = lane; c < kCols; c += 32)
              if (col0 + c < a.n) dst[static_cast<int64_t>(r) * a.n + c] = *cell(r, c);
          }
          __syncwarp();
        }
      };

      if (!inside) {
        release();
        if (has_bias) read_bias(next.tile_n);
      } else if (!whole) {
        const int64_t row = row0 + lane;
        float* dst = a.partial + (static_cast<int64_t>(t.split) * a.m + row) * a.n + col0;
#pragma unroll
        for (int s = 0; s < kTurns; ++s) {
          uint32_t v[32];
          tmem_load_32(v, from + s * 32);
          tmem_wait_load(v);
          if (s == kTurns - 1) release();
          if (row >= a.m || !live) continue;
          if ((a.n & 3) == 0 && col0 + s * 32 + 32 <= a.n) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
              reinterpret_cast<uint4*>(dst + s * 32)[j] =
                  make_uint4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
          } else {
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (col0 + s * 32 + j < a.n) dst[s * 32 + j] = __uint_as_float(v[j]);
          }
        }
      } else {
        if (has_pre) {
#pragma unroll
          for (int s = 0; s < kTurns; ++s) {
            uint32_t v[32];
            take(v, s);
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = __float_as_uint(keep_finite<T>(__uint_as_float(v[j])));
            if (s == 0) box_free();
            put(v, s);
          }
          send(&maps.pre, a.pre);
        }
        if (tma_res) {
          live = __all_sync(kFullMask, bounded_wait(res_bar, res_phase, dead) && live);
          res_phase ^= 1u;
        } else if (has_res && !straight) {
          // residual rows that do not start on 16 bytes: element by element, a lane a column
          box_free();
          const T* res = static_cast<const T*>(a.residual) + row0 * a.ld_res + col0;
#pragma unroll 8
          for (int r = 0; r < 32; ++r) {
#pragma unroll
            for (int c = lane; c < kCols; c += 32)
              *cell(r, c) = row0 + r < a.m && col0 + c < a.n ? res[r * a.ld_res + c] : from_float<T>(0.f);
          }
          __syncwarp();
        }
#pragma unroll
        for (int s = 0; s < kTurns; ++s) {
          uint4 direct[4];
          if (straight) {
            const int64_t row = row0 + lane;
            const T* res = static_cast<const T*>(a.residual) + row * a.ld_res + col0 + s * 32;
#pragma unroll
            for (int j = 0; j < 4; ++j)
              direct[j] = row < a.m && col0 + s * 32 + j * 8 < a.n ? reinterpret_cast<const uint4*>(res)[j]
                                                                   : make_uint4(0, 0, 0, 0);
          }
          uint32_t v[32];
          take(v, s);
          if (s == kTurns - 1) {
            release();
            if (has_bias) read_bias(next.tile_n);
          }
          if (ACT != RFM_ACT_NONE) {
#pragma unroll
            for (int j = 0; j < 32; j += 2) {
              const float2 f = split(activate(pair(__uint_as_float(v[j]), __uint_as_float(v[j + 1])), ACT));
              v[j] = __float_as_uint(f.x);
              v[j + 1] = __float_as_uint(f.y);
            }
          }
          if (has_res) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const uint4 q = straight ? direct[j] : *piece(s * 4 + j);
              const uint32_t words[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float2 two = unpack2<T>(words[i]);
                add2(v[8 * j + 2 * i], v[8 * j + 2 * i + 1], two.x, two.y);
              }
            }
          }
          if (s == 0 && (!has_res || straight)) box_free();  // a residual in the box has waited for it
          put(v, s);
        }
        send(&maps.out, a.out);
      }
      if (!live) break;
      acc ^= 1u;
      if (acc == 0) acc_phase ^= 1u;
    }
    if (lane == 0) tma_wait_read<0>();
  }
  __syncwarp();
  tc_fence_before();
  if (CG == 2) {
    cluster_sync();  // neither CTA leaves while the other's products read its memory
  } else {
    __syncthreads();
  }
  if (warp == S::kMmaWarp) {
    tc_fence_after();
    tmem_free<CG>(tmem, kTmemColumns);
  }
}

// ---- the parts of a split contraction, added in their order, and the epilogue

struct FinishArgs {
  const float* partial;
  const void* bias;
  const void* residual;
  void* out;
  void* pre;
  int64_t m;
  int64_t ld_res;
  int32_t n;
  int32_t splits;
  int32_t activation;
  int32_t bias_dtype;
};

template <typename T, int VEC>
__global__ void __launch_bounds__(256) finish_kernel(const FinishArgs a) {
  chain_start();
  const int64_t per_row = a.n / VEC;
  const int64_t total = a.m * per_row;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t row = i / per_row;
    const int col = static_cast<int>(i % per_row) * VEC;
    float v[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[j] = 0.f;
    for (int s = 0; s < a.splits; ++s) {
      const Pack<float, VEC> q =
          *reinterpret_cast<const Pack<float, VEC>*>(a.partial + (static_cast<int64_t>(s) * a.m + row) * a.n + col);
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[j] += q.v[j];
    }
    Pack<T, VEC> o;
    if (a.bias != nullptr) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[j] += load_param(a.bias, a.bias_dtype, col + j);
    }
    if (a.pre != nullptr) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) o.v[j] = from_float<T>(keep_finite<T>(v[j]));
      *reinterpret_cast<Pack<T, VEC>*>(static_cast<T*>(a.pre) + row * a.n + col) = o;
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      float x = activate(v[j], a.activation);
      if (a.residual != nullptr) x += to_float(static_cast<const T*>(a.residual)[row * a.ld_res + col + j]);
      o.v[j] = from_float<T>(x);
    }
    *reinterpret_cast<Pack<T, VEC>*>(static_cast<T*>(a.out) + row * a.n + col) = o;
  }
}

// ---- dP = dY act'(saved) and its column sums

// dP is rounded to 16 bits once, here: it is an operand of the tensor cores, which
// take no fp32 one (tf32 would run at half the rate on twice the bytes).  The
// column sums take it before that rounding, in fp32: a lane its rows, then the
// warps, then the slabs, each in order.

struct GradPreArgs {
  const void* dy;
  const void* saved;  // pre, or (relu without a residual) out; not read without an activation
  void* dp;           // null: not stored
  float* partial;     // [slabs][n] column sums, null: not wanted
  int64_t rows;
  int64_t ld_dy;
  int64_t ld_dp;
  int32_t n;
};

constexpr int kPreWarps = 8;

// A CTA owns 32 * VEC columns and every gridDim.y-th group of 8 rows (a row a
// warp); the sums of its warps are added in their order at the end.
template <typename T, int VEC, int ACT>
__global__ void __launch_bounds__(32 * kPreWarps, 3) grad_pre_kernel(const GradPreArgs a) {
  chain_start();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int col = (static_cast<int>(blockIdx.x) * 32 + lane) * VEC;
  const bool in = col < a.n;
  constexpr int kPairs = (VEC + 1) / 2;
  Pair sum[kPairs];
#pragma unroll
  for (int j = 0; j < kPairs; ++j) sum[j] = both(0.f);
  const int64_t stride = static_cast<int64_t>(gridDim.y) * kPreWarps;
  if (in) {
    // four rows' loads go out before the first row is used
    constexpr int kRows = 4;
    for (int64_t row = static_cast<int64_t>(blockIdx.y) * kPreWarps + warp; row < a.rows; row += kRows * stride) {
      Pack<T, VEC> g[kRows], p[kRows];
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        // rows past the end: the last one again, not counted and not stored
        const int64_t at = min(row + r * stride, a.rows - 1);
        g[r] = *reinterpret_cast<const Pack<T, VEC>*>(static_cast<const T*>(a.dy) + at * a.ld_dy + col);
        if (ACT != RFM_ACT_NONE) {
          p[r] = *reinterpret_cast<const Pack<T, VEC>*>(static_cast<const T*>(a.saved) + at * a.n + col);
        }
      }
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        const int64_t at = row + r * stride;
        const bool valid = at < a.rows;
        Pack<T, VEC> o;
#pragma unroll
        for (int j = 0; j < kPairs; ++j) {
          Pair v;
          if constexpr (VEC == 1) {
            v = times_activate_grad(both(to_float(g[r].v[0])), both(ACT != RFM_ACT_NONE ? to_float(p[r].v[0]) : 0.f), ACT);
            o.v[0] = from_float<T>(split(v).x);
          } else {
            v = load_pair(g[r], j);
            if (ACT != RFM_ACT_NONE) v = times_activate_grad(v, load_pair(p[r], j), ACT);
            store_pair(o, j, v);
          }
          if (valid) sum[j] = sum[j] + v;
        }
        if (valid && a.dp != nullptr) {
          *reinterpret_cast<Pack<T, VEC>*>(static_cast<T*>(a.dp) + at * a.ld_dp + col) = o;
        }
      }
    }
  }
  if (a.partial == nullptr) return;
  __shared__ float sums[kPreWarps][32 * VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) sums[warp][j * 32 + lane] = j % 2 == 0 ? split(sum[j / 2]).x : split(sum[j / 2]).y;
  __syncthreads();
  if (warp == 0 && in) {
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      float s = sums[0][j * 32 + lane];
#pragma unroll
      for (int k = 1; k < kPreWarps; ++k) s += sums[k][j * 32 + lane];
      a.partial[static_cast<int64_t>(blockIdx.y) * a.n + col + j] = s;
    }
  }
}

// The slabs' sums per column, in a fixed order: 32 columns per CTA, each of 32
// warps every 32nd slab, then the 32 sums.
__global__ void __launch_bounds__(1024) bias_sum_kernel(const float* partial, int slabs, int n, void* out, int dtype) {
  chain_start();
  __shared__ float sums[32][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int col = static_cast<int>(blockIdx.x) * 32 + lane;
  float s = 0.f;
  if (col < n) {
#pragma unroll 8
    for (int k = warp; k < slabs; k += 32) s += partial[static_cast<int64_t>(k) * n + col];
  }
  sums[warp][lane] = s;
  __syncthreads();
  // warp w adds the 32 sums of column w
  s = sums[lane][warp];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(kFullMask, s, o);
  const int mine = static_cast<int>(blockIdx.x) * 32 + warp;
  if (lane == 0 && mine < n) store_param(out, dtype, mine, s);
}

template <typename T, int VEC>
int launch_grad_pre(const GradPreArgs& a, int activation, const dim3& grid, cudaStream_t s) {
  const auto kernel = activation == RFM_ACT_RELU   ? grad_pre_kernel<T, VEC, RFM_ACT_RELU>
                      : activation == RFM_ACT_GELU ? grad_pre_kernel<T, VEC, RFM_ACT_GELU>
                                                   : grad_pre_kernel<T, VEC, RFM_ACT_NONE>;
  // Where dP is stored an ordinary launch: CTAs that start one by one as the forward's
  // leave find the SMs unevenly filled (31200 x 2048, relu, a training pass: 213 us,
  // 199 so).
  return launch_chained(a.dp != nullptr ? Chain::kNone : Chain::kFirst, kernel, grid, 32 * kPreWarps, 0, 1, s, a);
}

// ---- dP and dX = dP W in one pass, where a row of dX fits one tile

// Up to 384 columns of dX an activation's gradient needs no pass of its own: dY
// and `saved` come by TMA into the ring of the product's A operand, warps turn dY
// into dP in place (element by element, so the swizzle does not matter), and from
// there the tensor cores read it and TMA stores it for dW.  A warp owns 8 columns
// of a slice, so its bias sums need no other warp: over a lane's rows, over the
// lanes by shuffles, and over the CTA's tiles in shared memory, in a fixed order.
// Two groups of eight warps take the slices in turn: with one, gelu's gradient
// (some 30 instructions a pair) left the issue slots half idle.
//
// HBM-bound: dY, `saved` and dP, 6 bytes an element, where the dP pass and dX
// apart move 8.  Rows are dealt out in units of 32, up to four a tile, so that the
// last wave occupies every SM (31200 rows: 244 tiles of 128 on 148 SMs).  A lane
// takes its rows one after the other: all four at once spilled, and spills go to
// L2 where shared memory leaves no L1 (31200 x 256 -> 2048 bf16: 109 us, 74 so).
// Measured, the whole backward with relu: 31200 x 256 -> 2048 bf16 118 us (with
// the dP pass 138), dX alone 61 (92); 13608 x 384 -> 1536 fp16 with gelu 68 (85)
// and 34 (53).  Fewer than some 64 tiles of 128 rows go the other way: 4800 x 256
// -> 2048 47.5 and 47.6, 2400 43.7 and 40, 300 28.1 and 18.8.
template <int BN>
struct GradShape {
  static constexpr int kUnit = 32;      // rows
  static constexpr int kPreparers = 8;  // of a slice: a warp 8 of its 64 columns
  static constexpr int kGroups = 2;     // of preparers
  static constexpr int kEpiWarps = 4;
  static constexpr int kEpi = kGroups * kPreparers, kLoadWarp = kEpi + kEpiWarps, kWeightWarp = kLoadWarp + 1;
  static constexpr int kMmaWarp = kWeightWarp + 1, kStoreWarp = kMmaWarp + 1;
  static constexpr int kThreads = 32 * (kStoreWarp + 1);
  // Three rings: dY (then dP), saved, and the weight (384 columns: three half
  // slices, where only two whole ones had room).  A group waits for a stage's next
  // phase only after it has seen the phase before, or the wait would end at once:
  // so the first two rings have an even number of stages, and a stage's uses are
  // all one group's.
  static constexpr int kA = 4, kS = 4, kW = BN == 384 ? 3 : BN == 256 ? 2 : 8;
  static_assert(kA % kGroups == 0 && kS % kGroups == 0, "a group's stages are its own");
  static constexpr int kUnitBytes = kUnit * kBK * 2, kSliceBytes = kBM * kBK * 2;
  static constexpr int kWeightParts = BN == 256 ? 1 : 2;  // of a slice
  static constexpr int kWeightRows = kBK / kWeightParts, kWeightBytes = BN * kWeightRows * 2;
  // Columns of bias sums, 4 bytes each for every group: sized for 256 -> 2048, the
  // decoder's feed-forward block.  Beside the rings there is room for 350 more with
  // 384 columns of dX and for 1,370 with fewer; beyond the limit (256 -> 2056) dP has
  // its pass of its own.
  static constexpr int kMostOut = 2048;
  static constexpr int kAccs = BN == 384 ? 1 : 2;
  static constexpr int kTmemColumns = BN == 128 ? 256 : 512;
  static constexpr int kMmaN = BN == 384 ? 192 : BN;
  static constexpr int kBoxBytes = 32 * 32 * 2;
  static constexpr int kSaved = kA * kSliceBytes, kWeight = kSaved + kS * kSliceBytes;
  static constexpr int kBoxes = kWeight + kW * kWeightBytes;
  static constexpr int kSums = kBoxes + kEpiWarps * kBoxBytes;
  static constexpr int kBars = kSums + kGroups * kMostOut * 4;
  static constexpr int kNumBars = 3 * kA + 2 * kS + 2 * kW + 2 * kAccs;
  static constexpr int kFlags = kBars + kNumBars * 8;
  static constexpr int kBytes = kFlags + 16;
  static_assert(kBytes <= 232448, "shared memory of one CTA");
};

struct GradXArgs {
  int64_t m;
  int32_t n;         // columns of dX
  int32_t out;       // columns of dP
  int32_t units;     // of 32 rows
  int32_t k_blocks;
  int32_t store;     // dP is stored
  float* partial;    // [CTAs][out] column sums, null: not wanted
};

struct GradXMaps {
  CUtensorMap dy, saved, dp;                 // boxes of a tile's rows
  CUtensorMap dy_unit, saved_unit, dp_unit;  // of a unit's
  CUtensorMap weight, dx;
};

// A place in a ring of N stages.
template <int N>
struct Ring {
  uint32_t stage = 0, phase = 0;
  __device__ __forceinline__ void next() {
    if (++stage == N) {
      stage = 0;
      phase ^= 1u;
    }
  }
  // every stage has been given back
  __device__ __forceinline__ bool drained(uint32_t empty, volatile int* dead) {
    for (int i = 0; i < N; ++i) {
      if (!bounded_wait(empty + 8 * stage, phase ^ 1u, dead)) return false;
      next();
    }
    return true;
  }
  // after a failure: the copies of the last `issued` slices land before the shared memory is given up
  __device__ __forceinline__ void settle(uint32_t full, uint32_t issued) {
    for (uint32_t i = 0; i < (issued < N ? issued : N); ++i) {
      if (stage == 0) {
        stage = N;
        phase ^= 1u;
      }
      --stage;
      for (uint32_t k = 0; k < kWaitTries && !mbar_try(full + 8 * stage, phase); ++k) {
      }
    }
  }
};

template <typename T, int BN, int ACT>
__global__ void __launch_bounds__(GradShape<BN>::kThreads, 1)
    grad_x_kernel(const __grid_constant__ GradXMaps maps, const __grid_constant__ GradXArgs a) {
  using S = GradShape<BN>;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t base = smem_u32(smem);
  const uint32_t a_full = base + S::kBars, a_ready = a_full + 8 * S::kA, a_empty = a_ready + 8 * S::kA;
  const uint32_t s_full = a_empty + 8 * S::kA, s_empty = s_full + 8 * S::kS;
  const uint32_t w_full = s_empty + 8 * S::kS, w_empty = w_full + 8 * S::kW;
  const uint32_t acc_full = w_empty + 8 * S::kW, acc_empty = acc_full + 8 * S::kAccs;
  volatile int* dead = reinterpret_cast<volatile int*>(smem + S::kFlags);
  const int warp = static_cast<int>(threadIdx.x) >> 5, lane = static_cast<int>(threadIdx.x) & 31;

  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (threadIdx.x == 0) {
    *dead = 0;
    if ((base & 1023u) != 0) {  // the swizzles count on it; never expected
      *dead = 1;
      atomicExch(&g_linear_faults, 1);
    }
    for (int i = 0; i < S::kA; ++i) {
      mbar_init(a_full + 8 * i, 1);
      mbar_init(a_ready + 8 * i, S::kPreparers);
      mbar_init(a_empty + 8 * i, a.store ? 2 : 1);  // the products, the store
    }
    for (int i = 0; i < S::kS; ++i) {
      mbar_init(s_full + 8 * i, 1);
      mbar_init(s_empty + 8 * i, S::kPreparers);
    }
    for (int i = 0; i < S::kW; ++i) {
      mbar_init(w_full + 8 * i, 1);
      mbar_init(w_empty + 8 * i, 1);
    }
    for (int i = 0; i < S::kAccs; ++i) {
      mbar_init(acc_full + 8 * i, 1);
      mbar_init(acc_empty + 8 * i, S::kEpiWarps);
    }
    mbar_init_fence();
    tma_prefetch_map(&maps.dy);
    tma_prefetch_map(&maps.saved);
    tma_prefetch_map(&maps.weight);
  }
  if (warp == S::kMmaWarp) tmem_alloc<1>(base + S::kFlags + 4, S::kTmemColumns);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  grid_dependency_wait();  // the set-up above touches nothing that the kernel before writes
  const uint32_t tmem = *reinterpret_cast<const volatile uint32_t*>(smem + S::kFlags + 4);
  // This CTA's tiles: in every wave but the last the CTAs take four units each, one
  // behind the other; what is left is dealt out evenly.
  constexpr int kTile = kBM / S::kUnit;
  const int ctas = static_cast<int>(gridDim.x), waves = a.units / (kTile * ctas);
  const int left = a.units - waves * kTile * ctas;
  const int last0 = static_cast<int>(static_cast<int64_t>(left) * blockIdx.x / ctas);
  const int last1 = static_cast<int>(static_cast<int64_t>(left) * (blockIdx.x + 1) / ctas);
  const int tiles = waves + (last1 > last0 ? 1 : 0);
  const auto tile_units = [&](int t) { return t < waves ? kTile : last1 - last0; };
  const auto tile_first = [&](int t) {
    return t < waves ? (t * ctas + static_cast<int>(blockIdx.x)) * kTile : waves * kTile * ctas + last0;
  };

  if (warp < S::kEpi) {
    const int group = warp / S::kPreparers, chunk = warp % S::kPreparers;
    Ring<S::kA> ra;
    Ring<S::kS> rs;
    // this lane's 16-byte piece of rows lane, lane + 32, ..: the warp's 8 columns under the swizzle
    const int at = lane * 128 + ((chunk ^ (lane & 7)) << 4);
    float* all_sums = reinterpret_cast<float*>(smem + S::kSums);
    float* sums = all_sums + group * S::kMostOut + chunk * 8;
    // after the shuffles lane l holds the sum of column l / 4
    if (a.partial != nullptr && (lane & 3) == 0) {
      for (int kb = 0; kb < a.k_blocks; ++kb) sums[kb * kBK + (lane >> 2)] = 0.f;
    }
    bool ok = true;
    int turn = 0;  // the group whose slice it is
    for (int t = 0; ok && t < tiles; ++t) {
      const int units = tile_units(t);
      for (int kb = 0; kb < a.k_blocks; ++kb, ra.next(), rs.next(), turn = (turn + 1) % S::kGroups) {
        if (turn != group) continue;
        ok = bounded_wait(a_full + 8 * ra.stage, ra.phase, dead) && bounded_wait(s_full + 8 * rs.stage, rs.phase, dead);
        ok = __all_sync(kFullMask, ok);
        if (!ok) break;
        uint8_t* dy = smem + ra.stage * S::kSliceBytes + at;
        const uint8_t* saved = smem + S::kSaved + rs.stage * S::kSliceBytes + at;
        Pair sum[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) sum[j] = both(0.f);
#pragma unroll 1
        for (int r = 0; r < units; ++r) {
          const Pack<T, 8> g = *reinterpret_cast<const Pack<T, 8>*>(dy + r * S::kUnitBytes);
          const Pack<T, 8> p = *reinterpret_cast<const Pack<T, 8>*>(saved + r * S::kUnitBytes);
          Pack<T, 8> o;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const Pair v = times_activate_grad(load_pair(g, j), load_pair(p, j), ACT);
            store_pair(o, j, v);
            sum[j] = sum[j] + v;
          }
          *reinterpret_cast<Pack<T, 8>*>(dy + r * S::kUnitBytes) = o;
        }
        proxy_fence();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(a_ready + 8 * ra.stage);
          mbar_arrive(s_empty + 8 * rs.stage);
        }
        if (a.partial != nullptr) {
          // each step halves the columns a lane still sums
          float v[8];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 f = split(sum[j]);
            v[2 * j] = f.x;
            v[2 * j + 1] = f.y;
          }
#pragma unroll
          for (int half = 4, o = 16; half > 0; half >>= 1, o >>= 1) {
            const bool upper = (lane & o) != 0;
#pragma unroll
            for (int j = 0; j < half; ++j) {
              const float give = upper ? v[j] : v[j + half], keep = upper ? v[j + half] : v[j];
              v[j] = keep + __shfl_xor_sync(kFullMask, give, o);
            }
          }
          v[0] += __shfl_xor_sync(kFullMask, v[0], 2);
          v[0] += __shfl_xor_sync(kFullMask, v[0], 1);
          if ((lane & 3) == 0) sums[kb * kBK + (lane >> 2)] += v[0];
        }
      }
    }
    if (a.partial != nullptr) {
      // the groups' sums, in their order
      static_assert(S::kGroups == 2, "two sums");
      asm volatile("bar.sync 1, %0;" ::"n"(32 * S::kEpi) : "memory");
      for (int col = static_cast<int>(threadIdx.x); col < a.out; col += 32 * S::kEpi)
        a.partial[static_cast<int64_t>(blockIdx.x) * a.out + col] = all_sums[col] + all_sums[S::kMostOut + col];
    }
  } else if (warp < S::kEpi + S::kEpiWarps) {
    const int quarter = warp & 3;
    const uint32_t box = base + S::kBoxes + quarter * S::kBoxBytes;
    uint8_t* row_ptr = smem + S::kBoxes + quarter * S::kBoxBytes + lane * 64;
    const int swz = (lane >> 1) & 3;
    Ring<S::kAccs> acc;
    for (int t = 0; t < tiles; ++t) {
      const int64_t row0 = static_cast<int64_t>(tile_first(t) + quarter) * S::kUnit;
      if (!__all_sync(kFullMask, bounded_wait(acc_full + 8 * acc.stage, acc.phase, dead))) break;
      tc_fence_after();
      if (quarter < tile_units(t)) {
#pragma unroll 1
        for (int c = 0; c < BN && c < a.n; c += 32) {
          uint32_t v[32];
          tmem_load_32(v, tmem + (static_cast<uint32_t>(quarter * 32) << 16) + acc.stage * BN + c);
          if (lane == 0) tma_wait_read<0>();  // the box's last store has been read
          __syncwarp();
          tmem_wait_load(v);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint32_t q[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
              q[i] = pack2<T>(__uint_as_float(v[8 * j + 2 * i]), __uint_as_float(v[8 * j + 2 * i + 1]));
            *reinterpret_cast<uint4*>(row_ptr + ((j ^ swz) << 4)) = make_uint4(q[0], q[1], q[2], q[3]);
          }
          proxy_fence();
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(&maps.dx, c, static_cast<int>(row0), box);
            tma_commit();
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(acc_empty + 8 * acc.stage);
      acc.next();
    }
    if (lane == 0) tma_wait_read<0>();
  } else if (warp == S::kLoadWarp) {
    if (lane == 0) {
      Ring<S::kA> ra;
      Ring<S::kS> rs;
      uint32_t issued_a = 0, issued_s = 0;
      bool ok = true;
      for (int t = 0; ok && t < tiles; ++t) {
        const int u = tile_first(t), units = tile_units(t);
        const auto load = [&](uint32_t to, const CUtensorMap* tile, const CUtensorMap* unit, int kb, uint32_t bar) {
          mbar_expect(bar, units * S::kUnitBytes);
          if (units == kTile) {
            tma_load_2d(to, tile, kb * kBK, u * S::kUnit, bar);
          } else {
            for (int r = 0; r < units; ++r)
              tma_load_2d(to + r * S::kUnitBytes, unit, kb * kBK, (u + r) * S::kUnit, bar);
          }
        };
        for (int kb = 0; kb < a.k_blocks; ++kb) {
          ok = bounded_wait(a_empty + 8 * ra.stage, ra.phase ^ 1u, dead);
          if (!ok) break;
          load(base + ra.stage * S::kSliceBytes, &maps.dy, &maps.dy_unit, kb, a_full + 8 * ra.stage);
          ra.next();
          ++issued_a;
          ok = bounded_wait(s_empty + 8 * rs.stage, rs.phase ^ 1u, dead);
          if (!ok) break;
          load(base + S::kSaved + rs.stage * S::kSliceBytes, &maps.saved, &maps.saved_unit, kb, s_full + 8 * rs.stage);
          rs.next();
          ++issued_s;
        }
      }
      if (!ok || !ra.drained(a_empty, dead) || !rs.drained(s_empty, dead)) {
        ra.settle(a_full, issued_a);
        rs.settle(s_full, issued_s);
      }
    }
  } else if (warp == S::kWeightWarp) {
    if (lane == 0) {
      Ring<S::kW> rw;
      uint32_t issued = 0;
      bool ok = true;
      for (int t = 0; ok && t < tiles; ++t) {
        for (int kb = 0; kb < S::kWeightParts * a.k_blocks; ++kb) {
          ok = bounded_wait(w_empty + 8 * rw.stage, rw.phase ^ 1u, dead);
          if (!ok) break;
          const uint32_t bar = w_full + 8 * rw.stage, to = base + S::kWeight + rw.stage * S::kWeightBytes;
          mbar_expect(bar, S::kWeightBytes);
#pragma unroll
          for (int j = 0; j < BN / 64; ++j)
            tma_load_2d(to + j * 128 * S::kWeightRows, &maps.weight, j * 64, kb * S::kWeightRows, bar);
          rw.next();
          ++issued;
        }
      }
      if (!ok || !rw.drained(w_empty, dead)) rw.settle(w_full, issued);
    }
  } else if (warp == S::kMmaWarp) {
    if (lane == 0) {
      constexpr int kType = std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
      constexpr uint32_t kInstr = mma_instr(kType, false, true, kBM, S::kMmaN);
      constexpr uint32_t kGroup = 128 * S::kWeightRows;  // bytes of 64 columns of the weight
      Ring<S::kA> ra;
      Ring<S::kW> rw;
      Ring<S::kAccs> acc;
      bool ok = true;
      for (int t = 0; ok && t < tiles; ++t) {
        if (!bounded_wait(acc_empty + 8 * acc.stage, acc.phase ^ 1u, dead)) break;
        tc_fence_after();
        const uint32_t d = tmem + acc.stage * BN;
        for (int kb = 0; ok && kb < a.k_blocks; ++kb) {
          // rows past the tile's units hold what was there before: their products are not stored
          const uint32_t sa = base + ra.stage * S::kSliceBytes;
          for (int half = 0; half < S::kWeightParts; ++half) {
            ok = bounded_wait(w_full + 8 * rw.stage, rw.phase, dead) &&
                 (half > 0 || bounded_wait(a_ready + 8 * ra.stage, ra.phase, dead));
            if (!ok) break;
            tc_fence_after();
            const uint32_t sb = base + S::kWeight + rw.stage * S::kWeightBytes;
#pragma unroll
            for (int k = 0; k < S::kWeightRows / 16; ++k) {
#pragma unroll
              for (int part = 0; part < BN / S::kMmaN; ++part) {
                tc_mma_f16<1>(d + part * S::kMmaN, operand_desc(sa + half * S::kWeightRows * 2 + k * 32, 16, 1024),
                              operand_desc(sb + part * (S::kMmaN / 64) * kGroup + k * 2048, kGroup, 1024), kInstr,
                              kb > 0 || half > 0 || k > 0);
              }
            }
            tc_commit<1>(w_empty + 8 * rw.stage);
            rw.next();
          }
          if (!ok) break;
          tc_commit<1>(a_empty + 8 * ra.stage);
          ra.next();
        }
        if (!ok) break;
        tc_commit<1>(acc_full + 8 * acc.stage);
        acc.next();
      }
      // as in gemm_kernel: products in flight end before the tensor memory is given up
      if (*dead) {
        tc_commit<1>(acc_full + 8 * acc.stage);
        for (uint32_t k = 0; k < kWaitTries && !mbar_try(acc_full + 8 * acc.stage, acc.phase); ++k) {
        }
      }
    }
  } else if (lane == 0 && a.store) {
    Ring<S::kA> ra;
    bool ok = true;
    for (int t = 0; ok && t < tiles; ++t) {
      const int u = tile_first(t), units = tile_units(t);
      for (int kb = 0; kb < a.k_blocks; ++kb) {
        ok = bounded_wait(a_ready + 8 * ra.stage, ra.phase, dead);
        if (!ok) break;
        const uint32_t from = base + ra.stage * S::kSliceBytes;
        if (units == kTile) {
          tma_store_2d(&maps.dp, kb * kBK, u * S::kUnit, from);
        } else {
          for (int r = 0; r < units; ++r)
            tma_store_2d(&maps.dp_unit, kb * kBK, (u + r) * S::kUnit, from + r * S::kUnitBytes);
        }
        tma_commit();
        tma_wait_read<0>();
        mbar_arrive(a_empty + 8 * ra.stage);
        ra.next();
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == S::kMmaWarp) {
    tc_fence_after();
    tmem_free<1>(tmem, S::kTmemColumns);
  }
}

// ---- a few rows: the weight is read once and nothing is tiled

// One warp computes W columns of the output for R rows: lane l holds the 16-byte
// pieces l, l + 32, .. of the weight's rows and of x's, products and sums in fp32,
// one shuffle tree at the end.  With a tile of 128 rows the tensor cores would
// work on zeros, and the contraction would be split to occupy the SMs: two
// launches.  Here the weight's bytes in flight are all that counts.  Measured
// (4096 -> 4096, fp16, the kernels' own time): 1 row 8.4 us (4.0 TB/s), tiles 20.6;
// 2 rows 10.4 and 23.9; 4 rows 18.6 and 16.5, so two rows are the most.  A whole
// call of one row takes 9.5 us among others.
struct FewArgs {
  const void* x;
  const void* weight;
  const void* bias;
  const void* residual;
  void* out;
  void* pre;
  int64_t ld_x, ld_w, ld_res;
  int32_t rows, n, k;
  int32_t bias_dtype;
  int32_t activation;
};

constexpr int kFewWarps = 4;

template <typename T>
__device__ __forceinline__ Pack<T, 8> load_piece(const T* row, int k, int depth) {
  if (k + 8 <= depth) return *reinterpret_cast<const Pack<T, 8>*>(row + k);
  Pack<T, 8> p;
#pragma unroll
  for (int j = 0; j < 8; ++j) p.v[j] = k + j < depth ? row[k + j] : from_float<T>(0.f);
  return p;
}

template <typename T, int R, int W, int UNROLL>
__global__ void __launch_bounds__(32 * kFewWarps) few_rows_kernel(const FewArgs a) {
  chain_start();
  const int lane = threadIdx.x & 31;
  const int n0 = (static_cast<int>(blockIdx.x) * kFewWarps + (threadIdx.x >> 5)) * W;
  if (n0 >= a.n) return;
  const T* x = static_cast<const T*>(a.x);
  const T* w = static_cast<const T*>(a.weight) + n0 * a.ld_w;
  Pair acc[R][W];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int c = 0; c < W; ++c) acc[r][c] = pair(0.f, 0.f);
  for (int k0 = lane * 8; k0 < a.k; k0 += 256 * UNROLL) {
    Pack<T, 8> wp[UNROLL][W];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u)
#pragma unroll
      for (int c = 0; c < W; ++c)
        wp[u][c] = load_piece(w + (n0 + c < a.n ? c : 0) * a.ld_w, k0 + u * 256, a.k);  // a column past the end: twice
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const Pack<T, 8> xp = load_piece(x + (r < a.rows ? r : 0) * a.ld_x, k0 + u * 256, a.k);
#pragma unroll
        for (int c = 0; c < W; ++c)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[r][c] = fma(load_pair(xp, j), load_pair(wp[u][c], j), acc[r][c]);
      }
    }
  }
  // element e = r * W + c of the warp's block ends up with lane e
  float mine = 0.f;
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int c = 0; c < W; ++c) {
      const float2 f = split(acc[r][c]);
      float s = f.x + f.y;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(kFullMask, s, o);
      if (lane == r * W + c) mine = s;
    }
  const int row = lane / W, col = n0 + lane % W;
  if (lane >= R * W || row >= a.rows || col >= a.n) return;
  if (a.bias != nullptr) mine += load_param(a.bias, a.bias_dtype, col);
  const int64_t at = static_cast<int64_t>(row) * a.n + col;
  if (a.pre != nullptr) static_cast<T*>(a.pre)[at] = from_float<T>(keep_finite<T>(mine));
  mine = activate(mine, a.activation);
  if (a.residual != nullptr) mine += to_float(static_cast<const T*>(a.residual)[row * a.ld_res + col]);
  static_cast<T*>(a.out)[at] = from_float<T>(mine);
}

constexpr int kFewRows = 2;  // most rows of this form

template <typename T>
int launch_few_rows(const FewArgs& a, cudaStream_t s) {
  constexpr int kColumns = 2;  // of a warp
  const unsigned grid = static_cast<unsigned>((a.n + kFewWarps * kColumns - 1) / (kFewWarps * kColumns));
  const auto kernel = a.rows == 1 ? few_rows_kernel<T, 1, kColumns, 4> : few_rows_kernel<T, 2, kColumns, 4>;
  return launch_chained(Chain::kFirst, kernel, dim3(grid), 32 * kFewWarps, 0, 1, s, a);
}

// ---- host side

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                 const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encode_tiled() {
  static const EncodeTiled fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult found = cudaDriverEntryPointSymbolNotFound;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &found) != cudaSuccess ||
        found != cudaDriverEntryPointSuccess) {
      cudaGetLastError();
      return static_cast<EncodeTiled>(nullptr);
    }
    return reinterpret_cast<EncodeTiled>(p);
  }();
  return fn;
}

// A matrix of `outer` rows of `inner` elements, `ld` apart, moved in boxes of
// box_inner x box_outer.
bool make_map(CUtensorMap* map, int dtype, const void* p, int64_t inner, int64_t outer, int64_t ld, int box_inner,
              int box_outer, CUtensorMapSwizzle swizzle) {
  const EncodeTiled encode = encode_tiled();
  if (encode == nullptr) return false;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(inner), static_cast<cuuint64_t>(outer)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld) * 2};
  const cuuint32_t box[2] = {static_cast<cuuint32_t>(box_inner), static_cast<cuuint32_t>(box_outer)};
  const cuuint32_t ones[2] = {1, 1};
  return encode(map, dtype == RFM_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2,
                const_cast<void*>(p), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool tma_rows(const void* p, int64_t ld) { return aligned16(p) && ld % 8 == 0; }

// How a product is cut: the tile's columns, one CTA or a pair to a tile, and the
// parts of the contraction.
struct Cut {
  int bn = 64;
  int pair = 0;
  int splits = 1;
};

// Estimated cycles of the busiest SM for each cut: a tile's fixed part (fill and
// drain of its pipeline, its stores) and one part per 64-deep slice, fitted to
// measurements of 38 products (rows 16 to 31200, 64 to 4096 deep, forward and both
// backward products; the chosen cut is on average 2 % behind the best, 19 % at
// worst).  Shallow products go to one CTA a tile (31200 x 256 -> 2048: 42.9 us,
// pairs 49.2), deep ones to pairs, which bring a third less through L2 (16384 x
// 4096 -> 4096: 371 us, single 427); narrower tiles only fill SMs (300 x 2048 ->
// 256: 64 columns in 4 parts 12.4 us, 256 columns whole 16.5).  Splitting pays
// the fp32 sums' way through L2 and a second launch.
Cut choose_cut(int64_t m, int n, int k_blocks) {
  struct Cost {
    int bn, pair;
    double start, tile, slice;
  };
  constexpr Cost kCosts[] = {
      {256, 1, 7500, 4200, 650}, {256, 0, 5000, 3400, 820}, {128, 0, 5000, 1800, 590}, {64, 0, 5000, 1200, 550}};
  constexpr double kSecondKernel = 9000.0, kPartBytesPerCycle = 1650.0;
  constexpr int kLeastSlices = 5;  // of a part
  const int sms = device_sm_count();
  Cut best;
  double least = 1e300;
  for (const Cost& c : kCosts) {
    const int64_t rows = c.pair ? 2 * kBM : kBM;
    const int64_t tiles = ((m + rows - 1) / rows) * ((n + c.bn - 1) / c.bn);
    const int64_t workers = c.pair ? sms / 2 : sms;
    if (workers == 0) continue;  // no device: sizes are still asked for
    for (int splits = 1; splits <= kMaxSplits; ++splits) {
      if (splits > 1 && (k_blocks / splits < kLeastSlices || tiles * (splits - 1) >= 4 * workers)) break;
      const double waves = static_cast<double>((tiles * splits + workers - 1) / workers);
      double cycles = c.start + waves * (c.tile + (k_blocks + splits - 1) / splits * c.slice);
      if (splits > 1) cycles += kSecondKernel + 8.0 * splits * static_cast<double>(m) * n / kPartBytesPerCycle;
      if (cycles < least) {
        least = cycles;
        best = Cut{c.bn, c.pair, splits};
      }
    }
  }
  return best;
}

struct Product {
  const void* a;
  const void* b;
  int64_t ld_a, ld_b;
  int64_t m;
  int n;
  int64_t k;
  int dtype;
  Chain chain;
  GemmArgs args;  // epilogue fields filled in by the caller
};

template <typename T, int BN, int CG, bool A_MN, bool B_MN, int ACT>
int launch_gemm(const Product& p, GemmArgs& g, float* partial, cudaStream_t stream) {
  using S = Shape<BN, CG>;
  // The context whose shared-memory limit is raised.  Before the maps: in a thread
  // that has made no CUDA call yet (autograd's, in a process's first backward) this
  // makes the context current, which encoding a map needs.
  static thread_local unsigned long long ready = 0;
  const auto kernel = gemm_kernel<T, BN, CG, A_MN, B_MN, ACT>;
  const unsigned long long context = current_context_id();
  if (ready != context || context == 0) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kBytes) != cudaSuccess) {
      cudaGetLastError();
      return RFM_ERR_LAUNCH;
    }
    ready = context;
  }
  GemmMaps maps;
  const bool ok_a = A_MN ? make_map(&maps.a, p.dtype, p.a, p.m, p.k, p.ld_a, 64, kBK, CU_TENSOR_MAP_SWIZZLE_128B)
                         : make_map(&maps.a, p.dtype, p.a, p.k, p.m, p.ld_a, kBK, kBM, CU_TENSOR_MAP_SWIZZLE_128B);
  const bool ok_b = B_MN ? make_map(&maps.b, p.dtype, p.b, p.n, p.k, p.ld_b, 64, kBK, CU_TENSOR_MAP_SWIZZLE_128B)
                         : make_map(&maps.b, p.dtype, p.b, p.k, p.n, p.ld_b, kBK, S::kBRows, CU_TENSOR_MAP_SWIZZLE_128B);
  if (!ok_a || !ok_b) return RFM_ERR_LAUNCH;
  g.tiles_m = static_cast<int>((p.m + kBM * CG - 1) / (kBM * CG));
  g.tiles_n = (p.n + BN - 1) / BN;
  g.partial = partial;
  g.tma_out = g.splits == 1 && tma_rows(g.out, p.n) && (g.pre == nullptr || tma_rows(g.pre, p.n));
  g.tma_res = g.splits == 1 && g.residual != nullptr && tma_rows(g.residual, g.ld_res);
  maps.out = maps.pre = maps.res = maps.a;
  constexpr CUtensorMapSwizzle swizzle = S::kBoxCols == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B;
  if (g.tma_out) {
    if (!make_map(&maps.out, p.dtype, g.out, p.n, p.m, p.n, S::kBoxCols, 32, swizzle)) return RFM_ERR_LAUNCH;
    if (g.pre != nullptr &&
        !make_map(&maps.pre, p.dtype, g.pre, p.n, p.m, p.n, S::kBoxCols, 32, swizzle)) {
      return RFM_ERR_LAUNCH;
    }
  }
  if (g.tma_res &&
      !make_map(&maps.res, p.dtype, g.residual, p.n, p.m, g.ld_res, S::kBoxCols, 32, swizzle)) {
    return RFM_ERR_LAUNCH;
  }
  const int64_t items = static_cast<int64_t>(g.tiles_m) * g.tiles_n * g.splits;
  if (items >= (int64_t(1) << 31) - (1 << 16)) return RFM_ERR_UNSUPPORTED;
  const int sms = device_sm_count();
  const int64_t workers = sms / CG;
  const unsigned grid = static_cast<unsigned>((items < workers ? items : workers) * CG);
  return launch_chained(p.chain, kernel, dim3(grid), S::kThreads, S::kBytes, CG, stream, maps, g);
}

template <typename T, int BN, int CG, bool A_MN, bool B_MN>
int launch_act(const Product& p, GemmArgs& g, float* partial, cudaStream_t stream) {
  if constexpr (!A_MN && !B_MN) {  // the forward; a split product's activation comes in the second kernel
    if (g.splits == 1 && g.activation == RFM_ACT_RELU) {
      return launch_gemm<T, BN, CG, A_MN, B_MN, RFM_ACT_RELU>(p, g, partial, stream);
    }
    if (g.splits == 1 && g.activation == RFM_ACT_GELU) {
      return launch_gemm<T, BN, CG, A_MN, B_MN, RFM_ACT_GELU>(p, g, partial, stream);
    }
  }
  return launch_gemm<T, BN, CG, A_MN, B_MN, RFM_ACT_NONE>(p, g, partial, stream);
}

template <typename T, bool A_MN, bool B_MN>
int launch_cut(const Product& p, GemmArgs& g, const Cut& cut, float* partial, cudaStream_t stream) {
  if (cut.pair) return launch_act<T, 256, 2, A_MN, B_MN>(p, g, partial, stream);
  if (cut.bn == 256) return launch_act<T, 256, 1, A_MN, B_MN>(p, g, partial, stream);
  if (cut.bn == 128) return launch_act<T, 128, 1, A_MN, B_MN>(p, g, partial, stream);
  return launch_act<T, 64, 1, A_MN, B_MN>(p, g, partial, stream);
}

template <typename T, bool A_MN, bool B_MN>
int run_product(const Product& p, void* workspace, cudaStream_t stream) {
  const Cut cut = choose_cut(p.m, p.n, static_cast<int>((p.k + kBK - 1) / kBK));
  GemmArgs g = p.args;
  g.m = p.m;
  g.n = p.n;
  g.k_blocks = static_cast<int>((p.k + kBK - 1) / kBK);
  g.splits = cut.splits;
  float* partial = static_cast<float*>(workspace);
  const int rc = launch_cut<T, A_MN, B_MN>(p, g, cut, partial, stream);
  if (rc != RFM_OK || cut.splits == 1) return rc;
  FinishArgs f{partial, g.bias, g.residual, g.out, g.pre, p.m, g.ld_res, p.n, cut.splits, g.activation, g.bias_dtype};
  const bool quads = p.n % 4 == 0 && (reinterpret_cast<uintptr_t>(g.out) & 7) == 0 &&
                     (reinterpret_cast<uintptr_t>(g.pre) & 7) == 0;
  const int64_t cells = p.m * (p.n / (quads ? 4 : 1));
  const int64_t most = static_cast<int64_t>(device_sm_count()) * 8;
  const int64_t ctas = (cells + 255) / 256;
  const unsigned grid = static_cast<unsigned>(ctas < most ? ctas : most);
  if (quads) {
    return launch_chained(Chain::kNext, finish_kernel<T, 4>, dim3(grid), 256, 0, 1, stream, f);
  }
  return launch_chained(Chain::kNext, finish_kernel<T, 1>, dim3(grid), 256, 0, 1, stream, f);
}

template <bool A_MN, bool B_MN>
int run_typed(const Product& p, void* workspace, cudaStream_t stream) {
  return p.dtype == RFM_DTYPE_BF16 ? run_product<__nv_bfloat16, A_MN, B_MN>(p, workspace, stream)
                                   : run_product<__half, A_MN, B_MN>(p, workspace, stream);
}

// fp32 sums of a split product, 16-byte multiples.
int64_t partial_bytes(int64_t m, int64_t n, int64_t k) {
  if (m == 0) return 0;
  const Cut cut = choose_cut(m, static_cast<int>(n), static_cast<int>((k + kBK - 1) / kBK));
  return cut.splits == 1 ? 0 : ((cut.splits * m * n * 4 + 15) & ~int64_t(15));
}

// Row slabs of the bias sums: about eight CTAs an SM, no less than 32 rows each.
int bias_slabs(int64_t rows, int n, int vec) {
  const int64_t strips = (n + 32 * vec - 1) / (32 * vec);
  const int64_t want = static_cast<int64_t>(device_sm_count()) * 8 / strips + 1;
  const int64_t most = (rows + 31) / 32;
  const int64_t slabs = want < most ? want : most;
  return static_cast<int>(slabs < 1 ? 1 : (slabs > 4096 ? 4096 : slabs));
}

// The sums' bytes whichever way the columns are read: wider strips are fewer, and
// their rows are cut into more slabs; grad_x_kernel leaves one row of sums a CTA.
int64_t bias_bytes(int64_t rows, int n) {
  int64_t slabs = bias_slabs(rows, n, 8);
  const int64_t narrow = bias_slabs(rows, n, 1), units = (rows + 31) / 32, sms = device_sm_count();
  const int64_t ctas = units < sms ? units : sms;
  slabs = narrow > slabs ? narrow : slabs;
  slabs = ctas > slabs ? ctas : slabs;
  return (slabs * n * 4 + 15) & ~int64_t(15);
}

// dP and dX in one kernel: an activation, a row of dX in one tile, rows that TMA
// reads, and enough tiles to occupy most SMs.
bool grad_x_fused(const rfm_linear_grad* p) {
  const int in = p->in_features, out = p->out_features;
  return p->activation != RFM_ACT_NONE && p->grad_x != nullptr && in % 8 == 0 && out % 8 == 0 && in <= 384 &&
         (p->grad_bias == nullptr || out <= GradShape<384>::kMostOut) &&
         tma_rows(p->grad_out, p->ld_grad) && aligned16(p->saved) && aligned16(p->grad_x) &&
         (p->rows + kBM - 1) / kBM * 2 >= device_sm_count();
}

template <typename T, int BN, int ACT>
int launch_grad_x(const rfm_linear_grad* p, int* ctas, cudaStream_t stream) {
  using S = GradShape<BN>;
  const int in = p->in_features, out = p->out_features;
  GradXArgs a{};
  a.m = p->rows;
  a.n = in;
  a.out = out;
  a.units = static_cast<int>((p->rows + S::kUnit - 1) / S::kUnit);
  a.k_blocks = (out + kBK - 1) / kBK;
  a.store = p->grad_weight != nullptr;
  a.partial = p->grad_bias != nullptr ? static_cast<float*>(p->workspace) : nullptr;
  static thread_local unsigned long long ready = 0;  // as in launch_gemm: before the maps
  const auto kernel = grad_x_kernel<T, BN, ACT>;
  const unsigned long long context = current_context_id();
  if (ready != context || context == 0) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kBytes) != cudaSuccess) {
      cudaGetLastError();
      return RFM_ERR_LAUNCH;
    }
    ready = context;
  }
  GradXMaps maps;
  const auto slices = [&](CUtensorMap* tile, CUtensorMap* unit, const void* at, int64_t ld) {
    return make_map(tile, p->dtype, at, out, p->rows, ld, kBK, kBM, CU_TENSOR_MAP_SWIZZLE_128B) &&
           make_map(unit, p->dtype, at, out, p->rows, ld, kBK, S::kUnit, CU_TENSOR_MAP_SWIZZLE_128B);
  };
  if (!slices(&maps.dy, &maps.dy_unit, p->grad_out, p->ld_grad) ||
      !slices(&maps.saved, &maps.saved_unit, p->saved, out) ||
      !slices(&maps.dp, &maps.dp_unit, p->grad_pre, p->ld_grad_pre) ||
      !make_map(&maps.weight, p->dtype, p->weight, in, out, p->ld_weight, 64, S::kWeightRows,
                CU_TENSOR_MAP_SWIZZLE_128B) ||
      !make_map(&maps.dx, p->dtype, p->grad_x, in, p->rows, in, 32, 32, CU_TENSOR_MAP_SWIZZLE_64B)) {
    return RFM_ERR_LAUNCH;
  }
  const int sms = device_sm_count();
  *ctas = a.units < sms ? a.units : sms;
  return launch_chained(Chain::kFirst, kernel, dim3(*ctas), S::kThreads, S::kBytes, 1, stream, maps, a);
}

template <typename T, int ACT>
int launch_grad_x(const rfm_linear_grad* p, int* ctas, cudaStream_t stream) {
  if (p->in_features <= 128) return launch_grad_x<T, 128, ACT>(p, ctas, stream);
  if (p->in_features <= 256) return launch_grad_x<T, 256, ACT>(p, ctas, stream);
  return launch_grad_x<T, 384, ACT>(p, ctas, stream);
}

int run_grad_x(const rfm_linear_grad* p, int* ctas, cudaStream_t stream) {
  if (p->dtype == RFM_DTYPE_BF16) {
    return p->activation == RFM_ACT_RELU ? launch_grad_x<__nv_bfloat16, RFM_ACT_RELU>(p, ctas, stream)
                                         : launch_grad_x<__nv_bfloat16, RFM_ACT_GELU>(p, ctas, stream);
  }
  return p->activation == RFM_ACT_RELU ? launch_grad_x<__half, RFM_ACT_RELU>(p, ctas, stream)
                                       : launch_grad_x<__half, RFM_ACT_GELU>(p, ctas, stream);
}

int check_sizes(int64_t rows, int in_features, int out_features, int dtype) {
  if (rows < 0 || in_features < 1 || out_features < 1 || (dtype != RFM_DTYPE_BF16 && dtype != RFM_DTYPE_F16)) {
    return RFM_ERR_INVALID_ARGUMENT;
  }
  // TMA coordinates are 32-bit
  if (rows > (int64_t(1) << 31) - 512 || in_features > (1 << 30) || out_features > (1 << 30)) {
    return RFM_ERR_UNSUPPORTED;
  }
  return RFM_OK;
}

bool operand_rows(const void* p, int64_t ld, int64_t rows, int64_t cols) {
  return p != nullptr && tma_rows(p, ld) && (rows <= 1 || ld >= cols) && ld > 0 && ld < (int64_t(1) << 38);
}

}  // namespace
}  // namespace rfm

extern "C" int64_t rfm_linear_forward_workspace_bytes(int64_t rows, int in_features, int out_features) {
  using namespace rfm;
  const int rc = check_sizes(rows, in_features, out_features, RFM_DTYPE_BF16);
  if (rc != RFM_OK) return -rc;
  return rows <= kFewRows ? 0 : partial_bytes(rows, out_features, in_features);
}

extern "C" int rfm_linear_forward(const rfm_linear* p, void* stream) {
  using namespace rfm;
  if (p == nullptr || p->reserved != 0) return RFM_ERR_INVALID_ARGUMENT;
  const int rc = check_sizes(p->rows, p->in_features, p->out_features, p->dtype);
  if (rc != RFM_OK) return rc;
  if (p->activation < RFM_ACT_NONE || p->activation > RFM_ACT_GELU) return RFM_ERR_INVALID_ARGUMENT;
  if (p->rows == 0) return RFM_OK;
  const bool bias_ok = p->bias == nullptr || p->bias_dtype == p->dtype || p->bias_dtype == RFM_DTYPE_F32;
  if (!operand_rows(p->x, p->ld_x, p->rows, p->in_features) ||
      !operand_rows(p->weight, p->ld_weight, p->out_features, p->in_features) || p->out == nullptr || !bias_ok) {
    return RFM_ERR_INVALID_ARGUMENT;
  }
  if (p->residual != nullptr && p->rows > 1 && p->ld_residual < p->out_features) return RFM_ERR_INVALID_ARGUMENT;
  if (p->rows <= kFewRows) {
    FewArgs f{p->x,     p->weight,      p->bias,
              p->residual, p->out,      p->pre,
              p->ld_x,  p->ld_weight,   p->ld_residual,
              static_cast<int32_t>(p->rows), p->out_features, p->in_features,
              p->bias_dtype, p->activation};
    return p->dtype == RFM_DTYPE_BF16 ? launch_few_rows<__nv_bfloat16>(f, as_stream(stream))
                                      : launch_few_rows<__half>(f, as_stream(stream));
  }
  const int64_t need = partial_bytes(p->rows, p->out_features, p->in_features);
  if (need > 0 && (p->workspace == nullptr || !aligned16(p->workspace) || p->workspace_bytes < need)) {
    return RFM_ERR_INVALID_ARGUMENT;
  }
  Product g{};
  g.a = p->x;
  g.ld_a = p->ld_x;
  g.b = p->weight;
  g.ld_b = p->ld_weight;
  g.m = p->rows;
  g.n = p->out_features;
  g.k = p->in_features;
  g.dtype = p->dtype;
  g.chain = Chain::kFirst;
  g.args.activation = p->activation;
  g.args.bias = p->bias;
  g.args.bias_dtype = p->bias_dtype;
  g.args.residual = p->residual;
  g.args.ld_res = p->ld_residual;
  g.args.out = p->out;
  g.args.pre = p->pre;
  return run_typed<false, false>(g, p->workspace, as_stream(stream));
}

extern "C" int64_t rfm_linear_backward_workspace_bytes(int64_t rows, int in_features, int out_features) {
  using namespace rfm;
  const int rc = check_sizes(rows, in_features, out_features, RFM_DTYPE_BF16);
  if (rc != RFM_OK) return -rc;
  // the products run one after the other and share the space; the bias sums come first
  int64_t most = partial_bytes(rows, in_features, out_features);
  const int64_t dw = rows == 0 ? 0 : partial_bytes(out_features, in_features, rows);
  most = dw > most ? dw : most;
  const int64_t bias = bias_bytes(rows, out_features);
  return bias > most ? bias : most;
}

extern "C" int rfm_linear_backward(const rfm_linear_grad* p, void* stream) {
  using namespace rfm;
  if (p == nullptr || p->reserved != 0) return RFM_ERR_INVALID_ARGUMENT;
  const int rc = check_sizes(p->rows, p->in_features, p->out_features, p->dtype);
  if (rc != RFM_OK) return rc;
  if (p->activation < RFM_ACT_NONE || p->activation > RFM_ACT_GELU) return RFM_ERR_INVALID_ARGUMENT;
  if (p->grad_x == nullptr && p->grad_weight == nullptr && p->grad_bias == nullptr) return RFM_OK;
  const int64_t rows = p->rows;
  const int in = p->in_features, out = p->out_features;
  cudaStream_t s = as_stream(stream);
  if (p->grad_bias != nullptr && p->bias_dtype != p->dtype && p->bias_dtype != RFM_DTYPE_F32) {
    return RFM_ERR_INVALID_ARGUMENT;
  }
  if (rows == 0) {  // empty sums
    if (p->grad_weight != nullptr &&
        cudaMemsetAsync(p->grad_weight, 0, static_cast<size_t>(in) * out * 2, s) != cudaSuccess) {
      cudaGetLastError();
      return RFM_ERR_LAUNCH;
    }
    if (p->grad_bias != nullptr) {
      return launch_chained(Chain::kFirst, bias_sum_kernel, dim3((out + 31) / 32), 1024, 0, 1, s,
                            static_cast<const float*>(nullptr), 0, out, p->grad_bias, p->bias_dtype);
    }
    return RFM_OK;
  }
  const bool acts = p->activation != RFM_ACT_NONE;
  if (p->grad_out == nullptr || (rows > 1 && p->ld_grad < out) || (acts && p->saved == nullptr)) {
    return RFM_ERR_INVALID_ARGUMENT;
  }
  const bool products = p->grad_x != nullptr || p->grad_weight != nullptr;
  // dP is dY itself without an activation, where TMA can read it
  const bool own = products && (acts || !tma_rows(p->grad_out, p->ld_grad));
  if (own && !operand_rows(p->grad_pre, p->ld_grad_pre, rows, out)) return RFM_ERR_INVALID_ARGUMENT;
  if (p->grad_x != nullptr && !operand_rows(p->weight, p->ld_weight, out, in)) return RFM_ERR_INVALID_ARGUMENT;
  if (p->grad_weight != nullptr && !operand_rows(p->x, p->ld_x, rows, in)) return RFM_ERR_INVALID_ARGUMENT;
  const int64_t need = rfm_linear_backward_workspace_bytes(rows, in, out);
  if (need > 0 && (p->workspace == nullptr || !aligned16(p->workspace) || p->workspace_bytes < need)) {
    return RFM_ERR_INVALID_ARGUMENT;
  }

  const bool fused = grad_x_fused(p);
  if (fused) {
    int ctas = 0;
    int done = run_grad_x(p, &ctas, s);
    if (done == RFM_OK && p->grad_bias != nullptr) {
      done = launch_chained(Chain::kNext, bias_sum_kernel, dim3((out + 31) / 32), 1024, 0, 1, s,
                            static_cast<const float*>(p->workspace), ctas, out, p->grad_bias, p->bias_dtype);
    }
    if (done != RFM_OK) return done;
  } else if (own || p->grad_bias != nullptr) {
    GradPreArgs a{};
    a.dy = p->grad_out;
    a.ld_dy = rows > 1 ? p->ld_grad : out;
    a.saved = acts ? p->saved : nullptr;
    a.dp = own ? p->grad_pre : nullptr;
    a.ld_dp = p->ld_grad_pre;
    a.partial = p->grad_bias != nullptr ? static_cast<float*>(p->workspace) : nullptr;
    a.rows = rows;
    a.n = out;
    const bool vec = out % 8 == 0 && a.ld_dy % 8 == 0 && aligned16(a.dy) && aligned16(a.saved);
    const int width = 32 * (vec ? 8 : 1);
    const int slabs = bias_slabs(rows, out, vec ? 8 : 1);
    const dim3 grid((out + width - 1) / width, slabs);
    int done;
    if (p->dtype == RFM_DTYPE_BF16) {
      done = vec ? launch_grad_pre<__nv_bfloat16, 8>(a, p->activation, grid, s)
                 : launch_grad_pre<__nv_bfloat16, 1>(a, p->activation, grid, s);
    } else {
      done = vec ? launch_grad_pre<__half, 8>(a, p->activation, grid, s)
                 : launch_grad_pre<__half, 1>(a, p->activation, grid, s);
    }
    if (done != RFM_OK) return done;
    if (p->grad_bias != nullptr) {
      done = launch_chained(Chain::kNext, bias_sum_kernel, dim3((out + 31) / 32), 1024, 0, 1, s, a.partial, slabs, out,
                            p->grad_bias, p->bias_dtype);
      if (done != RFM_OK) return done;
    }
  }
  Chain chain = own || p->grad_bias != nullptr ? Chain::kNext : Chain::kFirst;  // of the next product
  const void* dp = own ? p->grad_pre : p->grad_out;
  const int64_t ld_dp = own ? p->ld_grad_pre : p->ld_grad;
  if (p->grad_x != nullptr && !fused) {
    Product g{};
    g.a = dp;
    g.ld_a = ld_dp;
    g.b = p->weight;
    g.ld_b = p->ld_weight;
    g.m = rows;
    g.n = in;
    g.k = out;
    g.dtype = p->dtype;
    g.chain = chain;
    g.args.out = p->grad_x;
    const int done = run_typed<false, true>(g, p->workspace, s);
    if (done != RFM_OK) return done;
    chain = Chain::kNext;
  }
  if (p->grad_weight != nullptr) {
    Product g{};
    g.a = dp;
    g.ld_a = ld_dp;
    g.b = p->x;
    g.ld_b = p->ld_x;
    g.m = out;
    g.n = in;
    g.k = rows;
    g.dtype = p->dtype;
    g.chain = chain;
    g.args.out = p->grad_weight;
    return run_typed<true, true>(g, p->workspace, s);
  }
  return RFM_OK;
}

extern "C" int rfm_linear_faults(int* faults) {
  using namespace rfm;
  if (faults == nullptr) return RFM_ERR_INVALID_ARGUMENT;
  // the copy alone waits for streams that synchronise with the default one; torch's own do not
  cudaError_t err = cudaDeviceSynchronize();
  if (err == cudaSuccess) err = cudaMemcpyFromSymbol(faults, g_linear_faults, sizeof(int));
  if (err == cudaSuccess) return RFM_OK;
  const int rc = launch_status();
  return rc == RFM_OK ? RFM_ERR_LAUNCH : rc;
}
