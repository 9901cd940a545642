// Layer norm over the last dimension, forward and backward, fp32 / bf16 / fp16.
//
//   mean = sum x / D,  rstd = 1 / sqrt(sum (x - mean)^2 / D + eps)
//   y    = (x - mean) rstd w + b
//   with u = (x - mean) rstd and t = dy w:
//   dx   = rstd (t - mean(t) - u mean(t u)),  dw = sum_rows dy u,  db = sum_rows dy
//
// All arithmetic is fp32; the only rounding to the tensors' type is the store
// of y, dx, dw and db.  The variance is the mean of squared deviations from the
// mean (two sums over registers, not E[x^2] - E[x]^2, which cancels for rows
// whose mean is large).
//
// HBM-bound: the forward moves 2 and the backward 3 arrays of rows x D.  A team
// of TEAM threads keeps one row in registers (TEAM * VEC * CH >= D), so every
// element is read once.  Teams of 8 lanes for short rows, a warp (no barrier) up to
// 1024 columns (512 where rows are read element by element; the backward of 16-bit
// rows has two warps beyond 512), 128 to 512 threads up to 8192; longer rows are
// re-read from L2.
// Each thread copies its own 16-byte pieces of the next DEPTH rows into shared
// memory ahead of time (cp.async; nobody else reads them, so no barrier is
// needed): bytes in flight, some 100 KB an SM, are what the bandwidth hangs on,
// and registers could hold only one row more.
// The weight and bias gradients are summed in registers over a team's rows (a
// thread always owns the same columns), then over the CTA's teams in shared
// memory, then over the CTAs by a second kernel, all in a fixed order: no
// atomics, and the same bits on every run.
#include <math.h>

#include "rfm_types.cuh"

namespace rfm {
namespace {

constexpr int kThreads = 256;  // of the kernels without teams
constexpr int kWarps = kThreads / 32;
constexpr int kWideDim = 8192;  // longest row held in registers
constexpr int kWideSlabs = 64;  // row slabs of the wide rows' parameter gradients

// Threads of a CTA of teams; `cols`: columns a thread owns.
__host__ __device__ constexpr int cta_threads(int team, int cols) { return team > 32 ? 512 : cols > 16 ? 128 : 256; }
// Rows a thread copies ahead (0: element loads, one row ahead in registers).
__host__ __device__ constexpr int ring_depth(int vec, int ch) { return vec == 1 ? 0 : ch == 1 ? 4 : ch <= 4 ? 3 : 2; }

struct NormArgs {
  const void* x;
  const void* dy;
  const void* weight;
  const void* bias;
  void* out;  // y or dx
  const float* mean_in;
  const float* rstd_in;
  float* mean_out;
  float* rstd_out;
  float* partial;  // [CTAs][2][D]
  int64_t rows;
  int64_t ld_x;
  int64_t ld_dy;
  int dim;
  int param_dtype;
  float eps;
  float inv_dim;
};

// One thread's pieces of rows to come: copied ahead into its own places of
// shared memory, or (element loads) one row ahead in registers.
template <typename T, int VEC, int TEAM, int CH>
struct Ahead {
  static constexpr int kDepth = ring_depth(VEC, CH);
  static constexpr int kThreadsCta = cta_threads(TEAM, CH * VEC);
  static constexpr int kBytes = kDepth * CH * kThreadsCta * 16;  // of one array
  static constexpr int kStep = TEAM * VEC;
  const T* at;     // the array
  int64_t ld;
  int dim, lane;
  uint8_t* smem;   // this array's ring
  Pack<T, VEC> next[kDepth == 0 ? CH : 1];

  __device__ __forceinline__ Ahead(const void* base, int64_t ld_, int dim_, int lane_, uint8_t* ring)
      : at(static_cast<const T*>(base)), ld(ld_), dim(dim_), lane(lane_), smem(ring) {}

  __device__ __forceinline__ uint8_t* place(int slot, int c) const {
    return smem + ((slot * CH + c) * kThreadsCta + static_cast<int>(threadIdx.x)) * 16;
  }

  __device__ __forceinline__ void request(int64_t row, bool valid, int slot) {
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int col = c * kStep + lane * VEC;
      if constexpr (kDepth > 0) {
        if (valid && col < dim) {
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                           static_cast<uint32_t>(__cvta_generic_to_shared(place(slot, c)))),
                       "l"(at + row * ld + col)
                       : "memory");
        }
      } else {
        if (valid && col < dim) {
          next[c] = *reinterpret_cast<const Pack<T, VEC>*>(at + row * ld + col);
        } else {
#pragma unroll
          for (int j = 0; j < VEC; ++j) next[c].v[j] = from_float<T>(0.f);
        }
      }
    }
  }

  __device__ __forceinline__ void take(Pack<T, VEC> (&r)[CH], bool valid, int slot) const {
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      if constexpr (kDepth > 0) {
        if (valid && c * kStep + lane * VEC < dim) {
          r[c] = *reinterpret_cast<const Pack<T, VEC>*>(place(slot, c));
        } else {
#pragma unroll
          for (int j = 0; j < VEC; ++j) r[c].v[j] = from_float<T>(0.f);
        }
      } else {
        r[c] = next[c];
      }
    }
  }
};

template <int DEPTH>
__device__ __forceinline__ void ring_commit() {
  if constexpr (DEPTH > 0) asm volatile("cp.async.commit_group;" ::: "memory");
}

// All but the newest DEPTH - 1 requests of this thread have landed.
template <int DEPTH>
__device__ __forceinline__ void ring_wait() {
  if constexpr (DEPTH > 0) asm volatile("cp.async.wait_group %0;" ::"n"(DEPTH - 1) : "memory");
}

// Sum of (a, b) over a team; every thread of the team gets it.  A team of more
// than a warp meets at a barrier of its own and uses the slots `parity` of its
// part of `slots`, so that two sums in a row need one barrier each.
template <int TEAM>
__device__ __forceinline__ float2 team_sum(float2 s, float2* slots, int parity) {
#pragma unroll
  for (int o = (TEAM < 32 ? TEAM : 32) / 2; o > 0; o >>= 1) {
    s.x += __shfl_xor_sync(kFullMask, s.x, o);
    s.y += __shfl_xor_sync(kFullMask, s.y, o);
  }
  if constexpr (TEAM > 32) {
    constexpr int kTeamWarps = TEAM / 32;
    const int team = static_cast<int>(threadIdx.x) / TEAM;
    float2* mine = slots + (team * 2 + parity) * kTeamWarps;
    if ((threadIdx.x & 31) == 0) mine[(threadIdx.x % TEAM) >> 5] = s;
    asm volatile("bar.sync %0, %1;" ::"r"(team + 1), "n"(TEAM) : "memory");
    s = mine[0];
#pragma unroll
    for (int w = 1; w < kTeamWarps; ++w) {
      s.x += mine[w].x;
      s.y += mine[w].y;
    }
  }
  return s;
}

// Weight (or bias) of a thread's columns as pairs: in registers, or (SHARE, beyond
// 16 columns) in shared memory.  The forward has the registers: reading them from
// shared memory for every row took its bandwidth (65536 x 1024 fp16: 57 us, 50
// with registers).  The backward needs its registers for the sums.
template <int VEC, int TEAM, int CH, bool SHARE>
struct Params {
  static constexpr int kCols = CH * VEC, kStep = TEAM * VEC;
  static constexpr bool kShared = SHARE && kCols > 16;
  Pair reg[kShared ? 1 : kCols / 2];
  const float* smem;

  __device__ __forceinline__ void load(const void* p, int dtype, int dim, float missing, int lane, float* shared) {
    smem = shared;
    if constexpr (kShared) {
      for (int i = threadIdx.x; i < kStep * CH; i += blockDim.x)
        shared[i] = i < dim && p != nullptr ? load_param(p, dtype, i) : missing;
    } else {
#pragma unroll
      for (int i = 0; i < kCols / 2; ++i) {
        float v[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int c = (2 * i + k) / VEC, j = (2 * i + k) % VEC;
          const int col = c * kStep + lane * VEC + j;
          v[k] = col < dim && p != nullptr ? load_param(p, dtype, col) : missing;
        }
        reg[i] = pair(v[0], v[1]);
      }
    }
  }

  // the thread's columns 2 i and 2 i + 1
  __device__ __forceinline__ Pair at(int i, int lane) const {
    if constexpr (kShared) {
      const int c = (2 * i) / VEC, j = (2 * i) % VEC;
      const float2 f = *reinterpret_cast<const float2*>(smem + c * kStep + lane * VEC + j);
      return pair(f.x, f.y);
    } else {
      return reg[i];
    }
  }
};

// The thread's elements 2 i, 2 i + 1 of a row (element loads: of two chunks).
template <typename T, int VEC, int CH>
__device__ __forceinline__ Pair element_pair(const Pack<T, VEC> (&r)[CH], int i) {
  if constexpr (VEC == 1) {
    return pair(to_float(r[2 * i].v[0]), to_float(r[2 * i + 1].v[0]));
  } else {
    return load_pair(r[2 * i / VEC], (2 * i % VEC) / 2);
  }
}

template <typename T, int VEC, int TEAM, int CH>
__global__ void __launch_bounds__(cta_threads(TEAM, CH* VEC)) norm_fwd_kernel(const NormArgs a) {
  using Rows = Ahead<T, VEC, TEAM, CH>;
  using P = Params<VEC, TEAM, CH, false>;
  extern __shared__ __align__(16) uint8_t ring[];
  __shared__ float2 slots[2 * Rows::kThreadsCta / 32];
  constexpr int kTeams = Rows::kThreadsCta / TEAM;
  constexpr int kStep = TEAM * VEC;
  constexpr int kPairs = CH * VEC / 2;
  constexpr int kDepth = Rows::kDepth > 0 ? Rows::kDepth : 1;
  const int lane = static_cast<int>(threadIdx.x) % TEAM;
  const int team = static_cast<int>(threadIdx.x) / TEAM;
  T* out = static_cast<T*>(a.out);
  const int64_t stride = static_cast<int64_t>(gridDim.x) * kTeams;
  int64_t row = static_cast<int64_t>(blockIdx.x) * kTeams + team;
  // the loop runs on the row of the warp's first team, so that a warp stays whole
  int64_t lead = TEAM >= 32 ? row : static_cast<int64_t>(blockIdx.x) * kTeams + (threadIdx.x & ~31u) / TEAM;

  chain_start();
  Rows rows(a.x, a.ld_x, a.dim, lane, ring);
#pragma unroll
  for (int d = 0; d < kDepth; ++d) {
    rows.request(row + d * stride, row + d * stride < a.rows, d);
    ring_commit<Rows::kDepth>();
  }
  P w, b;
  w.load(a.weight, a.param_dtype, a.dim, 1.f, lane, nullptr);
  b.load(a.bias, a.param_dtype, a.dim, 0.f, lane, nullptr);

  int slot = 0;
  for (; lead < a.rows; row += stride, lead += stride) {
    Pack<T, VEC> x[CH];
    ring_wait<Rows::kDepth>();
    rows.take(x, row < a.rows, slot);
    Pair v[kPairs];
    Pair s = pair(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      v[i] = element_pair<T, VEC, CH>(x, i);
      s = s + v[i];
    }
    rows.request(row + kDepth * stride, row + kDepth * stride < a.rows, slot);
    ring_commit<Rows::kDepth>();
    if (++slot == kDepth) slot = 0;
    float2 sums = split(s);
    const float mean = team_sum<TEAM>(make_float2(sums.x + sums.y, 0.f), slots, 0).x * a.inv_dim;
    const Pair minus = pair(-mean, -mean);
    s = pair(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      v[i] = v[i] + minus;
      if constexpr (VEC == 1) {  // columns past the row's end (a whole piece of a vector row) count nothing
        float2 f = split(v[i]);
        if (2 * i * kStep + lane >= a.dim) f.x = 0.f;
        if ((2 * i + 1) * kStep + lane >= a.dim) f.y = 0.f;
        v[i] = pair(f.x, f.y);
      } else if ((2 * i / VEC) * kStep + lane * VEC >= a.dim) {
        v[i] = pair(0.f, 0.f);
      }
      s = fma(v[i], v[i], s);
    }
    sums = split(s);
    const float var = team_sum<TEAM>(make_float2(sums.x + sums.y, 0.f), slots, 1).x;
    const float rstd = 1.f / sqrtf(fmaf(var, a.inv_dim, a.eps));
    if (row < a.rows) {
      const Pair scale = pair(rstd, rstd);
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        const int col = c * kStep + lane * VEC;
        if (col >= a.dim) continue;
        Pack<T, VEC> y;
        if constexpr (VEC == 1) {
          const float2 f = split(fma(v[c / 2] * scale, w.at(c / 2, lane), b.at(c / 2, lane)));
          y.v[0] = from_float<T>(c % 2 == 0 ? f.x : f.y);
        } else {
#pragma unroll
          for (int j = 0; j < VEC / 2; ++j) {
            const int i = c * VEC / 2 + j;
            store_pair(y, j, fma(v[i] * scale, w.at(i, lane), b.at(i, lane)));
          }
        }
        *reinterpret_cast<Pack<T, VEC>*>(out + row * a.dim + col) = y;
      }
      if (lane == 0 && a.mean_out != nullptr) {
        a.mean_out[row] = mean;
        a.rstd_out[row] = rstd;
      }
    }
  }
}

// PARAMS: also the sums of dy u and dy per column, one partial pair per CTA.  u
// and t are computed twice, for the sums and for dx: cheaper than the registers
// that would keep them.
template <typename T, int VEC, int TEAM, int CH, bool PARAMS>
__global__ void __launch_bounds__(cta_threads(TEAM, CH* VEC)) norm_bwd_kernel(const NormArgs a) {
  using Rows = Ahead<T, VEC, TEAM, CH>;
  using P = Params<VEC, TEAM, CH, true>;
  extern __shared__ __align__(16) uint8_t ring[];
  __shared__ float2 slots[2 * Rows::kThreadsCta / 32];
  constexpr int kStep = TEAM * VEC;
  __shared__ __align__(16) float params[P::kShared ? kStep * CH : 1];
  constexpr int kTeams = Rows::kThreadsCta / TEAM;
  constexpr int kPairs = CH * VEC / 2;
  constexpr int kDepth = Rows::kDepth > 0 ? Rows::kDepth : 1;
  const int lane = static_cast<int>(threadIdx.x) % TEAM;
  const int team = static_cast<int>(threadIdx.x) / TEAM;
  T* out = static_cast<T*>(a.out);
  const int64_t stride = static_cast<int64_t>(gridDim.x) * kTeams;
  int64_t row = static_cast<int64_t>(blockIdx.x) * kTeams + team;
  int64_t lead = TEAM >= 32 ? row : static_cast<int64_t>(blockIdx.x) * kTeams + (threadIdx.x & ~31u) / TEAM;

  chain_start();
  Rows xs(a.x, a.ld_x, a.dim, lane, ring);
  Rows dys(a.dy, a.ld_dy, a.dim, lane, ring + Rows::kBytes);
  float mean_ahead[kDepth], rstd_ahead[kDepth];
  const auto request = [&](int64_t r, int d) {
    const bool valid = r < a.rows;
    xs.request(r, valid, d);
    dys.request(r, valid, d);
    ring_commit<Rows::kDepth>();
    mean_ahead[d] = valid ? a.mean_in[r] : 0.f;
    rstd_ahead[d] = valid ? a.rstd_in[r] : 0.f;
  };
#pragma unroll
  for (int d = 0; d < kDepth; ++d) request(row + d * stride, d);
  P w;
  w.load(a.weight, a.param_dtype, a.dim, 1.f, lane, params);
  if (P::kShared) __syncthreads();
  Pair dw[PARAMS ? kPairs : 1], db[PARAMS ? kPairs : 1];
#pragma unroll
  for (int i = 0; i < (PARAMS ? kPairs : 1); ++i) dw[i] = db[i] = pair(0.f, 0.f);

  int parity = 0;
  while (lead < a.rows) {
#pragma unroll
    for (int d = 0; d < kDepth; ++d) {
      if (lead >= a.rows) break;
      const float mean = mean_ahead[d], rstd = rstd_ahead[d];
      Pack<T, VEC> x[CH], dy[CH];
      ring_wait<Rows::kDepth>();
      xs.take(x, row < a.rows, d);  // zeros past the row's end and past the last row
      dys.take(dy, row < a.rows, d);
      // u = x rstd - mean rstd would cancel for rows whose mean is large
      const Pair minus = pair(-mean, -mean), scale = pair(rstd, rstd);
      Pair s1 = pair(0.f, 0.f), s2 = pair(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < kPairs; ++i) {
        const Pair g = element_pair<T, VEC, CH>(dy, i);
        const Pair u = (element_pair<T, VEC, CH>(x, i) + minus) * scale;  // past the end: times dy, 0
        const Pair t = g * w.at(i, lane);
        s1 = s1 + t;
        s2 = fma(t, u, s2);
        if (PARAMS) {
          dw[i] = fma(g, u, dw[i]);
          db[i] = db[i] + g;
        }
      }
      const float2 f1 = split(s1), f2 = split(s2);
      const float2 s = team_sum<TEAM>(make_float2(f1.x + f1.y, f2.x + f2.y), slots, parity);
      parity ^= 1;
      if (out != nullptr && row < a.rows) {
        // dx = rstd (t - m1 - u m2)
        const float m1 = s.x * a.inv_dim, m2 = s.y * a.inv_dim;
        const Pair minus1 = pair(-m1, -m1), minus2 = pair(-m2, -m2);
#pragma unroll
        for (int c = 0; c < CH; ++c) {
          const int col = c * kStep + lane * VEC;
          if (col >= a.dim) continue;
          Pack<T, VEC> o;
          const auto dx = [&](int i) {
            const Pair u = (element_pair<T, VEC, CH>(x, i) + minus) * scale;
            const Pair t = fma(element_pair<T, VEC, CH>(dy, i), w.at(i, lane), minus1);
            return fma(u, minus2, t) * scale;
          };
          if constexpr (VEC == 1) {
            const float2 f = split(dx(c / 2));
            o.v[0] = from_float<T>(c % 2 == 0 ? f.x : f.y);
          } else {
#pragma unroll
            for (int j = 0; j < VEC / 2; ++j) store_pair(o, j, dx(c * VEC / 2 + j));
          }
          *reinterpret_cast<Pack<T, VEC>*>(out + row * a.dim + col) = o;
        }
      }
      request(row + kDepth * stride, d);
      row += stride;
      lead += stride;
    }
  }

  if constexpr (PARAMS) {
    float* pw = a.partial + static_cast<int64_t>(blockIdx.x) * 2 * a.dim;
    const auto column = [&](int e) { return (e / VEC) * kStep + lane * VEC + e % VEC; };
    if constexpr (kTeams == 1) {
#pragma unroll
      for (int i = 0; i < kPairs; ++i) {
        const float2 fw = split(dw[i]), fb = split(db[i]);
        if (column(2 * i) < a.dim) {
          pw[column(2 * i)] = fw.x;
          pw[a.dim + column(2 * i)] = fb.x;
        }
        if (column(2 * i + 1) < a.dim) {
          pw[column(2 * i + 1)] = fw.y;
          pw[a.dim + column(2 * i + 1)] = fb.y;
        }
      }
    } else {
      // the CTA's teams, summed in a fixed order, one register pair of every thread at a time
      __shared__ float2 slab[2][Rows::kThreadsCta];
#pragma unroll
      for (int i = 0; i < kPairs; ++i) {
        __syncthreads();
        slab[0][threadIdx.x] = split(dw[i]);
        slab[1][threadIdx.x] = split(db[i]);
        __syncthreads();
        for (int k = threadIdx.x; k < 2 * TEAM; k += Rows::kThreadsCta) {
          const int which = k / TEAM, from = k % TEAM;
          float2 sum = make_float2(0.f, 0.f);
#pragma unroll
          for (int m = 0; m < kTeams; ++m) {
            sum.x += slab[which][m * TEAM + from].x;
            sum.y += slab[which][m * TEAM + from].y;
          }
          const int c0 = (2 * i / VEC) * kStep + from * VEC + 2 * i % VEC;
          const int c1 = ((2 * i + 1) / VEC) * kStep + from * VEC + (2 * i + 1) % VEC;
          if (c0 < a.dim) pw[which * a.dim + c0] = sum.x;
          if (c1 < a.dim) pw[which * a.dim + c1] = sum.y;
        }
      }
    }
  }
}

// Rows longer than the registers hold: one CTA per row, the row re-read (from
// L2) for each sum.
template <typename T>
__global__ void __launch_bounds__(kThreads) norm_fwd_wide_kernel(const NormArgs a) {
  chain_start();
  __shared__ float2 slots[2 * kWarps];
  T* out = static_cast<T*>(a.out);
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(a.x) + row * a.ld_x;
    float2 s = make_float2(0.f, 0.f);
    for (int c = threadIdx.x; c < a.dim; c += kThreads) s.x += to_float(x[c]);
    const float mean = team_sum<kThreads>(s, slots, 0).x * a.inv_dim;
    s = make_float2(0.f, 0.f);
    for (int c = threadIdx.x; c < a.dim; c += kThreads) {
      const float d = to_float(x[c]) - mean;
      s.x = fmaf(d, d, s.x);
    }
    const float rstd = 1.f / sqrtf(fmaf(team_sum<kThreads>(s, slots, 1).x, a.inv_dim, a.eps));
    for (int c = threadIdx.x; c < a.dim; c += kThreads) {
      const float w = a.weight != nullptr ? load_param(a.weight, a.param_dtype, c) : 1.f;
      const float b = a.bias != nullptr ? load_param(a.bias, a.param_dtype, c) : 0.f;
      out[row * a.dim + c] = from_float<T>(fmaf((to_float(x[c]) - mean) * rstd, w, b));
    }
    if (threadIdx.x == 0 && a.mean_out != nullptr) {
      a.mean_out[row] = mean;
      a.rstd_out[row] = rstd;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) norm_bwd_wide_kernel(const NormArgs a) {
  chain_start();
  __shared__ float2 slots[2 * kWarps];
  T* out = static_cast<T*>(a.out);
  int parity = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, parity ^= 1) {
    const T* x = static_cast<const T*>(a.x) + row * a.ld_x;
    const T* dy = static_cast<const T*>(a.dy) + row * a.ld_dy;
    const float mean = a.mean_in[row], rstd = a.rstd_in[row];
    float2 s = make_float2(0.f, 0.f);
    for (int c = threadIdx.x; c < a.dim; c += kThreads) {
      const float w = a.weight != nullptr ? load_param(a.weight, a.param_dtype, c) : 1.f;
      const float t = to_float(dy[c]) * w;
      s.x += t;
      s.y = fmaf(t, (to_float(x[c]) - mean) * rstd, s.y);
    }
    s = team_sum<kThreads>(s, slots, parity);
    const float m1 = s.x * a.inv_dim, m2 = s.y * a.inv_dim;
    for (int c = threadIdx.x; c < a.dim; c += kThreads) {
      const float w = a.weight != nullptr ? load_param(a.weight, a.param_dtype, c) : 1.f;
      const float u = (to_float(x[c]) - mean) * rstd;
      out[row * a.dim + c] = from_float<T>(rstd * (to_float(dy[c]) * w - fmaf(u, m2, m1)));
    }
  }
}

// Parameter gradients of wide rows: a thread owns one column over one slab of
// rows (blockIdx.y).
template <typename T>
__global__ void __launch_bounds__(kThreads) norm_wide_params_kernel(const NormArgs a) {
  chain_start();
  const int col = static_cast<int>(blockIdx.x) * kThreads + static_cast<int>(threadIdx.x);
  if (col >= a.dim) return;
  float dw = 0.f, db = 0.f;
  for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
    const float g = to_float((static_cast<const T*>(a.dy) + row * a.ld_dy)[col]);
    const float u = (to_float((static_cast<const T*>(a.x) + row * a.ld_x)[col]) - a.mean_in[row]) * a.rstd_in[row];
    dw = fmaf(g, u, dw);
    db += g;
  }
  float* p = a.partial + static_cast<int64_t>(blockIdx.y) * 2 * a.dim;
  p[col] = dw;
  p[a.dim + col] = db;
}

// Sums the CTAs' partials per column in a fixed order: 32 columns per CTA, each
// of 32 warps every 32nd partial, then the 32 sums.  blockIdx.y picks dw or db.
__global__ void __launch_bounds__(1024) norm_param_sum_kernel(const float* partial, int parts, int dim,
                                                              void* dweight, void* dbias, int param_dtype) {
  chain_start();
  __shared__ float sums[32][33];
  void* out = blockIdx.y == 0 ? dweight : dbias;
  if (out == nullptr) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int col = static_cast<int>(blockIdx.x) * 32 + lane;
  float s = 0.f;
  if (col < dim) {
    const float* p = partial + static_cast<int64_t>(blockIdx.y) * dim + col;
#pragma unroll 8
    for (int k = warp; k < parts; k += 32) s += p[static_cast<int64_t>(k) * 2 * dim];
  }
  sums[warp][lane] = s;
  __syncthreads();
  // warp w adds the 32 sums of column w
  s = sums[lane][warp];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(kFullMask, s, o);
  const int mine = static_cast<int>(blockIdx.x) * 32 + warp;
  if (lane == 0 && mine < dim) store_param(out, param_dtype, mine, s);
}

// CTAs of a grid that walks `rows` in steps of `teams` rows: what is needed, at
// most `per_sm` a SM.
int norm_ctas(int64_t rows, int teams, int per_sm) {
  const int64_t need = (rows + teams - 1) / teams;
  const int64_t most = static_cast<int64_t>(device_sm_count()) * per_sm;
  return static_cast<int>(need < most ? need : most);
}

// Most CTAs of the backward on one SM, which bounds its workspace.
constexpr int kBwdPerSm = 6;

// CTAs of `kernel` that one SM holds (asked once: the library runs on one kind
// of GPU), after raising the kernel's shared-memory limit for this context.
template <typename Kernel>
int resident(Kernel kernel, int threads, int bytes, unsigned long long* ready, int* per_sm) {
  const unsigned long long context = current_context_id();
  if (*per_sm > 0 && *ready == context && context != 0) return *per_sm;
  int n = 0;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess ||
      cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, threads, bytes) != cudaSuccess || n < 1) {
    cudaGetLastError();
    return 0;
  }
  *ready = context;
  *per_sm = n;
  return n;
}

template <typename T, int VEC, int TEAM, int CH, bool PARAMS>
int launch_bwd(const NormArgs& a, int* ctas, cudaStream_t stream) {
  constexpr int threads = cta_threads(TEAM, CH * VEC), bytes = 2 * Ahead<T, VEC, TEAM, CH>::kBytes;
  static thread_local unsigned long long ready = 0;
  static thread_local int per_sm = 0;
  const auto kernel = norm_bwd_kernel<T, VEC, TEAM, CH, PARAMS>;
  const int fit = resident(kernel, threads, bytes, &ready, &per_sm);
  if (fit == 0) return RFM_ERR_LAUNCH;
  *ctas = norm_ctas(a.rows, threads / TEAM, fit < kBwdPerSm ? fit : kBwdPerSm);
  return launch_chained(Chain::kFirst, kernel, dim3(*ctas), threads, bytes, 1, stream, a);
}

// The backward may have another team (BTEAM, BCH) than the forward.
template <typename T, int VEC, int TEAM, int CH, int BTEAM = TEAM, int BCH = CH>
int launch_norm(const NormArgs& a, bool backward, int* ctas, cudaStream_t stream) {
  if (backward) {
    return a.partial != nullptr ? launch_bwd<T, VEC, BTEAM, BCH, true>(a, ctas, stream)
                                : launch_bwd<T, VEC, BTEAM, BCH, false>(a, ctas, stream);
  }
  constexpr int threads = cta_threads(TEAM, CH * VEC), bytes = Ahead<T, VEC, TEAM, CH>::kBytes;
  static thread_local unsigned long long ready = 0;
  static thread_local int per_sm = 0;
  const auto kernel = norm_fwd_kernel<T, VEC, TEAM, CH>;
  const int fit = resident(kernel, threads, bytes, &ready, &per_sm);
  if (fit == 0) return RFM_ERR_LAUNCH;
  const dim3 grid(norm_ctas(a.rows, threads / TEAM, fit));
  return launch_chained(Chain::kFirst, kernel, grid, threads, bytes, 1, stream, a);
}

// The smallest team and register count that hold a row.
template <typename T>
int dispatch_norm(const NormArgs& a, bool vectors, bool backward, int* ctas, cudaStream_t s) {
  constexpr int V = 16 / static_cast<int>(sizeof(T));
  const int d = a.dim;
  if (d > kWideDim) {
    const int grid = norm_ctas(a.rows, 1, 8);
    if (!backward) return launch_chained(Chain::kFirst, norm_fwd_wide_kernel<T>, dim3(grid), kThreads, 0, 1, s, a);
    if (a.out != nullptr) {
      const int rc = launch_chained(Chain::kFirst, norm_bwd_wide_kernel<T>, dim3(grid), kThreads, 0, 1, s, a);
      if (rc != RFM_OK) return rc;
    }
    if (a.partial == nullptr) return RFM_OK;
    *ctas = static_cast<int>(a.rows < kWideSlabs ? a.rows : kWideSlabs);
    return launch_chained(a.out == nullptr ? Chain::kFirst : Chain::kNext, norm_wide_params_kernel<T>,
                          dim3((d + kThreads - 1) / kThreads, *ctas), kThreads, 0, 1, s, a);
  }
  // A warp a row up to 1024 columns (32 a lane): a team of several warps pays its
  // shuffles in each of them and a barrier twice a row (65536 x 1024 fp16, four
  // warps a row: 67 and 98 us, forward and backward; one warp: 49 and 80 us).  The
  // backward of 16-bit rows takes two warps, for the registers: 71 us.  That is 5.5
  // and 5.7 TB/s.
  if (vectors) {
    if (d <= 8 * V) return launch_norm<T, V, 8, 1>(a, backward, ctas, s);
    if (d <= 32 * V) return launch_norm<T, V, 32, 1>(a, backward, ctas, s);
    if (d <= 64 * V) return launch_norm<T, V, 32, 2>(a, backward, ctas, s);
    if (d <= 128 * V) return launch_norm<T, V, 32, 4, V == 8 ? 64 : 32, V == 8 ? 2 : 4>(a, backward, ctas, s);
    if constexpr (V == 4) {
      if (d <= 1024) return launch_norm<T, V, 32, 8>(a, backward, ctas, s);
    }
    if (d <= 2048) return launch_norm<T, V, 128, 16 / V>(a, backward, ctas, s);
    if (d <= 4096) return launch_norm<T, V, 256, 16 / V>(a, backward, ctas, s);
    return launch_norm<T, V, 512, 16 / V>(a, backward, ctas, s);
  }
  if (d <= 32) return launch_norm<T, 1, 8, 4>(a, backward, ctas, s);
  if (d <= 128) return launch_norm<T, 1, 32, 4>(a, backward, ctas, s);
  if (d <= 512) return launch_norm<T, 1, 32, 16>(a, backward, ctas, s);
  if (d <= 2048) return launch_norm<T, 1, 128, 16>(a, backward, ctas, s);
  return launch_norm<T, 1, 512, 16>(a, backward, ctas, s);
}

int run_norm(const NormArgs& a, int dtype, bool backward, int* ctas, cudaStream_t s) {
  const int v = 16 / dtype_bytes(dtype);
  const bool vectors = a.dim % v == 0 && a.ld_x % v == 0 && a.ld_dy % v == 0 && aligned16(a.x) && aligned16(a.dy) &&
                       aligned16(a.out);
  if (dtype == RFM_DTYPE_F32) return dispatch_norm<float>(a, vectors, backward, ctas, s);
  if (dtype == RFM_DTYPE_BF16) return dispatch_norm<__nv_bfloat16>(a, vectors, backward, ctas, s);
  return dispatch_norm<__half>(a, vectors, backward, ctas, s);
}

int norm_args(NormArgs& a, const void* x, int64_t ld_x, const void* weight, int64_t rows, int dim, int dtype,
              int param_dtype) {
  if (rows < 0 || dim < 1 || !dtype_known(dtype) || !dtype_known(param_dtype) ||
      (ld_x < dim && rows > 1) || ld_x < 0) {
    return RFM_ERR_INVALID_ARGUMENT;
  }
  if (rows > (int64_t(1) << 40) || ld_x > (int64_t(1) << 40) || dim > (1 << 30)) return RFM_ERR_UNSUPPORTED;
  if (rows > 0 && x == nullptr) return RFM_ERR_INVALID_ARGUMENT;
  a = NormArgs{};
  a.x = x;
  a.ld_x = ld_x;
  a.weight = weight;
  a.rows = rows;
  a.dim = dim;
  a.param_dtype = param_dtype;
  a.inv_dim = 1.f / static_cast<float>(dim);
  return RFM_OK;
}

}  // namespace
}  // namespace rfm

extern "C" int rfm_layer_norm_forward(const void* x, int64_t ld_x, const void* weight, const void* bias, void* out,
                                      float* mean, float* rstd, int64_t rows, int dim, float eps, int dtype,
                                      int param_dtype, void* stream) {
  using namespace rfm;
  NormArgs a;
  const int rc = norm_args(a, x, ld_x, weight, rows, dim, dtype, param_dtype);
  if (rc != RFM_OK) return rc;
  if ((mean == nullptr) != (rstd == nullptr) || !(eps >= 0.f)) return RFM_ERR_INVALID_ARGUMENT;
  if (rows == 0) return RFM_OK;
  if (out == nullptr) return RFM_ERR_INVALID_ARGUMENT;
  a.bias = bias;
  a.out = out;
  a.mean_out = mean;
  a.rstd_out = rstd;
  a.eps = eps;
  return run_norm(a, dtype, false, nullptr, as_stream(stream));
}

extern "C" int64_t rfm_layer_norm_workspace_bytes(int64_t rows, int dim) {
  using namespace rfm;
  if (rows < 0 || dim < 1) return -RFM_ERR_INVALID_ARGUMENT;
  const int64_t most = static_cast<int64_t>(device_sm_count()) * kBwdPerSm;
  const int64_t parts = dim > kWideDim ? kWideSlabs : (rows < most ? rows : most);
  return parts * 2 * dim * static_cast<int64_t>(sizeof(float));
}

extern "C" int rfm_layer_norm_backward(const void* x, int64_t ld_x, const void* weight, const float* mean,
                                       const float* rstd, const void* grad_out, int64_t ld_grad, void* grad_x,
                                       void* grad_weight, void* grad_bias, int64_t rows, int dim, int dtype,
                                       int param_dtype, void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace rfm;
  NormArgs a;
  const int rc = norm_args(a, x, ld_x, weight, rows, dim, dtype, param_dtype);
  if (rc != RFM_OK) return rc;
  if ((ld_grad < dim && rows > 1) || ld_grad < 0) return RFM_ERR_INVALID_ARGUMENT;
  const bool params = grad_weight != nullptr || grad_bias != nullptr;
  if (rows > 0 && (mean == nullptr || rstd == nullptr || grad_out == nullptr)) return RFM_ERR_INVALID_ARGUMENT;
  if (params && rows > 0 &&
      (workspace == nullptr || workspace_bytes < rfm_layer_norm_workspace_bytes(rows, dim))) {
    return RFM_ERR_INVALID_ARGUMENT;
  }
  if (grad_x == nullptr && !params) return RFM_OK;
  a.dy = grad_out;
  a.ld_dy = ld_grad;
  a.out = grad_x;
  a.mean_in = mean;
  a.rstd_in = rstd;
  a.partial = params ? static_cast<float*>(workspace) : nullptr;
  int ctas = 0;
  if (rows > 0) {
    const int done = run_norm(a, dtype, true, &ctas, as_stream(stream));
    if (done != RFM_OK) return done;
  }
  if (!params) return RFM_OK;
  // with no rows the sums are empty: zeros
  return launch_chained(rows == 0 ? Chain::kFirst : Chain::kNext, norm_param_sum_kernel, dim3((dim + 31) / 32, 2), 1024,
                        0, 1, as_stream(stream), a.partial, ctas, dim, grad_weight, grad_bias, param_dtype);
}
