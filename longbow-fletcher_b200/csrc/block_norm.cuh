// The norms around a block, its gate and residual (Cuda_BlockNorm), and the weighted sum of experts'
// outputs in front of them (Cuda_Combine_Grouped): one pass over the rows, which stay in registers
// in fp32 from the first load to the last store.
//
// Bound: HBM, at (inputs + outputs) * rows * cols * element size.  A row belongs to a team of 1 to 8
// warps, whose lanes hold up to NV 16-byte vectors each; teams walk the rows with a stride.  Sums
// are warp shuffles, joined through shared memory and a named barrier of the team where it has
// several warps.  LayerNorm's variance is the mean of squared deviations (a second pass over
// registers), as in Cuda_LayerNorm.
#pragma once
#include <algorithm>
#include <atomic>
#include <cmath>

#include "routing.cuh"
#include "tc_common.cuh"

namespace fl {
namespace bnorm {

constexpr int kThreads = 256;
constexpr int kMaxCols = 49152;  // the generic kernel keeps a row of fp32 in shared memory

struct NormArgs {
  const void* y;         // [rows, cols], or the slots' rows (combine)
  const int32_t* slots;  // combine: [rows, top_k]
  const float* weights;
  int32_t top_k;
  int32_t num_slots;     // slots from here on are none (GroupedArgs)
  const void* residual;  // null: 0
  const void* gate;      // null: 1
  int64_t gate_step;     // elements from one row's gate to the next: 0 or cols
  void* u;               // null: not stored
  void* h;
  const float *post_gamma, *post_beta, *pre_gamma, *pre_beta;
  int32_t post, pre;
  float eps, residual_scale, branch_scale;
  int64_t rows;
  int32_t cols;
};

// VEC elements moved at once: 16 bytes, or what a row's width allows.
template <int BYTES>
struct RawOf;
template <>
struct RawOf<32> {
  struct R {
    uint4 lo, hi;
  };
};
template <>
struct RawOf<16> {
  typedef uint4 R;
};
template <>
struct RawOf<8> {
  typedef uint2 R;
};
template <>
struct RawOf<4> {
  typedef uint32_t R;
};
template <>
struct RawOf<2> {
  typedef uint16_t R;
};
template <typename T, int VEC>
union Pack {
  typename RawOf<VEC * sizeof(T)>::R q;
  T t[VEC];
};

// One step of S = 2 values in packed fp32, or of one.
template <int S>
__device__ __forceinline__ void fma_s(float* d, const float* a, float b0, float b1, const float* c) {
  if constexpr (S == 1)
    d[0] = fmaf(a[0], b0, c[0]);
  else
    fma2(d[0], d[1], a[0], a[1], b0, b1, c[0], c[1]);
}
template <int S>
__device__ __forceinline__ void mul_s(float* d, float b0, float b1) {
  if constexpr (S == 1)
    d[0] *= b0;
  else
    mul2(d[0], d[1], d[0], d[1], b0, b1);
}
template <int S>
__device__ __forceinline__ void add_s(float* d, float b) {
  if constexpr (S == 1)
    d[0] += b;
  else
    add2(d[0], d[1], b, b);
}

// Sum over the team's lanes.  `red` has kSlots turns of 8 floats; turns alternate so that a warp
// that is still reading one sum cannot meet the next sum's writes.
constexpr int kTurns = 8;
template <int WPR>
__device__ __forceinline__ float team_sum(float s, float (*red)[8], int& turn) {
  s = warp_sum(s);
  if constexpr (WPR > 1) {
    const int warp = threadIdx.x >> 5, team = warp / WPR;
    if ((threadIdx.x & 31) == 0) red[turn][warp] = s;
    asm volatile("bar.sync %0, %1;" ::"r"(team + 1), "r"(WPR * 32) : "memory");
    s = 0.f;
#pragma unroll
    for (int i = 0; i < WPR; i++) s += red[turn][team * WPR + i];
    turn = (turn + 1) % kTurns;
  }
  return s;
}

// Whether all lanes hold a vector j: in a FULL row each does, and with 4 or 8 values a vector all but the
// last (the launch takes no more of them than the row needs).
template <int VEC, int NV, bool FULL>
__device__ __forceinline__ constexpr bool kWhole(int j) {
  return FULL || (VEC >= 4 && j < NV - 1);
}

// v = norm(v) for the team's row: lane t holds vectors t, t + TPR, ...; what lies past the row is 0
// and stays out of the sums.  FULL: the lanes' vectors are exactly the row.  Packed pairs of fp32, with
// the uniform choices outside the loops: at 16-bit widths instructions weigh as much as bytes (with the
// choices inside, 1100 instructions a row of 1024 and 78 us for 49152 rows, against 67).
template <int VEC, int NV, int WPR, bool FULL>
__device__ __forceinline__ void norm_row(float (&v)[NV * VEC], int kind, const float* __restrict__ gamma,
                                         const float* __restrict__ beta, float eps, int t, int nvec, int cols,
                                         float (*red)[8], int& turn) {
  constexpr int TPR = 32 * WPR;
  constexpr int S = VEC == 1 ? 1 : 2, Q = VEC < 4 ? S : 4;  // values a step, and a load of gamma or beta
  if (kind == FLETCHER_NORM_NONE) return;
  if (kind == FLETCHER_NORM_LAYER) {
    float p[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NV * VEC; i += 2) add2(p[0], p[1], v[i], v[i + 1]);
    const float mean = team_sum<WPR>(p[0] + p[1], red, turn) / (float)cols;
#pragma unroll
    for (int j = 0; j < NV; j++)
      if (kWhole<VEC, NV, FULL>(j) || j * TPR + t < nvec) {
#pragma unroll
        for (int i = j * VEC; i < (j + 1) * VEC; i += S) add_s<S>(&v[i], -mean);
      }
  }
  float q[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < NV * VEC; i += 2) fma2(q[i & 2], q[(i & 2) + 1], v[i], v[i + 1], v[i], v[i + 1], q[i & 2], q[(i & 2) + 1]);
  const float inv = 1.0f / sqrtf(team_sum<WPR>((q[0] + q[1]) + (q[2] + q[3]), red, turn) / (float)cols + eps);
#pragma unroll
  for (int i = 0; i < NV * VEC; i += 2) mul2(v[i], v[i + 1], v[i], v[i + 1], inv, inv);
  auto table = [&](const float* src, float (&d)[Q], int at) {
    if constexpr (Q == 4) {
      const float4 f = __ldg(reinterpret_cast<const float4*>(src + at));
      d[0] = f.x, d[1] = f.y, d[2] = f.z, d[3] = f.w;
    } else {
#pragma unroll
      for (int k = 0; k < Q; k++) d[k] = __ldg(src + at + k);
    }
  };
  const float one = 1.0f;
  auto scale = [&](auto with_gamma, auto with_beta) {
#pragma unroll
    for (int j = 0; j < NV; j++)
      if (kWhole<VEC, NV, FULL>(j) || j * TPR + t < nvec) {
#pragma unroll
        for (int i = 0; i < VEC; i += Q) {
          float* x = &v[j * VEC + i];
          float g[Q], b[Q];
          const int at = (j * TPR + t) * VEC + i;
          if constexpr (decltype(with_gamma)::value) table(gamma, g, at);
          if constexpr (decltype(with_beta)::value) table(beta, b, at);
#pragma unroll
          for (int k = 0; k < Q; k += S) {
            if constexpr (decltype(with_gamma)::value && decltype(with_beta)::value)
              fma_s<S>(x + k, x + k, g[k], g[k + S - 1], &b[k]);
            else if constexpr (decltype(with_gamma)::value)
              mul_s<S>(x + k, g[k], g[k + S - 1]);
            else
              fma_s<S>(x + k, x + k, one, one, &b[k]);
          }
        }
      }
  };
  if (gamma && beta)
    scale(std::true_type{}, std::true_type{});
  else if (gamma)
    scale(std::true_type{}, std::false_type{});
  else if (beta)
    scale(std::false_type{}, std::true_type{});
}

// A row's inputs are asked for one row ahead: the next y (or the first kAhead choices' rows, whose slots
// are asked for two rows ahead) while this row is normed, the next residual once this one is used.
constexpr int kAhead = 2;  // one of fp32 slots beside 16-bit rows, which take the registers of two
// Blocks an SM, by the registers that a row's vectors need (two choices' rows and a residual in flight):
// 65536 x 768 norms take 78 us with 2, 90 with 3, which spills.
template <int VEC, int NV>
constexpr int kMinBlocks = VEC <= 2 || NV > 2 ? 2 : NV == 2 ? 3 : 4;
// TY: the type of y, T, or for a combine also fp32.
template <typename T, typename TY, int VEC, int NV, int WPR, bool FULL, bool COMBINE>
__global__ void __launch_bounds__(kThreads, kMinBlocks<VEC, NV>) k_block_norm(const NormArgs a) {
  constexpr int TPR = 32 * WPR, TEAMS = kThreads / TPR;
  constexpr int S = VEC == 1 ? 1 : 2;
  typedef Pack<T, VEC> P;
  typedef decltype(P::q) Raw;
  typedef Pack<TY, VEC> PY;
  static_assert(NV * VEC % 2 == 0, "sums go in pairs");
  constexpr int NY = COMBINE && sizeof(TY) == sizeof(T) ? kAhead : 1;
  __shared__ float red[kTurns][8];
  int turn = 0;
  const int lane = threadIdx.x & 31, t = threadIdx.x % TPR, team = threadIdx.x / TPR;
  const int nvec = a.cols / VEC;
  const int64_t step = (int64_t)gridDim.x * TEAMS;
  int64_t row = (int64_t)blockIdx.x * TEAMS + team;
  PY py[NY][NV];
  P pr[NV];
  auto load = [&](auto& p, const void* base, int64_t r) {
    typedef typename std::remove_reference<decltype(p[0].q)>::type R;
    const R* src = reinterpret_cast<const R*>(base) + r * nvec + t;
#pragma unroll
    for (int j = 0; j < NV; j++)
      if (kWhole<VEC, NV, FULL>(j) || j * TPR + t < nvec) {
        // A one-warp row's choices pass by L1, which keeps gamma and beta (32768 x 2 x 768: 39 us against
        // 43; rows of several warps are slower with it, 32768 x 1 x 2048 102 against 94).
        if constexpr (COMBINE && WPR == 1 && sizeof(R) == 16)
          asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                       : "=r"(p[j].q.x), "=r"(p[j].q.y), "=r"(p[j].q.z), "=r"(p[j].q.w)
                       : "l"(src + j * TPR));
        else
          p[j].q = src[j * TPR];
      }
  };
  // Combine: lane j < top_k holds choice j of the current and of the next row.
  int32_t slot = -1, slot_next = -1;
  float w = 0.f, w_next = 0.f;
  auto load_slot = [&](int64_t r, int32_t& s, float& f) {
    s = -1;
    if (r < a.rows && lane < a.top_k) {
      s = a.slots[r * a.top_k + lane];
      f = a.weights[r * a.top_k + lane];
    }
  };
  // Asked where a slot is used, not where it is loaded: that would wait for the load (32768 x 2 x 768: 41 us).
  auto some = [&](int32_t s) { return (uint32_t)s < (uint32_t)a.num_slots; };
  auto load_y = [&](int64_t r, int32_t s) {
    if constexpr (COMBINE) {
#pragma unroll
      for (int j = 0; j < NY; j++) {
        const int32_t sj = __shfl_sync(0xffffffffu, s, j);  // -1 past the choices
        if (some(sj)) load(py[j], a.y, sj);
      }
    } else if (r < a.rows) {
      load(py[0], a.y, r);
    }
  };
  pdl_wait();
  if constexpr (COMBINE) {
    load_slot(row, slot, w);
    load_slot(row + step, slot_next, w_next);
  }
  load_y(row, slot);
  if (a.residual && row < a.rows) load(pr, a.residual, row);
  for (; row < a.rows; row += step) {
    float v[NV * VEC];
    auto add = [&](const auto& p, float scale) {
      typedef typename std::remove_cv<typename std::remove_reference<decltype(p[0].t[0])>::type>::type E;
#pragma unroll
      for (int j = 0; j < NV; j++)
        if (kWhole<VEC, NV, FULL>(j) || j * TPR + t < nvec) {
#pragma unroll
          for (int i = 0; i < VEC; i += S) {
            const float f[2] = {to_f<E>(p[j].t[i]), to_f<E>(p[j].t[i + S - 1])};
            fma_s<S>(&v[j * VEC + i], f, scale, scale, &v[j * VEC + i]);
          }
        }
    };
    P pg[NV];
    if (a.gate) {
      const Raw* src = reinterpret_cast<const Raw*>(reinterpret_cast<const T*>(a.gate) + row * a.gate_step) + t;
#pragma unroll
      for (int j = 0; j < NV; j++)
        if (kWhole<VEC, NV, FULL>(j) || j * TPR + t < nvec) pg[j].q = src[j * TPR];
    }
#pragma unroll
    for (int i = 0; i < NV * VEC; i++) v[i] = 0.f;
    if constexpr (COMBINE) {
#pragma unroll
      for (int j = 0; j < NY; j++) {
        const float wj = __shfl_sync(0xffffffffu, w, j);
        if (some(__shfl_sync(0xffffffffu, slot, j))) add(py[j], wj);
      }
      for (int j = NY; j < a.top_k; j++) {
        const int32_t sj = __shfl_sync(0xffffffffu, slot, j);
        const float wj = __shfl_sync(0xffffffffu, w, j);
        if (some(sj)) {
          load(py[0], a.y, sj);
          add(py[0], wj);
        }
      }
      slot = slot_next;
      w = w_next;
      load_slot(row + 2 * step, slot_next, w_next);
    } else {
      add(py[0], 1.0f);
    }
    load_y(row + step, slot);
    norm_row<VEC, NV, WPR, FULL>(v, a.post, a.post_gamma, a.post_beta, a.eps, t, nvec, a.cols, red, turn);
    if (a.gate) {
#pragma unroll
      for (int j = 0; j < NV; j++)
        if (kWhole<VEC, NV, FULL>(j) || j * TPR + t < nvec) {
#pragma unroll
          for (int i = 0; i < VEC; i += S) mul_s<S>(&v[j * VEC + i], to_f<T>(pg[j].t[i]), to_f<T>(pg[j].t[i + S - 1]));
        }
    }
    if (a.branch_scale != 1.0f) {
#pragma unroll
      for (int i = 0; i < NV * VEC; i += 2) mul2(v[i], v[i + 1], v[i], v[i + 1], a.branch_scale, a.branch_scale);
    }
    if (a.residual) {
      add(pr, a.residual_scale);
      if (row + step < a.rows) load(pr, a.residual, row + step);
    }
    auto store = [&](void* to) {
      Raw* dst = reinterpret_cast<Raw*>(to) + row * nvec + t;
#pragma unroll
      for (int j = 0; j < NV; j++) {
        if (kWhole<VEC, NV, FULL>(j) || j * TPR + t < nvec) {
          P o;
          if constexpr (sizeof(T) == 2 && VEC > 1) {
#pragma unroll
            for (int i = 0; i < VEC; i += 2)
              reinterpret_cast<uint32_t*>(&o)[i / 2] = tc::pack2<T>(v[j * VEC + i], v[j * VEC + i + 1]);
          } else {
#pragma unroll
            for (int i = 0; i < VEC; i++) o.t[i] = from_f<T>(v[j * VEC + i]);
          }
          dst[j * TPR] = o.q;
        }
      }
    };
    if (a.u) store(a.u);
    if (a.pre != FLETCHER_NORM_NONE) {
      norm_row<VEC, NV, WPR, FULL>(v, a.pre, a.pre_gamma, a.pre_beta, a.eps, t, nvec, a.cols, red, turn);
      store(a.h);
    }
  }
}

__device__ __forceinline__ float block_sum(float s, float* red) {
  s = warp_sum(s);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
  __syncthreads();
  s = 0.f;
#pragma unroll
  for (int i = 0; i < kThreads / 32; i++) s += red[i];
  return s;
}

__device__ __forceinline__ void norm_generic(float* v, int kind, const float* gamma, const float* beta, float eps,
                                             int cols, float* red) {
  if (kind == FLETCHER_NORM_NONE) return;
  float s = 0.f, mean = 0.f;
  if (kind == FLETCHER_NORM_LAYER) {
    for (int c = threadIdx.x; c < cols; c += kThreads) s += v[c];
    mean = block_sum(s, red) / (float)cols;
    s = 0.f;
  }
  for (int c = threadIdx.x; c < cols; c += kThreads) {
    const float d = v[c] - mean;
    v[c] = d;
    s = fmaf(d, d, s);
  }
  const float inv = 1.0f / sqrtf(block_sum(s, red) / (float)cols + eps);
  for (int c = threadIdx.x; c < cols; c += kThreads)
    v[c] = fmaf(v[c] * inv, gamma ? gamma[c] : 1.0f, beta ? beta[c] : 0.0f);
}

// Any width: a block per row, the row in shared memory, each column always with the
// same thread (so outputs may lie over inputs).
template <typename T, typename TY, bool COMBINE>
__global__ void __launch_bounds__(kThreads) k_block_norm_generic(const NormArgs a) {
  extern __shared__ float v[];
  __shared__ float red[kThreads / 32];
  pdl_wait();
  const TY* y = reinterpret_cast<const TY*>(a.y);
  const T *res = reinterpret_cast<const T*>(a.residual), *gate = reinterpret_cast<const T*>(a.gate);
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    for (int c = threadIdx.x; c < a.cols; c += kThreads) {
      float s = 0.f;
      if constexpr (COMBINE) {
        for (int j = 0; j < a.top_k; j++) {
          const int32_t slot = a.slots[row * a.top_k + j];
          if ((uint32_t)slot < (uint32_t)a.num_slots) s = fmaf(a.weights[row * a.top_k + j], to_f<TY>(y[(int64_t)slot * a.cols + c]), s);
        }
      } else {
        s = to_f<TY>(y[row * a.cols + c]);
      }
      v[c] = s;
    }
    norm_generic(v, a.post, a.post_gamma, a.post_beta, a.eps, a.cols, red);
    for (int c = threadIdx.x; c < a.cols; c += kThreads) {
      float s = v[c];
      if (gate) s *= to_f<T>(gate[row * a.gate_step + c]);
      s *= a.branch_scale;
      if (res) s = fmaf(a.residual_scale, to_f<T>(res[row * a.cols + c]), s);
      v[c] = s;
      if (a.u) reinterpret_cast<T*>(a.u)[row * a.cols + c] = from_f<T>(s);
    }
    if (a.pre != FLETCHER_NORM_NONE) {
      norm_generic(v, a.pre, a.pre_gamma, a.pre_beta, a.eps, a.cols, red);
      for (int c = threadIdx.x; c < a.cols; c += kThreads) reinterpret_cast<T*>(a.h)[row * a.cols + c] = from_f<T>(v[c]);
    }
  }
}

template <typename T, typename TY, int VEC, int NV, int WPR, bool COMBINE, bool FULL = false>
int32_t launch_vec(Ctx* c, const NormArgs& a) {
  if constexpr (!FULL && VEC * sizeof(T) == 16)
    if (a.cols == NV * VEC * WPR * 32) return launch_vec<T, TY, VEC, NV, WPR, COMBINE, true>(c, a);
  constexpr int TEAMS = kThreads / (32 * WPR);
  // As few teams as walk the rows in the same number of turns.
  const int64_t most = (int64_t)c->num_sms * kMinBlocks<VEC, NV> * TEAMS;
  const int64_t turns = (a.rows + most - 1) / most;
  const int64_t blocks = (a.rows + turns * TEAMS - 1) / (turns * TEAMS);
  FL_CUDA(c, launch_pdl(k_block_norm<T, TY, VEC, NV, WPR, FULL, COMBINE>, dim3((unsigned)blocks), dim3(kThreads), 0, c->stream, a));
  FL_LAUNCH(c);
  return FLETCHER_OK;
}

// Widths that 16 bytes do not divide: pairs or single elements, more of them a lane.
template <typename T, typename TY, int VEC, bool COMBINE>
int32_t launch_narrow(Ctx* c, const NormArgs& a) {
  const int nvec = a.cols / VEC;
  if (nvec <= 256) return launch_vec<T, TY, VEC, 8, 1, COMBINE>(c, a);
  if (nvec <= 1024) return launch_vec<T, TY, VEC, 16, 2, COMBINE>(c, a);
  return launch_vec<T, TY, VEC, 16, 8, COMBINE>(c, a);
}
constexpr int kNarrowMost = 16 * 256;

template <typename T, typename TY, bool COMBINE>
int32_t launch_norm(Ctx* c, const NormArgs& a) {
  constexpr int VEC = 16 / sizeof(T);
  const int nvec = a.cols / VEC;
  if (a.cols % VEC == 0 && nvec <= 1024) {
    // The fewest warps a row whose lanes hold at most four vectors each (two vectors in twice the warps:
    // 49152 x 1024 in 87 us against 79, 65536 x 768 in 102 against 80).
    if (nvec <= 32) return launch_vec<T, TY, VEC, 1, 1, COMBINE>(c, a);
    if (nvec <= 64) return launch_vec<T, TY, VEC, 2, 1, COMBINE>(c, a);
    if (nvec <= 96) return launch_vec<T, TY, VEC, 3, 1, COMBINE>(c, a);
    if (nvec <= 128) return launch_vec<T, TY, VEC, 4, 1, COMBINE>(c, a);
    if (nvec <= 192) return launch_vec<T, TY, VEC, 3, 2, COMBINE>(c, a);
    if (nvec <= 256) return launch_vec<T, TY, VEC, 4, 2, COMBINE>(c, a);
    if (nvec <= 384) return launch_vec<T, TY, VEC, 3, 4, COMBINE>(c, a);
    if (nvec <= 512) return launch_vec<T, TY, VEC, 4, 4, COMBINE>(c, a);
    if (nvec <= 768) return launch_vec<T, TY, VEC, 3, 8, COMBINE>(c, a);
    return launch_vec<T, TY, VEC, 4, 8, COMBINE>(c, a);
  }
  if constexpr (sizeof(T) == 2) {
    if (a.cols % 2 == 0 && a.cols <= 2 * kNarrowMost) return launch_narrow<T, TY, 2, COMBINE>(c, a);
  }
  if (a.cols <= kNarrowMost) return launch_narrow<T, TY, 1, COMBINE>(c, a);
  auto kern = k_block_norm_generic<T, TY, COMBINE>;
  const int smem = a.cols * 4;
  static std::atomic<bool> attr_set[64] = {};  // per device; idempotent, replicas' threads may meet here
  if (!attr_set[c->device & 63].load(std::memory_order_acquire)) {
    FL_CUDA(c, cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxCols * 4));
    attr_set[c->device & 63].store(true, std::memory_order_release);
  }
  const int64_t blocks = std::min<int64_t>(a.rows, (int64_t)c->num_sms * 8);
  FL_CUDA(c, launch_pdl(kern, dim3((unsigned)blocks), dim3(kThreads), smem, c->stream, a));
  FL_LAUNCH(c);
  return FLETCHER_OK;
}

}  // namespace bnorm

// dtype: of the outputs and of what is not a table; slots_dtype: that, or f32.
int32_t launch_block_norm(Ctx* c, int32_t dtype, const bnorm::NormArgs& a);                     // block_norm.cu
int32_t launch_combine(Ctx* c, int32_t dtype, int32_t slots_dtype, const bnorm::NormArgs& a);  // combine.cu

}  // namespace fl
