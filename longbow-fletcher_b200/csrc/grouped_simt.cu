// Grouped product on the fp32 units: f32 (the parity type) and the 16-bit shapes the tensor-core
// kernels do not take (widths that 16 bytes do not divide, TANH).
#include <algorithm>

#include "routing.cuh"

namespace fl {
namespace {

// The block's group and rows: m-tile `tile` of all groups' m-tiles in order; the tile's first slot
// and the group's end, expert -1 when there are fewer tiles.  No slot lies past `pairs` (GroupedArgs).
// Called by one warp.
__device__ __forceinline__ void find_tile(const int32_t* __restrict__ offsets, int E, int32_t pairs, int tile,
                                          int rows_per_tile, int32_t* expert, int32_t* first, int32_t* end) {
  const int lane = threadIdx.x & 31;
  int before = 0, e_found = -1, f = 0, n = 0;
  for (int b = 0; b < E; b += 32) {
    const int e = b + lane;
    const int32_t o0 = e < E ? min(offsets[e], pairs) : 0, o1 = e < E ? min(offsets[e + 1], pairs) : 0;
    const int tiles = (o1 - o0 + rows_per_tile - 1) / rows_per_tile;
    int s = tiles;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += u;
    }
    const int at = tile - before - (s - tiles);  // the tile's index within this lane's expert
    const uint32_t hit = __ballot_sync(0xffffffffu, at >= 0 && at < tiles);
    if (hit) {
      const int src = __ffs(hit) - 1;
      e_found = b + src;
      f = __shfl_sync(0xffffffffu, o0 + at * rows_per_tile, src);
      n = __shfl_sync(0xffffffffu, o1, src);
      break;
    }
    before += __shfl_sync(0xffffffffu, s, 31);
  }
  if (lane == 0) {
    *expert = e_found;
    *first = f;
    *end = n;
  }
}

template <typename T, int ACT>
__device__ __forceinline__ float act1(float v) {
  if constexpr (ACT == FLETCHER_ACT_GELU) return sizeof(T) == 4 ? gelu_fast(v) : gelu_fast16(v);
  if constexpr (ACT == FLETCHER_ACT_TANH) return tanh_fast(v);
  return v;
}

// One BM x BN output tile a block (SwiGLU: its gate and up columns), TM x TN sums a thread in packed pairs
// along n, K in slabs of 16: the next slab's elements are on their way from memory while this one's are
// multiplied from shared memory.  Rows are gathered as they are loaded; single elements, so that any
// width does.  KS teams of threads take alternate slabs.  At 4000 x 2 rows of 8
// experts, 500 -> 500, it gives 34 TFLOP/s, under half of the fp32 units' rate (74 at 1.95 GHz): beside the packed
// multiply-adds stand single loads with a test each, transposing stores and the (x, x) pairs.  Few rows are
// bound by a slab's chain of load, store and multiply, which teams overlap.
template <typename T, int ACT, int BM, int BN, int TM, int TN, int KS>
__global__ void __launch_bounds__((BM / TM) * (BN / TN) * KS) k_grouped_simt(const GroupedArgs a) {
  constexpr int BK = 16, kThreads = (BM / TM) * (BN / TN);  // of one of the KS teams
  constexpr bool GATED = ACT == FLETCHER_ACT_SWIGLU;
  constexpr int NB = GATED ? 2 : 1;
  constexpr int XL = BM * BK / kThreads, WL = BN * BK / kThreads;  // elements a thread loads
  static_assert(kThreads % BK == 0 && kThreads % BN == 0 && TM % 4 == 0 && TN == 4, "thread layout");
  __shared__ __align__(16) float s_x[KS][2][BK][BM + 4], s_w[KS][2][NB][BK][BN];
  __shared__ int32_t s_tile[3];
  const int tid = threadIdx.x % kThreads, team = threadIdx.x / kThreads;
  auto& sx = s_x[team];
  auto& sw = s_w[team];
  auto team_sync = [&]() {
    if constexpr (KS > 1)
      asm volatile("bar.sync %0, %1;" ::"r"(team + 1), "n"(kThreads) : "memory");
    else
      __syncthreads();
  };
  const unsigned nt = (unsigned)((a.n_out + BN - 1) / BN);  // n-tiles, fastest
  pdl_wait();
  if (threadIdx.x < 32)
    find_tile(a.offsets, a.experts, (int32_t)a.pairs, (int)(blockIdx.x / nt), BM, &s_tile[0], &s_tile[1], &s_tile[2]);
  __syncthreads();
  const int e = s_tile[0];
  if (e < 0) return;
  const int first = s_tile[1], end = s_tile[2];
  const int64_t n0 = (int64_t)(blockIdx.x % nt) * BN;
  // This thread loads column xk of rows xm + i * (kThreads / BK), and column wn of rows wk + i * (kThreads / BN).
  const int xk = tid % BK, xm = tid / BK, wn = tid % BN, wk = tid / BN;
  const T* xrow[XL];
#pragma unroll
  for (int i = 0; i < XL; i++) {
    const int s = first + xm + i * (kThreads / BK);
    const int64_t r = s >= end ? -1 : a.pair_of ? min((int64_t)(a.pair_of[s] / a.top_k), a.x_rows - 1) : s;
    xrow[i] = r < 0 ? nullptr : reinterpret_cast<const T*>(a.x) + r * a.K + xk;
  }
  const T* w = reinterpret_cast<const T*>(a.w) + (int64_t)e * a.K * a.N + n0 + wn;
  const bool w_in = n0 + wn < a.n_out;
  T rx[XL], rw[NB][WL];
  auto load = [&](int64_t k0) {
#pragma unroll
    for (int i = 0; i < XL; i++) rx[i] = xrow[i] && k0 + xk < a.K ? xrow[i][k0] : from_f<T>(0.f);
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
      for (int i = 0; i < WL; i++) {
        const int64_t k = k0 + wk + i * (kThreads / BN);
        rw[b][i] = w_in && k < a.K ? w[k * a.N + b * a.n_out] : from_f<T>(0.f);
      }
  };
  auto store = [&](int buf) {
#pragma unroll
    for (int i = 0; i < XL; i++) sx[buf][xk][xm + i * (kThreads / BK)] = to_f<T>(rx[i]);
#pragma unroll
    for (int b = 0; b < NB; b++)
#pragma unroll
      for (int i = 0; i < WL; i++) sw[buf][b][wk + i * (kThreads / BN)][wn] = to_f<T>(rw[b][i]);
  };
  const int tx = tid % (BN / TN), ty = tid / (BN / TN);
  float acc[NB][TM][TN] = {};
  load(team * BK);
  store(0);
  team_sync();
  int buf = 0;
  for (int64_t k0 = team * BK; k0 < a.K; k0 += KS * BK, buf ^= 1) {
    const bool more = k0 + KS * BK < a.K;
    if (more) load(k0 + KS * BK);
#pragma unroll
    for (int k = 0; k < BK; k++) {
      float xv[TM];
#pragma unroll
      for (int i = 0; i < TM; i += 4) {
        const float4 q = *reinterpret_cast<const float4*>(&sx[buf][k][ty * TM + i]);
        xv[i] = q.x, xv[i + 1] = q.y, xv[i + 2] = q.z, xv[i + 3] = q.w;
      }
#pragma unroll
      for (int b = 0; b < NB; b++) {
        const float4 q = *reinterpret_cast<const float4*>(&sw[buf][b][k][tx * TN]);
#pragma unroll
        for (int i = 0; i < TM; i++) {
          float* c = acc[b][i];
          fma2(c[0], c[1], xv[i], xv[i], q.x, q.y, c[0], c[1]);
          fma2(c[2], c[3], xv[i], xv[i], q.z, q.w, c[2], c[3]);
        }
      }
    }
    if (more) store(buf ^ 1);
    team_sync();
  }
  if constexpr (KS > 1) {  // the teams' sums, added in their order by the first
    float* red = &s_x[0][0][0][0];
    static_assert(sizeof(s_x) >= sizeof(float) * (KS - 1) * kThreads * TM * TN, "room for one operand's sums");
#pragma unroll
    for (int b = 0; b < NB; b++) {
      __syncthreads();
      if (team > 0) {
#pragma unroll
        for (int i = 0; i < TM * TN; i++) red[((team - 1) * TM * TN + i) * kThreads + tid] = acc[b][i / TN][i % TN];
      }
      __syncthreads();
      if (team == 0) {
#pragma unroll
        for (int t = 0; t < KS - 1; t++)
#pragma unroll
          for (int i = 0; i < TM * TN; i++) acc[b][i / TN][i % TN] += red[(t * TM * TN + i) * kThreads + tid];
      }
    }
    if (team > 0) return;
  }
  const T* bias = a.bias ? reinterpret_cast<const T*>(a.bias) + (int64_t)e * a.N : nullptr;
  T* out = reinterpret_cast<T*>(a.out);
#pragma unroll
  for (int i = 0; i < TM; i++) {
    const int64_t s = first + ty * TM + i;
    if (s >= end) continue;
#pragma unroll
    for (int j = 0; j < TN; j++) {
      const int64_t n = n0 + tx * TN + j;
      if (n >= a.n_out) continue;
      float v = acc[0][i][j] + (bias ? to_f<T>(bias[n]) : 0.f);
      if constexpr (GATED) {
        const float u = acc[NB - 1][i][j] + (bias ? to_f<T>(bias[a.n_out + n]) : 0.f);
        v = sizeof(T) == 4 ? swiglu_exact(v, u) : a.out32 ? swiglu_f32(v, u) : swiglu_16(v, u);
      } else {
        v = act1<T, ACT>(v);
      }
      if (a.out32)
        reinterpret_cast<float*>(a.out)[s * a.n_out + n] = v;
      else
        out[s * a.n_out + n] = from_f<T>(v);
    }
  }
}

template <typename T, int ACT, int BM, int BN, int TM, int TN, int KS>
int32_t run(Ctx* c, const GroupedArgs& a) {
  const int64_t nt = (a.n_out + BN - 1) / BN;
  const int64_t mt = a.pairs / BM + std::min<int64_t>(a.experts, a.pairs);  // at most this many m-tiles
  FL_CHECK(c, nt * mt <= INT32_MAX, "Linear_Grouped: %lldx%lld is too large for the fp32 units", (long long)a.pairs,
           (long long)a.n_out);
  FL_CUDA(c, launch_pdl(k_grouped_simt<T, ACT, BM, BN, TM, TN, KS>, dim3((unsigned)(nt * mt)),
                        dim3((BM / TM) * (BN / TN) * KS), 0, c->stream, a));
  FL_LAUNCH(c);
  return FLETCHER_OK;
}

template <typename T, int ACT>
int32_t pick(Ctx* c, const GroupedArgs& a) {
  // 64 x 64 tiles where there are two for every SM, else 32 x 32 by four teams (SwiGLU's two operands: two),
  // so that more SMs and warps share few rows (509 rows of 5 experts, 129 -> 130: 8.6 us, 15.1 in 64 x 64 tiles).
  const int64_t tiles = (a.pairs / 64 + std::min<int64_t>(a.experts, a.pairs)) * ((a.n_out + 63) / 64);
  if (tiles >= 2 * c->num_sms) return run<T, ACT, 64, 64, 8, 4, 1>(c, a);
  return run<T, ACT, 32, 32, 4, 4, ACT == FLETCHER_ACT_SWIGLU ? 2 : 4>(c, a);
}

template <typename T>
int32_t launch(Ctx* c, const GroupedArgs& a) {
  switch (a.act) {
    case FLETCHER_ACT_IDENTITY:
      return pick<T, FLETCHER_ACT_IDENTITY>(c, a);
    case FLETCHER_ACT_GELU:
      return pick<T, FLETCHER_ACT_GELU>(c, a);
    case FLETCHER_ACT_TANH:
      return pick<T, FLETCHER_ACT_TANH>(c, a);
    default:
      return pick<T, FLETCHER_ACT_SWIGLU>(c, a);
  }
}

}  // namespace

int32_t launch_grouped_simt(Ctx* c, int32_t dtype, const GroupedArgs& a) {
  if (dtype == FLETCHER_BF16) return launch<__nv_bfloat16>(c, a);
  if (dtype == FLETCHER_F16) return launch<__half>(c, a);
  return launch<float>(c, a);
}

}  // namespace fl
