// Grouped product on the fp32 units: f32 (the parity type) and the 16-bit shapes the tensor-core
// kernels do not take (widths that 16 bytes do not divide, unaligned buffers, TANH).
#include <algorithm>

#include "routing.cuh"

namespace fl {
namespace {

constexpr int BM = 64, BN = 64, BK = 16, TM = 4, TN = 4;
constexpr int kThreads = (BM / TM) * (BN / TN);

// The block's group and rows: m-tile `tile` of all groups' m-tiles in order; the tile's first slot
// and the group's end, expert -1 when there are fewer tiles.  Called by one warp.
__device__ __forceinline__ void find_tile(const int32_t* __restrict__ offsets, int E, int tile, int rows_per_tile,
                                          int32_t* expert, int32_t* first, int32_t* end) {
  const int lane = threadIdx.x & 31;
  int before = 0, e_found = -1, f = 0, n = 0;
  for (int b = 0; b < E; b += 32) {
    const int e = b + lane;
    const int32_t o0 = e < E ? offsets[e] : 0, o1 = e < E ? offsets[e + 1] : 0;
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

// One 64 x 64 output tile a block (SwiGLU: its gate and up columns), 4 x 4 sums a thread, K in
// slabs of 16 through shared memory; rows are gathered as the slab is loaded.
template <typename T, int ACT>
__global__ void __launch_bounds__(kThreads) k_grouped_simt(const GroupedArgs a) {
  constexpr bool GATED = ACT == FLETCHER_ACT_SWIGLU;
  constexpr int NB = GATED ? 2 : 1;
  __shared__ float sx[BK][BM + 4], sw[NB][BK][BN];
  __shared__ int32_t s_tile[3];
  __shared__ int64_t s_row[BM];
  const unsigned nt = (unsigned)((a.n_out + BN - 1) / BN);  // n-tiles, fastest
  pdl_wait();
  if (threadIdx.x < 32) find_tile(a.offsets, a.experts, (int)(blockIdx.x / nt), BM, &s_tile[0], &s_tile[1], &s_tile[2]);
  __syncthreads();
  const int e = s_tile[0];
  if (e < 0) return;
  const int64_t first = s_tile[1], end = s_tile[2];
  for (int i = threadIdx.x; i < BM; i += kThreads) {
    const int64_t s = first + i;
    s_row[i] = s >= end ? -1 : a.pair_of ? a.pair_of[s] / a.top_k : s;
  }
  __syncthreads();
  const int64_t n0 = (int64_t)(blockIdx.x % nt) * BN;
  const T* x = reinterpret_cast<const T*>(a.x);
  const T* w = reinterpret_cast<const T*>(a.w) + (int64_t)e * a.K * a.N;
  const int tx = threadIdx.x % (BN / TN), ty = threadIdx.x / (BN / TN);
  float acc[NB][TM][TN] = {};
  for (int64_t k0 = 0; k0 < a.K; k0 += BK) {
    for (int i = threadIdx.x; i < BM * BK; i += kThreads) {
      const int m = i / BK, k = i % BK;
      const int64_t r = s_row[m];
      sx[k][m] = r >= 0 && k0 + k < a.K ? to_f<T>(x[r * a.K + k0 + k]) : 0.f;
    }
#pragma unroll
    for (int b = 0; b < NB; b++)
      for (int i = threadIdx.x; i < BK * BN; i += kThreads) {
        const int k = i / BN, n = i % BN;
        sw[b][k][n] = k0 + k < a.K && n0 + n < a.n_out ? to_f<T>(w[(k0 + k) * a.N + b * a.n_out + n0 + n]) : 0.f;
      }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < BK; k++) {
      float xv[TM];
#pragma unroll
      for (int i = 0; i < TM; i++) xv[i] = sx[k][ty * TM + i];
#pragma unroll
      for (int b = 0; b < NB; b++)
#pragma unroll
        for (int j = 0; j < TN; j++) {
          const float wv = sw[b][k][tx * TN + j];
#pragma unroll
          for (int i = 0; i < TM; i++) acc[b][i][j] = fmaf(xv[i], wv, acc[b][i][j]);
        }
    }
    __syncthreads();
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
        const float u = acc[1][i][j] + (bias ? to_f<T>(bias[a.n_out + n]) : 0.f);
        v = sizeof(T) == 4 ? swiglu_exact(v, u) : __fdividef(v, 1.0f + __expf(-v)) * u;
      } else {
        v = act1<T, ACT>(v);
      }
      out[s * a.n_out + n] = from_f<T>(v);
    }
  }
}

template <typename T>
int32_t launch(Ctx* c, const GroupedArgs& a) {
  const int64_t nt = (a.n_out + BN - 1) / BN;
  const int64_t mt = (a.pairs + BM - 1) / BM + std::min<int64_t>(a.experts, a.pairs);  // at most this many m-tiles
  FL_CHECK(c, nt * mt <= INT32_MAX, "Linear_Grouped: %lldx%lld is too large for the fp32 units", (long long)a.pairs,
           (long long)a.n_out);
  const dim3 grid((unsigned)(nt * mt));
#define FL_ACT(A)                                                                                      \
  case A:                                                                                              \
    FL_CUDA(c, launch_pdl(k_grouped_simt<T, A>, grid, dim3(kThreads), 0, c->stream, a));               \
    break
  switch (a.act) {
    FL_ACT(FLETCHER_ACT_IDENTITY);
    FL_ACT(FLETCHER_ACT_GELU);
    FL_ACT(FLETCHER_ACT_TANH);
    FL_ACT(FLETCHER_ACT_SWIGLU);
    default:
      return set_error(c, FLETCHER_ERR_INVALID, "Linear_Grouped: unknown activation %d", a.act);
  }
#undef FL_ACT
  FL_LAUNCH(c);
  return FLETCHER_OK;
}

}  // namespace

int32_t launch_grouped_simt(Ctx* c, int32_t dtype, const GroupedArgs& a) {
  if (dtype == FLETCHER_BF16) return launch<__nv_bfloat16>(c, a);
  if (dtype == FLETCHER_F16) return launch<__half>(c, a);
  return launch<float>(c, a);
}

}  // namespace fl
