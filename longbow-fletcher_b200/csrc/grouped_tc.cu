// Grouped products on tcgen05 / TMEM / TMA, bf16 and fp16: for every slot s of expert e,
// out[s] = act(x[row(s)] . W[e] + b[e]), W [E][K, N] as the framework stores Linear weights,
// (in, out).
//
// Layout: rows of x are K-major operands, TMA tiles in 128-byte-swizzled 64-wide slabs, in slot order:
// rows of tokens are first copied there (k_place_rows), once, instead of being gathered again for
// each column tile.  Gathering in the product itself was measured on 32768 tokens x 2 of 8 experts,
// 768 -> 2 x 2048: 445 TFLOP/s with TMA gathers of four rows (80 cycles each), 760 with cp.async by
// four warps (1450 cycles a 16 KB slab, whatever the rows' order), against 1250 from rows that lie
// together.  W is
// read as it is stored: its rows are K, its columns contiguous, so boxes of 64 K x 64 columns are
// MN-major operands (64 columns = one 128-byte swizzle row, 8-row K groups 1024 bytes apart, column
// blocks 8 KB apart).  No weight is packed or copied, and SwiGLU's gate and up columns are simply
// fetched from the two halves of a row into one tile.  Rows of K past the end read as zero on both
// sides (x by its width, W by its own dimension, so one expert's rows never meet the next one's).
//
// The number of rows of each group is known on the device only.  Every CTA reads the offsets,
// computes how many row tiles each group has, and walks the same list of (row tile, column tile)
// pairs with a stride; tiles never span groups, so the last tile of a group computes rows it does
// not store.
#include <cuda.h>

#include <algorithm>
#include <atomic>

#include "routing.cuh"
#include "tc_common.cuh"

namespace fl {

int32_t make_tma_map_2d(Ctx* c, CUtensorMap* m, int32_t dtype, const void* ptr, uint64_t rows, uint64_t cols,
                        uint64_t ld, uint32_t box_cols, uint32_t box_rows);
int32_t make_tma_map_3d(Ctx* c, CUtensorMap* m, int32_t dtype, const void* ptr, uint64_t planes, uint64_t rows,
                        uint64_t cols, uint32_t box_cols, uint32_t box_rows);

namespace tcg {

using namespace tc;

constexpr int BM = 128, BK = 64;
constexpr int kEpiWarps = 8;
constexpr int kThreads = 64 + 32 * kEpiWarps;
constexpr int kBox = 32 * 128;  // an epilogue warp's output box: 32 rows x 64 columns x 2 bytes
constexpr int kColBlock = 64 * BK * 2;  // 64 columns of W x 64 rows of K

// BN: accumulator columns of a tile.  PAIR: the tile is 256 rows, computed by two CTAs (two SMs) with
// cta_group::2; each loads its 128 rows of x and half of the columns of W.
template <int BN, bool PAIR>
struct Cfg {
  static constexpr int TILE_M = PAIR ? 2 * BM : BM;
  static constexpr int B_COLS = PAIR ? BN / 2 : BN;  // columns of W loaded by one CTA
  static constexpr int A_BYTES = BM * BK * 2;
  static constexpr int B_BYTES = B_COLS * BK * 2;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int OUT_BYTES = kEpiWarps * kBox;
  static constexpr int TABLE_BYTES = (kMaxExperts + 1 + 32) * 4;
  static constexpr int TAIL_BYTES = 384 + TABLE_BYTES;  // barriers, then the groups' table
  static constexpr int STAGES_FIT = (232448 - 1024 - TAIL_BYTES - OUT_BYTES) / STAGE_BYTES;
  static constexpr int STAGES = STAGES_FIT < 8 ? STAGES_FIT : 8;
  static constexpr int OUT_OFF = STAGES * STAGE_BYTES;
  static constexpr int BAR_OFF = OUT_OFF + OUT_BYTES;
  static constexpr int TABLE_OFF = BAR_OFF + 384;
  static constexpr int TMEM_COLS = 2 * BN;
  static constexpr int SMEM = BAR_OFF + TAIL_BYTES + 1024 /*alignment slack*/;
  static_assert((2 * STAGES + 8) * 8 <= 384, "barrier area");
  static_assert(SMEM <= 232448, "shared memory budget");
};

struct Args {
  const int32_t* offsets;
  const int32_t* pair_of;  // k_grouped_small: slot s reads row pair_of[s] / top_k
  const void* bias;
  void* out;
  int32_t* err;
  int64_t N, n_out;
  int32_t E, top_k, num_kb, n_tiles, act;
  int32_t out32;  // fp32 result
  int32_t pairs, last_row;  // bounds of the slots and of x's rows (GroupedArgs)
};

template <bool PAIR>
__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z) {
  if constexpr (PAIR)
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], "
        "[%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(dst)),
        "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
            smem_u32(dst)),
        "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z)
        : "memory");
}

// MN-major operand of several 64-column blocks: 128-byte swizzle, K groups of 8 rows 1024 bytes
// apart (SBO), column blocks kColBlock apart (LBO).
__device__ __forceinline__ uint64_t desc_mn(uint32_t saddr) {
  uint64_t d = 0;
  d |= (uint64_t)((saddr & 0x3FFFF) >> 4);
  d |= (uint64_t)(kColBlock >> 4) << 16;
  d |= (uint64_t)(1024 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}

// Copies the offsets to shared memory, none past `pairs`, and counts the groups' row tiles; by the whole block.
__device__ __forceinline__ int fill_table(const int32_t* offsets, int E, int32_t pairs, int tile_m, int32_t* offs,
                                          int32_t* tmp) {
  const int t = threadIdx.x, warp = t >> 5, warps = blockDim.x >> 5;
  int n = 0;
  for (int e = t; e <= E; e += blockDim.x) {
    const int o = min(offsets[e], pairs);
    offs[e] = o;
    if (e < E) n += (min(offsets[e + 1], pairs) - o + tile_m - 1) / tile_m;
  }
  n = __reduce_add_sync(0xffffffffu, n);
  if ((t & 31) == 0) tmp[warp] = n;
  __syncthreads();
  n = 0;
  for (int w = 0; w < warps; w++) n += tmp[w];
  return n;
}

struct Tile {
  int e, first, end, nb;  // expert, first slot, end of its group, column tile
};
// Tiles are asked for in ascending order.
struct Walk {
  const int32_t* offs;
  int n_tiles, tile_m, e = 0, before = 0;  // row tiles of the experts before e
  __device__ __forceinline__ Tile at(int tile) {
    const int mt = tile / n_tiles;
    for (;; e++) {
      const int first = offs[e], end = offs[e + 1], n = (end - first + tile_m - 1) / tile_m;
      if (mt < before + n) return {e, first + (mt - before) * tile_m, end, tile - mt * n_tiles};
      before += n;
    }
  }
};

template <typename T>
__device__ __forceinline__ void add_bias32(float (&v)[32], const T* b, int64_t col, int64_t cols) {
#pragma unroll
  for (int i = 0; i < 32; i += 8) {
    if (col + i < cols) {
      union {
        uint4 q;
        T t[8];
      } u;
      u.q = __ldg(reinterpret_cast<const uint4*>(b + col + i));
#pragma unroll
      for (int j = 0; j < 8; j++) v[i + j] += to_f<T>(u.t[j]);
    }
  }
}

// gelu_fast16 on two values in packed fp32, for fp32 results too: its division is off by two places, which
// leaves 0.5 x (1 + t) within two half places of |x| of what a rounded division gives.
__device__ __forceinline__ void gelu_pair(float& x0, float& x1) {
  float a0, a1, u0, u1, q0, q1, n0, n1, d0, d1;
  mul2(q0, q1, x0, x1, x0, x1);
  mul2(a0, a1, x0, x1, 0.044715f, 0.044715f);
  fma2(u0, u1, a0, a1, q0, q1, x0, x1);
  mul2(u0, u1, u0, u1, 0.7978846f, 0.7978846f);
  mul2(q0, q1, u0, u1, u0, u1);
  fma2(n0, n1, q0, q1, u0, u1, 27.0f * u0, 27.0f * u1);
  fma2(d0, d1, q0, q1, 9.0f, 9.0f, 27.0f, 27.0f);
  const float p0 = __fdividef(n0, d0), p1 = __fdividef(n1, d1);
  const float t0 = fabsf(u0) > 4.0f ? copysignf(1.0f, u0) : p0, t1 = fabsf(u1) > 4.0f ? copysignf(1.0f, u1) : p1;
  mul2(x0, x1, x0, x1, 0.5f, 0.5f);
  fma2(x0, x1, x0, x1, t0, t1, x0, x1);
}

// A lane's 32 gates and ups; F32: for an fp32 result.  (Chosen at run time, the form that is not taken cost the
// large product 1.5%: 292 against 287.5 us at 32768 x 2 rows of 8 experts, 768 -> 2 x 2048.)
template <bool F32>
__device__ __forceinline__ void swiglu32(const float (&g)[32], const float (&u)[32], float* v) {
#pragma unroll
  for (int i = 0; i < 32; i++) v[i] = F32 ? swiglu_f32(g[i], u[i]) : swiglu_16(g[i], u[i]);
}

__device__ __forceinline__ void prefetch_l1(const void* p) { asm volatile("prefetch.global.L1 [%0];" ::"l"(p)); }

template <typename T>
__device__ __forceinline__ uint4 pack8(const float* v) {
  return make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
}

// A lane's N values of a row, columns col.. of n_out, from registers.
template <typename T, int N>
__device__ __forceinline__ void store_row(const Args& args, const float* v, int64_t row, int64_t col) {
  if (args.out32) {
    float* dst = reinterpret_cast<float*>(args.out) + row * args.n_out + col;
#pragma unroll
    for (int j = 0; j < N; j += 8) {
      if (col + j < args.n_out)  // whole 32-byte sectors
        asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst + j), "f"(v[j]), "f"(v[j + 1]),
                     "f"(v[j + 2]), "f"(v[j + 3]), "f"(v[j + 4]), "f"(v[j + 5]), "f"(v[j + 6]), "f"(v[j + 7])
                     : "memory");
    }
  } else {
    T* dst = reinterpret_cast<T*>(args.out) + row * args.n_out + col;
#pragma unroll
    for (int j = 0; j < N; j += 8)
      if (col + j < args.n_out) *reinterpret_cast<uint4*>(dst + j) = pack8<T>(v + j);
  }
}

// Persistent: warp 0 loads by TMA, warp 1 issues the MMAs and owns the TMEM, warps 2-9 drain one
// accumulator while the next tile fills the other.  As the dense GEMM: bounded waits, and
// on expiry every role leaves after what it issued has landed.
template <typename T, int BN, bool PAIR, bool GATED, bool F32>
__global__ void __launch_bounds__(kThreads, 1)
    k_grouped_tc(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                 const __grid_constant__ CUtensorMap tmC, const Args args) {
  using C = Cfg<BN, PAIR>;
  constexpr int OUT_N = GATED ? BN / 2 : BN;  // output columns of a tile
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + (((raw + 1023u) & ~1023u) - raw);
  uint8_t* sA = smem;
  uint8_t* sB = smem + C::STAGES * C::A_BYTES;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::BAR_OFF);
  uint64_t* empty = full + C::STAGES;
  uint64_t* tfull = empty + C::STAGES;
  uint64_t* tempty = tfull + 2;
  uint64_t* drain = tempty + 2;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort = reinterpret_cast<volatile int*>(tmem_holder + 1);
  int32_t* offs = reinterpret_cast<int32_t*>(smem + C::TABLE_OFF);
  int32_t* tmp = offs + kMaxExperts + 1;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t crank = PAIR ? cluster_ctarank() : 0;
  const int first_tile = PAIR ? (int)(blockIdx.x >> 1) : (int)blockIdx.x;
  const int tile_stride = PAIR ? (int)(gridDim.x >> 1) : (int)gridDim.x;

  if (threadIdx.x == 0) {
    for (int i = 0; i < C::STAGES; i++) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; i++) {
      mbar_init(&tfull[i], 1);
      mbar_init(&tempty[i], kEpiWarps * (PAIR ? 2 : 1));
    }
    mbar_init(drain, 1);
    *abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&tmA) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&tmB) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&tmC) : "memory");
  }
  if (warp == 1) {
    if constexpr (PAIR) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_holder)),
                   "r"(C::TMEM_COLS)
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_holder)),
                   "r"(C::TMEM_COLS)
                   : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
  }
  pdl_wait();  // the routing and x are the previous kernels' work
  const int num_tiles = fill_table(args.offsets, args.E, args.pairs, C::TILE_M, offs, tmp) * args.n_tiles;
  tc_fence_before();
  if constexpr (PAIR)
    cluster_sync();  // both CTAs' barriers are initialised before any cross-CTA signal
  else
    __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;
  Walk walk{offs, args.n_tiles, C::TILE_M};

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0, issued = 0, issued_par = 0;
      // In a pair both CTAs' loads complete on the even CTA's barrier, which expects both.
      constexpr uint32_t kBytes = (PAIR ? 2 : 1) * C::STAGE_BYTES;
      bool ok = true;
      for (int tile = first_tile; tile < num_tiles && ok; tile += tile_stride) {
        const Tile t = walk.at(tile);
        for (int kb = 0; kb < args.num_kb; kb++) {
          if (!(ok = mbar_wait_spin(&empty[stage], phase ^ 1, abort, args.err))) break;
          uint8_t* a = sA + stage * C::A_BYTES;
          uint8_t* b = sB + stage * C::B_BYTES;
          const uint32_t fb = PAIR ? mapa_shared(smem_u32(&full[stage]), 0) : smem_u32(&full[stage]);
          if (crank == 0) mbar_expect_tx(&full[stage], kBytes);
          if constexpr (PAIR)
            tma_load_2d_pair(a, &tmA, fb, kb * BK, t.first + (int)crank * BM);
          else
            tma_load_2d(a, &tmA, &full[stage], kb * BK, t.first);
#pragma unroll
          for (int i = 0; i < C::B_COLS / 64; i++) {
            const int col = i * 64 + (int)crank * C::B_COLS;  // accumulator column
            const int x = GATED ? t.nb * OUT_N + col % OUT_N + (col >= OUT_N ? (int)args.n_out : 0) : t.nb * BN + col;
            tma_load_3d<PAIR>(b + i * kColBlock, &tmB, fb, x, kb * BK, t.e);
          }
          issued |= 1u << stage;
          issued_par = (issued_par & ~(1u << stage)) | (phase << stage);
          if (++stage == C::STAGES) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
      // Leaving early: the loads in flight land before the CTA exits (in a pair they complete on the even
      // CTA's barriers; the odd CTA cannot pass the last cluster barrier before that one has seen them).
      if (*abort && crank == 0)
        for (int s = 0; s < C::STAGES; s++)
          if ((issued >> s) & 1) mbar_drain(&full[s], (issued_par >> s) & 1);
    }
  } else if (warp == 1) {
    if (lane == 0 && crank == 0) {
      const uint32_t id = idesc<T, C::TILE_M, BN, true>();
      int stage = 0, it = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = first_tile; tile < num_tiles && ok; tile += tile_stride, ++it) {
        const int acc = it & 1;
        if (!mbar_wait_spin(&tempty[acc], ((it >> 1) & 1) ^ 1, abort, args.err)) break;
        tc_fence_after();
        const uint32_t d = tmem_base + acc * BN;
        for (int kb = 0; kb < args.num_kb; kb++) {
          if (!(ok = mbar_wait_spin(&full[stage], phase, abort, args.err))) break;
          tc_fence_after();
          const uint64_t da = sw128_desc(smem_u32(sA + stage * C::A_BYTES));
          const uint64_t db = desc_mn(smem_u32(sB + stage * C::B_BYTES));
#pragma unroll
          for (int k = 0; k < BK / 16; k++) {  // K += 16: 32 bytes along x's rows, 16 rows (2 KB) down W's blocks
            if constexpr (PAIR)
              mma_f16_pair(d, da + 2 * k, db + (uint64_t)k * (2048 >> 4), id, (kb | k) != 0);
            else
              mma_f16(d, da + 2 * k, db + (uint64_t)k * (2048 >> 4), id, (kb | k) != 0);
          }
          if constexpr (PAIR)
            mma_commit_pair(&empty[stage]);
          else
            mma_commit(&empty[stage]);
          if (++stage == C::STAGES) {
            stage = 0;
            phase ^= 1;
          }
        }
        if (!ok) break;
        if constexpr (PAIR)
          mma_commit_pair(&tfull[acc]);
        else
          mma_commit(&tfull[acc]);
      }
      if (*abort) {  // the MMAs issued so far complete before TMEM is freed
        if constexpr (PAIR)
          mma_commit_pair(drain);
        else
          mma_commit(drain);
        mbar_drain(drain, 0);
      }
    }
  } else {
    // Epilogue: warps 2-5 take the first half of a tile's output columns, warps 6-9 the second; warp w
    // reads TMEM lanes 32 * (w % 4) .., its lanes' rows.
    const int q = warp & 3, half = (warp - 2) >> 2;
    constexpr int UW = OUT_N >= 128 ? 64 : 32, UNITS = OUT_N / 2 / UW;  // a warp's units of UW columns
    uint8_t* box = smem + C::OUT_OFF + (warp - 2) * kBox;
    const uint32_t tempty_lead = PAIR ? mapa_shared(smem_u32(tempty), 0) : 0;
    int it = 0;
    for (int tile = first_tile; tile < num_tiles; tile += tile_stride, ++it) {
      const Tile t = walk.at(tile);
      const int acc = it & 1;
      const int row0 = t.first + (int)crank * BM + q * 32;
      const uint32_t tbase = tmem_base + ((uint32_t)(q * 32) << 16) + acc * BN;
      const T* bias = args.bias ? reinterpret_cast<const T*>(args.bias) + (int64_t)t.e * args.N : nullptr;
      if (bias && lane < 2 * UNITS) {  // a 128-byte line a unit, and one of the up columns
        const int64_t col = (int64_t)t.nb * OUT_N + half * (OUT_N / 2) + (lane >> 1) * UW;
        if (col < args.n_out && (GATED || (lane & 1) == 0)) prefetch_l1(bias + col + (lane & 1) * args.n_out);
      }
      if (!mbar_wait_spin(&tfull[acc], (it >> 1) & 1, abort, args.err)) break;
      tc_fence_after();
#pragma unroll 1
      for (int u = 0; u < UNITS; u++) {
        const int c0 = half * (OUT_N / 2) + u * UW;  // first output column of the unit within the tile
        const int64_t ocol = (int64_t)t.nb * OUT_N + c0;
        float v[64];
        float (&lo)[32] = *reinterpret_cast<float(*)[32]>(&v[0]);
        float (&hi)[32] = *reinterpret_cast<float(*)[32]>(&v[32]);
        auto release = [&]() {  // every TMEM read of this tile is done
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            if constexpr (PAIR)
              mbar_arrive_cluster(tempty_lead + acc * 8);
            else
              mbar_arrive(&tempty[acc]);
          }
        };
        if constexpr (GATED) {
#pragma unroll
          for (int s = 0; s < UW / 32; s++) {
            float g[32], w[32];
            tmem_ld32x2(tbase + c0 + s * 32, tbase + OUT_N + c0 + s * 32, g, w);
            if (u == UNITS - 1 && s == UW / 32 - 1) release();
            if (bias) {
              add_bias32<T>(g, bias, ocol + s * 32, args.n_out);
              add_bias32<T>(w, bias + args.n_out, ocol + s * 32, args.n_out);
            }
            swiglu32<F32>(g, w, &v[s * 32]);
          }
        } else {
          tmem_ld32x2(tbase + c0, lo, hi);
          if (u == UNITS - 1) release();
          if (bias) {
            add_bias32<T>(lo, bias, ocol, args.n_out);
            add_bias32<T>(hi, bias, ocol + 32, args.n_out);
          }
          if (args.act == FLETCHER_ACT_GELU) {
#pragma unroll
            for (int i = 0; i < 64; i += 2) gelu_pair(v[i], v[i + 1]);
          }
        }
        if (ocol >= args.n_out || row0 >= t.end) continue;
        if (UW == 64 && row0 + 32 <= t.end && !args.out32) {
          // 32 whole rows: staged in the swizzled box and stored by TMA, columns past the end clipped.
          if (lane == 0) bulk_wait_read0();  // the box's last store has left it
          __syncwarp();
#pragma unroll
          for (int j = 0; j < 8; j++)
            *reinterpret_cast<uint4*>(box + lane * 128 + ((j ^ (lane & 7)) << 4)) = pack8<T>(v + 8 * j);
          fence_async_smem();
          __syncwarp();
          if (lane == 0) {
            tma_store_2d(&tmC, box, (int)ocol, row0);
            bulk_commit();
          }
        } else if (row0 + lane < t.end) {  // the group's last rows (the next are another group's), or fp32
          store_row<T, UW>(args, v, row0 + lane, ocol);
        }
      }
    }
    if (lane == 0) bulk_wait0();
  }

  tc_fence_before();
  if constexpr (PAIR)
    cluster_sync();  // no cross-CTA signal or MMA is in flight past this point
  else
    __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    if constexpr (PAIR)
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(C::TMEM_COLS)
                   : "memory");
    else
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(C::TMEM_COLS)
                   : "memory");
  }
}

// ---------------------------------------------------------------- few rows a group
// Few rows a group: the weights' bytes are the work, so a tile takes at most 32 rows of x (4 KB a slab next
// to 16 KB of W; the MMA's other 96 rows read whatever lies behind and are never looked at), rows of
// tokens are gathered by TMA in quads, only as many as there are, and the rest of shared memory is a
// deep ring of W.  Warps 0 and 4 drain lanes 0-31 of the accumulator, half the columns each.  Where the
// tiles are too few for the SMs (a row or two), the slabs of a tile are split between the CTAs of a
// cluster (SPLIT), which add their sums through distributed shared memory.
struct SmallCfg {
  static constexpr int TILE_M = 32, BN = 128;
  static constexpr int kThreads = 160;
  static constexpr int A_BYTES = TILE_M * BK * 2;
  static constexpr int B_BYTES = BN * BK * 2;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int STAGES = 11;
  static constexpr int BAR_OFF = STAGES * STAGE_BYTES;
  static constexpr int TABLE_OFF = BAR_OFF + 384;
  static constexpr int TMEM_COLS = 2 * BN;
  static constexpr int SMEM = TABLE_OFF + (kMaxExperts + 1 + 32) * 4 + 1024;
  static_assert((2 * STAGES + 8) * 8 <= 384, "barrier area");
  static_assert(SMEM <= 232448, "shared memory budget");
  static_assert(STAGES * B_BYTES >= BM * BK * 2, "the MMA reads 128 rows from the last slab of x on");
};

__device__ __forceinline__ uint32_t cluster_ctas() {
  uint32_t n;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(n));
  return n;
}

// Four rows of a 2-D tensor by index, 64 columns from x, one below the other.
__device__ __forceinline__ void tma_gather4(void* dst, const CUtensorMap* map, uint64_t* bar, int x, const int (&r)[4]) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes [%0], "
      "[%1, {%3, %4, %5, %6, %7}], [%2];" ::"r"(smem_u32(dst)),
      "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3])
      : "memory");
}

template <typename T, bool GATED, bool GATHER, bool SPLIT, bool F32>
__global__ void __launch_bounds__(SmallCfg::kThreads, 1)
    k_grouped_small(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const Args args) {
  using C = SmallCfg;
  constexpr int BN = C::BN, OUT_N = GATED ? BN / 2 : BN;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + (((raw + 1023u) & ~1023u) - raw);
  uint8_t* sA = smem;
  uint8_t* sB = smem + C::STAGES * C::A_BYTES;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::BAR_OFF);
  uint64_t* empty = full + C::STAGES;
  uint64_t* tfull = empty + C::STAGES;
  uint64_t* tempty = tfull + 2;
  uint64_t* drain = tempty + 2;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort = reinterpret_cast<volatile int*>(tmem_holder + 1);
  int32_t* offs = reinterpret_cast<int32_t*>(smem + C::TABLE_OFF);
  int32_t* tmp = offs + kMaxExperts + 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 32) {
    for (int i = 0; i < C::STAGES; i++) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; i++) {
      mbar_init(&tfull[i], 1);
      mbar_init(&tempty[i], 2);
    }
    mbar_init(drain, 1);
    *abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&tmA) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&tmB) : "memory");
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_holder)),
                 "r"(C::TMEM_COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  pdl_wait();  // the routing and x are the previous kernels' work
  const int num_tiles = fill_table(args.offsets, args.E, args.pairs, C::TILE_M, offs, tmp) * args.n_tiles;
  // SPLIT: this CTA's tile (its cluster's) and range of K slabs; else all tiles with a stride, all slabs.
  const int ranks = SPLIT ? (int)cluster_ctas() : 1, rank = SPLIT ? (int)cluster_ctarank() : 0;
  const int first_tile = SPLIT ? (int)blockIdx.x / ranks : (int)blockIdx.x;
  const int tile_stride = SPLIT ? num_tiles : (int)gridDim.x;
  const int kb0 = SPLIT ? args.num_kb * rank / ranks : 0, kb1 = SPLIT ? args.num_kb * (rank + 1) / ranks : args.num_kb;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;
  Walk walk{offs, args.n_tiles, C::TILE_M};

  if (warp == 1) {
    int stage = 0;
    uint32_t phase = 0, issued = 0, issued_par = 0;
    bool ok = true;
    for (int tile = first_tile; tile < num_tiles && ok; tile += tile_stride) {
      const Tile t = walk.at(tile);
      const int quads = GATHER ? (min(t.end - t.first, C::TILE_M) + 3) / 4 : 0;
      int rows[4] = {};
      if (GATHER && lane < quads) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const int s = t.first + 4 * lane + i;
          // past the group: computed, not stored
          rows[i] = min(args.pair_of[s < t.end ? s : t.first] / args.top_k, args.last_row);
        }
      }
      for (int kb = kb0; kb < kb1; kb++) {
        ok = __all_sync(0xffffffffu, mbar_wait_spin(&empty[stage], phase ^ 1, abort, args.err));
        if (!ok) break;
        uint8_t* a = sA + stage * C::A_BYTES;
        uint8_t* b = sB + stage * C::B_BYTES;
        if (lane == 0) {
          mbar_expect_tx(&full[stage], C::B_BYTES + (GATHER ? quads * 512 : C::A_BYTES));
#pragma unroll
          for (int i = 0; i < BN / 64; i++) {
            const int x = GATED ? t.nb * OUT_N + i * (int)args.n_out : t.nb * BN + i * 64;
            tma_load_3d<false>(b + i * kColBlock, &tmB, smem_u32(&full[stage]), x, kb * BK, t.e);
          }
          if constexpr (!GATHER) tma_load_2d(a, &tmA, &full[stage], kb * BK, t.first);
        }
        if (GATHER && lane < quads) tma_gather4(a + lane * 512, &tmA, &full[stage], kb * BK, rows);
        issued |= 1u << stage;
        issued_par = (issued_par & ~(1u << stage)) | (phase << stage);
        if (++stage == C::STAGES) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
    if (lane == 0 && *abort)  // leaving early: the loads in flight land before the CTA exits
      for (int s = 0; s < C::STAGES; s++)
        if ((issued >> s) & 1) mbar_drain(&full[s], (issued_par >> s) & 1);
  } else if (warp == 2) {
    if (lane == 0) {
      const uint32_t id = idesc<T, BM, BN, true>();
      int stage = 0, it = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = first_tile; tile < num_tiles && ok; tile += tile_stride, ++it) {
        const int acc = it & 1;
        if (!mbar_wait_spin(&tempty[acc], ((it >> 1) & 1) ^ 1, abort, args.err)) break;
        tc_fence_after();
        const uint32_t d = tmem_base + acc * BN;
        for (int kb = kb0; kb < kb1; kb++) {
          if (!(ok = mbar_wait_spin(&full[stage], phase, abort, args.err))) break;
          tc_fence_after();
          const uint64_t da = sw128_desc(smem_u32(sA + stage * C::A_BYTES));
          const uint64_t db = desc_mn(smem_u32(sB + stage * C::B_BYTES));
#pragma unroll
          for (int k = 0; k < BK / 16; k++)
            mma_f16(d, da + 2 * k, db + (uint64_t)k * (2048 >> 4), id, kb > kb0 || k > 0);
          mma_commit(&empty[stage]);
          if (++stage == C::STAGES) {
            stage = 0;
            phase ^= 1;
          }
        }
        if (!ok) break;
        mma_commit(&tfull[acc]);
      }
      if (*abort) {
        mma_commit(drain);
        mbar_drain(drain, 0);
      }
    }
  }
  // Warps 0 and 4: bias, activation and rows of a tile's half, from v (gated: 32 gates, 32 ups).
  constexpr int COLS = OUT_N / 2;  // this warp's output columns: 32 (gated) or 64
  const int half = warp >> 2, c0 = half * COLS;
  auto finish = [&](const Tile& t, float (&v)[64]) {
    float (&lo)[32] = *reinterpret_cast<float(*)[32]>(&v[0]);
    float (&hi)[32] = *reinterpret_cast<float(*)[32]>(&v[32]);
    const int64_t ocol = (int64_t)t.nb * OUT_N + c0;
    if (args.bias) {
      const T* bias = reinterpret_cast<const T*>(args.bias) + (int64_t)t.e * args.N;
      add_bias32<T>(lo, bias, ocol, args.n_out);
      if constexpr (GATED)
        add_bias32<T>(hi, bias + args.n_out, ocol, args.n_out);
      else
        add_bias32<T>(hi, bias, ocol + 32, args.n_out);
    }
    if constexpr (GATED) {
      swiglu32<F32>(lo, hi, v);
    } else if (args.act == FLETCHER_ACT_GELU) {
#pragma unroll
      for (int i = 0; i < 64; i += 2) gelu_pair(v[i], v[i + 1]);
    }
    if (t.first + lane < t.end) store_row<T, COLS>(args, v, t.first + lane, ocol);
  };
  if (!SPLIT && (warp == 0 || warp == 4)) {
    int it = 0;
    for (int tile = first_tile; tile < num_tiles; tile += tile_stride, ++it) {
      const Tile t = walk.at(tile);
      const int acc = it & 1;
      const uint32_t tbase = tmem_base + acc * BN;
      if (!mbar_wait_spin(&tfull[acc], (it >> 1) & 1, abort, args.err)) break;
      tc_fence_after();
      float v[64];
      float (&lo)[32] = *reinterpret_cast<float(*)[32]>(&v[0]);
      float (&hi)[32] = *reinterpret_cast<float(*)[32]>(&v[32]);
      tmem_ld32x2(tbase + c0, tbase + c0 + (GATED ? OUT_N : 32), lo, hi);  // gated: gate and up
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&tempty[acc]);
      finish(t, v);
    }
  }
  if constexpr (SPLIT) {
    // The other ranks leave their sums in shared memory, over the ring, which is done with; rank 0 adds them in
    // their order.  Every thread takes both cluster barriers, whatever happened before them.
    constexpr int PITCH = 64 + 4;  // floats of a row of a warp's half
    float* mine = reinterpret_cast<float*>(smem) + (half * C::TILE_M + lane) * PITCH;
    float v[64];
    Tile t{};
    bool have = false;
    __syncwarp();
    if ((warp == 0 || warp == 4) && first_tile < num_tiles) {
      t = walk.at(first_tile);
      have = mbar_wait_spin(&tfull[0], 0, abort, args.err);
      have = __all_sync(0xffffffffu, have);
      if (have) {
        tc_fence_after();
        float (&lo)[32] = *reinterpret_cast<float(*)[32]>(&v[0]);
        float (&hi)[32] = *reinterpret_cast<float(*)[32]>(&v[32]);
        tmem_ld32x2(tmem_base + c0, tmem_base + c0 + (GATED ? OUT_N : 32), lo, hi);
        if (rank > 0 && t.first + lane < t.end) {
#pragma unroll
          for (int i = 0; i < 64; i += 4) *reinterpret_cast<float4*>(mine + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
        }
      }
    }
    cluster_sync();
    if (rank == 0 && have) {
      if (t.first + lane < t.end) {
        for (int r = 1; r < ranks; r++) {
          const uint32_t src = mapa_shared(smem_u32(mine), r);
#pragma unroll
          for (int i = 0; i < 64; i += 4) {
            float4 q;
            asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                         : "=f"(q.x), "=f"(q.y), "=f"(q.z), "=f"(q.w)
                         : "r"(src + i * 4)
                         : "memory");
            v[i] += q.x, v[i + 1] += q.y, v[i + 2] += q.z, v[i + 3] += q.w;
          }
        }
      }
      finish(t, v);
    }
    cluster_sync();  // rank 0 has read the others' sums
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 2) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(C::TMEM_COLS) : "memory");
  }
}

Args args_of(const Ctx* c, const GroupedArgs& g, int out_n) {
  Args a{};
  a.offsets = g.offsets;
  a.pair_of = g.pair_of;
  a.top_k = g.top_k;
  a.bias = g.bias;
  a.out = g.out;
  a.err = c->d_err;
  a.N = g.N;
  a.n_out = g.n_out;
  a.E = g.experts;
  a.num_kb = (int)((g.K + BK - 1) / BK);
  a.n_tiles = (int)((g.n_out + out_n - 1) / out_n);
  a.act = g.act;
  a.out32 = g.out32;
  a.pairs = (int32_t)g.pairs;
  a.last_row = (int32_t)g.x_rows - 1;
  return a;
}

// At most this many tiles, whatever the groups are.
int64_t most_tiles(const GroupedArgs& g, int tile_m, int n_tiles) {
  return (g.pairs / tile_m + std::min<int64_t>(g.experts, g.pairs)) * n_tiles;
}

template <typename T, bool GATED, bool GATHER, bool SPLIT, bool F32>
int32_t run_small(Ctx* c, int32_t dt, const GroupedArgs& g, int ranks) {
  using C = SmallCfg;
  CUtensorMap ma, mb;
  int32_t rc;
  if ((rc = make_tma_map_2d(c, &ma, dt, g.x, (uint64_t)g.x_rows, (uint64_t)g.K, (uint64_t)g.K, BK,
                            GATHER ? 1 : C::TILE_M)))
    return rc;
  if ((rc = make_tma_map_3d(c, &mb, dt, g.w, (uint64_t)g.experts, (uint64_t)g.K, (uint64_t)g.N, 64, BK))) return rc;
  const Args a = args_of(c, g, GATED ? C::BN / 2 : C::BN);
  auto kern = k_grouped_small<T, GATED, GATHER, SPLIT, F32>;
  static std::atomic<bool> attr_set[64] = {};  // per device; idempotent, replicas' threads may meet here
  if (!attr_set[c->device & 63].load(std::memory_order_acquire)) {
    FL_CUDA(c, cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
    attr_set[c->device & 63].store(true, std::memory_order_release);
  }
  const int64_t tiles = most_tiles(g, C::TILE_M, a.n_tiles);
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = ranks;
  at[1].val.clusterDim.y = 1;
  at[1].val.clusterDim.z = 1;
  cfg.gridDim = dim3((unsigned)(SPLIT ? tiles * ranks : std::min<int64_t>(tiles, c->num_sms)));
  cfg.blockDim = dim3(C::kThreads);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = c->stream;
  cfg.attrs = at;
  cfg.numAttrs = SPLIT ? 2 : 1;
  FL_CUDA(c, cudaLaunchKernelEx(&cfg, kern, ma, mb, a));
  FL_LAUNCH(c);
  return FLETCHER_OK;
}

template <typename T, bool GATED, bool GATHER, bool F32>
int32_t launch_small_g(Ctx* c, int32_t dt, const GroupedArgs& g) {
  // CTAs a tile: as many as the SMs have room for, at most 8, two slabs of K each at least.
  const int out_n = GATED ? SmallCfg::BN / 2 : SmallCfg::BN;
  const int64_t tiles = most_tiles(g, SmallCfg::TILE_M, (int)((g.n_out + out_n - 1) / out_n));
  int ranks = 1;
  while (ranks < 8 && tiles * ranks * 2 <= c->num_sms && g.K >= ranks * 4 * BK) ranks *= 2;
  return ranks > 1 ? run_small<T, GATED, GATHER, true, F32>(c, dt, g, ranks)
                   : run_small<T, GATED, GATHER, false, F32>(c, dt, g, 1);
}

template <typename T, bool GATHER>
int32_t launch_small_a(Ctx* c, int32_t dt, const GroupedArgs& g) {
  if (g.act != FLETCHER_ACT_SWIGLU) return launch_small_g<T, false, GATHER, false>(c, dt, g);
  return g.out32 ? launch_small_g<T, true, GATHER, true>(c, dt, g) : launch_small_g<T, true, GATHER, false>(c, dt, g);
}

template <typename T>
int32_t launch_small(Ctx* c, int32_t dt, const GroupedArgs& g) {
  return g.pair_of ? launch_small_a<T, true>(c, dt, g) : launch_small_a<T, false>(c, dt, g);
}

template <typename T, int BN, bool PAIR, bool GATED, bool F32>
int32_t run(Ctx* c, int32_t dt, const GroupedArgs& g) {
  using C = Cfg<BN, PAIR>;
  constexpr int OUT_N = GATED ? BN / 2 : BN;
  CUtensorMap ma, mb, mc;
  int32_t rc;
  if ((rc = make_tma_map_2d(c, &ma, dt, g.x, (uint64_t)g.x_rows, (uint64_t)g.K, (uint64_t)g.K, BK, BM)))
    return rc;
  if ((rc = make_tma_map_3d(c, &mb, dt, g.w, (uint64_t)g.experts, (uint64_t)g.K, (uint64_t)g.N, 64, BK))) return rc;
  mc = ma;  // not used for an fp32 result
  if (!g.out32 &&
      (rc = make_tma_map_2d(c, &mc, dt, g.out, (uint64_t)g.pairs, (uint64_t)g.n_out, (uint64_t)g.n_out, 64, 32)))
    return rc;
  const Args a = args_of(c, g, OUT_N);
  auto kern = k_grouped_tc<T, BN, PAIR, GATED, F32>;
  static std::atomic<bool> attr_set[64] = {};  // per device; idempotent, replicas' threads may meet here
  if (!attr_set[c->device & 63].load(std::memory_order_acquire)) {
    FL_CUDA(c, cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
    attr_set[c->device & 63].store(true, std::memory_order_release);
  }
  const int64_t tiles = most_tiles(g, C::TILE_M, a.n_tiles);
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = 2;
  at[1].val.clusterDim.y = 1;
  at[1].val.clusterDim.z = 1;
  const int units = PAIR ? c->num_sms / 2 : c->num_sms;
  cfg.gridDim = dim3((unsigned)(std::min<int64_t>(tiles, units) * (PAIR ? 2 : 1)));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = c->stream;
  cfg.attrs = at;
  cfg.numAttrs = PAIR ? 2 : 1;
  FL_CUDA(c, cudaLaunchKernelEx(&cfg, kern, ma, mb, mc, a));
  FL_LAUNCH(c);
  return FLETCHER_OK;
}

template <typename T, int BN, bool PAIR>
int32_t pick(Ctx* c, int32_t dt, const GroupedArgs& g) {
  if (g.act != FLETCHER_ACT_SWIGLU) return run<T, BN, PAIR, false, false>(c, dt, g);
  return g.out32 ? run<T, BN, PAIR, true, true>(c, dt, g) : run<T, BN, PAIR, true, false>(c, dt, g);
}

// Token rows copied to their slots: a warp a token, whose row is read once and written for each of its
// choices.  Bound by HBM at (1 + top_k) * rows * K * 2 bytes.
__global__ void __launch_bounds__(256) k_place_rows(const uint4* __restrict__ x, const int32_t* __restrict__ slots,
                                                    int64_t rows, int top_k, int vecs, int pairs,
                                                    uint4* __restrict__ out) {
  pdl_wait();
  const int lane = threadIdx.x & 31;
  for (int64_t t = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5; t < rows;
       t += ((int64_t)gridDim.x * blockDim.x) >> 5) {
    const uint4* src = x + t * vecs;
    const int slot_of = lane < top_k ? slots[t * top_k + lane] : -1, mine = slot_of < pairs ? slot_of : -1;
    for (int v0 = 0; v0 < vecs; v0 += 128) {
      uint4 q[4];
#pragma unroll
      for (int i = 0; i < 4; i++)
        if (v0 + i * 32 + lane < vecs) q[i] = __ldcs(src + v0 + i * 32 + lane);
      for (int j = 0; j < top_k; j++) {
        const int slot = __shfl_sync(0xffffffffu, mine, j);
        if (slot < 0) continue;
        uint4* dst = out + (int64_t)slot * vecs + v0 + lane;
#pragma unroll
        for (int i = 0; i < 4; i++)
          if (v0 + i * 32 + lane < vecs) dst[i * 32] = q[i];
      }
    }
  }
}

template <typename T>
int32_t launch(Ctx* c, int32_t dt, const GroupedArgs& g) {
  const bool gated = g.act == FLETCHER_ACT_SWIGLU;
  // 256 accumulator columns keep the tensor core fed (with 128 it reads x's rows from shared memory
  // for half the work: 32000 x 6 of 64 experts, 1024 -> 2 x 704, 678 against 552 us); 128 where all
  // tiles run at once either way, so that twice the SMs work (1536 of 12 experts, 776 -> 1000: 11.6
  // against 15.5 us).
  const int64_t groups = std::min<int64_t>(g.experts, g.pairs);
  const int64_t tiles = (2 * g.pairs / BM + groups) * ((g.n_out + (gated ? 63 : 127)) / (gated ? 64 : 128)) / 2;
  if (tiles <= c->num_sms) return pick<T, 128, false>(c, dt, g);
  // Pairs of SMs on 256 x 256 tiles where groups have rows for them on average (12000 x 2 of 8 experts,
  // 768 -> 2 x 2048: 134 against 147 us with 128 x 256; 128 rows an expert, 64 experts: 58 against 49).
  if (g.pairs >= 256 * groups) return pick<T, 256, true>(c, dt, g);
  return pick<T, 256, false>(c, dt, g);
}

}  // namespace tcg

bool grouped_tc_supported(int32_t dtype, const GroupedArgs& g) {
  return dtype != FLETCHER_F32 && g.K % 8 == 0 && g.n_out % 8 == 0 && g.act != FLETCHER_ACT_TANH;
}

// Rows an expert on average, counting no more experts than there are rows, decide between the kernels.
// Measured with weights from HBM, 768 -> 2 x 2048 of 8 and 1024 -> 2 x 704 of 64 experts, us:
//   rows an expert                         4            8            16           32
//   32-row tiles, rows gathered in them    12.8  37.8   13.6  41.6   15.1  45.7   23.9  67.4
//   32-row tiles, rows placed before       14.2  37.2   14.0  37.9   14.0  38.1   17.2  48.1
//   128-row tiles, rows placed before      15.3  39.5   15.2  41.1   14.3  41.6   14.3  42.4
static bool rows_per_expert_at_most(const GroupedArgs& g, int n) {
  return g.pairs <= n * std::min<int64_t>(g.experts, g.pairs);
}
static bool gathers(const GroupedArgs& g) { return g.slots && rows_per_expert_at_most(g, 4); }

int64_t grouped_tc_workspace(const GroupedArgs& g) { return g.slots && !gathers(g) ? g.pairs * g.K * 2 : 0; }

int32_t launch_grouped_tc(Ctx* c, int32_t dtype, const GroupedArgs& args, void* workspace) {
  GroupedArgs g = args;
  const bool small = rows_per_expert_at_most(g, 16);
  if (g.slots && !gathers(g)) {
    const int64_t blocks = std::min<int64_t>((g.x_rows + 7) / 8, (int64_t)c->num_sms * 8);
    FL_CUDA(c, launch_pdl(tcg::k_place_rows, dim3((unsigned)blocks), dim3(256), 0, c->stream, (const uint4*)g.x, g.slots,
                          g.x_rows, g.top_k, (int)(g.K / 8), (int)g.pairs, (uint4*)workspace));
    FL_LAUNCH(c);
    g.x = workspace;
    g.x_rows = g.pairs;
    g.slots = g.pair_of = nullptr;
  }
  if (small)
    return dtype == FLETCHER_BF16 ? tcg::launch_small<__nv_bfloat16>(c, dtype, g) : tcg::launch_small<__half>(c, dtype, g);
  if (dtype == FLETCHER_BF16) return tcg::launch<__nv_bfloat16>(c, dtype, g);
  return tcg::launch<__half>(c, dtype, g);
}

}  // namespace fl
