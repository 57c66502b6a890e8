// Routing of rows to experts: top-k choice, weights, and the order of the choices by expert.
//
// A row belongs to L lanes, which read its logits in chunks of eight.  A candidate is one integer key:
// the logit's bits in an order that compares like the value, above the complement of the expert's
// index, so the largest key is the largest logit and, among equals, the lowest expert (32 bits for
// 16-bit logits, else 64).  Each lane keeps its KM >= top_k largest keys in order (networks sort a chunk
// and merge it in; two choices are kept by insertion); then a round takes the largest of the lanes'
// first keys (log2 L shuffles) and its owner moves on.  Lane j mod L keeps
// choice j and computes its exponential, with the first winner as the maximum; exponentials and quotients
// are expf's and a division's (with the special-function unit's exponential 17.4 us where these take 18.4, and
// weights 30 below the maximum off by up to 14 units of their last place).  65536 x 64 -> 6: 18.4 us, 16.9 where only
// the chosen weights are summed.  Issuing the two kernels' 11.1 M warp instructions takes half of that; the rest is
// latency, of loads and of two dependent launches.  Four lanes a row for many rows (two and eight were within
// 1 us there, at 16384 x 128 -> 8 slower by 5 and 1).
//
// Grouping is a stable counting sort in two launches: k_route leaves, per block of rows and per run of
// kSpan blocks, how many choices each expert got; k_group sums the runs and blocks before its own, ranks
// its pairs within the block, and writes slots and their inverse.  (With the blocks' counts alone every
// block reads the same lines of L2 at once: 9 of 19 us; summed by the last block of k_route: 4 us.)
// Where a cluster of blocks can hold all pairs, its blocks read one another's counts and one launch does
// it all.  Only integers are added in no fixed order, so the slots are the same in every run.
#include <algorithm>
#include <new>
#include <vector>

#include "routing.cuh"

namespace fl {
namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kBlocksPerSM = 2;
constexpr int V = 8;  // logits per lane
constexpr int kSpan = 16;
// Keys of eight logits from expert e0 on, and the logits in fp32.  NaN counts as -inf and -0 as +0;
// a key that is not `valid` (-inf, or the 0 of an empty place) is never chosen.
template <typename T>
struct KeyOf {  // f32
  typedef unsigned long long K;
  static __device__ __forceinline__ void make(const float (&t)[V], int e0, K (&key)[V], float (&x)[V]) {
#pragma unroll
    for (int i = 0; i < V; i++) {
      x[i] = fmaxf(t[i], -INFINITY) + 0.0f;
      const uint32_t b = __float_as_uint(x[i]);
      key[i] = ((K)(b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u)) << 32) | (uint32_t)~(e0 + i);
    }
  }
  static __device__ __forceinline__ bool valid(K k) { return (uint32_t)(k >> 32) > 0x007fffffu; }
  static __device__ __forceinline__ int expert(K k) { return (int)~(uint32_t)k; }
  static __device__ __forceinline__ float value(K k) {
    const uint32_t o = (uint32_t)(k >> 32);
    return __uint_as_float((o & 0x80000000u) ? o & 0x7fffffffu : ~o);
  }
};
template <typename T, typename T2, uint32_t NEG_INF>
struct KeyOf16 {
  typedef uint32_t K;
  // Two logits a word: the maximum with -inf drops NaN, adding +0 turns -0 over, and flipping a negative
  // number's bits, a positive one's sign, orders both halves.
  static __device__ __forceinline__ void make(const T (&t)[V], int e0, K (&key)[V], float (&x)[V]) {
#pragma unroll
    for (int i = 0; i < V; i += 2) {
      const uint32_t inf2 = NEG_INF * 0x10001u, zero2 = 0;
      const T2 v = __hadd2(__hmax2(*reinterpret_cast<const T2*>(&t[i]), *reinterpret_cast<const T2*>(&inf2)),
                           *reinterpret_cast<const T2*>(&zero2));
      uint32_t u = *reinterpret_cast<const uint32_t*>(&v);
      x[i] = to_f<T>(v.x);
      x[i + 1] = to_f<T>(v.y);
      u ^= ((u >> 15) & 0x10001u) * 0xffffu | 0x80008000u;
      key[i] = (u << 16) | (uint32_t)(0xffff - e0 - i);
      key[i + 1] = (u & 0xffff0000u) | (uint32_t)(0xffff - e0 - i - 1);
    }
  }
  static __device__ __forceinline__ bool valid(K k) { return k >> 16 > (NEG_INF ^ 0xffffu); }
  static __device__ __forceinline__ int expert(K k) { return 0xffff - (int)(k & 0xffffu); }
  static __device__ __forceinline__ float value(K k) {
    const uint32_t o = k >> 16;
    const uint16_t b = (uint16_t)((o & 0x8000u) ? o & 0x7fffu : ~o);
    return to_f<T>(*reinterpret_cast<const T*>(&b));
  }
};
template <>
struct KeyOf<__half> : KeyOf16<__half, __half2, 0xfc00u> {};
template <>
struct KeyOf<__nv_bfloat16> : KeyOf16<__nv_bfloat16, __nv_bfloat162, 0xff80u> {};

template <typename K>
__device__ __forceinline__ void exchange(K& a, K& b) {
  const K hi = a > b ? a : b, lo = a > b ? b : a;
  a = hi;
  b = lo;
}
// Eight keys in descending order, by Batcher's odd-even merge sort: 19 exchanges.
template <typename K>
__device__ __forceinline__ void sort8(K (&k)[8]) {
  auto ex = [&](int i, int j) { exchange(k[i], k[j]); };
  ex(0, 1), ex(2, 3), ex(4, 5), ex(6, 7);
  ex(0, 2), ex(1, 3), ex(4, 6), ex(5, 7);
  ex(1, 2), ex(5, 6);
  ex(0, 4), ex(1, 5), ex(2, 6), ex(3, 7);
  ex(2, 4), ex(3, 5);
  ex(1, 2), ex(3, 4), ex(5, 6);
}

struct RouteArgs {
  const void* logits;  // null: `experts` is given
  int64_t rows;
  int32_t E, k;
  int32_t sigmoid, normalise;
  float scale;
  int64_t chunk;  // rows per block
  int32_t* experts;
  float* weights;
  int32_t* slots;
  int32_t* pair_of;
  int32_t* offsets;
  int32_t* hist;    // [blocks, E] choices of each expert in a block's rows
  int32_t* spans;   // [blocks / kSpan, E] the same for runs of blocks; 0 between calls
  int32_t* ticket;  // blocks of k_group that have read them; 0 between calls
};

// exp(x - m) where x may equal an infinite m.
__device__ __forceinline__ float exp_below(float x, float m) { return x == m ? 1.0f : expf(x - m); }

// The choices and weights of rows [r0, r1), into `hist` (shared) each expert's count, and, unless null,
// the choices into `ids` (shared).
template <typename T, int L, int KM>
__device__ __forceinline__ void choose(const RouteArgs& a, int64_t r0, int64_t r1, int32_t* hist, int16_t* ids) {
  typedef KeyOf<T> Key;
  typedef typename Key::K K;
  constexpr int KEEP = (KM + L - 1) / L;  // choices a lane keeps
  constexpr int kPass = kThreads / L;
  const int lane = threadIdx.x & 31, gl = lane & (L - 1);
  const int chunks = (a.E + V * L - 1) / (V * L);
  const T* z = reinterpret_cast<const T*>(a.logits);
  const bool vec = a.E % V == 0;
  struct alignas(16) Chunk {
    T t[V];
  };
  // Whole teams step together; a team past the end works on the last row and writes nothing.  Places past
  // the experts are -inf.
  auto load = [&](int64_t r, int e0, Chunk& u) {
    const T* row = z + (r < r1 ? r : r1 - 1) * a.E + e0;
    if (vec && e0 < a.E) {
#pragma unroll
      for (int i = 0; i < (int)sizeof(Chunk) / 16; i++)
        reinterpret_cast<uint4*>(&u)[i] = __ldg(reinterpret_cast<const uint4*>(row) + i);
    } else {
#pragma unroll
      for (int i = 0; i < V; i++) u.t[i] = e0 + i < a.E ? row[i] : from_f<T>(-INFINITY);
    }
  };
  const bool all = !a.sigmoid && !a.normalise;  // the weights' sum is over the whole row
  Chunk next;
  load(r0 + threadIdx.x / L, gl * V, next);
  for (int64_t base = r0; base < r1; base += kPass) {
    const int64_t mine = base + threadIdx.x / L;
    if (base + (threadIdx.x & ~31) / L >= r1) break;  // none of the warp's rows is left
    K list[KM] = {};
    float ref = 0.f, sum = 0.f, top = -INFINITY;  // sum of exp(x - ref) over the lane's logits, their maximum
    for (int c = 0; c < chunks; c++) {
      const int e0 = (c * L + gl) * V;
      const Chunk cur = next;
      if (c + 1 < chunks)  // on its way while this chunk is sorted
        load(mine, e0 + L * V, next);
      else if (base + kPass < r1)
        load(mine + kPass, gl * V, next);
      K key[V];
      float x[V];
      Key::make(cur.t, e0, key, x);
      if (all) {
#pragma unroll
        for (int i = 0; i < V; i++) top = fmaxf(top, x[i]);
        const float r = fabsf(top) == INFINITY ? 0.f : top;  // +inf is counted below instead
        sum = sum > 0.f ? sum * expf(ref - r) : 0.f;
        ref = r;
        float s1 = 0.f;
#pragma unroll
        for (int i = 0; i < V; i += 2) {
          add2(x[i], x[i + 1], -r, -r);
          add2(sum, s1, expf(x[i]), expf(x[i + 1]));
        }
        sum += s1;
      }
      if constexpr (KM >= V) {
        // The chunk in order; the larger of its i-th last and the list's last eight, pairwise, leave the KM
        // largest in a bitonic sequence, which log2 KM steps put in order.
        sort8(key);
        if (c == 0) {
#pragma unroll
          for (int i = 0; i < V; i++) list[i] = key[i];
        } else {
#pragma unroll
          for (int i = 0; i < V; i++) list[KM - V + i] = key[V - 1 - i] > list[KM - V + i] ? key[V - 1 - i] : list[KM - V + i];
#pragma unroll
          for (int d = KM / 2; d >= 1; d /= 2)
#pragma unroll
            for (int i = 0; i < KM; i++)
              if ((i & d) == 0) exchange(list[i], list[i + d]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < V; i++) {
          K k = key[i];
          if (k > list[KM - 1]) {
#pragma unroll
            for (int j = 0; j < KM; j++) exchange(list[j], k);
          }
        }
      }
    }
    float m = 0.f;
    K kept[KEEP] = {};
    if constexpr (L == 1) {
      m = Key::value(list[0]);
#pragma unroll
      for (int j = 0; j < KM; j++)
        if (j < a.k) kept[j] = list[j];
    } else {
#pragma unroll
      for (int j = 0; j < KM; j++) {
        if (j < a.k) {
          K best = list[0];
#pragma unroll
          for (int o = 1; o < L; o <<= 1) {
            const K other = __shfl_xor_sync(0xffffffffu, best, o);
            best = other > best ? other : best;
          }
          const bool own = list[0] == best;  // keys are unique: one lane (or, at 0, all with nothing left)
#pragma unroll
          for (int i = 0; i < KM; i++) list[i] = own ? (i + 1 < KM ? list[i + 1] : 0) : list[i];
          if (j == 0) m = Key::value(best);
          if ((j & (L - 1)) == gl) kept[j / L] = best;
        }
      }
    }
    float w[KEEP], total = 0.f;
#pragma unroll
    for (int j = 0; j < KEEP; j++) {
      w[j] = 0.f;
      if (Key::valid(kept[j])) {
        const float v = Key::value(kept[j]);
        w[j] = a.sigmoid ? 1.0f / (1.0f + expf(-v)) : exp_below(v, m);
      }
      total += w[j];
    }
    if (all) {
      total = sum > 0.f ? sum * expf(ref - m) : 0.f;
      if (m == INFINITY) {  // the row's +inf share the weight
        total = 0.f;
        for (int e = gl; e < a.E; e += L)
          total += to_f<T>(z[(mine < r1 ? mine : r1 - 1) * a.E + e]) == INFINITY ? 1.f : 0.f;
      }
    }
#pragma unroll
    for (int o = 1; o < L; o <<= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    // Divided by the sum first, so that no product overflows before it; 0 where the sum is 0.
    const float by = a.sigmoid && !a.normalise ? 1.0f : total > 0.f ? total : INFINITY;
    if (mine < r1) {
      const int64_t out = mine * a.k;
#pragma unroll
      for (int i = 0; i < KEEP; i++) {
        const int j = i * L + gl;
        if (j < a.k) {
          const int id = Key::valid(kept[i]) ? Key::expert(kept[i]) : -1;
          a.experts[out + j] = id;
          a.weights[out + j] = w[i] / by * a.scale;
          if (ids) ids[(int)(out - r0 * a.k) + j] = (int16_t)id;
          if (id >= 0) atomicAdd(&hist[id], 1);
        }
      }
    }
  }
}

// Slots of n <= kSub pairs from p0, whose experts are in ids (shared).  start[e] (shared): the first slot
// of expert e, moved on by what is assigned.  count (shared): [kWarps][E].  Each warp ranks a run of pairs
// against its own counters, the counters become the warps' first slots, and the ranks are added.
constexpr int kSub = 4096, kRun = kSub / kWarps / 32;
__device__ __forceinline__ void assign_slots(const RouteArgs& a, int64_t p0, int n, const int16_t* ids, int32_t* start,
                                             int32_t* count) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int per = ((n + kWarps - 1) / kWarps + 31) / 32 * 32, warps = (n + per - 1) / per;
  const int w0 = warp * per;
  int32_t* mine = count + warp * a.E;
  int rank[kRun];
  if (warp < warps) {
    for (int e = lane; e < a.E; e += 32) mine[e] = 0;
    __syncwarp();
#pragma unroll
    for (int i = 0; i < kRun; i++) {
      if (i * 32 < per) {
        const int p = w0 + i * 32 + lane;
        const int e = p < n ? ids[p] : -1;
        // The lanes with the same expert, bit by bit (__match_any_sync: three times the instructions).
        uint32_t same = __ballot_sync(0xffffffffu, e >= 0);
        for (int b = 0; (a.E - 1) >> b; b++) {
          const uint32_t ones = __ballot_sync(0xffffffffu, (e >> b) & 1);
          same &= (e >> b) & 1 ? ones : ~ones;
        }
        rank[i] = -1;
        if (e >= 0) rank[i] = mine[e] + __popc(same & ((1u << lane) - 1));
        __syncwarp();
        if (e >= 0 && lane == 31 - __clz(same)) mine[e] = rank[i] + 1;
        __syncwarp();
      }
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < a.E; e += kThreads) {
    int32_t at = start[e];
    for (int w = 0; w < warps; w++) {
      const int32_t c = count[w * a.E + e];
      count[w * a.E + e] = at;
      at += c;
    }
    start[e] = at;
  }
  __syncthreads();
  if (warp < warps) {
#pragma unroll
    for (int i = 0; i < kRun; i++) {
      if (i * 32 < per) {
        const int p = w0 + i * 32 + lane;
        if (p < n) {
          const int slot = rank[i] < 0 ? -1 : mine[ids[p]] + rank[i];
          a.slots[p0 + p] = slot;
          if (slot >= 0) a.pair_of[slot] = (int32_t)(p0 + p);
        }
      }
    }
  }
}

// Exclusive prefix of n (shared, kMaxExperts, 0 past E) into at[0..E), and the total into at[E]; by the
// block, whose first warp holds eight experts a lane.
__device__ __forceinline__ void scan_experts(const int32_t* n, int32_t* at, int E) {
  static_assert(kMaxExperts == 256, "eight a lane");
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    int4 v[2] = {reinterpret_cast<const int4*>(n)[2 * lane], reinterpret_cast<const int4*>(n)[2 * lane + 1]};
    const int32_t sum = (v[0].x + v[0].y + v[0].z + v[0].w) + (v[1].x + v[1].y + v[1].z + v[1].w);
    int32_t s = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int32_t u = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += u;
    }
    s -= sum;  // at[E] and what follows are the total, as nothing is counted there
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const int4 q = make_int4(s, s + v[i].x, s + v[i].x + v[i].y, s + v[i].x + v[i].y + v[i].z);
      reinterpret_cast<int4*>(at)[2 * lane + i] = q;
      s = q.w + v[i].w;
    }
    if (lane == 31) at[kMaxExperts] = s;
  }
  __syncthreads();
}

// The prefix's first slots become this block's, past `before` (null: none); the first block leaves the offsets.
__device__ __forceinline__ void first_slots(const RouteArgs& a, int32_t* at, const int32_t* before) {
  for (int e = threadIdx.x; e <= a.E; e += kThreads) {
    const int32_t v = at[e];
    if (blockIdx.x == 0) a.offsets[e] = v;
    if (before && e < a.E) at[e] = v + before[e];
  }
}

__device__ __forceinline__ int32_t load_shared_of(const int32_t* p, uint32_t rank) {
  int32_t v;
  asm volatile("{\n .reg .b32 a;\n mapa.shared::cluster.u32 a, %1, %2;\n ld.shared::cluster.s32 %0, [a];\n}"
               : "=r"(v)
               : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank)
               : "memory");
  return v;
}

// ONE: a cluster of up to kClusterMost blocks, with at most kSub pairs each, which see one another's counts
// and so group their pairs too.
constexpr int kClusterMost = 8;
template <typename T, int L, int KM, bool ONE>
__global__ void __launch_bounds__(kThreads, kBlocksPerSM) k_route(const RouteArgs a) {
  __shared__ __align__(16) int32_t hist[kMaxExperts], at[kMaxExperts + 1];
  extern __shared__ int32_t dyn[];  // ONE: count [kWarps][E], ids [kSub]
  int16_t* ids = ONE ? reinterpret_cast<int16_t*>(dyn + kWarps * a.E) : nullptr;
  for (int e = threadIdx.x; e < kMaxExperts; e += kThreads) hist[e] = 0;
  __syncthreads();
  pdl_wait();
  const int64_t r0 = (int64_t)blockIdx.x * a.chunk, r1 = r0 + a.chunk < a.rows ? r0 + a.chunk : a.rows;
  if (r0 < r1) {
    if (a.logits) {
      choose<T, L, KM>(a, r0, r1, hist, ids);
    } else {
      for (int64_t p = r0 * a.k + threadIdx.x; p < r1 * a.k; p += kThreads) {
        const int e = a.experts[p];
        if (ONE) ids[p - r0 * a.k] = (int16_t)e;
        if (e >= 0) atomicAdd(&hist[e], 1);
      }
    }
  }
  if constexpr (ONE) {
    __shared__ __align__(16) int32_t all[kMaxExperts], before[kMaxExperts];
    const bool cluster = gridDim.x > 1;  // the grid is the cluster
    if (cluster) {
      __syncwarp();
      asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
      for (int e = threadIdx.x; e < kMaxExperts; e += kThreads) {
        int32_t n = 0, b = 0;
        for (uint32_t r = 0; e < a.E && r < gridDim.x; r++) {
          const int32_t v = load_shared_of(&hist[e], r);
          n += v;
          if (r < blockIdx.x) b += v;
        }
        all[e] = n;
        before[e] = b;
      }
      __syncwarp();
      asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // the others' counts are read
    }
    __syncthreads();
    scan_experts(cluster ? all : hist, at, a.E);
    first_slots(a, at, cluster ? before : nullptr);
    __syncthreads();
    if (r0 < r1) assign_slots(a, r0 * a.k, (int)((r1 - r0) * a.k), ids, at, dyn);
    __syncwarp();
    if (cluster) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // nobody reads this block's now
  } else {
    __syncthreads();
    for (int e = threadIdx.x; e < a.E; e += kThreads) {
      const int32_t n = hist[e];
      a.hist[(int64_t)blockIdx.x * a.E + e] = n;
      if (n) atomicAdd(&a.spans[(int64_t)(blockIdx.x / kSpan) * a.E + e], n);
    }
  }
}

// One block per block of k_route, the same rows.
__global__ void __launch_bounds__(kThreads, kBlocksPerSM) k_group(const RouteArgs a) {
  __shared__ __align__(16) int32_t at[kMaxExperts + 1], before[kMaxExperts], all[kMaxExperts];
  __shared__ int16_t ids[kSub];
  __shared__ bool last;
  extern __shared__ int32_t count[];
  for (int e = threadIdx.x; e < kMaxExperts; e += kThreads) before[e] = all[e] = 0;
  __syncthreads();
  pdl_wait();
  const int64_t r0 = (int64_t)blockIdx.x * a.chunk, r1 = r0 + a.chunk < a.rows ? r0 + a.chunk : a.rows;
  const int64_t p0 = r0 * a.k, p1 = r0 < r1 ? r1 * a.k : p0;
  // A run's experts are on their way while the block finds its first slots, or ranks the run before.
  int32_t next[kSub / kThreads];
  auto fetch = [&](int64_t p) {
#pragma unroll
    for (int i = 0; i < kSub / kThreads; i++) {
      const int64_t at_p = p + i * kThreads + threadIdx.x;
      next[i] = at_p < p1 ? a.experts[at_p] : -1;
    }
  };
  fetch(p0);
  // kThreads / E threads share an expert's counts.
  const int spans = (gridDim.x + kSpan - 1) / kSpan, mine = blockIdx.x / kSpan;
  const int share = kThreads / a.E, e = threadIdx.x % a.E, part = threadIdx.x / a.E;
  if (part < share) {
    int32_t b = 0, n = 0;
#pragma unroll 4
    for (int i = part; i < spans; i += share) {
      const int32_t v = __ldcg(&a.spans[(int64_t)i * a.E + e]);
      n += v;
      b += i < mine ? v : 0;
    }
#pragma unroll 4
    for (int i = mine * kSpan + part; i < (int)blockIdx.x; i += share) b += __ldcg(&a.hist[(int64_t)i * a.E + e]);
    atomicAdd(&before[e], b);
    atomicAdd(&all[e], n);
  }
  __syncthreads();
  // The last block to have read the runs' counts clears them for the next call.
  if (threadIdx.x == 0) {
    __threadfence();
    last = atomicAdd(a.ticket, 1) == (int)gridDim.x - 1;
  }
  scan_experts(all, at, a.E);
  first_slots(a, at, before);
  if (last) {
    for (int i = threadIdx.x; i < spans * a.E; i += kThreads) a.spans[i] = 0;
    if (threadIdx.x == 0) *a.ticket = 0;
  }
  for (int64_t p = p0; p < p1; p += kSub) {
    __syncthreads();  // the first slots stand; the last run's ids and counts have been read
#pragma unroll
    for (int i = 0; i < kSub / kThreads; i++) ids[i * kThreads + threadIdx.x] = (int16_t)next[i];
    if (p + kSub < p1) fetch(p + kSub);
    __syncthreads();
    assign_slots(a, p, (int)(p1 - p < kSub ? p1 - p : kSub), ids, at, count);
  }
}

template <typename T, int L, int KM>
int32_t route_l(Ctx* c, const RouteArgs& a, int blocks, bool one) {
  const size_t smem = (size_t)kWarps * a.E * 4;  // at most 16 KB
  if constexpr (L < 32) {  // a warp a row: few rows, which one cluster always holds
    if (!one) {
      FL_CUDA(c, launch_pdl(k_route<T, L, KM, false>, dim3(blocks), dim3(kThreads), 0, c->stream, a));
      FL_LAUNCH(c);
      const cudaError_t e = launch_pdl(k_group, dim3(blocks), dim3(kThreads), smem, c->stream, a);
      if (e != cudaSuccess) {  // nobody clears the runs' counts
        cudaMemsetAsync(a.spans, 0, (size_t)((blocks + kSpan - 1) / kSpan) * a.E * 4, c->stream);
        FL_CUDA(c, e);
      }
      FL_LAUNCH(c);
      return FLETCHER_OK;
    }
  }
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = blocks;
  at[1].val.clusterDim.y = 1;
  at[1].val.clusterDim.z = 1;
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem + kSub * 2;
  cfg.stream = c->stream;
  cfg.attrs = at;
  cfg.numAttrs = blocks > 1 ? 2 : 1;
  FL_CUDA(c, cudaLaunchKernelEx(&cfg, k_route<T, L, KM, true>, a));
  FL_LAUNCH(c);
  return FLETCHER_OK;
}

template <typename T, int L>
int32_t route_k(Ctx* c, const RouteArgs& a, int blocks, bool one) {
  if (a.k <= 2) return route_l<T, L, 2>(c, a, blocks, one);
  if constexpr (L > 1)  // one lane: at most 8 experts
    if (a.k > 8) return route_l<T, L, 16>(c, a, blocks, one);
  return route_l<T, L, 8>(c, a, blocks, one);
}

// Lanes a row: one where a chunk holds all experts; a warp for few rows of many experts, where the chain of
// chunks is what takes time (128 x 256 -> 8: 5.8 us, 9.0 with four; 32 x 64 -> 6: 5.4 against 4.1).
constexpr int kWarpRowsMost = 128;
static_assert((kWarpRowsMost + kSub / kMaxTopK - 1) / (kSub / kMaxTopK) <= kClusterMost &&
                  (kWarpRowsMost + kWarps - 1) / kWarps <= 2 * kClusterMost,
              "one launch takes as many rows, whatever top_k");
int lanes_of(const RouteArgs& a) { return a.E <= V ? 1 : a.E > 8 * V && a.rows <= kWarpRowsMost ? 32 : 4; }

template <typename T>
int32_t route_t(Ctx* c, const RouteArgs& a, int blocks, bool one) {
  const int lanes = lanes_of(a);
  return lanes == 1   ? route_k<T, 1>(c, a, blocks, one)
         : lanes == 4 ? route_k<T, 4>(c, a, blocks, one)
                      : route_k<T, 32>(c, a, blocks, one);
}

int max_blocks(const Ctx* c) { return kBlocksPerSM * c->num_sms; }
int64_t max_spans(const Ctx* c) { return (max_blocks(c) + kSpan - 1) / kSpan; }

int32_t route(Routing* r, int32_t dtype, RouteArgs a) {
  Ctx* c = r->c;
  a.E = r->num_experts;
  a.k = r->top_k;
  a.experts = r->experts;
  a.weights = r->weights;
  a.slots = r->slots;
  a.pair_of = r->pair_of;
  a.offsets = r->offsets;
  a.hist = r->hist;
  a.spans = r->spans;
  a.ticket = r->ticket;
  const int64_t pass = kThreads / lanes_of(a);  // rows a block takes at once
  const int64_t passes = std::max<int64_t>(1, (a.rows + pass - 1) / pass);
  // One launch where a cluster's blocks hold the pairs and take no more than two turns (4096 x 64 -> 6 in
  // four turns: 15.4 us, in two launches 9.3; 4096 x 8 -> 2: 5.2 against 7.6).
  const int64_t fit = (a.rows + kSub / a.k - 1) / (kSub / a.k);  // blocks of at most kSub pairs
  const bool one = fit <= kClusterMost && passes <= 2 * kClusterMost;
  int64_t blocks = std::max(fit, std::min<int64_t>(passes, one ? kClusterMost : max_blocks(c)));
  if (one) {
    a.chunk = (a.rows + blocks - 1) / blocks;
  } else {
    blocks = std::min<int64_t>(blocks, max_blocks(c));
    a.chunk = (a.rows + blocks - 1) / blocks;
    blocks = (a.rows + a.chunk - 1) / a.chunk;
  }
  const int n = (int)blocks;
  if (dtype == FLETCHER_BF16) return route_t<__nv_bfloat16>(c, a, n, one);
  if (dtype == FLETCHER_F16) return route_t<__half>(c, a, n, one);
  return route_t<float>(c, a, n, one);
}

// For calls that allocate, read host arrays or wait: a graph cannot hold them.
int32_t refuse_capture(Ctx* c, const char* what) {
  cudaStreamCaptureStatus st = cudaStreamCaptureStatusNone;
  FL_CUDA(c, cudaStreamIsCapturing(c->stream, &st));
  FL_CHECK(c, st == cudaStreamCaptureStatusNone, "Routing: %s cannot be captured", what);
  return FLETCHER_OK;
}

}  // namespace

int32_t routing_workspace(Routing* r, int64_t bytes, void** out) {
  Ctx* c = r->c;
  const int n = r->num_work;
  if (n == 0 || r->work_bytes[n - 1] < bytes) {
    cudaStreamCaptureStatus st = cudaStreamCaptureStatusNone;
    FL_CUDA(c, cudaStreamIsCapturing(c->stream, &st));
    FL_CHECK(c, st == cudaStreamCaptureStatusNone,
             "Linear_Grouped: the routing's workspace must grow; make the call once before capturing it");
    FL_CHECK(c, n < Routing::kMaxBlocks, "Linear_Grouped: the routing's workspace cannot grow further");
    // Twice the last block: what was outgrown adds up to less than the newest, and that is less than twice the
    // largest need.
    const int64_t want = std::max(bytes, n ? 2 * r->work_bytes[n - 1] : 0);
    int32_t rc = dev_alloc(c, &r->work[n], want);
    r->work_bytes[n] = want;
    if (rc && want > bytes) {
      rc = dev_alloc(c, &r->work[n], bytes);
      r->work_bytes[n] = bytes;
    }
    if (rc) return rc;
    r->num_work++;
  }
  *out = r->work[r->num_work - 1];
  return FLETCHER_OK;
}

}  // namespace fl

using namespace fl;

extern "C" {

int32_t Cuda_Routing_Create(CudaContextRef ctx, int64_t max_rows, int32_t num_experts, int32_t top_k,
                            CudaRoutingRef* out) {
  Ctx* c = reinterpret_cast<Ctx*>(ctx);
  if (!c) return FLETCHER_ERR_INVALID;
  DeviceGuard g(c);
  FL_CHECK(c, out, "Routing: null result");
  *out = nullptr;
  FL_CHECK(c, num_experts >= 1 && num_experts <= kMaxExperts, "Routing: %d experts outside [1, %d]", num_experts,
           kMaxExperts);
  FL_CHECK(c, top_k >= 1 && top_k <= std::min(kMaxTopK, num_experts), "Routing: %d choices outside [1, %d]", top_k,
           std::min(kMaxTopK, num_experts));
  FL_CHECK(c, max_rows >= 0 && max_rows <= ((int64_t)1 << 30) / top_k, "Routing: %lld rows are too many",
           (long long)max_rows);
  int32_t rc = refuse_capture(c, "Create");
  if (rc) return rc;
  Routing* r = new (std::nothrow) Routing();
  if (!r) return set_error(c, FLETCHER_ERR_OOM, "Routing: out of host memory");
  r->c = c;
  r->device = c->device;
  r->max_rows = max_rows;
  r->num_experts = num_experts;
  r->top_k = top_k;
  const int64_t pairs = (max_rows * top_k + 3) / 4 * 4;  // keeps every array 16-byte aligned
  const int64_t ints = 4 * pairs + (num_experts + 1 + 3) / 4 * 4 + (max_blocks(c) + max_spans(c)) * num_experts + 1;
  r->bytes = ints * 4;
  if ((rc = dev_alloc(c, &r->mem, r->bytes))) {
    delete r;
    return rc;
  }
  r->experts = (int32_t*)r->mem;
  r->weights = (float*)(r->experts + pairs);
  r->slots = r->experts + 2 * pairs;
  r->pair_of = r->experts + 3 * pairs;
  r->offsets = r->experts + 4 * pairs;
  r->hist = r->offsets + (num_experts + 1 + 3) / 4 * 4;
  r->spans = r->hist + (int64_t)max_blocks(c) * num_experts;
  r->ticket = r->spans + max_spans(c) * num_experts;  // both 0, as dev_alloc fills
  *out = r;
  return FLETCHER_OK;
}

int32_t Cuda_Routing_Free(CudaRoutingRef routing) {
  Routing* r = as_routing(routing);
  if (!r) return FLETCHER_OK;
  DeviceGuard g(r->c);
  dev_free(r->c, r->mem, r->bytes);
  for (int i = 0; i < r->num_work; i++) dev_free(r->c, r->work[i], r->work_bytes[i]);
  delete r;
  return FLETCHER_OK;
}

int32_t Cuda_Routing_TopK(CudaRoutingRef routing, CudaBufferRef logits, int64_t rows, int32_t scoring,
                          int32_t normalise, float scale) {
  Routing* r = as_routing(routing);
  if (!r) return FLETCHER_ERR_INVALID;
  Ctx* c = r->c;
  DeviceGuard g(c);
  const Buf* z = reinterpret_cast<const Buf*>(logits);
  FL_CHECK(c, r->device == c->device, "Routing: made on another device");
  FL_CHECK(c, rows >= 0 && rows <= r->max_rows, "Routing: %lld rows outside [0, %lld]", (long long)rows,
           (long long)r->max_rows);
  FL_CHECK(c, holds(c, z, rows * r->num_experts), "Routing: logits must hold %lldx%d on the context's device",
           (long long)rows, r->num_experts);
  FL_CHECK(c, !overlap(z->ptr, rows * r->num_experts * dtype_size(z->dtype), r->mem, r->bytes),
           "Routing: the logits overlap the routing");
  FL_CHECK(c, scoring == FLETCHER_SCORE_SOFTMAX || scoring == FLETCHER_SCORE_SIGMOID, "Routing: unknown scoring %d",
           scoring);
  RouteArgs a{};
  a.logits = z->ptr;
  a.rows = rows;
  a.sigmoid = scoring == FLETCHER_SCORE_SIGMOID;
  a.normalise = normalise != 0;
  a.scale = scale;
  r->rows = -1;  // not valid unless all is enqueued
  const int32_t rc = route(r, z->dtype, a);
  if (rc) return rc;
  r->rows = rows;
  return FLETCHER_OK;
}

int32_t Cuda_Routing_Assign(CudaRoutingRef routing, const int32_t* experts, const float* weights, int64_t rows) {
  Routing* r = as_routing(routing);
  if (!r) return FLETCHER_ERR_INVALID;
  Ctx* c = r->c;
  DeviceGuard g(c);
  FL_CHECK(c, r->device == c->device, "Routing: made on another device");
  FL_CHECK(c, rows >= 0 && rows <= r->max_rows, "Routing: %lld rows outside [0, %lld]", (long long)rows,
           (long long)r->max_rows);
  FL_CHECK(c, experts || rows == 0, "Routing: null experts");
  const int64_t pairs = rows * r->top_k;
  for (int64_t i = 0; i < pairs; i++)
    FL_CHECK(c, experts[i] >= -1 && experts[i] < r->num_experts, "Routing: expert %d outside [-1, %d)", experts[i],
             r->num_experts);
  int32_t rc = refuse_capture(c, "Assign");
  if (rc) return rc;
  r->rows = -1;
  if ((rc = stage_to_device(c, r->experts, experts, pairs * 4))) return rc;
  if (weights) {
    rc = stage_to_device(c, r->weights, weights, pairs * 4);
  } else {
    try {
      const std::vector<float> ones((size_t)pairs, 1.0f);
      rc = stage_to_device(c, r->weights, ones.data(), pairs * 4);
    } catch (const std::bad_alloc&) {
      return set_error(c, FLETCHER_ERR_OOM, "Routing: out of host memory");
    }
  }
  if (rc) return rc;
  RouteArgs a{};
  a.rows = rows;
  if ((rc = route(r, FLETCHER_F32, a))) return rc;
  r->rows = rows;
  return FLETCHER_OK;
}

int32_t Cuda_Routing_Read(CudaRoutingRef routing, int32_t* experts, float* weights, int32_t* slots,
                          int32_t* offsets) {
  Routing* r = as_routing(routing);
  if (!r) return FLETCHER_ERR_INVALID;
  Ctx* c = r->c;
  DeviceGuard g(c);
  FL_CHECK(c, r->device == c->device, "Routing: made on another device");
  FL_CHECK(c, r->rows >= 0, "Routing: nothing routed yet");
  const int32_t rc = refuse_capture(c, "Read");
  if (rc) return rc;
  const size_t n = (size_t)r->pairs() * 4;
  const struct {
    void* to;
    const void* from;
    size_t bytes;
  } copies[] = {{experts, r->experts, n},
                {weights, r->weights, n},
                {slots, r->slots, n},
                {offsets, r->offsets, (size_t)(r->num_experts + 1) * 4}};
  for (const auto& k : copies)
    if (k.to && k.bytes) FL_CUDA(c, cudaMemcpyAsync(k.to, k.from, k.bytes, cudaMemcpyDeviceToHost, c->stream));
  FL_CUDA(c, cudaStreamSynchronize(c->stream));
  return FLETCHER_OK;
}

int32_t Cuda_Routing_DevicePointers(CudaRoutingRef routing, void** experts, void** weights, void** slots,
                                    void** offsets) {
  Routing* r = as_routing(routing);
  if (!r) return FLETCHER_ERR_INVALID;
  if (experts) *experts = r->experts;
  if (weights) *weights = r->weights;
  if (slots) *slots = r->slots;
  if (offsets) *offsets = r->offsets;
  return FLETCHER_OK;
}

}  // extern "C"
