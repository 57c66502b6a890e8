// Routing of rows to experts: top-k choice, weights, and the order of the choices by expert.
//
// A row's E logits lie in V = 8 consecutive values per lane of a group of G lanes (G the power of
// two >= E / 8, at most a warp), so one or two vector loads a lane read the row.  A candidate is one
// integer key: the logit's bits in an order that compares like the value, above the complement of the
// expert's index, so the largest key is the largest logit and, among equals, the lowest expert (32
// bits for 16-bit logits, else 64).  Each lane sorts its eight keys once (19 exchanges); a round
// then takes the largest of the lanes' first keys (log2 G shuffles) and its owner moves on, where
// comparing all eight again would cost 24 operations a round.  Lane j mod G keeps choice j and
// computes its exponential, with the first winner as the maximum.
//
// Grouping is a stable counting sort in two launches without atomics on memory: k_route leaves, per
// block of rows, how many choices each expert got; k_group sums the blocks before its own (and all
// of them, for the offsets), ranks its pairs within the block, and writes slots and their inverse.
// Up to kOneBlockPairs pairs one block does both in one launch.  Nothing depends on the order in
// which blocks or atomics run, so the slots are the same in every run.
#include <algorithm>
#include <new>
#include <vector>

#include "routing.cuh"

namespace fl {
namespace {

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kBlocksPerSM = 2;
constexpr int V = 8;  // logits per lane
// Keys.  0 for what is never chosen: -inf and NaN; +0 and -0 are equal.
template <typename T>
struct KeyOf {  // f32
  typedef unsigned long long K;
  static __device__ __forceinline__ K make(float x, int e) {
    if (!(x > -INFINITY)) return 0;
    if (x == 0.0f) x = 0.0f;
    const uint32_t b = __float_as_uint(x);
    return ((K)((b & 0x80000000u) ? ~b : b | 0x80000000u) << 32) | (uint32_t)~e;
  }
  static __device__ __forceinline__ int expert(K k) { return (int)~(uint32_t)k; }
  static __device__ __forceinline__ float value(K k) {
    const uint32_t o = (uint32_t)(k >> 32);
    return __uint_as_float((o & 0x80000000u) ? o & 0x7fffffffu : ~o);
  }
};
template <typename T>
struct KeyOf16 {
  typedef uint32_t K;
  static __device__ __forceinline__ K make(T x, int e) {
    const float f = to_f<T>(x);
    if (!(f > -INFINITY)) return 0;
    const uint32_t b = f == 0.0f ? 0 : *reinterpret_cast<const uint16_t*>(&x);
    return (((b & 0x8000u) ? ~b & 0xffffu : b | 0x8000u) << 16) | (uint32_t)(0xffff - e);
  }
  static __device__ __forceinline__ int expert(K k) { return 0xffff - (int)(k & 0xffffu); }
  static __device__ __forceinline__ float value(K k) {
    const uint32_t o = k >> 16;
    const uint16_t b = (uint16_t)((o & 0x8000u) ? o & 0x7fffu : ~o);
    return to_f<T>(*reinterpret_cast<const T*>(&b));
  }
};
template <>
struct KeyOf<__half> : KeyOf16<__half> {};
template <>
struct KeyOf<__nv_bfloat16> : KeyOf16<__nv_bfloat16> {};

// Eight keys in descending order.
template <typename K>
__device__ __forceinline__ void sort8(K (&k)[8]) {
  auto ex = [&](int i, int j) {
    const K hi = k[i] > k[j] ? k[i] : k[j], lo = k[i] > k[j] ? k[j] : k[i];
    k[i] = hi;
    k[j] = lo;
  };
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
  int32_t* hist;
};

// exp(x - m) where x may equal an infinite m.
__device__ __forceinline__ float exp_below(float x, float m) { return x == m ? 1.0f : expf(x - m); }

// The choices and weights of rows [r0, r1), and into `hist` (shared) each expert's count.
template <typename T, int G>
__device__ __forceinline__ void choose(const RouteArgs& a, int64_t r0, int64_t r1, int32_t* hist) {
  typedef KeyOf<T> Key;
  typedef typename Key::K K;
  constexpr int KEEP = (kMaxTopK + G - 1) / G;  // choices a lane keeps
  constexpr int kPass = kThreads / G;
  const int lane = threadIdx.x & 31, gl = lane & (G - 1), e0 = gl * V;
  const T* z = reinterpret_cast<const T*>(a.logits);
  const bool vec = a.E % V == 0 && ((uintptr_t)z & 15) == 0;
  union Row {
    uint4 q[sizeof(T) * V / 16];
    T t[V];
  };
  // Whole groups step together; a group past the end works on the last row and writes nothing.
  auto load = [&](int64_t r, Row& u) {
    const T* row = z + (r < r1 ? r : r1 - 1) * a.E + e0;
    if (vec) {
      if (e0 < a.E) {
#pragma unroll
        for (int i = 0; i < (int)(sizeof(T) * V / 16); i++) u.q[i] = __ldg(reinterpret_cast<const uint4*>(row) + i);
      }
    } else {
#pragma unroll
      for (int i = 0; i < V; i++)
        if (e0 + i < a.E) u.t[i] = row[i];
    }
  };
  Row next;
  load(r0 + threadIdx.x / G, next);
  for (int64_t base = r0; base < r1; base += kPass) {
    const int64_t mine = base + threadIdx.x / G;
    const Row cur = next;
    if (base + kPass < r1) load(mine + kPass, next);  // on its way while this row is sorted
    K key[V];
#pragma unroll
    for (int i = 0; i < V; i++) key[i] = e0 + i < a.E ? Key::make(cur.t[i], e0 + i) : 0;
    const bool all = !a.sigmoid && !a.normalise;  // the weights' sum is over the whole row
    float x[V];
    if (all) {
#pragma unroll
      for (int i = 0; i < V; i++) x[i] = key[i] ? to_f<T>(cur.t[i]) : -INFINITY;
    }
    sort8(key);
    float m = 0.f;
    K kept[KEEP] = {};
#pragma unroll
    for (int j = 0; j < kMaxTopK; j++) {
      if (j < a.k) {
        K best = key[0];
#pragma unroll
        for (int o = 1; o < G; o <<= 1) {
          const K other = __shfl_xor_sync(0xffffffffu, best, o);
          best = other > best ? other : best;
        }
        if (key[0] == best) {  // keys are unique: one lane (or, at 0, lanes with nothing left)
#pragma unroll
          for (int i = 0; i + 1 < V; i++) key[i] = key[i + 1];
          key[V - 1] = 0;
        }
        if (j == 0) m = Key::value(best);
        if ((j & (G - 1)) == gl) kept[j / G] = best;
      }
    }
    float w[KEEP], total = 0.f;
#pragma unroll
    for (int j = 0; j < KEEP; j++) {
      const float v = Key::value(kept[j]);
      w[j] = !kept[j] ? 0.f : a.sigmoid ? 1.0f / (1.0f + expf(-v)) : exp_below(v, m);
      total += w[j];
    }
    if (all) {
      total = 0.f;
#pragma unroll
      for (int i = 0; i < V; i++)
        if (x[i] > -INFINITY) total += exp_below(x[i], m);
    }
#pragma unroll
    for (int o = 1; o < G; o <<= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    const bool divide = !a.sigmoid || a.normalise;
    if (mine < r1) {
#pragma unroll
      for (int i = 0; i < KEEP; i++) {
        const int j = i * G + gl;
        if (j < a.k) {
          const int id = kept[i] ? Key::expert(kept[i]) : -1;
          a.experts[mine * a.k + j] = id;
          a.weights[mine * a.k + j] = (divide ? (total > 0.f ? w[i] / total : 0.f) : w[i]) * a.scale;
          if (id >= 0) atomicAdd(&hist[id], 1);
        }
      }
    }
  }
}

// Slots of the pairs [p0, p1).  start[e] (shared): the first slot of expert e in this block.
// count (shared): [kWarps][E].
__device__ __forceinline__ void assign_slots(const RouteArgs& a, int64_t p0, int64_t p1, const int32_t* start,
                                             int32_t* count) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i < kWarps * a.E; i += kThreads) count[i] = 0;
  __syncthreads();
  const int64_t per = ((p1 - p0 + kWarps - 1) / kWarps + 31) / 32 * 32;
  const int64_t w0 = p0 + warp * per, w1 = w0 + per < p1 ? w0 + per : p1;
  int32_t* mine = count + warp * a.E;
  for (int64_t p = w0 + lane; p < w1; p += 32) {
    const int e = a.experts[p];
    if (e >= 0) atomicAdd(&mine[e], 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < a.E; e += kThreads) {
    int32_t at = start[e];
    for (int w = 0; w < kWarps; w++) {
      const int32_t n = count[w * a.E + e];
      count[w * a.E + e] = at;
      at += n;
    }
  }
  __syncthreads();
  for (int64_t b = w0; b < w1; b += 32) {
    const int64_t p = b + lane;
    const int e = p < w1 ? a.experts[p] : -1;
    const uint32_t same = __match_any_sync(0xffffffffu, e);
    int32_t slot = -1;
    if (e >= 0) slot = mine[e] + __popc(same & ((1u << lane) - 1));
    __syncwarp();
    if (e >= 0 && lane == 31 - __clz(same)) mine[e] = slot + 1;
    __syncwarp();
    if (p < w1) {
      a.slots[p] = slot;
      if (slot >= 0) a.pair_of[slot] = (int32_t)p;
    }
  }
}

// Exclusive prefix of n[0..E) (shared) into at[0..E), and the total; E <= 256 <= kThreads.
__device__ __forceinline__ int32_t scan_experts(const int32_t* n, int32_t* at, int E, int32_t* tmp /*[17]*/) {
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
  int32_t v = t < E ? n[t] : 0, s = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int32_t u = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += u;
  }
  if (lane == 31) tmp[warp] = s;
  __syncthreads();
  int32_t before = 0, total = 0;
  for (int w = 0; w < kWarps; w++) {
    if (w < warp) before += tmp[w];
    total += tmp[w];
  }
  if (t < E) at[t] = before + s - v;
  __syncthreads();
  return total;
}

// ONE: a single block, which groups its pairs too.
template <typename T, int G, bool ONE>
__global__ void __launch_bounds__(kThreads, kBlocksPerSM) k_route(const RouteArgs a) {
  __shared__ int32_t hist[kMaxExperts];
  for (int e = threadIdx.x; e < a.E; e += kThreads) hist[e] = 0;
  __syncthreads();
  pdl_wait();
  const int64_t r0 = (int64_t)blockIdx.x * a.chunk, r1 = r0 + a.chunk < a.rows ? r0 + a.chunk : a.rows;
  if (r0 < r1) {
    if (a.logits) {
      choose<T, G>(a, r0, r1, hist);
    } else {
      for (int64_t p = r0 * a.k + threadIdx.x; p < r1 * a.k; p += kThreads) {
        const int e = a.experts[p];
        if (e >= 0) atomicAdd(&hist[e], 1);
      }
    }
  }
  __syncthreads();
  if constexpr (ONE) {
    __shared__ int32_t at[kMaxExperts], tmp[kWarps + 1];
    extern __shared__ int32_t count[];
    const int32_t total = scan_experts(hist, at, a.E, tmp);
    for (int e = threadIdx.x; e < a.E; e += kThreads) a.offsets[e] = at[e];
    if (threadIdx.x == 0) a.offsets[a.E] = total;
    assign_slots(a, r0 * a.k, r1 * a.k, at, count);
  } else {
    for (int e = threadIdx.x; e < a.E; e += kThreads) a.hist[(int64_t)blockIdx.x * a.E + e] = hist[e];
  }
}

// One block per block of k_route, the same rows.
__global__ void __launch_bounds__(kThreads, kBlocksPerSM) k_group(const RouteArgs a) {
  __shared__ int32_t before[kMaxExperts], all[kMaxExperts], at[kMaxExperts], tmp[kWarps + 1];
  extern __shared__ int32_t count[];
  for (int e = threadIdx.x; e < a.E; e += kThreads) before[e] = all[e] = 0;
  __syncthreads();
  pdl_wait();
  // kThreads / E threads share an expert's column of the blocks' counts.
  const int share = kThreads / a.E, e = threadIdx.x % a.E, part = threadIdx.x / a.E;
  if (part < share) {
    int32_t b = 0, n = 0;
#pragma unroll 16
    for (int i = part; i < (int)gridDim.x; i += share) {
      const int32_t v = a.hist[(int64_t)i * a.E + e];
      n += v;
      if (i < (int)blockIdx.x) b += v;
    }
    atomicAdd(&before[e], b);
    atomicAdd(&all[e], n);
  }
  __syncthreads();
  const int32_t total = scan_experts(all, at, a.E, tmp);
  if (blockIdx.x == 0) {
    for (int i = threadIdx.x; i < a.E; i += kThreads) a.offsets[i] = at[i];
    if (threadIdx.x == 0) a.offsets[a.E] = total;
  }
  for (int i = threadIdx.x; i < a.E; i += kThreads) at[i] += before[i];
  __syncthreads();
  const int64_t r0 = (int64_t)blockIdx.x * a.chunk, r1 = r0 + a.chunk < a.rows ? r0 + a.chunk : a.rows;
  if (r0 < r1) assign_slots(a, r0 * a.k, r1 * a.k, at, count);
}

constexpr int64_t kOneBlockPairs = 2048;

template <typename T, int G>
int32_t route_g(Ctx* c, const RouteArgs& a, int blocks) {
  const size_t smem = (size_t)kWarps * a.E * 4;  // at most 16 KB
  if (blocks == 1) {
    FL_CUDA(c, launch_pdl(k_route<T, G, true>, dim3(1), dim3(kThreads), smem, c->stream, a));
    FL_LAUNCH(c);
    return FLETCHER_OK;
  }
  FL_CUDA(c, launch_pdl(k_route<T, G, false>, dim3(blocks), dim3(kThreads), 0, c->stream, a));
  FL_LAUNCH(c);
  FL_CUDA(c, launch_pdl(k_group, dim3(blocks), dim3(kThreads), smem, c->stream, a));
  FL_LAUNCH(c);
  return FLETCHER_OK;
}

template <typename T>
int32_t route_t(Ctx* c, const RouteArgs& a, int blocks) {
  const int lanes = (a.E + V - 1) / V;
  if (lanes <= 1) return route_g<T, 1>(c, a, blocks);
  if (lanes <= 2) return route_g<T, 2>(c, a, blocks);
  if (lanes <= 4) return route_g<T, 4>(c, a, blocks);
  if (lanes <= 8) return route_g<T, 8>(c, a, blocks);
  if (lanes <= 16) return route_g<T, 16>(c, a, blocks);
  return route_g<T, 32>(c, a, blocks);
}

int max_blocks(const Ctx* c) { return kBlocksPerSM * c->num_sms; }

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
  const int64_t pairs = a.rows * a.k;
  // A block for every 256 pairs, to keep short batches wide, up to two blocks an SM.
  const int64_t want = pairs <= kOneBlockPairs ? 1 : (pairs + 255) / 256;
  const int blocks = (int)std::min<int64_t>(want, max_blocks(c));
  a.chunk = (a.rows + blocks - 1) / blocks;
  if (dtype == FLETCHER_BF16) return route_t<__nv_bfloat16>(c, a, blocks);
  if (dtype == FLETCHER_F16) return route_t<__half>(c, a, blocks);
  return route_t<float>(c, a, blocks);
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
    // Twice the last block: what was outgrown adds up to less than the newest.
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
  FL_CHECK(c, max_rows >= 0 && max_rows <= (int64_t)INT32_MAX / top_k, "Routing: %lld rows are too many",
           (long long)max_rows);
  Routing* r = new (std::nothrow) Routing();
  if (!r) return set_error(c, FLETCHER_ERR_OOM, "Routing: out of host memory");
  r->c = c;
  r->device = c->device;
  r->max_rows = max_rows;
  r->num_experts = num_experts;
  r->top_k = top_k;
  const int64_t pairs = (max_rows * top_k + 3) / 4 * 4;  // keeps every array 16-byte aligned
  const int64_t ints = 4 * pairs + (num_experts + 1 + 3) / 4 * 4 + (int64_t)max_blocks(c) * num_experts;
  r->bytes = ints * 4;
  const int32_t rc = dev_alloc(c, &r->mem, r->bytes);
  if (rc) {
    delete r;
    return rc;
  }
  r->experts = (int32_t*)r->mem;
  r->weights = (float*)(r->experts + pairs);
  r->slots = r->experts + 2 * pairs;
  r->pair_of = r->experts + 3 * pairs;
  r->offsets = r->experts + 4 * pairs;
  r->hist = r->offsets + (num_experts + 1 + 3) / 4 * 4;
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
  r->rows = -1;
  int32_t rc = stage_to_device(c, r->experts, experts, pairs * 4);
  if (rc) return rc;
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
