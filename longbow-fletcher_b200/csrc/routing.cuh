// The routing of rows to experts: what Cuda_Routing_* fill and the grouped products and the
// combine read.
#pragma once
#include "kernels.cuh"

namespace fl {

constexpr int kMaxExperts = 256;
constexpr int kMaxTopK = 16;

struct Routing {
  Ctx* c = nullptr;
  int device = 0;
  int64_t max_rows = 0;
  int32_t num_experts = 0, top_k = 0;
  int64_t rows = -1;  // rows of the last routing; -1: none yet
  void* mem = nullptr;  // one allocation for the arrays below
  int64_t bytes = 0;
  int32_t* experts = nullptr;  // [pairs]
  float* weights = nullptr;    // [pairs]
  int32_t* slots = nullptr;    // [pairs] slot of each pair, -1: none
  int32_t* pair_of = nullptr;  // [pairs] pair of each slot; behind the last slot unspecified
  int32_t* offsets = nullptr;  // [num_experts + 1]
  int32_t *hist = nullptr, *spans = nullptr, *ticket = nullptr;  // of the counting sort (routing.cu)
  // Cuda_Linear_Grouped's copy of token rows in slot order, grown on demand.  Blocks that were outgrown
  // stay until the routing is freed: captured graphs may still use them.
  static constexpr int kMaxBlocks = 48;
  void* work[kMaxBlocks] = {};
  int64_t work_bytes[kMaxBlocks] = {};
  int num_work = 0;
  int64_t pairs() const { return rows * top_k; }
};

// At least `bytes` of the routing's workspace; may allocate, but not while the stream is captured.
int32_t routing_workspace(Routing* r, int64_t bytes, void** out);

inline Routing* as_routing(CudaRoutingRef r) { return reinterpret_cast<Routing*>(r); }

// Whether [a, a+na) and [b, b+nb) share memory.
inline bool overlap(const void* a, int64_t na, const void* b, int64_t nb) {
  const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
  return na > 0 && nb > 0 && x < y + (uintptr_t)nb && y < x + (uintptr_t)na;
}

// A buffer of the context's device that holds `elems` elements.
inline bool holds(const Ctx* c, const Buf* b, int64_t elems) {
  return b && b->device == c->device && elems >= 0 && elems <= b->bytes / dtype_size(b->dtype);
}

// What a grouped product reads and writes (grouped_simt.cu, grouped_tc.cu).  Buffers are checked against the
// rows of the last call that routed, but the arrays on the device may be those of another one: a replayed
// graph's, or an earlier one's while a later one is only captured.  So kernels bound what they read there
// by `pairs` and `x_rows`, and Cuda_Combine_Grouped's by its slots.
struct GroupedArgs {
  const void* x;     // [tokens or slots, K]
  const void* w;     // [experts * K, N]
  const void* bias;  // [experts, N] or null
  void* out;         // [slots, n_out]
  int64_t K, N, n_out;
  int64_t x_rows;          // rows of x
  const int32_t* offsets;  // [experts + 1]
  const int32_t* slots;    // rows of x are tokens: [tokens, top_k] slots of each; null: rows are slots
  const int32_t* pair_of;  // with `slots`, the inverse: slot s reads row pair_of[s] / top_k
  int32_t top_k, experts;
  int64_t pairs;  // upper bound of the slots
  int32_t act;
  bool out32;  // 16-bit operands, fp32 result
};
// silu(g) * u of 16-bit operands.  An fp32 result takes expf and a division (under 5 half places off); one that is
// rounded to 16 bits the special-function unit's, up to 30 half places of fp32 off.
__device__ __forceinline__ float swiglu_f32(float g, float u) { return __fdiv_rn(g, 1.0f + expf(-g)) * u; }
__device__ __forceinline__ float swiglu_16(float g, float u) { return __fdividef(g, 1.0f + __expf(-g)) * u; }
bool grouped_tc_supported(int32_t dtype, const GroupedArgs& a);
int64_t grouped_tc_workspace(const GroupedArgs& a);  // bytes
int32_t launch_grouped_tc(Ctx* c, int32_t dtype, const GroupedArgs& a, void* workspace);
int32_t launch_grouped_simt(Ctx* c, int32_t dtype, const GroupedArgs& a);

}  // namespace fl
