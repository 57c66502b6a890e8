// Cuda_Linear_Grouped: checks and choice of the kernel.
#include "routing.cuh"

using namespace fl;

extern "C" {

int32_t Cuda_Linear_Grouped(CudaRoutingRef routing, CudaBufferRef input, int32_t inputOrder, int64_t inCols,
                            CudaBufferRef weight, int64_t outCols, CudaBufferRef bias, CudaBufferRef result,
                            int32_t activation) {
  Routing* r = as_routing(routing);
  if (!r) return FLETCHER_ERR_INVALID;
  Ctx* c = r->c;
  DeviceGuard g(c);
  const Buf *x = reinterpret_cast<Buf*>(input), *w = reinterpret_cast<Buf*>(weight), *b = reinterpret_cast<Buf*>(bias);
  Buf* y = reinterpret_cast<Buf*>(result);
  FL_CHECK(c, r->device == c->device, "Linear_Grouped: the routing was made on another device");
  FL_CHECK(c, r->rows >= 0, "Linear_Grouped: nothing routed yet");
  FL_CHECK(c, x && w && y, "Linear_Grouped: null buffer");
  const int32_t dt = x->dtype;
  FL_CHECK(c, w->dtype == dt && (y->dtype == dt || y->dtype == FLETCHER_F32) && (!b || b->dtype == dt),
           "Linear_Grouped: dtype mismatch");
  FL_CHECK(c, inputOrder == FLETCHER_ROWS_TOKENS || inputOrder == FLETCHER_ROWS_SLOTS,
           "Linear_Grouped: unknown input order %d", inputOrder);
  FL_CHECK(c, activation == FLETCHER_ACT_IDENTITY || activation == FLETCHER_ACT_GELU || activation == FLETCHER_ACT_TANH ||
                  activation == FLETCHER_ACT_SWIGLU,
           "Linear_Grouped: activation %d", activation);
  const bool swiglu = activation == FLETCHER_ACT_SWIGLU;
  constexpr int64_t kMaxCols = 1 << 24;
  FL_CHECK(c, inCols >= 1 && inCols <= kMaxCols && outCols >= 1 && outCols <= kMaxCols,
           "Linear_Grouped: %lld -> %lld columns outside [1, %lld]", (long long)inCols, (long long)outCols,
           (long long)kMaxCols);
  FL_CHECK(c, !swiglu || outCols % 2 == 0, "Linear_Grouped: SwiGLU needs an even output width");
  GroupedArgs a{};
  a.K = inCols;
  a.N = outCols;
  a.n_out = swiglu ? outCols / 2 : outCols;
  a.pairs = r->pairs();
  a.x_rows = inputOrder == FLETCHER_ROWS_TOKENS ? r->rows : a.pairs;
  a.experts = r->num_experts;
  a.top_k = r->top_k;
  FL_CHECK(c, holds(c, x, a.x_rows * inCols), "Linear_Grouped: input must hold %lldx%lld on the context's device",
           (long long)a.x_rows, (long long)inCols);
  FL_CHECK(c, holds(c, w, a.experts * inCols * outCols), "Linear_Grouped: weight must hold %d x %lldx%lld",
           a.experts, (long long)inCols, (long long)outCols);
  FL_CHECK(c, !b || holds(c, b, a.experts * outCols), "Linear_Grouped: bias must hold %dx%lld", a.experts,
           (long long)outCols);
  FL_CHECK(c, holds(c, y, a.pairs * a.n_out), "Linear_Grouped: result must hold %lldx%lld", (long long)a.pairs,
           (long long)a.n_out);
  const int64_t es = dtype_size(dt), ybytes = a.pairs * a.n_out * dtype_size(y->dtype);
  FL_CHECK(c, !overlap(y->ptr, ybytes, x->ptr, a.x_rows * inCols * es) &&
                  !overlap(y->ptr, ybytes, w->ptr, a.experts * inCols * outCols * es) &&
                  !(b && overlap(y->ptr, ybytes, b->ptr, a.experts * outCols * es)) &&
                  !overlap(y->ptr, ybytes, r->mem, r->bytes),
           "Linear_Grouped: the result overlaps an input");
  if (a.pairs == 0) return FLETCHER_OK;
  a.x = x->ptr;
  a.w = w->ptr;
  a.bias = b ? b->ptr : nullptr;
  a.out = y->ptr;
  a.offsets = r->offsets;
  a.slots = inputOrder == FLETCHER_ROWS_TOKENS ? r->slots : nullptr;
  a.pair_of = inputOrder == FLETCHER_ROWS_TOKENS ? r->pair_of : nullptr;
  a.act = activation;
  a.out32 = dt != FLETCHER_F32 && y->dtype == FLETCHER_F32;
  if (grouped_tc_supported(dt, a)) {
    void* ws = nullptr;
    const int64_t need = grouped_tc_workspace(a);
    const int32_t rc = need ? routing_workspace(r, need, &ws) : FLETCHER_OK;
    if (rc) return rc;
    touch(y);
    return launch_grouped_tc(c, dt, a, ws);
  }
  touch(y);
  return launch_grouped_simt(c, dt, a);
}

}  // extern "C"
