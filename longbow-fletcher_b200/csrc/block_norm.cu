// Cuda_BlockNorm and Cuda_Combine_Grouped: checks; the kernels without a combine.
#include "block_norm.cuh"

namespace fl {
namespace {

// Fills and checks what both entry points share.  `y` is [y_rows, cols]; combine: y may be fp32 beside
// 16-bit buffers, and no output may be y.
int32_t setup(Ctx* c, const char* op, const Buf* y, int64_t y_rows, bool combine, int64_t rows, int64_t cols,
              const FletcherBlockNorm* n, Buf* u, Buf* h, bnorm::NormArgs* a) {
  FL_CHECK(c, y, "%s: null buffer", op);
  FL_CHECK(c, u || h, "%s: no output", op);
  const int32_t dt = u ? u->dtype : h->dtype;
  FL_CHECK(c, y->dtype == dt || (combine && y->dtype == FLETCHER_F32), "%s: dtype mismatch", op);
  const int64_t ysize = dtype_size(y->dtype);
  FL_CHECK(c, cols >= 1 && cols <= bnorm::kMaxCols, "%s: %lld columns outside [1, %d]", op, (long long)cols, bnorm::kMaxCols);
  FL_CHECK(c, rows >= 0 && rows <= INT32_MAX, "%s: %lld rows", op, (long long)rows);
  FL_CHECK(c, holds(c, y, y_rows * cols), "%s: input must hold %lldx%lld on the context's device", op,
           (long long)y_rows, (long long)cols);
  const FletcherBlockNorm none{FLETCHER_NORM_NONE, FLETCHER_NORM_NONE, 0.f, 0.f, 1.f, 0, 0, nullptr, nullptr, nullptr,
                               nullptr, nullptr, nullptr};
  if (!n) n = &none;
  FL_CHECK(c, n->post_kind >= FLETCHER_NORM_NONE && n->post_kind <= FLETCHER_NORM_RMS && n->pre_kind >= FLETCHER_NORM_NONE &&
                  n->pre_kind <= FLETCHER_NORM_RMS,
           "%s: unknown norm", op);
  FL_CHECK(c, n->reserved == 0, "%s: the reserved field must be 0", op);
  FL_CHECK(c, n->eps >= 0.f && std::isfinite(n->eps), "%s: eps must be finite and not negative", op);
  FL_CHECK(c, (h != nullptr) == (n->pre_kind != FLETCHER_NORM_NONE),
           "%s: the normed output is given exactly when there is a pre norm", op);
  const int64_t total = rows * cols, es = dtype_size(dt), bytes = total * es;
  const Buf *res = reinterpret_cast<const Buf*>(n->residual), *gate = reinterpret_cast<const Buf*>(n->gate);
  FL_CHECK(c, !res || (res->dtype == dt && holds(c, res, total)), "%s: residual must be %lldx%lld of the input's dtype",
           op, (long long)rows, (long long)cols);
  FL_CHECK(c, !gate || n->gate_rows == 1 || n->gate_rows >= rows, "%s: gate_rows must be 1 or at least the rows", op);
  const bool wide_gate = gate && n->gate_rows != 1 && rows != 1;
  FL_CHECK(c, !gate || (gate->dtype == dt && holds(c, gate, (wide_gate ? rows : 1) * cols)),
           "%s: gate must be %lldx%lld of the input's dtype", op, (long long)(wide_gate ? rows : 1), (long long)cols);
  const struct {
    CudaBufferRef ref;
    const float** to;
    int32_t kind;
    bool shift;
  } affine[] = {{n->post_gamma, &a->post_gamma, n->post_kind, false},
                {n->post_beta, &a->post_beta, n->post_kind, true},
                {n->pre_gamma, &a->pre_gamma, n->pre_kind, false},
                {n->pre_beta, &a->pre_beta, n->pre_kind, true}};
  Buf* outs[2] = {u, h};
  for (Buf* o : outs) {
    if (!o) continue;
    FL_CHECK(c, o->dtype == dt && holds(c, o, total), "%s: outputs must be %lldx%lld of the input's dtype", op,
             (long long)rows, (long long)cols);
    // An output lies over an input either not at all or element for element.
    FL_CHECK(c, (!combine && o->ptr == y->ptr) || !overlap(o->ptr, bytes, y->ptr, y_rows * cols * ysize),
             "%s: an output overlaps the input", op);
    FL_CHECK(c, !res || o->ptr == res->ptr || !overlap(o->ptr, bytes, res->ptr, bytes),
             "%s: an output overlaps the residual", op);
    FL_CHECK(c, !gate || (o->ptr == gate->ptr && (wide_gate || rows == 1)) ||
                    !overlap(o->ptr, bytes, gate->ptr, (wide_gate ? rows : 1) * cols * es),
             "%s: an output overlaps the gate", op);
  }
  FL_CHECK(c, !u || !h || !overlap(u->ptr, bytes, h->ptr, bytes), "%s: the outputs overlap", op);
  for (const auto& f : affine) {
    const Buf* b = reinterpret_cast<const Buf*>(f.ref);
    *f.to = nullptr;
    if (!b) continue;
    FL_CHECK(c, f.kind != FLETCHER_NORM_NONE, "%s: gamma or beta without its norm", op);
    FL_CHECK(c, !(f.shift && f.kind == FLETCHER_NORM_RMS), "%s: the RMS norm takes no beta", op);
    FL_CHECK(c, b->dtype == FLETCHER_F32 && holds(c, b, cols), "%s: gamma/beta must be f32 [%lld]", op, (long long)cols);
    for (Buf* o : outs)
      FL_CHECK(c, !o || !overlap(o->ptr, bytes, b->ptr, cols * 4), "%s: an output overlaps gamma or beta", op);
    *f.to = (const float*)b->ptr;
  }
  a->y = y->ptr;
  a->residual = res ? res->ptr : nullptr;
  a->gate = gate ? gate->ptr : nullptr;
  a->gate_step = wide_gate ? cols : 0;
  a->u = u ? u->ptr : nullptr;
  a->h = h ? h->ptr : nullptr;
  a->post = n->post_kind;
  a->pre = n->pre_kind;
  a->eps = n->eps;
  a->residual_scale = n->residual_scale;
  a->branch_scale = n->branch_scale;
  a->rows = rows;
  a->cols = (int32_t)cols;
  return FLETCHER_OK;
}

}  // namespace

int32_t launch_block_norm(Ctx* c, int32_t dtype, const bnorm::NormArgs& a) {
  using namespace bnorm;
  if (dtype == FLETCHER_F32) return launch_norm<float, float, false>(c, a);
  return dtype == FLETCHER_BF16 ? launch_norm<__nv_bfloat16, __nv_bfloat16, false>(c, a)
                                : launch_norm<__half, __half, false>(c, a);
}

}  // namespace fl

using namespace fl;

extern "C" {

int32_t Cuda_BlockNorm(CudaContextRef ctx, CudaBufferRef y, int64_t rows, int64_t cols, const FletcherBlockNorm* norm,
                       CudaBufferRef outResidual, CudaBufferRef outNorm) {
  Ctx* c = reinterpret_cast<Ctx*>(ctx);
  if (!c) return FLETCHER_ERR_INVALID;
  DeviceGuard g(c);
  FL_CHECK(c, norm, "BlockNorm: null parameters");
  const Buf* yb = reinterpret_cast<Buf*>(y);
  Buf *u = reinterpret_cast<Buf*>(outResidual), *h = reinterpret_cast<Buf*>(outNorm);
  bnorm::NormArgs a{};
  const int32_t rc = setup(c, "BlockNorm", yb, rows, false, rows, cols, norm, u, h, &a);
  if (rc || rows == 0) return rc;
  touch(u);
  touch(h);
  return launch_block_norm(c, yb->dtype, a);
}

int32_t Cuda_Combine_Grouped(CudaRoutingRef routing, CudaBufferRef grouped, int64_t cols, const FletcherBlockNorm* norm,
                             CudaBufferRef outResidual, CudaBufferRef outNorm) {
  Routing* r = as_routing(routing);
  if (!r) return FLETCHER_ERR_INVALID;
  Ctx* c = r->c;
  DeviceGuard g(c);
  FL_CHECK(c, r->device == c->device, "Combine_Grouped: the routing was made on another device");
  FL_CHECK(c, r->rows >= 0, "Combine_Grouped: nothing routed yet");
  const Buf* yb = reinterpret_cast<Buf*>(grouped);
  Buf *u = reinterpret_cast<Buf*>(outResidual), *h = reinterpret_cast<Buf*>(outNorm);
  bnorm::NormArgs a{};
  const int32_t rc = setup(c, "Combine_Grouped", yb, r->pairs(), true, r->rows, cols, norm, u, h, &a);
  if (rc) return rc;
  for (const Buf* o : {u, h})
    FL_CHECK(c, !o || !overlap(o->ptr, r->rows * cols * dtype_size(o->dtype), r->mem, r->bytes),
             "Combine_Grouped: an output overlaps the routing");
  if (r->rows == 0) return FLETCHER_OK;
  touch(u);
  touch(h);
  a.slots = r->slots;
  a.weights = r->weights;
  a.top_k = r->top_k;
  a.num_slots = (int32_t)r->pairs();
  return launch_combine(c, u ? u->dtype : h->dtype, yb->dtype, a);
}

}  // extern "C"
