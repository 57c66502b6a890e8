// The kernels of Cuda_Combine_Grouped (a file of their own: they take as long to compile as the rest).
#include "block_norm.cuh"

namespace fl {

int32_t launch_combine(Ctx* c, int32_t dtype, int32_t slots_dtype, const bnorm::NormArgs& a) {
  using namespace bnorm;
  if (dtype == FLETCHER_F32) return launch_norm<float, float, true>(c, a);
  if (slots_dtype == FLETCHER_F32)
    return dtype == FLETCHER_BF16 ? launch_norm<__nv_bfloat16, float, true>(c, a) : launch_norm<__half, float, true>(c, a);
  return dtype == FLETCHER_BF16 ? launch_norm<__nv_bfloat16, __nv_bfloat16, true>(c, a)
                                : launch_norm<__half, __half, true>(c, a);
}

}  // namespace fl
