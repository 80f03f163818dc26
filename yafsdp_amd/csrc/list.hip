// Instantiations and dispatch of the list kernels.
#include "launch.h"
#include "list_kernels.hip.h"

namespace yafsdp {

hipError_t launch_list_norm(int norm, const ListArgs& a, double* partials, int grid, hipStream_t stream) {
  switch (norm) {
    case LIST_NORM_1:
      return launch_kernel(list_norm_kernel<LIST_NORM_1, kListBlock>, grid, kListBlock, stream, a, partials);
    case LIST_NORM_2:
      return launch_kernel(list_norm_kernel<LIST_NORM_2, kListBlock>, grid, kListBlock, stream, a, partials);
    case LIST_NORM_INF:
      return launch_kernel(list_norm_kernel<LIST_NORM_INF, kListBlock>, grid, kListBlock, stream, a, partials);
    default: return hipErrorInvalidValue;
  }
}

hipError_t launch_list_finish(int norm, const double* partials, int count, float max_norm, float* norm_and_coef,
                              hipStream_t stream) {
  switch (norm) {
    case LIST_NORM_1:
      return launch_kernel(list_finish_kernel<LIST_NORM_1, 1024>, 1, 1024, stream, partials, count, max_norm,
                           norm_and_coef);
    case LIST_NORM_2:
      return launch_kernel(list_finish_kernel<LIST_NORM_2, 1024>, 1, 1024, stream, partials, count, max_norm,
                           norm_and_coef);
    case LIST_NORM_INF:
      return launch_kernel(list_finish_kernel<LIST_NORM_INF, 1024>, 1, 1024, stream, partials, count, max_norm,
                           norm_and_coef);
    default: return hipErrorInvalidValue;
  }
}

hipError_t launch_list_scale(const ListArgs& a, const float* coef, int grid, hipStream_t stream) {
  return launch_kernel(list_scale_kernel<kListBlock>, grid, kListBlock, stream, a, coef);
}

namespace {
template <class G>
hipError_t adamw_by_out(int out_dt, const ListAdamArgs& a, const AdamScalars& s, const float* grad_scale, int grid,
                        hipStream_t stream) {
  switch (out_dt) {
    case DT_F32:
      return launch_kernel(list_adamw_kernel<G, F32, kListBlock>, grid, kListBlock, stream, a, s, grad_scale);
    case DT_BF16:
      return launch_kernel(list_adamw_kernel<G, BF16, kListBlock>, grid, kListBlock, stream, a, s, grad_scale);
    case DT_F16:
      return launch_kernel(list_adamw_kernel<G, F16, kListBlock>, grid, kListBlock, stream, a, s, grad_scale);
    default: return hipErrorInvalidValue;
  }
}
}  // namespace

hipError_t launch_list_adamw(int grad_dt, int out_dt, const ListAdamArgs& a, const AdamScalars& s,
                             const float* grad_scale, int grid, hipStream_t stream) {
  switch (grad_dt) {
    case DT_F32: return adamw_by_out<F32>(out_dt, a, s, grad_scale, grid, stream);
    case DT_BF16: return adamw_by_out<BF16>(out_dt, a, s, grad_scale, grid, stream);
    case DT_F16: return adamw_by_out<F16>(out_dt, a, s, grad_scale, grid, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace yafsdp
