// Instantiations and dispatch of the list kernels.
#include "launch.h"
#include "list_kernels.hip.h"

namespace yafsdp {

namespace {

// f(integral constant of the norm)
template <int N>
struct norm_t { static constexpr int value = N; };
template <class F>
hipError_t by_norm(int norm, F f) {
  switch (norm) {
    case LIST_NORM_1: return f(norm_t<LIST_NORM_1>());
    case LIST_NORM_2: return f(norm_t<LIST_NORM_2>());
    case LIST_NORM_INF: return f(norm_t<LIST_NORM_INF>());
    default: return hipErrorInvalidValue;
  }
}

}  // namespace

hipError_t launch_list_stage(const ListStageArgs& a, uint32_t* dst, hipStream_t stream) {
  return launch_kernel(list_stage_kernel, 1, kListStageWords / 4, stream, a, reinterpret_cast<u32x4*>(dst));
}

hipError_t launch_list_fetch(const void* src, void* dst, uint32_t n, uint32_t* done, uint32_t number, int grid,
                             hipStream_t stream) {
  return launch_kernel(list_fetch_kernel, grid, kListFetchBlock, stream, static_cast<const u32x4*>(src),
                       static_cast<u32x4*>(dst), n, done, number);
}

template <class META>
hipError_t launch_list_norm(int norm, const META& a, double* partials, int grid, hipStream_t stream) {
  return by_norm(norm, [&](auto n) {
    return launch_kernel(list_norm_kernel<decltype(n)::value, META, kListNormBlock>, grid, kListNormBlock, stream, a,
                         partials);
  });
}

hipError_t launch_list_finish(int norm, const double* partials, int count, float max_norm, float* norm_and_coef,
                              hipStream_t stream) {
  return by_norm(norm, [&](auto n) {
    return launch_kernel(list_finish_kernel<decltype(n)::value, kListClipBlock>, 1, kListClipBlock, stream, partials,
                         count, max_norm, norm_and_coef);
  });
}

hipError_t launch_list_small(int norm, bool clip, const ListArgs& a, float max_norm, float* norm_and_coef,
                             hipStream_t stream) {
  return by_norm(norm, [&](auto n) {
    if (clip)
      return launch_kernel(list_small_kernel<decltype(n)::value, true, kListSmallBlock>, 1, kListSmallBlock, stream, a,
                           max_norm, norm_and_coef);
    return launch_kernel(list_small_kernel<decltype(n)::value, false, kListSmallBlock>, 1, kListSmallBlock, stream, a,
                         max_norm, norm_and_coef);
  });
}

template <class META>
hipError_t launch_list_clip(int norm, const META& a, const double* partials, int count, float max_norm,
                            float* norm_and_coef, int grid, hipStream_t stream) {
  return by_norm(norm, [&](auto n) {
    return launch_kernel(list_clip_kernel<decltype(n)::value, META, kListClipBlock>, grid, kListClipBlock, stream, a,
                         partials, count, max_norm, norm_and_coef);
  });
}

namespace {
// f(first tile, workgroups) for one wave per tile in workgroups of one wave, at most kListMaxGrid of them per launch
template <class F>
hipError_t wave_per_tile(uint32_t n_tiles, F f) {
  for (uint32_t first = 0; first < n_tiles; first += kListMaxGrid) {
    const uint32_t left = n_tiles - first;
    const hipError_t e = f(first, int(left < kListMaxGrid ? left : kListMaxGrid));
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}
static_assert(kListScaleBlock == 64 && kListAdamBlock == 64, "wave_per_tile counts workgroups of one wave");
}  // namespace

template <class META>
hipError_t launch_list_scale(const META& a, const float* coef, hipStream_t stream) {
  return wave_per_tile(a.n_tiles, [&](uint32_t first, int grid) {
    return launch_kernel(list_scale_kernel<META, kListScaleBlock>, grid, kListScaleBlock, stream, a, first, coef);
  });
}

namespace {
template <class G, class O, class META>
hipError_t adamw_go(const META& a, const AdamScalars& s, const float* grad_scale, hipStream_t stream) {
  return wave_per_tile(a.n_tiles, [&](uint32_t first, int grid) {
    return launch_kernel(list_adamw_kernel<G, O, META, kListAdamBlock>, grid, kListAdamBlock, stream, a, first, s,
                         grad_scale);
  });
}
template <class G, class META>
hipError_t adamw_by_out(int out_dt, const META& a, const AdamScalars& s, const float* grad_scale, hipStream_t stream) {
  switch (out_dt) {
    case DT_F32: return adamw_go<G, F32>(a, s, grad_scale, stream);
    case DT_BF16: return adamw_go<G, BF16>(a, s, grad_scale, stream);
    case DT_F16: return adamw_go<G, F16>(a, s, grad_scale, stream);
    default: return hipErrorInvalidValue;
  }
}
}  // namespace

template <class META>
hipError_t launch_list_adamw(int grad_dt, int out_dt, const META& a, const AdamScalars& s, const float* grad_scale,
                             hipStream_t stream) {
  switch (grad_dt) {
    case DT_F32: return adamw_by_out<F32>(out_dt, a, s, grad_scale, stream);
    case DT_BF16: return adamw_by_out<BF16>(out_dt, a, s, grad_scale, stream);
    case DT_F16: return adamw_by_out<F16>(out_dt, a, s, grad_scale, stream);
    default: return hipErrorInvalidValue;
  }
}

#define YAFSDP_LIST_INSTANCES(META)                                                                               \
  template hipError_t launch_list_norm<META>(int, const META&, double*, int, hipStream_t);                        \
  template hipError_t launch_list_clip<META>(int, const META&, const double*, int, float, float*, int, hipStream_t); \
  template hipError_t launch_list_scale<META>(const META&, const float*, hipStream_t);
YAFSDP_LIST_INSTANCES(ListArgs)
YAFSDP_LIST_INSTANCES(ListRef)
#undef YAFSDP_LIST_INSTANCES
template hipError_t launch_list_adamw<ListAdamArgs>(int, int, const ListAdamArgs&, const AdamScalars&, const float*,
                                                    hipStream_t);
template hipError_t launch_list_adamw<ListAdamRef>(int, int, const ListAdamRef&, const AdamScalars&, const float*,
                                                   hipStream_t);

}  // namespace yafsdp
