// The arithmetic of one Adam(W) step on one element, shared by the flat kernel and the list kernel.
#pragma once
#include "launch.h"

namespace yafsdp {

// Per element, the operation order of torch.optim.AdamW / Adam (single-tensor
// and foreach forms alike) with every intermediate tensor rounded to binary32:
//   g   = grad * grad_scale                        (when a scale pointer is given)
//   g   = fma(p, wd, g)                            (Adam, L2 form: grad.add(param, alpha=wd))
//   p   = p * (1 - lr*wd)                          (AdamW: param.mul_)
//   m   = fma(w, g - m, m)          w = 1 - beta1 < 0.5      (exp_avg.lerp_(grad, w))
//       = fma(w - 1, g - m, g)      otherwise
//   v   = fma((1 - beta2) * g, g, v * beta2)       (mul_ then addcmul_)
//   den = sqrt(v) / sqrt(1 - beta2^t) + eps
//   p   = p + (-(lr / (1 - beta1^t)) * m) / den    (addcdiv_)
//   out16 = round16(p)                             (next iteration's all-gather input)
// The multiply-adds are fused exactly where torch's CPU kernels fuse them;
// division and square root are correctly rounded (the compiler's default for
// binary32 `/` and sqrtf in HIP code; the *_rn sqrt intrinsic is the 1-ulp one).

__device__ __forceinline__ void adam_elem(float& p, float g, float& m, float& v, const AdamScalars& s, bool scaled,
                                          float gs) {
  if (scaled) g = __fmul_rn(g, gs);
  if (s.flags & ADAM_L2) g = __fmaf_rn(p, s.l2, g);
  if (s.flags & ADAM_DECOUPLED) p = __fmul_rn(p, s.decay);
  const float d = __fsub_rn(g, m);
  m = (s.flags & ADAM_W_SMALL) ? __fmaf_rn(s.w, d, m) : __fmaf_rn(s.w_m1, d, g);
  v = __fmaf_rn(__fmul_rn(s.one_m_beta2, g), g, __fmul_rn(v, s.beta2));
  const float den = __fadd_rn(__fdiv_rn(__builtin_sqrtf(v), s.bc2_sqrt), s.eps);
  p = __fadd_rn(p, __fdiv_rn(__fmul_rn(s.neg_step, m), den));
}

}  // namespace yafsdp
