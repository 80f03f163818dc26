// The scalars of one Adam step, shared by the flat and the list entry points.
#pragma once
#include <cmath>
#include <cstring>

#include "../../include/yafsdp_hip.h"
#include "launch.h"

namespace yafsdp {

inline AdamScalars adam_scalars(double lr, double beta1, double beta2, double eps, double weight_decay, int64_t step,
                                int flags) {
  // scalars exactly as torch.optim computes them: Python floats (binary64),
  // rounded to binary32 where they enter a tensor op
  AdamScalars s;
  std::memset(&s, 0, sizeof(s));
  s.flags = 0;
  if (weight_decay != 0.0) {
    if (flags & YAFSDP_ADAM_DECOUPLED_DECAY) {
      s.flags |= ADAM_DECOUPLED;
      s.decay = static_cast<float>(1.0 - lr * weight_decay);
    } else {
      s.flags |= ADAM_L2;
      s.l2 = static_cast<float>(weight_decay);
    }
  }
  s.w = static_cast<float>(1.0 - beta1);
  s.w_m1 = s.w - 1.0f;
  if (std::fabs(s.w) < 0.5f) s.flags |= ADAM_W_SMALL;
  s.beta2 = static_cast<float>(beta2);
  s.one_m_beta2 = static_cast<float>(1.0 - beta2);
  const double bc1 = 1.0 - std::pow(beta1, double(step));
  const double bc2 = 1.0 - std::pow(beta2, double(step));
  s.bc2_sqrt = static_cast<float>(std::pow(bc2, 0.5));
  s.eps = static_cast<float>(eps);
  s.neg_step = static_cast<float>(-(lr / bc1));
  if (flags & YAFSDP_ADAM_ZERO_GRAD) s.flags |= ADAM_ZERO_GRAD;
  return s;
}

}  // namespace yafsdp
