// The gated block's activation, in its kernels of one row, few rows and many.
#pragma once
#include "glu_launch.h"

namespace mq {

// act(g), in float.
__device__ __forceinline__ float glu_act(float g, int act) {
  // the tanh form 0.5 g (1 + tanh(z / 2)) is g / (1 + exp(-z))
  const float z = act == kActSilu ? g : kGeluZ * (g + kGeluCubic * g * g * g);
  return g / (1.0f + expf(-z));
}

}  // namespace mq
