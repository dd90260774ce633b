// The linear layer's kernels for FP32 (a translation unit per element type: they compile side by side).
#include "afiv_linear_kernels.h"

AFIV_LINEAR_TYPE(float, f32)
