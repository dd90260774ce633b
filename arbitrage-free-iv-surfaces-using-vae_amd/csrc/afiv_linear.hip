// Entry of the linear layer: scratch sizes and the choice of the element type's kernels.
#include "afiv_internal.h"
#include "afiv_linear_plan.h"

#define DECLARE(NAME)                                                                                                                  \
    int afiv_linear_forward_##NAME(const void *, const void *, const void *, const void *, int, int64_t, int64_t, int64_t, void *,     \
                                   void *, uint8_t *, float *, hipStream_t);                                                           \
    int afiv_linear_backward_##NAME(const void *, const void *, const int8_t *, const uint8_t *, const void *, const void *,           \
                                    const uint8_t *, int, int64_t, int64_t, int64_t, void *, void *, void *, float *, hipStream_t);
DECLARE(f32)
DECLARE(bf16)
DECLARE(f16)

int64_t afiv_linear_forward_scratch(int64_t M, int64_t N, int64_t K, int dtype) { return forward_places(M, N, K, dtype == AFIV_F32).bytes; }
int64_t afiv_linear_backward_scratch(int64_t M, int64_t N, int64_t K, int dtype, int act, bool from_checkpoint)
{
    return backward_places(M, N, K, dtype == AFIV_F32, act != AFIV_ACT_NONE, from_checkpoint).bytes;
}

int afiv_launch_linear_act(const void *x, const void *w, const void *bias, const void *residual, int dtype, int act, int64_t M, int64_t N,
                           int64_t K, void *y, void *pre, uint8_t *dcodes, float *scratch, hipStream_t s)
{
    const auto f = dtype == AFIV_F32 ? afiv_linear_forward_f32 : dtype == AFIV_BF16 ? afiv_linear_forward_bf16 : afiv_linear_forward_f16;
    return f(x, w, bias, residual, act, M, N, K, y, pre, dcodes, scratch, s);
}

int afiv_launch_linear_act_backward(const void *dy, const void *x, const int8_t *codes, const uint8_t *scales, const void *w,
                                    const void *pre, const uint8_t *dcodes, int dtype, int act, int64_t M, int64_t N, int64_t K, void *dx,
                                    void *dw, void *db, float *scratch, hipStream_t s)
{
    const auto f = dtype == AFIV_F32 ? afiv_linear_backward_f32 : dtype == AFIV_BF16 ? afiv_linear_backward_bf16 : afiv_linear_backward_f16;
    return f(dy, x, codes, scales, w, pre, dcodes, act, M, N, K, dx, dw, db, scratch, s);
}
