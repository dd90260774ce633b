// 8-bit activation checkpoints: a tensor [rows, cols] as one byte an element and one scale byte per
// 32 elements of a row (format in afiv_layer.h), and back.  No counterpart in the reference, which
// keeps every activation of a training step in FP32.
//
// Both directions are one pass bound by HBM: packing reads the type's size and writes 33/32 bytes an
// element, restoring the reverse.  A lane owns 8 consecutive elements (one 16-byte load of a 16-bit
// type), so the four lanes of a block of 32 find its largest magnitude with two exchanges.  32768 x 4096 in BF16: packing
// 92 us (4.4 TB/s), restoring 106 us (3.8 TB/s; a copy reaches 4.95).
#include "afiv_layer.h"

namespace {

constexpr int THREADS = 256;

// lanes of a block of 32: 4 consecutive ones.  One lane per 8 elements; a row is padded to whole blocks.
template <class T>
__global__ __launch_bounds__(THREADS) void pack_kernel(const T *__restrict__ x, int64_t rows, int64_t cols, int64_t units,
                                                       int8_t *__restrict__ codes, uint8_t *__restrict__ scales)
{
    const int64_t nb = (cols + 31) / 32, per = nb * 4;
    for (int64_t u = (int64_t)blockIdx.x * THREADS + threadIdx.x; u < units; u += (int64_t)gridDim.x * THREADS) {
        const int64_t row = u / per, c = (u - row * per) * 8;
        const int n = (int)(cols - c < 8 ? cols - c : 8);            // may be <= 0 in a row's last block
        Pack<T, 8> v = {};
        if (n > 0) v = load_some<T, 8>(x + row * cols + c, n);
        float f[8], amax = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            f[i] = (float)v.v[i];
            amax = fmaxf(amax, finite_abs(f[i]));
        }
        amax = fmaxf(amax, __shfl_xor(amax, 1));
        amax = fmaxf(amax, __shfl_xor(amax, 2));
        const int e = scale_byte(amax);
        Pack<int8_t, 8> q;
#pragma unroll
        for (int i = 0; i < 8; ++i) q.v[i] = eight_code(f[i], e);
        if (n > 0) store_some<int8_t, 8>(codes + row * cols + c, q, n);
        if ((c & 31) == 0) scales[row * nb + c / 32] = (uint8_t)e;
    }
}

template <class T>
__global__ __launch_bounds__(THREADS) void restore_kernel(const int8_t *__restrict__ codes, const uint8_t *__restrict__ scales,
                                                          int64_t rows, int64_t cols, int64_t units, T *__restrict__ x)
{
    const int64_t nb = (cols + 31) / 32, per = (cols + 7) / 8;
    for (int64_t u = (int64_t)blockIdx.x * THREADS + threadIdx.x; u < units; u += (int64_t)gridDim.x * THREADS) {
        const int64_t row = u / per, c = (u - row * per) * 8;
        const int n = (int)(cols - c < 8 ? cols - c : 8);
        const Pack<int8_t, 8> q = load_some<int8_t, 8>(codes + row * cols + c, n);
        const int e = scales[row * nb + c / 32];
        Pack<T, 8> v;
#pragma unroll
        for (int i = 0; i < 8; ++i) v.v[i] = (T)eight_value(q.v[i], e);
        store_some<T, 8>(x + row * cols + c, v, n);
    }
}

unsigned blocks_for(int64_t units)
{
    const int64_t b = (units + THREADS - 1) / THREADS;
    return (unsigned)(b < 16384 ? b : 16384);
}

template <class T>
int pack(const void *x, int64_t rows, int64_t cols, int8_t *codes, uint8_t *scales, hipStream_t s)
{
    const int64_t units = rows * ((cols + 31) / 32 * 4);       // a multiple of 4: the lanes of a block stay together
    hipLaunchKernelGGL(pack_kernel<T>, dim3(blocks_for(units)), dim3(THREADS), 0, s, (const T *)x, rows, cols, units, codes, scales);
    return hipGetLastError() == hipSuccess ? AFIV_OK : AFIV_E_HIP;
}
template <class T>
int restore(const int8_t *codes, const uint8_t *scales, int64_t rows, int64_t cols, void *x, hipStream_t s)
{
    const int64_t units = rows * ((cols + 7) / 8);
    hipLaunchKernelGGL(restore_kernel<T>, dim3(blocks_for(units)), dim3(THREADS), 0, s, codes, scales, rows, cols, units, (T *)x);
    return hipGetLastError() == hipSuccess ? AFIV_OK : AFIV_E_HIP;
}

}  // namespace

int afiv_launch_checkpoint8_pack(const void *x, int dtype, int64_t rows, int64_t cols, int8_t *codes, uint8_t *scales, hipStream_t s)
{
    if (rows == 0 || cols == 0) return AFIV_OK;
    if (dtype == AFIV_F32) return pack<float>(x, rows, cols, codes, scales, s);
    if (dtype == AFIV_BF16) return pack<__bf16>(x, rows, cols, codes, scales, s);
    return pack<_Float16>(x, rows, cols, codes, scales, s);
}

int afiv_launch_checkpoint8_restore(const int8_t *codes, const uint8_t *scales, int dtype, int64_t rows, int64_t cols, void *x,
                                    hipStream_t s)
{
    if (rows == 0 || cols == 0) return AFIV_OK;
    if (dtype == AFIV_F32) return restore<float>(codes, scales, rows, cols, x, s);
    if (dtype == AFIV_BF16) return restore<__bf16>(codes, scales, rows, cols, x, s);
    return restore<_Float16>(codes, scales, rows, cols, x, s);
}
