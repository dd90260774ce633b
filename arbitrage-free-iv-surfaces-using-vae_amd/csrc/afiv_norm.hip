// Training-mode batch normalisation, activation and dropout of a hidden layer in one operator,
// forward and backward, for x [M,N] in FP32 / BF16 / FP16.  Replaces, per hidden layer, the
// BatchNorm1d -> activation -> Dropout chain of the reference's stacks (cvae_model.py:64-105).
//
//   mu, var = column mean and (biased) variance;  rstd = 1/sqrt(var + eps);  h = (x - mu) rstd
//   y = k s f(gamma h + beta),            k = keep mask, s = 1/(1-p), f = activation
//   g = dy k s f'(gamma h + beta);        dbeta = sum g;  dgamma = sum g h
//   dx = gamma rstd (g - dbeta/M - h dgamma/M)
//
// All of it is a few operations per element, so HBM bounds it: the forward pass reads x twice (the
// statistics need every row before the first output), the backward pass reads x or its 8-bit
// checkpoint, dy and keep twice.  Column sums go row chunk by row chunk: P chunks give P partial
// sums, added in chunk order by a second kernel, so results do not depend on scheduling.
//
// Statistics are summed in FP64 (plain sum and sum of squares: the squares are exact, and the
// cancellation in var = E[x^2] - mu^2 costs 1e-16 mu^2/var), and h and the pre-activation are FP64
// operations rounded to FP32 at their end: on this chip they cost what FP32 ones do, x - mu does not
// cancel, and the sign of the pre-activation, where relu's derivative jumps, does not hang on an FP32
// rounding.
#include "afiv_layer.h"

namespace {

constexpr int THREADS = 256;

template <class T> struct Vec { static constexpr int N = 16 / (int)sizeof(T); };   // elements of a 16-byte access

struct NormArgs {
    int64_t M, N, rows_per;              // rows of a chunk
    int act;
    double eps, momentum;
    float scale;                         // 1 / (1 - p)
    const float *gamma, *beta;
    const uint8_t *keep;
    float *run_mean, *run_var;
    double *stats;                       // [2,N]: mu, rstd
    double *partial;                     // [chunks,N,2]
    int64_t chunks;
    double *means;                       // backward: [2,N]: dbeta / M, dgamma / M
    int8_t *codes;
    uint8_t *scales;
    float *dgamma, *dbeta;
};

// Threads stand as TX lanes across columns (V elements each) by TY rows.  Sums of a column over the
// TY rows of the workgroup: result at the threads of row 0, in row order.
template <int V, int TX>
__device__ __forceinline__ void reduce_rows(double (&a)[V], double (&b)[V], double *lds, int tx, int ty)
{
    constexpr int TY = THREADS / TX, W = TX * V;
#pragma unroll
    for (int half = TY / 2; half >= 1; half /= 2) {
        if (ty >= half && ty < 2 * half) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                lds[((ty - half) * W + tx * V + i) * 2] = a[i];
                lds[((ty - half) * W + tx * V + i) * 2 + 1] = b[i];
            }
        }
        __syncthreads();
        if (ty < half) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                a[i] += lds[(ty * W + tx * V + i) * 2];
                b[i] += lds[(ty * W + tx * V + i) * 2 + 1];
            }
        }
        __syncthreads();
    }
}

template <class T, int V, int TX>
__device__ __forceinline__ void sum_x(const NormArgs &p, const T *__restrict__ x, int64_t r0, int64_t r1, int64_t col, int n,
                                      int ty, double (&s1)[V], double (&s2)[V])
{
    constexpr int TY = THREADS / TX;
#pragma unroll
    for (int i = 0; i < V; ++i) s1[i] = s2[i] = 0.0;
    if (n <= 0) return;
#pragma unroll 4
    for (int64_t r = r0 + ty; r < r1; r += TY) {
        const Pack<T, V> v = load_some<T, V>(x + r * p.N + col, n);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const double d = (double)(float)v.v[i];
            s1[i] += d;
            s2[i] = __builtin_fma(d, d, s2[i]);
        }
    }
}

// statistics of one column from its sums
__device__ __forceinline__ void finish_stats(const NormArgs &p, int64_t col, double s1, double s2, double &mu, double &rstd)
{
    const double m = (double)p.M;
    mu = s1 / m;
    const double d = s2 / m - mu * mu;
    const double var = d < 0.0 ? 0.0 : d;                 // NaN stays NaN
    rstd = 1.0 / sqrt(var + p.eps);
    p.stats[col] = mu;
    p.stats[p.N + col] = rstd;
    if (p.run_mean) {
        p.run_mean[col] = (float)((1.0 - p.momentum) * (double)p.run_mean[col] + p.momentum * mu);
        p.run_var[col] = (float)((1.0 - p.momentum) * (double)p.run_var[col] + p.momentum * (var * (m / (m - 1.0))));
    }
}

// outputs (and the checkpoint) of rows r0..r1 at columns col..col+n, a = gamma rstd
template <class T, int V, int TX>
__device__ __forceinline__ void apply_rows(const NormArgs &p, const T *__restrict__ x, T *__restrict__ y, int64_t r0, int64_t r1,
                                           int64_t col, int n, int ty, const double (&mu)[V], const double (&a)[V], const float (&beta)[V])
{
    constexpr int TY = THREADS / TX, LANES = 32 / V;        // lanes of a checkpoint block
    const int64_t nb = (p.N + 31) / 32;
#pragma unroll 2
    for (int64_t r = r0 + ty; r < r1; r += TY) {
        const int64_t at = r * p.N + col;
        Pack<T, V> v = {};
        if (n > 0) v = load_some<T, V>(x + at, n);
        Pack<uint8_t, V> k;
        if (p.keep && n > 0) k = load_some<uint8_t, V>(p.keep + at, n);
        Pack<T, V> out;
        float f[V], z[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            f[i] = (float)v.v[i];
            z[i] = (float)__builtin_fma((double)f[i] - mu[i], a[i], (double)beta[i]);
        }
        with_act(p.act, [&](auto act) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                float o, d;
                act_both<decltype(act)::value>(z[i], o, d);
                z[i] = o;
            }
        });
#pragma unroll
        for (int i = 0; i < V; ++i) out.v[i] = (T)(p.keep ? (k.v[i] ? z[i] * p.scale : 0.0f) : z[i]);
        if (n > 0) store_some<T, V>(y + at, out, n);
        if (p.codes) {
            float amax = 0.0f;
#pragma unroll
            for (int i = 0; i < V; ++i) amax = fmaxf(amax, finite_abs(f[i]));
#pragma unroll
            for (int d = 1; d < LANES; d *= 2) amax = fmaxf(amax, __shfl_xor(amax, d));
            const int e = scale_byte(amax);
            Pack<int8_t, V> q;
#pragma unroll
            for (int i = 0; i < V; ++i) q.v[i] = eight_code(f[i], e);
            if (n > 0) {
                store_some<int8_t, V>(p.codes + at, q, n);
                if ((col & 31) == 0) p.scales[r * nb + col / 32] = (uint8_t)e;
            }
        }
    }
}

template <int V>
__device__ __forceinline__ void column_affine(const NormArgs &p, int64_t col, int n, double (&mu)[V], double (&a)[V], float (&beta)[V])
{
#pragma unroll
    for (int i = 0; i < V; ++i) {
        mu[i] = a[i] = 0.0;
        beta[i] = 0.0f;
        if (i < n) {
            mu[i] = p.stats[col + i];
            a[i] = (double)p.gamma[col + i] * p.stats[p.N + col + i];
            beta[i] = p.beta[col + i];
        }
    }
}

constexpr int WIDE = 16;       // TX of the chunked kernels

template <class T>
__global__ __launch_bounds__(THREADS) void stats_kernel(NormArgs p, const T *__restrict__ x)
{
    constexpr int V = Vec<T>::N, TX = WIDE;
    __shared__ double lds[THREADS / TX / 2 * TX * V * 2];
    const int tx = threadIdx.x % TX, ty = threadIdx.x / TX;
    const int64_t col = ((int64_t)blockIdx.x * TX + tx) * V;
    const int n = (int)(p.N - col < V ? p.N - col : V);
    const int64_t r0 = (int64_t)blockIdx.y * p.rows_per, r1 = r0 + p.rows_per < p.M ? r0 + p.rows_per : p.M;
    double s1[V], s2[V];
    sum_x<T, V, TX>(p, x, r0, r1, col, n, ty, s1, s2);
    reduce_rows<V, TX>(s1, s2, lds, tx, ty);
    if (ty == 0) {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i < n) {
                double *o = p.partial + ((int64_t)blockIdx.y * p.N + col + i) * 2;
                o[0] = s1[i];
                o[1] = s2[i];
            }
    }
}

// 16 columns a workgroup, 16 threads each over the chunks
template <bool FORWARD>
__global__ __launch_bounds__(THREADS) void finish_kernel(NormArgs p)
{
    __shared__ double lds[16][16][2];
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    const int64_t col = (int64_t)blockIdx.x * 16 + tx;
    double a = 0.0, b = 0.0;
    if (col < p.N)
        for (int64_t c = ty; c < p.chunks; c += 16) {
            a += p.partial[(c * p.N + col) * 2];
            b += p.partial[(c * p.N + col) * 2 + 1];
        }
    lds[ty][tx][0] = a;
    lds[ty][tx][1] = b;
    __syncthreads();
    if (ty == 0 && col < p.N) {
        for (int i = 1; i < 16; ++i) {
            a += lds[i][tx][0];
            b += lds[i][tx][1];
        }
        if (FORWARD) {
            double mu, rstd;
            finish_stats(p, col, a, b, mu, rstd);
        } else {
            p.dbeta[col] = (float)a;
            p.dgamma[col] = (float)b;
            p.means[col] = a / (double)p.M;
            p.means[p.N + col] = b / (double)p.M;
        }
    }
}

template <class T>
__global__ __launch_bounds__(THREADS) void apply_kernel(NormArgs p, const T *__restrict__ x, T *__restrict__ y)
{
    constexpr int V = Vec<T>::N, TX = WIDE;
    const int tx = threadIdx.x % TX, ty = threadIdx.x / TX;
    const int64_t col = ((int64_t)blockIdx.x * TX + tx) * V;
    const int n = (int)(p.N - col < V ? p.N - col : V);
    const int64_t r0 = (int64_t)blockIdx.y * p.rows_per, r1 = r0 + p.rows_per < p.M ? r0 + p.rows_per : p.M;
    double mu[V], a[V];
    float beta[V];
    column_affine<V>(p, col, n, mu, a, beta);
    apply_rows<T, V, TX>(p, x, y, r0, r1, col, n, ty, mu, a, beta);
}

// A batch of few rows: one workgroup does 32 columns from the sums to the outputs, in one launch.
template <class T>
__global__ __launch_bounds__(THREADS) void small_forward_kernel(NormArgs p, const T *__restrict__ x, T *__restrict__ y)
{
    constexpr int V = Vec<T>::N, TX = 32 / V;
    __shared__ double lds[THREADS / TX / 2 * TX * V * 2];
    const int tx = threadIdx.x % TX, ty = threadIdx.x / TX;
    const int64_t col = ((int64_t)blockIdx.x * TX + tx) * V;
    const int n = (int)(p.N - col < V ? p.N - col : V);
    double s1[V], s2[V];
    sum_x<T, V, TX>(p, x, 0, p.M, col, n, ty, s1, s2);
    reduce_rows<V, TX>(s1, s2, lds, tx, ty);
    if (ty == 0) {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i < n) {
                double mu, rstd;
                finish_stats(p, col + i, s1[i], s2[i], mu, rstd);
                lds[(tx * V + i) * 2] = mu;
                lds[(tx * V + i) * 2 + 1] = (double)p.gamma[col + i] * rstd;
            }
    }
    __syncthreads();
    double mu[V], a[V];
    float beta[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        mu[i] = i < n ? lds[(tx * V + i) * 2] : 0.0;
        a[i] = i < n ? lds[(tx * V + i) * 2 + 1] : 0.0;
        beta[i] = i < n ? p.beta[col + i] : 0.0f;
    }
    apply_rows<T, V, TX>(p, x, y, 0, p.M, col, n, ty, mu, a, beta);
}

// ---- backward --------------------------------------------------------------------------------
template <int V> struct Column { double mu[V], rstd[V]; float gamma[V], beta[V]; };

template <int V>
__device__ __forceinline__ void column_back(const NormArgs &p, int64_t col, int n, Column<V> &k)
{
#pragma unroll
    for (int i = 0; i < V; ++i) {
        k.mu[i] = k.rstd[i] = 0.0;
        k.gamma[i] = k.beta[i] = 0.0f;
        if (i < n) {
            k.mu[i] = p.stats[col + i];
            k.rstd[i] = p.stats[p.N + col + i];
            k.gamma[i] = p.gamma[col + i];
            k.beta[i] = p.beta[col + i];
        }
    }
}

// g and h of V elements of a row
template <class T, int V, bool EIGHT>
__device__ __forceinline__ void g_and_h(const NormArgs &p, const T *__restrict__ x, const T *__restrict__ dy, int64_t r, int64_t nb,
                                        int64_t col, int n, const Column<V> &k, float (&g)[V], float (&h)[V])
{
    const int64_t at = r * p.N + col;
    const Pack<T, V> d = load_some<T, V>(dy + at, n);
    Pack<uint8_t, V> m;
    if (p.keep) m = load_some<uint8_t, V>(p.keep + at, n);
    float f[V], z[V];
    if (EIGHT) {
        const Pack<int8_t, V> q = load_some<int8_t, V>(p.codes + at, n);
        const int e = p.scales[r * nb + col / 32];
#pragma unroll
        for (int i = 0; i < V; ++i) f[i] = eight_value(q.v[i], e);
    } else {
        const Pack<T, V> v = load_some<T, V>(x + at, n);
#pragma unroll
        for (int i = 0; i < V; ++i) f[i] = (float)v.v[i];
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const double hd = ((double)f[i] - k.mu[i]) * k.rstd[i];
        h[i] = (float)hd;
        g[i] = (float)d.v[i];
        z[i] = (float)__builtin_fma(hd, (double)k.gamma[i], (double)k.beta[i]);
    }
    if (p.act != AFIV_ACT_NONE)
        with_act(p.act, [&](auto act) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                float f, d;
                act_both<decltype(act)::value>(z[i], f, d);
                g[i] *= d;
            }
        });
    if (p.keep) {
#pragma unroll
        for (int i = 0; i < V; ++i) g[i] = m.v[i] ? g[i] * p.scale : 0.0f;
    }
}

template <class T, int V, int TX, bool EIGHT>
__device__ __forceinline__ void sum_g(const NormArgs &p, const T *__restrict__ x, const T *__restrict__ dy, int64_t r0, int64_t r1,
                                      int64_t col, int n, int ty, const Column<V> &k, double (&s1)[V], double (&s2)[V])
{
    constexpr int TY = THREADS / TX;
    const int64_t nb = (p.N + 31) / 32;
#pragma unroll
    for (int i = 0; i < V; ++i) s1[i] = s2[i] = 0.0;
    if (n <= 0) return;
#pragma unroll 2
    for (int64_t r = r0 + ty; r < r1; r += TY) {
        float g[V], h[V];
        g_and_h<T, V, EIGHT>(p, x, dy, r, nb, col, n, k, g, h);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            s1[i] += (double)g[i];
            s2[i] = __builtin_fma((double)g[i], (double)h[i], s2[i]);
        }
    }
}

// mb = dbeta / M, mg = dgamma / M
template <class T, int V, int TX, bool EIGHT>
__device__ __forceinline__ void back_rows(const NormArgs &p, const T *__restrict__ x, const T *__restrict__ dy, T *__restrict__ dx,
                                          int64_t r0, int64_t r1, int64_t col, int n, int ty, const Column<V> &k, const float (&mb)[V],
                                          const float (&mg)[V])
{
    constexpr int TY = THREADS / TX;
    const int64_t nb = (p.N + 31) / 32;
    if (n <= 0) return;
#pragma unroll 2
    for (int64_t r = r0 + ty; r < r1; r += TY) {
        float g[V], h[V];
        g_and_h<T, V, EIGHT>(p, x, dy, r, nb, col, n, k, g, h);
        Pack<T, V> o;
#pragma unroll
        for (int i = 0; i < V; ++i) o.v[i] = (T)((float)(k.gamma[i] * k.rstd[i]) * (g[i] - mb[i] - h[i] * mg[i]));
        store_some<T, V>(dx + r * p.N + col, o, n);
    }
}

template <class T, bool EIGHT>
__global__ __launch_bounds__(THREADS) void back_sums_kernel(NormArgs p, const T *__restrict__ x, const T *__restrict__ dy)
{
    constexpr int V = Vec<T>::N, TX = WIDE;
    __shared__ double lds[THREADS / TX / 2 * TX * V * 2];
    const int tx = threadIdx.x % TX, ty = threadIdx.x / TX;
    const int64_t col = ((int64_t)blockIdx.x * TX + tx) * V;
    const int n = (int)(p.N - col < V ? p.N - col : V);
    const int64_t r0 = (int64_t)blockIdx.y * p.rows_per, r1 = r0 + p.rows_per < p.M ? r0 + p.rows_per : p.M;
    Column<V> k;
    column_back<V>(p, col, n, k);
    double s1[V], s2[V];
    sum_g<T, V, TX, EIGHT>(p, x, dy, r0, r1, col, n, ty, k, s1, s2);
    reduce_rows<V, TX>(s1, s2, lds, tx, ty);
    if (ty == 0) {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i < n) {
                double *o = p.partial + ((int64_t)blockIdx.y * p.N + col + i) * 2;
                o[0] = s1[i];
                o[1] = s2[i];
            }
    }
}

template <class T, bool EIGHT>
__global__ __launch_bounds__(THREADS) void back_dx_kernel(NormArgs p, const T *__restrict__ x, const T *__restrict__ dy, T *__restrict__ dx)
{
    constexpr int V = Vec<T>::N, TX = WIDE;
    const int tx = threadIdx.x % TX, ty = threadIdx.x / TX;
    const int64_t col = ((int64_t)blockIdx.x * TX + tx) * V;
    const int n = (int)(p.N - col < V ? p.N - col : V);
    const int64_t r0 = (int64_t)blockIdx.y * p.rows_per, r1 = r0 + p.rows_per < p.M ? r0 + p.rows_per : p.M;
    Column<V> k;
    column_back<V>(p, col, n, k);
    float mb[V], mg[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        mb[i] = i < n ? (float)p.means[col + i] : 0.0f;
        mg[i] = i < n ? (float)p.means[p.N + col + i] : 0.0f;
    }
    back_rows<T, V, TX, EIGHT>(p, x, dy, dx, r0, r1, col, n, ty, k, mb, mg);
}

template <class T, bool EIGHT>
__global__ __launch_bounds__(THREADS) void small_backward_kernel(NormArgs p, const T *__restrict__ x, const T *__restrict__ dy,
                                                                 T *__restrict__ dx)
{
    constexpr int V = Vec<T>::N, TX = 32 / V;
    __shared__ double lds[THREADS / TX / 2 * TX * V * 2];
    const int tx = threadIdx.x % TX, ty = threadIdx.x / TX;
    const int64_t col = ((int64_t)blockIdx.x * TX + tx) * V;
    const int n = (int)(p.N - col < V ? p.N - col : V);
    Column<V> k;
    column_back<V>(p, col, n, k);
    double s1[V], s2[V];
    sum_g<T, V, TX, EIGHT>(p, x, dy, 0, p.M, col, n, ty, k, s1, s2);
    reduce_rows<V, TX>(s1, s2, lds, tx, ty);
    if (ty == 0) {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i < n) {
                p.dbeta[col + i] = (float)s1[i];
                p.dgamma[col + i] = (float)s2[i];
                lds[(tx * V + i) * 2] = s1[i] / (double)p.M;
                lds[(tx * V + i) * 2 + 1] = s2[i] / (double)p.M;
            }
    }
    __syncthreads();
    if (!dx) return;
    float mb[V], mg[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        mb[i] = i < n ? (float)lds[(tx * V + i) * 2] : 0.0f;
        mg[i] = i < n ? (float)lds[(tx * V + i) * 2 + 1] : 0.0f;
    }
    back_rows<T, V, TX, EIGHT>(p, x, dy, dx, 0, p.M, col, n, ty, k, mb, mg);
}

// Rows up to which one launch of N/32 workgroups is taken instead of three.
constexpr int64_t SMALL_ROWS = 1024;

// row chunks of the chunked kernels: enough workgroups for eight waves a SIMD, at least 16 rows each
int64_t chunks_for(int64_t M, int64_t col_blocks)
{
    int64_t c = (2048 + col_blocks - 1) / col_blocks;
    if (c > AFIV_NORM_CHUNKS) c = AFIV_NORM_CHUNKS;
    if (c > (M + 15) / 16) c = (M + 15) / 16;
    return c < 1 ? 1 : c;
}

int ok() { return hipGetLastError() == hipSuccess ? AFIV_OK : AFIV_E_HIP; }

template <class T>
int forward(NormArgs p, const void *xv, void *yv, hipStream_t s)
{
    const T *x = (const T *)xv;
    T *y = (T *)yv;
    if (p.M <= SMALL_ROWS) {
        hipLaunchKernelGGL(small_forward_kernel<T>, dim3((unsigned)((p.N + 31) / 32)), dim3(THREADS), 0, s, p, x, y);
        return ok();
    }
    const int64_t cb = (p.N + WIDE * Vec<T>::N - 1) / (WIDE * Vec<T>::N);
    p.chunks = chunks_for(p.M, cb);
    p.rows_per = (p.M + p.chunks - 1) / p.chunks;
    const dim3 grid((unsigned)cb, (unsigned)p.chunks);
    hipLaunchKernelGGL(stats_kernel<T>, grid, dim3(THREADS), 0, s, p, x);
    hipLaunchKernelGGL(finish_kernel<true>, dim3((unsigned)((p.N + 15) / 16)), dim3(THREADS), 0, s, p);
    hipLaunchKernelGGL(apply_kernel<T>, grid, dim3(THREADS), 0, s, p, x, y);
    return ok();
}

template <class T, bool EIGHT>
int backward(NormArgs p, const void *xv, const void *dyv, void *dxv, hipStream_t s)
{
    const T *x = (const T *)xv, *dy = (const T *)dyv;
    T *dx = (T *)dxv;
    if (p.M <= SMALL_ROWS) {
        hipLaunchKernelGGL((small_backward_kernel<T, EIGHT>), dim3((unsigned)((p.N + 31) / 32)), dim3(THREADS), 0, s, p, x, dy, dx);
        return ok();
    }
    const int64_t cb = (p.N + WIDE * Vec<T>::N - 1) / (WIDE * Vec<T>::N);
    p.chunks = chunks_for(p.M, cb);
    p.rows_per = (p.M + p.chunks - 1) / p.chunks;
    const dim3 grid((unsigned)cb, (unsigned)p.chunks);
    hipLaunchKernelGGL((back_sums_kernel<T, EIGHT>), grid, dim3(THREADS), 0, s, p, x, dy);
    hipLaunchKernelGGL(finish_kernel<false>, dim3((unsigned)((p.N + 15) / 16)), dim3(THREADS), 0, s, p);
    if (dx) hipLaunchKernelGGL((back_dx_kernel<T, EIGHT>), grid, dim3(THREADS), 0, s, p, x, dy, dx);
    return ok();
}

}  // namespace

int afiv_launch_norm_act(const void *x, const float *gamma, const float *beta, const uint8_t *keep, int dtype, int act, int64_t M,
                         int64_t N, double eps, double momentum, double drop_p, float *run_mean, float *run_var, void *y, double *stats,
                         int8_t *codes, uint8_t *scales, double *scratch, hipStream_t s)
{
    NormArgs p = {};
    p.M = M; p.N = N; p.act = act; p.eps = eps; p.momentum = momentum;
    p.scale = (float)(1.0 / (1.0 - drop_p));
    p.gamma = gamma; p.beta = beta; p.keep = keep; p.run_mean = run_mean; p.run_var = run_var;
    p.stats = stats; p.partial = scratch; p.codes = codes; p.scales = scales;
    if (dtype == AFIV_F32) return forward<float>(p, x, y, s);
    if (dtype == AFIV_BF16) return forward<__bf16>(p, x, y, s);
    return forward<_Float16>(p, x, y, s);
}

int afiv_launch_norm_act_backward(const void *dy, const void *x, const int8_t *codes, const uint8_t *scales, const float *gamma,
                                  const float *beta, const uint8_t *keep, const double *stats, int dtype, int act, int64_t M, int64_t N,
                                  double drop_p, void *dx, float *dgamma, float *dbeta, double *scratch, hipStream_t s)
{
    NormArgs p = {};
    p.M = M; p.N = N; p.act = act;
    p.scale = (float)(1.0 / (1.0 - drop_p));
    p.gamma = gamma; p.beta = beta; p.keep = keep;
    p.stats = const_cast<double *>(stats);                       // read only in this direction
    p.partial = scratch;
    p.means = scratch + (int64_t)AFIV_NORM_CHUNKS * N * 2;
    p.codes = const_cast<int8_t *>(codes);
    p.scales = const_cast<uint8_t *>(scales);
    p.dgamma = dgamma; p.dbeta = dbeta;
    if (codes) {
        if (dtype == AFIV_F32) return backward<float, true>(p, x, dy, dx, s);
        if (dtype == AFIV_BF16) return backward<__bf16, true>(p, x, dy, dx, s);
        return backward<_Float16, true>(p, x, dy, dx, s);
    }
    if (dtype == AFIV_F32) return backward<float, false>(p, x, dy, dx, s);
    if (dtype == AFIV_BF16) return backward<__bf16, false>(p, x, dy, dx, s);
    return backward<_Float16, false>(p, x, dy, dx, s);
}
