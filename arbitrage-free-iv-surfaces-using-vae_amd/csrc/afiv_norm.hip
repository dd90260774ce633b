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
// 131072 x 1024 in BF16 with dropout and an 8-bit checkpoint: statistics 68 us (3.9 TB/s), outputs 164 us (4.9 TB/s),
// backward sums 168 us (3.2 TB/s), dx 183 us (4.4 TB/s); a copy reaches 4.95.  64 x 128: 7.2 and 6.4 us, one launch each.
//
// Statistics are FP64 sums of d = x - x0 and d^2, x0 = the column's first element: var = E[d^2] - E[d]^2 then cancels
// only as far as x0 lies from the mean (without the shift a column of mean 1e5 and variance 1 lost five
// digits, and showed it in FP32 outputs).  What follows is FP32 on mu split into two
// parts, h = ((x - mu1) - mu2) rstd: x and mu1 are exact, so nothing is lost where they cancel, and h is within a few
// roundings of its own size (all of it in FP64 took twice the registers and, with its conversions, twice
// the time).  relu's derivative jumps at zero, so there a pre-activation within 2^-20 |beta| of zero, that is,
// within reach of its rounding, is taken again in FP64, and its side is right to 1e-16.
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

// Rows come in groups of four (or two): their loads are issued together, so that a wave has several rows in flight (a row
// at a time left HBM at 1.5 TB/s).  FULL: the workgroup's lanes have all V of their columns, or none.  Otherwise all of
// them load as the ragged one must, without branches: its own way, row by row, held the others up (131072 x 299, bf16,
// backward 307 -> 226 us).

template <bool FULL, class E, int V>
__device__ __forceinline__ Pack<E, V> take(const NormArgs &a, const E *p, int n)
{
    if constexpr (FULL) return load_pack<E, V>(p);
    else return load_ending<E, V>(p, n, a.N >= V);
}
template <bool FULL, class E, int V>
__device__ __forceinline__ void give(E *p, const Pack<E, V> &v, int n)
{
    if constexpr (FULL) store_pack<E, V>(p, v);
    else store_some<E, V>(p, v, n);
}

// calls f(first row, rows) for the rows r0 + ty, + TY, ... below r1, U at a time and then one by one
template <bool FULL, int TY, class F>
__device__ __forceinline__ void each_group(int64_t r0, int64_t r1, int ty, F &&f)
{
    int64_t r = r0 + ty;
    constexpr int U = FULL ? 4 : 2;                 // moving a ragged row's elements into place takes registers
    for (; r + (U - 1) * TY < r1; r += U * TY) f(r, std::integral_constant<int, U>());
    for (; r < r1; r += TY) f(r, std::integral_constant<int, 1>());
}

// Threads stand as TX lanes across columns (V elements each) by TY rows.  Sums of a column over the TY rows of the
// workgroup, in a fixed order: among a wave's rows by exchanges, then over the waves in LDS.  Result at the threads
// of row 0.
constexpr int SUMS_LDS = THREADS / 64;                 // doubles of LDS for each of a column's two sums

template <int V, int TX>
__device__ __forceinline__ void reduce_rows(double (&a)[V], double (&b)[V], double *lds, int tx, int ty)
{
    constexpr int WAVES = THREADS / 64, W = TX * V;
#pragma unroll
    for (int d = TX; d < 64; d *= 2)
#pragma unroll
        for (int i = 0; i < V; ++i) {
            a[i] += __shfl_xor(a[i], d);
            b[i] += __shfl_xor(b[i], d);
        }
    const int wave = threadIdx.x / 64;
    if (threadIdx.x % 64 < TX) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            lds[(wave * W + tx * V + i) * 2] = a[i];
            lds[(wave * W + tx * V + i) * 2 + 1] = b[i];
        }
    }
    __syncthreads();
    if (ty == 0) {
#pragma unroll
        for (int w = 1; w < WAVES; ++w)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                a[i] += lds[(w * W + tx * V + i) * 2];
                b[i] += lds[(w * W + tx * V + i) * 2 + 1];
            }
    }
    __syncthreads();
}

template <bool FULL, class T, int V, int TX>
__device__ __forceinline__ void sum_x(const NormArgs &p, const T *__restrict__ x, int64_t r0, int64_t r1, int64_t col, int n,
                                      int ty, double (&s1)[V], double (&s2)[V])
{
    constexpr int TY = THREADS / TX;
#pragma unroll
    for (int i = 0; i < V; ++i) s1[i] = s2[i] = 0.0;
    if (n <= 0) return;
    const Pack<T, V> x0 = take<FULL, T, V>(p, x + col, n);
    each_group<FULL, TY>(r0, r1, ty, [&](int64_t r, auto rows) {
        constexpr int U = decltype(rows)::value;
        Pack<T, V> v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = take<FULL, T, V>(p, x + (r + u * TY) * p.N + col, n);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const double d = (double)(float)v[u].v[i] - (double)(float)x0.v[i];
                s1[i] += d;
                s2[i] = __builtin_fma(d, d, s2[i]);
            }
    });
}

// statistics of one column from its sums and first element
__device__ __forceinline__ void finish_stats(const NormArgs &p, int64_t col, double s1, double s2, double x0, double &mu, double &rstd)
{
    const double m = (double)p.M, e = s1 / m;
    mu = x0 + e;
    const double d = s2 / m - e * e;
    const double var = d < 0.0 ? 0.0 : d;                 // NaN stays NaN
    rstd = 1.0 / sqrt(var + p.eps);
    p.stats[col] = mu;
    p.stats[p.N + col] = rstd;
    if (p.run_mean) {
        p.run_mean[col] = (float)((1.0 - p.momentum) * (double)p.run_mean[col] + p.momentum * mu);
        p.run_var[col] = (float)((1.0 - p.momentum) * (double)p.run_var[col] + p.momentum * (var * (m / (m - 1.0))));
    }
}

// what a thread holds of its V columns
template <int V> struct Column { float mu1[V], mu2[V], rstd[V], gamma[V], beta[V]; };

__device__ __forceinline__ void set_column(float &mu1, float &mu2, float &rstd, double mu, double r)
{
    mu1 = (float)mu;
    mu2 = (float)(mu - (double)mu1);
    rstd = (float)r;
}

template <int V>
__device__ __forceinline__ void columns(const NormArgs &p, int64_t col, int n, Column<V> &k)
{
#pragma unroll
    for (int i = 0; i < V; ++i) {
        k.mu1[i] = k.mu2[i] = k.rstd[i] = k.gamma[i] = k.beta[i] = 0.0f;
        if (i < n) {
            set_column(k.mu1[i], k.mu2[i], k.rstd[i], p.stats[col + i], p.stats[p.N + col + i]);
            k.gamma[i] = p.gamma[col + i];
            k.beta[i] = p.beta[col + i];
        }
    }
}

// h and the pre-activation z of V elements f.  sides: z's sign matters
template <int V>
__device__ __forceinline__ void normalise(const NormArgs &p, const float (&f)[V], int64_t col, int n, const Column<V> &k, bool sides, float (&h)[V],
                                          float (&z)[V])
{
    bool near = false;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        h[i] = ((f[i] - k.mu1[i]) - k.mu2[i]) * k.rstd[i];
        z[i] = __builtin_fmaf(h[i], k.gamma[i], k.beta[i]);
        near |= fabsf(z[i]) <= 0x1p-20f * fabsf(k.beta[i]);
    }
    if (sides && near) {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i < n) z[i] = (float)__builtin_fma(((double)f[i] - p.stats[col + i]) * p.stats[p.N + col + i], (double)k.gamma[i], (double)k.beta[i]);
    }
}

// outputs (and the checkpoint) of rows r0..r1 at columns col..col+n.  Lanes behind the last column are
// among those that find a checkpoint block's largest magnitude: they take the last lane's columns and store nothing.
template <bool FULL, class T, int V, int TX>
__device__ __forceinline__ void apply_rows(const NormArgs &p, const T *__restrict__ x, T *__restrict__ y, int64_t r0, int64_t r1,
                                           int64_t col, int n, int ty, const Column<V> &c, bool mine)
{
    constexpr int TY = THREADS / TX, LANES = 32 / V;        // lanes of a checkpoint block
    const int64_t nb = (p.N + 31) / 32;
    with_act(p.act, [&](auto act) {
        each_group<FULL, TY>(r0, r1, ty, [&](int64_t r, auto rows) {
            constexpr int U = decltype(rows)::value;
            Pack<T, V> v[U];
            Pack<uint8_t, V> k[U];
#pragma unroll
            for (int u = 0; u < U; ++u) v[u] = take<FULL, T, V>(p, x + (r + u * TY) * p.N + col, n);
            if (p.keep) {
#pragma unroll
                for (int u = 0; u < U; ++u) k[u] = take<FULL, uint8_t, V>(p, p.keep + (r + u * TY) * p.N + col, n);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t at = (r + u * TY) * p.N + col;
                Pack<T, V> out;
                float f[V], h[V], z[V];
#pragma unroll
                for (int i = 0; i < V; ++i) f[i] = (float)v[u].v[i];
                normalise<V>(p, f, col, n, c, false, h, z);             // f itself does not jump
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    float o, d;
                    act_both<decltype(act)::value>(z[i], o, d);
                    out.v[i] = (T)(p.keep ? (k[u].v[i] ? o * p.scale : 0.0f) : o);
                }
                if (mine) give<FULL, T, V>(y + at, out, n);
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
                    if (mine) {
                        give<FULL, int8_t, V>(p.codes + at, q, n);
                        if ((col & 31) == 0) p.scales[(r + u * TY) * nb + col / 32] = (uint8_t)e;
                    }
                }
            }
        });
    });
}

constexpr int WIDE = 16;       // TX of the chunked kernels

template <class T>
__global__ __launch_bounds__(THREADS) void stats_kernel(NormArgs p, const T *__restrict__ x)
{
    constexpr int V = Vec<T>::N, TX = WIDE;
    __shared__ double lds[SUMS_LDS * TX * V * 2];
    const int tx = threadIdx.x % TX, ty = threadIdx.x / TX;
    const int64_t col = ((int64_t)blockIdx.x * TX + tx) * V;
    const int n = (int)(p.N - col < V ? p.N - col : V);
    const bool whole = p.N % V == 0 || (int64_t)(blockIdx.x + 1) * TX * V <= p.N;
    const int64_t r0 = (int64_t)blockIdx.y * p.rows_per, r1 = r0 + p.rows_per < p.M ? r0 + p.rows_per : p.M;
    double s1[V], s2[V];
    if (whole) sum_x<true, T, V, TX>(p, x, r0, r1, col, n, ty, s1, s2);
    else sum_x<false, T, V, TX>(p, x, r0, r1, col, n, ty, s1, s2);
    reduce_rows<V, TX>(s1, s2, lds, tx, ty);
    if (ty == 0) {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i < n) {
                double *o = p.partial + ((int64_t)blockIdx.y * p.N + col + i) * 2;
                o[0] = s1[i];
                o[1] = s2[i];
                if (blockIdx.y == 0) p.stats[col + i] = (double)(float)x[col + i];      // for finish_kernel
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
            finish_stats(p, col, a, b, p.stats[col], mu, rstd);
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
    const int64_t first = ((int64_t)blockIdx.x * TX + tx) * V;
    const bool mine = first < p.N;
    const int64_t col = mine ? first : (p.N - 1) / V * V;
    const int n = (int)(p.N - col < V ? p.N - col : V);
    const bool whole = p.N % V == 0;
    const int64_t r0 = (int64_t)blockIdx.y * p.rows_per, r1 = r0 + p.rows_per < p.M ? r0 + p.rows_per : p.M;
    Column<V> k;
    columns<V>(p, col, n, k);
    if ((int64_t)(blockIdx.x + 1) * TX * V <= p.N) apply_rows<true, T, V, TX>(p, x, y, r0, r1, col, n, ty, k, true);      // no guards
    else if (whole) apply_rows<true, T, V, TX>(p, x, y, r0, r1, col, n, ty, k, mine);
    else apply_rows<false, T, V, TX>(p, x, y, r0, r1, col, n, ty, k, mine);
}

// A batch of few rows: one workgroup does 32 columns from the sums to the outputs, in one launch.
template <class T>
__global__ __launch_bounds__(THREADS) void small_forward_kernel(NormArgs p, const T *__restrict__ x, T *__restrict__ y)
{
    constexpr int V = Vec<T>::N, TX = 32 / V;
    __shared__ double lds[SUMS_LDS * TX * V * 2];
    const int tx = threadIdx.x % TX, ty = threadIdx.x / TX;
    const int64_t first = ((int64_t)blockIdx.x * TX + tx) * V;
    const bool mine = first < p.N;
    const int64_t col = mine ? first : (p.N - 1) / V * V;
    const int n = (int)(p.N - col < V ? p.N - col : V);
    const bool whole = p.N % V == 0 || (int64_t)(blockIdx.x + 1) * TX * V <= p.N;
    double s1[V], s2[V];
    if (whole) sum_x<true, T, V, TX>(p, x, 0, p.M, col, n, ty, s1, s2);
    else sum_x<false, T, V, TX>(p, x, 0, p.M, col, n, ty, s1, s2);
    reduce_rows<V, TX>(s1, s2, lds, tx, ty);
    if (ty == 0 && mine) {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i < n) {
                double mu, rstd;
                finish_stats(p, col + i, s1[i], s2[i], (double)(float)x[col + i], mu, rstd);
                lds[(tx * V + i) * 2] = mu;
                lds[(tx * V + i) * 2 + 1] = rstd;
            }
    }
    __syncthreads();
    Column<V> k;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        k.mu1[i] = k.mu2[i] = k.rstd[i] = k.gamma[i] = k.beta[i] = 0.0f;
        if (i < n) {
            set_column(k.mu1[i], k.mu2[i], k.rstd[i], lds[(tx * V + i) * 2], lds[(tx * V + i) * 2 + 1]);
            k.gamma[i] = p.gamma[col + i];
            k.beta[i] = p.beta[col + i];
        }
    }
    if ((int64_t)(blockIdx.x + 1) * TX * V <= p.N) apply_rows<true, T, V, TX>(p, x, y, 0, p.M, col, n, ty, k, true);      // no guards
    else if (whole) apply_rows<true, T, V, TX>(p, x, y, 0, p.M, col, n, ty, k, mine);
    else apply_rows<false, T, V, TX>(p, x, y, 0, p.M, col, n, ty, k, mine);
}

// ---- backward --------------------------------------------------------------------------------
// what the backward pass reads of U rows, TY apart
template <class T, int V, bool EIGHT, int U>
struct BackRows {
    Pack<T, V> d[U], x[EIGHT ? 1 : U];
    Pack<uint8_t, V> k[U];
    Pack<int8_t, V> q[EIGHT ? U : 1];
    uint8_t e[U];

    template <bool FULL>
    __device__ __forceinline__ void load(const NormArgs &p, const T *__restrict__ xs, const T *__restrict__ dy, int64_t r, int ty_step, int64_t nb,
                                         int64_t col, int n)
    {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t row = r + u * ty_step, at = row * p.N + col;
            d[u] = take<FULL, T, V>(p, dy + at, n);
            if constexpr (EIGHT) {
                q[u] = take<FULL, int8_t, V>(p, p.codes + at, n);
                e[u] = p.scales[row * nb + col / 32];
            } else x[u] = take<FULL, T, V>(p, xs + at, n);
        }
        if (p.keep) {
#pragma unroll
            for (int u = 0; u < U; ++u) k[u] = take<FULL, uint8_t, V>(p, p.keep + (r + u * ty_step) * p.N + col, n);
        }
    }
    // g and h of row u
    template <int ACT>
    __device__ __forceinline__ void g_and_h(const NormArgs &p, int u, int64_t col, int n, const Column<V> &c, float (&g)[V], float (&h)[V]) const
    {
        float f[V], z[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            if constexpr (EIGHT) f[i] = eight_value(q[u].v[i], e[u]);
            else f[i] = (float)x[u].v[i];
        }
        normalise<V>(p, f, col, n, c, ACT == AFIV_ACT_RELU || ACT == AFIV_ACT_LEAKY_RELU, h, z);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            float y, s;
            act_both<ACT>(z[i], y, s);
            g[i] = ACT == AFIV_ACT_NONE ? (float)d[u].v[i] : (float)d[u].v[i] * s;
            if (p.keep) g[i] = k[u].v[i] ? g[i] * p.scale : 0.0f;
        }
    }
};

template <bool FULL, class T, int V, int TX, bool EIGHT>
__device__ __forceinline__ void sum_g(const NormArgs &p, const T *__restrict__ x, const T *__restrict__ dy, int64_t r0, int64_t r1,
                                      int64_t col, int n, int ty, const Column<V> &c, double (&s1)[V], double (&s2)[V])
{
    constexpr int TY = THREADS / TX;
    const int64_t nb = (p.N + 31) / 32;
#pragma unroll
    for (int i = 0; i < V; ++i) s1[i] = s2[i] = 0.0;
    if (n <= 0) return;
    with_act(p.act, [&](auto act) {
        each_group<FULL, TY>(r0, r1, ty, [&](int64_t r, auto rows) {
            BackRows<T, V, EIGHT, decltype(rows)::value> b;
            b.template load<FULL>(p, x, dy, r, TY, nb, col, n);
#pragma unroll
            for (int u = 0; u < decltype(rows)::value; ++u) {
                float g[V], h[V];
                b.template g_and_h<decltype(act)::value>(p, u, col, n, c, g, h);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    s1[i] += (double)g[i];
                    s2[i] = __builtin_fma((double)g[i], (double)h[i], s2[i]);
                }
            }
        });
    });
}

// mb = dbeta / M, mg = dgamma / M
template <bool FULL, class T, int V, int TX, bool EIGHT>
__device__ __forceinline__ void back_rows(const NormArgs &p, const T *__restrict__ x, const T *__restrict__ dy, T *__restrict__ dx,
                                          int64_t r0, int64_t r1, int64_t col, int n, int ty, const Column<V> &c, const float (&mb)[V],
                                          const float (&mg)[V])
{
    constexpr int TY = THREADS / TX;
    const int64_t nb = (p.N + 31) / 32;
    if (n <= 0) return;
    with_act(p.act, [&](auto act) {
        each_group<FULL, TY>(r0, r1, ty, [&](int64_t r, auto rows) {
            BackRows<T, V, EIGHT, decltype(rows)::value> b;
            b.template load<FULL>(p, x, dy, r, TY, nb, col, n);
#pragma unroll
            for (int u = 0; u < decltype(rows)::value; ++u) {
                float g[V], h[V];
                b.template g_and_h<decltype(act)::value>(p, u, col, n, c, g, h);
                Pack<T, V> o;
#pragma unroll
                for (int i = 0; i < V; ++i) o.v[i] = (T)(c.gamma[i] * c.rstd[i] * (g[i] - mb[i] - h[i] * mg[i]));
                give<FULL, T, V>(dx + (r + u * TY) * p.N + col, o, n);
            }
        });
    });
}

template <class T, bool EIGHT>
__global__ __launch_bounds__(THREADS, 2) void back_sums_kernel(NormArgs p, const T *__restrict__ x, const T *__restrict__ dy)
{
    constexpr int V = Vec<T>::N, TX = WIDE;
    __shared__ double lds[SUMS_LDS * TX * V * 2];
    const int tx = threadIdx.x % TX, ty = threadIdx.x / TX;
    const int64_t col = ((int64_t)blockIdx.x * TX + tx) * V;
    const int n = (int)(p.N - col < V ? p.N - col : V);
    const bool whole = p.N % V == 0 || (int64_t)(blockIdx.x + 1) * TX * V <= p.N;
    const int64_t r0 = (int64_t)blockIdx.y * p.rows_per, r1 = r0 + p.rows_per < p.M ? r0 + p.rows_per : p.M;
    Column<V> k;
    columns<V>(p, col, n, k);
    double s1[V], s2[V];
    if (whole) sum_g<true, T, V, TX, EIGHT>(p, x, dy, r0, r1, col, n, ty, k, s1, s2);
    else sum_g<false, T, V, TX, EIGHT>(p, x, dy, r0, r1, col, n, ty, k, s1, s2);
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
__global__ __launch_bounds__(THREADS, 2) void back_dx_kernel(NormArgs p, const T *__restrict__ x, const T *__restrict__ dy, T *__restrict__ dx)
{
    constexpr int V = Vec<T>::N, TX = WIDE;
    const int tx = threadIdx.x % TX, ty = threadIdx.x / TX;
    const int64_t col = ((int64_t)blockIdx.x * TX + tx) * V;
    const int n = (int)(p.N - col < V ? p.N - col : V);
    const bool whole = p.N % V == 0 || (int64_t)(blockIdx.x + 1) * TX * V <= p.N;
    const int64_t r0 = (int64_t)blockIdx.y * p.rows_per, r1 = r0 + p.rows_per < p.M ? r0 + p.rows_per : p.M;
    Column<V> k;
    columns<V>(p, col, n, k);
    float mb[V], mg[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        mb[i] = i < n ? (float)p.means[col + i] : 0.0f;
        mg[i] = i < n ? (float)p.means[p.N + col + i] : 0.0f;
    }
    if (whole) back_rows<true, T, V, TX, EIGHT>(p, x, dy, dx, r0, r1, col, n, ty, k, mb, mg);
    else back_rows<false, T, V, TX, EIGHT>(p, x, dy, dx, r0, r1, col, n, ty, k, mb, mg);
}

template <class T, bool EIGHT>
__global__ __launch_bounds__(THREADS, 2) void small_backward_kernel(NormArgs p, const T *__restrict__ x, const T *__restrict__ dy,
                                                                 T *__restrict__ dx)
{
    constexpr int V = Vec<T>::N, TX = 32 / V;
    __shared__ double lds[SUMS_LDS * TX * V * 2];
    const int tx = threadIdx.x % TX, ty = threadIdx.x / TX;
    const int64_t col = ((int64_t)blockIdx.x * TX + tx) * V;
    const int n = (int)(p.N - col < V ? p.N - col : V);
    const bool whole = p.N % V == 0 || (int64_t)(blockIdx.x + 1) * TX * V <= p.N;
    Column<V> k;
    columns<V>(p, col, n, k);
    double s1[V], s2[V];
    if (whole) sum_g<true, T, V, TX, EIGHT>(p, x, dy, 0, p.M, col, n, ty, k, s1, s2);
    else sum_g<false, T, V, TX, EIGHT>(p, x, dy, 0, p.M, col, n, ty, k, s1, s2);
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
    if (whole) back_rows<true, T, V, TX, EIGHT>(p, x, dy, dx, 0, p.M, col, n, ty, k, mb, mg);
    else back_rows<false, T, V, TX, EIGHT>(p, x, dy, dx, 0, p.M, col, n, ty, k, mb, mg);
}

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
    if (p.M <= AFIV_NORM_SMALL_ROWS) {
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
    if (p.M <= AFIV_NORM_SMALL_ROWS) {
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
