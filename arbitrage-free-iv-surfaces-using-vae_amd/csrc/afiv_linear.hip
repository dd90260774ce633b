// A linear layer with its epilogue, y = f(x W^T + b) + r, and its backward products, for FP32, BF16
// and FP16.  Replaces nn.Linear (+ activation) of the reference's stacks and their autograd
// (cvae_model.py:64-105), for layers of any width.
//
//   forward    z[m,n] = sum_k x[m,k] W[n,k] + b[n];   y = f(z) + r
//   backward   dz = dy f'(z);   dx = dz W;   dW = dz^T x;   db = sum_m dz
//
// The three products are one tiled kernel: C[i,j] = sum_l A[i,l] B[j,l], where an operand is stored
// along l (x and W forward, dz for dx) or across it (W for dx; dz and x for dW).  Either way it
// lies in LDS along l, 32 steps of l a row of 64 bytes, so one matrix instruction's operand is one
// 16-byte LDS read; operands stored across l are transposed in registers, 4 x 4 elements at a time, on
// their way in.  dz is formed there too (dy, and z or its 8-bit derivative codes), and so is an 8-bit
// x: neither ever exists in memory.
//
// 16-bit types go to v_mfma_f32_16x16x32.  FP32 operands are split into three BF16 parts,
// a = a1 + a2 + a3 (8 bits each, every difference exact), and the six products a1 b1, a1 b2, a2 b1,
// a1 b3, a2 b2, a3 b1 are summed in FP32: what is dropped is 2^-26 of the product, a quarter of an FP32
// rounding, and six BF16 products cost 6/16 of one FP32 matrix instruction's time.  Magnitudes
// of 2^127 and above (infinities too) do not split; a workgroup that has loaded one does its
// tile again with FP32 multiply-adds.  Parts below 2^-133 are lost, that is, an element under 2^-110
// keeps fewer than 24 bits.
//
// Few rows (up to 16) take another kernel: W is read once, straight from memory into the matrix
// instruction, by as many waves as the layer has.
#include "afiv_layer.h"

#include <algorithm>

namespace {

constexpr int THREADS = 256;
constexpr int BK = 32;                    // steps of l in LDS

struct LinArgs {
    // operands: A stored along l [R,L] or across [L,R]; B likewise [C,L] or [L,C]
    const void *A, *B;
    const void *pre;                      // A is dy: z, in the element type, or
    const uint8_t *dcodes;                // its derivative codes (both NULL: dz = dy)
    const int8_t *codes;                  // B is an 8-bit checkpoint
    const uint8_t *scales;
    int64_t R, C, L;
    int act;
    int64_t splits, l_per;                // the sum is cut into `splits` runs of l_per (a multiple of BK)
    // epilogue of C[i,j]: + bias[j], activation (act_out), + residual[i,j]
    const void *bias, *residual;
    int act_out;
    void *out, *pre_out;
    uint8_t *dcodes_out;
    float *partial;                       // splits > 1: [splits,R,C], finished by another kernel
    void *db;                             // dW: db[i] = sum over l of A, by the workgroups of the first tile column
    float *db_partial;                    // splits > 1: [splits,R]
};

enum Kind { ALONG, ALONG_DZ, ACROSS, ACROSS_DZ, ACROSS_EIGHT };
constexpr bool across(Kind k) { return k >= ACROSS; }
constexpr bool is_dz(Kind k) { return k == ALONG_DZ || k == ACROSS_DZ; }

// what a thread holds of an operand between its global loads and its LDS stores: 8 steps of l of one
// row (along) or 4 steps of 4 rows (across)
template <class T, Kind K> struct Held {
    static constexpr int N = across(K) ? 16 : 8;
    Pack<T, (K == ACROSS_EIGHT ? 1 : N)> v;
    Pack<T, (is_dz(K) ? N : 1)> z;                        // z, or the derivative codes in its first bytes
    Pack<int8_t, (K == ACROSS_EIGHT ? 16 : 1)> q;
    uint8_t e[4];
};

template <class T, Kind K>
__device__ __forceinline__ void fetch(const LinArgs &a, const void *base, int64_t R, int64_t row, int64_t l, int64_t l_end, Held<T, K> &h)
{
    if constexpr (!across(K)) {
        const int n = row < R ? (int)(l_end - l < 8 ? l_end - l : 8) : 0;      // may be negative
        if (n <= 0) {
            h.v = {};
            if (is_dz(K)) h.z = {};
            return;
        }
        const int64_t at = row * a.L + l;
        h.v = load_some<T, 8>((const T *)base + at, n);
        if constexpr (is_dz(K)) {
            if (a.pre) h.z = load_some<T, 8>((const T *)a.pre + at, n);
            else if (a.dcodes) {
                const Pack<uint8_t, 8> c = load_some<uint8_t, 8>(a.dcodes + at, n);
                __builtin_memcpy(&h.z, &c, 8);
            }
        }
    } else {
        const int n = (int)(R - row < 4 ? R - row : 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bool in = l + i < l_end && n > 0;
            const int64_t at = (l + i) * R + row;
            if constexpr (K == ACROSS_EIGHT) {
                Pack<int8_t, 4> q = {};
                uint8_t e = 1;
                if (in) {
                    q = load_some<int8_t, 4>(a.codes + at, n);
                    e = a.scales[(l + i) * ((R + 31) / 32) + row / 32];
                }
                __builtin_memcpy(&h.q.v[4 * i], &q, 4);
                h.e[i] = e;
            } else {
                Pack<T, 4> v = {};
                if (in) v = load_some<T, 4>((const T *)base + at, n);
                __builtin_memcpy(&h.v.v[4 * i], &v, sizeof v);
                if constexpr (is_dz(K)) {
                    if (a.pre) {
                        Pack<T, 4> z = {};
                        if (in) z = load_some<T, 4>((const T *)a.pre + at, n);
                        __builtin_memcpy(&h.z.v[4 * i], &z, sizeof z);
                    } else if (a.dcodes) {
                        Pack<uint8_t, 4> c = {};
                        if (in) c = load_some<uint8_t, 4>(a.dcodes + at, n);
                        __builtin_memcpy((char *)&h.z + 4 * i, &c, 4);
                    }
                }
            }
        }
    }
}

// the held elements in FP32
template <class T, Kind K>
__device__ __forceinline__ void values(const LinArgs &a, const Held<T, K> &h, float (&f)[Held<T, K>::N])
{
    constexpr int N = Held<T, K>::N;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if constexpr (K == ACROSS_EIGHT) f[i] = eight_value(h.q.v[i], h.e[i / 4]);
        else f[i] = (float)h.v.v[i];
        if constexpr (is_dz(K)) {
            if (a.pre) f[i] *= act_derivative((float)h.z.v[i], a.act);
            else if (a.dcodes) {
                uint8_t c;
                __builtin_memcpy(&c, (const char *)&h.z + i, 1);
                f[i] *= derivative_of_code(c, a.act);
            }
        }
    }
}

// one element, for the FP32 path of unsplittable tiles
template <class T, Kind K>
__device__ __forceinline__ float element(const LinArgs &a, const void *base, int64_t R, int64_t row, int64_t l)
{
    const int64_t at = across(K) ? l * R + row : row * a.L + l;
    float f;
    if constexpr (K == ACROSS_EIGHT) f = eight_value(a.codes[at], a.scales[l * ((R + 31) / 32) + row / 32]);
    else f = (float)((const T *)base)[at];
    if constexpr (is_dz(K)) {
        if (a.pre) f *= act_derivative((float)((const T *)a.pre)[at], a.act);
        else if (a.dcodes) f *= derivative_of_code(a.dcodes[at], a.act);
    }
    return f;
}

// LDS: row r's 16-byte chunk c (8 steps of l) of a tile stands at chunk c ^ swizzle(r): the 8 rows a
// read touches at once, and the rows 4 apart that a transposing store does, fall on different banks
__device__ __forceinline__ int swizzle(int r) { return ((r >> 1) ^ (r >> 3)) & 3; }
__device__ __forceinline__ int lds_at(int r, int l) { return r * BK + (((l >> 3) ^ swizzle(r)) << 3) + (l & 7); }

template <class T> struct Mma;
template <> struct Mma<__bf16> {
    static constexpr int PARTS = 1;
    typedef bf16x8 frag;
    static __device__ __forceinline__ f32x4 mul(frag a, frag b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <> struct Mma<_Float16> {
    static constexpr int PARTS = 1;
    typedef f16x8 frag;
    static __device__ __forceinline__ f32x4 mul(frag a, frag b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
template <> struct Mma<float> : Mma<__bf16> { static constexpr int PARTS = 3; };

// element type in LDS
template <class T> struct Part { typedef T type; };
template <> struct Part<float> { typedef __bf16 type; };

// N values to consecutive places of each part's plane
template <class T, int N>
__device__ __forceinline__ void put(typename Part<T>::type *lds, int plane, const float (&f)[N])
{
    typedef typename Part<T>::type P;
    if constexpr (Mma<T>::PARTS == 1) {
        Pack<P, N> o;
#pragma unroll
        for (int i = 0; i < N; ++i) o.v[i] = (P)f[i];
        __builtin_memcpy(__builtin_assume_aligned(lds, sizeof o), &o, sizeof o);
    } else {
        Pack<P, N> o[3];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const P a = (P)f[i];
            const float r = f[i] - (float)a;
            const P b = (P)r;
            o[0].v[i] = a;
            o[1].v[i] = b;
            o[2].v[i] = (P)(r - (float)b);
        }
#pragma unroll
        for (int p = 0; p < 3; ++p) __builtin_memcpy(__builtin_assume_aligned(lds + p * plane, sizeof o[0]), &o[p], sizeof o[0]);
    }
}

template <class T, Kind K, int ROWS>
struct Operand {
    // units of work of a tile: 8 steps x 1 row, or 4 steps x 4 rows
    static constexpr int UNITS = across(K) ? (BK / 4) * (ROWS / 4) : (BK / 8) * ROWS;
    static constexpr int PER = (UNITS + THREADS - 1) / THREADS;
    Held<T, K> h[PER];

    static __device__ __forceinline__ void place(int u, int &row, int &l)
    {
        if (across(K)) {                  // neighbouring lanes: neighbouring rows, in pairs of l for the LDS stores
            row = (u % (ROWS / 4)) * 4;
            l = (u / (ROWS / 4)) * 4;
        } else {
            row = u / (BK / 8);
            l = (u % (BK / 8)) * 8;
        }
    }
    __device__ __forceinline__ void load(const LinArgs &a, const void *base, int64_t R, int64_t row0, int64_t l0, int64_t l_end, int tid)
    {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int u = i * THREADS + tid;
            if (UNITS % THREADS == 0 || u < UNITS) {
                int row, l;
                place(u, row, l);
                fetch<T, K>(a, base, R, row0 + row, l0 + l, l_end, h[i]);
            }
        }
    }
    // to LDS; sums[4 i + j]: running sums over l of the four rows of unit i (across only)
    template <bool SUMS>
    __device__ __forceinline__ void store(const LinArgs &a, typename Part<T>::type *lds, int tid, float &amax, float *sums)
    {
        constexpr int N = Held<T, K>::N, PLANE = ROWS * BK;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int u = i * THREADS + tid;
            if (UNITS % THREADS == 0 || u < UNITS) {
                int row, l;
                place(u, row, l);
                float f[N];
                values<T, K>(a, h[i], f);
                if constexpr (Mma<T>::PARTS == 3) {
#pragma unroll
                    for (int j = 0; j < N; ++j) amax = fmaxf(amax, fabsf(f[j]));
                }
                if constexpr (!across(K)) put<T, 8>(lds + lds_at(row, l), PLANE, f);
                else {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float t[4] = {f[j], f[4 + j], f[8 + j], f[12 + j]};
                        put<T, 4>(lds + lds_at(row + j, l), PLANE, t);
                        if (SUMS) sums[4 * i + j] += (t[0] + t[1]) + (t[2] + t[3]);
                    }
                }
            }
        }
    }
};

// C[i, j..j+3] = z, finished: j is a multiple of 4
template <class T>
__device__ __forceinline__ void finish(const LinArgs &a, int64_t i, int64_t j, const float (&z0)[4])
{
    if (!a.out) return;                    // only db was asked for
    const int n = (int)(a.C - j < 4 ? a.C - j : 4);
    const int64_t at = i * a.C + j;
    float z[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) z[q] = z0[q];
    if (a.bias) {
        const Pack<T, 4> b = load_some<T, 4>((const T *)a.bias + j, n);
#pragma unroll
        for (int q = 0; q < 4; ++q) z[q] += (float)b.v[q];
    }
    if (a.pre_out) {
        Pack<T, 4> o;
#pragma unroll
        for (int q = 0; q < 4; ++q) o.v[q] = (T)z[q];
        store_some<T, 4>((T *)a.pre_out + at, o, n);
    }
    if (a.dcodes_out) {
        Pack<uint8_t, 4> o;
#pragma unroll
        for (int q = 0; q < 4; ++q) o.v[q] = derivative_code(z[q], a.act_out);
        store_some<uint8_t, 4>(a.dcodes_out + at, o, n);
    }
    Pack<T, 4> r = {};
    if (a.residual) r = load_some<T, 4>((const T *)a.residual + at, n);
    Pack<T, 4> o;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        float y = act_value(z[q], a.act_out);
        if (a.residual) y += (float)r.v[q];
        o.v[q] = (T)y;
    }
    store_some<T, 4>((T *)a.out + at, o, n);
}

// Tile of 32 TR x 32 TC outputs, four waves of 16 TR x 16 TC.  The matrix instruction gets B as its
// first operand: a lane then holds four neighbouring columns of one row of C.
template <class T, Kind KA, Kind KB, int TR, int TC>
__global__ __launch_bounds__(THREADS) void tile_kernel(LinArgs a)
{
    constexpr int BR = 32 * TR, BC = 32 * TC, PARTS = Mma<T>::PARTS;
    typedef typename Part<T>::type P;
    typedef typename Mma<T>::frag frag;
    constexpr bool SUMS = KA == ACROSS_DZ;
    __shared__ __align__(16) P sA[PARTS * BR * BK];
    __shared__ __align__(16) P sB[PARTS * BC * BK];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int wr = (wave & 1) * 16 * TR, wc = (wave >> 1) * 16 * TC;

    // tile columns run fastest within a band of 8 tile rows, so that workgroups at work together share
    // both operands' tiles in L2
    const int64_t tiles_r = (a.R + BR - 1) / BR, tiles_c = (a.C + BC - 1) / BC, tiles = tiles_r * tiles_c;
    int64_t b = blockIdx.x;
    const int64_t split = b / tiles;
    b -= split * tiles;
    const int64_t band = b / (8 * tiles_c), in = b - band * 8 * tiles_c;
    const int64_t rows_here = tiles_r - band * 8 < 8 ? tiles_r - band * 8 : 8;
    const int64_t tr = band * 8 + in % rows_here, tc = in / rows_here;
    const int64_t row0 = tr * BR, col0 = tc * BC;
    const int64_t l_begin = split * a.l_per, l_end = l_begin + a.l_per < a.L ? l_begin + a.l_per : a.L;

    f32x4 acc[TR][TC] = {};
    Operand<T, KA, BR> oa;
    Operand<T, KB, BC> ob;
    float amax = 0.0f;
    float sums[SUMS ? 4 * Operand<T, KA, BR>::PER : 1] = {};
    const bool want_sums = SUMS && a.db && tc == 0;

    if (l_begin < l_end) {
        oa.load(a, a.A, a.R, row0, l_begin, l_end, tid);
        ob.load(a, a.B, a.C, col0, l_begin, l_end, tid);
    }
    for (int64_t l0 = l_begin; l0 < l_end; l0 += BK) {
        __syncthreads();
        oa.template store<SUMS>(a, sA, tid, amax, sums);
        ob.template store<false>(a, sB, tid, amax, nullptr);
        __syncthreads();
        if (l0 + BK < l_end) {
            oa.load(a, a.A, a.R, row0, l0 + BK, l_end, tid);
            ob.load(a, a.B, a.C, col0, l0 + BK, l_end, tid);
        }
        frag fa[PARTS][TR], fb[PARTS][TC];
#pragma unroll
        for (int p = 0; p < PARTS; ++p) {
#pragma unroll
            for (int i = 0; i < TR; ++i) fa[p][i] = *(const frag *)&sA[p * BR * BK + lds_at(wr + 16 * i + (lane & 15), (lane >> 4) * 8)];
#pragma unroll
            for (int j = 0; j < TC; ++j) fb[p][j] = *(const frag *)&sB[p * BC * BK + lds_at(wc + 16 * j + (lane & 15), (lane >> 4) * 8)];
        }
#pragma unroll
        for (int p = PARTS - 1; p >= 0; --p)                  // small products first
#pragma unroll
            for (int q = 0; q <= p; ++q)
#pragma unroll
                for (int i = 0; i < TR; ++i)
#pragma unroll
                    for (int j = 0; j < TC; ++j) acc[i][j] = Mma<T>::mul(fb[q][j], fa[p - q][i], acc[i][j]);
    }

    if constexpr (PARTS == 3) {
        if (__syncthreads_or(!(amax < 0x1p127f))) {
#pragma unroll 1
            for (int i = 0; i < TR; ++i)
#pragma unroll 1
                for (int j = 0; j < TC; ++j)
#pragma unroll 1
                    for (int q = 0; q < 4; ++q) {
                        const int64_t row = row0 + wr + 16 * i + (lane & 15), col = col0 + wc + 16 * j + (lane >> 4) * 4 + q;
                        float s = 0.0f;
                        if (row < a.R && col < a.C)
                            for (int64_t l = l_begin; l < l_end; ++l)
                                s = __builtin_fmaf(element<T, KA>(a, a.A, a.R, row, l), element<T, KB>(a, a.B, a.C, col, l), s);
#pragma unroll
                        for (int ii = 0; ii < TR; ++ii)
#pragma unroll
                            for (int jj = 0; jj < TC; ++jj)
#pragma unroll
                                for (int qq = 0; qq < 4; ++qq)
                                    if (ii == i && jj == j && qq == q) acc[ii][jj][qq] = s;
                    }
        }
    }

    if (want_sums) {                       // the same for the whole workgroup
        float *s = (float *)sA;            // [BK / 4][BR]
        __syncthreads();
#pragma unroll
        for (int i = 0; i < Operand<T, KA, BR>::PER; ++i) {
            const int u = i * THREADS + tid;
            if (u < Operand<T, KA, BR>::UNITS) {
                int row, l;
                Operand<T, KA, BR>::place(u, row, l);
#pragma unroll
                for (int j = 0; j < 4; ++j) s[(l / 4) * BR + row + j] = sums[4 * i + j];
            }
        }
        __syncthreads();
        for (int r = tid; r < BR; r += THREADS)
            if (row0 + r < a.R) {
                float t = 0.0f;
                for (int i = 0; i < BK / 4; ++i) t += s[i * BR + r];
                if (a.splits > 1) a.db_partial[split * a.R + row0 + r] = t;
                else ((T *)a.db)[row0 + r] = (T)t;
            }
    }

#pragma unroll
    for (int i = 0; i < TR; ++i) {
        const int64_t row = row0 + wr + 16 * i + (lane & 15);
#pragma unroll
        for (int j = 0; j < TC; ++j) {
            const int64_t col = col0 + wc + 16 * j + (lane >> 4) * 4;
            if (row < a.R && col < a.C) {
                const float z[4] = {acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]};
                if (a.splits > 1) {
                    Pack<float, 4> o = {z[0], z[1], z[2], z[3]};
                    store_some<float, 4>(a.partial + (split * a.R + row) * a.C + col, o, (int)(a.C - col < 4 ? a.C - col : 4));
                } else finish<T>(a, row, col, z);
            }
        }
    }
}

// the splits' sums, in their order, and the epilogue
template <class T>
__global__ __launch_bounds__(THREADS) void join_kernel(LinArgs a)
{
    const int64_t quads = (a.C + 3) / 4, total = a.R * quads;
    for (int64_t u = (int64_t)blockIdx.x * THREADS + threadIdx.x; u < total; u += (int64_t)gridDim.x * THREADS) {
        const int64_t i = u / quads, j = (u - i * quads) * 4;
        const int n = (int)(a.C - j < 4 ? a.C - j : 4);
        float z[4] = {};
#pragma unroll 4
        for (int64_t s = 0; s < a.splits; ++s) {
            const Pack<float, 4> v = load_some<float, 4>(a.partial + (s * a.R + i) * a.C + j, n);
#pragma unroll
            for (int q = 0; q < 4; ++q) z[q] += v.v[q];
        }
        finish<T>(a, i, j, z);
    }
    if (a.db)
        for (int64_t i = (int64_t)blockIdx.x * THREADS + threadIdx.x; i < a.R; i += (int64_t)gridDim.x * THREADS) {
            float t = 0.0f;
            for (int64_t s = 0; s < a.splits; ++s) t += a.db_partial[s * a.R + i];
            ((T *)a.db)[i] = (T)t;
        }
}

// ---- few rows ----------------------------------------------------------------------------------
// R <= 16 rows of A (stored along l) against 16 rows of B a workgroup: the matrix instruction's 16 columns
// are the rows of A, its rows those of B, and both operands go from memory to registers 16 bytes a
// lane.  The workgroup's waves take steps of l in turn and are summed in LDS, wave by wave.
constexpr int FEW = 16;

template <class T, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void few_rows_kernel(LinArgs a)
{
    __shared__ float part[WAVES][16][FEW + 1];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t col0 = (int64_t)blockIdx.x * 16, col = col0 + (lane & 15), row = lane & 15;
    f32x4 acc = {};
    constexpr int STEP = 32;
    const T *pa = (const T *)a.A + row * a.L, *pb = (const T *)a.B + col * a.L;
    const bool ina = row < a.R, inb = col < a.C;
#pragma unroll 4
    for (int64_t l = (int64_t)wave * STEP + (lane >> 4) * 8; l - (lane >> 4) * 8 < a.L; l += WAVES * STEP) {
        const int n = (int)(a.L - l < 8 ? a.L - l : 8);
        Pack<T, 8> va = {}, vb = {};
        if (n > 0 && ina) va = load_some<T, 8>(pa + l, n);
        if (n > 0 && inb) vb = load_some<T, 8>(pb + l, n);
        if constexpr (sizeof(T) == 2) {
            typename Mma<T>::frag fa, fb;
            __builtin_memcpy(&fa, &va, 16);
            __builtin_memcpy(&fb, &vb, 16);
            acc = Mma<T>::mul(fb, fa, acc);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(vb.v[i], va.v[i], acc, 0, 0, 0);
        }
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) part[wave][(lane >> 4) * 4 + q][lane & 15] = acc[q];
    __syncthreads();
    if (tid < 64) {                                            // lane: row = lane & 15, four columns
        float z[4] = {};
        for (int w = 0; w < WAVES; ++w)
#pragma unroll
            for (int q = 0; q < 4; ++q) z[q] += part[w][(lane >> 4) * 4 + q][lane & 15];
        const int64_t j = col0 + (lane >> 4) * 4;
        if (ina && j < a.C) finish<T>(a, row, j, z);
    }
}

// ---- launches ----------------------------------------------------------------------------------
int ok() { return hipGetLastError() == hipSuccess ? AFIV_OK : AFIV_E_HIP; }

struct Plan { bool big; int64_t tiles, splits, l_per; };

// Tile and split of a product of R x C outputs and L steps.  128 x 128 tiles once they give every CU
// one; below that 64 x 64, and below 512 workgroups the sum is cut into runs of at least 256 steps.
Plan plan_for(int64_t R, int64_t C, int64_t L)
{
    auto tiles = [&](int64_t t) { return ((R + t - 1) / t) * ((C + t - 1) / t); };
    Plan p;
    p.big = tiles(128) >= 256;
    p.tiles = tiles(p.big ? 128 : 64);
    p.splits = 1;
    const int64_t steps = (L + BK - 1) / BK;
    if (p.tiles > 0 && p.tiles < 256 && steps >= 16) p.splits = std::min((512 + p.tiles - 1) / p.tiles, steps / 8);
    p.l_per = std::max<int64_t>(1, (steps + p.splits - 1) / p.splits) * BK;
    p.splits = std::max<int64_t>(1, (L + p.l_per - 1) / p.l_per);
    return p;
}

template <class T, Kind KA, Kind KB>
int product(LinArgs a, float *scratch, hipStream_t s)
{
    const Plan p = plan_for(a.R, a.C, a.L);
    if (p.tiles == 0) return AFIV_OK;
    a.splits = p.splits;
    a.l_per = p.l_per;
    a.partial = scratch;
    a.db_partial = scratch + p.splits * a.R * a.C;
    const dim3 grid((unsigned)(p.tiles * p.splits));
    if (p.big) hipLaunchKernelGGL((tile_kernel<T, KA, KB, 4, 4>), grid, dim3(THREADS), 0, s, a);
    else hipLaunchKernelGGL((tile_kernel<T, KA, KB, 2, 2>), grid, dim3(THREADS), 0, s, a);
    if (p.splits > 1) {
        const int64_t units = a.R * ((a.C + 3) / 4), blocks = (units + THREADS - 1) / THREADS;
        hipLaunchKernelGGL(join_kernel<T>, dim3((unsigned)(blocks < 4096 ? blocks : 4096)), dim3(THREADS), 0, s, a);
    }
    return ok();
}

int64_t scratch_floats(int64_t R, int64_t C, int64_t L)
{
    const Plan p = plan_for(R, C, L);
    return p.splits > 1 ? p.splits * (R * C + R) : 0;
}

template <class T>
int forward(const LinArgs &a, float *scratch, hipStream_t s)
{
    if (a.R <= FEW && a.R > 0 && a.C > 0) {
        const dim3 grid((unsigned)((a.C + 15) / 16));
        // 16 waves where the layer has few workgroups to fill the chip with
        if (grid.x < 512 && a.L >= 512) hipLaunchKernelGGL((few_rows_kernel<T, 16>), grid, dim3(1024), 0, s, a);
        else hipLaunchKernelGGL((few_rows_kernel<T, 4>), grid, dim3(256), 0, s, a);
        return ok();
    }
    return product<T, ALONG, ALONG>(a, scratch, s);
}

template <class T>
int backward(const void *dy, const void *x, const int8_t *codes, const uint8_t *scales, const void *w, const void *pre,
             const uint8_t *dcodes, int act, int64_t M, int64_t N, int64_t K, void *dx, void *dw, void *db, float *scratch, hipStream_t s)
{
    LinArgs a = {};
    a.A = dy; a.act = act;
    if (act != AFIV_ACT_NONE) { a.pre = pre; a.dcodes = dcodes; }
    if (dx) {
        LinArgs d = a;
        d.B = w; d.R = M; d.C = K; d.L = N; d.out = dx;
        const int rc = product<T, ALONG_DZ, ACROSS>(d, scratch, s);
        if (rc) return rc;
    }
    if (dw || db) {
        LinArgs d = a;
        d.B = x; d.codes = codes; d.scales = scales;
        d.R = N; d.C = K; d.L = M; d.out = dw; d.db = db;
        return codes ? product<T, ACROSS_DZ, ACROSS_EIGHT>(d, scratch, s) : product<T, ACROSS_DZ, ACROSS>(d, scratch, s);
    }
    return AFIV_OK;
}

}  // namespace

int64_t afiv_linear_forward_scratch(int64_t M, int64_t N, int64_t K) { return M <= FEW ? 0 : scratch_floats(M, N, K) * 4; }

int64_t afiv_linear_backward_scratch(int64_t M, int64_t N, int64_t K)
{
    return std::max(scratch_floats(M, K, N), scratch_floats(N, K, M)) * 4;
}

int afiv_launch_linear_act(const void *x, const void *w, const void *bias, const void *residual, int dtype, int act, int64_t M, int64_t N,
                           int64_t K, void *y, void *pre, uint8_t *dcodes, float *scratch, hipStream_t s)
{
    LinArgs a = {};
    a.A = x; a.B = w; a.R = M; a.C = N; a.L = K;
    a.bias = bias; a.residual = residual; a.act_out = act; a.out = y; a.pre_out = pre; a.dcodes_out = dcodes;
    if (dtype == AFIV_F32) return forward<float>(a, scratch, s);
    if (dtype == AFIV_BF16) return forward<__bf16>(a, scratch, s);
    return forward<_Float16>(a, scratch, s);
}

int afiv_launch_linear_act_backward(const void *dy, const void *x, const int8_t *codes, const uint8_t *scales, const void *w,
                                    const void *pre, const uint8_t *dcodes, int dtype, int act, int64_t M, int64_t N, int64_t K, void *dx,
                                    void *dw, void *db, float *scratch, hipStream_t s)
{
    if (dtype == AFIV_F32) return backward<float>(dy, x, codes, scales, w, pre, dcodes, act, M, N, K, dx, dw, db, scratch, s);
    if (dtype == AFIV_BF16) return backward<__bf16>(dy, x, codes, scales, w, pre, dcodes, act, M, N, K, dx, dw, db, scratch, s);
    return backward<_Float16>(dy, x, codes, scales, w, pre, dcodes, act, M, N, K, dx, dw, db, scratch, s);
}
