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
// x: neither exists in memory (but for large products, below).
//
// 16-bit types go to v_mfma_f32_16x16x32, and dz is rounded to T for it (db is summed before): held in two parts it would
// double both products, 820 of 1460 us at 16384 x 4096 x 4096, and layers whose gradients are of type T round there anyway.  FP32 operands are cut into three BF16 parts of 8 bits,
// a = a1 + a2 + a3 exactly (each the upper half of what is left), and the six products a1 b1, a1 b2, a2 b1,
// a1 b3, a2 b2, a3 b1 are summed in FP32: what is dropped is at most 2^-21 of a product (a2 b3 and a3 b2, 2^-22 each) and
// 2^-25 in the mean, half an FP32 rounding, and six BF16 products cost 6/16 of one FP32 matrix instruction's time.
// An infinity does not split (its rest is NaN); a workgroup that has met one does its tile again with FP32
// multiply-adds.  Parts below 2^-133 are lost, that is, an element under 2^-110 keeps fewer than 24 bits.
//
// Few rows (up to 32), and small products, take another kernel: W goes straight from memory into the matrix
// instruction, by as many waves as the layer has.  Large products take a third, whose operands go from memory to LDS
// as they are; what cannot be read so (dz, an 8-bit x, rows that are not whole 16-byte chunks) is written out first.
#pragma once

#include "afiv_layer.h"

#include <type_traits>

#include "afiv_linear_plan.h"

namespace {

constexpr int THREADS = 256;

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

// INSIDE: all of it lies in the matrix, and nothing is guarded
template <class T, Kind K, bool INSIDE>
__device__ __forceinline__ void fetch(const LinArgs &a, const void *base, int64_t R, int64_t row, int64_t l, int64_t l_end, Held<T, K> &h)
{
    if constexpr (!across(K)) {
        const int n = INSIDE ? 8 : row < R ? (int)(l_end - l < 8 ? l_end - l : 8) : 0;      // may be negative
        if (!INSIDE && n <= 0) {
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
        const int n = INSIDE ? 4 : (int)(R - row < 4 ? R - row : 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bool in = INSIDE || (l + i < l_end && n > 0);
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
    }
    if constexpr (is_dz(K)) {
        if (a.pre || a.dcodes)
            with_act(a.act, [&](auto act) {
                constexpr int ACT = decltype(act)::value;
                if (a.pre) {
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        float y, d;
                        act_both<ACT>((float)h.z.v[i], y, d);
                        f[i] *= d;
                    }
                } else {
                    uint8_t c[N];
                    __builtin_memcpy(c, &h.z, N);
#pragma unroll
                    for (int i = 0; i < N; ++i) f[i] *= derivative_of_code<ACT>(c[i]);
                }
            });
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
        if (a.pre || a.dcodes)
            with_act(a.act, [&](auto act) {
                float y, d = 1.0f;
                if (a.pre) act_both<decltype(act)::value>((float)((const T *)a.pre)[at], y, d);
                else d = derivative_of_code<decltype(act)::value>(a.dcodes[at]);
                f *= d;
            });
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

// The three parts of eight FP32 values, two to a word: the upper halves of a, of a - a1 and of a - a1 - a2
__device__ __forceinline__ void split8(const float (&a)[8], uint32_t (&p1)[4], uint32_t (&p2)[4], uint32_t (&p3)[4])
{
    float b[8], c[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        b[i] = a[i] - __uint_as_float(__float_as_uint(a[i]) & 0xffff0000u);
        c[i] = b[i] - __uint_as_float(__float_as_uint(b[i]) & 0xffff0000u);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        p1[i] = __builtin_amdgcn_perm(__float_as_uint(a[2 * i + 1]), __float_as_uint(a[2 * i]), 0x07060302);
        p2[i] = __builtin_amdgcn_perm(__float_as_uint(b[2 * i + 1]), __float_as_uint(b[2 * i]), 0x07060302);
        p3[i] = __builtin_amdgcn_perm(__float_as_uint(c[2 * i + 1]), __float_as_uint(c[2 * i]), 0x07060302);
    }
}

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
        uint32_t o[3][4];
        float v[8] = {};
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = f[i];
        split8(v, o[0], o[1], o[2]);
#pragma unroll
        for (int p = 0; p < 3; ++p) __builtin_memcpy(__builtin_assume_aligned(lds + p * plane, 2 * N), o[p], 2 * N);
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
        // the same for the workgroup: tiles inside load without guards, so that a wave's loads go out together
        if (row0 + ROWS <= R && l0 + BK <= l_end) load_units<true>(a, base, R, row0, l0, l_end, tid);
        else load_units<false>(a, base, R, row0, l0, l_end, tid);
    }
    template <bool INSIDE>
    __device__ __forceinline__ void load_units(const LinArgs &a, const void *base, int64_t R, int64_t row0, int64_t l0, int64_t l_end, int tid)
    {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int u = i * THREADS + tid;
            if (UNITS % THREADS == 0 || u < UNITS) {
                int row, l;
                place(u, row, l);
                fetch<T, K, INSIDE>(a, base, R, row0 + row, l0 + l, l_end, h[i]);
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

// db without dW, where no pass over dz sums it: a workgroup sums 128 columns of dz over one run of rows and reads nothing
// of the layer's input.  A lane holds what it would in the tile kernel (4 columns, every eighth quad of rows), and the runs
// are that kernel's, so db has the same bits with and without dW.  block: runs by blocks of columns.  Loads bound it, one step
// on its way behind the step before: 131072 x 64 in BF16 with gelu's derivative 36 us (0.9 TB/s; with the product that took
// 68), 64 x 4096 6 us (41).
template <class T>
__device__ __forceinline__ void sum_dz(const LinArgs &a, int64_t block)
{
    typedef Operand<T, ACROSS_DZ, 128> Dz;
    typedef Held<T, ACROSS_DZ> H;
    static_assert(Dz::UNITS == THREADS, "a unit a thread");
    __shared__ float lds[BK / 4][128];
    int c, l;
    Dz::place(threadIdx.x, c, l);
    const int64_t blocks = (a.R + 127) / 128, split = block / blocks;
    const int64_t col0 = (block - split * blocks) * 128, l_begin = split * a.l_per;
    const int64_t l_end = l_begin + a.l_per < a.L ? l_begin + a.l_per : a.L;
    float sums[4] = {};
    Dz next;
    if (l_begin < l_end) next.load(a, a.A, a.R, col0, l_begin, l_end, threadIdx.x);
    for (int64_t l0 = l_begin; l0 < l_end; l0 += BK) {
        const H h = next.h[0];
        if (l0 + BK < l_end) next.load(a, a.A, a.R, col0, l0 + BK, l_end, threadIdx.x);
        float f[H::N];
        values<T, ACROSS_DZ>(a, h, f);
#pragma unroll
        for (int j = 0; j < 4; ++j) sums[j] += (f[j] + f[4 + j]) + (f[8 + j] + f[12 + j]);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) lds[l / 4][c + j] = sums[j];
    __syncthreads();
    if (threadIdx.x < 128 && col0 + threadIdx.x < a.R) {
        float t = 0.0f;
        for (int i = 0; i < BK / 4; ++i) t += lds[i][threadIdx.x];
        if (a.splits > 1) a.db_partial[split * a.R + col0 + threadIdx.x] = t;
        else ((T *)a.db)[col0 + threadIdx.x] = (T)t;
    }
}

// W outputs of row i from column j on, from their sums z.  EPI: the forward epilogue.
template <class T, bool EPI, int W>
__device__ __forceinline__ void finish(const LinArgs &a, int64_t i, int64_t j, float (&z)[W])
{
    const int n = (int)(a.C - j < W ? a.C - j : W);
    const int64_t at = i * a.C + j;
    if constexpr (EPI) {
        if (a.bias) {
            const Pack<T, W> b = load_some<T, W>((const T *)a.bias + j, n);
#pragma unroll
            for (int q = 0; q < W; ++q) z[q] += (float)b.v[q];
        }
        if (a.pre_out) {
            Pack<T, W> o;
#pragma unroll
            for (int q = 0; q < W; ++q) o.v[q] = (T)z[q];
            store_some<T, W>((T *)a.pre_out + at, o, n);
        }
        Pack<uint8_t, W> c = {};
        with_act(a.act_out, [&](auto act) {
            constexpr int ACT = decltype(act)::value;
#pragma unroll
            for (int q = 0; q < W; ++q) {
                float y, d;
                act_both<ACT>(z[q], y, d);
                if (a.dcodes_out) c.v[q] = derivative_code<ACT>(z[q], d);
                z[q] = y;
            }
        });
        if (a.dcodes_out) store_some<uint8_t, W>(a.dcodes_out + at, c, n);
        if (a.residual) {
            const Pack<T, W> r = load_some<T, W>((const T *)a.residual + at, n);
#pragma unroll
            for (int q = 0; q < W; ++q) z[q] += (float)r.v[q];
        }
    }
    Pack<T, W> o;
#pragma unroll
    for (int q = 0; q < W; ++q) o.v[q] = (T)z[q];
    store_some<T, W>((T *)a.out + at, o, n);
}

// A wave's 16 TR x 16 TC outputs from its accumulators (lane = row lane & 15, four columns from 4 (lane >> 4) of
// each 16 x 16 block) by way of LDS, SLABS blocks of 16 rows at a time in the wave's own room: a lane then
// has 8 neighbouring columns, the memory accesses are whole lines, and the epilogue's code stands once.
// The 16-byte chunks of a row are permuted by the row so that a column of writes meets all banks.
// Tiles inside the matrix take the forward epilogue four rows at a time, the residual's loads first: one by one they
// were a fifth of a large layer's time.
template <class T, bool EPI, int TR, int TC, int SLABS>
__device__ __forceinline__ void write_out(const LinArgs &a, const f32x4 (&acc)[TR][TC], int64_t row0, int64_t col0, int64_t split, int lane,
                                          float *room)
{
    constexpr int COLS = 16 * TC, CHUNKS = COLS / 4, UNITS = 16 * COLS / 8;      // of a slab
    static_assert(TR % SLABS == 0 && UNITS % 64 == 0 && 64 % (COLS / 8) == 0, "whole passes, a lane's column stays");
    const bool inside = row0 + 16 * TR <= a.R && col0 + COLS <= a.C && a.splits == 1;
    const int c0 = lane % (COLS / 8) * 2;                                          // a lane's first chunk
    const int64_t col = col0 + c0 * 4;
    float bias[8] = {};
    if (EPI && inside && a.bias) {
        const Pack<T, 8> b = load_pack<T, 8>((const T *)a.bias + col);
#pragma unroll
        for (int q = 0; q < 8; ++q) bias[q] = (float)b.v[q];
    }
    auto from_room = [&](int r, float (&z)[8]) {
        const f32x4 lo = *(const f32x4 *)&room[r * COLS + ((c0 ^ (r & (CHUNKS - 1))) * 4)];
        const f32x4 hi = *(const f32x4 *)&room[r * COLS + (((c0 + 1) ^ (r & (CHUNKS - 1))) * 4)];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            z[q] = lo[q];
            z[4 + q] = hi[q];
        }
    };
    constexpr int RSTEP = 64 / (COLS / 8), ROWS = SLABS * 16, G = ROWS / RSTEP < 4 ? ROWS / RSTEP : 4;   // rows from unit to unit
#pragma unroll 1
    for (int phase = 0; phase < TR / SLABS; ++phase) {
#pragma unroll
        for (int ph = 0; ph < TR / SLABS; ++ph)
            if (ph == phase) {
#pragma unroll
                for (int i = 0; i < SLABS; ++i)
#pragma unroll
                    for (int j = 0; j < TC; ++j) {
                        const int r = lane & 15, c = (4 * j + (lane >> 4)) ^ (r & (CHUNKS - 1));
                        *(f32x4 *)&room[(i * 16 + r) * COLS + c * 4] = acc[ph * SLABS + i][j];
                    }
            }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        const int64_t first = row0 + phase * ROWS;
        if (EPI && inside) {
#pragma unroll 1
            for (int r0 = lane / (COLS / 8); r0 < ROWS; r0 += G * RSTEP) {
                Pack<T, 8> res[G];
                if (a.residual) {
#pragma unroll
                    for (int g = 0; g < G; ++g) res[g] = load_pack<T, 8>((const T *)a.residual + (first + r0 + g * RSTEP) * a.C + col);
                }
                with_act(a.act_out, [&](auto act) {
                    constexpr int ACT = decltype(act)::value;
#pragma unroll
                    for (int g = 0; g < G; ++g) {
                        const int64_t at = (first + r0 + g * RSTEP) * a.C + col;
                        float z[8];
                        from_room(r0 + g * RSTEP, z);
                        Pack<T, 8> o, pre;
                        Pack<uint8_t, 8> code;
#pragma unroll
                        for (int q = 0; q < 8; ++q) {
                            z[q] += bias[q];
                            float y, d;
                            act_both<ACT>(z[q], y, d);
                            pre.v[q] = (T)z[q];
                            if (a.dcodes_out) code.v[q] = derivative_code<ACT>(z[q], d);
                            if (a.residual) y += (float)res[g].v[q];
                            o.v[q] = (T)y;
                        }
                        if (a.pre_out) store_pack<T, 8>((T *)a.pre_out + at, pre);
                        if (a.dcodes_out) store_pack<uint8_t, 8>(a.dcodes_out + at, code);
                        store_pack<T, 8>((T *)a.out + at, o);
                    }
                });
            }
        } else {
#pragma unroll 1
            for (int r = lane / (COLS / 8); r < ROWS; r += RSTEP) {
                const int64_t row = first + r;
                if (row < a.R && col < a.C) {
                    float z[8];
                    from_room(r, z);
                    if (a.splits > 1) {
                        Pack<float, 8> o;
#pragma unroll
                        for (int q = 0; q < 8; ++q) o.v[q] = z[q];
                        store_some<float, 8>(a.partial + (split * a.R + row) * a.C + col, o, (int)(a.C - col < 8 ? a.C - col : 8));
                    } else finish<T, EPI, 8>(a, row, col, z);
                }
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
}

// workgroup -> split and tile: tile columns run fastest within a band of 8 tile rows, so that workgroups at work
// together share both operands' tiles; consecutive workgroups go round the 8 XCDs, each with an L2 of its own, so
// each XCD is given a run of consecutive tiles
__device__ __forceinline__ void place_tile(const LinArgs &a, int br, int bc, int64_t block, int64_t all, int64_t &split, int64_t &tr, int64_t &tc)
{
    const int64_t tiles_r = (a.R + br - 1) / br, tiles_c = (a.C + bc - 1) / bc, tiles = tiles_r * tiles_c;
    const int64_t each = all / 8, spare = all % 8, xcd = block % 8;
    int64_t b = xcd * each + (xcd < spare ? xcd : spare) + block / 8;
    split = b / tiles;
    b -= split * tiles;
    const int64_t band = b / (8 * tiles_c), in = b - band * 8 * tiles_c;
    const int64_t rows_here = tiles_r - band * 8 < 8 ? tiles_r - band * 8 : 8;
    tr = band * 8 + in % rows_here;
    tc = in / rows_here;
}

// sums over l for a tile's outputs one by one, in FP32: for operands that do not split into parts
template <class T, Kind KA, Kind KB, int TR, int TC>
__device__ __forceinline__ void plain_sums(const LinArgs &a, f32x4 (&acc)[TR][TC], int64_t row0, int64_t col0, int64_t l_begin, int64_t l_end,
                                           int lane)
{
#pragma unroll 1
    for (int i = 0; i < TR; ++i)
#pragma unroll 1
        for (int j = 0; j < TC; ++j)
#pragma unroll 1
            for (int q = 0; q < 4; ++q) {
                const int64_t row = row0 + 16 * i + (lane & 15), col = col0 + 16 * j + (lane >> 4) * 4 + q;
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

// Tile of 32 TR x 32 TC outputs, four waves of 16 TR x 16 TC.  The matrix instruction gets B as its
// first operand: a lane then holds four neighbouring columns of one row of C.  For products too small for the direct
// kernel, where latency bounds: one step's loads are on their way behind the step before.  Backward of 64 rows, 13 -> 128, in
// FP32: 9.5 us for dx, dW and db.
template <class T, Kind KA, Kind KB, int TR, int TC>
__device__ __forceinline__ void tile(const LinArgs &a, int64_t block, int64_t blocks)
{
    constexpr int BR = 32 * TR, BC = 32 * TC, PARTS = Mma<T>::PARTS;
    typedef typename Part<T>::type P;
    typedef typename Mma<T>::frag frag;
    constexpr bool SUMS = KA == ACROSS_DZ;
    constexpr int ROOM = 16 * 16 * TC;                                      // floats of a wave's epilogue
    constexpr int BYTES = PARTS * (BR + BC) * BK * 2;
    static_assert(BYTES >= 4 * ROOM * 4, "the epilogue's room");
    __shared__ __align__(16) char lds[BYTES];
    P *const sA = (P *)lds, *const sB = sA + PARTS * BR * BK;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int wr = (wave & 1) * 16 * TR, wc = (wave >> 1) * 16 * TC;

    int64_t split, tr, tc;
    place_tile(a, BR, BC, block, blocks, split, tr, tc);
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
        if (__syncthreads_or(!(amax < __builtin_inff())))
            plain_sums<T, KA, KB, TR, TC>(a, acc, row0 + wr, col0 + wc, l_begin, l_end, lane);
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

    __syncthreads();
    write_out<T, KA == ALONG, TR, TC, 1>(a, acc, row0 + wr, col0 + wc, split, lane, (float *)lds + wave * ROOM);
}

template <class T, Kind KA, Kind KB>
__global__ __launch_bounds__(THREADS) void tile_kernel(LinArgs a)
{
    tile<T, KA, KB, 2, 2>(a, blockIdx.x, gridDim.x);
}

// dx and dW in one launch: the first dx_blocks workgroups are dx's.  Neither fills the chip where the tile kernel takes
// both, and neither waits for the other.
template <class T, Kind KX>
__global__ __launch_bounds__(THREADS) void both_kernel(LinArgs dx, LinArgs dw, int64_t dx_blocks)
{
    const int64_t block = blockIdx.x;
    if (block < dx_blocks) tile<T, ALONG_DZ, ACROSS, 2, 2>(dx, block, dx_blocks);
    else tile<T, ACROSS_DZ, KX, 2, 2>(dw, block - dx_blocks, gridDim.x - dx_blocks);
}

template <class T>
__global__ __launch_bounds__(THREADS) void db_alone_kernel(LinArgs dw)
{
    sum_dz<T>(dw, blockIdx.x);
}

// dx and db in one launch, as above
template <class T>
__global__ __launch_bounds__(THREADS) void dx_db_kernel(LinArgs dx, LinArgs dw, int64_t dx_blocks)
{
    const int64_t block = blockIdx.x;
    if (block < dx_blocks) tile<T, ALONG_DZ, ACROSS, 2, 2>(dx, block, dx_blocks);
    else sum_dz<T>(dw, block - dx_blocks);
}

// The splits' sums, in a fixed order, and the epilogue: SLICES threads an output of four columns, each over every
// SLICES-th split, their sums added in LDS in slice order.  One thread over hundreds of splits waits for one
// load after the other (131072 x 64 x 32: 0.2 ms of a 0.22 ms backward pass).
template <class T, bool EPI, int SLICES>
__global__ __launch_bounds__(THREADS) void join_kernel(LinArgs a)
{
    constexpr int PER = THREADS / SLICES;
    __shared__ float lds[SLICES > 1 ? SLICES : 1][PER][5];
    const int unit = threadIdx.x % PER, slice = threadIdx.x / PER;
    const int64_t quads = (a.C + 3) / 4, outs = a.R * quads, total = outs + (a.db ? a.R : 0);
    for (int64_t first = (int64_t)blockIdx.x * PER; first < total; first += (int64_t)gridDim.x * PER) {      // the same for the workgroup
        const int64_t u = first + unit, i = u / quads, j = (u - i * quads) * 4;
        const int n = (int)(a.C - j < 4 ? a.C - j : 4);
        float z[4] = {};
        if (u < outs) {
#pragma unroll 4
            for (int64_t s = slice; s < a.splits; s += SLICES) {
                const Pack<float, 4> v = load_some<float, 4>(a.partial + (s * a.R + i) * a.C + j, n);
#pragma unroll
                for (int q = 0; q < 4; ++q) z[q] += v.v[q];
            }
        } else if (u < total) {
#pragma unroll 4
            for (int64_t s = slice; s < a.splits; s += SLICES) z[0] += a.db_partial[s * a.R + u - outs];
        }
        if constexpr (SLICES > 1) {
            __syncthreads();
#pragma unroll
            for (int q = 0; q < 4; ++q) lds[slice][unit][q] = z[q];
            __syncthreads();
            if (slice == 0) {
#pragma unroll
                for (int s = 1; s < SLICES; ++s)
#pragma unroll
                    for (int q = 0; q < 4; ++q) z[q] += lds[s][unit][q];
            }
        }
        if (slice == 0) {
            if (u < outs) finish<T, EPI, 4>(a, i, j, z);
            else if (u < total) ((T *)a.db)[u - outs] = (T)z[0];
        }
    }
}

// ---- large products -------------------------------------------------------------------------------
// The same product from operands that go from memory to LDS as they are: rows of whole 16-byte chunks.  Operands of
// that kind are read where they stand; others are written so first, by prepare_kernel: rows of another length, dz, an
// 8-bit x.
// Steps of 64 (FP32: 32): a tile's rows are 128 bytes along l, or its steps of l are rows of BR elements
// (across), and lie in LDS as the loads leave them, 1024 consecutive bytes an instruction; what keeps the
// reads off each other's banks is therefore a permutation of the global addresses: 16-byte chunk c of row r stands
// at c ^ (r & 7), block c of 16 elements of step l at c ^ key(l).  16-bit operands across l are transposed by the LDS
// read itself (ds_read_b64_tr_b16), FP32 ones are read an element at a time.
// Two buffers; one barrier a step: the loads of the next step run behind this one's products.
typedef __attribute__((address_space(3))) void *lds_ptr;

// P: element, ROWS: rows of the tile, TN: blocks of 16 rows of a wave
template <class P, bool XS, int ROWS, int WAVES, int TN>
struct Direct {
    static constexpr int ES = sizeof(P), FK = 128 / ES;           // steps of l
    static constexpr int BYTES = ROWS * 128, PER = BYTES / 1024 / WAVES;      // loads of a wave
    static_assert(PER * WAVES * 1024 == BYTES, "whole loads");
    static constexpr int LSTEP = XS ? 1024 / (ES * ROWS) : 0;     // steps of l from one load of a wave to the next
    static constexpr int BASES = XS ? TN : 2;
    uint32_t off[PER];                    // byte offset from the tile's corner; beyond the matrix: out of range
    uint32_t l_first;                     // step of l of the first load
    uint32_t at[BASES];                   // where a lane's reads start

    // across: blocks of 16 elements stand at block ^ key(l)
    static __device__ __forceinline__ int key(int l) { return ES == 2 ? (l & 3) | ((l >> 1) & 4) : (l >> 2) & 3; }

    // w0: first of the wave's 16 TN rows
    __device__ __forceinline__ void init(int64_t R, int64_t ld, int64_t row0, int w0, int wave, int lane)
    {
        constexpr int CB = 16 * ES / 16;                          // 16-byte chunks of a block of 16 elements
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int byte = (wave * PER + i) * 1024 + lane * 16;
            if (!XS) {
                const int r = byte / 128, c = (lane & 7) ^ (lane >> 3);
                off[i] = row0 + r < R ? (uint32_t)(r * ld * ES + c * 16) : 0x80000000u;
            } else {
                const int l = byte / (ES * ROWS), pos = byte % (ES * ROWS) / 16;
                const int col = ((pos / CB) ^ key(l)) * 16 + pos % CB * (16 / ES);
                off[i] = row0 + col < R ? (uint32_t)((l * ld + col) * ES) : 0x80000000u;
            }
        }
        if (!XS) {
            l_first = ((lane & 7) ^ (lane >> 3)) * (16 / ES);
            // chunks (lane >> 4) and 4 + (lane >> 4): a slice each in 16 bit, together one fragment in FP32
#pragma unroll
            for (int k = 0; k < 2; ++k) at[k] = (w0 + (lane & 15)) * 128 + (((k * 4 + (lane >> 4)) ^ (lane & 7)) << 4);
        } else {
            l_first = (wave * PER * 1024 + lane * 16) / (ES * ROWS);
            // 16 bit: 16 lanes read 4 steps x 16 rows, 8 bytes each, and get 4 steps of a row each; FP32: a lane reads its own
            const int l = ES == 2 ? (lane >> 4) * 8 + ((lane >> 2) & 3) : (lane >> 4) * 4;
#pragma unroll
            for (int i = 0; i < TN; ++i)
                at[i] = l * (ES * ROWS) + (((w0 >> 4) + i) ^ key(l)) * (16 * ES) + (ES == 2 ? (lane & 3) * 8 : (lane & 15) * 4);
        }
    }
    __device__ __forceinline__ void load(const P *base, int64_t ld, int64_t row0, int64_t l0, int64_t l_end, char *lds, int wave) const
    {
#if defined(__HIP_DEVICE_COMPILE__)             // buffer resources have no host type
        const P *corner = base + (XS ? l0 * ld + row0 : row0 * ld + l0);
        const auto rsrc = __builtin_amdgcn_make_buffer_rsrc((void *)corner, 0, 0x7fffffff, 0x00020000);
        const int left = (int)(l_end - l0 < FK ? (l_end > l0 ? l_end - l0 : 0) : FK);
#pragma unroll
        for (int i = 0; i < PER; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_ptr)(lds + (wave * PER + i) * 1024), 16,
                                                     (int)l_first < left - i * LSTEP ? off[i] : 0x80000000u, 0, 0, 0);
#endif
    }
    // 16 bit: rows 16 i + (lane & 15) of the wave's, steps 32 kk + 8 (lane >> 4) ..+7
    __device__ __forceinline__ typename Mma<P>::frag read(const char *lds, int i, int kk) const
    {
        typename Mma<P>::frag f;
        if constexpr (!XS) f = *(const typename Mma<P>::frag *)(lds + at[kk] + i * 2048);
        else {
            typedef short s16x4 __attribute__((ext_vector_type(4)));
            s16x4 h[2];
#pragma unroll
            for (int p = 0; p < 2; ++p)
                h[p] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(lds + at[i] + (kk * 32 + p * 4) * (2 * ROWS)));
            __builtin_memcpy(&f, h, 16);
        }
        return f;
    }
    // FP32: the same rows, steps 4 (lane >> 4) ..+3 and 16 + 4 (lane >> 4) ..+3: any order of the steps will do that both
    // operands share, and this one reads the chunks that 16-bit fragments do
    __device__ __forceinline__ void read(const char *lds, int i, float (&f)[8]) const
    {
        if constexpr (!XS) {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const f32x4 v = *(const f32x4 *)(lds + at[k] + i * 2048);
#pragma unroll
                for (int q = 0; q < 4; ++q) f[4 * k + q] = v[q];
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = *(const float *)(lds + at[i] + (e < 4 ? e : 12 + e) * (4 * ROWS));
        }
    }
};

// what the direct kernels read of an operand
struct Source {
    const void *p;
    int64_t ld;                           // elements from row to row (of l across)
};

// nothing of memory or LDS moves across; all but this wave's last LEFT loads have arrived and its LDS reads are done
// (__syncthreads would wait for every load)
template <int LEFT>
__device__ __forceinline__ void arrive()
{
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(0x0070 | (LEFT & 15) | (LEFT >> 4 << 14));
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" ::: "memory");
}

// 16-bit types.  WR x WC waves of 16 TR x 16 TC outputs.  The matrix units bound it: 16384 x 4096 x 8192 in BF16 with gelu
// and residual takes 0.92 ms (1.19 PFLOP/s, 57 % of their cycles; the rest is the epilogue and the start of each tile),
// dW of 16384 x 4096 x 4096 0.38 ms (1.44 PFLOP/s).  DEEP: four buffers instead of two, for a grid of at most one
// workgroup a CU, which has no other to hide its loads behind: 777 x 1003 x 2055 19.4 -> 17.0 us, of which the steps
// take 0.21 us each, what the matrix units need and L2 gives; where two fit a CU two buffers are faster (26 and
// 20 us for a product of 315 workgroups).
template <class T, Kind KA, Kind KB, int WR, int WC, int TR, int TC, bool DEEP>
__global__ __launch_bounds__(64 * WR * WC) void direct_kernel(LinArgs a, Source sa, Source sb)
{
    constexpr int W = WR * WC, BR = 16 * TR * WR, BC = 16 * TC * WC, FK = 64;
    typedef typename Mma<T>::frag frag;
    typedef Direct<T, across(KA), BR, W, TR> DA;
    typedef Direct<T, across(KB), BC, W, TC> DB;
    // each buffer an array of its own, named where it is used: the compiler then knows that loads into one do not
    // touch reads of the other, and does not make those wait
    __shared__ __align__(1024) char a0[DA::BYTES];
    __shared__ __align__(1024) char a1[DA::BYTES];
    __shared__ __align__(1024) char b0[DB::BYTES];
    __shared__ __align__(1024) char b1[DB::BYTES];
    __shared__ __align__(1024) char a2[DA::BYTES];
    __shared__ __align__(1024) char a3[DA::BYTES];
    __shared__ __align__(1024) char b2[DB::BYTES];
    __shared__ __align__(1024) char b3[DB::BYTES];
    // the epilogue's room of a wave: a quarter of the waves share an array
    static_assert(W % 4 == 0 && DA::BYTES == DB::BYTES, "four arrays of one size");
    constexpr int SLAB = 16 * 16 * TC, FIT = DA::BYTES / (W / 4) / 4 / SLAB, SLABS = FIT >= TR ? TR : FIT >= TR / 2 ? TR / 2 : FIT >= TR / 4 ? TR / 4 : 1;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wr = (wave % WR) * 16 * TR, wc = (wave / WR) * 16 * TC;
    int64_t split, tr, tc;
    place_tile(a, BR, BC, blockIdx.x, gridDim.x, split, tr, tc);
    const int64_t row0 = tr * BR, col0 = tc * BC;
    const int64_t l_begin = split * a.l_per, l_end = l_begin + a.l_per < a.L ? l_begin + a.l_per : a.L;
    DA da;
    DB db;
    da.init(a.R, sa.ld, row0, wr, wave, lane);
    db.init(a.C, sb.ld, col0, wc, wave, lane);
    f32x4 acc[TR][TC] = {};

    auto load = [&](char *la, char *lb, int64_t l0) {           // from l_end on: zeros
        da.load((const T *)sa.p, sa.ld, row0, l0, l_end, la, wave);
        db.load((const T *)sb.p, sb.ld, col0, l0, l_end, lb, wave);
    };
    // Fragments of one 32-step slice at a time: while row block i of this slice is multiplied, its registers take
    // the next slice's (those of B, shared by the row blocks, have a second set), so the matrix units need not
    // wait for LDS, nor the reads for a barrier that comes once a step.
    frag fa[TR], fb[2][TC];
    auto slice = [&](int set, const char *na, const char *nb, int next_kk) {
#pragma unroll
        for (int i = 0; i < TR; ++i) {
#pragma unroll
            for (int j = 0; j < TC; ++j) acc[i][j] = Mma<T>::mul(fb[set][j], fa[i], acc[i][j]);
            fa[i] = da.read(na, i, next_kk);
            if (i < TC) fb[set ^ 1][i] = db.read(nb, i, next_kk);
            __builtin_amdgcn_sched_group_barrier(0x008, TC, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, across(KA) ? 2 : 1, 0);
            if (i < TC) __builtin_amdgcn_sched_group_barrier(0x100, across(KB) ? 2 : 1, 0);
        }
    };
    static_assert(TC <= TR, "a row block for every column block's reads");
    constexpr int LATER = DEEP ? 2 * (DA::PER + DB::PER) : 0;   // a wave's loads that may still be on their way at a barrier
    load(a0, b0, l_begin);
    load(a1, b1, l_begin + FK);
    if constexpr (DEEP) {
        load(a2, b2, l_begin + 2 * FK);
        load(a3, b3, l_begin + 3 * FK);
    }
    arrive<DEEP ? 3 * (DA::PER + DB::PER) : 0>();
#pragma unroll
    for (int i = 0; i < TR; ++i) fa[i] = da.read(a0, i, 0);
#pragma unroll
    for (int j = 0; j < TC; ++j) fb[0][j] = db.read(b0, j, 0);
    // every load of this wave for the next tile has arrived and its reads are done before any wave reads that tile or
    // loads over this one; loads are issued before the products, not among them
    auto step = [&](char *ta, char *tb, char *na, char *nb, int64_t l0) {      // this tile, the next one, what comes into this one's place
        slice(0, ta, tb, 1);
        arrive<LATER>();
        load(ta, tb, l0);
        __builtin_amdgcn_sched_barrier(0);
        slice(1, na, nb, 0);
    };
    constexpr int BUFFERS = DEEP ? 4 : 2;
#pragma unroll 1
    for (int64_t l0 = l_begin; l0 < l_end; l0 += BUFFERS * FK) {               // steps from l_end on are multiplied with zeros
        step(a0, b0, a1, b1, l0 + BUFFERS * FK);
        if constexpr (DEEP) {
            step(a1, b1, a2, b2, l0 + 5 * FK);
            step(a2, b2, a3, b3, l0 + 6 * FK);
            step(a3, b3, a0, b0, l0 + 7 * FK);
        } else step(a1, b1, a0, b0, l0 + 3 * FK);
    }
    __builtin_amdgcn_s_waitcnt(0x0070);                         // the last loads and reads, before LDS is used again
    __syncthreads();
    write_out<T, KA == ALONG && KB == ALONG, TR, TC, SLABS>(a, acc, row0 + wr, col0 + wc, split, lane,
                                                            (float *)(wave % 4 == 0 ? a0 : wave % 4 == 1 ? a1 : wave % 4 == 2 ? b0 : b1) + wave / 4 * SLABS * SLAB);
}

// whether rows row0..row0 + 127 of an operand hold an infinity in l_begin..l_end (the whole workgroup asks)
template <bool XS>
__device__ __forceinline__ bool infinities(const Source &s, int64_t R, int64_t row0, int64_t l_begin, int64_t l_end)
{
    bool any = false;
    const int64_t run = XS ? 128 : l_end - l_begin, all = 128 * (l_end - l_begin);
    for (int64_t i = threadIdx.x; i < all; i += blockDim.x) {
        const int64_t outer = i / run, inner = i % run, row = row0 + (XS ? inner : outer), l = l_begin + (XS ? outer : inner);
        if (row < R) any |= fabsf(((const float *)s.p)[XS ? l * s.ld + row : row * s.ld + l]) == __builtin_inff();
    }
    return any;
}

// FP32: 128 x 128 tiles, four waves of 64 x 64, two workgroups a CU.  The operands lie in LDS as they are, 32 steps to a
// row of 128 bytes, and each wave splits its fragments on the way to the matrix units: 44 vector instructions a fragment
// beside the 12 matrix instructions it feeds, which the two units of a SIMD run side by side.  (Parts written to memory
// as three planes first were 10 bytes an element of extra traffic and half again as many through L2: forward and backward
// of 8192 x 1024 x 512 took 221 us, 191 now: forward 61 to 66 from card to card, dx 53 to 57, dW 53 to 56.)  Instruction issue bounds it: a matrix
// instruction (16 cycles) and its 3.7 vector instructions (15) take 34 cycles of a SIMD with two waves, 50 of one with a
// lone wave, however the two kinds are ordered.  `a` describes the operands as they came, sa and sb as they are read.
template <Kind KA, Kind KB>
__global__ __launch_bounds__(256, 2) void direct32_kernel(LinArgs a, Source sa, Source sb)
{
    constexpr int TR = 4, TC = 4, FK = 32;
    typedef Direct<float, across(KA), 128, 4, TR> DA;
    typedef Direct<float, across(KB), 128, 4, TC> DB;
    __shared__ __align__(1024) char a0[DA::BYTES];
    __shared__ __align__(1024) char a1[DA::BYTES];
    __shared__ __align__(1024) char b0[DB::BYTES];
    __shared__ __align__(1024) char b1[DB::BYTES];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wr = (wave & 1) * 64, wc = (wave >> 1) * 64;
    int64_t split, tr, tc;
    place_tile(a, 128, 128, blockIdx.x, gridDim.x, split, tr, tc);
    const int64_t row0 = tr * 128, col0 = tc * 128;
    const int64_t l_begin = split * a.l_per, l_end = l_begin + a.l_per < a.L ? l_begin + a.l_per : a.L;
    DA da;
    DB db;
    da.init(a.R, sa.ld, row0, wr, wave, lane);
    db.init(a.C, sb.ld, col0, wc, wave, lane);
    f32x4 acc[TR][TC] = {};

    auto load = [&](char *la, char *lb, int64_t l0) {           // from l_end on: zeros
        da.load((const float *)sa.p, sa.ld, row0, l0, l_end, la, wave);
        db.load((const float *)sb.p, sb.ld, col0, l0, l_end, lb, wave);
    };
    auto parts = [](const float (&f)[8], bf16x8 (&p)[3]) {
        uint32_t w[3][4];
        split8(f, w[0], w[1], w[2]);
        __builtin_memcpy(p, w, sizeof w);
    };
    float fa[TR][8], fb[TC][8];
    bf16x8 pb[TC][3];
    // One step of 32: its fragments are in fa and fb, whose registers take the next step's as they are split.  The split of
    // row block i + 1 stands among the products of block i.
    auto step = [&](const char *na, const char *nb) {
        constexpr int READS_A = across(KA) ? 8 : 2, READS_B = across(KB) ? 8 : 2;
#pragma unroll
        for (int j = 0; j < TC; ++j) {
            parts(fb[j], pb[j]);
            db.read(nb, j, fb[j]);
            __builtin_amdgcn_sched_group_barrier(0x002, 44, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, READS_B, 0);
        }
        bf16x8 pa[2][3];
        parts(fa[0], pa[0]);
        da.read(na, 0, fa[0]);
        __builtin_amdgcn_sched_group_barrier(0x002, 44, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, READS_A, 0);
#pragma unroll
        for (int i = 0; i < TR; ++i) {
            if (i + 1 < TR) {
                parts(fa[i + 1], pa[(i + 1) & 1]);
                da.read(na, i + 1, fa[i + 1]);
            }
#pragma unroll
            for (int p = 2; p >= 0; --p)                          // small products first
#pragma unroll
                for (int q = 0; q <= p; ++q)
#pragma unroll
                    for (int j = 0; j < TC; ++j) {
                        acc[i][j] = Mma<float>::mul(pb[j][q], pa[i & 1][p - q], acc[i][j]);
                        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                        if (i + 1 < TR) __builtin_amdgcn_sched_group_barrier(0x002, 2, 0);
                    }
            if (i + 1 < TR) __builtin_amdgcn_sched_group_barrier(0x100, READS_A, 0);
        }
    };
    load(a0, b0, l_begin);
    load(a1, b1, l_begin + FK);
    arrive<0>();
#pragma unroll
    for (int i = 0; i < TR; ++i) da.read(a0, i, fa[i]);
#pragma unroll
    for (int j = 0; j < TC; ++j) db.read(b0, j, fb[j]);
#pragma unroll 1
    for (int64_t l0 = l_begin; l0 < l_end; l0 += 2 * FK) {
        arrive<0>();
        load(a0, b0, l0 + 2 * FK);
        __builtin_amdgcn_sched_barrier(0);
        step(a1, b1);
        arrive<0>();
        load(a1, b1, l0 + 3 * FK);
        __builtin_amdgcn_sched_barrier(0);
        step(a0, b0);
    }
    __builtin_amdgcn_s_waitcnt(0x0070);                         // the last loads and reads, before LDS is used again
    // an infinity's parts are infinity and NaN: a tile with NaNs is looked over for infinities
    bool nan = false;
#pragma unroll
    for (int i = 0; i < TR; ++i)
#pragma unroll
        for (int j = 0; j < TC; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) nan |= acc[i][j][q] != acc[i][j][q];
    if (__syncthreads_or(nan)) {
        const bool any = infinities<across(KA)>(sa, a.R, row0, l_begin, l_end) || infinities<across(KB)>(sb, a.C, col0, l_begin, l_end);
        if (__syncthreads_or(any)) plain_sums<float, KA, KB, TR, TC>(a, acc, row0 + wr, col0 + wc, l_begin, l_end, lane);
    }
    __syncthreads();
    write_out<float, KA == ALONG && KB == ALONG, TR, TC, 4>(a, acc, row0 + wr, col0 + wc, split, lane,
                                                            (float *)(wave == 0 ? a0 : wave == 1 ? a1 : wave == 2 ? b0 : b1));
}

// An operand for the direct kernels, [rows, cols] -> [rows, ldp], zeros behind cols.  src: x itself, dy with z or its
// derivative codes (dz = dy f'(z); with `partial`, also the partial column sums of dz in FP32), or an 8-bit checkpoint.
// rows_per rows a workgroup of 64 lanes (8 columns each) by 4 rows.  out may be NULL (db alone).  HBM bounds it: dz of
// 16384 x 4096 in BF16 from derivative codes 78 us (4.3 TB/s), an 8-bit x 42 us (4.8 TB/s).
enum Made { COPY, DZ, EIGHT };
struct PrepArgs {
    const void *src, *pre;
    const uint8_t *dcodes;
    const int8_t *codes;
    const uint8_t *scales;
    int act;
    int64_t rows, cols, ldp, rows_per, chunks, blocks;      // workgroups: chunks of rows by blocks of 512 columns
    void *out;
    float *partial;
};

template <class T, Made MADE>
__device__ __forceinline__ void prepare(const PrepArgs &a)
{
    __shared__ float lds[MADE == DZ ? 4 : 1][512];
    const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6;
    const int64_t col = ((int64_t)blockIdx.x * 64 + tx) * 8;
    const int n = (int)(a.cols - col < 8 ? a.cols - col : 8);
    const int64_t r0 = (int64_t)blockIdx.y * a.rows_per, r1 = r0 + a.rows_per < a.rows ? r0 + a.rows_per : a.rows;
    float sum[8] = {};
    auto rows = [&](auto full, auto act) {
        constexpr bool FULL = decltype(full)::value;              // the workgroup's lanes have 8 columns, or none
        constexpr int ACT = decltype(act)::value, U = 4;
        auto take = [&](auto *p) {                                // rows have at least 8 elements
            typedef std::remove_const_t<std::remove_pointer_t<decltype(p)>> E;
            if constexpr (FULL) return load_pack<E, 8>(p);
            else return load_ending<E, 8>(p, n, true);
        };
        const int64_t nb = (a.cols + 31) / 32;
        // U rows' loads together, the last ones again where fewer are left
        for (int64_t r = r0 + ty; r < r1; r += 4 * U) {
            Pack<T, 8> v[U], z[MADE == DZ ? U : 1];
            Pack<uint8_t, 8> c[MADE == DZ ? U : 1];
            Pack<int8_t, 8> q[MADE == EIGHT ? U : 1];
            int e[MADE == EIGHT ? U : 1];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t row = r + 4 * u < r1 ? r + 4 * u : r, at = row * a.cols + col;
                if constexpr (MADE == EIGHT) {
                    q[u] = take(a.codes + at);
                    e[u] = a.scales[row * nb + col / 32];
                } else v[u] = take((const T *)a.src + at);
            }
            if constexpr (MADE == DZ && ACT != AFIV_ACT_NONE) {
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int64_t row = r + 4 * u < r1 ? r + 4 * u : r, at = row * a.cols + col;
                    if (a.pre) z[u] = take((const T *)a.pre + at);
                    else c[u] = take(a.dcodes + at);
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (u > 0 && r + 4 * u >= r1) break;
                float f[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    if constexpr (MADE == EIGHT) f[i] = eight_value(q[u].v[i], e[u]);
                    else f[i] = (float)v[u].v[i];
                    if constexpr (MADE == DZ && ACT != AFIV_ACT_NONE) {
                        float y, d;
                        if (a.pre) act_both<ACT>((float)z[u].v[i], y, d);
                        else d = derivative_of_code<ACT>(c[u].v[i]);
                        f[i] *= d;
                    }
                    if (!FULL && i >= n) f[i] = 0.0f;
                    if constexpr (MADE == DZ) sum[i] += f[i];
                }
                if (MADE == DZ && !a.out) continue;
                Pack<T, 8> b;
#pragma unroll
                for (int i = 0; i < 8; ++i) b.v[i] = (T)f[i];
                store_pack<T, 8>((T *)a.out + (r + 4 * u) * a.ldp + col, b);
            }
        }
    };
    auto with = [&](auto act) {
        if (n <= 0) return;
        if (a.cols % 8 == 0 || (int64_t)(blockIdx.x + 1) * 512 <= a.cols) rows(std::true_type(), act);
        else rows(std::false_type(), act);
    };
    if constexpr (MADE == DZ) with_act(a.act, with);
    else with(std::integral_constant<int, AFIV_ACT_NONE>());
    if constexpr (MADE == DZ) {
        if (!a.partial) return;
#pragma unroll
        for (int i = 0; i < 8; ++i) lds[ty][tx * 8 + i] = sum[i];
        __syncthreads();
        for (int c = threadIdx.x; c < 512; c += THREADS)
            if ((int64_t)blockIdx.x * 512 + c < a.cols)
                a.partial[(int64_t)blockIdx.y * a.cols + (int64_t)blockIdx.x * 512 + c] = (lds[0][c] + lds[1][c]) + (lds[2][c] + lds[3][c]);
    }
}

template <class T, Made MADE>
__global__ __launch_bounds__(THREADS) void prepare_kernel(PrepArgs a)
{
    prepare<T, MADE>(a);
}

// both operands of a forward product in one launch
template <class T>
__global__ __launch_bounds__(THREADS) void prepare_two_kernel(PrepArgs a, PrepArgs b)
{
    const PrepArgs &p = blockIdx.z == 0 ? a : b;
    if ((int64_t)blockIdx.x < p.blocks && (int64_t)blockIdx.y < p.chunks) prepare<T, COPY>(p);      // the same for the workgroup
}

// db from the partial sums: 16 columns a workgroup, 16 threads each over the chunks
template <class T>
__global__ __launch_bounds__(THREADS) void db_kernel(const float *__restrict__ partial, int64_t chunks, int64_t N, T *__restrict__ db)
{
    __shared__ float lds[16][16];
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    const int64_t col = (int64_t)blockIdx.x * 16 + tx;
    float s = 0.0f;
    if (col < N)
        for (int64_t c = ty; c < chunks; c += 16) s += partial[c * N + col];
    lds[ty][tx] = s;
    __syncthreads();
    if (ty == 0 && col < N) {
        for (int i = 1; i < 16; ++i) s += lds[i][tx];
        db[col] = (T)s;
    }
}

// ---- few rows ----------------------------------------------------------------------------------
// 16 GROUPS rows of A (stored along l) against 16 rows of B a workgroup: the matrix instruction's 16 columns
// are rows of A, its rows those of B, and both operands go from memory to registers 16 bytes a lane, four
// steps' loads together (FP32 by its own matrix instruction: memory, not arithmetic, bounds this).  The workgroup's
// waves take steps of l in turn and are summed in LDS, wave by wave.  It reads A again for every 16 columns and B for
// every 32 rows, so beyond 32 rows only products too small for that to matter take it: one round of loads, where
// a tile waits for one after the other.  One row of 4096 -> 4096 in BF16: 8.7 us (3.9 TB/s); 100 rows of 128 -> 64 in
// FP32: 4.1 us.
template <class T, int WAVES, int GROUPS>
__global__ __launch_bounds__(64 * WAVES) void few_rows_kernel(LinArgs a)
{
    constexpr int STEP = 32, U = 4;
    __shared__ float part[WAVES][16][16 * GROUPS + 1];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, sub = (lane >> 4) * 8;
    const int64_t col0 = (int64_t)blockIdx.x * 16, col = col0 + (lane & 15), row0 = (int64_t)blockIdx.y * 16 * GROUPS;
    // lanes beyond the matrices read a row inside: what they multiply is not stored
    const T *pb = (const T *)a.B + (col < a.C ? col : a.C - 1) * a.L, *pa[GROUPS];
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
        const int64_t row = row0 + g * 16 + (lane & 15);
        pa[g] = (const T *)a.A + (row < a.R ? row : a.R - 1) * a.L;
    }
    f32x4 acc[GROUPS] = {};
    auto multiply = [&](const Pack<T, 8> &vb, const Pack<T, 8> &va, f32x4 &c) {
        if constexpr (sizeof(T) == 2) {
            typename Mma<T>::frag fa, fb;
            __builtin_memcpy(&fa, &va, 16);
            __builtin_memcpy(&fb, &vb, 16);
            c = Mma<T>::mul(fb, fa, c);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(vb.v[i], va.v[i], c, 0, 0, 0);
        }
    };
    int64_t l = (int64_t)wave * STEP;                          // the same for the wave's lanes
    for (; l + (U - 1) * WAVES * STEP + STEP <= a.L; l += U * WAVES * STEP) {
        Pack<T, 8> vb[U], va[U][GROUPS];
#pragma unroll
        for (int u = 0; u < U; ++u) vb[u] = load_pack<T, 8>(pb + l + u * WAVES * STEP + sub);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int g = 0; g < GROUPS; ++g) va[u][g] = load_pack<T, 8>(pa[g] + l + u * WAVES * STEP + sub);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int g = 0; g < GROUPS; ++g) multiply(vb[u], va[u][g], acc[g]);
    }
    for (; l < a.L; l += WAVES * STEP) {
        const int n = (int)(a.L - l - sub < 8 ? a.L - l - sub : 8);
        Pack<T, 8> vb = {};
        if (n > 0) vb = load_some<T, 8>(pb + l + sub, n);
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
            Pack<T, 8> va = {};
            if (n > 0) va = load_some<T, 8>(pa[g] + l + sub, n);
            multiply(vb, va, acc[g]);
        }
    }
#pragma unroll
    for (int g = 0; g < GROUPS; ++g)
#pragma unroll
        for (int q = 0; q < 4; ++q) part[wave][(lane >> 4) * 4 + q][g * 16 + (lane & 15)] = acc[g][q];
    __syncthreads();
    if (wave < GROUPS) {                                       // a wave a group; lane: row = lane & 15, four columns
        const int64_t row = row0 + wave * 16 + (lane & 15), j = col0 + (lane >> 4) * 4;
        float z[4] = {};
#pragma unroll
        for (int w = 0; w < WAVES; ++w)
#pragma unroll
            for (int q = 0; q < 4; ++q) z[q] += part[w][(lane >> 4) * 4 + q][wave * 16 + (lane & 15)];
        if (row < a.R && j < a.C) finish<T, true, 4>(a, row, j, z);
    }
}

// ---- launches ----------------------------------------------------------------------------------
int ok() { return hipGetLastError() == hipSuccess ? AFIV_OK : AFIV_E_HIP; }

template <class T, bool EPI>
void join(const LinArgs &a, hipStream_t s)
{
    const int64_t units = a.R * ((a.C + 3) / 4) + (a.db ? a.R : 0);
    auto blocks = [&](int64_t per) { return dim3((unsigned)std::min<int64_t>((units + per - 1) / per, 4096)); };
    if (a.splits > 16) hipLaunchKernelGGL((join_kernel<T, EPI, 16>), blocks(THREADS / 16), dim3(THREADS), 0, s, a);
    else hipLaunchKernelGGL((join_kernel<T, EPI, 1>), blocks(THREADS), dim3(THREADS), 0, s, a);
}

// the tile kernel's part of a product's arguments; returns its workgroups
int64_t tiled(LinArgs &a, float *scratch)
{
    const Plan p = plan_for(a.R, a.C, a.L);
    a.splits = p.splits;
    a.l_per = p.l_per;
    a.partial = scratch;
    a.db_partial = scratch + p.splits * a.R * a.C;
    return p.tiles * p.splits;
}

template <class T, Kind KA, Kind KB>
int product(LinArgs a, float *scratch, hipStream_t s)
{
    const int64_t blocks = tiled(a, scratch);
    if (blocks == 0) return AFIV_OK;
    hipLaunchKernelGGL((tile_kernel<T, KA, KB>), dim3((unsigned)blocks), dim3(THREADS), 0, s, a);
    if (a.splits > 1) join<T, KA == ALONG>(a, s);
    return ok();
}

// both backward products (d: dx, e: dW), neither empty
template <class T, Kind KX>
int products(LinArgs d, LinArgs e, float *scratch, hipStream_t s)
{
    const int64_t blocks = tiled(d, scratch), more = tiled(e, scratch + tile_floats(d.R, d.C, d.L));
    hipLaunchKernelGGL((both_kernel<T, KX>), dim3((unsigned)(blocks + more)), dim3(THREADS), 0, s, d, e, blocks);
    if (d.splits > 1) join<T, false>(d, s);
    if (e.splits > 1) join<T, false>(e, s);
    return ok();
}

// db of e (dW's arguments, of which dW is not wanted) and dx, if d describes it
template <class T>
int db_alone(const LinArgs *d, LinArgs e, float *scratch, hipStream_t s)
{
    tiled(e, d ? scratch + tile_floats(d->R, d->C, d->L) : scratch);
    const int64_t blocks = (e.R + 127) / 128 * e.splits;
    if (d) {
        LinArgs dx = *d;
        const int64_t dx_blocks = tiled(dx, scratch);
        hipLaunchKernelGGL(dx_db_kernel<T>, dim3((unsigned)(dx_blocks + blocks)), dim3(THREADS), 0, s, dx, e, dx_blocks);
        if (dx.splits > 1) join<T, false>(dx, s);
    } else hipLaunchKernelGGL(db_alone_kernel<T>, dim3((unsigned)blocks), dim3(THREADS), 0, s, e);
    if (e.splits > 1)
        hipLaunchKernelGGL(db_kernel<T>, dim3((unsigned)((e.R + 15) / 16)), dim3(THREADS), 0, s, e.db_partial, e.splits, e.R, (T *)e.db);
    return ok();
}

template <class T, Kind KA, Kind KB>
int direct(LinArgs a, const Source &sa, const Source &sb, float *scratch, hipStream_t s)
{
    const Plan p = direct_plan(a.R, a.C, a.L, sizeof(T) == 4);
    a.splits = p.splits;
    a.l_per = p.l_per;
    a.partial = scratch;
    a.db = nullptr;
    const dim3 grid((unsigned)(p.tiles * p.splits));
    if constexpr (sizeof(T) == 4) hipLaunchKernelGGL((direct32_kernel<KA, KB>), grid, dim3(256), 0, s, a, sa, sb);
    else if (huge_tiles(a.R, a.C)) hipLaunchKernelGGL((direct_kernel<T, KA, KB, 2, 4, 8, 4, false>), grid, dim3(512), 0, s, a, sa, sb);
    else if (p.tiles * p.splits <= CUS) hipLaunchKernelGGL((direct_kernel<T, KA, KB, 2, 4, 4, 2, true>), grid, dim3(512), 0, s, a, sa, sb);
    else hipLaunchKernelGGL((direct_kernel<T, KA, KB, 2, 4, 4, 2, false>), grid, dim3(512), 0, s, a, sa, sb);
    if (p.splits > 1) join<T, KA == ALONG && KB == ALONG>(a, s);
    return ok();
}

// how an operand is written to `room`, and how the direct kernel reads it
template <class T>
Source placed(PrepArgs &a, const Room &room, char *scratch, float *partial, bool write)
{
    a.blocks = (a.cols + 511) / 512;
    a.chunks = prep_chunks(a.rows, a.cols);
    a.ldp = padded(a.cols);
    a.rows_per = (a.rows + a.chunks - 1) / a.chunks;
    a.out = write ? scratch + room.at : nullptr;
    a.partial = partial;
    const Source o = {a.out, a.ldp};
    return o;
}
template <class T, Made MADE>
Source prepared(PrepArgs a, const Room &room, char *scratch, float *partial, bool write, hipStream_t s)
{
    const Source o = placed<T>(a, room, scratch, partial, write);
    hipLaunchKernelGGL((prepare_kernel<T, MADE>), dim3((unsigned)a.blocks, (unsigned)a.chunks), dim3(THREADS), 0, s, a);
    return o;
}

// an operand that may be read where it stands
Source standing(const void *p, int64_t ld)
{
    const Source o = {p, ld};
    return o;
}
PrepArgs copy_of(const void *p, int64_t rows, int64_t cols)
{
    PrepArgs q = {};
    q.src = p; q.rows = rows; q.cols = cols;
    return q;
}
template <class T>
Source plain_source(const void *p, int64_t rows, int64_t cols, const Room &room, char *scratch, hipStream_t s)
{
    return room.bytes ? prepared<T, COPY>(copy_of(p, rows, cols), room, scratch, nullptr, true, s) : standing(p, cols);
}

template <class T>
int forward(const LinArgs &a, float *scratch, hipStream_t s)
{
    if (few_rows(a.R, a.C, a.L)) {
        const dim3 grid((unsigned)((a.C + 15) / 16), (unsigned)((a.R + 31) / 32));
        // 16 waves where the layer has few workgroups to fill the chip with
        const bool many = grid.x * grid.y < 512 && a.L >= 512;
        if (a.R <= 16) {
            if (many) hipLaunchKernelGGL((few_rows_kernel<T, 16, 1>), grid, dim3(1024), 0, s, a);
            else hipLaunchKernelGGL((few_rows_kernel<T, 4, 1>), grid, dim3(256), 0, s, a);
        } else {
            if (many) hipLaunchKernelGGL((few_rows_kernel<T, 16, 2>), grid, dim3(1024), 0, s, a);
            else hipLaunchKernelGGL((few_rows_kernel<T, 4, 2>), grid, dim3(256), 0, s, a);
        }
        return ok();
    }
    const Places p = forward_places(a.R, a.C, a.L, sizeof(T) == 4);
    if (p.direct && (p.x.bytes || aligned(a.A)) && (p.w.bytes || aligned(a.B)) && aligned(scratch)) {
        if (!p.x.bytes) return direct<T, ALONG, ALONG>(a, standing(a.A, a.L), standing(a.B, a.L), scratch, s);
        char *at = (char *)scratch;
        PrepArgs qx = copy_of(a.A, a.R, a.L), qw = copy_of(a.B, a.C, a.L);
        const Source x = placed<T>(qx, p.x, at, nullptr, true), w = placed<T>(qw, p.w, at, nullptr, true);
        hipLaunchKernelGGL(prepare_two_kernel<T>, dim3((unsigned)std::max(qx.blocks, qw.blocks), (unsigned)std::max(qx.chunks, qw.chunks), 2),
                           dim3(THREADS), 0, s, qx, qw);
        return direct<T, ALONG, ALONG>(a, x, w, scratch, s);
    }
    return product<T, ALONG, ALONG>(a, scratch, s);
}

template <class T>
int backward(const void *dy, const void *x, const int8_t *codes, const uint8_t *scales, const void *w, const void *pre,
             const uint8_t *dcodes, int act, int64_t M, int64_t N, int64_t K, void *dx, void *dw, void *db, float *scratch, hipStream_t s)
{
    if (act == AFIV_ACT_NONE) {
        pre = nullptr;
        dcodes = nullptr;
    }
    LinArgs a = {};
    a.A = dy; a.act = act; a.pre = pre; a.dcodes = dcodes;
    LinArgs d = a, e = a;
    d.B = w; d.R = M; d.C = K; d.L = N; d.out = dx;
    e.B = x; e.codes = codes; e.scales = scales; e.R = N; e.C = K; e.L = M; e.out = dw; e.db = db;

    // operands that the direct kernel cannot read in place are written first; a misaligned one of a kind that it
    // could sends the product to the tile kernel
    constexpr int WHOLE = 16 / sizeof(T);
    const Places p = backward_places(M, N, K, sizeof(T) == 4, act != AFIV_ACT_NONE, dw && !x);
    char *const at = (char *)scratch;
    const bool make_dz = act != AFIV_ACT_NONE || N % WHOLE, make_x = codes || K % WHOLE;
    const bool ready = aligned(scratch) && (make_dz || aligned(dy));
    const bool direct_dx = dx && p.direct && ready && (p.w.bytes || aligned(w));
    const bool direct_dw = dw && p.direct_dw && ready && (make_x || aligned(x));
    Source g = standing(dy, N);
    // db as column sums of the pass that makes dz: beside a direct dW, or where no dW is asked for (tiles would multiply
    // all of dz by x for it: 16384 x 4096 x 4096 in bf16 11.9 ms, 75 us here)
    const bool sums = db && p.direct_dw && ready && (direct_dw || !dw), write = make_dz && (direct_dx || direct_dw);
    if (write || sums) {
        float *const partial = sums ? (float *)(at + p.db) : nullptr;
        PrepArgs q = {};
        q.src = dy; q.pre = pre; q.dcodes = dcodes; q.act = act; q.rows = M; q.cols = N;
        const Source made = prepared<T, DZ>(q, p.dz, at, partial, write, s);
        if (write) g = made;
        if (sums) hipLaunchKernelGGL(db_kernel<T>, dim3((unsigned)((N + 15) / 16)), dim3(THREADS), 0, s, partial, prep_chunks(M, N), N, (T *)db);
    }
    int rc = ok();
    const bool only_db = !dw && db && !sums;                     // the input may be missing: no product with it
    const bool joint = dx && M > 0 && one_launch(M, N, K);
    if (!rc && joint && only_db && !direct_dx) return db_alone<T>(&d, e, scratch, s);
    if (!rc && joint && dw && !direct_dx && !direct_dw)
        return codes ? products<T, ACROSS_EIGHT>(d, e, scratch, s) : products<T, ACROSS>(d, e, scratch, s);
    if (!rc && dx) {
        if (direct_dx) rc = direct<T, ALONG_DZ, ACROSS>(d, g, plain_source<T>(w, N, K, p.w, at, s), scratch, s);
        else rc = product<T, ALONG_DZ, ACROSS>(d, scratch, s);
    }
    if (!rc && only_db) rc = db_alone<T>(nullptr, e, scratch, s);
    if (rc || !dw) return rc;
    if (!direct_dw) return codes ? product<T, ACROSS_DZ, ACROSS_EIGHT>(e, scratch, s) : product<T, ACROSS_DZ, ACROSS>(e, scratch, s);
    if (!codes) {
        const Room none = {};
        return direct<T, ACROSS_DZ, ACROSS>(e, g, plain_source<T>(x, M, K, make_x ? p.x : none, at, s), scratch, s);
    }
    PrepArgs q = {};
    q.codes = codes; q.scales = scales; q.rows = M; q.cols = K;
    const Source xs = prepared<T, EIGHT>(q, p.x, at, nullptr, true, s);
    if constexpr (sizeof(T) == 4) return direct<T, ACROSS_DZ, ACROSS_EIGHT>(e, g, xs, scratch, s);
    else return direct<T, ACROSS_DZ, ACROSS>(e, g, xs, scratch, s);
}

// ---- one translation unit per element type instantiates these ------------------------------------
template <class T>
int linear_forward(const void *x, const void *w, const void *bias, const void *residual, int act, int64_t M, int64_t N, int64_t K, void *y,
                   void *pre, uint8_t *dcodes, float *scratch, hipStream_t s)
{
    LinArgs a = {};
    a.A = x; a.B = w; a.R = M; a.C = N; a.L = K;
    a.bias = bias; a.residual = residual; a.act_out = act; a.out = y; a.pre_out = pre; a.dcodes_out = dcodes;
    return forward<T>(a, scratch, s);
}

}  // namespace

#define AFIV_LINEAR_TYPE(T, NAME)                                                                                                      \
    int afiv_linear_forward_##NAME(const void *x, const void *w, const void *bias, const void *residual, int act, int64_t M, int64_t N, \
                                   int64_t K, void *y, void *pre, uint8_t *dcodes, float *scratch, hipStream_t s)                       \
    {                                                                                                                                  \
        return linear_forward<T>(x, w, bias, residual, act, M, N, K, y, pre, dcodes, scratch, s);                                      \
    }                                                                                                                                  \
    int afiv_linear_backward_##NAME(const void *dy, const void *x, const int8_t *codes, const uint8_t *scales, const void *w,           \
                                    const void *pre, const uint8_t *dcodes, int act, int64_t M, int64_t N, int64_t K, void *dx,        \
                                    void *dw, void *db, float *scratch, hipStream_t s)                                                 \
    {                                                                                                                                  \
        return backward<T>(dy, x, codes, scales, w, pre, dcodes, act, M, N, K, dx, dw, db, scratch, s);                                \
    }
