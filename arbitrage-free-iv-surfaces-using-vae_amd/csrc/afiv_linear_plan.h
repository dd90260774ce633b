// How the linear layer's products are cut into tiles and runs, and the scratch memory that takes: shared by the
// launches (afiv_linear_kernels.h) and the size queries.
#pragma once

#include <algorithm>
#include <cstdint>

#include "afiv.h"

namespace {

constexpr int BK = 32;                    // steps of l in LDS, tile kernel
constexpr int CUS = 256;

// the few-rows kernel's products
bool few_rows(int64_t R, int64_t C, int64_t L)
{
    return R > 0 && (R <= 32 || (R <= 4096 && (double)R * (double)C * (double)L <= 1 << 21));
}

int64_t tiles_of(int64_t R, int64_t C, int64_t t) { return ((R + t - 1) / t) * ((C + t - 1) / t); }

struct Plan { int64_t tiles, splits, l_per; };

// runs of l: with fewer than `few` tiles the sum is cut, for `want` workgroups, into runs of at least `least` steps
Plan cut(int64_t tiles, int64_t L, int64_t step, int64_t few, int64_t want, int64_t least)
{
    Plan p = {tiles, 1, 1};
    const int64_t steps = (L + step - 1) / step;
    if (tiles > 0 && tiles < few && steps >= 2 * least) p.splits = std::min(want / tiles, steps / least);
    p.l_per = std::max<int64_t>(1, (steps + p.splits - 1) / p.splits) * step;
    p.splits = std::max<int64_t>(1, (L + p.l_per - 1) / p.l_per);
    return p;
}

// Tile kernel: 64 x 64 tiles; below 256 workgroups the sum is cut into runs of at least 256 steps.
Plan plan_for(int64_t R, int64_t C, int64_t L) { return cut(tiles_of(R, C, 64), L, BK, 256, 512, 8); }

// Both backward products in one launch: it has fewer than 2^32 work items, 256 a workgroup, and each product alone may
// come near that.
bool one_launch(int64_t M, int64_t N, int64_t K)
{
    const Plan dx = plan_for(M, K, N), dw = plan_for(N, K, M);
    return dx.tiles * dx.splits + dw.tiles * dw.splits < 1 << 24;
}

// The direct kernel: 256 x 256 tiles where they fill the chip at least once and little of them lies outside the matrix
// (131072 x 128 x 128, bf16: 26 us by 128 x 128 tiles, 46 by the large ones), else 128 x 128 (FP32: always).  Below 96
// tiles the sum is cut, 16 bit for one workgroup a CU with four buffers, FP32 for two with two; above, the kernel that
// joins the runs costs more than the idle CUs.
bool huge_tiles(int64_t R, int64_t C) { return tiles_of(R, C, 256) >= CUS && 16 * tiles_of(R, C, 256) <= 5 * tiles_of(R, C, 128); }
Plan direct_plan(int64_t R, int64_t C, int64_t L, bool f32)
{
    if (f32) return cut(tiles_of(R, C, 128), L, 32, 96, 512, 8);
    return huge_tiles(R, C) ? cut(tiles_of(R, C, 256), L, 64, 0, 0, 1) : cut(tiles_of(R, C, 128), L, 64, 96, CUS, 8);
}

// What the direct kernel takes: at least a tile each way, rows within 2^31 bytes of a tile's corner, and enough work that
// its few, large tiles fill the chip.  us in a captured graph, by it and by the tile kernel, forward / dx / dW:
//   16 bit, whole rows   256^3  6.1 6.7 / 7.5 10 / 7.7 13       512^3  7.7 10.7 / 9.2 13.7 / 9.6 16.6     1024^3  17 17 / 17 31 / 17 43
//   16 bit, ragged rows  300^3  11.6 10.4 / 14.5 14.4 / 15 21   777 x 333 x 500  13 10.5 / 15.9 17 / 19.5 26
//   FP32                 512^3  20 14 / 21 17 / 20 22           768^3  25 20.5 / 25 23 / 24.5 27          1024^3  31 31 / 31 43 / 31 62
// One threshold a type stands for all of these: 16 bit, between whole rows, which it does faster from 2^24 on, and ragged
// ones, which a pass has to write out for it first; FP32, where dW gains (2^27) before dx and the forward product do (2^30).
bool direct_takes(int64_t R, int64_t C, int64_t L, bool f32)
{
    return R >= 128 && C >= 128 && L >= 128 && (double)R * (double)C * (double)L >= (f32 ? 1 << 28 : 1 << 27);
}
bool direct_rows(int64_t len) { return len <= 1 << 20; }
bool aligned(const void *p) { return ((uintptr_t)p & 15) == 0; }

// floats that the tile kernel's split takes, and either kernel's
int64_t tile_floats(int64_t R, int64_t C, int64_t L)
{
    const Plan p = plan_for(R, C, L);
    return p.splits > 1 ? p.splits * (R * C + R) : 0;
}
int64_t scratch_floats(int64_t R, int64_t C, int64_t L, bool f32)
{
    const Plan d = direct_plan(R, C, L, f32);
    return std::max(tile_floats(R, C, L), d.splits > 1 ? d.splits * R * C : 0);
}

// Scratch of a call: the splits' floats, then the operands written for the direct kernel, then the partial sums of db.
int64_t padded(int64_t cols) { return (cols + 7) / 8 * 8; }
constexpr int64_t PREP_CHUNKS = 256;
int64_t prep_chunks(int64_t rows, int64_t cols)
{
    const int64_t cb = (cols + 511) / 512;
    return std::max<int64_t>(1, std::min(PREP_CHUNKS, std::min((2048 + cb - 1) / cb, (rows + 15) / 16)));
}
struct Room { int64_t at, bytes; };
struct Places { bool direct, direct_dw; Room x, w, dz; int64_t db, bytes; };      // direct: the forward product, or dx's

Room place(int64_t &end, bool wanted, int64_t rows, int64_t cols, bool f32)
{
    Room r = {0, 0};
    if (!wanted) return r;
    r.at = (end + 255) / 256 * 256;
    r.bytes = rows * padded(cols) * (f32 ? 4 : 2);
    end = r.at + r.bytes;
    return r;
}

Places forward_places(int64_t M, int64_t N, int64_t K, bool f32)
{
    Places p = {};
    if (few_rows(M, N, K)) return p;
    p.bytes = scratch_floats(M, N, K, f32) * 4;
    p.direct = direct_takes(M, N, K, f32) && direct_rows(K);
    const bool make = p.direct && K % (f32 ? 4 : 8);
    p.x = place(p.bytes, make, M, K, f32);
    p.w = place(p.bytes, make, N, K, f32);
    return p;
}

// act: dz differs from dy; eight: x is a checkpoint
Places backward_places(int64_t M, int64_t N, int64_t K, bool f32, bool act, bool eight)
{
    const int64_t whole = f32 ? 4 : 8;                   // elements of 16 bytes
    Places p = {};
    p.bytes = std::max(std::max(scratch_floats(M, K, N, f32), scratch_floats(N, K, M, f32)), tile_floats(M, K, N) + tile_floats(N, K, M)) * 4;
    p.direct = direct_takes(M, K, N, f32) && direct_rows(N) && direct_rows(K);
    p.direct_dw = direct_takes(N, K, M, f32) && direct_rows(N) && direct_rows(K);
    p.dz = place(p.bytes, (p.direct || p.direct_dw) && (act || N % whole), M, N, f32);
    p.x = place(p.bytes, p.direct_dw && (eight || K % whole), M, K, f32);
    p.w = place(p.bytes, p.direct && K % whole, N, K, f32);
    p.db = (p.bytes + 255) / 256 * 256;
    if (p.direct_dw) p.bytes = p.db + PREP_CHUNKS * N * 4;
    return p;
}

}  // namespace
