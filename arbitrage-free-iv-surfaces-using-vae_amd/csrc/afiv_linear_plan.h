// How the linear layer's products are cut into tiles and runs, and the scratch memory that takes: shared by the
// launches (afiv_linear_kernels.h) and the size queries.
#pragma once

#include <algorithm>
#include <cstdint>

#include "afiv.h"

namespace {

constexpr int BK = 32;                    // steps of l in LDS, tile kernel
constexpr int FK = 64;                    // and direct kernel
constexpr int FEW = 16;                   // rows of the few-rows kernel

int64_t tiles_of(int64_t R, int64_t C, int64_t t) { return ((R + t - 1) / t) * ((C + t - 1) / t); }

struct Plan { int64_t tiles, splits, l_per; };

// runs of l: below `want` workgroups the sum is cut, into runs of at least `least` steps
Plan cut(int64_t tiles, int64_t L, int64_t step, int64_t want, int64_t least)
{
    Plan p = {tiles, 1, 1};
    const int64_t steps = (L + step - 1) / step;
    if (tiles > 0 && tiles < want / 2 && steps >= 2 * least) p.splits = std::min((want + tiles - 1) / tiles, steps / least);
    p.l_per = std::max<int64_t>(1, (steps + p.splits - 1) / p.splits) * step;
    p.splits = std::max<int64_t>(1, (L + p.l_per - 1) / p.l_per);
    return p;
}

// Tile and split of a product of R x C outputs and L steps.  128 x 128 tiles once they give every CU
// one; below that 64 x 64, and below 512 workgroups the sum is cut into runs of at least 256 steps.
bool big_tiles(int64_t R, int64_t C) { return tiles_of(R, C, 128) >= 256; }
Plan plan_for(int64_t R, int64_t C, int64_t L) { return cut(tiles_of(R, C, big_tiles(R, C) ? 128 : 64), L, BK, 512, 8); }

// The direct kernel: 256 x 256 tiles where they fill the chip at least once, else 128 x 128 (cut like the above).
bool huge_tiles(int64_t R, int64_t C) { return tiles_of(R, C, 256) >= 256; }
Plan direct_plan(int64_t R, int64_t C, int64_t L)
{
    return huge_tiles(R, C) ? cut(tiles_of(R, C, 256), L, FK, 0, 1) : cut(tiles_of(R, C, 128), L, FK, 512, 8);
}

// what the direct kernel takes: rows of whole 16-byte chunks within 2^31 bytes of a tile's corner, and enough
// work that its tiles are not mostly padding
bool direct_rows(int64_t len) { return len % 8 == 0 && len <= (1 << 21); }
bool direct_pays(int64_t R, int64_t C, int64_t L) { return R >= 128 && C >= 128 && L >= 128 && R * C >= 128 * 128 * 32; }
bool aligned(const void *p) { return ((uintptr_t)p & 15) == 0; }

// floats that either kernel's split takes
int64_t scratch_floats(int64_t R, int64_t C, int64_t L)
{
    const Plan p = plan_for(R, C, L), d = direct_plan(R, C, L);
    return std::max(p.splits > 1 ? p.splits * (R * C + R) : 0, d.splits > 1 ? d.splits * R * C : 0);
}

// The backward pass by the direct kernel: dz and, from a checkpoint, x are written to memory first (they are read
// by many tiles; the products are long), 16-byte aligned behind the splits' floats.
int64_t align16(int64_t bytes) { return (bytes + 15) / 16 * 16; }
constexpr int64_t DB_CHUNKS = 256;
bool direct_backward(int64_t M, int64_t N, int64_t K)
{
    return direct_rows(N) && direct_rows(K) && direct_pays(M, K, N) && direct_pays(N, K, M);
}
struct Places { int64_t floats, dz, x, db, bytes; };
Places places(int64_t M, int64_t N, int64_t K)
{
    Places p;
    p.floats = 0;
    p.dz = align16(std::max(scratch_floats(M, K, N), scratch_floats(N, K, M)) * 4);
    const bool direct = direct_backward(M, N, K);
    p.x = p.dz + (direct ? M * N * 2 : 0);              // N, K multiples of 8: aligned
    p.db = p.x + (direct ? M * K * 2 : 0);
    p.bytes = p.db + (direct ? DB_CHUNKS * N * 4 : 0);
    return p;
}

}  // namespace
