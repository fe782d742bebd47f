// cuddle_rows_plan.hpp — sizes of 4-bit rows and the rules that pick a distance kernel's shape. Plain C++, so that a host
// program can walk them over every size.
#pragma once

#include <cstdint>

namespace cuddle {

constexpr uint32_t kInt4Unit = 64;      // components per unit
constexpr uint32_t kInt4UnitBytes = 512; // 16 rows x 32 bytes

constexpr uint32_t int4_units(uint32_t dim) { return (dim + kInt4Unit - 1) / kInt4Unit; }
constexpr uint32_t int4_gstride(uint32_t dim, uint32_t group) {
    const uint32_t groups = (dim + group - 1) / group, m = groups > 4 ? 8 : groups > 2 || group == 32 ? 4 : 2;
    return (groups + m - 1) / m * m;
}

// Threads. Five and eight quartets of one tile: sixteen waves around one copy of the digits (1M x 960, 64 queries: 431 us,
// 625 with eight waves of two tiles each; 20 queries: 207 and 252).
constexpr int int4_block(int qt, int t) { return qt >= 5 && t == 1 ? 1024 : qt >= 3 ? 512 : 256; }

constexpr uint32_t int4_lds_kb(int qt) { return qt >= 5 ? 128u : qt >= 3 ? 144u : 64u; } // digits per block: one large block per CU, or several
// Up to four queries whose digits fit a block's LDS: the distance kernel makes them itself. A round of a call is fused if
// its queries are this few, so a call of more queries lays out room for digits also for a last, smaller round.
constexpr bool int4_fused(uint64_t nq, uint32_t dim) { return nq <= 4 && (int4_units(dim) + 7) / 8 * 8 <= int4_lds_kb(1); }

// Scales that a lane loads at once beside `p` units. A row of scales has to be a multiple of that, or the load takes in the
// next row's and, behind the last row, what is not the array's.
constexpr uint32_t int4_scales(int p, uint32_t group) { return (uint32_t)p * 64 / group; }

// Launch shapes of the distance kernel: a wave takes `t` tiles against `qt` quartets of queries, codes of `p` units at a
// time. One quartet of queries: codes are the bound, so many of them are requested at a time (four pieces of 1 KB per
// wave; short rows: more tiles and fewer units). More: `qt` quartets per wave, the count among those built that costs least.
// A wave's pass over its codes unpacks them once and multiplies them qt times; unpacking, addresses and the wait cost
// about as much as three quartets' products (1M x 960, one pass: 140 us with 5 quartets, 190 with 8, 114 with 4, 98 with
// 3). 20 queries: 161 us with 5, 210 with 8; 64: 401 with 8, 498 with 5, 471 with 4; 100: 682 with 5, 730 with 8, 779
// with 4. Six and seven quartets were built and won nowhere by more than 4 %. Digits that do not fit the block's LDS at
// once are fetched anew for every 256 rows, from the L2, and change nothing in the order (100k x 4096, 64 queries: 221 us
// with 8, 264 with 5, 289 with 4).
// Rows of one or two units have one pair of units to request ahead, and their scales are too few for more (int4_scales).
// Five quartets then take two tiles, which keeps the wave busy (1M x 128, 100 queries: 245 us against 295; from 192
// dimensions on equal or slower, 100k x 4096: 455 against 345); with eight, two tiles do not fit the registers. Eight
// against five for such rows (1M x 128; search, k = 10: 64 queries 132 us and 137, 128 207 and 221, 200 345 and 308, 1000
// 1200 and 1560; distances, mostly their own writes, 267 and 290 at 101, 345 and 334 at 128, 522 and 445 at 200). The rule is
// kept the same for all rows; 160 to 200 queries are where it loses on such short ones.
struct Int4Shape {
    int qt, t, p;
};
constexpr Int4Shape int4_shape(uint32_t units, uint32_t nq, bool fused) {
    if (fused) return units < 6 ? Int4Shape{1, 4, 2} : Int4Shape{1, 2, 4};
    const uint32_t quads = (nq + 3) / 4;
    int best = 1;
    uint32_t cost = ~0u; // (of equal costs the larger: its codes are unpacked less often)
    for (int qt : {1, 2, 3, 4, 5, 8}) {
        const uint32_t c = (quads + qt - 1) / qt * (qt + 3);
        if (c <= cost) {
            cost = c;
            best = qt;
        }
    }
    if (best == 1) return {1, 4, 2};
    if (best < 5) return {best, 2, 2};
    if (units < 3) return {best, best == 5 ? 2 : 1, 2};
    return {best, 1, 4};
}

} // namespace cuddle
