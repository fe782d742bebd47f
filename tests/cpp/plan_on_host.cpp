// Walks the launch rule of the 4-bit distances (vectordb_amd/csrc/cuddle_rows_plan.hpp) over all dimensions, groups and up
// to 4096 queries: whatever shape is picked, what a lane loads of a row's scales is the row's own and aligned.
#include <cstdio>
#include <set>

#include "cuddle_rows_plan.hpp"

using namespace cuddle;

int main() {
    unsigned long bad = 0, seen = 0;
    for (uint32_t units = 1; units <= 512; ++units) {
        std::set<int> pieces;
        for (uint32_t nq = 1; nq <= 4096; ++nq)
            for (bool fused : {false, true})
                if (!fused || int4_fused(nq, units * kInt4Unit)) pieces.insert(int4_shape(units, nq, fused).p);
        for (uint32_t dim = (units - 1) * kInt4Unit + 1; dim <= units * kInt4Unit; ++dim)
            for (uint32_t group : {32u, 64u, 128u})
                for (int p : pieces) {
                    const uint32_t gs = int4_gstride(dim, group), sc = int4_scales(p, group), last = (units - 1) / p * p;
                    ++seen;
                    if (sc && (uint32_t)p * 64 % group == 0 && gs % sc == 0 && last * 64 / group + sc <= gs && gs >= (dim + group - 1) / group) continue;
                    if (bad++ < 5) std::printf("dim %u, group %u, %d units at a time: %u scales of a row of %u\n", dim, group, p, sc, gs);
                }
    }
    std::printf("%lu of %lu\n", bad, seen);
    return bad ? 1 : 0;
}
