// muon_plan.h — who does which tile of a phase of the Newton-Schulz products (muon.cu): the kernel's walk, and the
// host's choice of the shares. Without CUDA it compiles as host code.
#pragma once

#include <stdint.h>

#include <algorithm>

#ifdef __CUDACC__
#define ARCQML_PLAN __host__ __device__ __forceinline__
#else
#define ARCQML_PLAN inline
#endif

namespace arcqml {

constexpr uint32_t kMatrices = 64; // of a launch

// Who does which tile. Units (blocks, or pairs of them) take the tiles of each depth, deepest first, in whole
// rounds: neighbouring tiles at a time, which share their operands in L2. The steps that are left of all depths
// are cut into equal runs, one for each unit. Cuts move to the next tile's edge, or (where it is worth what
// it costs, see share_out()) go through a tile, which the unit that finishes last then sums up in the order of
// its depth.
struct TilePlan {
    uint32_t classes; // of depth
    uint32_t tile[kMatrices + 1], rounds[kMatrices], depth[kMatrices];
    uint32_t left[kMatrices + 1]; // steps left before the class; a tile counts for kLeast of them at least
    uint32_t runs;                // units that share the steps left
    uint32_t snap;                // a cut this near to a tile's edge moves there
};

constexpr uint32_t kLeast = 16; // taking a tile's sums out takes as long
ARCQML_PLAN uint32_t weight(uint32_t depth) { return depth > kLeast ? depth : kLeast; }

// The class that step `at` of those left belongs to.
ARCQML_PLAN uint32_t class_of(const TilePlan &p, uint32_t at) {
    uint32_t c = 0;
    while (p.left[c + 1] <= at) ++c;
    return c;
}
// Where the unit's run of the steps left begins.
ARCQML_PLAN uint32_t cut(const TilePlan &p, uint32_t unit) {
    const uint32_t all = p.left[p.classes];
    if (unit >= p.runs) return all;
    const uint32_t at = uint32_t(uint64_t(unit) * all / p.runs);
    if (at == 0) return 0;
    const uint32_t c = class_of(p, at), w = weight(p.depth[c]), past = (at - p.left[c]) % w, behind = w - past;
    return past < p.snap && past < behind          ? at - past
           : past < p.snap || past + p.snap > p.depth[c] || past + p.snap < past ? at + behind
                                                                                 : at;
}
struct Part {
    uint32_t tile, begin, end, depth; // steps of the tile's depth
    uint32_t start;                   // the tile's first step among those left
    ARCQML_PLAN bool whole() const { return begin == 0 && end == depth; }
};
struct Walk {
    const TilePlan &p;
    uint32_t unit, units, c = 0, round = 0, at, end;
    ARCQML_PLAN Walk(const TilePlan &plan, uint32_t u, uint32_t n) : p(plan), unit(u), units(n) {
        at = cut(p, unit);
        end = cut(p, unit + 1);
    }
    ARCQML_PLAN bool next(Part &r) {
        for (; c < p.classes; ++c, round = 0)
            if (round < p.rounds[c]) {
                r.tile = p.tile[c] + round++ * units + unit;
                r.begin = 0;
                r.end = r.depth = p.depth[c];
                return true;
            }
        if (at >= end) return false;
        const uint32_t k = class_of(p, at), w = weight(p.depth[k]), n = (at - p.left[k]) / w;
        r.depth = p.depth[k];
        r.start = p.left[k] + n * w;
        r.tile = p.tile[k] + p.rounds[k] * units + n;
        r.begin = at - r.start;
        r.end = end - r.start < r.depth ? end - r.start : r.depth;
        at = r.start + (r.end == r.depth ? w : r.end);
        return true;
    }
};

// Of a tile that is cut: the unit with its first step, and how many units have parts of it.
ARCQML_PLAN void sharers(const TilePlan &p, const Part &r, uint32_t &first, uint32_t &count) {
    first = uint32_t(uint64_t(r.start) * p.runs / p.left[p.classes]);
    while (cut(p, first) > r.start) --first;
    while (cut(p, first + 1) <= r.start) ++first;
    count = 1;
    while (cut(p, first + count) < r.start + r.depth) ++count;
}
// Which of a unit's two parts it is, the unit's run beginning at `from`: 0 of a tile that began earlier.
ARCQML_PLAN uint32_t slot_of(const Part &r, uint32_t from) { return r.start < from ? 0 : 1; }

// Cuts the steps left into shares, and gives the longest one's steps.
inline uint32_t share_out(TilePlan &p, uint32_t units, bool split) {
    // whole tiles, or runs of equal length, of 16 steps and a sixth of a tile at least: writing parts and putting
    // them together takes about 18 us, 40 steps of 11-bit operands and 20 of 22-bit ones
    const uint32_t all = p.left[p.classes];
    uint32_t longest[2];
    const auto cut_up = [&](bool parts) {
        p.snap = parts ? 8 : 0xffffffffu;
        p.runs = parts ? std::max(1u, std::min(units, all / std::max(16u, (p.depth[0] + 5) / 6))) : units;
    };
    for (int parts = 0; parts < 2; ++parts) {
        cut_up(parts != 0);
        uint32_t run = 0;
        for (uint32_t u = 0; u < p.runs; ++u) run = std::max(run, cut(p, u + 1) - cut(p, u));
        longest[parts] = run + (parts ? (split ? 20 : 40) : 0);
    }
    const bool parts = longest[1] < longest[0];
    cut_up(parts);
    return longest[parts];
}

}  // namespace arcqml
