// Walks the plans of muon_plan.h on the CPU: every step of every tile is taken once, by units that agree on who
// puts a cut tile together and where its parts lie. Prints "plans tiles cut"; 1 with a message for the first fault.
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <map>
#include <random>
#include <set>
#include <vector>

#include "muon_plan.h"

using namespace arcqml;

#define CHECK(what)                                                                     \
    if (!(what)) {                                                                      \
        printf("plan %d: %s\n", plan, #what);                                           \
        return 1;                                                                       \
    }

int main() {
    std::mt19937_64 g(1);
    const auto pick = [&](uint64_t low, uint64_t high) { return low + g() % (high - low + 1); };
    uint64_t tiles = 0, cuts = 0;
    for (int plan = 0; plan < 6000; ++plan) {
        const uint32_t units = pick(0, 1) ? 74 : 148;
        TilePlan p{};
        // classes by depth, deepest first, as make_plan puts them down
        std::set<uint32_t, std::greater<uint32_t>> depths;
        const uint32_t most = plan % 10 == 0 ? kMatrices : 5;
        const uint32_t classes = pick(1, most);
        while (depths.size() < classes) depths.insert(uint32_t(pick(0, 3) ? pick(1, 140) : pick(1, 3000)));
        std::vector<uint32_t> has;
        uint32_t all = 0;
        for (uint32_t d : depths) {
            const uint32_t c = p.classes++;
            static const uint32_t usual[] = {1, 2, 3, 10, 36, 73, 74, 75, 136, 148, 300};
            has.push_back(pick(0, 1) ? usual[pick(0, 10)] : uint32_t(pick(1, 400)));
            p.tile[c] = all;
            p.depth[c] = d;
            p.rounds[c] = has[c] / units;
            p.left[c + 1] = p.left[c] + has[c] % units * weight(d);
            all += has[c];
        }
        const uint32_t longest = share_out(p, units, pick(0, 1) != 0);
        CHECK(p.runs >= 1 && p.runs <= units);
        std::vector<std::vector<uint8_t>> taken(all);
        std::vector<uint32_t> depth(all);
        for (uint32_t c = 0, t = 0; c < p.classes; ++c)
            for (uint32_t i = 0; i < has[c]; ++i, ++t) taken[t].assign(depth[t] = p.depth[c], 0);
        struct Share {
            uint32_t unit, first, count, slot, begin;
        };
        std::map<uint32_t, std::vector<Share>> shares; // of tiles that are cut
        std::set<std::pair<uint32_t, uint32_t>> slots;
        for (uint32_t unit = 0; unit < units; ++unit) {
            const uint32_t from = cut(p, unit);
            CHECK(from <= cut(p, unit + 1));
            Walk walk(p, unit, units);
            Part part;
            uint32_t steps = 0;
            while (walk.next(part)) {
                CHECK(part.tile < all && part.depth == depth[part.tile]);
                CHECK(part.begin < part.end && part.end <= part.depth);
                CHECK(++steps <= all);
                for (uint32_t d = part.begin; d < part.end; ++d) CHECK(!taken[part.tile][d]++);
                if (part.whole()) continue;
                CHECK(part.end - part.begin >= 8); // worth its way through memory
                Share s{unit, 0, 0, slot_of(part, from), part.begin};
                sharers(p, part, s.first, s.count);
                CHECK(slots.insert({unit, s.slot}).second); // a unit's parts do not overwrite one another
                shares[part.tile].push_back(s);
            }
        }
        for (uint32_t t = 0; t < all; ++t)
            for (uint32_t d = 0; d < depth[t]; ++d) CHECK(taken[t][d]);
        std::set<uint32_t> counters;
        for (const auto &[tile, list] : shares) {
            (void)tile;
            CHECK(list.size() >= 2 && counters.insert(list[0].first).second); // a counter for each cut tile
            for (uint32_t i = 0; i < list.size(); ++i) {
                const Share &s = list[i]; // units in order are parts in the order of depth
                CHECK(s.first == list[0].first && s.count == list.size());
                CHECK(s.unit == s.first + i && s.slot == (i ? 0u : 1u));
                CHECK(i == 0 ? s.begin == 0 : s.begin > list[i - 1].begin);
            }
        }
        uint32_t run = 0;
        for (uint32_t unit = 0; unit < p.runs; ++unit) run = std::max(run, cut(p, unit + 1) - cut(p, unit));
        CHECK(longest >= run && longest <= run + 40);
        tiles += all;
        cuts += shares.size();
    }
    printf("6000 %llu %llu\n", (unsigned long long)tiles, (unsigned long long)cuts);
    return 0;
}
