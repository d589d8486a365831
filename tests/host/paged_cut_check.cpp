// Host check of how paged decode attention's partial results find their join
// (mg_paged_plan.hpp): each team of many batches walks its run as the kernel does,
// leaving notes and partial results; the join, walked through the notes alone, takes
// every partial result once, each request's in order. Prints "ok" or the first mistake.
#include "../../muse-glimmer-intel-serve_amd/csrc/mg_paged_plan.hpp"

#include <cstdio>
#include <random>
#include <utility>
#include <vector>

using namespace mg;

#define CHECK(c)                                                                     \
    do {                                                                             \
        if (!(c)) {                                                                  \
            std::printf("%s (batch %d, line %d)\n", #c, batch, __LINE__);            \
            return 1;                                                                \
        }                                                                            \
    } while (0)

int main()
{
    std::mt19937_64 rng(11);
    auto upto = [&](int64_t n) { return int64_t(rng() % uint64_t(n + 1)); };
    int64_t joined = 0, notes_by_team = 0;
    for (int batch = 0; batch < 6000; ++batch) {
        const int R = 1 + int(upto(batch % 3 ? 12 : 300));
        const int asked = 1 + int(upto(batch % 5 ? 40 : 700)); // the launch's teams; fewer work where units are fewer
        const int cap = 1 << (7 + upto(10));
        std::vector<int> units(R), first(R + 1, 0);
        for (int b = 0; b < R; ++b) {
            units[b] = paged_span(int(upto(3) ? upto(cap) : upto(200)), cap, batch % 2 ? 0 : 1 + upto(500)).units;
            first[b + 1] = first[b] + units[b];
        }
        const PagedTeams d = paged_teams(first[R], asked);
        const bool by_team = cuts_by_team(asked, R);
        notes_by_team += by_team;
        const PagedCut unwritten{-1, -1, -1, -1};
        std::vector<PagedCut> cut(by_team ? asked : R, unwritten);
        std::vector<std::pair<int, int>> at_place(size_t(2 * asked), {-1, -1}); // (request, its unit) of a partial result
        for (int t = 0; t < asked; ++t) {
            if (t >= d.teams) { // without a run
                if (by_team) cut[t] = PagedCut{};
                continue;
            }
            const int u0 = team_first(d, t), u1 = team_first(d, t + 1);
            int b = 0;
            while (first[b + 1] <= u0) ++b;
            for (int u = u0; u < u1; ++b) {
                const int at = u - first[b], end = first[b + 1] < u1 ? units[b] : u1 - first[b], behind = u1 - first[b] - end;
                if (leaves_cut(by_team, at, behind)) {
                    PagedCut &c = cut[by_team ? t : b];
                    CHECK(c.parts == -1); // one writer
                    c = at == 0 ? paged_cut(d, t, b, first[b], units[b]) : PagedCut{};
                }
                if (at != 0 || end != units[b]) {
                    const int place = team_place(d, t, first[b]);
                    CHECK(place >= 0 && place < 2 * asked && at_place[place].first == -1);
                    at_place[place] = {b, at};
                }
                u = first[b] + end;
            }
        }
        const int64_t kept = cuts_kept(asked, R);
        CHECK(kept <= int64_t(cut.size()));
        for (int64_t i = kept; i < int64_t(cut.size()); ++i) CHECK(cut[i].parts == 0); // the last team's
        std::vector<int> taken(2 * size_t(asked), 0), joins(R, 0);
        for (int64_t i = 0; i < kept; ++i) {
            const PagedCut c = cut[i];
            CHECK(c.parts == 0 || c.parts > 1); // written
            if (c.parts == 0) continue;
            CHECK(c.request >= 0 && c.request < R && ++joins[c.request] == 1);
            int unit = -1;
            for (int s = 0; s < c.parts; ++s) {
                const int place = cut_place(c, s);
                CHECK(place >= 0 && place < 2 * asked && ++taken[place] == 1);
                CHECK(at_place[place].first == c.request && at_place[place].second > unit);
                CHECK(s > 0 || at_place[place].second == 0);
                unit = at_place[place].second;
                ++joined;
            }
        }
        for (int p = 0; p < 2 * asked; ++p) CHECK((at_place[p].first >= 0) == (taken[p] == 1));
    }
    if (joined < 10000 || notes_by_team < 1000) {
        std::printf("the batches cut too little\n");
        return 1;
    }
    std::printf("ok\n");
    return 0;
}
