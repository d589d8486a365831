// Host check of mg_paged_plan.hpp for each number of keys that a wave takes at once,
// 32 and 64: a request's keys lie in its units, no more of them than paged_most_units
// says; each team walks its run as the kernel does, every unit once, and the join,
// walked through the notes alone, takes every partial result once, in order. Prints
// "ok" or the first mistake.
#include "../../muse-glimmer-intel-serve_amd/csrc/mg_paged_plan.hpp"

#include <cstdio>
#include <random>
#include <utility>
#include <vector>

using namespace mg;

#define CHECK(c)                                                                     \
    do {                                                                             \
        if (!(c)) {                                                                  \
            std::printf("%s (step %d, batch %d, line %d)\n", #c, STEP, batch, __LINE__); \
            return false;                                                            \
        }                                                                            \
    } while (0)

template <int STEP>
bool sweep()
{
    constexpr int U = 4 * STEP;
    std::mt19937_64 rng(STEP);
    auto upto = [&](int64_t n) { return int64_t(rng() % uint64_t(n + 1)); };
    int64_t joined = 0, fullest = 0;
    for (int batch = 0; batch < 5000; ++batch) {
        const int R = 1 + int(upto(batch % 3 ? 12 : 300));
        const int cap = 1 << (batch % 5 == 0 ? (batch % 3 ? 30 : 22) : 5 + upto(12));
        const int64_t window = batch % 2 ? 0 : batch % 8 == 0 ? 1 + upto(4 * int64_t(cap)) : 1 + upto(2000);
        const int64_t most = paged_most_units(cap, window, STEP);
        const int asked = 1 + int(upto(batch % 7 ? 60 : 600));
        std::vector<int> units(R);
        std::vector<int64_t> first(R + 1, 0);
        for (int b = 0; b < R; ++b) {
            const int64_t pick = upto(6);
            const int len = pick == 0 ? 0 : pick == 1 ? -5 : pick == 2 ? cap : pick == 3 ? int(upto(300))
                            : pick == 4 ? int(window + U * upto(3) + upto(2) - 1) : int(upto(cap));
            const PagedSpan s = paged_span<STEP>(len, cap, window);
            CHECK(s.n == (len < 0 ? 0 : len > cap ? cap : len));
            CHECK(s.lo == (window > 0 && s.n > window ? s.n - window : 0));
            CHECK(s.base % STEP == 0 && s.base <= s.lo && s.lo - s.base < STEP);
            CHECK(s.units >= 1 && s.units <= most);
            CHECK(int64_t(s.base) + int64_t(s.units) * U >= s.n);
            CHECK(s.units == 1 || int64_t(s.base) + int64_t(s.units - 1) * U < s.n);
            fullest += s.units == most;
            units[b] = s.units;
            first[b + 1] = first[b] + s.units;
        }
        CHECK(first[R] < (int64_t(1) << 31));
        const PagedTeams d = paged_teams(int(first[R]), asked);
        const bool by_team = cuts_by_team(asked, R);
        std::vector<PagedCut> cut(by_team ? asked : R, PagedCut{-1, -1, -1, -1});
        std::vector<std::pair<int, int64_t>> at_place(size_t(2 * asked), {-1, -1}); // (request, its unit) of a partial result
        std::vector<int64_t> done(R, 0);
        for (int t = 0; t < asked; ++t) {
            if (t >= d.teams) { // without a run
                if (by_team) cut[t] = PagedCut{};
                continue;
            }
            const int64_t u0 = team_first(d, t), u1 = team_first(d, t + 1);
            CHECK(u0 < u1);
            int b = 0;
            while (first[b + 1] <= u0) ++b;
            for (int64_t u = u0; u < u1; ++b) {
                const int64_t at = u - first[b], end = first[b + 1] < u1 ? units[b] : u1 - first[b], behind = u1 - first[b] - end;
                CHECK(done[b] == at);
                done[b] = end;
                if (leaves_cut(by_team, int(at), int(behind))) {
                    PagedCut &c = cut[by_team ? t : b];
                    CHECK(c.parts == -1); // one writer
                    c = at == 0 ? paged_cut(d, t, b, int(first[b]), units[b]) : PagedCut{};
                }
                if (at != 0 || end != units[b]) {
                    const int place = team_place(d, t, int(first[b]));
                    CHECK(place >= 0 && place < 2 * asked && at_place[place].first == -1);
                    at_place[place] = {b, at};
                }
                u = first[b] + end;
            }
        }
        for (int b = 0; b < R; ++b) CHECK(done[b] == units[b]);
        const int64_t kept = cuts_kept(asked, R);
        std::vector<int> taken(2 * size_t(asked), 0);
        for (int64_t i = 0; i < kept; ++i) {
            const PagedCut c = cut[size_t(i)];
            CHECK(c.parts == 0 || c.parts > 1);
            int64_t unit = -1;
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
    if (joined < 10000 || fullest < 1000) {
        std::printf("the batches cut or fill too little: %ld, %ld\n", long(joined), long(fullest));
        return false;
    }
    return true;
}

int main()
{
    if (!sweep<32>() || !sweep<64>()) return 1;
    std::printf("ok\n");
    return 0;
}
