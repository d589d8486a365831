// Host check of mg_paged_plan.hpp: for many batches of request lengths and team
// counts, every attended key is covered once, by the team that team_of names,
// each team's partial results go to places of its own, and the join finds
// exactly the teams that leave one. Prints "ok" or the first mistake.
#include "../../muse-glimmer-intel-serve_amd/csrc/mg_paged_plan.hpp"

#include <cstdio>
#include <map>
#include <random>
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
    std::mt19937_64 rng(7);
    auto upto = [&](int64_t n) { return int64_t(rng() % uint64_t(n + 1)); };
    for (int batch = 0; batch < 4000; ++batch) {
        const int R = 1 + int(upto(batch % 3 ? 12 : 300));
        const int cap = 1 << (batch % 5 == 0 ? (batch % 3 ? 30 : 24) : 5 + upto(12));
        const int64_t window = batch % 2 ? 0 : 1 + upto(2000);
        const int teams_asked = 1 + int(upto(batch % 7 ? 80 : 600));
        std::vector<PagedSpan> sp(R);
        std::vector<int64_t> first(R + 1, 0);
        for (int b = 0; b < R; ++b) {
            const int64_t pick = upto(5);
            const int len = pick == 0 ? 0 : pick == 1 ? -5 : pick == 2 ? cap : pick == 3 ? int(upto(300)) : int(upto(cap));
            const PagedSpan s = sp[b] = paged_span(len, cap, window);
            CHECK(s.n == (len < 0 ? 0 : len > cap ? cap : len));
            CHECK(s.lo == (window > 0 && s.n > window ? s.n - window : 0));
            CHECK(s.base % kPagedStep == 0 && s.base <= s.lo && s.lo - s.base < kPagedStep);
            CHECK(s.units >= 1 && int64_t(s.base) + int64_t(s.units) * kPagedUnit >= s.n);
            CHECK(s.units == 1 || int64_t(s.base) + int64_t(s.units - 1) * kPagedUnit < s.n);
            first[b + 1] = first[b] + s.units;
        }
        CHECK(first[R] < (int64_t(1) << 31));
        const PagedTeams d = paged_teams(int(first[R]), teams_asked);
        const int64_t total = first[R], teams = d.teams;
        CHECK(d.total == total && teams == (teams_asked < total ? teams_asked : total));
        std::vector<int64_t> done(R, 0);              // units of each request walked so far, in order
        std::vector<std::vector<int64_t>> left(R);    // the teams that leave a partial result, in order
        std::map<int64_t, int> places;
        CHECK(team_first(d, 0) == 0 && team_first(d, int(teams)) == total);
        for (int64_t t = 0; t < teams; ++t) {
            const int64_t u0 = team_first(d, int(t)), u1 = team_first(d, int(t) + 1);
            CHECK(u0 < u1);
            CHECK(team_of(d, int(u0)) == t && team_of(d, int(u1) - 1) == t);
            int b = 0;
            while (first[b + 1] <= u0) ++b;
            const int b0 = b;
            for (int64_t u = u0; u < u1; ++b) {
                const int64_t at = u - first[b], end = first[b + 1] < u1 ? sp[b].units : u1 - first[b];
                CHECK(done[b] == at);
                done[b] = end;
                if (!(at == 0 && end == sp[b].units)) {
                    const int64_t place = 2 * t + (b == b0 ? 0 : 1);
                    CHECK(places.emplace(place, b).second);
                    CHECK(place == team_place(d, int(t), int(first[b])));
                    left[b].push_back(t);
                }
                u = first[b] + end;
            }
        }
        for (int b = 0; b < R; ++b) {
            CHECK(done[b] == sp[b].units);
            const int64_t t0 = team_of(d, int(first[b])), t1 = team_of(d, int(first[b + 1]) - 1);
            if (t0 == t1) {
                CHECK(left[b].empty());
            } else {
                CHECK(int64_t(left[b].size()) == t1 - t0 + 1);
                for (int64_t t = t0; t <= t1; ++t) CHECK(left[b][size_t(t - t0)] == t);
            }
        }
    }
    std::printf("ok\n");
    return 0;
}
