// How decode attention over a paged cache divides its keys among work-groups:
// plain arithmetic, the same on the host (its host test) and on the device.
//
// A request's attended keys [lo, n) are cut into units of 128 keys from `base`,
// lo rounded down to a step of 32 (a request without keys has one empty unit,
// so that somebody writes its zeros). The units of all requests form one line
// of T; it is cut into `teams` equal runs, whatever requests they cross, and
// each team has a work-group for every group of query heads. A request inside
// one team is finished there; one that a team's edge cuts leaves a partial
// result in each of its teams, at most two a team: that of the team's first
// request (place 2 t) and that of its last (2 t + 1).
#pragma once

#include <stdint.h>

#ifdef __HIP__
#define MG_HD __host__ __device__ __forceinline__
#else
#define MG_HD inline
#endif

namespace mg
{
    constexpr int kPagedStep = 32;  // keys a wave takes at once
    constexpr int kPagedUnit = 128; // a step of each of a work-group's four waves

    struct PagedSpan
    {
        int lo, n, base, units;
    };

    // `cap`: the tokens a table row can hold
    MG_HD PagedSpan paged_span(int len, int cap, int64_t window)
    {
        PagedSpan s;
        s.n = len < 0 ? 0 : len > cap ? cap : len;
        s.lo = window > 0 && s.n > window ? int(s.n - window) : 0;
        s.base = s.lo / kPagedStep * kPagedStep;
        const int u = (s.n - s.base) / kPagedUnit + ((s.n - s.base) % kPagedUnit != 0);
        s.units = u > 0 ? u : 1;
        return s;
    }

    // The line's division among `teams` <= total teams: `per` units each, the first `rem` one more.
    // total < 2^31 (the caller's check), so 32 bits do.
    struct PagedTeams
    {
        int total, teams, per, rem;
    };
    MG_HD PagedTeams paged_teams(int total, int teams)
    {
        PagedTeams d;
        d.total = total;
        d.teams = teams < total ? teams : total; // no team is empty
        d.per = total / d.teams;
        d.rem = total - d.per * d.teams;
        return d;
    }
    // first unit of team t (of t = teams: the total)
    MG_HD int team_first(const PagedTeams &d, int t) { return t * d.per + (t < d.rem ? t : d.rem); }
    // the team that holds unit u
    MG_HD int team_of(const PagedTeams &d, int u)
    {
        const int big = d.rem * (d.per + 1);
        return u < big ? u / (d.per + 1) : d.rem + (u - big) / d.per;
    }
    // where team t leaves its partial result of the request whose first unit is p
    MG_HD int team_place(const PagedTeams &d, int t, int p) { return 2 * t + (team_first(d, t) < p ? 1 : 0); }
} // namespace mg
