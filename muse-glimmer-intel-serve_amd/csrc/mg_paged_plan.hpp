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

    // What the join of a request reads: how many partial results it has (0: finished in its team), the place of the
    // first and the team of the second. Every team behind the first begins with the request.
    struct alignas(16) PagedCut
    {
        int request, parts, first, second;
    };
    // the request of `units` units from unit p on, which begins in team t
    MG_HD PagedCut paged_cut(const PagedTeams &d, int t, int request, int p, int units)
    {
        const int behind = team_of(d, p + units - 1) - t;
        return PagedCut{request, behind > 0 ? behind + 1 : 0, team_place(d, t, p), t + 1};
    }
    // the place of a request's partial result s < parts
    MG_HD int cut_place(const PagedCut &c, int s) { return s == 0 ? c.first : 2 * (c.second + s - 1); }

    // Notes are kept for each request by the team it begins in, or, of fewer teams than requests, for each team
    // but the last by the team itself: of its last part, which only the team's end can cut.
    MG_HD bool cuts_by_team(int64_t teams, int64_t requests) { return teams < requests; }
    MG_HD int64_t cuts_kept(int64_t teams, int64_t requests) { return cuts_by_team(teams, requests) ? teams - 1 : requests; }
    // whether a team's part from its request's unit `at` on, with `behind` units of the team behind it, leaves a note
    MG_HD bool leaves_cut(bool by_team, int at, int behind) { return by_team ? behind == 0 : at == 0; }
} // namespace mg
