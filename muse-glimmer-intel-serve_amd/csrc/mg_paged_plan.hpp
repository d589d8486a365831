// How decode attention over a paged cache divides its keys among work-groups:
// plain arithmetic, the same on the host (its checker) and on the device.
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

    // first unit of team t of `teams` (teams <= total: no team is empty)
    MG_HD int64_t team_first(int64_t t, int64_t total, int64_t teams) { return t * total / teams; }
    // the team that holds unit u
    MG_HD int64_t team_of(int64_t u, int64_t total, int64_t teams) { return ((u + 1) * teams - 1) / total; }
    // where team t leaves its partial result of the request whose first unit is p
    MG_HD int64_t team_place(int64_t t, int64_t p, int64_t total, int64_t teams)
    {
        return 2 * t + (team_first(t, total, teams) < p ? 1 : 0);
    }
} // namespace mg
