// What the kernels of decode attention over a paged cache share: their
// arguments, a work-group's way to its run of the line of units, the weighing of
// partial results, and the host's side of a call.
#pragma once

#include "mg_device.hpp"
#include "mg_internal.hpp"
#include "mg_paged_plan.hpp"

namespace mg
{
    struct PagedArgs
    {
        const void *q, *kc, *vc;
        const uint16_t *kd, *vd;
        const int32_t *table, *lens;
        void *out;
        float *part;     // [2 teams, vh, hw, D] outputs, then [2 teams, vh, hw] maxima and sums
        PagedCut *cut;   // [requests] or, by_team, [teams]: what the second kernel joins
        int by_team;
        int64_t ldq, ldt, ldo, window;
        int R, nkv, W, sh, num_pages;
        int hpg, hw, vh; // query heads a kv head, a work-group; work-groups a team
        int teams;
        float scale2;    // scaling * log2(e)
    };

    // the factor of a part whose maximum is m beside the maximum `top` >= m of all (both may be -inf)
    MG_DEV float weight_of(float m, float top) { return m == top ? 1.0f : __builtin_amdgcn_exp2f(m - top); }
    // what an output is multiplied by: 1 / sum; without a score above -inf 0 where there is no key, else NaN
    MG_DEV float inverse(float sum, float top)
    {
        return top > -__builtin_huge_valf() ? 1.0f / sum : sum == 0.0f ? 0.0f : __builtin_nanf("");
    }

    // the work-group's run [u0, u1) of its team, the request it starts in and that request's first unit p
    struct Run
    {
        PagedTeams d;
        int u0, u1, p, b;
    };
    template <int STEP = kPagedStep>
    MG_DEV Run find_run(const PagedArgs &a, int team)
    {
        const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
        if (a.R <= 64) {
            // each wave by itself, a request a lane
            const int own = lane < a.R ? paged_span<STEP>(a.lens[lane], a.W << a.sh, a.window).units : 0;
            const int pre = wave_prefix_sum(own);
            Run r;
            r.d = paged_teams(__builtin_amdgcn_readlane(pre, 63), a.teams);
            r.u0 = r.u1 = r.p = r.b = 0;
            if (team >= r.d.teams) return r;
            r.u0 = team_first(r.d, team);
            r.u1 = team_first(r.d, team + 1);
            r.b = wave_count(pre <= r.u0); // the requests that end before it
            r.p = r.b > 0 ? __builtin_amdgcn_readlane(pre, r.b - 1) : 0;
            return r;
        }
        __shared__ int red[4], found[2];
        const int per = (a.R + 255) / 256, b0 = tid * per, b1 = min(b0 + per, a.R);
        const int cap = a.W << a.sh;
        int mine = 0;
        for (int b = b0; b < b1; ++b) mine += paged_span<STEP>(a.lens[b], cap, a.window).units;
        int pre = wave_prefix_sum(mine);
        if (lane == 63) red[wv] = pre;
        __syncthreads();
        for (int w = 0; w < wv; ++w) pre += red[w];
        Run r;
        // (uniform values read from LDS go to scalar registers)
        r.d = paged_teams(__builtin_amdgcn_readfirstlane(red[0] + red[1] + red[2] + red[3]), a.teams);
        int p = pre - mine; // the thread's first unit
        r.u0 = r.u1 = 0;
        if (team >= r.d.teams) return r;
        r.u0 = team_first(r.d, team);
        r.u1 = team_first(r.d, team + 1);
        if (r.u0 >= p && r.u0 < pre) {
            int b = b0;
            for (;; ++b) {
                const int u = paged_span<STEP>(a.lens[b], cap, a.window).units;
                if (r.u0 < p + u) break;
                p += u;
            }
            found[0] = p;
            found[1] = b;
        }
        __syncthreads();
        r.p = __builtin_amdgcn_readfirstlane(found[0]);
        r.b = __builtin_amdgcn_readfirstlane(found[1]);
        return r;
    }

    // The host's side of a call. Checks what every format asks for, fills the arguments but for the cache's own
    // and the work's division: the query heads a work-group takes and the work-groups a team.
    PagedArgs paged_args(const void *q, int64_t ldq, const void *kc, const void *vc, const void *kd, const void *vd,
                         const int32_t *table, int64_t ldt, int64_t max_pages, const int32_t *lens, int64_t seqs, int64_t nq,
                         int64_t nkv, int64_t D, int64_t page_size, int64_t num_pages, int64_t window, double scaling,
                         void *out, int64_t ldo, int dt, int dt_out);
    // Divides the line of units of STEP keys a wave among teams for `per_cu` work-groups a CU, and the workspace
    // among their partial results.
    void paged_divide(mg_ctx *c, PagedArgs &a, int64_t D, int per_cu, int step);
    // Joins the partial results, where any request can be cut (a.teams > 1).
    void paged_join(mg_ctx *c, const PagedArgs &a, int64_t D, int dt_out);
} // namespace mg
