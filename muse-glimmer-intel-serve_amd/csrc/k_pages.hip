// Page tables and slot maps of a paged KV cache, from request lengths, for gfx950.
//
// R requests hold pages of 2^sh tokens: row i of the table lists request i's
// pages in order. A step takes every request from o tokens to n. With
//   add_i  = max(0, n - o),             starts = the exclusive sum of add,
//   have_i = ceil(o / ps), want_i = ceil(n / ps),
//   grow_i = max(0, want - have), off  = the exclusive sum of grow,
//   back_i = max(0, have - want), boff = the exclusive sum of back,
// a growing request takes pages free[(head + off_i + k) % N], a shrinking one
// puts its last back_i pages at free[(tail + boff_i + k) % N]: the free pages
// are a queue in a ring of N entries, so what is taken and what is given back
// never meet, and no step of the call waits for another's writes. Token
// starts_i + j of the step is position p = o_i + j and slot
// table[i, p / ps] ps + p % ps; a page taken in this call is read from the
// queue, not from the table.
//
// A request is granted its growth when its tokens fit the maps, its pages fit
// the table's row, and off_i + grow_i pages are there; grow_i counts for the
// requests behind it either way, so the granted ones take a prefix of the
// queue. Every sum is of whole numbers: results do not depend on the order.
//
// A work-group takes the three sums (prefix sums over 1024 requests at a time)
// into LDS; every item of the step (a token, a page taken, a page given back)
// then finds its request by bisection there. Small steps run in one work-group;
// larger ones in a work-group for every 1024 tokens, each with all the sums for itself
// (R lengths from L2: cheaper than sums from memory in a second launch; 1000
// requests, 94 000 tokens 13.3 -> 7.3 us a call, 200 requests, 520 000 tokens 11.2 -> 7.3),
// and the first also writes the new lengths and counters. Where those replace their
// old values, which the others still read, they are left to a second launch of one
// work-group, from 4096 tokens on (10.4 us, what one work-group takes at 4000).
//
// Latency bounds it: traced 4.8 us (median) for a decode step of 48 requests, in place or not, 7.7
// and 8.2 for the two above, of which a stream of calls hides 0.5 to 1: a launch, the sums, then
// chains of a bisection and two or three dependent loads. The work-groups follow the tokens alone:
// pages are taken and given back by as many, so one of them takes a step of few tokens that ends
// long requests, at 0.5 (few requests to bisect) to 1.1 us a thousand pages: 8 requests of 131072
// tokens in pages of 16 38 us, 256 of 4096 61, 256 of 131072 2.3 ms.
#include "mg_device.hpp"
#include "mg_internal.hpp"

namespace mg
{
    constexpr int kPagesMax = 4096;   // requests: three sums of each fit 64 KiB of LDS
    constexpr int kPagesGroup = 1024; // tokens a work-group
    constexpr int kPagesAlone = 4096; // tokens up to which one does the whole of a step in place

    enum : int { kPagesItems = 1, kPagesEnd = 2 }; // what a launch does: the items, the lengths and counters

    struct PagesArgs
    {
        int32_t *table;
        const int32_t *old_lens, *new_lens;
        int32_t *ring;
        const int64_t *ends;
        int32_t *lens;
        int64_t *ends_out;
        int32_t *starts;
        int64_t *slots, *pos;
        int64_t ldt;
        int R, W, N, T, sh;
        int what;
    };

    // the last index in [0, n) whose sum is at most x (sums: n + 1 entries from 0, not
    // falling): the owner of item x where x < sums[n]
    MG_DEV int owner(const int *sums, int n, int x)
    {
        int lo = 0, hi = n; // sums[lo] <= x
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (sums[mid] <= x)
                lo = mid;
            else
                hi = mid;
        }
        return lo;
    }

    MG_DEV uint32_t add_sat(uint32_t a, uint32_t b) { return __builtin_elementwise_add_sat(a, b); }
    // wave_prefix_sum with sums that stop at 2^32 - 1
    MG_DEV uint32_t wave_prefix_sat(uint32_t u)
    {
        uint32_t t = u;
        t = add_sat(t, dpp32<0x111, 0xf>(0u, u));
        t = add_sat(t, dpp32<0x112, 0xf>(0u, u));
        t = add_sat(t, dpp32<0x113, 0xf>(0u, u));
        t = add_sat(t, dpp32<0x114, 0xf, 0xe>(0u, t));
        t = add_sat(t, dpp32<0x118, 0xf, 0xc>(0u, t));
        t = add_sat(t, dpp32<0x142, 0xa>(0u, t));
        t = add_sat(t, dpp32<0x143, 0xc>(0u, t));
        return t;
    }
    // inclusive sums of three values over the work-group's first `waves` waves (the others hold none) on top of
    // their carries, which move on; they stop at 2^32 - 1
    template <int NT>
    MG_DEV void group_prefix(uint32_t (&u)[3], uint32_t (&carry)[3], uint32_t (&red)[3][NT / 64], int waves)
    {
        const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        if (wv < waves) {
#pragma unroll
            for (int k = 0; k < 3; ++k) {
                u[k] = wave_prefix_sat(u[k]);
                if (lane == 63) red[k][wv] = u[k];
            }
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            const int r = int(wave_prefix_sat(lane < waves ? red[k][lane] : 0u));
            const uint32_t before = wv > 0 ? uint32_t(__builtin_amdgcn_readlane(r, wv - 1)) : 0u;
            u[k] = add_sat(add_sat(u[k], before), carry[k]);
            carry[k] = add_sat(carry[k], uint32_t(__builtin_amdgcn_readlane(r, 63)));
        }
        __syncthreads();
    }

    MG_DEV int pages_of(int len, int sh) { return (len >> sh) + ((len & ((1 << sh) - 1)) != 0); }
    // a queue counter's place in the ring
    MG_DEV int ring_at(int64_t c, int N)
    {
        const int r = int(c % N);
        return r < 0 ? r + N : r;
    }

    // One step's state, the sums in LDS. Lengths are clamped to what a row can hold
    // (old) and to 0 (both); a row holds W << sh <= 2^30 tokens (checked on the host).
    struct PagesStep
    {
        const PagesArgs &a;
        const int *st, *go, *bo; // sums of tokens (up to T + 1, which no request's fits), pages taken, pages given back
        const int32_t *olds, *news;
        int avail, h0, t0;

        MG_DEV void lens(int i, int &o, int &n) const
        {
            o = min(max(olds[i], 0), a.W << a.sh);
            n = max(news[i], 0);
        }
        MG_DEV bool granted(int i, int o, int n) const
        {
            return n <= o || (n <= (a.W << a.sh) && st[i + 1] <= a.T && (go[i + 1] == go[i] || go[i + 1] <= avail));
        }
        MG_DEV int queued(int start, int k) const // the ring's place of entry k behind `start`
        {
            const int64_t r = int64_t(start) + k;
            return int(r >= a.N ? r - a.N : r);
        }
        MG_DEV void token(int t) const
        {
            int64_t slot = -1, p = -1;
            if (t < st[a.R]) {
                const int i = owner(st, a.R, t);
                int o, n;
                lens(i, o, n);
                if (granted(i, o, n)) {
                    const int at = o + (t - st[i]), pi = at >> a.sh, have = pages_of(o, a.sh);
                    const int page = pi < have ? a.table[i * a.ldt + pi] : a.ring[queued(h0, go[i] + (pi - have))];
                    p = at;
                    if (page >= 0 && page < a.N) slot = (int64_t(page) << a.sh) + (at & ((1 << a.sh) - 1));
                }
            }
            if (a.slots) a.slots[t] = slot;
            if (a.pos) a.pos[t] = p;
        }
        MG_DEV void take(int g) const
        {
            const int i = owner(go, a.R, g);
            int o, n;
            lens(i, o, n);
            if (granted(i, o, n)) a.table[i * a.ldt + pages_of(o, a.sh) + (g - go[i])] = a.ring[queued(h0, g)];
        }
        MG_DEV void give(int g) const
        {
            const int i = owner(bo, a.R, g);
            int o, n;
            lens(i, o, n);
            a.ring[queued(t0, g)] = a.table[i * a.ldt + pages_of(n, a.sh) + (g - bo[i])];
        }
        // items first, first + step, ... of one line of them all: tokens, pages taken, pages given back
        MG_DEV void items(int first, int step) const
        {
            const int64_t taken = min(go[a.R], avail), given = min(bo[a.R], a.N), all = a.T + taken + given;
            for (int64_t x = first; x < all; x += step) {
                if (x < a.T)
                    token(int(x));
                else if (x < a.T + taken)
                    take(int(x - a.T));
                else
                    give(int(x - a.T - taken));
            }
        }
    };

    template <int NT>
    __global__ __launch_bounds__(NT) void k_kv_pages(PagesArgs a)
    {
        extern __shared__ int sums[];
        __shared__ uint32_t red[3][NT / 64];
        __shared__ int place[2];
        int *st = sums, *go = sums + a.R + 1, *bo = sums + 2 * (a.R + 1);
        const int tid = threadIdx.x;
        const int64_t head = a.ends[0], tail = a.ends[1];
        const int64_t left = tail - head;
        const int avail = left < 0 ? 0 : left > a.N ? a.N : int(left);
        PagesStep s{a, st, go, bo, a.old_lens, a.new_lens, avail, 0, 0};
        if (tid == NT - 1) { // (two long divisions, beside the first waves' sums)
            st[0] = go[0] = bo[0] = 0;
            place[0] = ring_at(head, a.N);
            place[1] = ring_at(tail, a.N);
        }
        // the sums: first as if the maps held every token, again without those that do not fit where they do not
        for (bool again = false;; again = true) {
            uint32_t carry[3] = {0, 0, 0}; // tokens, pages taken, pages given back (fewer than 2^31, as the table's)
            for (int b = 0; b < a.R; b += NT) {
                const int i = b + tid;
                int o = 0, n = 0;
                if (i < a.R) s.lens(i, o, n);
                const bool fits = n <= (a.W << a.sh) && (!again || i >= a.R || st[i + 1] <= a.T);
                const int d = pages_of(n, a.sh) - pages_of(o, a.sh);
                uint32_t u[3] = {uint32_t(max(n - o, 0)), d > 0 && fits ? uint32_t(d) : 0u, uint32_t(max(-d, 0))};
                group_prefix<NT>(u, carry, red, min(NT / 64, (a.R - b + 63) / 64));
                if (i < a.R) {
                    st[i + 1] = int(min(u[0], uint32_t(a.T) + 1));
                    go[i + 1] = int(u[1]);
                    bo[i + 1] = int(u[2]);
                }
            }
            __syncthreads();
            if (again || carry[0] <= uint32_t(a.T)) break;
        }
        s.h0 = place[0];
        s.t0 = place[1];
        if (a.what & kPagesItems) s.items(blockIdx.x * NT + tid, gridDim.x * NT);
        if (!(a.what & kPagesEnd) || blockIdx.x != 0) return;
        __syncthreads(); // the lengths may be updated in place: every thread is done with them
        for (int i = tid; i < a.R; i += NT) {
            int o, n;
            s.lens(i, o, n);
            a.lens[i] = s.granted(i, o, n) ? n : o;
            if (a.starts) a.starts[i + 1] = min(st[i + 1], a.T);
        }
        if (tid == 0) {
            if (a.starts) a.starts[0] = 0;
            // a request that is refused for its pages is followed by refused ones only: the granted pages are
            // the largest sum that the queue covers
            const int used = go[a.R] <= avail ? go[a.R] : go[owner(go, a.R, avail)];
            a.ends_out[0] = head + used;
            a.ends_out[1] = tail + bo[a.R];
        }
    }

    void launch_kv_pages(mg_ctx *c, int32_t *table, int64_t ldt, int64_t requests, int64_t max_pages,
                         const int32_t *old_lens, const int32_t *new_lens, int64_t page_size, int32_t *ring,
                         int64_t num_pages, const int64_t *ends, int32_t *lens, int64_t *ends_out, int32_t *starts,
                         int64_t *slots, int64_t *pos, int64_t tokens)
    {
        const int sh = page_shift(page_size, "kv_pages");
        need(requests >= 0 && requests <= kPagesMax,
             "kv_pages: at most " + std::to_string(kPagesMax) + " requests (got " + std::to_string(requests) + ")");
        need(max_pages > 0 && num_pages > 0 && num_pages < (int64_t(1) << 31), "kv_pages: bad table or pool size");
        need(max_pages <= (int64_t(1) << 30) >> sh, "kv_pages: a table row must stand for at most 2^30 tokens");
        need(requests * max_pages < (int64_t(1) << 31), "kv_pages: a table must have fewer than 2^31 pages");
        need(tokens >= 0 && tokens <= (int64_t(1) << 30), "kv_pages: bad token count");
        need(requests == 0 || (table && old_lens && new_lens && lens), "kv_pages: NULL tensor");
        need(ring && ends && ends_out, "kv_pages: NULL tensor");
        if (ldt == 0) ldt = max_pages;
        need(ldt >= max_pages, "kv_pages: row stride smaller than a row");
        PagesArgs a{table, old_lens, new_lens, ring, ends, lens, ends_out, starts, slots, pos,
                    ldt, int(requests), int(max_pages), int(num_pages), int(tokens), sh, 0};
        const size_t lds = 3 * size_t(requests + 1) * sizeof(int);
        auto go = [&](int what, int64_t groups) {
            a.what = what;
            hipLaunchKernelGGL((k_kv_pages<1024>), dim3(unsigned(groups)), dim3(1024), lds, c->stream, a);
            check_launch("k_kv_pages");
        };
        const int64_t most = 2 * int64_t(c->num_cus), all = (tokens + kPagesGroup - 1) / kPagesGroup;
        const int64_t groups = all < 1 ? 1 : all < most ? all : most;
        const bool in_place = lens == old_lens || lens == new_lens || ends_out == ends;
        if (!in_place || tokens <= kPagesAlone) {
            go(kPagesItems | kPagesEnd, in_place ? 1 : groups);
        } else {
            go(kPagesItems, groups);
            go(kPagesEnd, 1);
        }
    }
} // namespace mg
