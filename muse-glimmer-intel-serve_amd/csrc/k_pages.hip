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
// One work-group takes the three sums (prefix sums over 1024 requests at a time)
// into LDS; every item of the step (a token, a page taken, a
// page given back) then finds its request by bisection there. A step with few
// tokens ends in that launch. One with more leaves the sums in the workspace and
// a second launch of many work-groups, each with the sums in its own LDS, does
// the items. Measured, us a call (64 requests): 2191 tokens 8.1 in one launch, 11.0
// in two; 4344 10.0 and 11.0; 8803 15.0 and 11.4; 17570 25.2 and 10.7. Latency bounds
// both: a launch, then chains of a bisection and two or three dependent loads.
#include "mg_device.hpp"
#include "mg_internal.hpp"

namespace mg
{
    constexpr int kPagesMax = 4096;   // requests: three sums of each fit 64 KiB of LDS
    constexpr int kPagesAlone = 4096; // tokens up to which one work-group does the whole step

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
        int *sums;    // workspace: the three sums, R + 1 each, then old and new lengths, then head and tail in the ring
        int64_t ldt;
        int R, W, N, T, sh;
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

    // inclusive sums of two values over the work-group's threads on top of their carries, which move on
    template <int NT>
    MG_DEV void group_prefix_u64(uint64_t &u, uint64_t &v, uint64_t &cu, uint64_t &cv, uint64_t (&red)[2][NT / 64])
    {
        const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) {
            const uint64_t x = __shfl_up(u, m, 64), y = __shfl_up(v, m, 64);
            u += lane >= m ? x : 0;
            v += lane >= m ? y : 0;
        }
        if (lane == 63) {
            red[0][wv] = u;
            red[1][wv] = v;
        }
        __syncthreads();
        u += cu;
        v += cv;
        for (int w = 0; w < NT / 64; ++w) {
            const uint64_t x = red[0][w], y = red[1][w];
            u += w < wv ? x : 0;
            v += w < wv ? y : 0;
            cu += x;
            cv += y;
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

    template <int NT, bool ALONE>
    __global__ __launch_bounds__(NT) void k_kv_pages(PagesArgs a)
    {
        extern __shared__ int sums[];
        __shared__ uint64_t red[2][NT / 64];
        int *st = sums, *go = sums + a.R + 1, *bo = sums + 2 * (a.R + 1);
        const int tid = threadIdx.x;
        const int64_t head = a.ends[0], tail = a.ends[1];
        const int64_t left = tail - head;
        const int avail = left < 0 ? 0 : left > a.N ? a.N : int(left);
        const PagesStep s{a, st, go, bo, a.old_lens, a.new_lens, avail, ring_at(head, a.N), ring_at(tail, a.N)};
        if (tid == 0) st[0] = go[0] = bo[0] = 0;
        // the sums: first as if the maps held every token, again without those that do not fit where they do not
        for (bool again = false;; again = true) {
            uint64_t tokens = 0, pages = 0; // pages: taken in the low half, given back in the high half
            for (int b = 0; b < a.R; b += NT) {
                const int i = b + tid;
                int o = 0, n = 0;
                if (i < a.R) s.lens(i, o, n);
                const bool fits = n <= (a.W << a.sh) && (!again || i >= a.R || st[i + 1] <= a.T);
                const int d = pages_of(n, a.sh) - pages_of(o, a.sh);
                uint64_t te = uint64_t(max(n - o, 0)), pe = d >= 0 ? (fits ? uint64_t(d) : 0) : uint64_t(-d) << 32;
                group_prefix_u64<NT>(te, pe, tokens, pages, red);
                if (i < a.R) {
                    st[i + 1] = int(te <= uint64_t(a.T) ? te : uint64_t(a.T) + 1);
                    go[i + 1] = int(uint32_t(pe));
                    bo[i + 1] = int(pe >> 32);
                }
            }
            __syncthreads();
            if (again || tokens <= uint64_t(a.T)) break;
        }
        if constexpr (ALONE) {
            s.items(tid, NT);
        } else {
            const int n3 = 3 * (a.R + 1);
            for (int i = tid; i < n3; i += NT) a.sums[i] = sums[i];
            for (int i = tid; i < a.R; i += NT) {
                a.sums[n3 + i] = a.old_lens[i];
                a.sums[n3 + a.R + i] = a.new_lens[i];
            }
            if (tid == 0) {
                int *e = a.sums + n3 + 2 * a.R;
                e[0] = s.avail;
                e[1] = s.h0;
                e[2] = s.t0;
            }
        }
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

    __global__ __launch_bounds__(256) void k_kv_pages_items(PagesArgs a)
    {
        extern __shared__ int sums[];
        const int n1 = a.R + 1;
        for (int i = threadIdx.x; i < 3 * n1; i += 256) sums[i] = a.sums[i];
        const int *lens = a.sums + 3 * n1, *e = lens + 2 * a.R;
        const PagesStep s{a, sums, sums + n1, sums + 2 * n1, lens, lens + a.R, e[0], e[1], e[2]};
        __syncthreads();
        s.items(blockIdx.x * 256 + threadIdx.x, gridDim.x * 256);
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
        const PagesArgs a{table,    old_lens, new_lens, ring, ends, lens, ends_out, starts, slots, pos, static_cast<int *>(c->work),
                          ldt, int(requests), int(max_pages), int(num_pages), int(tokens), sh};
        const size_t lds = 3 * size_t(requests + 1) * sizeof(int);
        const int64_t room = c->work_bytes / int64_t(sizeof(int));
        if (tokens <= kPagesAlone || 5 * requests + 6 > room) {
            hipLaunchKernelGGL((k_kv_pages<1024, true>), dim3(1), dim3(1024), lds, c->stream, a);
            check_launch("k_kv_pages");
            return;
        }
        hipLaunchKernelGGL((k_kv_pages<1024, false>), dim3(1), dim3(1024), lds, c->stream, a);
        check_launch("k_kv_pages");
        // a token a thread, at most a few rounds of work-groups
        const int64_t most = 8 * int64_t(c->num_cus), groups = (tokens + 255) / 256;
        hipLaunchKernelGGL(k_kv_pages_items, dim3(unsigned(groups < most ? groups : most)), dim3(256), lds, c->stream, a);
        check_launch("k_kv_pages_items");
    }
} // namespace mg
