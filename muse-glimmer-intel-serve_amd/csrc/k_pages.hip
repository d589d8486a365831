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
#include "mg_device.hpp"
#include "mg_internal.hpp"

namespace mg
{
    constexpr int kPagesMax = 4096; // requests: three sums of each fit 64 KiB of LDS

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

    MG_DEV uint64_t wave_prefix_u64(uint64_t v, int lane)
    {
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) {
            const uint64_t u = __shfl_up(v, m, 64);
            v += lane >= m ? u : 0;
        }
        return v;
    }

    // inclusive sum over the work-group's threads on top of `carry`, which moves on
    template <int NT>
    MG_DEV uint64_t group_prefix_u64(uint64_t v, uint64_t &carry, uint64_t *red)
    {
        const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
        v = wave_prefix_u64(v, lane);
        if (lane == 63) red[wv] = v;
        __syncthreads();
        uint64_t before = carry, all = carry;
        for (int w = 0; w < NT / 64; ++w) {
            before += w < wv ? red[w] : 0;
            all += red[w];
        }
        __syncthreads();
        carry = all;
        return v + before;
    }

    MG_DEV void lens_of(const PagesArgs &a, int i, int &o, int &n)
    {
        // capacity W << sh is at most 2^30 (checked on the host)
        o = min(max(a.old_lens[i], 0), a.W << a.sh);
        n = max(a.new_lens[i], 0);
    }
    MG_DEV int pages_of(int len, int sh) { return (len >> sh) + ((len & ((1 << sh) - 1)) != 0); }
    // a queue counter's place in the ring
    MG_DEV int ring_at(int64_t c, int N)
    {
        const int r = int(c % N);
        return r < 0 ? r + N : r;
    }

    template <int NT>
    __global__ __launch_bounds__(NT) void k_kv_pages(PagesArgs a)
    {
        extern __shared__ int sums[];
        __shared__ uint64_t red[NT / 64];
        int *st = sums, *go = sums + a.R + 1, *bo = sums + 2 * (a.R + 1);
        const int tid = threadIdx.x;
        const int64_t head = a.ends[0], tail = a.ends[1];
        const int64_t left = tail - head;
        const int avail = left < 0 ? 0 : left > a.N ? a.N : int(left);
        const int h0 = ring_at(head, a.N), t0 = ring_at(tail, a.N);
        // the sums; token sums stop at T + 1, which no request's fits
        uint64_t tokens = 0, pages = 0; // taken in the low half, given back in the high half
        if (tid == 0) st[0] = go[0] = bo[0] = 0;
        for (int b = 0; b < a.R; b += NT) {
            const int i = b + tid;
            int o = 0, n = 0;
            if (i < a.R) lens_of(a, i, o, n);
            const uint64_t te = group_prefix_u64<NT>(uint64_t(max(n - o, 0)), tokens, red);
            const bool fits = n <= o || (n <= (a.W << a.sh) && te <= uint64_t(a.T));
            const int d = pages_of(n, a.sh) - pages_of(o, a.sh);
            const uint64_t pe =
                group_prefix_u64<NT>(d >= 0 ? (fits ? uint64_t(d) : 0) : uint64_t(-d) << 32, pages, red);
            if (i < a.R) {
                st[i + 1] = int(te <= uint64_t(a.T) ? te : uint64_t(a.T) + 1);
                go[i + 1] = int(uint32_t(pe));
                bo[i + 1] = int(pe >> 32);
            }
        }
        __syncthreads();
        auto granted = [&](int i, int o, int n) {
            return n <= o || (n <= (a.W << a.sh) && st[i + 1] <= a.T && (go[i + 1] == go[i] || go[i + 1] <= avail));
        };
        const int ps1 = (1 << a.sh) - 1;
        const int total = st[a.R];
        for (int t = tid; t < a.T; t += NT) {
            int64_t slot = -1, p = -1;
            if (t < total) {
                const int i = owner(st, a.R, t);
                int o, n;
                lens_of(a, i, o, n);
                if (granted(i, o, n)) {
                    const int at = o + (t - st[i]), pi = at >> a.sh, have = pages_of(o, a.sh);
                    int page;
                    if (pi < have) {
                        page = a.table[i * a.ldt + pi];
                    } else {
                        const int64_t r = int64_t(h0) + go[i] + (pi - have);
                        page = a.ring[r >= a.N ? r - a.N : r];
                    }
                    p = at;
                    if (page >= 0 && page < a.N) slot = (int64_t(page) << a.sh) + (at & ps1);
                }
            }
            if (a.slots) a.slots[t] = slot;
            if (a.pos) a.pos[t] = p;
        }
        const int taken = min(go[a.R], avail);
        for (int g = tid; g < taken; g += NT) {
            const int i = owner(go, a.R, g);
            int o, n;
            lens_of(a, i, o, n);
            const int64_t r = int64_t(h0) + g;
            if (granted(i, o, n)) a.table[i * a.ldt + pages_of(o, a.sh) + (g - go[i])] = a.ring[r >= a.N ? r - a.N : r];
        }
        const int given = min(bo[a.R], a.N);
        for (int g = tid; g < given; g += NT) {
            const int i = owner(bo, a.R, g);
            int o, n;
            lens_of(a, i, o, n);
            const int64_t r = int64_t(t0) + g;
            a.ring[r >= a.N ? r - a.N : r] = a.table[i * a.ldt + pages_of(n, a.sh) + (g - bo[i])];
        }
        __syncthreads(); // the lengths may be updated in place: every thread is done with them
        for (int b = 0; b < a.R; b += NT) {
            const int i = b + tid;
            if (i >= a.R) break;
            int o, n;
            lens_of(a, i, o, n);
            const bool ok = granted(i, o, n);
            a.lens[i] = ok ? n : o;
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
        need(tokens >= 0 && tokens < (int64_t(1) << 31) - 1, "kv_pages: bad token count");
        need(requests == 0 || (table && old_lens && new_lens && lens), "kv_pages: NULL tensor");
        need(ring && ends && ends_out, "kv_pages: NULL tensor");
        if (ldt == 0) ldt = max_pages;
        need(ldt >= max_pages, "kv_pages: row stride smaller than a row");
        const PagesArgs a{table, old_lens, new_lens, ring, ends,          lens,           ends_out,       starts,    slots,
                          pos,   ldt,      int(requests), int(max_pages), int(num_pages), int(tokens), sh};
        const size_t lds = 3 * size_t(requests + 1) * sizeof(int);
        hipLaunchKernelGGL(k_kv_pages<1024>, dim3(1), dim3(1024), lds, c->stream, a);
        check_launch("k_kv_pages");
    }
} // namespace mg
