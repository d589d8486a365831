// Decode attention over a paged KV cache for gfx950: one new token for each of
// many requests of different lengths.
//
// For request b of n = lens[b] keys (the new token's among them) and query head
// h (KV head g = h / groups), over keys j in [lo, n), lo = window > 0 ?
// max(0, n - window) : 0, key j in slot table[b, j / ps] ps + j % ps of the pool
// [slots, kv_heads, head_dim]:
//   s_j = (q_bh . k_j) * scaling,   out_bh = sum_j softmax(s)_j v_j.
// A request without keys gives zeros. A key whose page is outside the pool is
// left out, as a masked one. Q8_0 pages hold k_j and v_j as q * d, exactly.
#include "mg_device.hpp"
#include "mg_internal.hpp"

namespace mg
{
    struct PagedArgs
    {
        const void *q, *kc, *vc;
        const uint16_t *kd, *vd;
        const int32_t *table, *lens;
        void *out;
        int64_t ldq, ldt, ldo, window, num_pages;
        int nq, nkv, W, sh;
        float scale;
    };

    // first and one past the last key of request b
    MG_DEV void key_range(const PagedArgs &a, int b, int &lo, int &n)
    {
        n = min(max(a.lens[b], 0), a.W << a.sh);
        lo = a.window > 0 && n > a.window ? int(n - a.window) : 0;
    }

    // one work-group per (request, query head): a tile of 256 keys, one a thread, then the
    // tile's weights over the values, a thread per dim
    template <class S, class SO, bool Q8>
    __global__ __launch_bounds__(256) void k_attn_paged(PagedArgs a, int D)
    {
        using raw = typename S::raw;
        __shared__ float qf[128], p[256], red[4];
        __shared__ int64_t sl[256];
        const int b = blockIdx.x, h = blockIdx.y, g = h / (a.nq / a.nkv), tid = threadIdx.x;
        int lo, n;
        key_range(a, b, lo, n);
        if (tid < D) qf[tid] = S::dec(static_cast<const raw *>(a.q)[b * a.ldq + h * D + tid]);
        __syncthreads();
        float m = -__builtin_huge_valf(), l = 0.0f, o = 0.0f;
        auto val = [&](const void *c, const uint16_t *d, int64_t i) {
            if constexpr (Q8)
                return float(static_cast<const int8_t *>(c)[i]) * f16_f32(d[i / 32]);
            else
                return S::dec(static_cast<const raw *>(c)[i]);
        };
        for (int j0 = lo; j0 < n; j0 += 256) {
            const int j = j0 + tid;
            float s = -__builtin_huge_valf();
            int64_t at = -1;
            if (j < n) {
                const int page = a.table[b * a.ldt + (j >> a.sh)];
                if (page >= 0 && page < a.num_pages) {
                    at = (((int64_t(page) << a.sh) + (j & ((1 << a.sh) - 1))) * a.nkv + g) * D;
                    float dot = 0.0f;
                    for (int i = 0; i < D; ++i) dot = __builtin_fmaf(qf[i], val(a.kc, a.kd, at + i), dot);
                    s = dot * a.scale;
                }
            }
            float mt = dpp_max(s);
            if ((tid & 63) == 0) red[tid >> 6] = mt;
            __syncthreads();
            mt = __builtin_fmaxf(__builtin_fmaxf(red[0], red[1]), __builtin_fmaxf(red[2], red[3]));
            const float mn = __builtin_fmaxf(m, mt);
            const float ref = mn == -__builtin_huge_valf() ? 0.0f : mn;
            const float w = at < 0 ? 0.0f : exp_f32(s - ref);
            p[tid] = w;
            sl[tid] = at;
            __syncthreads();
            const float corr = exp_f32(m - ref);
            l *= corr;
            o *= corr;
            m = mn;
            for (int i = 0; i < 256; ++i) {
                const int64_t ai = sl[i];
                if (ai < 0) continue;
                l += p[i];
                if (tid < D) o = __builtin_fmaf(p[i], val(a.vc, a.vd, ai + tid), o);
            }
            __syncthreads();
        }
        if (tid < D) {
            const float r = l == 0.0f ? 0.0f : o / l;
            static_cast<typename SO::raw *>(a.out)[b * a.ldo + h * D + tid] = SO::enc32(r);
        }
    }

    void launch_attn_decode_paged(mg_ctx *c, const void *q, int64_t ldq, const void *kc, const void *vc,
                                  const uint16_t *kd, const uint16_t *vd, const int32_t *table, int64_t ldt,
                                  int64_t max_pages, const int32_t *lens, int64_t seqs, int64_t nq, int64_t nkv,
                                  int64_t D, int64_t page_size, int64_t num_pages, int64_t window, double scaling,
                                  void *out, int64_t ldo, int dt, int dt_out)
    {
        const int sh = page_shift(page_size, "attn_decode_paged");
        need(seqs >= 0 && nq > 0 && nkv > 0 && nq % nkv == 0,
             "attn_decode_paged: q_heads must be a multiple of kv_heads");
        need(nq <= 65535, "attn_decode_paged: too many heads");
        need(D == 64 || D == 128, "attn_decode_paged: head_dim must be 64 or 128");
        need(dt == BF16 || dt == F16, "attn_decode_paged: dtype must be bf16 or f16");
        need(dt_out == dt || dt_out == F32, "attn_decode_paged: dtype_out must be f32 or q's dtype");
        need(max_pages > 0 && num_pages > 0 && num_pages < (int64_t(1) << 31), "attn_decode_paged: bad table or pool size");
        need(max_pages <= ((int64_t(1) << 31) - 1) >> sh, "attn_decode_paged: a row's tokens must be below 2^31");
        if (seqs == 0) return;
        need(q && kc && vc && table && lens && out, "attn_decode_paged: NULL tensor");
        need((kd == nullptr) == (vd == nullptr), "attn_decode_paged: give both k_scale and v_scale, or neither");
        if (ldq == 0) ldq = nq * D;
        if (ldo == 0) ldo = nq * D;
        if (ldt == 0) ldt = max_pages;
        need(ldq >= nq * D && ldo >= nq * D && ldt >= max_pages, "attn_decode_paged: row stride smaller than a row");
        need(aligned16(q) && aligned16(kc) && aligned16(vc) && ldq % 8 == 0,
             "attn_decode_paged: q rows and caches must be 16-byte aligned");
        need(seqs < (int64_t(1) << 31), "attn_decode_paged: too many requests");
        const PagedArgs a{q,   kc,  vc,     kd,        vd,      table,    lens,           out, ldq,
                          ldt, ldo, window, num_pages, int(nq), int(nkv), int(max_pages), sh,  float(scaling)};
        auto go = [&](auto kern) {
            hipLaunchKernelGGL(kern, dim3(unsigned(seqs), unsigned(nq)), dim3(256), 0, c->stream, a, int(D));
            check_launch("k_attn_paged");
        };
        auto typed = [&](auto s) {
            using S = decltype(s);
            if (dt_out == F32)
                kd ? go(k_attn_paged<S, SF32, true>) : go(k_attn_paged<S, SF32, false>);
            else
                kd ? go(k_attn_paged<S, S, true>) : go(k_attn_paged<S, S, false>);
        };
        dt == BF16 ? typed(SBf16{}) : typed(SF16{});
    }
} // namespace mg
