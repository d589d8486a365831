// Decode attention over MXFP4 pages for gfx950: the operator of k_attn_paged.hip
// (one new token for each of many requests, its division of the keys among teams
// and its join) where a key's row of a head is head_dim / 2 bytes of e2m1 codes
// and head_dim / 32 bytes of powers of two.
//
// A wave takes steps of 64 keys, lane l the slot and the scales of key l; rows
// come as there, in 16-byte pieces a step ahead, through LDS.
//   S^T = K Q^T: 16 x 16 x 32 bf16 products, lane (key n, c) holding dims
// c D/4 .. of its key, all of one block: codes become bf16 with that block's scale,
// exactly, two an instruction. (bf16 holds every code at every scale; f16 queries
// enter as the exact sum of two bf16 parts.) Row 4 a + b of tile t is key
// 16 a + 4 t + b, so that lane (head n, c) ends with the scores of keys 16 c .. + 15.
//   O += P V: a transposing 4-bit read gives lane (dim n, c) the codes of those
// keys for one dim, a pair of keys a byte, so they become bf16 without a scale. A V
// block's scale goes to its weights: they are split into bf16 parts once, the
// first by truncation, which keeps every part positive or zero, and each part takes
// the power of two in its exponent field, for two keys at once by one saturating
// subtraction of 254 - s from the field of 2^127 p. What falls below bf16's smallest
// exponent becomes zero or less than 2^-126: weights times scales down to 2^-118 keep
// 2^-16 of themselves. Block scales of 255 are looked for: the codes of such a pair
// become NaN (0 of the other key's weight times NaN would be as wrong, but both are
// attended, and the sums are NaN either way).
#include "mg_attn_paged.hpp"
#include "mg_mxfp4.hpp"

namespace mg
{
    constexpr int kMxStep = 64; // keys a wave takes at once

    // each half less d's, not below 0
    MG_DEV uint32_t pk_subsat_u16(uint32_t a, uint32_t d)
    {
        return __builtin_bit_cast(uint32_t,
                                  __builtin_elementwise_sub_sat(__builtin_bit_cast(u16x2, a), __builtin_bit_cast(u16x2, d)));
    }
    // the upper halves of a and b as a pair
    MG_DEV uint32_t high_halves(float a, float b)
    {
        return __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, b), __builtin_bit_cast(uint32_t, a), 0x07060302u);
    }

    template <class S, class SO, int KB> // KB = head_dim / 32
    __global__ __launch_bounds__(256, 2) void k_attn_mxfp4(PagedArgs a)
    {
        constexpr int D = 32 * KB, NT = 2 * KB; // NT output tiles of 16 dims
        constexpr int U = 4 * kMxStep;
        constexpr int RB = D / 2;               // bytes of a row
        constexpr int LPR = RB / 16;            // lanes a row
        constexpr int RPI = 64 / LPR;           // rows a load instruction covers
        constexpr int NLD = kMxStep / RPI;
        constexpr int KW = D / 32;              // a lane's words of a key: 32 / 4 (or 16 / 4) dims of 8
        // LDS rows: padded against bank conflicts, and every 16 of them by another 64 bytes (a K read takes rows
        // 16 a + b)
        constexpr int SR = RB + 16, SG = 16 * SR + 64;
        constexpr int WB = 4 * SG;              // LDS bytes of a wave's K or V
        constexpr int SO4 = D + 4;              // row stride of a wave's output in LDS (floats)
        static_assert(16 * SO4 * 4 <= 2 * WB, "a wave's output takes the place of its K and V");
        using raw = typename SO::raw;
        constexpr bool QF16 = S::dt == F16;
        constexpr int NP = SO::dt == F32 ? 3 : 2; // bf16 parts of a weight
        constexpr float kLow = -__builtin_huge_valf();
        using KV = std::conditional_t<KB == 4, uint32_t, uint16_t>; // a key's scales
        __shared__ __align__(16) char lds[4][2 * WB];
        __shared__ __align__(16) uint16_t vsc[4][KB][kMxStep]; // (254 - s) << 7 of a key's V blocks, 0x8000 for NaN
        __shared__ float wm[4][16], wl[4][16];
        const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
        // runs of eight work-groups (a key's heads) on one XCD: two heads' rows share a 128-byte line, eight heads' scales one
        constexpr int G = 8;
        int wg = blockIdx.x;
        if (wg < int(gridDim.x) / (8 * G) * (8 * G)) {
            const int xcd = wg % 8, turn = wg / 8;
            wg = turn / G * (8 * G) + xcd * G + turn % G;
        }
        const int team = wg / a.vh, v = wg - team * a.vh;
        const Run run = find_run<kMxStep>(a, team);
        const bool notes = a.teams > 1 && v == 0 && threadIdx.x == 0; // who writes the cuts down
        if (run.u0 >= run.u1) { // the whole work-group
            if (notes && a.by_team) a.cut[team] = PagedCut{};
            return;
        }
        const int nsub = a.hpg / a.hw, g = v / nsub;
        const int h0 = g * a.hpg + (v - g * nsub) * a.hw;
        const int n = lane & 15, c = lane >> 4;
        char *sk = lds[wv], *sv = sk + WB;
        const int pc = lane % LPR, pr = lane / LPR;
        const int64_t rowb = int64_t(a.nkv) * RB; // bytes between slots
        const char *kg = static_cast<const char *>(a.kc) + int64_t(g) * RB;
        const char *vg = static_cast<const char *>(a.vc) + int64_t(g) * RB;
        const KV *ksg = reinterpret_cast<const KV *>(a.kd) + g, *vsg = reinterpret_cast<const KV *>(a.vd) + g;
        const uint32_t lane_off = uint32_t(pr * rowb) + 16 * pc; // (checked on the host: below 2^32)
        const int cap = a.W << a.sh, psm = (1 << a.sh) - 1;
        auto at_row = [](int row) { return row * SR + (row >> 4) * 64; };

        // a part of a request in the run: units [at, end), attended keys [klo, khi), and the
        // units of the run behind it
        struct Part
        {
            int b, at, end, units, k0, klo, khi, behind;
        };
        auto part_of = [&](int b, int at, int left) {
            const PagedSpan sp = paged_span<kMxStep>(__builtin_amdgcn_readfirstlane(a.lens[b]), cap, a.window);
            Part s;
            s.b = b;
            s.at = at;
            s.units = sp.units;
            s.end = sp.units - at < left ? sp.units : at + left;
            s.behind = left - (s.end - at);
            s.k0 = sp.base + at * U;
            s.klo = s.k0 > sp.lo ? s.k0 : sp.lo;
            const int64_t ke = int64_t(sp.base) + int64_t(s.end) * U;
            s.khi = ke < sp.n ? int(ke) : sp.n;
            return s;
        };
        Part cur = part_of(run.b, run.u0 - run.p, run.u1 - run.u0);

        // the step whose table entries are read next: every wave takes a step of each part, which may be empty
        Part ahead = cur;
        int akb = cur.k0 + kMxStep * wv;
        bool more_ahead = true;
        auto advance = [&]() {
            akb += U;
            if (akb < ahead.khi) return;
            more_ahead = ahead.behind > 0;
            if (!more_ahead) return;
            ahead = part_of(ahead.b + 1, 0, ahead.behind);
            akb = ahead.k0 + kMxStep * wv;
        };
        // the slot of key akb + lane, or -1
        auto slot_of = [&]() {
            const int key = akb + lane;
            if (!more_ahead || key < ahead.klo || key >= ahead.khi) return -1;
            const int page = a.table[ahead.b * a.ldt + (key >> a.sh)];
            return page >= 0 && page < a.num_pages ? (page << a.sh) + (key & psm) : -1;
        };
        Vec<uint32_t, 4> stk[NLD], stv[NLD];
        uint32_t ssk, ssv; // scales of key `lane`
        auto stage = [&](int slot, uint64_t seen) {
            ssk = ssv = 0;
            if (slot >= 0) {
                ssk = ksg[int64_t(slot) * a.nkv];
                ssv = vsg[int64_t(slot) * a.nkv];
            }
            if (seen == ~uint64_t(0) && psm + 1 >= RPI) {
#pragma unroll
                for (int i = 0; i < NLD; ++i) {
                    int64_t o = __builtin_amdgcn_readlane(slot, RPI * i) * rowb;
                    __asm__("" : "+s"(o)); // the rows' base stays in scalar registers, the lane's offset in one
                    const char *kp = kg + o, *vp = vg + o;
                    stk[i] = ld16_stream<uint32_t, 4>(reinterpret_cast<const uint32_t *>(kp + lane_off));
                    stv[i] = ld16_stream<uint32_t, 4>(reinterpret_cast<const uint32_t *>(vp + lane_off));
                }
                return;
            }
#pragma unroll
            for (int i = 0; i < NLD; ++i) {
                const int s = __shfl(slot, pr + RPI * i, 64);
                stk[i] = Vec<uint32_t, 4>{{0u, 0u, 0u, 0u}};
                stv[i] = stk[i];
                if (s >= 0) {
                    const int64_t o = s * rowb + 16 * pc;
                    stk[i] = ld16_stream<uint32_t, 4>(reinterpret_cast<const uint32_t *>(kg + o));
                    stv[i] = ld16_stream<uint32_t, 4>(reinterpret_cast<const uint32_t *>(vg + o));
                }
            }
        };
        int slot = slot_of();
        uint64_t seen = __builtin_amdgcn_ballot_w64(slot >= 0); // keys of the staged step, one bit each
        stage(slot, seen);
        advance();
        slot = slot_of();

        // B of S^T: lane (head n, c) holds q[n][c D / 4 + 8 i ..], zero for padding heads; f16 as two bf16 parts
        bf16x8 qop[QF16 ? 2 : 1][KW];
        auto load_q = [&](int b) {
#pragma unroll
            for (int i = 0; i < KW; ++i) {
                const uint16_t *qp = static_cast<const uint16_t *>(a.q) + b * a.ldq + int64_t(h0 + n) * D + c * (D / 4) + 8 * i;
                Vec<uint32_t, 4> w{{0u, 0u, 0u, 0u}};
                if (n < a.hw) w = *reinterpret_cast<const Vec<uint32_t, 4> *>(qp);
                if constexpr (QF16) {
                    Vec<uint32_t, 4> hi, lo;
#pragma unroll
                    for (int k = 0; k < 4; ++k) mx_halves(w.v[k], hi.v[k], lo.v[k]);
                    qop[0][i] = __builtin_bit_cast(bf16x8, hi);
                    qop[1][i] = __builtin_bit_cast(bf16x8, lo);
                } else {
                    qop[0][i] = __builtin_bit_cast(bf16x8, w);
                }
            }
        };
        load_q(cur.b);
        for (;;) {
            f32x4 o[NT];
#pragma unroll
            for (int t = 0; t < NT; ++t) o[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            float m = kLow, l = 0.0f; // head n (replicated over c)
            bool any = false;         // the wave has seen a key that is not masked
            int kb = cur.k0 + kMxStep * wv;
            bool more;
            do {
                kb += U;
                more = kb < cur.khi;
                const uint64_t now = seen;
                uint32_t ks[4]; // the scales of this lane's key of each tile
                bool nan_v = false;
                if (now != 0) {
#pragma unroll
                    for (int i = 0; i < NLD; ++i) {
                        const int row = at_row(pr + RPI * i);
                        *reinterpret_cast<Vec<uint32_t, 4> *>(sk + row + 16 * pc) = stk[i];
                        *reinterpret_cast<Vec<uint32_t, 4> *>(sv + row + 16 * pc) = stv[i];
                    }
                    bool bad = false;
#pragma unroll
                    for (int i = 0; i < KB; ++i) {
                        const uint32_t s = ssv >> (8 * i) & 0xffu;
                        bad |= s == 255u;
                        vsc[wv][i][lane] = s == 255u ? uint16_t(0x8000) : uint16_t((254u - s) << 7);
                    }
                    nan_v = __builtin_amdgcn_ballot_w64(bad) != 0;
#pragma unroll
                    for (int t = 0; t < 4; ++t)
                        ks[t] = uint32_t(__shfl(int(ssk), 16 * (n >> 2) + 4 * t + (n & 3), 64)) >> (KB == 4 ? 8 * c : 8 * (c >> 1)) & 0xffu;
                    wave_lds_sync();
                }
                // the next step's rows and the table entries of the one behind it are requested now
                if (more_ahead) {
                    seen = __builtin_amdgcn_ballot_w64(slot >= 0);
                    stage(slot, seen);
                    advance();
                    slot = slot_of();
                }
                if (now == 0) continue;
                any = true;
                // scores of keys 16 c + 4 t + r for head n
                float sc[4][4], mx = kLow;
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    const Vec<uint32_t, KW> kw =
                        *reinterpret_cast<const Vec<uint32_t, KW> *>(sk + at_row(16 * (n >> 2) + 4 * t + (n & 3)) + 4 * KW * c);
                    f32x4 st = {0.0f, 0.0f, 0.0f, 0.0f};
                    const float f = mx_scale(ks[t]);
#pragma unroll
                    for (int i = 0; i < KW; ++i) {
                        const bf16x8 k = __builtin_bit_cast(bf16x8, mx_bf16(kw.v[i], f));
                        if constexpr (QF16) st = mfma_bf16(k, qop[1][i], st);
                        st = mfma_bf16(k, qop[0][i], st);
                    }
#pragma unroll
                    for (int r = 0; r < 4; ++r) sc[t][r] = st[r] * a.scale2;
                    if (now != ~uint64_t(0)) {
                        const uint32_t bits = uint32_t(now >> (16 * c + 4 * t));
#pragma unroll
                        for (int r = 0; r < 4; ++r) sc[t][r] = (bits >> r & 1) != 0 ? sc[t][r] : kLow;
                    }
#pragma unroll
                    for (int r = 0; r < 4; ++r) mx = __builtin_fmaxf(mx, sc[t][r]);
                }
                mx = rows4_max(mx);
                const float mn = __builtin_fmaxf(m, mx);
                // no score above -inf yet: a zero reference, so that -inf scores weigh 0
                // and only NaN ones reach the sum
                const float mref = mn == kLow ? 0.0f : mn;
                // weights: element 4 t + r of lane (head n, c) is key 16 c + 4 t + r
                float p[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) p[e] = __builtin_amdgcn_exp2f(sc[e >> 2][e & 3] - mref);
                if (__builtin_amdgcn_ballot_w64(mn != m) != 0) {
                    // some head's running max moved: rescale its sum and its O row
                    // (rows are heads 4c + r; their factors come from lanes 4c + r)
                    const float corr = __builtin_amdgcn_exp2f(m - mref); // first step: 2^-inf = 0
                    l *= corr;
                    float cr[4];
#pragma unroll
                    for (int r = 0; r < 4; ++r) cr[r] = __shfl(corr, 4 * c + r, 64);
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int r = 0; r < 4; ++r) o[t][r] *= cr[r];
                }
                m = mn;
#pragma unroll
                for (int e = 0; e < 16; e += 8)
                    l += ((p[e] + p[e + 1]) + (p[e + 2] + p[e + 3])) + ((p[e + 4] + p[e + 5]) + (p[e + 6] + p[e + 7]));
                // parts of 2^127 p, pairs of keys
                uint32_t w[NP][8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    float p0 = p[2 * i] * 0x1p127f, p1 = p[2 * i + 1] * 0x1p127f;
#pragma unroll
                    for (int k = 0; k < NP; ++k) {
                        w[k][i] = k + 1 < NP ? high_halves(p0, p1) : bf_pack(p0, p1);
                        p0 -= bf_lo(w[k][i]);
                        p1 -= bf_hi(w[k][i]);
                    }
                }
                // V as B of P V: lane (dim n, c) needs keys 16 c .. + 15 of dim 16 s + n
                const char *vr = sv + at_row(16 * c + n);
#pragma unroll
                for (int b = 0; b < KB; ++b) {
                    Vec<uint32_t, 4> d[2];
                    d[0] = *reinterpret_cast<const Vec<uint32_t, 4> *>(&vsc[wv][b][16 * c]);
                    d[1] = *reinterpret_cast<const Vec<uint32_t, 4> *>(&vsc[wv][b][16 * c + 8]);
                    Vec<uint32_t, 4> ws[NP][2];
#pragma unroll
                    for (int k = 0; k < NP; ++k)
#pragma unroll
                        for (int i = 0; i < 8; ++i) ws[k][i >> 2].v[i & 3] = pk_subsat_u16(w[k][i], d[i >> 2].v[i & 3]);
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const int t = 2 * b + u;
                        const Vec<uint32_t, 2> x = lds_read_tr4(vr + 8 * t);
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            Vec<uint32_t, 4> vb = mx_bf16(x.v[h], 1.0f);
                            if (nan_v) {
#pragma unroll
                                for (int i = 0; i < 4; ++i)
                                    if ((d[h].v[i] & 0x80008000u) != 0) vb.v[i] = 0x7fc07fc0u;
                            }
#pragma unroll
                            for (int k = 0; k < NP; ++k)
                                o[t] = mfma_bf16(__builtin_bit_cast(bf16x8, ws[k][h]), __builtin_bit_cast(bf16x8, vb), o[t]);
                        }
                    }
                }
                wave_lds_sync(); // this step's reads are done before the next one's writes
            } while (more);
            // the next request, while the waves join
            const bool go_on = cur.behind > 0;
            Part next = cur;
            if (go_on) {
                next = part_of(cur.b + 1, 0, cur.behind);
                load_q(next.b);
            }

            // join the four waves: their outputs take the place of K and V in LDS
            l = rows4_sum(l);
            float *so = reinterpret_cast<float *>(lds[wv]);
            // keys, but none above -inf: the sum, 0 (or NaN), says so by 1. Beside a maximum it weighs 0; where no
            // part has one the parts' sums are added as they are, and 0 means that nothing was attended.
            if (c == 0) {
                wm[wv][n] = m;
                wl[wv][n] = any && m == kLow ? l + 1.0f : l;
            }
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) so[(4 * c + r) * SO4 + 16 * t + n] = o[t][r];
            __syncthreads();
            const bool whole = cur.at == 0 && cur.end == cur.units;
            const int first = run.u1 - cur.behind - cur.end; // the request's first unit
            if (notes && leaves_cut(a.by_team, cur.at, cur.behind))
                a.cut[a.by_team ? team : cur.b] =
                    cur.at == 0 ? paged_cut(run.d, team, cur.b, first, cur.units) : PagedCut{};
            const int hh = threadIdx.x >> 4, d0 = (threadIdx.x & 15) * (D / 16);
            if (hh < a.hw) {
                const float top = __builtin_fmaxf(__builtin_fmaxf(wm[0][hh], wm[1][hh]), __builtin_fmaxf(wm[2][hh], wm[3][hh]));
                float sum = 0.0f, acc[D / 16];
#pragma unroll
                for (int e = 0; e < D / 16; ++e) acc[e] = 0.0f;
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const float f = weight_of(wm[w][hh], top);
                    sum = __builtin_fmaf(f, wl[w][hh], sum);
                    const float *src = reinterpret_cast<const float *>(lds[w]) + hh * SO4 + d0;
#pragma unroll
                    for (int e = 0; e < D / 16; e += 4) {
                        const Vec<float, 4> x = *reinterpret_cast<const Vec<float, 4> *>(src + e);
#pragma unroll
                        for (int i = 0; i < 4; ++i) acc[e + i] = __builtin_fmaf(f, x.v[i], acc[e + i]);
                    }
                }
                if (whole) {
                    const float inv = inverse(sum, top);
                    raw *dst = static_cast<raw *>(a.out) + cur.b * a.ldo + int64_t(h0 + hh) * D + d0;
#pragma unroll
                    for (int e = 0; e < D / 16; ++e) dst[e] = SO::enc32(acc[e] * inv);
                } else {
                    const int64_t row = (int64_t(team_place(run.d, team, first)) * a.vh + v) * a.hw + hh;
                    float *dst = a.part + row * D + d0;
#pragma unroll
                    for (int e = 0; e < D / 16; e += 4)
                        *reinterpret_cast<Vec<float, 4> *>(dst + e) = Vec<float, 4>{{acc[e], acc[e + 1], acc[e + 2], acc[e + 3]}};
                    if (d0 == 0) {
                        float *ml = a.part + 2 * int64_t(a.teams) * a.vh * a.hw * D + 2 * row;
                        ml[0] = top;
                        ml[1] = sum;
                    }
                }
            }
            __syncthreads(); // the next part's first step writes where the outputs were
            if (!go_on) break;
            cur = next;
        }
    }

    void launch_attn_decode_mxfp4(mg_ctx *c, const void *q, int64_t ldq, const uint8_t *kc, const uint8_t *vc,
                                  const uint8_t *ks, const uint8_t *vs, const int32_t *table, int64_t ldt,
                                  int64_t max_pages, const int32_t *lens, int64_t seqs, int64_t nq, int64_t nkv,
                                  int64_t D, int64_t page_size, int64_t num_pages, int64_t window, double scaling,
                                  void *out, int64_t ldo, int dt, int dt_out)
    {
        PagedArgs a = paged_args(q, ldq, kc, vc, ks, vs, table, ldt, max_pages, lens, seqs, nq, nkv, D, page_size,
                                 num_pages, window, scaling, out, ldo, dt, dt_out);
        if (a.R == 0) return;
        need(ks && vs, "attn_decode_paged: MXFP4 pages need their scales");
        a.kd = reinterpret_cast<const uint16_t *>(ks), a.vd = reinterpret_cast<const uint16_t *>(vs);
        paged_divide(c, a, D, 2, kMxStep);
        auto go = [&](auto kern) {
            hipLaunchKernelGGL(kern, dim3(unsigned(a.teams * a.vh)), dim3(256), 0, c->stream, a);
            check_launch("k_attn_mxfp4");
        };
        auto sized = [&](auto s, auto so) {
            using S = decltype(s);
            using SO = decltype(so);
            D == 128 ? go(k_attn_mxfp4<S, SO, 4>) : go(k_attn_mxfp4<S, SO, 2>);
        };
        if (dt_out == F32)
            dt == BF16 ? sized(SBf16{}, SF32{}) : sized(SF16{}, SF32{});
        else
            dt == BF16 ? sized(SBf16{}, SBf16{}) : sized(SF16{}, SF16{});
        paged_join(c, a, D, dt_out);
    }
} // namespace mg
