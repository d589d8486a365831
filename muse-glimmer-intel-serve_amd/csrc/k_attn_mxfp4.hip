// Decode attention over MXFP4 pages for gfx950: the operator of k_attn_paged.hip
// (one new token for each of many requests, its division of the keys among teams
// and its join) where a key's row of a head is head_dim / 2 bytes of e2m1 codes
// and head_dim / 32 bytes of powers of two.
//
// A wave takes steps of 64 rows: 64 keys of a head, or 32 keys of two heads that lie beside
// each other. Rows, their scales and the table entries that lead to them are loaded
// into LDS two steps ahead, counted by the kernel. (A step ahead through registers, with a
// wait for table entries amid the rows on their way, took 88 us where this takes 66: 64
// ragged requests of up to 8000 keys, 40 / 8 heads, 256 MB from HBM.)
//   S^T = K Q^T: 16 x 16 x 32 bf16 products, lane (row n, c) holding dims c D/4 .. of
// its row, all of one block: codes become bf16 with that block's scale, exactly, two an
// instruction. (bf16 holds every code up to scale 252, a quarter of it past that; f16
// queries enter as the exact sum of two bf16 parts.) Row 4 a + b of tiles is such that lane
// (query head n, c) ends with the scores that O += P V wants of it, 16 keys'; of two heads with up to eight queries each,
// columns below 8 are the first's, and a lane keeps its own head's eight scores of each:
// exponentials and weights are then no more than a head's.
//   O += P V: a transposing 4-bit read gives lane (dim n, c) the codes of 16 rows
// for one dim, a pair of keys a byte, so they become bf16 without a scale. A V
// block's scale goes to its weights: they are split into bf16 parts once, the
// first by truncation, which keeps every part positive or zero (two parts for 16-bit
// outputs, 2^-16 of a weight; three for f32), and each part takes the power of two in its
// exponent field, for two keys at once by one saturating subtraction of 127 - s (254 -
// s from the field of 2^127 p where an s is above 127). What falls below bf16's
// smallest exponent becomes zero or less than 2^-126: weights times scales down to 2^-118
// keep 2^-16 of themselves. V scales of 255 are looked for, and their blocks' outputs made NaN.
//   A step of two heads is about 390 vector instructions and 48 products a wave; two waves
// a SIMD (153 to 253 registers, 75 KB of LDS a work-group) are busy with them half of the
// time, 6 TB/s in the run's middle. The rest is the start (sums of lengths, table, rows:
// three trips to memory, 7 us for a single step), a last step shorter than others' and the
// join's launch, 5 us.
#include "mg_attn_paged.hpp"
#include "mg_mxfp4.hpp"

namespace mg
{
    template <class T>
    MG_DEV T uniform_load(const T *p) // through scalar registers: p is the same in every lane
    {
        return *reinterpret_cast<const __attribute__((address_space(4))) T *>(reinterpret_cast<uintptr_t>(p));
    }

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

    // KB = head_dim / 32; HP: kv heads a wave takes, two with up to eight query heads each
    template <class S, class SO, int KB, int HP>
    __global__ __launch_bounds__(256, 2) void k_attn_mxfp4(PagedArgs a)
    {
        constexpr int D = 32 * KB, NT = 2 * KB; // NT output tiles of 16 dims
        constexpr int KS = 64 / HP, U = 4 * KS; // keys of a step, of a unit
        constexpr int RB = D / 2;               // bytes of a row
        constexpr int LPR = RB / 16;            // lanes a row
        constexpr int RPI = 64 / LPR;           // rows a load instruction covers
        constexpr int NLD = 64 / RPI;
        constexpr int OPS = 2 * NLD + 3;        // loads of a step: its rows, its scales, another's table entries
        constexpr int KW = D / 32;              // a lane's words of a key: D / 4 dims
        constexpr int WB = 64 * RB;             // LDS bytes of a step's K or V
        constexpr int NV = 16 / HP;             // a lane's keys of its query head
        using raw = typename SO::raw;
        constexpr bool QF16 = S::dt == F16;
        constexpr int NP = SO::dt == F32 ? 3 : 2; // bf16 parts of a weight
        constexpr float kLow = -__builtin_huge_valf();
        static_assert(2 * WB >= 16 * 64 * 4, "64 dims of a wave's output take the place of a step");
        __shared__ __align__(16) char lds[4][2][2 * WB];       // K and V of two steps
        __shared__ uint32_t scales[4][2][2][64];               // of two steps, K's and V's, a row's a word
        __shared__ int32_t entries[4][2][64];                  // of two steps
        __shared__ __align__(16) uint16_t vsc[4][KB][64];      // exponents to take from weights, for a row's V blocks
        __shared__ float wm[4][16], wl[4][16];
        __shared__ uint32_t place[4];                          // of a wave's output
        const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
        // runs of eight work-groups on one XCD: a key's heads share lines of rows and scales
        constexpr int G = 8;
        int wg = blockIdx.x;
        if (wg < int(gridDim.x) / (8 * G) * (8 * G)) {
            const int xcd = wg % 8, turn = wg / 8;
            wg = turn / G * (8 * G) + xcd * G + turn % G;
        }
        const int wgs = a.vh / HP, team = wg / wgs, v = wg - team * wgs;
        const Run run = find_run<KS>(a, team);
        const bool notes = a.teams > 1 && v == 0 && threadIdx.x == 0; // who writes the cuts down
        if (run.u0 >= run.u1) { // the whole work-group
            if (notes && a.by_team) a.cut[team] = PagedCut{};
            return;
        }
        const int nsub = a.hpg / a.hw, g0 = v / nsub * HP, sub = v % nsub;
        const int n = lane & 15, c = lane >> 4;
        // of column `col` of 16: the kv head, the query head's place in its group and among all
        auto kv_of = [&](int col) { return g0 + (HP == 2 ? col >> 3 : 0); };
        auto place_of = [](int col) { return HP == 2 ? col & 7 : col; };
        auto head_of = [&](int col) { return kv_of(col) * a.hpg + sub * a.hw + place_of(col); };
        // In LDS a step is 64 rows, a key's two heads one behind the other. A lane's values of it: (e, j), e the head
        // (or 8 keys' half of 16), j the key, which are this row.
        auto row_of = [](int cc, int e, int j) { return HP == 1 ? 16 * cc + 8 * e + j : 16 * cc + 2 * j + e; };
        // A row's 16-byte pieces lie in turned order, so that 16 rows' reads of one piece meet fewer banks twice: rows with
        // equal row % 4 differ in one of these. (A third of the LDS cycles are conflicts still, of a pair; 28 % of one head.)
        auto turned = [](int row) { return LPR == 4 ? ((row >> 2) ^ (row >> 4)) & 3 : ((row >> 3) ^ (row >> 4)) & 1; };
        const int pr = lane / LPR;
        const int64_t rowb = int64_t(a.nkv) * RB; // bytes between slots
        const uint8_t *kg = static_cast<const uint8_t *>(a.kc) + int64_t(g0) * RB;
        const uint8_t *vg = static_cast<const uint8_t *>(a.vc) + int64_t(g0) * RB;
        const int sg = (g0 + (HP == 2 ? lane & 1 : 0)) * KB; // of the lane's row's scales, from their slot's
        // of load i's row `pr`: (row >> 4 is i more there, or the same)
        const uint32_t lane_piece = 16 * ((lane % LPR) ^ turned(pr));
        auto piece = [&](int i) { return LPR == 4 ? lane_piece ^ 16u * i : lane_piece; };
        const uint32_t lane_row = uint32_t(pr / HP * rowb) + pr % HP * RB; // (checked on the host: below 2^32)
        const int cap = a.W << a.sh, psm = (1 << a.sh) - 1;
        // The scaling comes with the weights' exponent, as a positive number: a negative one turns the queries' signs, and
        // at zero they are zeros (infinities and NaN stay, for their product with zero is NaN).
        const float scale2 = a.scale2 == 0.0f ? 1.0f : __builtin_fabsf(a.scale2);
        const uint32_t flip = a.scale2 < 0.0f ? 0x80008000u : 0u;

        // a part of a request in the run: units [at, end), attended keys [klo, khi), and the
        // units of the run behind it
        struct Part
        {
            int b, at, end, units, k0, klo, khi, behind;
        };
        auto part_of = [&](int b, int at, int left) {
            const PagedSpan sp = paged_span<KS>(uniform_load(a.lens + __builtin_amdgcn_readfirstlane(b)), cap, a.window);
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

        // Steps are asked for in this order: their table entries four ahead, their rows and scales two ahead. All of that
        // goes to LDS, so that the kernel alone counts what is under way: a wait in the middle for an older load would be
        // a wait for the younger ones' rows, too.
        Part ahead = cur;
        int akb = cur.k0 + KS * wv;
        bool more_ahead = true;
        auto advance = [&]() { // every wave takes a step of each part, which may be empty
            akb += U;
            if (akb < ahead.khi) return;
            more_ahead = ahead.behind > 0;
            if (!more_ahead) return;
            ahead = part_of(ahead.b + 1, 0, ahead.behind);
            akb = ahead.k0 + KS * wv;
        };
        struct Ask
        {
            int kb;
            uint64_t rows; // those of attended keys
            bool is;
        };
        auto ask = [&](int par) { // the entries of step akb's keys, a row each
            Ask s;
            s.is = more_ahead;
            s.kb = akb;
            s.rows = 0;
            const int32_t *p = a.lens;
            if (more_ahead) {
                const int key = akb + lane / HP;
                s.rows = __builtin_amdgcn_ballot_w64(key >= ahead.klo && key < ahead.khi);
                const int in = key < ahead.klo ? ahead.klo : key < ahead.khi ? key : ahead.khi - 1;
                if (s.rows != 0) p = a.table + (ahead.b * a.ldt + (in >> a.sh));
                advance();
            }
            lds_load_at<4>(p, lds_address(reinterpret_cast<const char *>(entries[wv][par])));
            return s;
        };
        Ask next0 = ask(0), next1 = ask(1);
        // Asks for step next0's rows and scales, into the place `par`, and for the entries of the step two behind it.
        // Returns the rows that are there; those that are not may stay what they were or be others: any finite codes.
        bool full = false; // all OPS loads
        auto stage = [&](int par) {
            const int32_t entry = entries[wv][par][lane];
            const bool there = (next0.rows >> lane & 1) != 0 && entry >= 0 && entry < a.num_pages;
            const int slot = there ? (entry << a.sh) + ((next0.kb + lane / HP) & psm) : -1;
            const uint64_t seen = __builtin_amdgcn_ballot_w64(there);
            const uint32_t to = lds_address(lds[wv][par]);
            full = seen != 0;
            if (full) {
                const int f = __builtin_ctzll(seen), first = __builtin_amdgcn_readlane(slot, f);
                if ((psm + 1) * HP >= RPI) {
                    // a load's keys lie in one page: from the first that is there (of the step, if the load has none)
#pragma unroll
                    for (int i = 0; i < NLD; ++i) {
                        const uint64_t bits = seen >> (RPI * i) & ((uint64_t(1) << RPI) - 1);
                        const int r = bits != 0 ? RPI * i + __builtin_ctzll(bits) : f;
                        const int64_t o = (__builtin_amdgcn_readlane(slot, r) - r % RPI / HP) * rowb;
                        const uint32_t off = lane_row + piece(i);
                        lds_load(kg + o, off, to + 1024 * i);
                        lds_load(vg + o, off, to + WB + 1024 * i);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < NLD; ++i) {
                        int s = __shfl(slot, pr + RPI * i, 64);
                        s = s >= 0 ? s : first;
                        const int64_t o = s * rowb + (pr % HP * RB + piece(i));
                        lds_load_at(kg + o, to + 1024 * i);
                        lds_load_at(vg + o, to + WB + 1024 * i);
                    }
                }
                const int64_t o = int64_t(there ? slot : first) * (a.nkv * KB) + sg;
                const uint32_t ts = lds_address(reinterpret_cast<const char *>(scales[wv][par][0]));
                lds_load_at<KB>(reinterpret_cast<const uint8_t *>(a.kd) + o, ts);
                lds_load_at<KB>(reinterpret_cast<const uint8_t *>(a.vd) + o, ts + 256);
            }
            __asm__ volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); // the entries are read
            next0 = next1;
            if (next0.is) next1 = ask(par);
            else full = false;
            return seen;
        };
        __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");
        uint64_t now = stage(0), then = 0; // rows that are there, of the step that is next and of the one behind it
        if (next0.is) then = stage(1);
        else full = false;

        // B of S^T: lane (head n, c) holds q[n][c D / 4 + 8 i ..], zero for padding heads; f16 as two bf16 parts
        bf16x8 qop[QF16 ? 2 : 1][KW];
        auto load_q = [&](int b) {
#pragma unroll
            for (int i = 0; i < KW; ++i) {
                const uint16_t *qp = static_cast<const uint16_t *>(a.q) + b * a.ldq + int64_t(head_of(n)) * D + c * (D / 4) + 8 * i;
                Vec<uint32_t, 4> w{{0u, 0u, 0u, 0u}};
                if (place_of(n) < a.hw) w = *reinterpret_cast<const Vec<uint32_t, 4> *>(qp);
#pragma unroll
                for (int k = 0; k < 4; ++k) w.v[k] ^= flip;
                if (a.scale2 == 0.0f) {
                    constexpr uint32_t top = QF16 ? 0x7c00u : 0x7f80u; // the exponent of what is not finite
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        w.v[k] &= ((w.v[k] & top) == top ? 0xffffu : 0u) | ((w.v[k] >> 16 & top) == top ? 0xffff0000u : 0u);
                }
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
        int par = 0;
        for (;;) {
            f32x4 o[HP][NT];
#pragma unroll
            for (int e = 0; e < HP; ++e)
#pragma unroll
                for (int t = 0; t < NT; ++t) o[e][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            float m = kLow, l = 0.0f; // of head n (replicated over c)
            bool any = false;   // the wave has seen a key that is not masked
            uint32_t nan_v = 0; // V blocks that hold a NaN, a bit each, a head's eight
            int kb = cur.k0 + KS * wv;
            bool more;
            do {
                kb += U;
                more = kb < cur.khi;
                if (full)
                    __asm__ volatile("s_waitcnt vmcnt(%0)" ::"n"(OPS) : "memory"); // but for the next step's
                else
                    __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");
                // the step's operands, all at once: its place takes another one's
                Vec<uint32_t, KW> kw[4]; // row 4 a + b of tile 2 e + t is value (e, 4 t + b) of lanes c = a
                float kf[4];             // the scales of this lane's row of each tile
                Vec<uint32_t, 2> vx[NT];
                bool raised = false, past = false;
                if (now != 0) {
                    const char *sk = lds[wv][par], *sv = sk + WB;
#pragma unroll
                    for (int t = 0; t < 4; ++t) {
                        const int row = row_of(n >> 2, t >> 1, 4 * (t & 1) + (n & 3)), at = 4 * KW * c;
                        kw[t] = *reinterpret_cast<const Vec<uint32_t, KW> *>(sk + row * RB + (at & 15) + ((at & ~15) ^ 16 * turned(row)));
                        kf[t] = mx_scale(reinterpret_cast<const uint8_t *>(&scales[wv][par][0][row])[KB == 4 ? c : c >> 1]);
                    }
                    const int vrow = row_of(c, n >> 3, n & 7);
#pragma unroll
                    for (int t = 0; t < NT; ++t)
                        vx[t] = lds_read_tr4(sv + vrow * RB + 8 * (t & 1) + ((8 * (t & ~1)) ^ 16 * turned(vrow)));
                    const uint32_t ssk = scales[wv][par][0][lane], ssv = scales[wv][par][1][lane];
                    // V blocks' scales; past 127 anywhere they are taken from 254 and the weights by 2^127 higher, and
                    // a NaN is among those. So are K scales from 192 on, which want another way (below).
                    const uint32_t far = ssk & ssk << 1;
                    raised = (__builtin_amdgcn_ballot_w64(((ssv | far) & 0x80808080u) != 0) & now) != 0;
                    const uint32_t from = raised ? 0x00fe00feu : 0x007f007fu;
                    const int at = HP == 1 ? lane : (lane & 48) + 8 * (lane & 1) + (lane & 15) / 2;
                    const uint32_t even = KB == 4 ? ssv & 0x00ff00ffu : (ssv & 0xffu) | (ssv & 0xff00u) << 8;
                    const uint32_t d0 = pk_subsat_u16(from, even) << 7;
                    vsc[wv][0][at] = uint16_t(d0);
                    vsc[wv][KB / 2][at] = uint16_t(d0 >> 16);
                    if constexpr (KB == 4) {
                        const uint32_t d1 = pk_subsat_u16(from, ssv >> 8 & 0x00ff00ffu) << 7;
                        vsc[wv][1][at] = uint16_t(d1);
                        vsc[wv][3][at] = uint16_t(d1 >> 16);
                    }
                    if (raised) {
                        past = (__builtin_amdgcn_ballot_w64((far & 0x80808080u) != 0) & now) != 0;
#pragma unroll
                        for (int e = 0; e < HP; ++e) {
                            const uint64_t of = HP == 1 ? now : now & (0x5555555555555555u << e);
#pragma unroll
                            for (int i = 0; i < KB; ++i)
                                if ((__builtin_amdgcn_ballot_w64((ssv >> (8 * i) & 0xffu) == 255u) & of) != 0) nan_v |= 1u << (8 * e + i);
                        }
                    }
                    wave_lds_sync();
                    __asm__ volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); // (loads into LDS keep no order with its reads)
                }
                const uint64_t rows = now;
                const int mine = par;
                now = then;
                then = 0;
                par ^= 1;
                if (more) { // (else its place takes the outputs first)
                    full = false;
                    if (next0.is) then = stage(mine);
                }
                if (rows == 0) continue;
                // scores of values (e, 4 t + r) for head n, without their scaling
                f32x4 sc[4];
#pragma unroll
                for (int t = 0; t < 4; ++t) sc[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int i = 0; i < KW; ++i)
#pragma unroll
                    for (int t = 0; t < 4; ++t) {
                        const bf16x8 k = __builtin_bit_cast(bf16x8, mx_bf16(kw[t].v[i], kf[t]));
                        if constexpr (QF16) sc[t] = mfma_bf16(k, qop[1][i], sc[t]);
                        sc[t] = mfma_bf16(k, qop[0][i], sc[t]);
                    }
                // a pair's: lanes of columns below 8 take the first head's
                float p[NV], mx = kLow;
                auto pick = [&]() {
#pragma unroll
                    for (int i = 0; i < NV; ++i)
                        p[i] = HP == 1 || n < 8 ? sc[i >> 2][i & 3] : sc[(2 + (i >> 2)) & 3][i & 3];
                };
                pick();
                if (past || rows != ~uint64_t(0)) {
                    if (past) {
                        // Anew, with keys less 2^2, for scales of 253 and 254, and f16 queries' parts less 2^24, so that none
                        // of their sums passes f32 (from 192 on they can, with either sign, which is NaN).
#pragma unroll
                        for (int t = 0; t < 4; ++t) sc[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                        for (int i = 0; i < KW; ++i) {
                            bf16x8 q[QF16 ? 2 : 1];
#pragma unroll
                            for (int h = 0; h < (QF16 ? 2 : 1); ++h) {
                                Vec<uint32_t, 4> w = __builtin_bit_cast(Vec<uint32_t, 4>, qop[h][i]);
#pragma unroll
                                for (int e = 0; e < (QF16 ? 4 : 0); ++e) {
                                    __asm__ volatile("" : "+v"(w.v[e])); // (not ahead of the steps' loop, where they would take registers)
                                    w.v[e] = bf_pack(bf_lo(w.v[e]) * 0x1p-24f, bf_hi(w.v[e]) * 0x1p-24f);
                                }
                                q[h] = __builtin_bit_cast(bf16x8, w);
                            }
#pragma unroll
                            for (int t = 0; t < 4; ++t) {
                                const bf16x8 k =
                                    __builtin_bit_cast(bf16x8, mx_bf16_quarter(kw[t].v[i], __builtin_bit_cast(uint32_t, kf[t]) >> 23));
                                if constexpr (QF16) sc[t] = mfma_bf16(k, q[1], sc[t]);
                                sc[t] = mfma_bf16(k, q[0], sc[t]);
                            }
                        }
#pragma unroll
                        for (int t = 0; t < 4; ++t)
#pragma unroll
                            for (int r = 0; r < 4; ++r) sc[t][r] *= QF16 ? 0x1p26f : 0x1p2f;
                        pick();
                    }
                    const uint32_t bits = uint32_t(rows >> (16 * c)) & 0xffffu;
#pragma unroll
                    for (int i = 0; i < NV; ++i) p[i] = (bits >> (HP * i) & 1) != 0 ? p[i] : kLow;
                }
#pragma unroll
                for (int i = 0; i < NV; ++i) mx = __builtin_fmaxf(mx, p[i]);
                mx = rows4_max(mx);
                // no less than any score times its scaling, unrounded
                const float top = mx * scale2;
                mx = mx == kLow ? kLow : __builtin_fmaf(__builtin_fabsf(top), 0x1p-23f, top);
                // The reference moves when a score passes it by 8 (weights are then up to 2^8; to 1 where 2^127 is still to
                // come), which most steps do not see.
                const bool moves = mx > m + (raised ? 0.0f : 8.0f);
                const float mn = moves ? mx : m;
                // no score above -inf yet: a zero reference, so that -inf scores weigh 0
                // and only NaN ones reach the sum
                const float mref = mn == kLow ? 0.0f : mn;
#pragma unroll
                for (int i = 0; i < NV; ++i) p[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(p[i], scale2, -mref));
                if (any && __builtin_amdgcn_ballot_w64(moves) != 0) {
                    // some head's reference moved: rescale its sum and its O row
                    // (rows are heads 4c + r; their factors come from lanes 4c + r)
                    const float corr = __builtin_amdgcn_exp2f(m - mref); // from -inf: 0
                    l *= corr;
                    float cr[4];
#pragma unroll
                    for (int r = 0; r < 4; ++r) cr[r] = __shfl(corr, 4 * c + r, 64);
#pragma unroll
                    for (int e = 0; e < HP; ++e)
#pragma unroll
                        for (int t = 0; t < NT; ++t)
#pragma unroll
                            for (int r = 0; r < 4; ++r) o[e][t][r] *= cr[r];
                }
                m = mn;
                any = true;
#pragma unroll
                for (int i = 0; i < NV; i += 8)
                    l += ((p[i] + p[i + 1]) + (p[i + 2] + p[i + 3])) + ((p[i + 4] + p[i + 5]) + (p[i + 6] + p[i + 7]));
                if (raised) {
#pragma unroll
                    for (int i = 0; i < NV; ++i) p[i] *= 0x1p127f;
                    __asm__ volatile("" : "+v"(p[0])); // (a branch, not selections)
                }
                // parts of the weights, pairs of keys
                uint32_t w[NP][NV / 2];
#pragma unroll
                for (int i = 0; i < NV / 2; ++i) {
                    float p0 = p[2 * i], p1 = p[2 * i + 1];
#pragma unroll
                    for (int k = 0; k < NP; ++k) {
                        w[k][i] = k + 1 < NP ? high_halves(p0, p1) : bf_pack(p0, p1);
                        p0 -= bf_lo(w[k][i]);
                        p1 -= bf_hi(w[k][i]);
                    }
                }
                // V as B of P V: lane (dim n, c) has values (e, j) of dim 16 t + n. Of a pair, columns' weights meet both
                // heads' values: rows of O below 8 count of the first head's, the others of the second's.
#pragma unroll
                for (int b = 0; b < KB; ++b) {
                    Vec<uint32_t, 4> ws[NP];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        if (HP == 1 || e == 0) {
                            const Vec<uint32_t, 4> d =
                                *reinterpret_cast<const Vec<uint32_t, 4> *>(&vsc[wv][b][16 * c + 8 * (HP == 2 ? n >> 3 : e)]);
#pragma unroll
                            for (int k = 0; k < NP; ++k)
#pragma unroll
                                for (int i = 0; i < 4; ++i)
                                    ws[k].v[i] = pk_subsat_u16(w[k][HP == 1 ? 4 * e + i : i], d.v[i]);
                        }
                        bf16x8 vb[2];
#pragma unroll
                        for (int u = 0; u < 2; ++u) vb[u] = __builtin_bit_cast(bf16x8, mx_bf16(vx[2 * b + u].v[e], 1.0f));
#pragma unroll
                        for (int k = 0; k < NP; ++k)
#pragma unroll
                            for (int u = 0; u < 2; ++u)
                                o[e % HP][2 * b + u] = mfma_bf16(__builtin_bit_cast(bf16x8, ws[k]), vb[u], o[e % HP][2 * b + u]);
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

            // join the four waves, 64 dims at a time, in the places of the steps they took last
            const int mine = par ^ 1;
            l = rows4_sum(l);
            // keys, but none above -inf: the sum, 0 (or NaN), says so by 1. Beside a maximum it weighs 0; where no
            // part has one the parts' sums are added as they are, and 0 means that nothing was attended.
            if (c == 0) {
                wm[wv][n] = m;
                wl[wv][n] = any && m == kLow ? l + 1.0f : l;
            }
            if (lane == 0) place[wv] = uint32_t(2 * WB * mine);
            if (nan_v != 0) {
#pragma unroll
                for (int e = 0; e < HP; ++e)
#pragma unroll
                    for (int t = 0; t < NT; ++t)
                        if ((nan_v >> (8 * e + t / 2) & 1) != 0)
                            o[e][t] = f32x4{__builtin_nanf(""), __builtin_nanf(""), __builtin_nanf(""), __builtin_nanf("")};
            }
            const bool whole = cur.at == 0 && cur.end == cur.units;
            const int first = run.u1 - cur.behind - cur.end; // the request's first unit
            if (notes && leaves_cut(a.by_team, cur.at, cur.behind))
                a.cut[a.by_team ? team : cur.b] =
                    cur.at == 0 ? paged_cut(run.d, team, cur.b, first, cur.units) : PagedCut{};
            const int hh = threadIdx.x >> 4, d0 = (threadIdx.x & 15) * 4;
            float *so = reinterpret_cast<float *>(lds[wv][mine]);
#pragma unroll
            for (int part = 0; part < D / 64; ++part) {
                if (part > 0) __syncthreads(); // those before are read
#pragma unroll
                for (int t = 0; t < 4; ++t)
#pragma unroll
                    for (int r = 0; r < 4; ++r) // (rows 4 c + r, in turned order)
                        so[(4 * c + r) * 64 + ((16 * t + n) ^ (16 * c))] =
                            HP == 1 || c < 2 ? o[0][4 * part + t][r] : o[HP - 1][4 * part + t][r];
                __syncthreads();
                if (place_of(hh) < a.hw) {
                    const float top = __builtin_fmaxf(__builtin_fmaxf(wm[0][hh], wm[1][hh]), __builtin_fmaxf(wm[2][hh], wm[3][hh]));
                    float sum = 0.0f;
                    Vec<float, 4> acc{{0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        const float f = weight_of(wm[w][hh], top);
                        sum = __builtin_fmaf(f, wl[w][hh], sum);
                        const float *from = reinterpret_cast<const float *>(lds[w][0] + place[w]) + hh * 64 + (d0 ^ (16 * (hh >> 2)));
                        const Vec<float, 4> x = *reinterpret_cast<const Vec<float, 4> *>(from);
#pragma unroll
                        for (int i = 0; i < 4; ++i) acc.v[i] = __builtin_fmaf(f, x.v[i], acc.v[i]);
                    }
                    const int d = 64 * part + d0;
                    if (whole) {
                        const float inv = inverse(sum, top);
                        raw *dst = static_cast<raw *>(a.out) + cur.b * a.ldo + int64_t(head_of(hh)) * D + d;
#pragma unroll
                        for (int i = 0; i < 4; ++i) dst[i] = SO::enc32(acc.v[i] * inv);
                    } else {
                        const int vi = kv_of(hh) * nsub + sub;
                        const int64_t row = (int64_t(team_place(run.d, team, first)) * a.vh + vi) * a.hw + place_of(hh);
                        *reinterpret_cast<Vec<float, 4> *>(a.part + row * D + d) = acc;
                        if (d == 0) {
                            float *ml = a.part + 2 * int64_t(a.teams) * a.vh * a.hw * D + 2 * row;
                            ml[0] = top;
                            ml[1] = sum;
                        }
                    }
                }
            }
            __syncthreads(); // the places are free
            if (!go_on) break;
            full = false;
            if (next0.is) then = stage(mine);
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
        // A pair of heads at a time, where their queries fit 16 columns: half the work a score takes, and lines of 128
        // bytes where a head's row is 64 (40 / 8 heads, 64 ragged requests of up to 8000: 66 us, one at a time 76; 32 / 2
        // heads in sets of their own 46, one at a time 42, five of 100003).
        const bool pair = nkv % 2 == 0 && a.hw <= 8;
        paged_divide(c, a, D, pair ? 4 : 2, pair ? 32 : 64);
        auto go = [&](auto kern) {
            hipLaunchKernelGGL(kern, dim3(unsigned(a.teams * (pair ? a.vh / 2 : a.vh))), dim3(256), 0, c->stream, a);
            check_launch("k_attn_mxfp4");
        };
        auto sized = [&](auto s, auto so, auto kb) {
            using S = decltype(s);
            using SO = decltype(so);
            constexpr int KB = decltype(kb)::value;
            pair ? go(k_attn_mxfp4<S, SO, KB, 2>) : go(k_attn_mxfp4<S, SO, KB, 1>);
        };
        auto with = [&](auto s, auto so) {
            D == 128 ? sized(s, so, std::integral_constant<int, 4>{}) : sized(s, so, std::integral_constant<int, 2>{});
        };
        if (dt_out == F32)
            dt == BF16 ? with(SBf16{}, SF32{}) : with(SF16{}, SF32{});
        else
            dt == BF16 ? with(SBf16{}, SBf16{}) : with(SF16{}, SF16{});
        paged_join(c, a, D, dt_out);
    }
} // namespace mg
