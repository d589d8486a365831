// Decode attention over a paged KV cache for gfx950: one new token for each of
// many requests of different lengths.
//
// For request b of n = lens[b] keys (the new token's among them) and query head
// h (KV head g = h / groups), over keys j in [lo, n), lo = window > 0 ?
// max(0, n - window) : 0, key j in slot table[b, j / ps] ps + j % ps of the pool
// [slots, kv_heads, head_dim]:
//   s_j = (q_bh . k_j) * scaling,   out_bh = sum_j softmax(s)_j v_j.
// A request without keys gives zeros. A key whose page is outside the pool is
// left out, as a masked one. A score of -inf weighs nothing beside a larger one;
// a request that has only such scores gives NaN, as the quotient 0 / 0 is. Q8_0
// pages hold k_j and v_j as q * d, exactly.
//
// Division of the work (mg_paged_plan.hpp): the requests' keys form one line of
// units, cut into equal runs; a team of work-groups, one for every KV head (and
// for every 16 query heads of a larger group), walks a run, so the heads of one
// key, neighbours in memory, are read at about the same time. Lengths stay on
// the device: each work-group sums them itself. A request that lies in one run
// is finished there; the others leave partial results (maximum, sum,
// unnormalized output), which a second kernel joins in team order. (Joined by the
// last of a request's own work-groups instead, behind device-wide fences, a call
// took 19 to 52 us longer: a fence writes back an XCD's whole L2.)
//
// A work-group's four waves take steps of 32 keys of the run in turn, with no
// barrier until the request ends. Per step, as in the
// ring's decode kernel: whole rows are loaded in 16-byte pieces one step ahead,
// across the end of a request, and written to LDS;
// S^T = K Q^T and O += P V run on the matrix cores (16 query heads of the
// group, zero-padded, as columns), the weights entering as a high and a low
// 16-bit part (three of bf16 for f32 outputs), so each is within 2^-16 of p relative
// down to 2^-90 of the largest (a Q8_0 scale may take 2^-24 of bf16's range, a low
// part 2^-17). Online softmax in f32 on scores scaled by log2(e).
//   Pages: lane l holds the slot of key l of the step (its table entry was
// requested a step before); a load instruction covers 4 to 16 rows, which lie
// in one page where the page is that large, so one readlane gives their base;
// else, or where a key is masked, each row's slot comes by a shuffle. The mask
// is one bit a key, and rows of masked keys are never loaded: what they hold
// (NaN too) cannot reach the sums.
//   f16: two parts of 2^15 p are within 2^-19 of p down to p = 2^-21, where the low part
// ends at f16's smallest step; below it few bits would be left of a weight, which are all
// that counts behind a key that takes nearly everything and whose value is near zero. A
// step that holds a smaller weight takes its product in bf16, a value as the exact sum of
// two bf16 ones. (All steps in bf16: 32 windowed requests 22.3 us for 21.1, 250 short
// ones 75.2 for 70.6.) The factor multiplies the weight: beside a maximum past 2^26 an
// exponent would lose it.
//   Q8_0: quants become bf16, or f16 beside f16 queries, on their way from LDS,
// exactly (8 bits); a K block's scale multiplies its 32-dim part of the score, a
// V block's its weights before they are split, so no value is rounded to 16 bits.
//
// What bounds it: HBM where requests are long. 8 requests of 131072 keys (40/8
// heads of 128, bf16): 657 us, 6.5 TB/s of the 7.04 that a plain read reaches; 64
// ragged ones of up to 8000: 156, 6.2; 250 of up to 700: 67, 5.1 (waves wait 61 % of
// their cycles: a request's last step and the waves' meeting leave little in flight).
// About 6 us of each is launch, sums and the first step's chain of table entry, rows
// and products; the join adds 4 to 6. Q8_0: 5 of 100003 keys (32/2 heads) 56 us, 4.8
// TB/s; 550 vector instructions a step and wave keep the SIMDs 57 % busy and three
// waves each do not cover the rest of the step's chain.
#include "mg_attn_paged.hpp"

namespace mg
{
    typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
    MG_DEV f32x4 mfma_f16(f16x8 a, f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

    // the 16-bit storage types as matrix operands
    template <class S>
    struct Mm;
    template <>
    struct Mm<SBf16>
    {
        using x8 = bf16x8;
        static MG_DEV f32x4 mma(x8 a, x8 b, f32x4 c) { return mfma_bf16(a, b, c); }
        static MG_DEV uint32_t pack(float a, float b) // (bf_pack, without its copies of values that live on)
        {
            typedef float f2 __attribute__((ext_vector_type(2)));
            typedef __bf16 h2 __attribute__((ext_vector_type(2)));
            return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2{a, b}), h2));
        }
        static MG_DEV float low(uint32_t w) { return bf_lo(w); }
        static MG_DEV float high(uint32_t w) { return bf_hi(w); }
    };
    template <>
    struct Mm<SF16>
    {
        using x8 = f16x8;
        static MG_DEV f32x4 mma(x8 a, x8 b, f32x4 c) { return mfma_f16(a, b, c); }
        static MG_DEV uint32_t pack(float a, float b)
        {
            typedef _Float16 h2 __attribute__((ext_vector_type(2)));
            return __builtin_bit_cast(uint32_t, h2{_Float16(a), _Float16(b)});
        }
        static MG_DEV float low(uint32_t w) { return f16_f32(uint16_t(w)); }
        static MG_DEV float high(uint32_t w) { return f16_f32(uint16_t(w >> 16)); }
    };

    template <class X8>
    MG_DEV X8 ld_x8(const uint16_t *p)
    {
        return __builtin_bit_cast(X8, *reinterpret_cast<const Vec<uint32_t, 4> *>(p));
    }
    // two values as sums of NP 16-bit parts, each the rest's nearest, as the pair `at` of NP operands
    template <class M, int NP>
    MG_DEV void split(float p0, float p1, Vec<uint32_t, 4> (&w)[NP], int at)
    {
#pragma unroll
        for (int k = 0; k < NP; ++k) {
            w[k].v[at] = M::pack(p0, p1);
            if (k + 1 < NP) {
                p0 -= M::low(w[k].v[at]);
                p1 -= M::high(w[k].v[at]);
            }
        }
    }

    // eight quants as bf16, exactly
    MG_DEV bf16x8 q8_bf16(Vec<uint32_t, 2> x)
    {
        Vec<uint32_t, 4> w;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t u = x.v[i];
            w.v[2 * i] = Mm<SBf16>::pack(float(int8_t(u)), float(int8_t(u >> 8)));
            w.v[2 * i + 1] = Mm<SBf16>::pack(float(int8_t(u >> 16)), float(int32_t(u) >> 24));
        }
        return __builtin_bit_cast(bf16x8, w);
    }
    // eight quants as f16, exactly: 1024 + u in the mantissa of u = q + 128, less 1152
    MG_DEV f16x8 q8_f16(Vec<uint32_t, 2> x)
    {
        typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
        const f16x2 off = {_Float16(-1152.0f), _Float16(-1152.0f)};
        Vec<uint32_t, 4> w;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t u = x.v[i] ^ 0x80808080u;
            w.v[2 * i] = __builtin_bit_cast(
                uint32_t, __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) + off);
            w.v[2 * i + 1] = __builtin_bit_cast(
                uint32_t, __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) + off);
        }
        return __builtin_bit_cast(f16x8, w);
    }
    // ds_read_b64_tr_b8: within each 16-lane group, lane i receives byte i % 8 of the
    // 8-byte pieces addressed by lanes 2j + i / 8, j = 0..7
    MG_DEV Vec<uint32_t, 2> lds_read_tr8(const char *p)
    {
        typedef int i32x2 __attribute__((ext_vector_type(2)));
        typedef __attribute__((address_space(3))) i32x2 lds_i32x2;
        return __builtin_bit_cast(Vec<uint32_t, 2>, __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i32x2 *)(p)));
    }

    // (Q8_0 with 168 registers for three waves a SIMD: f16 queries with f32 outputs over head_dim 128 keep 12 bytes a
    // lane in scratch, and take 62.8 us where bf16's, without, take 62.3)
    template <class S, class SO, bool Q8, int KB> // KB = head_dim / 32
    __global__ __launch_bounds__(256, Q8 ? 3 : 2) void k_attn_paged(PagedArgs a)
    {
        constexpr int D = 32 * KB, NT = 2 * KB;   // NT output tiles of 16 dims
        constexpr int U = kPagedUnit;
        constexpr int EPL = Q8 ? 16 : 8;          // elements a lane loads at once
        constexpr int LPR = D / EPL;              // lanes a row
        constexpr int RPI = 64 / LPR;             // rows a load instruction covers
        constexpr int NLD = kPagedStep / RPI;     // load instructions a half
        // LDS row strides (bytes): conflict-free reads (V's quants: two-way)
        constexpr int SK = Q8 ? D + 16 : 2 * (D + 8), SV = Q8 ? D + 16 : 2 * (D + 16);
        constexpr int SO4 = D + 4;                // row stride of a wave's output in LDS (floats)
        constexpr int WB = 32 * (SK + SV);        // LDS bytes of a wave's K and V
        static_assert(16 * SO4 * 4 <= WB, "a wave's output takes the place of its K and V");
        using MS = Mm<S>; // the scores' product, at q's type
        using raw = typename SO::raw;
        // f16 values: the output's product in f16 where a step's weights allow, else in bf16
        constexpr bool F = S::dt == F16 && !Q8;
        constexpr float up = F ? 0x1p15f : 1.0f; // the weights' factor
        constexpr float kSmall = 0x1p-6f;        // a weight below 2^-21, with its factor
        // bf16 parts of a weight: two leave 2^-17 of it at most, 1.5e-6 of an output (2-norm), which f32
        // outputs would show (three: 3e-7) and 16-bit ones do not
        constexpr int NPB = SO::dt == F32 ? 3 : 2;
        constexpr float kLow = -__builtin_huge_valf();
        __shared__ __align__(16) char lds[4][WB];
        __shared__ __align__(16) float scl[Q8 ? 4 : 1][2][KB][32];
        __shared__ float wm[4][16], wl[4][16];
        const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
        // Work-groups go to the XCDs in turn. A Q8_0 key's scales of all heads share a 64-byte piece or two, so runs
        // of eight work-groups (a key's heads) are put on one XCD, whose L2 then fetches it once: 5 requests of
        // 100003 keys, 40/8 heads, 240 -> 209 us (head_dim 64: 190 -> 158); 32/2 heads 60.7 -> 61.5. 16-bit rows
        // are better off spread (40/8 heads of 64: 375 us, 388 in runs; of 128: 643, 700 all heads on one XCD).
        constexpr int G = Q8 ? 8 : 1;
        int wg = blockIdx.x;
        if (wg < int(gridDim.x) / (8 * G) * (8 * G)) {
            const int xcd = wg % 8, turn = wg / 8;
            wg = turn / G * (8 * G) + xcd * G + turn % G;
        }
        const int team = wg / a.vh, v = wg - team * a.vh;
        const Run run = find_run(a, team);
        const bool notes = a.teams > 1 && v == 0 && threadIdx.x == 0; // who writes the cuts down
        if (run.u0 >= run.u1) { // the whole work-group
            if (notes && a.by_team) a.cut[team] = PagedCut{};
            return;
        }
        const int nsub = a.hpg / a.hw, g = v / nsub;
        const int h0 = g * a.hpg + (v - g * nsub) * a.hw;
        const int n = lane & 15, c = lane >> 4;
        char *sk = lds[wv], *sv = sk + 32 * SK;
        const int pc = lane % LPR, pr = lane / LPR;
        const int64_t rowb = int64_t(a.nkv) * D * (Q8 ? 1 : 2); // bytes between slots
        const char *kg = static_cast<const char *>(a.kc) + int64_t(g) * D * (Q8 ? 1 : 2);
        const char *vg = static_cast<const char *>(a.vc) + int64_t(g) * D * (Q8 ? 1 : 2);
        const uint32_t lane_off = uint32_t(pr * rowb) + 16 * pc; // (checked on the host: below 2^32)
        const int cap = a.W << a.sh, psm = (1 << a.sh) - 1;

        // a part of a request in the run: units [at, end), attended keys [klo, khi), and the
        // units of the run behind it
        struct Part
        {
            int b, at, end, units, k0, klo, khi, behind;
        };
        auto part_of = [&](int b, int at, int left) {
            const PagedSpan sp = paged_span(__builtin_amdgcn_readfirstlane(a.lens[b]), cap, a.window);
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
        int akb = cur.k0 + kPagedStep * wv;
        bool more_ahead = true;
        auto advance = [&]() {
            akb += U;
            if (akb < ahead.khi) return;
            more_ahead = ahead.behind > 0;
            if (!more_ahead) return;
            ahead = part_of(ahead.b + 1, 0, ahead.behind);
            akb = ahead.k0 + kPagedStep * wv;
        };
        // the slot of key akb + lane % 32, or -1
        auto slot_of = [&]() {
            const int key = akb + (lane & 31);
            if (!more_ahead || key < ahead.klo || key >= ahead.khi) return -1;
            const int page = a.table[ahead.b * a.ldt + (key >> a.sh)];
            return page >= 0 && page < a.num_pages ? (page << a.sh) + (key & psm) : -1;
        };
        Vec<uint32_t, 4> stk[NLD], stv[NLD];
        Vec<uint16_t, KB> sts; // scales of key lane % 32: K's in the lower half of the wave, V's in the upper
        auto stage = [&](int slot, uint32_t seen) {
            if constexpr (Q8) {
                sts = Vec<uint16_t, KB>{};
                const uint16_t *sc = lane < 32 ? a.kd : a.vd;
                if (slot >= 0)
                    sts = *reinterpret_cast<const Vec<uint16_t, KB> *>(sc + (int64_t(slot) * a.nkv + g) * KB);
            }
            if (seen == 0xffffffffu && psm + 1 >= RPI) {
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
        uint32_t seen = uint32_t(__builtin_amdgcn_ballot_w64(slot >= 0)); // keys of the staged step, one bit each
        stage(slot, seen);
        advance();
        slot = slot_of();

        // B of S^T: lane (head n, c) holds q[n][32 i + 8c ..], zero for padding heads
        typename MS::x8 qop[KB];
        auto load_q = [&](int b) {
#pragma unroll
            for (int i = 0; i < KB; ++i) {
                const uint16_t *qp = static_cast<const uint16_t *>(a.q) + b * a.ldq + int64_t(h0 + n) * D + 32 * i + 8 * c;
                qop[i] = n < a.hw ? ld_x8<typename MS::x8>(qp) : typename MS::x8{};
            }
        };
        load_q(cur.b);
        for (;;) {
            f32x4 o[NT];
#pragma unroll
            for (int t = 0; t < NT; ++t) o[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            float m = kLow, l = 0.0f; // head n (replicated over c)
            bool any = false;         // the wave has seen a key that is not masked
            int kb = cur.k0 + kPagedStep * wv;
            bool more;
            do {
                kb += U;
                more = kb < cur.khi;
                const uint32_t now = seen;
                if (now != 0) {
#pragma unroll
                    for (int i = 0; i < NLD; ++i) {
                        const int key = pr + RPI * i;
                        *reinterpret_cast<Vec<uint32_t, 4> *>(sk + key * SK + 16 * pc) = stk[i];
                        *reinterpret_cast<Vec<uint32_t, 4> *>(sv + key * SV + 16 * pc) = stv[i];
                    }
                    if constexpr (Q8)
#pragma unroll
                        for (int i = 0; i < KB; ++i) scl[wv][lane >> 5][i][lane & 31] = f16_f32(sts.v[i]);
                    wave_lds_sync();
                }
                // the next step's rows and the table entries of the one behind it are requested now
                if (more_ahead) {
                    seen = uint32_t(__builtin_amdgcn_ballot_w64(slot >= 0));
                    stage(slot, seen);
                    advance();
                    slot = slot_of();
                }
                if (now == 0) continue;
                any = true;
                // K as A of S^T: lane (key n, c) holds dims 32 i + 8c.. of key 16 t + n
                Vec<uint32_t, EPL == 16 ? 2 : 4> kt[2][KB];
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int i = 0; i < KB; ++i)
                        kt[t][i] = *reinterpret_cast<const decltype(&kt[0][0])>(sk + (16 * t + n) * SK +
                                                                                (32 * i + 8 * c) * (16 / EPL));
                // scores of keys 16 t + 4c + r for head n
                float sc[2][4], mx = kLow;
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    f32x4 st = {0.0f, 0.0f, 0.0f, 0.0f};
                    if constexpr (Q8) {
#pragma unroll
                        for (int i = 0; i < KB; ++i) {
                            typename MS::x8 k;
                            if constexpr (S::dt == BF16)
                                k = q8_bf16(kt[t][i]);
                            else
                                k = q8_f16(kt[t][i]);
                            const f32x4 part = MS::mma(k, qop[i], f32x4{0.0f, 0.0f, 0.0f, 0.0f});
                            const Vec<float, 4> d =
                                *reinterpret_cast<const Vec<float, 4> *>(scl[wv][0][i] + 16 * t + 4 * c);
#pragma unroll
                            for (int r = 0; r < 4; ++r) st[r] = __builtin_fmaf(d.v[r], part[r], st[r]);
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < KB; ++i) st = MS::mma(__builtin_bit_cast(typename MS::x8, kt[t][i]), qop[i], st);
                    }
#pragma unroll
                    for (int r = 0; r < 4; ++r) sc[t][r] = st[r] * a.scale2;
                    if (now != 0xffffffffu) {
                        const uint32_t bits = now >> (16 * t + 4 * c);
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
                // weights: element 4t + r of lane (head n, c) is key 16 t + 4c + r
                float p[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) p[e] = up * __builtin_amdgcn_exp2f(sc[e >> 2][e & 3] - mref);
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
                l += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
                // V as B of P V: lane (dim n, c) needs keys 4c + r and 16 + 4c + r
                // of dim 16 s + n, through the transposing read
                const char *vr = Q8 ? sv + (16 * (n >> 3) + 4 * c + (n >> 1 & 3)) * SV + 8 * (n & 1)
                                    : sv + (4 * c + (n >> 2)) * SV + 8 * (n & 3);
                auto outputs = [&](auto in_f16) {
                    using M = Mm<std::conditional_t<decltype(in_f16)::value, SF16, SBf16>>;
                    using x8 = typename M::x8;
                    constexpr int NP = decltype(in_f16)::value ? 2 : NPB; // parts of a weight
                    constexpr int NV = F && !decltype(in_f16)::value ? 2 : 1; // parts of a value: f16's 11 bits are 8 and 3
                    Vec<uint32_t, 4> w[NP];
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        if constexpr (Q8) {
                            if (t % 2 == 0) {
                                const float *d = scl[wv][1][t / 2] + 4 * c;
                                const Vec<float, 4> d0 = *reinterpret_cast<const Vec<float, 4> *>(d);
                                const Vec<float, 4> d1 = *reinterpret_cast<const Vec<float, 4> *>(d + 16);
#pragma unroll
                                for (int e = 0; e < 4; e += 2) {
                                    split<M, NP>(p[e] * d0.v[e], p[e + 1] * d0.v[e + 1], w, e / 2);
                                    split<M, NP>(p[4 + e] * d1.v[e], p[5 + e] * d1.v[e + 1], w, 2 + e / 2);
                                }
                            }
                        } else if (t == 0) {
#pragma unroll
                            for (int e = 0; e < 8; e += 2) split<M, NP>(p[e], p[e + 1], w, e / 2);
                        }
                        Vec<uint32_t, 4> vb[NV];
                        if constexpr (Q8) {
                            vb[0] = __builtin_bit_cast(Vec<uint32_t, 4>, q8_bf16(lds_read_tr8(vr + 16 * t)));
                        } else {
                            const bf16x4 v0 = lds_read_tr(reinterpret_cast<const uint16_t *>(vr + 32 * t));
                            const bf16x4 v1 = lds_read_tr(reinterpret_cast<const uint16_t *>(vr + 16 * SV + 32 * t));
                            vb[0] = __builtin_bit_cast(Vec<uint32_t, 4>,
                                                       bf16x8{v0[0], v0[1], v0[2], v0[3], v1[0], v1[1], v1[2], v1[3]});
                            if constexpr (NV == 2) {
                                const Vec<uint32_t, 4> x = vb[0];
#pragma unroll
                                for (int i = 0; i < 4; ++i)
                                    split<M, NV>(f16_f32(uint16_t(x.v[i])), f16_f32(uint16_t(x.v[i] >> 16)), vb, i);
                            }
                        }
                        // (a weight's third part times a value's second, 2^-26 of their product, is left out)
#pragma unroll
                        for (int k = 0; k < NP; ++k)
#pragma unroll
                            for (int i = 0; i < NV && k + i < 3; ++i)
                                o[t] = M::mma(__builtin_bit_cast(x8, w[k]), __builtin_bit_cast(x8, vb[i]), o[t]);
                    }
                };
                if constexpr (F) {
                    uint32_t least = 0xffffffffu; // of the weights' bits, less 1: a zero weight (a masked key's) is none
#pragma unroll
                    for (int e = 0; e < 8; ++e) least = min(least, __builtin_bit_cast(uint32_t, p[e]) - 1u);
                    if (__builtin_amdgcn_ballot_w64(least < __builtin_bit_cast(uint32_t, kSmall) - 1u) == 0)
                        outputs(std::true_type{});
                    else
                        outputs(std::false_type{});
                } else {
                    outputs(std::false_type{});
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

    // Joins the partial results of one request and work-group of heads: top = max m_s,
    // out = sum_s 2^(m_s - top) acc_s / sum_s 2^(m_s - top) l_s. A work-group takes 4 E of the
    // outputs, thread (e, sg) four of them over every SG-th part from sg; SG threads' shares
    // are added in LDS, in the order of sg.
    template <class SO, int E>
    __global__ __launch_bounds__(256) void k_attn_paged_join(PagedArgs a, int D)
    {
        constexpr int SG = 256 / E;
        __shared__ float tops[SG][E], sums[SG][E];
        __shared__ Vec<float, 4> accs[SG][E];
        const PagedCut cut = a.cut[blockIdx.x];
        const int nt = cut.parts;
        if (nt == 0) return; // finished in its team
        const int v = blockIdx.y, e = threadIdx.x % E, sg = threadIdx.x / E;
        const int i0 = (int(blockIdx.z) * E + e) * 4; // the thread's outputs among [hw, D]
        const bool live = i0 < a.hw * D;
        const int hh = live ? i0 / D : 0; // (a work-group's outputs may be of several heads)
        const float *ml = a.part + 2 * int64_t(a.teams) * a.vh * a.hw * D;
        auto row = [&](int s) { return (int64_t(cut_place(cut, s)) * a.vh + v) * a.hw; };
        // P parts' maxima, sums and outputs are in flight at once (5 requests of 77 parts: 6.4 us with four, 4.8 with
        // eight); a thread with more takes them in batches, joined as scores are
        constexpr int P = E <= 16 ? 8 : 4;
        constexpr float kLow = -__builtin_huge_valf();
        float pm[P], pl[P], top = kLow, sum = 0.0f;
        Vec<float, 4> px[P], acc{{0.0f, 0.0f, 0.0f, 0.0f}};
        auto load = [&](int s0) {
#pragma unroll
            for (int k = 0; k < P; ++k) {
                const int s = s0 + k * SG;
                pm[k] = kLow;
                pl[k] = 0.0f;
                px[k] = Vec<float, 4>{{0.0f, 0.0f, 0.0f, 0.0f}};
                if (s < nt && live) {
                    const int64_t r = row(s);
                    pm[k] = ml[2 * (r + hh)];
                    pl[k] = ml[2 * (r + hh) + 1];
                    px[k] = *reinterpret_cast<const Vec<float, 4> *>(a.part + r * D + i0);
                }
            }
#pragma unroll
            for (int k = 0; k < P; ++k) top = __builtin_fmaxf(top, pm[k]);
        };
        auto add = [&](float ref) {
#pragma unroll
            for (int k = 0; k < P; ++k) {
                const float f = weight_of(pm[k], ref);
                sum = __builtin_fmaf(f, pl[k], sum);
#pragma unroll
                for (int i = 0; i < 4; ++i) acc.v[i] = __builtin_fmaf(f, px[k].v[i], acc.v[i]);
            }
        };
        auto scale = [&](float f) {
            sum *= f;
#pragma unroll
            for (int i = 0; i < 4; ++i) acc.v[i] *= f;
        };
        const bool few = nt <= P * SG; // one batch: weighed by the maximum of all threads at once
        load(sg);
        if (!few) {
            add(top);
            for (int s0 = sg + P * SG; s0 < nt; s0 += P * SG) {
                const float was = top;
                load(s0);
                scale(weight_of(was, top));
                add(top);
            }
        }
        tops[sg][e] = top;
        __syncthreads();
        float all = top;
#pragma unroll
        for (int s = 0; s < SG; ++s) all = __builtin_fmaxf(all, tops[s][e]);
        if (few)
            add(all);
        else
            scale(weight_of(top, all));
        sums[sg][e] = sum;
        accs[sg][e] = acc;
        __syncthreads();
        if (sg != 0 || !live) return;
        sum = sums[0][e];
        acc = accs[0][e];
#pragma unroll
        for (int s = 1; s < SG; ++s) {
            sum += sums[s][e];
#pragma unroll
            for (int i = 0; i < 4; ++i) acc.v[i] += accs[s][e].v[i];
        }
        const float inv = inverse(sum, all);
        const int nsub = a.hpg / a.hw, g = v / nsub;
        const int h0 = g * a.hpg + (v - g * nsub) * a.hw;
        typename SO::raw *dst = static_cast<typename SO::raw *>(a.out) + cut.request * a.ldo + int64_t(h0) * D + i0;
#pragma unroll
        for (int i = 0; i < 4; ++i) dst[i] = SO::enc32(acc.v[i] * inv);
    }

    PagedArgs paged_args(const void *q, int64_t ldq, const void *kc, const void *vc, const void *kd, const void *vd,
                         const int32_t *table, int64_t ldt, int64_t max_pages, const int32_t *lens, int64_t seqs, int64_t nq,
                         int64_t nkv, int64_t D, int64_t page_size, int64_t num_pages, int64_t window, double scaling,
                         void *out, int64_t ldo, int dt, int dt_out)
    {
        const int sh = page_shift(page_size, "attn_decode_paged");
        need(seqs >= 0 && nq > 0 && nkv > 0 && nq % nkv == 0,
             "attn_decode_paged: q_heads must be a multiple of kv_heads");
        need(nq <= 65535, "attn_decode_paged: too many heads"); // (16 rows of a load stay below 2^32 bytes)
        need(D == 64 || D == 128, "attn_decode_paged: head_dim must be 64 or 128");
        need(dt == BF16 || dt == F16, "attn_decode_paged: dtype must be bf16 or f16");
        need(dt_out == dt || dt_out == F32, "attn_decode_paged: dtype_out must be f32 or q's dtype");
        need(max_pages > 0 && num_pages > 0, "attn_decode_paged: bad table or pool size");
        need(num_pages <= ((int64_t(1) << 31) - 1) >> sh, "attn_decode_paged: a pool must have fewer than 2^31 slots");
        need(max_pages <= (int64_t(1) << 30) >> sh, "attn_decode_paged: a table row must stand for at most 2^30 tokens");
        need((kd == nullptr) == (vd == nullptr), "attn_decode_paged: give both k_scale and v_scale, or neither");
        if (ldq == 0) ldq = nq * D;
        if (ldo == 0) ldo = nq * D;
        if (ldt == 0) ldt = max_pages;
        need(ldq >= nq * D && ldo >= nq * D && ldt >= max_pages, "attn_decode_paged: row stride smaller than a row");
        need(aligned16(q) && aligned16(kc) && aligned16(vc) && ldq % 8 == 0,
             "attn_decode_paged: q rows and caches must be 16-byte aligned");
        need(reinterpret_cast<uintptr_t>(kd) % 8 == 0 && reinterpret_cast<uintptr_t>(vd) % 8 == 0,
             "attn_decode_paged: scales must be 8-byte aligned");
        need(seqs <= 65535, "attn_decode_paged: at most 65535 requests");
        PagedArgs a{};
        if (seqs == 0) return a;
        need(q && kc && vc && table && lens && out, "attn_decode_paged: NULL tensor");
        // a wave serves up to 16 query heads (the matrix cores' 16 columns); larger
        // groups split over work-groups of the largest divisor <= 16
        const int64_t hpg = nq / nkv;
        int64_t hw = hpg;
        while (hw > 16 || hpg % hw != 0) --hw;
        a.q = q, a.kc = kc, a.vc = vc, a.table = table, a.lens = lens, a.out = out;
        a.ldq = ldq, a.ldt = ldt, a.ldo = ldo, a.window = window;
        a.R = int(seqs), a.nkv = int(nkv), a.W = int(max_pages), a.sh = sh, a.num_pages = int(num_pages);
        a.hpg = int(hpg), a.hw = int(hw), a.vh = int(nkv * (hpg / hw));
        a.scale2 = float(double(float(scaling)) * 1.4426950408889634);
        return a;
    }

    void paged_divide(mg_ctx *c, PagedArgs &a, int64_t D, int per_cu, int step)
    {
        const int64_t most = a.R * paged_most_units(int64_t(a.W) << a.sh, a.window, step);
        need(most < (int64_t(1) << 31), "attn_decode_paged: the table must stand for fewer than 2^38 keys");
        // not more teams than there can be units, nor than the workspace has room for
        int64_t teams = per_cu * int64_t(c->num_cus) / a.vh;
        teams = teams < most ? teams : most;
        // (the cuts, then the partial results' outputs, then their maxima and sums)
        const int64_t tbytes = 2 * int64_t(a.vh) * a.hw * (D + 2) * int64_t(sizeof(float)) + int64_t(sizeof(PagedCut));
        teams = teams < c->work_bytes / tbytes ? teams : c->work_bytes / tbytes;
        teams = teams > 1 ? teams : 1;
        a.by_team = cuts_by_team(teams, a.R); // else there is room for a cut of each request among the teams'
        a.cut = static_cast<PagedCut *>(c->work);
        a.part = reinterpret_cast<float *>(a.cut + teams);
        a.teams = int(teams);
    }

    void paged_join(mg_ctx *c, const PagedArgs &a, int64_t D, int dt_out)
    {
        if (a.teams == 1) return; // nothing is cut
        const int64_t who = cuts_kept(a.teams, a.R);
        auto join = [&](auto kern, int e) {
            const dim3 grid{unsigned(who), unsigned(a.vh), unsigned((a.hw * D + 4 * e - 1) / (4 * e))};
            hipLaunchKernelGGL(kern, grid, dim3(256), 0, c->stream, a, int(D));
            check_launch("k_attn_paged_join");
        };
        // few requests over many teams: threads over the teams; else over the outputs (one request of 131072 keys,
        // 32/2 heads, 256 teams, 4 / 16: 31.3 us, 32.7; 8/1 heads, 512 teams: 21.7, 27.8; two of 60000, 32/2 heads, 128
        // teams each: 31.4, 29.9)
        const int64_t parts = a.teams / who;
        auto to = [&](auto so) {
            using SO = decltype(so);
            if (parts >= 256)
                join(k_attn_paged_join<SO, 4>, 4);
            else
                parts >= 8 ? join(k_attn_paged_join<SO, 16>, 16) : join(k_attn_paged_join<SO, 64>, 64);
        };
        dt_out == F32 ? to(SF32{}) : dt_out == BF16 ? to(SBf16{}) : to(SF16{});
    }

    void launch_attn_decode_paged(mg_ctx *c, const void *q, int64_t ldq, const void *kc, const void *vc,
                                  const uint16_t *kd, const uint16_t *vd, const int32_t *table, int64_t ldt,
                                  int64_t max_pages, const int32_t *lens, int64_t seqs, int64_t nq, int64_t nkv,
                                  int64_t D, int64_t page_size, int64_t num_pages, int64_t window, double scaling,
                                  void *out, int64_t ldo, int dt, int dt_out)
    {
        PagedArgs a = paged_args(q, ldq, kc, vc, kd, vd, table, ldt, max_pages, lens, seqs, nq, nkv, D, page_size,
                                 num_pages, window, scaling, out, ldo, dt, dt_out);
        if (a.R == 0) return;
        a.kd = kd, a.vd = vd;
        // Teams for 2 to 4 work-groups a CU: as many as its registers take, but three, not four, for 16-bit rows of
        // 64 (10 requests of 100003 keys 351 us, four 372, two 358; Q8_0: four 69, three 72, two 81 at 64 ragged
        // requests of up to 8000).
        paged_divide(c, a, D, kd ? (D == 128 ? 3 : 4) : (D == 128 ? 2 : 3), kPagedStep);
        auto go = [&](auto kern) {
            hipLaunchKernelGGL(kern, dim3(unsigned(a.teams * a.vh)), dim3(256), 0, c->stream, a);
            check_launch("k_attn_paged");
        };
        auto sized = [&](auto s, auto so) {
            using S = decltype(s);
            using SO = decltype(so);
            if (kd)
                D == 128 ? go(k_attn_paged<S, SO, true, 4>) : go(k_attn_paged<S, SO, true, 2>);
            else
                D == 128 ? go(k_attn_paged<S, SO, false, 4>) : go(k_attn_paged<S, SO, false, 2>);
        };
        if (dt_out == F32)
            dt == BF16 ? sized(SBf16{}, SF32{}) : sized(SF16{}, SF32{});
        else
            dt == BF16 ? sized(SBf16{}, SBf16{}) : sized(SF16{}, SF16{});
        paged_join(c, a, D, dt_out);
    }
} // namespace mg
