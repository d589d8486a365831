// Products of an MXFP4 weight with few tokens, for gfx950: y[t, o] = sum_i W[o, i]
// x[t, i], x in 16 bits or in MXFP4 itself.
//
// Weights go straight into LDS, steps ahead: of 512 elements, a wave by itself in a
// ring of two (up to four tokens of 16 bits, and MXFP4's, 16 a pass over the weight),
// or of 256, shared by eight waves, in a ring of three (five to 64 tokens of 16 bits).
// Products are 16 x 16 (weight rows x tokens) of 128 elements: lane (n, c) holds block c
// of weight row n, 16 bytes, and of token n.
// MXFP4 activations: one scaled product over 128. 16-bit ones: four over 32, the
// codes become bf16 with their scale, exactly up to 2^125 (past that mx_far_sums takes
// them); beside f16 activations f16 where that is exact too (scales of 2^-23 to 2^13,
// blocks of zeros, NaN), else the activations are split into two bf16 parts.
#include "mg_device.hpp"
#include "mg_internal.hpp"
#include "mg_mxfp4.hpp"

namespace mg
{
    struct MxGemvArgs
    {
        const uint8_t *w, *ws, *x, *xs; // x: 16-bit rows, or codes with scales xs
        void *y;
        int64_t ldx, ldy, rows, T;
        int64_t ysplit;    // elements of y between splits' results
        int nblk, steps;   // in / 32; the kernel's steps of a row (set by its launcher), of 512 or of 256 elements
        int splits;        // steps a split takes
    };

    // a token's operand of a step: 32 elements of 16 bits, or a block
    template <class A>
    struct MxTok
    {
        Vec<uint32_t, 4> v[A::dt == kMxFp4 ? 1 : 4];
        uint32_t s;
    };

    // A step's products. acc[..][k]: sums of every NA-th product, which keeps chains short.
    template <class A, int RT, int TT, int NA>
    MG_DEV void mx_step(const Vec<uint32_t, 4> (&w)[RT], const uint32_t (&ws)[RT], const MxTok<A> (&x)[TT],
                        f32x4 (&acc)[RT][TT][NA])
    {
        if constexpr (A::dt == kMxFp4) {
#pragma unroll
            for (int t = 0; t < RT; ++t)
#pragma unroll
                for (int u = 0; u < TT; ++u) acc[t][u][0] = mfma_mxfp4(w[t], ws[t], x[u].v[0], x[u].s, acc[t][u][0]);
        } else {
            bool wide = false; // f16: some block needs bf16's range
            if constexpr (A::dt == F16) {
                bool far = false;
#pragma unroll
                for (int t = 0; t < RT; ++t)
                    far |= ws[t] - 104u > 36u && ws[t] != 255u && ((w[t].v[0] | w[t].v[1] | w[t].v[2] | w[t].v[3]) & 0x77777777u) != 0;
                wide = __builtin_amdgcn_ballot_w64(far) != 0;
            }
            if (A::dt == F16 && !wide) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int t = 0; t < RT; ++t) {
                        const mxf16x8 wh = __builtin_bit_cast(mxf16x8, mx_f16(w[t].v[i], mx_scale(ws[t])));
#pragma unroll
                        for (int u = 0; u < TT; ++u)
                            acc[t][u][i % NA] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wh, __builtin_bit_cast(mxf16x8, x[u].v[i]),
                                                                                       acc[t][u][i % NA], 0, 0, 0);
                    }
                return;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int t = 0; t < RT; ++t) {
                    const bf16x8 wb = __builtin_bit_cast(bf16x8, mx_bf16(w[t].v[i], mx_scale(ws[t])));
#pragma unroll
                    for (int u = 0; u < TT; ++u) {
                        if constexpr (A::dt == F16) {
                            Vec<uint32_t, 4> hi, lo;
#pragma unroll
                            for (int k = 0; k < 4; ++k) mx_halves(x[u].v[i].v[k], hi.v[k], lo.v[k]);
                            acc[t][u][i % NA] = mfma_bf16(wb, __builtin_bit_cast(bf16x8, lo), acc[t][u][i % NA]);
                            acc[t][u][i % NA] = mfma_bf16(wb, __builtin_bit_cast(bf16x8, hi), acc[t][u][i % NA]);
                        } else {
                            acc[t][u][i % NA] = mfma_bf16(wb, __builtin_bit_cast(bf16x8, x[u].v[i]), acc[t][u][i % NA]);
                        }
                    }
                }
        }
    }
    template <int NA>
    MG_DEV f32x4 mx_total(const f32x4 (&a)[NA])
    {
        if constexpr (NA == 4)
            return (a[0] + a[1]) + (a[2] + a[3]);
        else if constexpr (NA == 2)
            return a[0] + a[1];
        else
            return a[0];
    }

    // Where weights pass bf16's largest value (scales of 253 and 254), or products with an f16 value's two bf16 parts may
    // each pass f32's, so that what the two are together is lost (from 192 on: 6 2^63 by 2^16 is far from that for any
    // number of them), the sums above are not these products'. A wave keeps the least of its scales less the first such
    // (in the steps' loop a branch of its own took 20 % at one token), and then takes its sums anew.
    template <class A>
    MG_DEV uint32_t mx_past(uint32_t s)
    {
        return s - (A::dt == F16 ? 192u : 253u);
    }
    template <class A>
    MG_DEV bool mx_any_past(uint32_t least) // (255 is NaN, whatever it meets)
    {
        return A::dt != kMxFp4 && __builtin_amdgcn_ballot_w64(least < (A::dt == F16 ? 63u : 2u)) != 0;
    }
    // The sums of RT tiles of 16 rows from row0 on with TT of 16 tokens from tok0 on, over the 128 elements of steps
    // step(0), step(1) ..: weights less 2^2, f16 parts less 2^24, all exactly, the sums so far less both while a step is added
    // (below 2^-123 they lose bits then). Straight from memory, for rows that are hardly ever there.
    template <class A, int RT, int TT, class F>
    MG_DEV void mx_far_sums(const MxGemvArgs &a, int64_t row0, int64_t tok0, int count, F step, f32x4 (&acc)[RT][TT])
    {
        constexpr float by = A::dt == F16 ? 0x1p-26f : 0x1p-2f;
        const int lane = threadIdx.x & 63, n = lane & 15, c = lane >> 4;
        auto times = [&](float f) {
#pragma unroll
            for (int t = 0; t < RT; ++t)
#pragma unroll
                for (int u = 0; u < TT; ++u)
#pragma unroll
                    for (int r = 0; r < 4; ++r) acc[t][u][r] *= f;
        };
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
            for (int u = 0; u < TT; ++u) acc[t][u] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        for (int k = 0; k < count; ++k) {
            const int64_t blk = 4 * int64_t(step(k)) + c;
            const bool in = blk < a.nblk;
            const Vec<uint32_t, 4> zero{{0u, 0u, 0u, 0u}};
            Vec<uint32_t, 4> w[RT];
            uint32_t ws[RT];
#pragma unroll
            for (int t = 0; t < RT; ++t) {
                const int64_t r = row0 + 16 * t + n, row = r < a.rows ? r : a.rows - 1;
                w[t] = zero;
                ws[t] = 127u;
                if (in) {
                    w[t] = *reinterpret_cast<const Vec<uint32_t, 4> *>(a.w + 16 * (row * a.nblk + blk));
                    ws[t] = a.ws[row * a.nblk + blk];
                }
            }
            times(by);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                bf16x8 wb[RT];
#pragma unroll
                for (int t = 0; t < RT; ++t) wb[t] = __builtin_bit_cast(bf16x8, mx_bf16_quarter(w[t].v[i], ws[t]));
#pragma unroll
                for (int u = 0; u < TT; ++u) {
                    const int64_t t0 = tok0 + 16 * u + n, tok = t0 < a.T ? t0 : a.T - 1;
                    Vec<uint32_t, 4> hi = zero, lo = zero;
                    if (in) hi = *reinterpret_cast<const Vec<uint32_t, 4> *>(a.x + 2 * (tok * a.ldx + 32 * blk + 8 * i));
                    if constexpr (A::dt == F16) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) mx_halves(hi.v[e], hi.v[e], lo.v[e], 0x1p-24f);
                    }
#pragma unroll
                    for (int t = 0; t < RT; ++t) {
                        if constexpr (A::dt == F16) acc[t][u] = mfma_bf16(wb[t], __builtin_bit_cast(bf16x8, lo), acc[t][u]);
                        acc[t][u] = mfma_bf16(wb[t], __builtin_bit_cast(bf16x8, hi), acc[t][u]);
                    }
                }
            }
            times(1.0f / by);
        }
    }

    template <int N>
    MG_DEV void mx_wait() // all but the last N loads into LDS have landed
    {
        __asm__ volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
    }

    // ------------------------------------------- a wave by itself: 16-bit rows of up to four tokens, MXFP4 of up to 16
    // A wave takes 16 weight rows in steps of 512 elements, 256 bytes a row an instruction (64 bytes of 16 rows: 19.3 us
    // for 16.4 at [25600, 5120], one token), with its own ring of two of them in LDS and no barrier. Four waves, a
    // work-group, share a row's steps in turn and add their sums at the end. That weight, 70 MB, from HBM, as in the run of a
    // model (17 of them in turn): one token 17.0 us, 4.1 TB/s, four 19.6 (f16: 20.4 and 21.8); three in turn stay in the
    // last cache, 14.0. Not bound by HBM, whose 9.9 it is far from: a ring starts empty for every 16 rows, and ten steps
    // are shared as three, three, two and two.
    template <class A, class SO, int XR, bool AL> // XR: token rows; AL: scales in whole 16s, aligned
    __global__ __launch_bounds__(256) void k_mxfp4_gemv_wave(MxGemvArgs a)
    {
        constexpr bool MX = A::dt == kMxFp4;
        constexpr int KS = 4, NB = 2, NA = MX ? 1 : 4;
        constexpr int SS = AL ? 256 : 1024;               // scales of a step: 16 bytes a row, or each a word
        constexpr int XB = MX ? 4096 + SS : 1024 * XR;    // tokens
        constexpr int SB = 4096 + SS + XB;
        constexpr int LS = AL ? 1 : 4, L = 4 + LS + (MX ? 4 + LS : XR);
        __shared__ __align__(16) char lds[KS][NB * SB];
        const int wv = __builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6)), lane = threadIdx.x & 63;
        const int n = lane & 15, c = lane >> 4;
        const int64_t r0 = 16 * int64_t(blockIdx.x), t0 = int64_t(blockIdx.y) * XR;
        const int nblk = a.nblk, steps = a.steps;
        const uint32_t base = lds_address(lds[wv]);
        // Load j brings rows 4 j .. + 3, lane l piece (l % 16) ^ (row % 16) of row l / 16: reads of 16 rows' same piece hit
        // all banks. A block past the rows' ends is taken from their first, and counts as zeros (below).
        auto rows16 = [&](const uint8_t *p, int64_t last, int m, uint32_t to) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int lr = 4 * j + c;
                const int64_t row = lr < last ? lr : last;
                const int blk = 16 * m + (n ^ lr);
                lds_load(p, uint32_t(row) * (16u * uint32_t(nblk)) + 16u * uint32_t(blk < nblk ? blk : 0), to + 1024 * j);
            }
        };
        auto scales16 = [&](const uint8_t *p, int64_t last, int m, uint32_t to) {
            const int64_t row = n < last ? n : last;
            if constexpr (AL) {
                if (lane < 16) lds_load(p, uint32_t(row) * uint32_t(nblk) + 16u * uint32_t(m), to);
            } else {
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    const int blk = 16 * m + 4 * s + c;
                    lds_load<1>(p, uint32_t(row) * uint32_t(nblk) + uint32_t(blk < nblk ? blk : 0), to + 256 * s);
                }
            }
        };
        const uint8_t *wb = a.w + r0 * (16 * int64_t(nblk)), *wsb = a.ws + r0 * nblk;
        const uint8_t *xb = MX ? a.x + t0 * (16 * int64_t(nblk)) : a.x, *xsb = MX ? a.xs + t0 * nblk : nullptr;
        auto load = [&](int m, int buf) {
            const uint32_t to = base + buf * SB;
            rows16(wb, a.rows - 1 - r0, m, to);
            scales16(wsb, a.rows - 1 - r0, m, to + 4096);
            if constexpr (MX) {
                rows16(xb, a.T - 1 - t0, m, to + 4096 + SS);
                scales16(xsb, a.T - 1 - t0, m, to + 8192 + SS);
            } else {
#pragma unroll
                for (int r = 0; r < XR; ++r) { // token r: lane l eight elements, piece l ^ r
                    const int64_t tok = t0 + r < a.T ? t0 + r : a.T - 1;
                    const int e = 512 * m + 8 * (lane ^ r);
                    lds_load(xb + 2 * tok * a.ldx, 2u * uint32_t(e < 32 * nblk ? e : 0), to + 4096 + SS + 1024 * r);
                }
            }
        };
        f32x4 acc[1][1][NA];
#pragma unroll
        for (int k = 0; k < NA; ++k) acc[0][0][k] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        uint32_t past = ~0u; // the least scale's place from where bf16 and f32 end
        const int mine = steps > wv ? (steps - wv + KS - 1) / KS : 0; // steps wv, wv + KS ..
#pragma unroll
        for (int p = 0; p < NB; ++p)
            if (p < mine) load(wv + p * KS, p);
        int buf = 0;
        for (int k = 0; k < mine; ++k) {
            const int m = wv + k * KS;
            if (k + NB <= mine)
                mx_wait<(NB - 1) * L>();
            else
                mx_wait<0>();
            const char *b = lds[wv] + buf * SB;
            Vec<uint32_t, 4> w[4][1];
            uint32_t ws[4][1];
            MxTok<A> x[4][1];
            auto block = [&](const char *p, int s) { return *reinterpret_cast<const Vec<uint32_t, 4> *>(p + 256 * n + 16 * ((4 * s + c) ^ n)); };
            auto scale = [&](const char *p, uint32_t (&out)[4]) {
                if constexpr (AL) {
                    const Vec<uint32_t, 4> v = *reinterpret_cast<const Vec<uint32_t, 4> *>(p + 16 * n);
#pragma unroll
                    for (int s = 0; s < 4; ++s) out[s] = v.v[s] >> (8 * c) & 0xffu;
                } else {
#pragma unroll
                    for (int s = 0; s < 4; ++s) out[s] = *reinterpret_cast<const uint32_t *>(p + 256 * s + 4 * lane);
                }
            };
            uint32_t sw[4], sx[4];
            scale(b + 4096, sw);
            if constexpr (MX) scale(b + 8192 + SS, sx);
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                w[s][0] = block(b, s);
                ws[s][0] = sw[s];
                const char *xl = b + 4096 + SS;
                if constexpr (MX) {
                    x[s][0].v[0] = block(xl, s);
                    x[s][0].s = sx[s];
                } else {
                    const int r = n < XR ? n : XR - 1; // (tokens past the last repeat it, and are not stored)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        x[s][0].v[i] = *reinterpret_cast<const Vec<uint32_t, 4> *>(xl + 1024 * r + 16 * ((16 * s + 4 * c + i) ^ r));
                }
            }
            __asm__ volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); // the buffer is read
            if (k + NB < mine) load(m + NB * KS, buf);
            buf = buf + 1 < NB ? buf + 1 : 0;
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                if (16 * m + 16 > nblk && 16 * m + 4 * s + c >= nblk) {
                    w[s][0] = Vec<uint32_t, 4>{{0u, 0u, 0u, 0u}};
                    ws[s][0] = x[s][0].s = 127u;
#pragma unroll
                    for (int i = 0; i < (MX ? 1 : 4); ++i) x[s][0].v[i] = Vec<uint32_t, 4>{{0u, 0u, 0u, 0u}};
                }
                if constexpr (!MX) past = min(past, mx_past<A>(ws[s][0]));
                mx_step<A, 1, 1, NA>(w[s], ws[s], x[s], acc);
            }
        }
        // lane (token n, c) holds rows 4 c .. 4 c + 3
        typename SO::raw *y = static_cast<typename SO::raw *>(a.y);
        f32x4 sum = mx_total(acc[0][0]);
        if constexpr (!MX) {
            if (mx_any_past<A>(past)) {
                f32x4 far[1][1];
                mx_far_sums<A, 1, 1>(a, r0, t0, 4 * mine, [&](int k) { return 4 * (wv + KS * (k / 4)) + k % 4; }, far);
                sum = far[0][0];
            }
        }
        *reinterpret_cast<f32x4 *>(lds[wv] + 16 * lane) = sum;
        __syncthreads();
        if (wv != 0) return;
#pragma unroll
        for (int k = 1; k < KS; ++k) sum += *reinterpret_cast<const f32x4 *>(lds[k] + 16 * lane);
        const int64_t tok = t0 + n, o = r0 + 4 * c;
        if (n >= XR || tok >= a.T) return;
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (o + r < a.rows) y[tok * a.ldy + o + r] = SO::enc32(sum[r]);
    }

    // ------------------------------------------- a work-group for more tokens of 16 bits: they are shared by its waves
    // 128 rows over 16 TT tokens in a ring of three steps of 256 elements, loaded by all of eight waves; waves 2 g and
    // 2 g + 1 take 32 rows, half of each step's elements each, and add at the end: a wave's reads of tokens, what bounds this
    // kernel beside its waits at the barrier, then serve two tiles of rows ([25600, 5120] by 64, bf16: 40 us, eight waves of
    // 16 rows and whole steps 48; by 8: 22.9 / 24.1, where the weight alone takes 10). Weights from HBM, 17 in turn: 40.7 by 64, 23.2 by 8. Reading a step's operands beneath
    // the products of the one before gains nothing (by 64: 49), nor do rings of two steps (by 5: 29.6) or four (22.7).
    template <class A, class SO, int TT>
    __global__ __launch_bounds__(512) void k_mxfp4_gemv(MxGemvArgs a)
    {
        constexpr int NW = 8, RT = 2, ES = 2, NB = 3;
        constexpr int NA = TT == 1 ? 4 : TT == 2 ? 2 : 1;
        constexpr int BM = 16 * NW, P = 4 * ES;                  // pieces (blocks) of a weight row's step
        constexpr int WB = BM * 16 * P, SCB = BM * 4 * P, XB = 16 * TT * 64 * P; // bytes of codes, scales (a word each), tokens
        constexpr int SB = WB + SCB + XB;
        constexpr int XL = (XB / 1024 + NW - 1) / NW;            // token loads a wave (the last ones may repeat)
        constexpr int L = 2 * ES + XL;
        __shared__ __align__(16) char lds[NB * SB];
        const int wv = __builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6)), lane = threadIdx.x & 63;
        const int n = lane & 15, c = lane >> 4;
        const int g = wv >> 1, half = wv & 1;
        const int64_t r0 = int64_t(blockIdx.x) * BM + 16 * wv; // the rows it loads
        const int nblk = a.nblk;
        const int s0 = int(blockIdx.y) * a.splits, s1 = min(s0 + a.splits, a.steps);
        const uint32_t base = lds_address(lds);
        // (a wave past the last row reads it again, and stores nothing)
        const int64_t first = r0 < a.rows ? r0 : a.rows - 1, last = a.rows - 1 - first;
        const uint8_t *wb = a.w + first * (16 * int64_t(nblk)), *wsb = a.ws + first * nblk;
        // A load brings 64 / P rows, lane l piece (l % P) ^ f(row) of its row, f so that reads of 16 rows' same piece hit
        // all banks; of tokens 4 / ES, lane l piece (l % 4 P) ^ (token % 16). (A read of tokens takes a lane's own c's piece,
        // four pieces from the next c's: lanes whose tokens differ by four meet, four cycles a read, 44 % of the LDS cycles at
        // [6656, 19968] by 48.) A block past the rows' ends is taken from their last, and counts as zeros (below).
        auto f = [](int row) { return row >> 1 & 7; };
        uint32_t off[ES], xoff[XL];
        int piece[ES], xp[XL];
#pragma unroll
        for (int t = 0; t < ES; ++t) {
            const int lr = t * (64 / P) + lane / P, row = lr < last ? lr : int(last);
            piece[t] = lane % P ^ f(lr);
            off[t] = uint32_t(row) * (16u * uint32_t(nblk)) + 16u * uint32_t(piece[t]);
        }
        const uint32_t soff = uint32_t(n < last ? n : int(last)) * uint32_t(nblk) + uint32_t(c);
        const uint8_t *xb[XL];
        int xat[XL];
#pragma unroll
        for (int u = 0; u < XL; ++u) {
            const int i = wv + u * NW < XB / 1024 ? wv + u * NW : XB / 1024 - 1;
            const int64_t t0 = i * (4 / ES) < a.T ? i * (4 / ES) : a.T - 1; // (uniform; the load's other tokens follow)
            const int64_t tok = t0 + lane / (4 * P) < a.T ? t0 + lane / (4 * P) : a.T - 1;
            xp[u] = lane % (4 * P) ^ (i * (4 / ES) + lane / (4 * P)) % 16;
            xb[u] = a.x + 2 * t0 * a.ldx;
            xoff[u] = uint32_t(2 * (tok - t0) * a.ldx) + 16u * uint32_t(xp[u]); // (checked on the host: 32 bits do)
            xat[u] = __builtin_amdgcn_readfirstlane(1024 * i);
        }
        auto load = [&](int m, int buf) {
            const uint32_t to = base + buf * SB;
            const int64_t at = int64_t(P) * m; // the step's first block
            const bool tail = P * m + P > nblk;
#pragma unroll
            for (int t = 0; t < ES; ++t) {
                uint32_t o = off[t];
                if (tail && P * m + piece[t] >= nblk) o -= 16u * uint32_t(P * m + piece[t] - nblk + 1);
                lds_load(wb + 16 * at, o, to + 1024 * (ES * wv + t));
            }
#pragma unroll
            for (int s = 0; s < ES; ++s) {
                uint32_t o = soff + 4u * s;
                if (tail && P * m + 4 * s + c >= nblk) o -= uint32_t(P * m + 4 * s + c - nblk + 1);
                lds_load<1>(wsb + at, o, to + WB + 256 * (ES * wv + s));
            }
#pragma unroll
            for (int u = 0; u < XL; ++u) {
                uint32_t o = xoff[u];
                if (tail && 32 * P * m + 8 * xp[u] >= 32 * nblk) o -= 16u * uint32_t(4 * P * m + xp[u] - 4 * nblk + 1);
                lds_load(xb[u] + 64 * at, o, to + WB + SCB + xat[u]);
            }
        };
        f32x4 acc[RT][TT][NA];
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
            for (int u = 0; u < TT; ++u)
#pragma unroll
                for (int k = 0; k < NA; ++k) acc[t][u][k] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        struct Part // a half step's operands
        {
            Vec<uint32_t, 4> w[RT];
            uint32_t ws[RT];
            MxTok<A> x[TT];
        };
        auto read = [&](Part &q, int buf) {
            const char *b = lds + buf * SB;
#pragma unroll
            for (int t = 0; t < RT; ++t) {
                q.w[t] = *reinterpret_cast<const Vec<uint32_t, 4> *>(b + 1024 * ES * (RT * g + t) + 16 * P * n + 16 * ((4 * half + c) ^ f(n)));
                q.ws[t] = *reinterpret_cast<const uint32_t *>(b + WB + 256 * (ES * (RT * g + t) + half) + 4 * lane);
            }
#pragma unroll
            for (int u = 0; u < TT; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    q.x[u].v[i] = *reinterpret_cast<const Vec<uint32_t, 4> *>(b + WB + SCB + 64 * P * (16 * u + n) + 16 * ((16 * half + 4 * c + i) ^ n));
        };
        uint32_t past = ~0u; // the least scale's place from where bf16 and f32 end
        auto products = [&](Part &q, int m) {
            if (P * m + P > nblk && P * m + 4 * half + c >= nblk) {
#pragma unroll
                for (int t = 0; t < RT; ++t) {
                    q.w[t] = Vec<uint32_t, 4>{{0u, 0u, 0u, 0u}};
                    q.ws[t] = 127u;
                }
#pragma unroll
                for (int u = 0; u < TT; ++u)
#pragma unroll
                    for (int i = 0; i < 4; ++i) q.x[u].v[i] = Vec<uint32_t, 4>{{0u, 0u, 0u, 0u}};
            }
#pragma unroll
            for (int t = 0; t < RT; ++t) past = min(past, mx_past<A>(q.ws[t]));
            mx_step<A, RT, TT, NA>(q.w, q.ws, q.x, acc);
        };
        int buf = 0, next = NB - 1; // of the step that arrives next, of the one to be loaded then
        auto arrive = [&](int m) {
            // step m has landed for every wave, and every wave has read step m - 1, whose buffer step m + NB - 1 takes
            if (NB > 2 && m + NB - 1 <= s1)
                __asm__ volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((NB - 2) * L) : "memory");
            else
                __asm__ volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
            if (m + NB - 1 < s1) load(m + NB - 1, next);
            next = next + 1 < NB ? next + 1 : 0;
        };
#pragma unroll
        for (int p = 0; p < NB - 1; ++p)
            if (s0 + p < s1) load(s0 + p, p);
        for (int m = s0; m < s1; ++m) {
            arrive(m);
            Part q;
            read(q, buf);
            buf = buf + 1 < NB ? buf + 1 : 0;
            products(q, m);
        }
        // lane (token n, c) holds rows 4 c .. 4 c + 3 of a tile; the second half's sums pass through LDS
        f32x4 own[RT][TT];
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
            for (int u = 0; u < TT; ++u) own[t][u] = mx_total(acc[t][u]);
        if (mx_any_past<A>(past))
            mx_far_sums<A, RT, TT>(a, int64_t(blockIdx.x) * BM + 16 * RT * g, 0, s1 - s0, [&](int k) { return 2 * (s0 + k) + half; }, own);
        __syncthreads();
        f32x4 *sums = reinterpret_cast<f32x4 *>(lds) + RT * TT * 64 * g + lane;
        static_assert(4 * RT * TT * 1024 <= NB * SB, "room for them");
        if (half == 1) {
#pragma unroll
            for (int t = 0; t < RT; ++t)
#pragma unroll
                for (int u = 0; u < TT; ++u) sums[64 * (TT * t + u)] = own[t][u];
        }
        __syncthreads();
        if (half == 1) return;
        typename SO::raw *y = static_cast<typename SO::raw *>(a.y) + blockIdx.y * a.ysplit;
#pragma unroll
        for (int u = 0; u < TT; ++u) {
            const int64_t tok = 16 * u + n;
            if (tok >= a.T) continue;
#pragma unroll
            for (int t = 0; t < RT; ++t) {
                const f32x4 s = own[t][u] + sums[64 * (TT * t + u)];
                const int64_t o = int64_t(blockIdx.x) * BM + 16 * (RT * g + t) + 4 * c;
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (o + r < a.rows) y[tok * a.ldy + o + r] = SO::enc32(s[r]);
            }
        }
    }

    namespace
    {
        // (of one token: two waves sharing a row's steps 16.9 us, four 16.4, none 16.4 at [25600, 5120]; 20.2, 18.9 and 34.7
        // at [5120, 25600])
        template <class A, class SO, int XR>
        void go_wave(mg_ctx *c, MxGemvArgs a)
        {
            const int64_t tiles = (a.rows + 15) / 16;
            need(launchable(tiles, 256), "mxfp4 product: too many rows");
            a.steps = (a.nblk + 15) / 16;
            const bool aligned = a.nblk % 16 == 0 && aligned16(a.ws) && (A::dt != kMxFp4 || aligned16(a.xs));
            auto go = [&](auto kern, int64_t passes) {
                hipLaunchKernelGGL(kern, dim3(unsigned(tiles), unsigned(passes)), dim3(256), 0, c->stream, a);
                check_launch("k_mxfp4_gemv_wave");
            };
            // (16-bit tokens are one pass)
            for (const int64_t most = 65535 * XR; a.T > 0; a.T -= most) {
                const int64_t passes = ((a.T < most ? a.T : most) + XR - 1) / XR;
                aligned ? go(k_mxfp4_gemv_wave<A, SO, XR, true>, passes) : go(k_mxfp4_gemv_wave<A, SO, XR, false>, passes);
                if constexpr (A::dt == kMxFp4) {
                    a.x += most * 16 * a.nblk;
                    a.xs += most * a.nblk;
                    a.y = static_cast<typename SO::raw *>(a.y) + most * a.ldy;
                }
            }
        }

        // five to 64 tokens of 16 bits
        template <class A, class SO>
        void go_shared(mg_ctx *c, MxGemvArgs a)
        {
            a.steps = (a.nblk + 7) / 8;
            const int64_t tiles = (a.rows + 127) / 128;
            need(launchable(tiles, 512), "mxfp4 product: too many rows");
            // parts of a row that fill the chip's CUs, of five steps at least ([6656, 19968] by 48, f16: four 40 us, one 112;
            // a second work-group a CU waits for its turn: nine 45; [5120, 25600] by 64: six 42, twelve 52)
            int64_t s = tiles < c->num_cus ? c->num_cus / tiles : 1;
            s = s < a.steps / 5 ? s : a.steps / 5;
            while (s > 1 && s * a.T * a.rows * 4 > c->work_bytes) --s;
            a.splits = s > 1 ? int((a.steps + s - 1) / s) : a.steps;
            const int ns = a.splits > 0 ? (a.steps + a.splits - 1) / a.splits : 1;
            void *y = a.y;
            const int64_t ldy = a.ldy;
            if (ns > 1) {
                a.y = c->work;
                a.ldy = a.rows;
                a.ysplit = a.rows * a.T;
            }
            auto tile = [&](auto so) {
                using O = decltype(so);
                auto go = [&](auto kern) {
                    hipLaunchKernelGGL(kern, dim3(unsigned(tiles), unsigned(ns)), dim3(512), 0, c->stream, a);
                    check_launch("k_mxfp4_gemv");
                };
                if (a.T <= 32)
                    a.T <= 16 ? go(k_mxfp4_gemv<A, O, 1>) : go(k_mxfp4_gemv<A, O, 2>);
                else
                    a.T <= 48 ? go(k_mxfp4_gemv<A, O, 3>) : go(k_mxfp4_gemv<A, O, 4>);
            };
            if (ns > 1) {
                tile(SF32{});
                join_splits(c, static_cast<const float *>(c->work), ns, y, ldy, a.rows, a.T, SO::dt);
            } else {
                tile(SO{});
            }
        }
    }

    void launch_gemv_mxfp4(mg_ctx *c, const uint8_t *qs, const uint8_t *s, const void *x, int64_t ldx, int64_t batch,
                           int64_t rows, int64_t in, void *y, int64_t ldy, int dt, int dt_out)
    {
        need(rows >= 0 && in >= 0 && batch >= 1 && batch <= 64, "gemv_mxfp4: batch must be in [1, 64]");
        need(in % 32 == 0, "gemv_mxfp4: input dim must be a multiple of 32 (got " + std::to_string(in) + ")");
        need(dt == BF16 || dt == F16, "gemv_mxfp4: dtype must be bf16 or f16");
        need(dt_out == dt || dt_out == F32, "gemv_mxfp4: dtype_out must be f32 or the activations' dtype");
        if (rows == 0) return;
        if (ldx == 0) ldx = in;
        if (ldy == 0) ldy = rows;
        need(y && (in == 0 || (qs && s && x)), "gemv_mxfp4: NULL tensor");
        need(ldx >= in && ldy >= rows, "gemv_mxfp4: leading dimension too small");
        need(in == 0 || (aligned16(qs) && aligned16(x) && ldx % 8 == 0), "gemv_mxfp4: codes and activations must be 16-byte aligned");
        need(ldx < (int64_t(1) << 30), "gemv_mxfp4: leading dimension too large");
        need(in <= (int64_t(1) << 27), "gemv_mxfp4: input dim too large");
        const int nblk = int(in / 32);
        const MxGemvArgs a{qs, s, static_cast<const uint8_t *>(x), nullptr, y, ldx, ldy, rows, batch, 0, nblk, 0, 0};
        auto go = [&](auto s_, auto so) {
            using S = decltype(s_);
            using SO = decltype(so);
            if (batch == 1)
                go_wave<S, SO, 1>(c, a);
            else
                batch <= 4 ? go_wave<S, SO, 4>(c, a) : go_shared<S, SO>(c, a);
        };
        if (dt == BF16)
            dt_out == F32 ? go(SBf16{}, SF32{}) : go(SBf16{}, SBf16{});
        else
            dt_out == F32 ? go(SF16{}, SF32{}) : go(SF16{}, SF16{});
    }

    void launch_gemm_mxfp4(mg_ctx *c, const uint8_t *aq, const uint8_t *as, int64_t tokens, const uint8_t *qs, const uint8_t *s,
                           int64_t rows, int64_t in, void *y, int64_t ldy, int dt_out)
    {
        need(rows >= 0 && in >= 0 && tokens >= 0, "gemm_mxfp4: bad shape");
        need(in % 32 == 0, "gemm_mxfp4: input dim must be a multiple of 32 (got " + std::to_string(in) + ")");
        need(dt_out == BF16 || dt_out == F16 || dt_out == F32, "gemm_mxfp4: dtype_out must be bf16, f16 or f32");
        if (rows == 0 || tokens == 0) return;
        if (ldy == 0) ldy = rows;
        need(y && (in == 0 || (aq && as && qs && s)), "gemm_mxfp4: NULL tensor");
        need(ldy >= rows, "gemm_mxfp4: leading dimension too small");
        need(in == 0 || (aligned16(aq) && aligned16(qs)), "gemm_mxfp4: codes must be 16-byte aligned");
        need(in <= (int64_t(1) << 27), "gemm_mxfp4: input dim too large");
        // The waves' form reads the weight once for every 16 tokens and starts soonest: up to 16 tokens, and up to 128 where
        // that is little to read, the tiles else ([5120, 5120] by 64: 10.5 us, tiles 12.6; by 128: 17.7 / 14.0;
        // [25600, 5120] by 17: 27 / 19; [25600, 1024] by 40: 17 / 7).
        const int64_t passes = (tokens + 15) / 16;
        const bool few = passes == 1 || (passes <= 8 && in >= 2048 && passes <= (int64_t(10) << 24) / (rows * in));
        if (!few && launch_mxfp4_tiles(c, aq, as, tokens, qs, s, rows, in, y, ldy, dt_out)) return;
        const int nblk = int(in / 32);
        const MxGemvArgs a{qs, s, aq, as, y, 0, ldy, rows, tokens, 0, nblk, 0, 0};
        if (dt_out == F32)
            go_wave<SMxFp4, SF32, 16>(c, a);
        else
            dt_out == BF16 ? go_wave<SMxFp4, SBf16, 16>(c, a) : go_wave<SMxFp4, SF16, 16>(c, a);
    }
} // namespace mg
