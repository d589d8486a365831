// Products of two MXFP4 operands over many tokens, for gfx950: y[t, o] = sum_i
// W[o, i] A[t, i], codes and scales of both as they lie (mg_mxfp4.hpp).
//
// A work-group of four waves takes a tile of BM weight rows and BN tokens; a wave
// WM x WN of it, as 32 x 32 x 64 scaled products (v_mfma_scale_f32_32x32x64_f8f6f4:
// lane 32 h + n holds block h of two, 16 bytes, of row n and its scale). Steps are of
// 128 elements, loaded straight into LDS in pairs, 128 bytes a row an instruction (a step at a
// time, 64 bytes a row, was bound by requests to the L2: [5120, 25600] by 333 tokens 50 us
// for 44, [5120, 19968] by 4096 302 for 269), and read there one half ahead; the four steps of
// a round are one straight line of code, each product followed by a load or an LDS
// read of what comes next (in runs of their own they cost 387 us where this takes 355 at
// [25600, 5120] by 4096). Results go out through LDS in 16-byte pieces.
//   At [25600, 5120] by 4096 (bf16 out) 305-320 us, 3.4-3.5 PFLOP/s: 1600 tiles are 6.25
// rounds of the CUs, paid as seven (15 % of the cycles a CU has none); 8192^3, four
// rounds, reaches 3.8. What holds that is power (zeros 5.6; from registers 6.2 and 9.0)
// and the reads from LDS: 39 % of its cycles are conflicts, by their counts those of the
// scales, a word a row 16 bytes apart. A bf16 product of 8192^3 by the library
// reaches 1.13 here. Rows that are not whole 512s are taken as if they were, their loads
// checked one by one, after a launch that lays both operands' scales out, at every call:
// [5120, 25632] by 333 64 us where 25600 takes 48, [5120, 5152] by 512 27 for 20, [25600,
// 5152] by 4096 412 for 342 (weights in turn, from HBM).
#include "mg_device.hpp"
#include "mg_internal.hpp"
#include "mg_mxfp4.hpp"

namespace mg
{
    struct MxGemmArgs
    {
        const uint8_t *w, *ws, *x, *xs;
        void *y;
        int64_t ldy, rows, T, ysplit; // elements of y between splits' results
        int nblk, spitch;             // in / 32; bytes between rows' scales, whole 16s
        int steps, splits;            // steps of 128 elements, whole fours, and how many of them a split takes
        int tm, tn;                   // tiles
        bool vec;                     // y takes 16-byte stores
    };

    template <int OA, int OB>
    MG_DEV f32x16 mfma_mxfp4_32(Vec<uint32_t, 4> a, uint32_t sa, Vec<uint32_t, 4> b, uint32_t sb, f32x16 c)
    {
        typedef int i32x8 __attribute__((ext_vector_type(8)));
        const i32x8 av = {int(a.v[0]), int(a.v[1]), int(a.v[2]), int(a.v[3]), 0, 0, 0, 0};
        const i32x8 bv = {int(b.v[0]), int(b.v[1]), int(b.v[2]), int(b.v[3]), 0, 0, 0, 0};
        return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(av, bv, c, 4, 4, OA, int(sa), OB, int(sb));
    }

    template <int N>
    MG_DEV void wait_and_meet() // all but the last N such loads have landed, in every wave
    {
        __builtin_amdgcn_sched_barrier(0);
        __asm__ volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
        __builtin_amdgcn_sched_barrier(0);
    }

    // a pair rounded to 16 bits, a NaN as the conversion leaves it
    template <class SO>
    MG_DEV uint32_t pack16(float a, float b)
    {
        if constexpr (SO::dt == BF16)
            return bf_pack(a, b);
        else
            return uint32_t(SF16::enc_finite(a)) | uint32_t(SF16::enc_finite(b)) << 16;
    }

    // The tile's place: work-groups go to the XCDs in turn; each XCD takes a run of tiles, in
    // groups of 4 token tiles by all weight tiles, so that its L2 holds what its CUs share.
    MG_DEV void tile_of(const MxGemmArgs &a, int id, int &m, int &n)
    {
        const int total = a.tm * a.tn, q = total / 8, r = total % 8;
        const int xcd = id % 8, turn = id / 8;
        int t = xcd * q + (xcd < r ? xcd : r) + turn;
        constexpr int GN = 4;
        const int per = GN * a.tm, grp = t / per, first = grp * GN, in = t - grp * per;
        const int width = a.tn - first < GN ? a.tn - first : GN;
        m = in / width;
        n = first + in % width;
    }

    // TAIL: the last steps reach past the rows' ends. Blocks there take codes of block 0 and scales of 0 on both
    // sides: 2^-254 of a product of at most 36 is far below f32's smallest value, and adds nothing.
    // NB: steps in LDS.
    template <class SO, int BM, int BN, int WM, int WN, int NB, bool TAIL>
    __global__ __launch_bounds__(256, BM * BN * NB > 128 * 128 * 4 ? 1 : 2) void k_mxfp4_gemm(MxGemmArgs a)
    {
        static_assert((BM / WM) * (BN / WN) == 4, "four waves");
        static_assert(NB == 4 || NB == 8, "a round of four steps in LDS, or two");
        constexpr int R = BM + BN, NU = NB / 2, RP = 128; // a step's rows; pairs of steps in LDS; bytes of a pair's row
        constexpr int TM = WM / 32, TN = WN / 32;
        constexpr int L = R / 32, LS = R / 256 > 0 ? R / 256 : 1; // loads a wave: of a pair's codes, of four steps' scales
        constexpr int CB = R * RP, SB = R * 16;
        __shared__ __align__(16) char lds[NU * CB + 2 * SB];
        const int wv = __builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6)), lane = threadIdx.x & 63;
        const int split = blockIdx.y;
        int tm, tn;
        tile_of(a, blockIdx.x, tm, tn);
        tm = __builtin_amdgcn_readfirstlane(tm); // (the division leaves them in vector registers)
        tn = __builtin_amdgcn_readfirstlane(tn);
        const int64_t m0 = int64_t(tm) * BM, n0 = int64_t(tn) * BN;
        const int s0 = split * a.splits, s1 = min(s0 + a.splits, a.steps), S = s1 - s0;
        const uint32_t base = lds_address(lds);
        const uint32_t wbytes = 16u * uint32_t(a.nblk); // of a row
        // Rows are the tile's weight rows, then its tokens. Load j of wave w brings 128 bytes of rows 8 (4 j + w) .. + 7, lane
        // l piece (l % 8) ^ turned(row) of row l / 8, so that reads of 16 rows' same piece hit all banks.
        auto turned = [](int row) { return row >> 1 & 7; };
        const int lp = lane % 8 ^ turned(8 * wv + lane / 8); // (32 j rows more turn it the same)
        uint32_t off[L], soff[LS];
#pragma unroll
        for (int j = 0; j < L; ++j) {
            const int r = 8 * (4 * j + wv) + lane / 8;
            const bool isw = 8 * (4 * j + wv) < BM;
            const int64_t last = isw ? a.rows - 1 - m0 : a.T - 1 - n0;
            const int rr = isw ? r : r - BM, row = rr < last ? rr : int(last);
            off[j] = uint32_t(row) * wbytes + 16u * uint32_t(lp);
        }
#pragma unroll
        for (int j = 0; j < LS; ++j) {
            const int r = 64 * (4 * j + wv) + lane;
            const bool isw = 64 * (4 * j + wv) < BM;
            const int64_t last = isw ? a.rows - 1 - m0 : a.T - 1 - n0;
            const int rr = isw ? r : r - BM, row = rr < last ? rr : int(last);
            soff[j] = uint32_t(row) * uint32_t(a.spitch);
        }
        const uint8_t *wb = a.w + m0 * wbytes, *xb = a.x + n0 * wbytes;
        const uint8_t *wsb = a.ws + m0 * a.spitch, *xsb = a.xs + n0 * a.spitch;
        auto load_codes = [&](int u, auto J) { // load j of pair u, steps s0 + 2 u, + 1
            constexpr int j = decltype(J)::value;
            const bool isw = 8 * (4 * j + wv) < BM;
            const uint32_t to = base + (u % NU) * CB + 1024 * (4 * j + wv);
            const int pair = s0 / 2 + u;
            if constexpr (TAIL)
                lds_load(isw ? wb : xb, 8 * pair + lp < a.nblk ? off[j] + uint32_t(RP) * uint32_t(pair) : off[j] - 16u * uint32_t(lp), to);
            else
                lds_load((isw ? wb : xb) + RP * int64_t(pair), off[j], to);
        };
        auto load_scales = [&](int g, auto J) { // load j of the scales of steps s0 + 4 g .. + 3
            constexpr int j = decltype(J)::value;
            const bool isw = 64 * (4 * j + wv) < BM;
            lds_load((isw ? wsb : xsb) + 16 * (int64_t(s0 / 4) + g), soff[j], base + NU * CB + (g & 1) * SB + 1024 * (4 * j + wv));
        };
        auto all_codes = [&](int u) { each<0, L>([&](auto J) { load_codes(u, J); }); };
        auto all_scales = [&](int g) { each<0, LS>([&](auto J) { load_scales(g, J); }); };
        const int n = lane & 31, h = lane >> 5;
        const int wr = wv / (BN / WN) * WM, wc = wv % (BN / WN) * WN; // the wave's place in the tile
        f32x16 acc[TM][TN];
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;
        struct Frag
        {
            Vec<uint32_t, 4> a[TM], b[TN];
            uint32_t sa[TM], sb[TN];
        };
        // half s of a step: blocks 2 s + h; its scales come with the first, four to a word
        const char *fa = lds + (wr + n) * RP, *fb = lds + (BM + wc + n) * RP;
        int pieces[4]; // of a pair's halves
#pragma unroll
        for (int i = 0; i < 4; ++i) pieces[i] = 16 * ((2 * i + h) ^ turned(n));
        auto read = [&](Frag &f, int pair, auto half, auto I) { // operand i of the wave's rows, then tokens
            constexpr int s = decltype(half)::value, i = decltype(I)::value;
            if constexpr (i < TM)
                f.a[i] = *reinterpret_cast<const Vec<uint32_t, 4> *>(fa + pair * CB + pieces[s] + 32 * RP * i);
            else
                f.b[i - TM] = *reinterpret_cast<const Vec<uint32_t, 4> *>(fb + pair * CB + pieces[s] + 32 * RP * (i - TM));
        };
        const char *ga = lds + NU * CB + 16 * (wr + n), *gb = lds + NU * CB + 16 * (BM + wc + n);
        auto read_scale = [&](Frag &f, int buf, int at, auto I) {
            constexpr int i = decltype(I)::value;
            if constexpr (i < TM)
                f.sa[i] = *reinterpret_cast<const uint32_t *>(ga + buf * SB + 4 * at + 512 * i);
            else
                f.sb[i - TM] = *reinterpret_cast<const uint32_t *>(gb + buf * SB + 4 * at + 512 * (i - TM));
        };
        using H0 = std::integral_constant<int, 0>;
        using H1 = std::integral_constant<int, 1>;
        constexpr int NM = TM * TN, NR = TM + TN;
        // a half's products, with `beside` issued after each: a wave has its SIMD's matrix core to itself, which would
        // wait while loads and reads are issued in one run
        auto products = [&](const Frag &f, const uint32_t (&sa)[TM], const uint32_t (&sb)[TN], auto half, auto beside) {
            constexpr int O = 2 * decltype(half)::value;
            each<0, NM>([&](auto M) {
                constexpr int i = decltype(M)::value / TN, j = decltype(M)::value % TN;
                acc[i][j] = mfma_mxfp4_32<O, O>(f.a[i], sa[i], f.b[j], sb[j], acc[i][j]);
                beside(M);
                __builtin_amdgcn_sched_barrier(0);
            });
        };
        // A pair's buffer takes the pair NU behind it as soon as every wave has read its second step, whose second half
        // is read beneath the products of its first; the next pair has to have landed there, too: the waves meet once a
        // pair. Scales of four steps come with the fourth step of the round two before (of the last one again, so that
        // the counts hold).
        const int last_g = S / 4 - 1;
        all_scales(0);
        all_scales(last_g > 0 ? 1 : 0);
        all_codes(0);
        all_codes(1); // (S >= 4)
        if (NU > 2 && last_g > 0) {
            all_codes(2);
            all_codes(3);
            wait_and_meet<3 * L>();
        } else {
            wait_and_meet<L>();
        }
        Frag f0, f1;
        each<0, NR>([&](auto I) {
            read(f0, 0, H0{}, I);
            read_scale(f0, 0, 0, I);
        });
        // LEFT: rounds behind this one, two for any number
        auto step = [&](int g, auto P, auto left) {
            constexpr int p = decltype(P)::value, LEFT = decltype(left)::value;
            constexpr bool loads = LEFT >= NB / 4, ends = p % 2 == 1; // a pair's second step
            // the step's pair's place, and the next step's
            const int pair = NB == 8 ? (g & 1) * 2 + p / 2 : p / 2;
            const int next = p < 3 ? (NB == 8 ? (g & 1) * 2 : 0) + (p + 1) / 2 : NB == 8 ? (~g & 1) * 2 : 0;
            uint32_t sa[TM], sb[TN]; // the lane's blocks in bytes 0 and 2
#pragma unroll
            for (int i = 0; i < TM; ++i) sa[i] = f0.sa[i] >> (8 * h);
#pragma unroll
            for (int j = 0; j < TN; ++j) sb[j] = f0.sb[j] >> (8 * h);
            // items 0 .. N - 1 spread over products `from` .. `to` - 1
            auto spread = [](auto M, auto N, auto from, auto to, auto item) {
                constexpr int m = decltype(M)::value, k = decltype(N)::value, a = decltype(from)::value, b = decltype(to)::value;
                if constexpr (m >= a && m < b) each<(m - a) * k / (b - a), (m - a + 1) * k / (b - a)>(item);
            };
            using Half = std::integral_constant<int, (NM + 1) / 2>;
            products(f0, sa, sb, H0{}, [&](auto M) {
                spread(M, std::integral_constant<int, NR>{}, H0{}, Half{},
                       [&](auto I) { read(f1, pair, std::integral_constant<int, 2 * (p % 2) + 1>{}, I); });
            });
            // the next pair has landed, but for those that were asked for behind it
            if constexpr (ends && LEFT == 0 && p < 3)
                wait_and_meet<0>();
            else if constexpr (ends && LEFT > 0)
                wait_and_meet<loads || p < 3 ? (NU - 2) * L : L>();
            products(f1, sa, sb, H1{}, [&](auto M) {
                if constexpr (p < 3 || LEFT > 0)
                    spread(M, std::integral_constant<int, NR>{}, H0{}, Half{}, [&](auto I) {
                        read(f0, next, std::integral_constant<int, 2 * ((p + 1) % 2)>{}, I);
                        read_scale(f0, (g + (p == 3)) & 1, (p + 1) % 4, I);
                    });
                if constexpr (loads && p == 3 && decltype(M)::value == 0) all_scales(g + 2 < last_g ? g + 2 : last_g);
                if constexpr (loads && ends)
                    spread(M, std::integral_constant<int, L>{}, H0{}, Half{}, [&](auto J) { load_codes(2 * g + p / 2 + NU, J); });
            });
        };
        auto four = [&](int g, auto left) {
            step(g, std::integral_constant<int, 0>{}, left);
            step(g, std::integral_constant<int, 1>{}, left);
            step(g, std::integral_constant<int, 2>{}, left);
            step(g, std::integral_constant<int, 3>{}, left);
        };
        using R0 = std::integral_constant<int, 0>;
        using R1 = std::integral_constant<int, 1>;
        using R2 = std::integral_constant<int, 2>;
        if constexpr (NB == 4) {
            for (int g = 0; g < last_g; ++g) four(g, R1{});
        } else {
            for (int g = 0; g + 1 < last_g; ++g) four(g, R2{});
            if (last_g > 0) four(last_g - 1, R1{});
        }
        four(last_g, R0{});
        // Lane (token n, h) holds rows 8 (e / 4) + 4 h + e % 4 of its column. 32 tokens at a time go through LDS, so
        // that a store instruction writes whole runs of a token's row.
        // (the sums are final here: without this the last products sink into the stores' branches, with copies and spills)
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j) {
                if constexpr (TM * TN > 8)
                    __asm__ volatile("" : "+a"(acc[i][j]));
                else
                    __asm__ volatile("" : "+v"(acc[i][j]));
            }
        __syncthreads();
        using raw = typename SO::raw;
        constexpr int ES = sizeof(raw), PITCH = WM * ES + 16, PL = WM * ES / 16; // lanes of 16 bytes a token
        static_assert(4 * 32 * PITCH <= int(sizeof(lds)), "a wave's 32 tokens");
        char *lo = lds + wv * 32 * PITCH;
        raw *y = static_cast<raw *>(a.y) + split * a.ysplit;
#pragma unroll
        for (int j = 0; j < TN; ++j) {
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int e = 0; e < 16; e += 4) {
                    char *to = lo + n * PITCH + (32 * i + 2 * e + 4 * h) * ES;
                    if constexpr (ES == 4)
                        *reinterpret_cast<Vec<float, 4> *>(to) =
                            Vec<float, 4>{{acc[i][j][e], acc[i][j][e + 1], acc[i][j][e + 2], acc[i][j][e + 3]}};
                    else
                        *reinterpret_cast<Vec<uint32_t, 2> *>(to) = Vec<uint32_t, 2>{
                            {pack16<SO>(acc[i][j][e], acc[i][j][e + 1]), pack16<SO>(acc[i][j][e + 2], acc[i][j][e + 3])}};
                }
            wave_lds_sync();
#pragma unroll
            for (int r = 0; r < 32; r += 64 / PL) {
                const int row = r + lane / PL, pc = lane % PL;
                Vec<uint32_t, 4> v = *reinterpret_cast<const Vec<uint32_t, 4> *>(lo + row * PITCH + 16 * pc);
                if constexpr (ES == 2) { // NaNs in the library's one pattern
                    uint32_t mag = 0;
#pragma unroll
                    for (int e = 0; e < 4; ++e) mag = pk_max_u16(mag, v.v[e] & 0x7fff7fffu);
                    if (max(mag & 0xffffu, mag >> 16) > (SO::dt == BF16 ? 0x7f80u : 0x7c00u)) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) v.v[e] = SO::dt == BF16 ? bf_canon(v.v[e]) : hf_canon(v.v[e]);
                    }
                }
                const int64_t t = n0 + wc + 32 * j + row, o = m0 + wr + pc * (16 / ES);
                if (t >= a.T) continue;
                raw *to = y + t * a.ldy + o;
                if (a.vec && o + 16 / ES <= a.rows) {
                    st16_stream<raw, 16 / ES>(to, __builtin_bit_cast(Vec<raw, 16 / ES>, v));
                } else {
                    const Vec<raw, 16 / ES> w = __builtin_bit_cast(Vec<raw, 16 / ES>, v);
#pragma unroll
                    for (int e = 0; e < 16 / ES; ++e)
                        if (o + e < a.rows) to[e] = w.v[e];
                }
            }
            wave_lds_sync();
        }
    }

    // the splits' sums, [n][T][rows], added in their order
    template <class SO, int V>
    __global__ __launch_bounds__(256) void k_mxfp4_gemm_join(const float *part, int n, typename SO::raw *y, int64_t ldy,
                                                             int64_t rows, int64_t T)
    {
        const int64_t i = (int64_t(blockIdx.x) * 256 + threadIdx.x) * V, all = T * rows;
        if (i >= all) return;
        Vec<float, V> s = *reinterpret_cast<const Vec<float, V> *>(part + i);
        for (int k = 1; k < n; ++k) {
            const Vec<float, V> x = *reinterpret_cast<const Vec<float, V> *>(part + k * all + i);
#pragma unroll
            for (int e = 0; e < V; ++e) s.v[e] += x.v[e];
        }
        const int64_t t = i / rows;
        Vec<typename SO::raw, V> o;
#pragma unroll
        for (int e = 0; e < V; ++e) o.v[e] = SO::enc32(s.v[e]);
        typename SO::raw *to = y + t * ldy + (i - t * rows);
#pragma unroll
        for (int e = 0; e < V; ++e) to[e] = o.v[e];
    }

    // scales of rows of nblk blocks, then of more rows, as rows of whole 16s, zeros behind a row's end
    __global__ __launch_bounds__(256) void k_mxfp4_scales(const uint8_t *a, int64_t rows_a, const uint8_t *b, int64_t rows,
                                                          int nblk, int pitch, uint32_t *out)
    {
        const int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x;
        const int per = pitch / 4;
        const int64_t r = i / per;
        if (r >= rows) return;
        const int at = int(i - r * per) * 4;
        const uint8_t *src = r < rows_a ? a + r * nblk : b + (r - rows_a) * nblk;
        uint32_t w = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (at + k < nblk) w |= uint32_t(src[at + k]) << (8 * k);
        out[i] = w;
    }

    void join_splits(mg_ctx *c, const float *part, int ns, void *y, int64_t ldy, int64_t rows, int64_t T, int dt_out)
    {
        const bool v = rows % 4 == 0;
        auto join = [&](auto so, auto kern) {
            using raw = typename decltype(so)::raw;
            const int64_t blocks = (T * rows + (v ? 1023 : 255)) / (v ? 1024 : 256);
            hipLaunchKernelGGL(kern, dim3(unsigned(blocks)), dim3(256), 0, c->stream, part, ns, static_cast<raw *>(y), ldy, rows, T);
            check_launch("k_mxfp4_gemm_join");
        };
        auto to = [&](auto so) {
            using SO = decltype(so);
            v ? join(so, k_mxfp4_gemm_join<SO, 4>) : join(so, k_mxfp4_gemm_join<SO, 1>);
        };
        dt_out == F32 ? to(SF32{}) : dt_out == BF16 ? to(SBf16{}) : to(SF16{});
    }

    namespace
    {
        // How a product is divided: into 256 x 256 tiles, one a CU, or 128 x 128 ones, eight steps of one in LDS or four of
        // each of two a CU, the sums into up to eight parts, whichever this estimate in us has soonest. Large tiles read
        // half as much a product and take 0.78 us a step and 7 to start and end; of the small ones a deep one takes 0.26 a
        // step and 2, two on a CU 0.57 for both, one's start and end beneath the other's steps; the parts' sums are written
        // and read once more. Fitted to 77 products of 1024 to 19968 by 512 to 25600 weights, whole 512s, and 129 to 4096 tokens; what
        // it picks takes 1.2% more than the best of up to 11 tried there on average, 13% at worst. (Large, deep and two, the
        // best parts of the first two: [25600, 5120] x 4096 313, 440, 380 us; x 200: 48, 38, 37; [25600, 1024] x
        // 4096: 113, 134, 88; [5120, 5120] x 512: 35, 15, 17; x 4096: 88, 77, 68; [5120, 19968] x 1024: 88, 111, 105; x
        // 200: 57, 31, 79.)
        enum Tile
        {
            kLarge,
            kDeep,
            kTwo
        };
        struct Tiling
        {
            Tile tile;
            int splits;
        };
        Tiling tiling(int64_t rows, int64_t T, int groups, int64_t room, int64_t cus)
        {
            auto tiles = [&](int64_t b) { return ((rows + b - 1) / b) * ((T + b - 1) / b); };
            Tiling best{kDeep, 1};
            float soonest = 0;
            for (const Tile tile : {kDeep, kTwo, kLarge})
                for (int s = 1; s <= (tile == kTwo ? 1 : groups < 8 ? groups : 8); ++s) {
                    const int64_t parts = int64_t(s) * T * rows * 4;
                    if (s > 1 && (parts > room || !launchable((T * rows + 255) / 256, 256))) break; // (the join's)
                    const int64_t n = tiles(tile == kLarge ? 256 : 128) * s, rounds = (n + cus - 1) / cus;
                    const float steps = float((groups + s - 1) / s * 4);
                    float t = s > 1 ? 2.5f + float(parts) * (2 / 4.1e6f) : 0.f;
                    if (tile == kLarge)
                        t += float(rounds) * (0.78f * steps + 7.f);
                    else if (tile == kDeep)
                        t += float(rounds) * (0.26f * steps + 2.1f);
                    else
                        t += n <= cus ? 0.33f * steps + 1.2f : (n <= 2 * cus ? 1.f : float(n) / float(2 * cus)) * (0.57f * steps + 1.8f);
                    if ((tile == kDeep && s == 1) || t < soonest) {
                        soonest = t;
                        best = {tile, s};
                    }
                }
            return best;
        }

        template <class SO>
        void tiles_t(mg_ctx *c, MxGemmArgs a, Tile tile, int ns, bool tail)
        {
            const int B = tile == kLarge ? 256 : 128;
            const int64_t tm = (a.rows + B - 1) / B, tn = (a.T + B - 1) / B;
            need(launchable(tm * tn, 256), "gemm_mxfp4: too many rows or tokens");
            a.tm = int(tm);
            a.tn = int(tn);
            constexpr int64_t per = 16 / sizeof(typename SO::raw); // elements of a 16-byte store
            a.vec = aligned16(a.y) && a.ldy % per == 0 && a.ysplit % per == 0;
            auto go = [&](auto kern) {
                hipLaunchKernelGGL(kern, dim3(unsigned(tm * tn), unsigned(ns)), dim3(256), 0, c->stream, a);
                check_launch("k_mxfp4_gemm");
            };
            auto of = [&](auto tail_) {
                constexpr bool TAIL = decltype(tail_)::value;
                if (tile == kLarge)
                    go(k_mxfp4_gemm<SO, 256, 256, 128, 128, 4, TAIL>);
                else
                    tile == kDeep ? go(k_mxfp4_gemm<SO, 128, 128, 64, 64, 8, TAIL>) : go(k_mxfp4_gemm<SO, 128, 128, 64, 64, 4, TAIL>);
            };
            tail ? of(std::true_type{}) : of(std::false_type{});
        }
    }

    bool launch_mxfp4_tiles(mg_ctx *c, const uint8_t *aq, const uint8_t *as, int64_t tokens, const uint8_t *qs, const uint8_t *s,
                            int64_t rows, int64_t in, void *y, int64_t ldy, int dt_out)
    {
        // (a tile's rows lie within 32-bit offsets)
        if (in == 0 || in > (int64_t(1) << 24)) return false;
        const int nblk = int(in / 32), groups = (nblk + 15) / 16;
        const bool tail = nblk % 16 != 0;
        char *work = static_cast<char *>(c->work);
        int64_t room = c->work_bytes;
        MxGemmArgs a{qs, s, aq, as, y, ldy, rows, tokens, 0, nblk, nblk, 4 * groups, 0, 0, 0, false};
        if (tail || !aligned16(as) || !aligned16(s)) {
            a.spitch = 16 * groups;
            const int64_t words = (rows + tokens) * (a.spitch / 4), blocks = (words + 255) / 256;
            const int64_t bytes = (4 * words + 255) / 256 * 256;
            if (bytes > room || !launchable(blocks, 256)) return false;
            hipLaunchKernelGGL(k_mxfp4_scales, dim3(unsigned(blocks)), dim3(256), 0, c->stream, s, rows, as, rows + tokens, nblk,
                               a.spitch, reinterpret_cast<uint32_t *>(work));
            check_launch("k_mxfp4_scales");
            a.ws = reinterpret_cast<const uint8_t *>(work);
            a.xs = a.ws + rows * a.spitch;
            work += bytes;
            room -= bytes;
        }
        const Tiling t = tiling(rows, tokens, groups, room, c->num_cus);
        const int per = (groups + t.splits - 1) / t.splits, ns = (groups + per - 1) / per;
        a.splits = 4 * per;
        if (ns == 1) {
            dt_out == F32 ? tiles_t<SF32>(c, a, t.tile, 1, tail)
                          : dt_out == BF16 ? tiles_t<SBf16>(c, a, t.tile, 1, tail) : tiles_t<SF16>(c, a, t.tile, 1, tail);
            return true;
        }
        float *part = reinterpret_cast<float *>(work);
        a.y = part;
        a.ldy = rows;
        a.ysplit = tokens * rows;
        tiles_t<SF32>(c, a, t.tile, ns, tail);
        join_splits(c, part, ns, y, ldy, rows, tokens, dt_out);
        return true;
    }
} // namespace mg
