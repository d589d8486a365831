// MXFP4 for gfx950: rows in 4.25 bits an element, their quantizer and its
// inverse, and products with weights held so.
//
// The format is the OCP microscaling one: 32 consecutive elements of a row
// share a power of two, 2^(s - 127) with s one byte (e8m0; 255 is NaN), and each
// is a 4-bit code c: sign, two exponent bits, one mantissa bit (e2m1), worth
// 0 .5 1 1.5 2 3 4 6 with the sign. Codes are [rows, in / 2] bytes, element 2 i
// in the low four bits of byte i; scales [rows, in / 32].
#include "mg_device.hpp"
#include "mg_internal.hpp"
#include "mg_mxfp4.hpp"

namespace mg
{
    // ------------------------------------------------------------- quantizer
    // One scale a block: s = floor(log2 amax) - 2 + 127 within [0, 254], so that
    // amax, in [4, 8) of it, meets the largest code's 6 (the format's own rule: what
    // is past 6 becomes 6); codes are the nearest values, ties to the even code.
    // A block that holds an infinity or a NaN gets s = 255.
    // Lane L of a wave holds elements 8 L .. 8 L + 7 of 512, so a quad holds a block.
    template <class S>
    __global__ __launch_bounds__(256) void k_quantize_mxfp4(const typename S::raw *__restrict__ x, int64_t ldx, int64_t in,
                                                            uint32_t *__restrict__ qs, uint8_t *__restrict__ sc,
                                                            int64_t pieces)
    {
        const int64_t p = int64_t(blockIdx.x) * 256 + threadIdx.x; // eight elements of a row
        const bool live = p < pieces;
        const int64_t per = in / 8, r = live ? p / per : 0, at = live ? (p - r * per) * 8 : 0;
        const Mx8<S> v = mx_load8<S>(x + r * ldx + at);
        const uint32_t s = mx_scale_byte(mx_quad_max(v.amax()));
        if (!live) return;
        qs[p] = v.codes(s);
        if (p % 4 == 0) sc[p / 4] = uint8_t(s);
    }

    // ----------------------------------------------------------- dequantizer
    template <class SO>
    __global__ __launch_bounds__(256) void k_dequant_mxfp4(const uint32_t *__restrict__ qs, const uint8_t *__restrict__ sc,
                                                           typename SO::raw *__restrict__ out, int64_t pieces)
    {
        const int64_t p = int64_t(blockIdx.x) * 256 + threadIdx.x;
        if (p >= pieces) return;
        mx_store8<SO>(out + 8 * p, qs[p], sc[p >> 2]);
    }

    // -------------------------------------------------------------- products
    // y[t, o] = sum_i W[o, i] x[t, i] for a few tokens t. A work-group of NW waves
    // serves 16 RT weight rows and 16 TT tokens; its waves take chunks of 128
    // elements in turn, and their sums meet in LDS in wave order. Lane (n, c) holds
    // block 4 m + c, 16 bytes of codes, of weight row n and of token n: of a product
    // over 32 elements its eight, four times, or the whole operand of one over 128.
    struct MxArgs
    {
        const uint8_t *w, *ws, *x, *xs; // x: 16-bit rows, or codes with scales xs
        void *y;
        int64_t ldx, ldy, rows, T;
        int nblk; // in / 32
    };

    template <class A>
    struct MxTok // a token's operand of a chunk: 32 elements of 16 bits, or a block
    {
        Vec<uint32_t, 4> v[A::dt == kMxFp4 ? 1 : 4];
        uint32_t s;
    };

    // One chunk's products. 16-bit activations: the codes become bf16, exactly. Beside
    // f16 activations they become f16 where that is exact too (scales of 2^-23 to
    // 2^13, blocks of zeros, NaN), else the activations are split into two bf16 parts.
    template <class A, int RT, int TT>
    MG_DEV void mx_chunk(const Vec<uint32_t, 4> (&w)[RT], const uint32_t (&ws)[RT], const MxTok<A> (&x)[TT],
                         f32x4 (&acc)[RT][TT])
    {
        if constexpr (A::dt == kMxFp4) {
#pragma unroll
            for (int t = 0; t < RT; ++t)
#pragma unroll
                for (int u = 0; u < TT; ++u) acc[t][u] = mfma_mxfp4(w[t], ws[t], x[u].v[0], x[u].s, acc[t][u]);
        } else {
            bool wide = false; // f16: some block needs bf16's range
            if constexpr (A::dt == F16) {
                bool far = false;
#pragma unroll
                for (int t = 0; t < RT; ++t)
                    far |= ws[t] - 104u > 36u && ws[t] != 255u && ((w[t].v[0] | w[t].v[1] | w[t].v[2] | w[t].v[3]) & 0x77777777u) != 0;
                wide = __builtin_amdgcn_ballot_w64(far) != 0;
            }
#pragma unroll
            for (int t = 0; t < RT; ++t) {
                const float f = mx_scale(ws[t]);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if constexpr (A::dt == F16) {
                        if (!wide) {
                            const mxf16x8 wh = __builtin_bit_cast(mxf16x8, mx_f16(w[t].v[i], f));
#pragma unroll
                            for (int u = 0; u < TT; ++u)
                                acc[t][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wh, __builtin_bit_cast(mxf16x8, x[u].v[i]), acc[t][u], 0, 0, 0);
                            continue;
                        }
                    }
                    const bf16x8 wb = __builtin_bit_cast(bf16x8, mx_bf16(w[t].v[i], f));
#pragma unroll
                    for (int u = 0; u < TT; ++u) {
                        if constexpr (A::dt == F16) {
                            Vec<uint32_t, 4> hi, lo;
#pragma unroll
                            for (int k = 0; k < 4; ++k) mx_halves(x[u].v[i].v[k], hi.v[k], lo.v[k]);
                            acc[t][u] = mfma_bf16(wb, __builtin_bit_cast(bf16x8, lo), acc[t][u]);
                            acc[t][u] = mfma_bf16(wb, __builtin_bit_cast(bf16x8, hi), acc[t][u]);
                        } else {
                            acc[t][u] = mfma_bf16(wb, __builtin_bit_cast(bf16x8, x[u].v[i]), acc[t][u]);
                        }
                    }
                }
            }
        }
    }

    template <class A, class SO, int RT, int TT, int NW, int P>
    __global__ __launch_bounds__(64 * NW) void k_mxfp4_rows(MxArgs a)
    {
        constexpr bool MX = A::dt == kMxFp4;
        const int wv = __builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6)), lane = threadIdx.x & 63;
        const int n = lane & 15, c = lane >> 4;
        const int64_t r0 = int64_t(blockIdx.x) * (16 * RT), t0 = int64_t(blockIdx.y) * (16 * TT);
        const int nblk = a.nblk, chunks = (nblk + 3) / 4;
        const uint8_t *wp[RT], *sp[RT], *xp[TT], *xsp[TT];
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            const int64_t r = r0 + 16 * t + n, row = r < a.rows ? r : a.rows - 1;
            wp[t] = a.w + row * (16 * int64_t(nblk)) + 16 * c;
            sp[t] = a.ws + row * nblk + c;
        }
#pragma unroll
        for (int t = 0; t < TT; ++t) {
            const int64_t b = t0 + 16 * t + n, tok = b < a.T ? b : a.T - 1;
            if constexpr (MX) {
                xp[t] = a.x + tok * (16 * int64_t(nblk)) + 16 * c;
                xsp[t] = a.xs + tok * nblk + c;
            } else {
                xp[t] = a.x + (tok * a.ldx + 32 * c) * 2;
            }
        }
        Vec<uint32_t, 4> w[P][RT];
        uint32_t ws[P][RT];
        MxTok<A> x[P][TT];
        auto load = [&](int p, int m) {
            // a block past the row's end counts as zeros
            const bool in = 4 * m + c < nblk;
#pragma unroll
            for (int t = 0; t < RT; ++t) {
                w[p][t] = Vec<uint32_t, 4>{{0u, 0u, 0u, 0u}};
                ws[p][t] = 127u;
                if (in) {
                    w[p][t] = ld16_stream<uint32_t, 4>(reinterpret_cast<const uint32_t *>(wp[t] + 64 * int64_t(m)));
                    ws[p][t] = sp[t][4 * int64_t(m)];
                }
            }
#pragma unroll
            for (int t = 0; t < TT; ++t) {
                constexpr int NV = MX ? 1 : 4;
#pragma unroll
                for (int i = 0; i < NV; ++i) x[p][t].v[i] = Vec<uint32_t, 4>{{0u, 0u, 0u, 0u}};
                x[p][t].s = 127u;
                if (in) {
#pragma unroll
                    for (int i = 0; i < NV; ++i)
                        x[p][t].v[i] = *reinterpret_cast<const Vec<uint32_t, 4> *>(xp[t] + (MX ? 64 : 256) * int64_t(m) + 16 * i);
                    if constexpr (MX) x[p][t].s = xsp[t][4 * int64_t(m)];
                }
            }
        };
        f32x4 acc[RT][TT];
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
            for (int u = 0; u < TT; ++u) acc[t][u] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int p = 0; p < P; ++p)
            if (wv + p * NW < chunks) load(p, wv + p * NW);
        for (int m = wv; m < chunks; m += P * NW) {
#pragma unroll
            for (int p = 0; p < P; ++p) {
                if (m + p * NW >= chunks) break;
                mx_chunk<A, RT, TT>(w[p], ws[p], x[p], acc);
                if (m + (p + P) * NW < chunks) load(p, m + (p + P) * NW);
            }
        }
        __shared__ __align__(16) f32x4 part[NW][RT * TT][64];
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
            for (int u = 0; u < TT; ++u) part[wv][t * TT + u][lane] = acc[t][u];
        __syncthreads();
        // element i: weight row i % 16 of tile t, token b of tile u; lane (b, c) holds rows 4 c .. 4 c + 3
        typename SO::raw *y = static_cast<typename SO::raw *>(a.y);
        for (int i = threadIdx.x; i < 256 * RT * TT; i += 64 * NW) {
            const int r = i % (16 * RT), b = i / (16 * RT); // of the tokens 16 TT
            const int64_t o = r0 + r, tok = t0 + b;
            if (o >= a.rows || tok >= a.T) continue;
            const int l = 16 * ((r & 15) >> 2) + (b & 15), tile = (r >> 4) * TT + (b >> 4);
            float s = 0.0f;
#pragma unroll
            for (int k = 0; k < NW; ++k) s += part[k][tile][l][r & 3];
            y[tok * a.ldy + o] = SO::enc32(s);
        }
    }

    // ------------------------------------------------------------- launchers
    void launch_quantize_mxfp4(mg_ctx *c, const void *x, int64_t ldx, int64_t rows, int64_t in, int dt, uint8_t *qs, uint8_t *s)
    {
        need(rows >= 0 && in >= 0, "quantize_mxfp4: bad shape");
        need(in % 32 == 0, "quantize_mxfp4: input dim must be a multiple of 32 (got " + std::to_string(in) + ")");
        need(dt == BF16 || dt == F16 || dt == F32, "quantize_mxfp4: dtype must be bf16, f16 or f32");
        if (rows == 0 || in == 0) return;
        if (ldx == 0) ldx = in;
        need(x && qs && s, "quantize_mxfp4: NULL tensor");
        need(ldx >= in, "quantize_mxfp4: row stride smaller than a row");
        need(aligned16(x) && ldx % (16 / dt_size(dt)) == 0 && reinterpret_cast<uintptr_t>(qs) % 4 == 0,
             "quantize_mxfp4: rows must be 16-byte and codes 4-byte aligned");
        need(rows <= (int64_t(1) << 38) / in, "quantize_mxfp4: tensor too large");
        const int64_t pieces = rows * (in / 8);
        auto go = [&](auto s_) {
            using S = decltype(s_);
            hipLaunchKernelGGL(k_quantize_mxfp4<S>, dim3(unsigned((pieces + 255) / 256)), dim3(256), 0, c->stream,
                               static_cast<const typename S::raw *>(x), ldx, in, reinterpret_cast<uint32_t *>(qs), s, pieces);
            check_launch("k_quantize_mxfp4");
        };
        dt == BF16 ? go(SBf16{}) : dt == F16 ? go(SF16{}) : go(SF32{});
    }

    void launch_dequant_mxfp4(mg_ctx *c, const uint8_t *qs, const uint8_t *s, void *out, int64_t rows, int64_t in, int dt)
    {
        need(rows >= 0 && in >= 0, "dequant_mxfp4: bad shape");
        need(in % 32 == 0, "dequant_mxfp4: input dim must be a multiple of 32 (got " + std::to_string(in) + ")");
        need(dt == BF16 || dt == F16 || dt == F32, "dequant_mxfp4: output dtype must be bf16, f16 or f32");
        if (rows == 0 || in == 0) return;
        need(qs && s && out, "dequant_mxfp4: NULL tensor");
        need(aligned16(out) && reinterpret_cast<uintptr_t>(qs) % 4 == 0,
             "dequant_mxfp4: output must be 16-byte and codes 4-byte aligned");
        need(rows <= (int64_t(1) << 38) / in, "dequant_mxfp4: tensor too large");
        const int64_t pieces = rows * (in / 8);
        auto go = [&](auto so) {
            using SO = decltype(so);
            hipLaunchKernelGGL(k_dequant_mxfp4<SO>, dim3(unsigned((pieces + 255) / 256)), dim3(256), 0, c->stream,
                               reinterpret_cast<const uint32_t *>(qs), s, static_cast<typename SO::raw *>(out), pieces);
            check_launch("k_dequant_mxfp4");
        };
        dt == BF16 ? go(SBf16{}) : dt == F16 ? go(SF16{}) : go(SF32{});
    }

    namespace
    {
        template <class A, class SO>
        void go_rows(mg_ctx *c, const MxArgs &a)
        {
            auto go = [&](auto kern, int64_t rt, int64_t tt, int nw) {
                const int64_t gx = (a.rows + 16 * rt - 1) / (16 * rt), gy = (a.T + 16 * tt - 1) / (16 * tt);
                need(gx < (int64_t(1) << 31) && gy <= 65535, "mxfp4 product: too many rows or tokens");
                hipLaunchKernelGGL(kern, dim3(unsigned(gx), unsigned(gy)), dim3(unsigned(64 * nw)), 0, c->stream, a);
                check_launch("k_mxfp4_rows");
            };
            if (a.T <= 16)
                go(k_mxfp4_rows<A, SO, 1, 1, 4, 2>, 1, 1, 4);
            else if (a.T <= 32)
                go(k_mxfp4_rows<A, SO, 2, 2, 4, 1>, 2, 2, 4);
            else
                go(k_mxfp4_rows<A, SO, 2, 4, 4, 1>, 2, 4, 4);
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
        need(in <= (int64_t(1) << 30), "gemv_mxfp4: input dim too large");
        const MxArgs a{qs, s, static_cast<const uint8_t *>(x), nullptr, y, ldx, ldy, rows, batch, int(in / 32)};
        if (dt == BF16)
            dt_out == F32 ? go_rows<SBf16, SF32>(c, a) : go_rows<SBf16, SBf16>(c, a);
        else
            dt_out == F32 ? go_rows<SF16, SF32>(c, a) : go_rows<SF16, SF16>(c, a);
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
        need(in <= (int64_t(1) << 30), "gemm_mxfp4: input dim too large");
        const MxArgs a{qs, s, aq, as, y, 0, ldy, rows, tokens, int(in / 32)};
        if (dt_out == F32)
            go_rows<SMxFp4, SF32>(c, a);
        else
            dt_out == BF16 ? go_rows<SMxFp4, SBf16>(c, a) : go_rows<SMxFp4, SF16>(c, a);
    }
} // namespace mg
