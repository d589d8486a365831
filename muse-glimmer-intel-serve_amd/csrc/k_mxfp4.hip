// MXFP4 for gfx950: rows in 4.25 bits an element, their quantizer and its inverse.
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
    // Lane L of a wave holds elements 8 L .. 8 L + 7 of 512, so a quad holds a block, and two such pieces. Bound by HBM:
    // [25600, 5120] bf16, 332 MB, 51 us, 6.5 TB/s as a copy (one piece a lane 54; with a division for every lane's row, now
    // taken only where rows are not dense, 59). The dequantizer takes 46.
    template <class S>
    __global__ __launch_bounds__(256) void k_quantize_mxfp4(const typename S::raw *__restrict__ x, int64_t ldx, int64_t in,
                                                            uint32_t *__restrict__ qs, uint8_t *__restrict__ sc,
                                                            int64_t pieces)
    {
        constexpr int N = 2;
        const int64_t p0 = int64_t(blockIdx.x) * (256 * N) + threadIdx.x; // eight elements of a row each
        Mx8<S> v[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int64_t p = p0 + 256 * i;
            int64_t at = p < pieces ? 8 * p : 0;
            if (ldx != in) at += at / in * (ldx - in);
            v[i] = mx_load8<S>(x + at);
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int64_t p = p0 + 256 * i;
            const uint32_t s = mx_scale_byte(mx_quad_max(v[i].amax()));
            if (p >= pieces) return;
            qs[p] = v[i].codes(s);
            if (p % 4 == 0) sc[p / 4] = uint8_t(s);
        }
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
        need(launchable((pieces + 511) / 512, 256), "quantize_mxfp4: tensor too large");
        auto go = [&](auto s_) {
            using S = decltype(s_);
            hipLaunchKernelGGL(k_quantize_mxfp4<S>, dim3(unsigned((pieces + 511) / 512)), dim3(256), 0, c->stream,
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
        need(launchable((pieces + 255) / 256, 256), "dequant_mxfp4: tensor too large");
        auto go = [&](auto so) {
            using SO = decltype(so);
            hipLaunchKernelGGL(k_dequant_mxfp4<SO>, dim3(unsigned((pieces + 255) / 256)), dim3(256), 0, c->stream,
                               reinterpret_cast<const uint32_t *>(qs), s, static_cast<typename SO::raw *>(out), pieces);
            check_launch("k_dequant_mxfp4");
        };
        dt == BF16 ? go(SBf16{}) : dt == F16 ? go(SF16{}) : go(SF32{});
    }
} // namespace mg
