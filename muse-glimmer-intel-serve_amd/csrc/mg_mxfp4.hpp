// MXFP4 on the device: gfx950's conversions of e2m1 codes with a power-of-two
// scale, and products of codes on the matrix cores. A conversion's scale operand
// is an f32 whose exponent field alone counts: the e8m0 byte shifted there. All
// are exact or round once, to nearest even, for every scale (2^-127 and NaN, byte
// 255, among them), with subnormals; a quantized value past 6 becomes 6.
#pragma once

#include <type_traits>

#include "mg_device.hpp"

namespace mg
{
    constexpr int kMxFp4 = 16; // among the storage formats' dt: codes with scales
    struct SMxFp4
    {
        static constexpr int dt = kMxFp4;
    };

    typedef _Float16 mxf16x8 __attribute__((ext_vector_type(8)));
    typedef __bf16 mxbf16x2 __attribute__((ext_vector_type(2)));
    typedef _Float16 mxf16x2 __attribute__((ext_vector_type(2)));

    MG_DEV float mx_scale(uint32_t s) { return __builtin_bit_cast(float, s << 23); }

    // the scale byte of a block whose largest magnitude has the f32 bits `amax`
    MG_DEV uint32_t mx_scale_byte(uint32_t amax)
    {
        const uint32_t e = amax >> 23;
        return e == 255u ? 255u : e > 2u ? e - 2u : 0u;
    }
    MG_DEV uint32_t mx_quad_max(uint32_t v)
    {
        v = max(v, dpp_mov<0xB1, 0xf>(v, v)); // quad_perm [1,0,3,2]
        v = max(v, dpp_mov<0x4E, 0xf>(v, v)); // quad_perm [2,3,0,1]
        return v;
    }

    // eight elements on their way to codes; amax() gives f32 bits (an infinity or a NaN: the largest)
    template <class S>
    struct Mx8
    {
        Vec<uint32_t, S::dt == F32 ? 8 : 4> v;
        MG_DEV uint32_t amax() const
        {
            uint32_t m = 0;
            if constexpr (S::dt == F32) {
#pragma unroll
                for (int i = 0; i < 8; ++i) m = max(m, v.v[i] & 0x7fffffffu);
                return m;
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) m = pk_max_u16(m, v.v[i] & 0x7fff7fffu);
                m = max(m & 0xffffu, m >> 16);
                return S::dt == BF16 ? m << 16 : __builtin_bit_cast(uint32_t, f16_f32(uint16_t(m)));
            }
        }
        MG_DEV uint32_t codes(uint32_t s) const
        {
            const float f = mx_scale(s);
            uint32_t q = 0;
            if constexpr (S::dt == F32) {
                auto at = [&](int i) { return __builtin_bit_cast(float, v.v[i]); };
                q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, at(0), at(1), f, 0);
                q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, at(2), at(3), f, 1);
                q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, at(4), at(5), f, 2);
                q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, at(6), at(7), f, 3);
            } else if constexpr (S::dt == BF16) {
                auto at = [&](int i) { return __builtin_bit_cast(mxbf16x2, v.v[i]); };
                q = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q, at(0), f, 0);
                q = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q, at(1), f, 1);
                q = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q, at(2), f, 2);
                q = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q, at(3), f, 3);
            } else {
                auto at = [&](int i) { return __builtin_bit_cast(mxf16x2, v.v[i]); };
                q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(q, at(0), f, 0);
                q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(q, at(1), f, 1);
                q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(q, at(2), f, 2);
                q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(q, at(3), f, 3);
            }
            return q;
        }
    };
    template <class S>
    MG_DEV Mx8<S> mx_load8(const typename S::raw *p)
    {
        Mx8<S> x;
        if constexpr (S::dt == F32) {
            const Vec<uint32_t, 4> a = ld16_stream<uint32_t, 4>(reinterpret_cast<const uint32_t *>(p));
            const Vec<uint32_t, 4> b = ld16_stream<uint32_t, 4>(reinterpret_cast<const uint32_t *>(p) + 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) x.v.v[i] = a.v[i], x.v.v[4 + i] = b.v[i];
        } else {
            x.v = ld16_stream<uint32_t, 4>(reinterpret_cast<const uint32_t *>(p));
        }
        return x;
    }

    // eight codes as bf16 or f16 pairs, as f32 (a NaN scale gives the format's one NaN)
    MG_DEV Vec<uint32_t, 4> mx_bf16(uint32_t q, float f)
    {
        return Vec<uint32_t, 4>{{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, f, 0)),
                                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, f, 1)),
                                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, f, 2)),
                                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(q, f, 3))}};
    }
    MG_DEV Vec<uint32_t, 4> mx_f16(uint32_t q, float f)
    {
        return Vec<uint32_t, 4>{{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(q, f, 0)),
                                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(q, f, 1)),
                                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(q, f, 2)),
                                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(q, f, 3))}};
    }
    // The same less 2^2, exactly: 6 2^127 of scale 254 is past bf16's largest value. (What is left of the smallest scales' 2^-128
    // is a subnormal that bf16 holds.)
    MG_DEV Vec<uint32_t, 4> mx_bf16_quarter(uint32_t q, uint32_t s)
    {
        Vec<uint32_t, 4> w = mx_bf16(q, mx_scale(s == 255u ? s : s > 2u ? s - 2u : 0u));
        const float f = s == 0u ? 0.25f : s == 1u ? 0.5f : 1.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) w.v[i] = bf_pack(bf_lo(w.v[i]) * f, bf_hi(w.v[i]) * f);
        return w;
    }
    // f16 pairs of a word, times a power of two, as sums of two bf16 pairs: 11 bits are 8 and 3 (an infinity or a NaN is its
    // high part)
    MG_DEV void mx_halves(uint32_t w, uint32_t &hi, uint32_t &lo, float f = 1.0f)
    {
        const float a = f16_f32(uint16_t(w)) * f, b = f16_f32(uint16_t(w >> 16)) * f;
        hi = bf_pack(a, b);
        lo = bf_pack(__builtin_isfinite(a) ? a - bf_lo(hi) : 0.0f, __builtin_isfinite(b) ? b - bf_hi(hi) : 0.0f);
    }

    template <class SO>
    MG_DEV void mx_store8(typename SO::raw *out, uint32_t q, uint32_t s)
    {
        const float f = mx_scale(s);
        if constexpr (SO::dt == F32) {
            typedef float f32x2 __attribute__((ext_vector_type(2)));
            f32x2 v[4];
            v[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, f, 0);
            v[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, f, 1);
            v[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, f, 2);
            v[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, f, 3);
            st16_stream<float, 4>(out, Vec<float, 4>{{v[0][0], v[0][1], v[1][0], v[1][1]}});
            st16_stream<float, 4>(out + 4, Vec<float, 4>{{v[2][0], v[2][1], v[3][0], v[3][1]}});
        } else {
            Vec<uint32_t, 4> w = SO::dt == BF16 ? mx_bf16(q, f) : mx_f16(q, f);
            if (s == 255u) // the library's NaN (the conversion's has a sign)
                w = SO::dt == BF16 ? Vec<uint32_t, 4>{{0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u}}
                                   : Vec<uint32_t, 4>{{0x7e007e00u, 0x7e007e00u, 0x7e007e00u, 0x7e007e00u}};
            st16_stream<uint32_t, 4>(reinterpret_cast<uint32_t *>(out), w);
        }
    }

    // ds_read_b64_tr_b4: within each 16-lane group, lane i receives four-bit element i of the 8-byte pieces
    // addressed by lanes 0 .. 15, lane j's in place j
    MG_DEV Vec<uint32_t, 2> lds_read_tr4(const char *p)
    {
        typedef int i32x2 __attribute__((ext_vector_type(2)));
        typedef __attribute__((address_space(3))) i32x2 lds_i32x2;
        return __builtin_bit_cast(Vec<uint32_t, 2>, __builtin_amdgcn_ds_read_tr4_b64_v2i32((lds_i32x2 *)(p)));
    }

    // f(0), f(1) .. of compile-time numbers
    template <int I, int N, class F>
    MG_DEV void each(F f)
    {
        if constexpr (I < N) {
            f(std::integral_constant<int, I>{});
            each<I + 1, N>(f);
        }
    }

    // 64 lanes' 16 bytes (or one, as a word) from base + off, each lane its own, to LDS at `to` + 16 (or 4) * lane.
    // (The compiler's own form would make every LDS read wait for all of them; here the kernel counts.) A load may read
    // scalar registers five wait states after a vector instruction wrote them, m0 one after a scalar one; the compiler
    // does not look in here: the move of m0 is one and s_nop 3 four. (m0 is reserved: it cannot be named as overwritten.
    // The compiler writes it anew where it wants it, which it does nowhere in these kernels: the host test of the built
    // code looks.)
    template <int BYTES = 16>
    MG_DEV void lds_load(const uint8_t *base, uint32_t off, uint32_t to)
    {
        // (uniform, but the compiler keeps some selections of them in vector registers)
        const uint64_t b = reinterpret_cast<uint64_t>(base);
        const uint64_t sb = uint64_t(uint32_t(__builtin_amdgcn_readfirstlane(int(b >> 32)))) << 32 |
                            uint32_t(__builtin_amdgcn_readfirstlane(int(uint32_t(b))));
        to = uint32_t(__builtin_amdgcn_readfirstlane(int(to)));
        if constexpr (BYTES == 16)
            __asm__ volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(off), "s"(sb) : "memory");
        else
            __asm__ volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tglobal_load_lds_ubyte %1, %2" ::"s"(to), "v"(off), "s"(sb) : "memory");
    }
    // the same from any address of each lane; 4 bytes, or two as a word, at `to` + 4 * lane
    template <int BYTES = 16>
    MG_DEV void lds_load_at(const void *p, uint32_t to)
    {
        to = uint32_t(__builtin_amdgcn_readfirstlane(int(to)));
        if constexpr (BYTES == 16)
            __asm__ volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(to), "v"(p) : "memory");
        else if constexpr (BYTES == 4)
            __asm__ volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(to), "v"(p) : "memory");
        else
            __asm__ volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_ushort %1, off" ::"s"(to), "v"(p) : "memory");
    }
    MG_DEV uint32_t lds_address(const char *p) { return uint32_t(uintptr_t((__attribute__((address_space(3))) const char *)p)); }

    // f32 sums of 16 x 16 products over 128 codes each: lane l = 16 c + n holds block c (32 codes, 16 bytes) of
    // row n of A (column n of B) and its scale byte; C as the other 16 x 16 products'
    MG_DEV f32x4 mfma_mxfp4(Vec<uint32_t, 4> a, uint32_t sa, Vec<uint32_t, 4> b, uint32_t sb, f32x4 c)
    {
        typedef int i32x8 __attribute__((ext_vector_type(8)));
        const i32x8 av = {int(a.v[0]), int(a.v[1]), int(a.v[2]), int(a.v[3]), 0, 0, 0, 0};
        const i32x8 bv = {int(b.v[0]), int(b.v[1]), int(b.v[2]), int(b.v[3]), 0, 0, 0, 0};
        return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(av, bv, c, 4, 4, 0, int(sa), 0, int(sb));
    }
} // namespace mg
