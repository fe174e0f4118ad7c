// Microscaled FP4: the two formats, the layout of their block scales, and the quantize of one block.
//
// A row of k values is stored as k / 2 bytes of e2m1 codes (the even element in the low nibble) and one scale byte per block:
//   nvfp4  blocks of 16, scale e4m3 (never negative), and a tensor scale g, a power of two, beside both:  value = code * s * g
//   mxfp4  blocks of 32, scale e8m0, a power of two:                                                      value = code * s
// Block scales lie in atoms of 512 bytes, 128 rows x 4 consecutive blocks, in the order in which tcgen05.cp spreads them over tensor
// memory: byte (row % 32) * 16 + (row % 128) / 32 * 4 + block % 4; the atoms of 128 rows follow each other along k, then the next 128 rows.
// Blocks of a row beyond k (k is a multiple of 32, an atom spans 64 or 128 values) have scale 0; rows beyond the last are never read
// into a result and stay as they were.
#pragma once

#include "common.cuh"

namespace lyraq {

__host__ __device__ constexpr int fp4_group(int format) { return format == LYRAQ_NVFP4 ? 16 : 32; }
// atoms along k, and the values of a row one atom scales
__host__ __device__ constexpr int    fp4_atom_k(int format) { return 4 * fp4_group(format); }
__host__ __device__ constexpr size_t fp4_atoms(size_t k, int format) { return (k + (size_t)fp4_atom_k(format) - 1) / (size_t)fp4_atom_k(format); }

__host__ __device__ inline size_t fp4_scale_offset(size_t row, size_t atoms, size_t atom)
{
    return ((row >> 7) * atoms + atom) * 512 + (row & 31) * 16 + ((row & 127) >> 5) * 4;
}

// Eight floats -> eight e2m1 codes (nearest, ties to the even code, saturating at 6), element j at bits 4 j.
__device__ __forceinline__ uint32_t f32x8_to_e2m1x8(const float* v)
{
    uint32_t r;
    asm("{\n\t"
        ".reg .b8 b0, b1, b2, b3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
        "mov.b32 %0, {b0, b1, b2, b3};\n\t"
        "}\n"
        : "=r"(r)
        : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return r;
}

// 1 / v, off by an ulp at most.
__device__ __forceinline__ float rcp_approx(float v)
{
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}

// A power of two that brings a divisor to where neither its reciprocal nor a remainder over- or underflows.  Dividends are multiplied by it too; what
// that over- or underflows has a quotient that saturates or rounds to zero.
__device__ __forceinline__ float fp4_range(float v) { return v < 7.9e-31f ? 1.2089258e24f : v > 1.2e30f ? 8.271806e-25f : 1.0f; }   // 2^-100, 2^80, 2^100, 2^-80

// What the blocks of a tensor share: its scale g, and with c = fp4_range(g): c, 6 g c and about 1 / (6 g c).
struct Fp4Tensor {
    float g, c, g6, r6;
};
template<int FORMAT> __device__ __forceinline__ Fp4Tensor fp4_tensor(const float* tensor_scale)
{
    Fp4Tensor t{1.0f, 1.0f, 6.0f, 0.0f};
    if (FORMAT == LYRAQ_NVFP4) {
        t.g  = tensor_scale != nullptr ? ld_f32(tensor_scale) : 1.0f;
        t.c  = fp4_range(t.g);
        t.g6 = 6.0f * (t.g * t.c);
        t.r6 = t.g6 > 0.0f ? rcp_approx(t.g6) : 0.0f;
    }
    return t;
}

// Quotients without a division: q0 = a r with r about 1 / b, then q0 + (a - q0 b) r.  The remainder is exact, so what is rounded to the result is off
// by 2^-45 of it.  Here b has few significant bits (three times or a four-bit number times a power of two), and so does every tie of the number
// formats times b: a quotient that is a tie comes out as it, one that is not lies more than half an ulp and 2^-31 away from any.  So
// roundings decide as the exact quotient would, ties included.
//
// Scale of one block from the largest magnitude in it: the stored byte and what the block's values are divided by.
struct Fp4Block {
    uint32_t code;
    float    t;      // 0: every code is 0
    float    r;      // 1 / t: exact for mxfp4, about so for nvfp4; 0 where t is
    bool     plain;  // finite, and nothing over- or underflows on the way of the values' quotients
};

// amax_bits: the largest |x| of the block as fp32 bits, taken as an integer maximum, so that a NaN beats an infinity and both beat every
// number.  A block that holds either gets the scale NaN and zero codes: all of it reads back as NaN.
//   nvfp4: s = e4m3(amax / (6 g)), t = s g;  mxfp4: s = t = 2^(floor(log2 amax) - 2), at least 2^-127
template<int FORMAT> __device__ __forceinline__ Fp4Block fp4_block(uint32_t amax_bits, const Fp4Tensor& s)
{
    Fp4Block b;
    if (amax_bits >= 0x7f800000u) {
        b.code  = FORMAT == LYRAQ_NVFP4 ? 0x7fu : 0xffu;
        b.t     = 0.0f;
        b.r     = 0.0f;
        b.plain = false;
        return b;
    }
    if (FORMAT == LYRAQ_NVFP4) {
        const float amax  = __uint_as_float(amax_bits);
        const float a     = fminf(amax * s.c, s.g6 * 1024.0f);   // saturates at 448
        const float q0    = a * s.r6;
        const float ratio = fmaf(fmaf(-q0, s.g6, a), s.r6, q0);
        b.code = f32x2_to_e4m3x2(ratio, 0.0f) & 0xffu;
        // e4m3 -> fp32: the code's seven bits under fp16's exponent read 2^-8 times its value, subnormals included
        b.t     = __half2float(__ushort_as_half((unsigned short)(b.code << 7))) * 256.0f * s.g;
        b.r     = b.t > 0.0f ? rcp_approx(b.t) : 0.0f;
        b.plain = b.t == 0.0f || (b.t >= 7.9e-31f && b.t <= 1.2e30f && amax <= b.t * 1048576.0f);
    } else {
        const uint32_t e = amax_bits >> 23;                                  // biased; 0 for subnormals
        b.code           = e > 2u ? e - 2u : 0u;
        b.t              = b.code != 0u ? __uint_as_float(b.code << 23) : __uint_as_float(0x00400000u);
        // 2^-(code - 127) is a number for every code (2^127 down to 2^-125), so the product with it is the quotient itself
        b.r     = __uint_as_float((254u - b.code) << 23);
        b.plain = true;
    }
    return b;
}

// The codes of eight values of a block.
template<int FORMAT> __device__ __forceinline__ uint32_t fp4_encode8(const float* x, const Fp4Block& b)
{
    float q[8], t = b.t, r = b.r;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        q[j] = x[j];
    }
    if (FORMAT == LYRAQ_NVFP4 && __builtin_expect(!b.plain, 0)) {   // no divisions here either: they are long, and every launch would fetch them on its way past
        const float c = fp4_range(t);
        t *= c;
        r = t > 0.0f ? rcp_approx(t) : 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            q[j] = t > 0.0f ? fminf(fmaxf(q[j] * c, t * -1048576.0f), t * 1048576.0f) : 0.0f;
        }
    }
    // with t = r = 0 every quotient comes out as 0
    const float2 r2 = make_float2(r, r);
    const float2 m2 = make_float2(-t, -t);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float2 v = make_float2(q[2 * j], q[2 * j + 1]);
        float2       p = mul_f32x2(v, r2);
        if (FORMAT == LYRAQ_NVFP4) {
            p = fma_f32x2(fma_f32x2(p, m2, v), r2, p);
        }
        q[2 * j]     = p.x;
        q[2 * j + 1] = p.y;
    }
    const uint32_t codes = f32x8_to_e2m1x8(q);
    return FORMAT == LYRAQ_NVFP4 || b.plain ? codes : 0u;   // mxfp4: not plain is not finite
}

// Largest magnitude of a 16-byte vector of T, as fp32 bits (see fp4_block).
template<typename T> __device__ __forceinline__ uint32_t amax_bits_of(const Vec16& v);
template<> __device__ __forceinline__ uint32_t amax_bits_of<float>(const Vec16& v)
{
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        m = max(m, v.w[i] & 0x7fffffffu);
    }
    return m;
}
// Of two 16-bit pairs the larger magnitudes, NaN before all (the sign is of no use).
template<typename T> __device__ __forceinline__ uint32_t max_abs2(uint32_t a, uint32_t b);
template<> __device__ __forceinline__ uint32_t max_abs2<__nv_bfloat16>(uint32_t a, uint32_t b)
{
    uint32_t r;
    asm("max.NaN.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
template<> __device__ __forceinline__ uint32_t max_abs2<__half>(uint32_t a, uint32_t b)
{
    uint32_t r;
    asm("max.NaN.xorsign.abs.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
template<typename T> __device__ __forceinline__ uint32_t amax16_of(const Vec16& v)
{
    const uint32_t m = max_abs2<T>(max_abs2<T>(v.w[0], v.w[1]), max_abs2<T>(v.w[2], v.w[3])) & 0x7fff7fffu;
    return max(m & 0xffffu, m >> 16);
}
template<> __device__ __forceinline__ uint32_t amax_bits_of<__nv_bfloat16>(const Vec16& v) { return amax16_of<__nv_bfloat16>(v) << 16; }
template<> __device__ __forceinline__ uint32_t amax_bits_of<__half>(const Vec16& v)
{
    // half -> float keeps order, infinities and NaN
    return __float_as_uint(__half2float(__ushort_as_half((unsigned short)amax16_of<__half>(v)))) & 0x7fffffffu;
}

// A block's vectors -> its codes, eight to a word, and its scale byte.
template<typename T, int FORMAT> __device__ __forceinline__ uint32_t fp4_encode_block(const Vec16* v, const Fp4Tensor& tensor, uint32_t* words)
{
    constexpr int kGroup = fp4_group(FORMAT);
    constexpr int kV     = kGroup * (int)sizeof(T) / 16;
    uint32_t      amax   = 0;
#pragma unroll
    for (int a = 0; a < kV; ++a) {
        amax = max(amax, amax_bits_of<T>(v[a]));
    }
    const Fp4Block blk = fp4_block<FORMAT>(amax, tensor);
#pragma unroll
    for (int a = 0; a < kGroup / 8; ++a) {
        float f[8];
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                f[e] = __uint_as_float(v[2 * a + (e >> 2)].w[e & 3]);
            }
        } else {
            unpack8<T>(v[a], f);
        }
        words[a] = fp4_encode8<FORMAT>(f, blk);
    }
    return blk.code;
}

// 32 consecutive values of a row, two blocks or one: their codes, and their scale bytes from the lowest on.  SHORT: one block after the other by the
// same instructions, for a kernel that runs them once: [1, 3072, 12288] 6.9 us instead of 7.1, [1, 256, 256] 2.75 instead of 2.9.
template<typename T, int FORMAT, bool SHORT> __device__ __forceinline__ uint32_t fp4_encode32(Vec16* v, const Fp4Tensor& tensor, Vec16& o)
{
    if constexpr (FORMAT == LYRAQ_MXFP4) {
        return fp4_encode_block<T, FORMAT>(v, tensor, o.w);
    } else {
        constexpr int kV   = (int)sizeof(T);   // vectors of a block
        uint32_t      code = 0;
        if constexpr (SHORT) {
#pragma unroll 1
            for (int b = 0; b < 2; ++b) {
                o.w[0] = o.w[2];
                o.w[1] = o.w[3];
                code   = code >> 8 | fp4_encode_block<T, FORMAT>(v, tensor, o.w + 2) << 8;
#pragma unroll
                for (int a = 0; a < kV; ++a) {
                    v[a] = v[a + kV];
                }
            }
        } else {
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                code |= fp4_encode_block<T, FORMAT>(v + b * kV, tensor, o.w + 2 * b) << (8 * b);
            }
        }
        return code;
    }
}

// What lyraq_quant_fp4 asks of its arguments (fp4_quant.cu).
int check_fp4(const void* q, const void* sf, const void* x, int dtype, size_t ldx, int format, size_t rows, size_t k);

}  // namespace lyraq
