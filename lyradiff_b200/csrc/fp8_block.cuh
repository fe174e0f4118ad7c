// FP8 with a scale for each block of 128 values: the format, the quantize of a block, and the problem its products share.
//
// A row of k values is stored as k bytes of e4m3 codes (k a multiple of 16) and one fp32 scale for each 128 of them, the last block of a row
// being shorter where k is no multiple of 128; a weight has one scale for each 128 rows x 128 columns.  value = code * s.
//   s = fl(max|x| / 448), at least 2^-100; code = e4m3(fl(x / s))
// The least scale keeps a block of zeros from a division by 0, and the arithmetic of the quotients among normal numbers; blocks below 448 * 2^-100 = 3.5e-28 are
// held in steps of 2^-109.
// with fl rounding to fp32.  A block that holds an infinity or a NaN gets the scale NaN and zero codes: all of it reads back as NaN.
#pragma once

#include "common.cuh"
#include "fp4.cuh"
#include "views.h"

namespace lyraq {
namespace fp8b {

constexpr int   kBlock     = 128;
constexpr int   kMaxSize   = 0x7fffff00;      // of m, n and k: row, column and block numbers of a last tile stay within 31 bits
constexpr float kLeast     = 7.888609052210118e-31f;   // 2^-100
constexpr int   kFewRows   = 16;              // most rows of X that gemm_fp8_block_rows.cu takes

__host__ __device__ constexpr size_t blocks_of(size_t k) { return (k + kBlock - 1) / kBlock; }
// pitch of a block's scales where the quantizer and the product share a workspace: [blocks of k][rows], whole 16-byte vectors
__host__ __device__ constexpr size_t scale_pitch(size_t rows) { return (rows + 3) / 4 * 4; }

// Where the scales of X lie: element (row, block) at row * row_step + block * block_step.
struct Scales {
    const float* p;
    size_t       row_step, block_step;
};

// The left operand: codes with their scales, or (codes null) rows of a 16- or 32-bit type that the few-row kernel quantizes itself.
struct Input {
    const uint8_t* codes;
    Scales         scales;
    const void*    x;
    int            dtype;
    size_t         ldx;
};

struct GemmParams {
    int           M, N, K;
    int           m_tiles, n_tiles;
    int           splits;     // CTAs along K
    unsigned int* status;
    void*         C;          // [M, N] of c_dtype: F16, BF16 or F32
    int           c_dtype;
    int           tma_store;  // 16-bit output whose row pitch allows TMA stores
    Scales        xs;
    const float*  ws;         // [blocks of N][blocks of K]
    const void*   bias;       // [N] of c_dtype or null
    const void*   residual;   // [M, N] of c_dtype or null
    float         beta;
    int           gelu;
    unsigned long long wait_limit_ns;   // of the tiled kernel's waits
    int           stalled_rank;         // test hook: this CTA of a cluster issues no loads there (-1: none)
};

// What a block's values are divided by, and how.
struct Divisor {
    float s;      // the scale
    float c;      // a power of two that keeps the remainders of the division normal numbers: dividend and divisor are multiplied by it
    float t, r;   // s c, and fl(1 / (s c)); r = 0 where the block is not finite, which makes every code 0
};

// amax_bits: the largest |x| of the block as fp32 bits, taken as an integer maximum, so that a NaN beats an infinity and both beat every number.
__device__ __forceinline__ Divisor divisor_of(uint32_t amax_bits)
{
    Divisor d;
    if (amax_bits >= 0x7f800000u) {
        d.s = __uint_as_float(0x7fc00000u);
        d.c = 0.0f;
        d.t = 1.0f;
        d.r = 0.0f;
        return d;
    }
    d.s = fmaxf(__fdiv_rn(__uint_as_float(amax_bits), 448.0f), kLeast);
    d.c = d.s < 8.673617379884035e-19f ? 1.8446744073709552e19f : 1.0f;   // 2^-60, 2^64
    d.t = d.s * d.c;
    d.r = __frcp_rn(d.t);
    return d;
}

// Codes of eight values.  The quotient is rounded to fp32 as a division rounds it, so that a quotient on a tie of e4m3 comes out as that tie; it
// is found without one, by corrections with the remainder (P. Markstein, "Computation of elementary functions on the IBM RISC System/6000 processor",
// 1990: r within half an ulp of 1 / t).  Two corrections round any quotient correctly.
// One is enough for 16-bit values (SHORT).  Behind it the quotient is off by 2^-45 before it is rounded, which could only matter if x lay within 2^-45 of t (q + ulp / 2) for
// a tie q of e4m3.  In units of the last places, with q = a 2^19 (a of five bits) and T the 24 bits of t, that is T (a 2^20 + 1) within 16 of a number of 11
// bits times 2^36, so T within 16 of a multiple of 2^20.  T is the quotient of an 11-bit number by 7, shifted: either its bits repeat every three places, and 15 equal
// ones never follow one another, or it has nine bits, and is a multiple of 2^15 (too far from one of 2^20) or b 2^20, and T (a 2^20 + 1) is b 2^20 off.
template<bool SHORT> __device__ __forceinline__ uint2 encode8(const float* x, const Divisor& d)
{
    const float2 r2 = make_float2(d.r, d.r), m2 = make_float2(-d.t, -d.t), c2 = make_float2(d.c, d.c);
    uint32_t     h[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        float2 v = make_float2(x[2 * j], x[2 * j + 1]);
        if (__builtin_expect(d.c != 1.0f, 0)) {
            // a block that is not finite: its values are replaced, not multiplied, so that no NaN reaches a code
            v = d.r == 0.0f ? make_float2(0.0f, 0.0f) : mul_f32x2(v, c2);
        }
        float2 q = mul_f32x2(v, r2);
        q        = fma_f32x2(fma_f32x2(q, m2, v), r2, q);
        if (!SHORT) {
            q = fma_f32x2(fma_f32x2(q, m2, v), r2, q);
        }
        h[j] = f32x2_to_e4m3x2(q.x, q.y);
    }
    return make_uint2(h[0] | h[1] << 16, h[2] | h[3] << 16);
}

// 16 values of a lane's: T vectors -> their largest magnitude (fp32 bits)
template<typename T> __device__ __forceinline__ uint32_t amax16_values(const Vec16* v)
{
    uint32_t m = 0;
#pragma unroll
    for (int a = 0; a < (int)sizeof(T); ++a) {
        m = max(m, amax_bits_of<T>(v[a]));
    }
    return m;
}
// ... and their codes
template<typename T> __device__ __forceinline__ Vec16 encode16(const Vec16* v, const Divisor& d)
{
    Vec16 o;
#pragma unroll
    for (int a = 0; a < 2; ++a) {
        float f[8];
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                f[e] = __uint_as_float(v[2 * a + (e >> 2)].w[e & 3]);
            }
        } else {
            unpack8<T>(v[a], f);
        }
        const uint2 w  = encode8<sizeof(T) == 2>(f, d);
        o.w[2 * a]     = w.x;
        o.w[2 * a + 1] = w.y;
    }
    return o;
}

int check_quant(const void* q, const void* scale, const void* x, int dtype, size_t ldx, size_t rows, size_t k);   // fp8_block_quant.cu
bool few_rows(int m, int n, int k);              // whether a product takes the few-row kernel (gemm_fp8_block.cu),
bool few_rows_quantize(int m, int n, int k);     // and whether a linear leaves the quantize to it
bool rows_fit(int n, int k, int sms);            // gemm_fp8_block_rows.cu: whether a CTA's shared memory holds its part of the rows
bool rows_quantize_pays(int m, int n, int k, int sms);
int  launch_rows(const Input& X, const uint8_t* W, const GemmParams& p, int sms, cudaStream_t stream);
// lyraq_gemm_fp8_block behind its checks (gemm_fp8_block.cu); rows that are not FP8 yet only where few_rows
int  product(const Input& X, const uint8_t* W, const float* ws, void* Y, int c_dtype, const void* bias, const void* residual, float beta, int epilogue, int m,
             int n, int k, cudaStream_t stream);

}  // namespace fp8b
}  // namespace lyraq
