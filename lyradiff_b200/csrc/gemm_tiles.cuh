// What the persistent tcgen05 GEMMs with microscaled or block-scaled operands share: the order of the tiles and the end of the epilogue.
#pragma once

#include "common.cuh"
#include "sm100_ptx.cuh"

namespace lyraq {
namespace tiles {

// 16 bytes, on a miss the 256 around them into L2
__device__ __forceinline__ Vec16 ld_16_l2_256(const void* p)
{
    Vec16 v;
    asm volatile("ld.global.L2::256B.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.w[0]), "=r"(v.w[1]), "=r"(v.w[2]), "=r"(v.w[3]) : "l"(p));
    return v;
}

// Bands of 8 tile rows swept along N: the tiles that run at the same time share A and B tiles through L2.
__device__ __forceinline__ void tile_coords(int tile, int m_tiles, int n_tiles, int& m_blk, int& n_blk)
{
    constexpr int kGroupM = 8;
    const int per_group = kGroupM * n_tiles;
    const int group     = tile / per_group;
    const int first_m   = group * kGroupM;
    const int rows      = min(kGroupM, m_tiles - first_m);
    const int in_group  = tile - group * per_group;
    m_blk               = first_m + in_group % rows;
    n_blk               = in_group / rows;
}

// 32 columns of one row: accumulators -> fp32 results, in the order beta R, bias, GELU.  bias: the columns' own in shared memory;
// staged: the row's residual in the warp's box, or null (then it is fetched here).  P has M, N,
// bias, residual, beta and gelu.  SCALED: the accumulators still want the factor `scale`.
template<typename T, bool RES, bool SCALED = true, typename P>
__device__ __forceinline__ void finish32(const P& p, const uint32_t* acc, const uint8_t* bias, const uint8_t* staged, int swizzle, float scale, int row,
                                         int col0, int valid, bool vec_ok, float* v)
{
    constexpr int kPer = 16 / (int)sizeof(T);
    const float2  s2 = make_float2(scale, scale);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const float2 a = make_float2(__uint_as_float(acc[2 * i]), __uint_as_float(acc[2 * i + 1]));
        const float2 t = SCALED ? mul_f32x2(a, s2) : a;
        v[2 * i]       = t.x;
        v[2 * i + 1]   = t.y;
    }
    if (RES && staged != nullptr) {
        if constexpr (sizeof(T) == 2) {
            const float2 b2 = make_float2(p.beta, p.beta);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                float2 f[4];
                unpack4x2<T>(*reinterpret_cast<const Vec16*>(staged + ((q ^ swizzle) << 4)), f);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float2 a = fma_f32x2(b2, f[j], make_float2(v[8 * q + 2 * j], v[8 * q + 2 * j + 1]));
                    v[8 * q + 2 * j]     = a.x;
                    v[8 * q + 2 * j + 1] = a.y;
                }
            }
        }
    } else if (RES && p.residual != nullptr && row < p.M) {
        const T* r = reinterpret_cast<const T*>(p.residual) + (size_t)row * (size_t)p.N + (size_t)col0;
        if (vec_ok && valid >= 32) {
#pragma unroll
            for (int q = 0; q < 32 / kPer; ++q) {
                const Vec16 x = ld_16(r + q * kPer);   // Y may be R
                float       f[8];
                if constexpr (sizeof(T) == 4) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        f[j] = __uint_as_float(x.w[j]);
                    }
                } else {
                    unpack8<T>(x, f);
                }
#pragma unroll
                for (int j = 0; j < kPer; ++j) {
                    v[q * kPer + j] = fmaf(p.beta, f[j], v[q * kPer + j]);
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                if (i < valid) {
                    v[i] = fmaf(p.beta, to_f32(r[i]), v[i]);
                }
            }
        }
    }
    if (p.bias != nullptr) {   // every lane reads the same 16 bytes
#pragma unroll
        for (int q = 0; q < 32 / kPer; ++q) {
            const Vec16 x = *reinterpret_cast<const Vec16*>(bias + 16 * q);
            float       f[8];
            if constexpr (sizeof(T) == 4) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    f[j] = __uint_as_float(x.w[j]);
                }
            } else {
                unpack8<T>(x, f);
            }
#pragma unroll
            for (int j = 0; j < kPer; j += 2) {
                const float2 a = add_f32x2(make_float2(v[q * kPer + j], v[q * kPer + j + 1]), make_float2(f[j], f[j + 1]));
                v[q * kPer + j]     = a.x;
                v[q * kPer + j + 1] = a.y;
            }
        }
    }
    if (p.gelu) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float2 t = gelu_tanh_f32x2(make_float2(v[2 * i], v[2 * i + 1]));
            v[2 * i]       = t.x;
            v[2 * i + 1]   = t.y;
        }
    }
}

// 32 values of one row to memory without TMA: fp32 outputs, or rows whose pitch is no multiple of 16 bytes.
template<typename T> __device__ __forceinline__ void store32(T* c, int valid, bool vec_ok, const float* v)
{
    if (vec_ok && valid >= 32) {
#pragma unroll
        for (int q = 0; q < 32 * (int)sizeof(T) / 16; ++q) {
            if constexpr (sizeof(T) == 4) {
                Vec16 w;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    w.w[j] = __float_as_uint(v[4 * q + j]);
                }
                st_16(c + 4 * q, w);
            } else {
                st_16(c + 8 * q, pack8<T>(v + 8 * q));
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            if (i < valid) {
                c[i] = from_f32<T>(v[i]);
            }
        }
    }
}

}  // namespace tiles
}  // namespace lyraq
