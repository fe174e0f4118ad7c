// What the FP4 kernels share: the problem, and the tcgen05 forms with block scales.
#pragma once

#include "fp4.cuh"
#include "gemm_tiles.cuh"
#include "sm100_ptx.cuh"
#include "views.h"

namespace lyraq {

struct Fp4GemmParams {
    int           M, N, K;
    int           m_tiles, n_tiles;
    unsigned int* status;
    void*         C;          // [M, N] of c_dtype: F16, BF16 or F32
    int           c_dtype;
    int           tma_store;  // 16-bit output whose row pitch allows TMA stores
    const float*  s_x;        // tensor scales, null = 1
    const float*  s_w;
    const void*   bias;       // [N] of c_dtype or null
    const void*   residual;   // [M, N] of c_dtype or null
    float         beta;
    int           gelu;
};

namespace fp4 {
constexpr int kFp4SkinnyRows = 16;   // most rows of X that gemm_fp4_skinny.cu takes
constexpr int kMaxSize       = 0x7fffff00;   // of m, n and k: row, column and block numbers of a last tile stay within 31 bits

// The left operand: FP4 codes with their block scales, or (codes null) rows of a 16- or 32-bit type that the few-row kernel quantizes itself.
struct Fp4Input {
    const uint8_t* codes;
    const uint8_t* scales;
    const void*    x;
    int            dtype;
    size_t         ldx;
};

int  launch_skinny(const Fp4Input& X, const uint8_t* W, const uint8_t* ws, int format, const Fp4GemmParams& p, int sms, cudaStream_t stream);
bool skinny_quantize_pays(int m, int n, int k, int sms);
bool few_rows(int m, int k);                  // whether a product takes the few-row kernel,
bool few_rows_quantize(int m, int n, int k);  // and whether a linear leaves the quantize to it
// lyraq_gemm_fp4 behind its checks; rows that are not FP4 yet only where few_rows
int product(const Fp4Input& X, const float* g_x, const uint8_t* W, const uint8_t* ws, const float* g_w, int format, void* Y, int c_dtype, const void* bias,
            const void* residual, float beta, int epilogue, int m, int n, int k, cudaStream_t stream);
}  // namespace fp4

__device__ __forceinline__ float fp4_tensor_scale(const Fp4GemmParams& p)
{
    return (p.s_x != nullptr ? ld_f32(p.s_x) : 1.0f) * (p.s_w != nullptr ? ld_f32(p.s_w) : 1.0f);
}

namespace sm100 {

__device__ __forceinline__ void tma_load_3d(uint32_t smem_dst, const CUtensorMap* m, uint32_t bar, int x, int y, int z)
{
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
        ::"r"(smem_dst), "l"(reinterpret_cast<uint64_t>(m)), "r"(bar), "r"(x), "r"(y), "r"(z)
        : "memory");
}
// one CTA of a pair; the bytes are counted on the leader's barrier (see tma_load_2d_pair)
__device__ __forceinline__ void tma_load_3d_pair(uint32_t smem_dst, const CUtensorMap* m, uint32_t leader_bar, int x, int y, int z)
{
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
        ::"r"(smem_dst), "l"(reinterpret_cast<uint64_t>(m)), "r"(leader_bar), "r"(x), "r"(y), "r"(z)
        : "memory");
}

// Shared memory -> tensor memory, 32 rows of 16 bytes, the same to each of the four lane quadrants: one atom of block scales, four columns.
// Runs in order before the MMAs that the same thread issues after it.  With a CTA pair each CTA's own shared memory goes to its own
// tensor memory.
template<int CTAS> __device__ __forceinline__ void tmem_copy_scales(uint32_t taddr, uint64_t sdesc)
{
    if (CTAS == 2) {
        asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(sdesc) : "memory");
    } else {
        asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(sdesc) : "memory");
    }
}

// Descriptor of an atom in shared memory: no swizzle, core matrices of 8 rows x 16 bytes one after the other (stride byte offset 128).
__device__ __forceinline__ uint64_t umma_desc_scales(uint32_t smem_addr)
{
    uint64_t d = 0;
    d |= (uint64_t)((smem_addr & 0x3ffff) >> 4);
    d |= (uint64_t)(128 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    return d;
}

// Instruction descriptor of the block-scaled kinds with packed e2m1 operands, both K-major.  sf_id: which bytes of a scale word the
// instruction takes: 0 for four blocks of 16 (all of them), 0 or 2 for two blocks of 32.
__host__ __device__ constexpr uint32_t umma_idesc_fp4(int format, uint32_t m, uint32_t n, uint32_t sf_id)
{
    return (sf_id << 4) | (1u << 7) | (1u << 10) | ((n >> 3) << 17) | ((format == LYRAQ_MXFP4 ? 1u : 0u) << 23) | ((m >> 4) << 24) | (sf_id << 29);
}

// D[tmem] (+)= (A * SA) (B * SB)^T over 64 values of K (32 bytes of a K-major row).
template<int FORMAT, int CTAS>
__device__ __forceinline__ void mma_fp4(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t accumulate)
{
    if (FORMAT == LYRAQ_NVFP4) {
        if (CTAS == 2) {
            asm volatile(
                "{\n\t"
                ".reg .pred p;\n\t"
                "setp.ne.b32 p, %4, 0;\n\t"
                "tcgen05.mma.cta_group::2.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%5], [%6], p;\n\t"
                "}\n" ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(sfa), "r"(sfb) : "memory");
        } else {
            asm volatile(
                "{\n\t"
                ".reg .pred p;\n\t"
                "setp.ne.b32 p, %4, 0;\n\t"
                "tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%5], [%6], p;\n\t"
                "}\n" ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(sfa), "r"(sfb) : "memory");
        }
    } else {
        if (CTAS == 2) {
            asm volatile(
                "{\n\t"
                ".reg .pred p;\n\t"
                "setp.ne.b32 p, %4, 0;\n\t"
                "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%5], [%6], p;\n\t"
                "}\n" ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(sfa), "r"(sfb) : "memory");
        } else {
            asm volatile(
                "{\n\t"
                ".reg .pred p;\n\t"
                "setp.ne.b32 p, %4, 0;\n\t"
                "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%5], [%6], p;\n\t"
                "}\n" ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(sfa), "r"(sfb) : "memory");
        }
    }
}

}  // namespace sm100
}  // namespace lyraq
