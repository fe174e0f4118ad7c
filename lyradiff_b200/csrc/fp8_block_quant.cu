// Quantizers of FP8 with a scale for each block of 128 (fp8_block.cuh has the format and the arithmetic of a block).
#include "fp8_block.cuh"

namespace lyraq {
namespace fp8b {

// Activations, blocks of 1 x 128.  A pass over memory: 2 bytes a value are read, one and a 32nd are written.  A lane owns 16 values of each of two blocks, eight
// lanes a block, a warp 256 columns of four rows (whole lines of each; their scales are 16 bytes where scales of a block lie together), the warps of a
// thread block neighbouring columns.
template<typename T>
__global__ void __launch_bounds__(256)
fp8_block_quant_kernel(uint8_t* q, float* scale, size_t scale_row, size_t scale_block, const T* x, size_t ldx, size_t rows, size_t k, unsigned pairs_k,
                       size_t pieces, int wide)
{
    constexpr int kPer  = 16 / (int)sizeof(T);
    constexpr int kVecs = (int)sizeof(T);
    grid_launch_dependents();
    const size_t   piece = (size_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    const unsigned lane  = threadIdx.x & 31;
    const size_t   quad  = piece / pairs_k, kb = (piece - quad * pairs_k) * 2;
    const size_t   row   = quad * 4 + (lane >> 3), col = kb * kBlock + (lane & 7) * 16;
    const bool     there = piece < pieces && row < rows;
    grid_dependency_wait();

    Vec16 v[2][kVecs] = {};
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        if (there && col + u * kBlock < k) {   // k is a multiple of 16: a lane's values are there or not
            const T* src = x + row * ldx + col + u * kBlock;
            if (wide) {
#pragma unroll
                for (int a = 0; a < kVecs; a += 2) {
                    ld_nc_32(src + a * kPer, v[u][a], v[u][a + 1]);
                }
            } else {
#pragma unroll
                for (int a = 0; a < kVecs; ++a) {
                    v[u][a] = ld_nc_16(src + a * kPer);
                }
            }
        }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        uint32_t amax = amax16_values<T>(v[u]);
#pragma unroll
        for (int d = 1; d < 8; d *= 2) {
            amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, d));
        }
        const Divisor d = divisor_of(amax);
        if (there && col + u * kBlock < k) {
            st_16(q + row * k + col + u * kBlock, encode16<T>(v[u], d));
            if ((lane & 7) == 0) {
                scale[row * scale_row + (kb + u) * scale_block] = d.s;
            }
        }
    }
}

// Weights, blocks of 128 x 128: a thread block each, 64 values a thread, kept in registers between the maximum and the codes.
template<typename T>
__global__ void __launch_bounds__(256) fp8_block_weight_kernel(uint8_t* q, float* scale, const T* w, size_t n, size_t k, unsigned blocks_k)
{
    constexpr int kPer  = 16 / (int)sizeof(T);
    constexpr int kVecs = (int)sizeof(T);
    grid_launch_dependents();
    const size_t by = blockIdx.x / blocks_k, bx = blockIdx.x - by * blocks_k;
    const size_t col = bx * kBlock + (threadIdx.x & 7) * 16;
    grid_dependency_wait();

    Vec16    v[4][kVecs] = {};
    uint32_t amax        = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const size_t row = by * kBlock + i * 32 + (threadIdx.x >> 3);
        if (row < n && col < k) {
#pragma unroll
            for (int a = 0; a < kVecs; ++a) {
                v[i][a] = ld_nc_16(w + row * k + col + a * kPer);
            }
        }
        amax = max(amax, amax16_values<T>(v[i]));
    }
    __shared__ uint32_t part[8];
    amax = __reduce_max_sync(0xffffffffu, amax);
    if ((threadIdx.x & 31) == 0) {
        part[threadIdx.x >> 5] = amax;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        amax = max(amax, part[i]);
    }
    const Divisor d = divisor_of(amax);
    if (threadIdx.x == 0) {
        scale[blockIdx.x] = d.s;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const size_t row = by * kBlock + i * 32 + (threadIdx.x >> 3);
        if (row < n && col < k) {
            st_16(q + row * k + col, encode16<T>(v[i], d));
        }
    }
}

int check_quant(const void* q, const void* scale, const void* x, int dtype, size_t ldx, size_t rows, size_t k)
{
    if (dtype != LYRAQ_F16 && dtype != LYRAQ_BF16 && dtype != LYRAQ_F32) {
        return LYRAQ_ERR_UNSUPPORTED;
    }
    if ((k & 15u) != 0 || k > (size_t)kMaxSize || rows > (size_t)kMaxSize) {
        return LYRAQ_ERR_UNSUPPORTED;
    }
    if (q == nullptr || scale == nullptr || x == nullptr || !aligned16(q) || (reinterpret_cast<uintptr_t>(scale) & 3u) != 0 || !aligned16(x)) {
        return LYRAQ_ERR_INVALID_ARG;
    }
    if (ldx < k || (ldx * (dtype == LYRAQ_F32 ? 4u : 2u) & 15u) != 0) {
        return LYRAQ_ERR_INVALID_ARG;
    }
    return LYRAQ_OK;
}

}  // namespace fp8b
}  // namespace lyraq

using namespace lyraq;

extern "C" {

int lyraq_quant_fp8_block(uint8_t* q, float* scale, size_t scale_row, size_t scale_block, const void* x, int x_dtype, size_t ldx, size_t rows, size_t k,
                          void* stream)
{
    if (rows == 0 || k == 0) {
        return LYRAQ_OK;
    }
    const int st = fp8b::check_quant(q, scale, x, x_dtype, ldx, rows, k);
    if (st != LYRAQ_OK) {
        return st;
    }
    const size_t blocks_k = fp8b::blocks_of(k), bytes = x_dtype == LYRAQ_F32 ? 4 : 2;
    const View   vs = view_of(scale, 4, rows, scale_row, blocks_k, scale_block, 1, 0, 1), vq = view_of(q, rows * k);
    const View   vx = view_of(x, bytes, rows, ldx, 1, 0, 1, 0, k);
    // rows of scales and of blocks must not fall on one another: the larger step lies past the smaller one's run
    const bool   nested = rows == 1 ? blocks_k == 1 || scale_block != 0
                        : blocks_k == 1 ? scale_row != 0
                        : scale_row < scale_block ? scale_row != 0 && (rows - 1) <= (scale_block - 1) / scale_row
                                                  : scale_block != 0 && (blocks_k - 1) <= (scale_row - 1) / scale_block;
    if (!nested || views_meet(vs, vq) || views_meet(vx, vq) || views_meet(vx, vs)) {
        return LYRAQ_ERR_INVALID_ARG;
    }
    const size_t pairs_k = (blocks_k + 1) / 2, pieces = (rows + 3) / 4 * pairs_k, blocks = (pieces + 7) / 8;
    if (blocks > 0x7fffffffu) {
        return LYRAQ_ERR_UNSUPPORTED;
    }
    const int wide   = ((reinterpret_cast<uintptr_t>(x) | ldx * bytes) & 31u) == 0;   // rows on 32 bytes
    auto      launch = [&](auto type) {
        using T = decltype(type);
        return launch_kernel(fp8b::fp8_block_quant_kernel<T>, (unsigned)blocks, 256u, (size_t)0, (cudaStream_t)stream, 1u, q, scale, scale_row, scale_block,
                             (const T*)x, ldx, rows, k, (unsigned)pairs_k, pieces, wide);
    };
    const cudaError_t e = x_dtype == LYRAQ_BF16 ? launch(__nv_bfloat16{}) : x_dtype == LYRAQ_F16 ? launch(__half{}) : launch(float{});
    return cuda_status(e, "cudaLaunchKernelEx(fp8_block_quant_kernel)");
}

int lyraq_weight_quant_fp8_block(uint8_t* qw, float* w_scale, const void* w, int w_dtype, size_t n, size_t k, void* stream)
{
    if (n == 0 || k == 0) {
        return LYRAQ_OK;
    }
    const int st = fp8b::check_quant(qw, w_scale, w, w_dtype, k, n, k);
    if (st != LYRAQ_OK) {
        return st;
    }
    const size_t blocks_k = fp8b::blocks_of(k), blocks = fp8b::blocks_of(n) * blocks_k;
    const View   vs = view_of(w_scale, blocks * 4), vq = view_of(qw, n * k), vw = view_of(w, n * k * (w_dtype == LYRAQ_F32 ? 4 : 2));
    if (views_meet(vs, vq) || views_meet(vw, vq) || views_meet(vw, vs)) {
        return LYRAQ_ERR_INVALID_ARG;
    }
    if (blocks > 0x7fffffffu) {
        return LYRAQ_ERR_UNSUPPORTED;
    }
    auto launch = [&](auto type) {
        using T = decltype(type);
        return launch_kernel(fp8b::fp8_block_weight_kernel<T>, (unsigned)blocks, 256u, (size_t)0, (cudaStream_t)stream, 1u, qw, w_scale, (const T*)w, n, k,
                             (unsigned)blocks_k);
    };
    const cudaError_t e = w_dtype == LYRAQ_BF16 ? launch(__nv_bfloat16{}) : w_dtype == LYRAQ_F16 ? launch(__half{}) : launch(float{});
    return cuda_status(e, "cudaLaunchKernelEx(fp8_block_weight_kernel)");
}

}  // extern "C"
