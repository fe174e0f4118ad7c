// Quantizers of the microscaled FP4 formats (fp4.cuh has the formats, the scale layout and the arithmetic of a block).
#include "fp4.cuh"

namespace lyraq {

int device_sm_count();  // gemm_dense.cu

// Activations (and weights, once their tensor scale is known).  A pass over memory: 2 bytes a value are read, half a byte and a
// sixteenth or a thirty-second of one are written.  A thread owns 32 values, two blocks or one, four lanes 128 of a row; nothing is exchanged
// but the scale bytes of an atom's row, which one lane stores as a word.  A warp takes the same 128 columns of eight rows, r and r + 1 in
// each quarter of the 128: whole lines of every row, and scale words that fill 32-byte sectors.
template<typename T, int FORMAT>
__global__ void __launch_bounds__(256)
fp4_quant_kernel(uint8_t* q, uint8_t* sf, const T* x, size_t ldx, const float* tensor_scale, size_t rows, size_t k, unsigned blocks_k, int warps_k_log2,
                 int wide)
{
    constexpr int kGroup  = fp4_group(FORMAT);
    constexpr int kBlocks = 32 / kGroup;            // of one thread
    constexpr int kPer    = 16 / (int)sizeof(T);    // values of a 16-byte vector
    constexpr int kVecs   = 32 / kPer;
    grid_launch_dependents();
    // a block's eight warps: 2^warps_k_log2 neighbouring pieces of 128 columns, the rest of them further rows
    const unsigned by = blockIdx.x / blocks_k, bx = blockIdx.x - by * blocks_k;
    const unsigned warp  = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const unsigned chunk = (bx << warps_k_log2) + (warp & ((1u << warps_k_log2) - 1u));
    const unsigned octet = (by << (3 - warps_k_log2)) + (warp >> warps_k_log2);      // 16 to 128 rows
    const unsigned i     = lane >> 2, j = lane & 3;
    const size_t   row   = (size_t)(octet >> 4) * 128 + 2 * (octet & 15) + (i >> 2) + 32 * (i & 3);
    const size_t   col   = (size_t)chunk * 128 + (size_t)j * 32;
    const bool     in    = row < rows && col < k;   // k is a multiple of 32: a thread's values are there or not
    grid_dependency_wait();

    Vec16 v[kVecs];
    if (in) {
        const T* src = x + row * ldx + col;
        if (wide) {   // [4608, 3072]: nvfp4 8.7 -> 7.2 us, mxfp4 7.3 -> 5.0
#pragma unroll
            for (int a = 0; a < kVecs; a += 2) {
                ld_nc_32(src + a * kPer, v[a], v[a + 1]);
            }
        } else {
#pragma unroll
            for (int a = 0; a < kVecs; ++a) {
                v[a] = ld_nc_16(src + a * kPer);
            }
        }
    }
    const Fp4Tensor tensor = fp4_tensor<FORMAT>(tensor_scale);
    uint32_t        code   = 0;
    if (in) {
        Vec16 o;
        code = fp4_encode32<T, FORMAT, false>(v, tensor, o);
        st_16(q + row * (k >> 1) + (col >> 1), o);
    }
    // blocks beyond k have scale 0, so the word of an existing row is always written whole
    constexpr unsigned kLanes = 4 / kBlocks;    // that share a word
    uint32_t           word   = code << (8 * kBlocks * (j % kLanes));
    word |= __shfl_xor_sync(0xffffffffu, word, 1);
    if (kLanes == 4) {
        word |= __shfl_xor_sync(0xffffffffu, word, 2);
    }
    const size_t atom = (size_t)chunk * (4 / kLanes) + j / kLanes, atoms = fp4_atoms(k, FORMAT);
    if (j % kLanes == 0 && row < rows && atom < atoms) {
        *reinterpret_cast<uint32_t*>(sf + fp4_scale_offset(row, atoms, atom)) = word;
    }
}

// The tensor scale of a weight: the least power of two g with max|w| <= 6 * 448 * g, over the numbers in it (an infinity or a NaN spoils its
// own block only), 0 for a weight of zeros, never below 2^-126.  A power of two loses nothing against max / 2688, since a block scale has
// its own exponent, and it keeps every decision of the quantizer exact.  g grows with the maximum, so the blocks' own scales are joined with an
// integer maximum, whose order does not matter.
__device__ __forceinline__ uint32_t fp4_tensor_scale_bits(uint32_t amax_bits)
{
    if (amax_bits == 0u) {
        return 0u;
    }
    const uint32_t v = __float_as_uint(__uint_as_float(amax_bits) / 2688.0f);
    const uint32_t e = (v + 0x007fffffu) & 0xff800000u;   // up to the next power of two
    return e < 0x00800000u ? 0x00800000u : e;
}

template<typename T>
__global__ void __launch_bounds__(256) fp4_tensor_scale_kernel(float* tensor_scale, const T* w, size_t n_vec)
{
    constexpr int kPer = 16 / (int)sizeof(T);
    grid_launch_dependents();
    grid_dependency_wait();
    uint32_t     amax   = 0;
    const size_t stride = (size_t)gridDim.x * blockDim.x;
    for (size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x; i < n_vec; i += stride) {
        const Vec16 v = ld_nc_16(w + i * kPer);
        uint32_t    m = amax_bits_of<T>(v);
        if (m >= 0x7f800000u) {
            m = 0;
#pragma unroll
            for (int e = 0; e < kPer; ++e) {
                uint32_t b;
                if constexpr (sizeof(T) == 4) {
                    b = v.w[e] & 0x7fffffffu;
                } else {
                    const unsigned short h = (unsigned short)(v.w[e >> 1] >> (16 * (e & 1)));
                    b = __float_as_uint(to_f32(*reinterpret_cast<const T*>(&h))) & 0x7fffffffu;
                }
                m = b < 0x7f800000u ? max(m, b) : m;
            }
        }
        amax = max(amax, m);
    }
    amax = __reduce_max_sync(0xffffffffu, amax);
    __shared__ uint32_t part[8];
    if ((threadIdx.x & 31) == 0) {
        part[threadIdx.x >> 5] = amax;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < 8; ++i) {
            amax = max(amax, part[i]);
        }
        const uint32_t g = fp4_tensor_scale_bits(amax);
        if (g != 0u) {
            atomicMax(reinterpret_cast<unsigned int*>(tensor_scale), g);
        }
    }
}

int check_fp4(const void* q, const void* sf, const void* x, int dtype, size_t ldx, int format, size_t rows, size_t k)
{
    if (format != LYRAQ_NVFP4 && format != LYRAQ_MXFP4) {
        return LYRAQ_ERR_INVALID_ARG;
    }
    if (dtype != LYRAQ_F16 && dtype != LYRAQ_BF16 && dtype != LYRAQ_F32) {
        return LYRAQ_ERR_UNSUPPORTED;
    }
    if ((k & 31u) != 0 || k > 0x7fffffffu || rows > 0x7fffffffu) {
        return LYRAQ_ERR_UNSUPPORTED;
    }
    if (q == nullptr || sf == nullptr || x == nullptr || !aligned16(q) || !aligned16(sf) || !aligned16(x)) {
        return LYRAQ_ERR_INVALID_ARG;
    }
    if (ldx < k || (ldx * (dtype == LYRAQ_F32 ? 4u : 2u) & 15u) != 0) {
        return LYRAQ_ERR_INVALID_ARG;
    }
    return LYRAQ_OK;
}

static int run_quant(uint8_t* q, uint8_t* sf, const void* x, int dtype, size_t ldx, const float* tensor_scale, int format, size_t rows,
                     size_t k, cudaStream_t s)
{
    const size_t chunks  = (k + 127) / 128;
    const size_t octets  = rows >= 32 ? (rows + 127) / 128 * 16 : (rows + 1) / 2;   // fewer than 32 rows lie in the first quarter of their 128
    int          warps_k = 0;
    while (warps_k < 3 && (size_t)1 << warps_k < chunks) {
        ++warps_k;
    }
    const size_t blocks_k = (chunks + ((size_t)1 << warps_k) - 1) >> warps_k;
    const size_t blocks   = blocks_k * ((octets + ((size_t)8 >> warps_k) - 1) >> (3 - warps_k));
    if (blocks > 0x7fffffffu) {
        return LYRAQ_ERR_UNSUPPORTED;
    }
    const int wide = ((reinterpret_cast<uintptr_t>(x) | ldx * (dtype == LYRAQ_F32 ? 4u : 2u)) & 31u) == 0;   // rows on 32 bytes
    auto launch = [&](auto* kernel, auto type) {
        using T = decltype(type);
        return launch_kernel(kernel, (unsigned)blocks, 256u, (size_t)0, s, 1u, q, sf, (const T*)x, ldx, tensor_scale, rows, k, (unsigned)blocks_k,
                             warps_k, wide);
    };
    auto pick = [&](auto type) {
        using T = decltype(type);
        return format == LYRAQ_NVFP4 ? launch(fp4_quant_kernel<T, LYRAQ_NVFP4>, type) : launch(fp4_quant_kernel<T, LYRAQ_MXFP4>, type);
    };
    const cudaError_t e = dtype == LYRAQ_BF16 ? pick(__nv_bfloat16{}) : dtype == LYRAQ_F16 ? pick(__half{}) : pick(float{});
    return cuda_status(e, "cudaLaunchKernelEx(fp4_quant_kernel)");
}

}  // namespace lyraq

using namespace lyraq;

extern "C" {

size_t lyraq_fp4_scale_bytes(size_t rows, size_t k, int format)
{
    if (format != LYRAQ_NVFP4 && format != LYRAQ_MXFP4) {
        return 0;
    }
    return (rows + 127) / 128 * fp4_atoms(k, format) * 512;
}

int lyraq_quant_fp4(uint8_t* q, uint8_t* q_scale, const void* x, int x_dtype, size_t ldx, const float* tensor_scale, int format, size_t rows,
                    size_t k, void* stream)
{
    if (format != LYRAQ_NVFP4 && format != LYRAQ_MXFP4) {
        return LYRAQ_ERR_INVALID_ARG;
    }
    if (rows == 0 || k == 0) {
        return LYRAQ_OK;
    }
    const int st = check_fp4(q, q_scale, x, x_dtype, ldx, format, rows, k);
    if (st != LYRAQ_OK) {
        return st;
    }
    return run_quant(q, q_scale, x, x_dtype, ldx, format == LYRAQ_NVFP4 ? tensor_scale : nullptr, format, rows, k, (cudaStream_t)stream);
}

int lyraq_weight_quant_fp4(uint8_t* qw, uint8_t* w_scale, float* tensor_scale, const void* w, int w_dtype, int format, size_t n, size_t k,
                           void* stream)
{
    if (format != LYRAQ_NVFP4 && format != LYRAQ_MXFP4) {
        return LYRAQ_ERR_INVALID_ARG;
    }
    if (n == 0 || k == 0) {
        return LYRAQ_OK;
    }
    const int st = check_fp4(qw, w_scale, w, w_dtype, k, format, n, k);
    if (st != LYRAQ_OK) {
        return st;
    }
    if (format == LYRAQ_MXFP4) {
        return run_quant(qw, w_scale, w, w_dtype, k, nullptr, format, n, k, (cudaStream_t)stream);
    }
    if (tensor_scale == nullptr) {
        return LYRAQ_ERR_INVALID_ARG;
    }
    const int sms = device_sm_count();
    if (sms <= 0) {
        return LYRAQ_ERR_CUDA;
    }
    cudaError_t e = cudaMemsetAsync(tensor_scale, 0, sizeof(float), (cudaStream_t)stream);
    if (e != cudaSuccess) {
        return cuda_status(e, "cudaMemsetAsync(tensor scale)");
    }
    const size_t   n_vec = n * k / (w_dtype == LYRAQ_F32 ? 4 : 8);
    const size_t   want  = (n_vec + 255) / 256, most = (size_t)sms * 8;
    const unsigned grid  = (unsigned)(want < most ? want : most);
    if (w_dtype == LYRAQ_BF16) {
        e = launch_kernel(fp4_tensor_scale_kernel<__nv_bfloat16>, grid, 256u, (size_t)0, (cudaStream_t)stream, 1u, tensor_scale,
                          (const __nv_bfloat16*)w, n_vec);
    } else if (w_dtype == LYRAQ_F16) {
        e = launch_kernel(fp4_tensor_scale_kernel<__half>, grid, 256u, (size_t)0, (cudaStream_t)stream, 1u, tensor_scale, (const __half*)w, n_vec);
    } else {
        e = launch_kernel(fp4_tensor_scale_kernel<float>, grid, 256u, (size_t)0, (cudaStream_t)stream, 1u, tensor_scale, (const float*)w, n_vec);
    }
    if (e != cudaSuccess) {
        return cuda_status(e, "cudaLaunchKernelEx(fp4_tensor_scale_kernel)");
    }
    return run_quant(qw, w_scale, w, w_dtype, k, tensor_scale, format, n, k, (cudaStream_t)stream);
}

}  // extern "C"
