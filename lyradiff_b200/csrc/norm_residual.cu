// The end of one block and the start of the next in a single pass over the tokens:
//
//   u = post(y) * w1          post: none, RMS or LayerNorm of the block's output
//   v = r x + gate_b * u      the residual stream, scaled by r
//   x' = T(v)
//   h = T( pre(v) * w2 * (1 + scale_b) + shift_b )      pre: RMS or LayerNorm, of v before its rounding
//
// Everything is fp32 from load to store and is rounded once.  h leaves in T, as e4m3 codes of T(h) / s, or in FP4 (fp4.cuh), the codes that
// the separate quantizers make of T(h).
//
// Bound by memory: two rows in, two out (or one and a quantized one).  A row stays in registers, so it is read once: its statistics are sums
// over a warp, or over a block and one exchange through shared memory each.  LayerNorm takes two such sums, the second over the distances from the
// mean (a difference of sums of squares would lose what a large mean covers).  The five parameter vectors are shared by a batch entry's rows and
// come from L1.
#include "fp4.cuh"
#include "views.h"

namespace lyraq {

int device_sm_count();  // gemm_dense.cu

struct NormParams {
    const void*  y;
    const void*  x;
    void*        x_out;
    void*        h;
    uint8_t*     qf8;
    uint8_t*     q4;
    uint8_t*     q4_sf;
    const void*  gate;
    const void*  scale;
    const void*  shift;
    const void*  w1;
    const void*  w2;
    const float* f8_scale;
    const float* q4_scale;
    size_t       y_batch, y_row, x_batch, x_row, xo_batch, xo_row, h_batch, h_row;   // strides in elements
    size_t       gate_batch, scale_batch, shift_batch;
    size_t       atoms;
    unsigned     rows, seq;      // batch * seq_len and seq_len
    int          dim, post, pre;
    float        r, eps;
};

// FORMAT: -1 without an FP4 output.  ALL: every parameter and the new stream are there.  FULL: every vector of every thread is.  Asking costs a sixth of the
// instructions: [4608, 3072] with everything 25.1 us without either, 22.3 with ALL, 21.2 with both.  Calls with parts absent ask: without post norm and
// weights 22.6, without a modulation too 18.1.
template<typename T, int VPT, int FORMAT, bool WARP, bool ALL, bool FULL>
__global__ void __launch_bounds__(WARP ? 256 : 512, 2)
norm_residual_kernel(const NormParams p)
{
    __shared__ float part[4][16];
    const int nvec    = p.dim >> 3;
    const int threads = WARP ? 32 : (int)blockDim.x;       // of the row
    const int t       = WARP ? (int)(threadIdx.x & 31) : (int)threadIdx.x;
    const float inv_d = 1.0f / (float)p.dim;
    grid_launch_dependents();
    grid_dependency_wait();

    const unsigned row = WARP ? blockIdx.x * 8 + (threadIdx.x >> 5) : blockIdx.x;
    if (row >= p.rows) {
        return;   // whole warps, and never part of a block that meets at a barrier
    }
    const unsigned b = row / p.seq, s = row - b * p.seq;
    // slot: which exchange of the row this is; every exchange has its own words, so one barrier each is enough
    auto total = [&](float2 v2, int slot) {
        float v = v2.x + v2.y;
#pragma unroll
        for (int m = 16; m > 0; m >>= 1) {
            v += __shfl_xor_sync(0xffffffffu, v, m);
        }
        if (!WARP) {
            if ((threadIdx.x & 31) == 0) {
                part[slot][threadIdx.x >> 5] = v;
            }
            __syncthreads();
            v = 0.0f;
            for (int i = 0; i < (int)(blockDim.x >> 5); ++i) {
                v += part[slot][i];
            }
        }
        return v;
    };
    const T* yr = reinterpret_cast<const T*>(p.y) + b * p.y_batch + s * p.y_row;
    const T* xr = reinterpret_cast<const T*>(p.x) + b * p.x_batch + s * p.x_row;
    Vec16 yv[VPT], xv[VPT];
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        const int vi = t + i * threads;
        yv[i] = Vec16{};
        xv[i] = Vec16{};
        if (FULL || vi < nvec) {
            yv[i] = ld_16(yr + vi * 8);
            xv[i] = ld_16(xr + vi * 8);
        }
    }

    // u = (y - mean) * inv as one fma: y * inv + (-mean * inv).  Vectors beyond the row are zeros that no sum takes in.
    float2 v[VPT][4];
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        unpack4x2<T>(yv[i], v[i]);
    }
    float mean = 0.0f, inv = 1.0f;
    if (p.post == LYRAQ_NORM_LAYER) {
        float2 a = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                a = add_f32x2(a, v[i][j]);
            }
        }
        mean = total(a, 0) * inv_d;
    }
    if (p.post != LYRAQ_NORM_NONE) {
        const float2 m2 = make_float2(-mean, -mean);
        float2       a  = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            if (FULL || t + i * threads < nvec) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    v[i][j] = add_f32x2(v[i][j], m2);
                    a       = fma_f32x2(v[i][j], v[i][j], a);
                }
            }
        }
        inv = rsqrtf(total(a, 1) * inv_d + p.eps);
    }
    const T*     gate = reinterpret_cast<const T*>(p.gate) + b * p.gate_batch;
    T*           xo   = reinterpret_cast<T*>(p.x_out) + b * p.xo_batch + s * p.xo_row;
    const float2 r2   = make_float2(p.r, p.r);
    float2       sum  = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        const int vi = t + i * threads;
        if (FULL || vi < nvec) {
            float2 f[4], c[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                c[j] = make_float2(inv, inv);
            }
            if (ALL || p.w1 != nullptr) {
                unpack4x2<T>(ld_nc_16_keep(reinterpret_cast<const T*>(p.w1) + vi * 8), f);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    c[j] = mul_f32x2(c[j], f[j]);
                }
            }
            if (ALL || p.gate != nullptr) {
                unpack4x2<T>(ld_nc_16_keep(gate + vi * 8), f);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    c[j] = mul_f32x2(c[j], f[j]);
                }
            }
            unpack4x2<T>(xv[i], f);
            float o[8];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                v[i][j]      = fma_f32x2(v[i][j], c[j], mul_f32x2(r2, f[j]));
                sum          = add_f32x2(sum, v[i][j]);
                o[2 * j]     = v[i][j].x;
                o[2 * j + 1] = v[i][j].y;
            }
            if (ALL || p.x_out != nullptr) {
                st_16(xo + vi * 8, pack8<T>(o));
            }
        }
    }
    mean = p.pre == LYRAQ_NORM_LAYER ? total(sum, 2) * inv_d : 0.0f;
    const float2 m2 = make_float2(-mean, -mean);
    float2       sq = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        if (FULL || t + i * threads < nvec) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                v[i][j] = add_f32x2(v[i][j], m2);
                sq      = fma_f32x2(v[i][j], v[i][j], sq);
            }
        }
    }
    inv = rsqrtf(total(sq, 3) * inv_d + p.eps);

    const T*    scale = reinterpret_cast<const T*>(p.scale) + b * p.scale_batch;
    const T*    shift = reinterpret_cast<const T*>(p.shift) + b * p.shift_batch;
    T*          hr    = reinterpret_cast<T*>(p.h) + b * p.h_batch + s * p.h_row;
    const float r8    = p.qf8 != nullptr ? 1.0f / ld_f32(p.f8_scale) : 0.0f;
    constexpr int   kFmt   = FORMAT < 0 ? 0 : FORMAT;
    const Fp4Tensor tensor = FORMAT >= 0 ? fp4_tensor<kFmt>(p.q4_scale) : Fp4Tensor{};
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        const int  vi = t + i * threads;
        const bool in = FULL || vi < nvec;
        Vec16      o{};
        if (in) {
            float2 f[4], c[4];
            float  h[8];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                c[j] = make_float2(inv, inv);
            }
            if (ALL || p.w2 != nullptr) {
                unpack4x2<T>(ld_nc_16_keep(reinterpret_cast<const T*>(p.w2) + vi * 8), f);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    c[j] = mul_f32x2(c[j], f[j]);
                }
            }
            if (ALL || p.scale != nullptr) {
                unpack4x2<T>(ld_nc_16_keep(scale + vi * 8), f);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    c[j] = fma_f32x2(c[j], f[j], c[j]);
                }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                f[j] = make_float2(0.0f, 0.0f);
            }
            if (ALL || p.shift != nullptr) {
                unpack4x2<T>(ld_nc_16_keep(shift + vi * 8), f);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 w = fma_f32x2(v[i][j], c[j], f[j]);
                h[2 * j]       = w.x;
                h[2 * j + 1]   = w.y;
            }
            o = pack8<T>(h);
            if (p.h != nullptr) {
                st_16(hr + vi * 8, o);
            }
            if (p.qf8 != nullptr) {
                unpack8<T>(o, h);
                st_8(p.qf8 + (size_t)row * (size_t)p.dim + vi * 8, f32x2_to_e4m3x2(h[0] * r8, h[1] * r8) | (f32x2_to_e4m3x2(h[2] * r8, h[3] * r8) << 16),
                     f32x2_to_e4m3x2(h[4] * r8, h[5] * r8) | (f32x2_to_e4m3x2(h[6] * r8, h[7] * r8) << 16));
            }
        }
        if (FORMAT >= 0) {
            // a block lies in two or four neighbouring lanes, the scale word of an atom's row in eight or sixteen; lanes beyond the row
            // add nothing to either
            constexpr int kLanes = fp4_group(kFmt) / 8;
            uint32_t amax = amax_bits_of<T>(o);
            amax          = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
            if (kLanes == 4) {
                amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
            }
            const Fp4Block blk  = fp4_block<kFmt>(amax, tensor);
            uint32_t       word = (in ? blk.code : 0u) << (8 * ((vi / kLanes) & 3));
            word |= __shfl_xor_sync(0xffffffffu, word, kLanes);
            word |= __shfl_xor_sync(0xffffffffu, word, 2 * kLanes);
            if (in) {
                float f[8];
                unpack8<T>(o, f);
                *reinterpret_cast<uint32_t*>(p.q4 + (size_t)row * (size_t)(p.dim >> 1) + vi * 4) = fp4_encode8<kFmt>(f, blk);
                if (vi % (4 * kLanes) == 0) {
                    *reinterpret_cast<uint32_t*>(p.q4_sf + fp4_scale_offset(row, p.atoms, (size_t)(vi / (4 * kLanes)))) = word;
                }
            }
        }
    }
}

// Threads of a row.  Up to 1280 elements a warp may have it (up to five vectors a lane) and no barrier; whether it does depends on how many rows there are to
// fill the chip with.  A warp against a block, us: 640 elements, 300 rows 3.6 / 3.6, 2400 4.6 / 6.0, 16384 16.9 / 20.1; 1024 elements, 450 rows 4.4 / 3.1, 900
// 4.7 / 4.7, 16384 27.1 / 29.2; 1280 elements, 600 rows 5.0 / 4.5, 900 5.2 / 5.6, 4608 9.7 / 10.7, 8192 16.4 / 17.5, 12288 29.0 / 27.2 (two blocks of five
// vectors a lane are all an SM holds).
// Longer rows have a block, best one without absent vectors (FULL): as many threads as let all rows run at once (1024 threads an SM), since a thread's part of
// the sums weighs more the fewer vectors it has, and three or four vectors a thread where rows take turns.  Vectors a thread, us: 2048 elements, 1000 rows two
// 4.5, three (not FULL) 6.1, four 6.9, 4608 rows 14.0 / 15.2 / 13.0; 3072 elements, 4608 rows 26.2 / 21.3 / 22.9; 8192 elements, 4608 rows 73 / 75 / 55; 2560
// elements, 4608 rows 20.3 (FULL) / 18.8 / 19.4.
struct NormSplit {
    int  vpt, threads;
    bool warp;
};
static NormSplit norm_split(size_t rows, int dim, int sms)
{
    const int nvec = dim / 8;
    const size_t fill = (size_t)sms * (nvec <= 80 ? 2 : 6);
    if (nvec <= 32 || (nvec <= 128 && rows > fill) || (nvec <= 160 && rows > fill && rows <= (size_t)sms * 64)) {
        return NormSplit{nvec <= 32 ? 1 : nvec <= 64 ? 2 : nvec <= 96 ? 3 : nvec <= 128 ? 4 : 5, 256, true};
    }
    auto whole = [&](int vpt) { return nvec % (32 * vpt) == 0 && nvec / vpt <= 512; };
    for (int vpt = rows <= (size_t)sms * 2 ? 1 : 2; vpt <= 4; ++vpt) {
        if (whole(vpt) && rows <= (size_t)sms * (size_t)(1024 * vpt / nvec)) {
            return NormSplit{vpt, nvec / vpt, false};
        }
    }
    int vpt = rows <= (size_t)sms * 2 ? 1 : !whole(3) && whole(4) ? 4 : 3;
    while ((nvec + vpt - 1) / vpt > 512) {
        ++vpt;
    }
    return NormSplit{vpt, ((nvec + vpt - 1) / vpt + 31) / 32 * 32, false};
}

// Rows are written while others are read: x_out and h are x or y, element for element, or apart from them; all outputs are apart from each other, the
// quantized ones from x and y too.
static bool outputs_clash(const lyraq_gated_norm_t& a)
{
    auto rows = [&](const void* p, size_t batch, size_t row) { return view_of(p, 2, a.batch, batch, a.seq_len, row, 1, 0, a.dim); };
    const size_t n = a.batch * a.seq_len;
    const View   in[2]  = {rows(a.y, a.y_batch, a.y_row), rows(a.x, a.x_batch, a.x_row)};
    const View   out[5] = {rows(a.x_out, a.x_out_batch, a.x_out_row), rows(a.h, a.h_batch, a.h_row), view_of(a.qf8, n * a.dim), view_of(a.q4, n * a.dim / 2),
                           view_of(a.q4 != nullptr ? a.q4_scales : nullptr, lyraq_fp4_scale_bytes(n, a.dim, a.q4_format))};
    for (int i = 0; i < 5; ++i) {
        for (const View& v : in) {
            if (!(i < 2 && views_same(out[i], v)) && views_meet(out[i], v)) {
                return true;
            }
        }
        for (int j = 0; j < i; ++j) {
            if (views_meet(out[i], out[j])) {
                return true;
            }
        }
    }
    return false;
}

static bool rows_ok(const void* p, size_t batch, size_t row) { return aligned16(p) && (batch & 7u) == 0 && (row & 7u) == 0; }

}  // namespace lyraq

using namespace lyraq;

extern "C" int lyraq_gated_residual_norm(const lyraq_gated_norm_t* a, void* stream)
{
    if (a == nullptr || a->post < LYRAQ_NORM_NONE || a->post > LYRAQ_NORM_LAYER ||
        (a->pre != LYRAQ_NORM_RMS && a->pre != LYRAQ_NORM_LAYER)) {
        return LYRAQ_ERR_INVALID_ARG;
    }
    if ((a->dtype != LYRAQ_F16 && a->dtype != LYRAQ_BF16) || (a->dim & 7u) != 0 || a->dim > 16384 || a->batch > 0x7fffffffu ||
        a->seq_len > 0x7fffffffu || a->batch * a->seq_len > 0x7fffffffu) {
        return LYRAQ_ERR_UNSUPPORTED;
    }
    if (a->batch * a->seq_len * a->dim == 0) {
        return LYRAQ_OK;
    }
    if (a->y == nullptr || a->x == nullptr || (a->x_out == nullptr && a->h == nullptr && a->qf8 == nullptr && a->q4 == nullptr) ||
        (a->qf8 != nullptr && a->f8_scale == nullptr) || (a->q4 != nullptr && a->q4_scales == nullptr)) {
        return LYRAQ_ERR_INVALID_ARG;
    }
    if (!rows_ok(a->y, a->y_batch, a->y_row) || !rows_ok(a->x, a->x_batch, a->x_row) || !rows_ok(a->x_out, a->x_out_batch, a->x_out_row) ||
        !rows_ok(a->h, a->h_batch, a->h_row) || !rows_ok(a->gate, a->gate_batch, 0) || !rows_ok(a->scale, a->scale_batch, 0) ||
        !rows_ok(a->shift, a->shift_batch, 0) || !aligned16(a->post_weight) || !aligned16(a->pre_weight) ||
        (reinterpret_cast<uintptr_t>(a->qf8) & 7u) != 0 || !aligned16(a->q4) || !aligned16(a->q4_scales)) {
        return LYRAQ_ERR_INVALID_ARG;
    }
    if (a->q4 != nullptr) {
        if (a->q4_format != LYRAQ_NVFP4 && a->q4_format != LYRAQ_MXFP4) {
            return LYRAQ_ERR_INVALID_ARG;
        }
        if ((a->dim & 31u) != 0) {
            return LYRAQ_ERR_UNSUPPORTED;
        }
    }
    if (outputs_clash(*a)) {
        return LYRAQ_ERR_INVALID_ARG;
    }
    const int sms = device_sm_count();
    if (sms <= 0) {
        return LYRAQ_ERR_CUDA;
    }
    NormParams p{};
    p.y = a->y; p.x = a->x; p.x_out = a->x_out; p.h = a->h; p.qf8 = a->qf8; p.q4 = a->q4; p.q4_sf = a->q4_scales;
    p.gate = a->gate; p.scale = a->scale; p.shift = a->shift; p.w1 = a->post_weight; p.w2 = a->pre_weight;
    p.f8_scale = a->f8_scale; p.q4_scale = a->q4_tensor_scale;
    p.y_batch = a->y_batch; p.y_row = a->y_row; p.x_batch = a->x_batch; p.x_row = a->x_row;
    p.xo_batch = a->x_out_batch; p.xo_row = a->x_out_row; p.h_batch = a->h_batch; p.h_row = a->h_row;
    p.gate_batch = a->gate_batch; p.scale_batch = a->scale_batch; p.shift_batch = a->shift_batch;
    p.rows = (unsigned)(a->batch * a->seq_len); p.seq = (unsigned)a->seq_len; p.dim = (int)a->dim; p.post = a->post; p.pre = a->pre;
    p.r = a->residual_scale; p.eps = a->eps;
    p.atoms = a->q4 != nullptr ? fp4_atoms(a->dim, a->q4_format) : 0;
    const NormSplit split = norm_split(p.rows, p.dim, sms);
    const unsigned  grid  = split.warp ? (p.rows + 7) / 8 : p.rows;
    auto launch = [&](auto* kernel) {
        return launch_kernel(kernel, grid, (unsigned)split.threads, (size_t)0, (cudaStream_t)stream, 1u, p);
    };
    const bool all  = p.w1 != nullptr && p.gate != nullptr && p.w2 != nullptr && p.scale != nullptr && p.shift != nullptr && p.x_out != nullptr;
    const bool full = !split.warp && p.dim == 8 * split.vpt * split.threads;
    auto pick_split = [&](auto type, auto fmt, auto every) {
        using T             = decltype(type);
        constexpr int  kFmt = decltype(fmt)::value;
        constexpr bool kAll = decltype(every)::value;
        if (split.warp) {
            return split.vpt == 1   ? launch(norm_residual_kernel<T, 1, kFmt, true, kAll, false>)
                   : split.vpt == 2 ? launch(norm_residual_kernel<T, 2, kFmt, true, kAll, false>)
                   : split.vpt == 3 ? launch(norm_residual_kernel<T, 3, kFmt, true, kAll, false>)
                   : split.vpt == 4 ? launch(norm_residual_kernel<T, 4, kFmt, true, kAll, false>)
                                    : launch(norm_residual_kernel<T, 5, kFmt, true, kAll, false>);
        }
        if (kAll && full) {
            return split.vpt == 1   ? launch(norm_residual_kernel<T, 1, kFmt, false, true, true>)
                   : split.vpt == 2 ? launch(norm_residual_kernel<T, 2, kFmt, false, true, true>)
                   : split.vpt == 3 ? launch(norm_residual_kernel<T, 3, kFmt, false, true, true>)
                                    : launch(norm_residual_kernel<T, 4, kFmt, false, true, true>);
        }
        return split.vpt == 1               ? launch(norm_residual_kernel<T, 1, kFmt, false, kAll, false>)
               : split.vpt == 2               ? launch(norm_residual_kernel<T, 2, kFmt, false, kAll, false>)
               : split.vpt == 3               ? launch(norm_residual_kernel<T, 3, kFmt, false, kAll, false>)
                                              : launch(norm_residual_kernel<T, 4, kFmt, false, kAll, false>);
    };
    auto pick_all = [&](auto type, auto fmt) {
        return all ? pick_split(type, fmt, std::integral_constant<bool, true>{}) : pick_split(type, fmt, std::integral_constant<bool, false>{});
    };
    auto pick_fmt = [&](auto type) {
        return a->q4 == nullptr                ? pick_all(type, std::integral_constant<int, -1>{})
               : a->q4_format == LYRAQ_NVFP4   ? pick_all(type, std::integral_constant<int, LYRAQ_NVFP4>{})
                                               : pick_all(type, std::integral_constant<int, LYRAQ_MXFP4>{});
    };
    const cudaError_t e = a->dtype == LYRAQ_BF16 ? pick_fmt(__nv_bfloat16{}) : pick_fmt(__half{});
    return cuda_status(e, "cudaLaunchKernelEx(norm_residual_kernel)");
}
