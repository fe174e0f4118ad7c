// FP8 linear with block scales for few tokens: Y[m,n] = T(epi(sum_kb s_x s_w (X W^T of the block) + beta R + bias)) with up to 16 rows of X.
//
// What bounds it is the weight: every byte of it is read once (26 MB for [5120, 5120], 4.0 us of HBM), the arithmetic is negligible.  So the operands
// change places, 128 rows of W on the M side of the MMA, the rows of X (16) on its N side, and K is split over the CTAs of a cluster until all
// SMs stream (measured: 9.4, 16.4 for the 71 MB of [13824, 5120], 5.4 for [1280, 5120]).  The scales are any fp32 numbers, so each K block of 128 is a product of its own; with 16 columns each, tensor memory holds 16 of them, and
// the warps that add them up, times their factors, are never waited for.  The CTAs' partial sums meet through distributed shared memory: each CTA of
// the cluster owns a share of the token columns, receives the others' partials for them and adds them in rank order, so the result does not depend
// on timing.  Not kept: mma.sync with W from global memory to registers, 16 rows of W a thread block (11.7 us) or an equal share of them an SM (13.2): rounds of
// loads that wait for one another.
//
//   warp 0   : TMA producer of W (128 x 128 B a stage), and of X where it is FP8.  Before it waits for the kernels in front of it, it asks its share of W
//              into L2: the weight stream starts while those still run.  A prefetch is not a read: whatever they write is what the loads behind the
//              wait see.
//   warp 1   : MMAs; the warp owns tensor memory
//   warps 2-5: rows of X that are not FP8 yet, quantized for the K blocks that the CTA reads, behind the weight stream (saves a launch and the way through
//              memory); then products -> sums -> shared memory of the owning CTA -> sum, epilogue, store
// All waits are bounded.  A timeout sets the status word and the abort flag of every CTA of the cluster: the sums a CTA stores need the partial
// sums of all of them, so when one gives up none of the cluster stores anything.
#include "fp8_block.cuh"
#include "sm100_ptx.cuh"

namespace lyraq {

using namespace sm100;

int make_tmap_bytes_2d(CUtensorMap* map, const void* base, uint64_t rows, uint64_t k_bytes, uint64_t row_stride_bytes,    // gemm_dense.cu
                       uint32_t box_rows, uint32_t box_bytes, bool swizzle128);

namespace fp8b {
namespace rows {

constexpr int kWRows    = 128;
constexpr int kRows     = kFewRows;
constexpr int kThreads  = 192;
constexpr int kMaxStages = 4;
constexpr int kWTile    = kWRows * kBlock;      // 16 KB
constexpr int kBufs     = 16;                   // products in tensor memory, 16 columns each
constexpr int kTmemCols = kBufs * kRows;        // 256: two CTAs share an SM
constexpr int kHalfSm   = 114000;               // shared memory with which they do

// Shared memory: W stages | X [K block][8 or 16 rows x 128 B] | partial sums of the cluster [rank][column][row of W] | scales of X [K block][16] | of W [K block] |
// barriers.  Up to eight rows of X take half a tile; the MMA's other eight columns come from whatever lies behind it and are not looked at.
struct Layout {
    int stages, kbs, x_tile;
    __host__ __device__ constexpr int x() const { return stages * kWTile; }
    __host__ __device__ constexpr int red() const { return x() + kbs * x_tile; }
    __host__ __device__ constexpr int scales() const { return red() + kRows * kWRows * 4; }
    __host__ __device__ constexpr int bars() const { return scales() + kbs * (kRows + 4) * 4; }
    __host__ __device__ constexpr int bytes() const { return bars() + 8 * (2 * kMaxStages + 2 * kBufs + 1) + 16 + 1024; }
};
constexpr int kMaxKb = 64;                      // K blocks of a CTA: their X stays in shared memory
static_assert(Layout{kMaxStages, kMaxKb, kRows * kBlock}.bytes() <= 227 * 1024 && Layout{2, 18, kRows * kBlock}.bytes() <= kHalfSm, "");
// four stages, or two or three where that lets two CTAs share an SM
constexpr Layout layout_of(int m, int kbs)
{
    const int x_tile = (m <= 8 ? 8 : kRows) * kBlock;
    for (int s = kMaxStages; s >= 2; --s) {
        if (Layout{s, kbs, x_tile}.bytes() <= kHalfSm) {
            return Layout{s, kbs, x_tile};
        }
    }
    return Layout{kMaxStages, kbs, x_tile};
}

__device__ __forceinline__ void tma_prefetch_2d(const CUtensorMap* m, int x, int y)
{
    asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global [%0, {%1, %2}];" ::"l"(reinterpret_cast<uint64_t>(m)), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ void st_cluster_f32(uint32_t cluster_addr, float v)
{
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(cluster_addr), "f"(v) : "memory");
}
__device__ __forceinline__ void st_cluster_u32(uint32_t cluster_addr, uint32_t v)
{
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(cluster_addr), "r"(v) : "memory");
}
// the four warps of the sums
__device__ __forceinline__ void sync_sums() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

template<typename T> __device__ __forceinline__ void finish(const GemmParams& p, float acc, int m, int n)
{
    const size_t at = (size_t)m * (size_t)p.N + (size_t)n;
    float        t  = acc;
    if (p.residual != nullptr) {
        t = fmaf(p.beta, to_f32(reinterpret_cast<const T*>(p.residual)[at]), t);
    }
    if (p.bias != nullptr) {
        t += to_f32(reinterpret_cast<const T*>(p.bias)[n]);
    }
    if (p.gelu) {
        t = gelu_tanh_f32x2(make_float2(t, t)).x;   // as the other kernel forms it
    }
    reinterpret_cast<T*>(p.C)[at] = from_f32<T>(t);
}

// X: the type of the rows, or void where they are FP8
template<typename X>
__global__ void __launch_bounds__(kThreads, 2)
gemm_fp8_block_rows_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x, const GemmParams p, const Input in,
                           const int num_kb, const int splits, const Layout lay, const int stalled_rank, const unsigned wait_limit_ms)
{
    constexpr bool     kQuantize = !std::is_void_v<X>;
    constexpr uint32_t kIdesc    = umma_idesc(1u, 0u, kWRows, kRows);
    extern __shared__ uint8_t smem_raw[];
    // the dynamic shared window starts at the same offset in every CTA of the kernel, so the layout is that of the peers too
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t*       gen_base  = smem_raw + (smem_base - smem_u32(smem_raw));
    const uint32_t bars      = smem_base + (uint32_t)lay.bars();
    auto full_bar      = [&](int s) { return bars + 8u * (uint32_t)s; };
    auto empty_bar     = [&](int s) { return bars + 8u * (uint32_t)(kMaxStages + s); };
    auto acc_full_bar  = [&](int b) { return bars + 8u * (uint32_t)(2 * kMaxStages + b); };
    auto acc_empty_bar = [&](int b) { return bars + 8u * (uint32_t)(2 * kMaxStages + kBufs + b); };
    const uint32_t x_bar      = bars + 8u * (2 * kMaxStages + 2 * kBufs);
    uint32_t*      tmem_slot  = reinterpret_cast<uint32_t*>(gen_base + lay.bars() + 8 * (2 * kMaxStages + 2 * kBufs + 1));
    volatile int*  abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int      warp = warp_index();
    const int      lane = threadIdx.x & 31;
    const int      rank = (int)cluster_ctarank();
    const int      tile = (int)blockIdx.x / splits;
    const int      n0   = tile * kWRows;
    const int      kb0  = (int)((long long)num_kb * rank / splits);
    const int      n_kb = (int)((long long)num_kb * (rank + 1) / splits) - kb0;
    const uint64_t wait_limit_ns = (uint64_t)wait_limit_ms * 1000000u;
    // records a wait that ran out and stops the whole cluster; its writes are visible to the peers behind the barrier in front of the sums
    auto give_up = [&](unsigned code) {
        report_timeout(p.status, code);
        for (int r = 0; r < splits; ++r) {
            st_cluster_u32(map_to_cta(smem_u32(const_cast<int*>(abort_flag)), (uint32_t)r), 1u);
        }
    };

    grid_launch_dependents();
    if (threadIdx.x == 0) {
        for (int s = 0; s < lay.stages; ++s) {
            mbar_init(full_bar(s), 1);
            mbar_init(empty_bar(s), 1);
        }
        for (int b = 0; b < kBufs; ++b) {
            mbar_init(acc_full_bar(b), 1);
            mbar_init(acc_empty_bar(b), 4);
        }
        mbar_init(x_bar, kQuantize ? 4 : 1);
        *abort_flag = 0;
        fence_barrier_init();
        for (int i = 0; i < n_kb; ++i) {
            tma_prefetch_2d(&tmap_w, (kb0 + i) * kBlock, n0);
        }
        prefetch_tensormap(&tmap_x);
    }
    if (warp == 1) {
        tmem_alloc(smem_u32(tmem_slot), kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before_sync();
    cluster_sync_all();   // every CTA of the cluster runs before a peer writes to its shared memory
    tc_fence_after_sync();
    const uint32_t tmem_base = *tmem_slot;
    grid_dependency_wait();

    float* const sx = reinterpret_cast<float*>(gen_base + lay.scales());    // [K block][16]
    float* const sw = sx + lay.kbs * kRows;
    if (warp == 0) {
        int      stage = 0, issued = 0;
        uint32_t phase = 0;
        if (!kQuantize && rank != stalled_rank && elect_one()) {
            mbar_arrive_expect_tx(x_bar, (uint32_t)(n_kb * lay.x_tile));
            for (int i = 0; i < n_kb; ++i) {
                tma_load_2d(smem_base + (uint32_t)(lay.x() + i * lay.x_tile), &tmap_x, x_bar, (kb0 + i) * kBlock, 0);
            }
        }
        __syncwarp();
        for (int i = 0; i < n_kb && rank != stalled_rank; ++i) {
            if (!mbar_wait_warp(empty_bar(stage), phase ^ 1u, abort_flag, wait_limit_ns)) {
                if (lane == 0) {
                    give_up(0xa100u | (unsigned)stage);
                }
                break;
            }
            if (elect_one()) {
                mbar_arrive_expect_tx(full_bar(stage), (uint32_t)kWTile);
                tma_load_2d(smem_base + (uint32_t)(stage * kWTile), &tmap_w, full_bar(stage), (kb0 + i) * kBlock, n0);
            }
            ++issued;
            if (++stage == lay.stages) {
                stage = 0;
                phase ^= 1u;
            }
        }
        // no copy may be in flight when the block leaves
        auto settle = [&](uint32_t bar, uint32_t parity, unsigned code) {
            const uint64_t t0 = global_timer_ns();
            while (!mbar_try_wait(bar, parity)) {
                if (global_timer_ns() - t0 > wait_limit_ns) {
                    report_timeout(p.status, code);
                    break;
                }
            }
        };
        int      s  = stage;
        uint32_t ph = phase;
        for (int i = 0; i < lay.stages && i < issued; ++i) {
            if (s == 0) {
                s = lay.stages;
                ph ^= 1u;
            }
            --s;
            settle(full_bar(s), ph, 0xa500u | (unsigned)s);
        }
        if (!kQuantize && rank != stalled_rank) {
            settle(x_bar, 0u, 0xa510u);
        }
    } else if (warp == 1) {
        int      stage = 0;
        uint32_t phase = 0;
        bool     ok    = mbar_wait_warp(x_bar, 0u, abort_flag, wait_limit_ns);
        if (!ok && lane == 0) {
            give_up(0xa210u);
        }
        for (int i = 0; ok && i < n_kb; ++i) {
            const int buf = i % kBufs;
            if (!mbar_wait_warp(acc_empty_bar(buf), (uint32_t)(i / kBufs & 1) ^ 1u, abort_flag, wait_limit_ns) ||
                !mbar_wait_warp(full_bar(stage), phase, abort_flag, wait_limit_ns)) {
                if (lane == 0) {
                    give_up(0xa200u | (unsigned)stage);
                }
                break;
            }
            tc_fence_after_sync();
            if (elect_one()) {
                const uint64_t adesc = umma_desc_k_sw128(smem_base + (uint32_t)(stage * kWTile)), bdesc = umma_desc_k_sw128(smem_base + (uint32_t)(lay.x() + i * lay.x_tile));
                const uint32_t d     = tmem_base + (uint32_t)(buf * kRows);
                const int      steps = min(kBlock, p.K - (kb0 + i) * kBlock + 31) / 32;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    if (k < steps) {
                        mma_f8f6f4(d, adesc + (uint64_t)(2 * k), bdesc + (uint64_t)(2 * k), kIdesc, k > 0 ? 1u : 0u);
                    }
                }
                tc_commit(empty_bar(stage));
                tc_commit(acc_full_bar(buf));
            }
            if (++stage == lay.stages) {
                stage = 0;
                phase ^= 1u;
            }
        }
    } else {
        const int at = (int)threadIdx.x - 64;
        for (int i = at; i < n_kb; i += 128) {
            sw[i] = ld_f32(p.ws + (size_t)tile * (size_t)num_kb + (size_t)(kb0 + i));
        }
        if constexpr (kQuantize) {
            constexpr int kPer  = 16 / (int)sizeof(X);
            constexpr int kVecs = (int)sizeof(X);
            constexpr int kTwo  = 2;      // eight lanes a block, two blocks of each lane at a time
            const int blocks = p.M * n_kb, lane8 = at & 7;
            for (int i0 = 0; i0 < blocks; i0 += kTwo * 16) {
                Vec16 v[kTwo][kVecs];
#pragma unroll
                for (int u = 0; u < kTwo; ++u) {
                    const int i = i0 + u * 16 + at / 8, row = i / n_kb, kb = i - row * n_kb, col = (kb0 + kb) * kBlock + lane8 * 16;
#pragma unroll
                    for (int a = 0; a < kVecs; ++a) {
                        v[u][a] = Vec16{};
                        if (i < blocks && col < p.K) {      // K is a multiple of 16: a lane's values are there or not
                            v[u][a] = ld_nc_16(reinterpret_cast<const X*>(in.x) + (size_t)row * in.ldx + (size_t)(col + a * kPer));
                        }
                    }
                }
#pragma unroll
                for (int u = 0; u < kTwo; ++u) {
                    const int i = i0 + u * 16 + at / 8, row = i / n_kb, kb = i - row * n_kb;
                    uint32_t  amax = amax16_values<X>(v[u]);
#pragma unroll
                    for (int d = 1; d < 8; d *= 2) {
                        amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, d));
                    }
                    const Divisor d = divisor_of(amax);
                    if (i < blocks) {      // 16 bytes of a row of 128, in the 128-byte swizzle
                        *reinterpret_cast<Vec16*>(gen_base + lay.x() + kb * lay.x_tile + row * kBlock + ((lane8 ^ (row & 7)) << 4)) = encode16<X>(v[u], d);
                        if (lane8 == 0) {
                            sx[kb * kRows + row] = d.s;
                        }
                    }
                }
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(x_bar);
            }
        } else {
            for (int i = at; i < p.M * n_kb; i += 128) {
                const int kb = i / p.M, row = i - kb * p.M;
                sx[kb * kRows + row] = ld_f32(in.scales.p + (size_t)row * in.scales.row_step + (size_t)(kb0 + kb) * in.scales.block_step);
            }
        }
        sync_sums();      // the scales are there
    }
    // ---- accumulator lane = row of W; the CTA of rank r owns the token columns [r kRows / S, (r + 1) kRows / S)
    const int slice = kRows / splits;
    const int wrow  = (warp & 3) * 32 + lane;
    if (warp >= 2) {
        float acc[kRows];
#pragma unroll
        for (int c = 0; c < kRows; ++c) {
            acc[c] = 0.0f;
        }
        bool ok = true;
        for (int i = 0; i < n_kb; ++i) {
            const int buf = i % kBufs;
            if (!mbar_wait_warp(acc_full_bar(buf), (uint32_t)(i / kBufs & 1), abort_flag, wait_limit_ns)) {
                if (lane == 0) {
                    give_up(0xa300u);
                }
                ok = false;
                break;
            }
            tc_fence_after_sync();
            uint32_t v[kRows];
            tmem_ld_32x16(tmem_base + ((uint32_t)((warp & 3) * 32) << 16) + (uint32_t)(buf * kRows), v);
            tmem_ld_wait();
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(acc_empty_bar(buf));
            }
            const float s = sw[i];
#pragma unroll
            for (int c = 0; c < kRows; c += 4) {
                const float4 f = *reinterpret_cast<const float4*>(sx + i * kRows + c);
                acc[c]     = fmaf(f.x * s, __uint_as_float(v[c]), acc[c]);
                acc[c + 1] = fmaf(f.y * s, __uint_as_float(v[c + 1]), acc[c + 1]);
                acc[c + 2] = fmaf(f.z * s, __uint_as_float(v[c + 2]), acc[c + 2]);
                acc[c + 3] = fmaf(f.w * s, __uint_as_float(v[c + 3]), acc[c + 3]);
            }
        }
        if (ok) {
#pragma unroll
            for (int c = 0; c < kRows; ++c) {
                if (c < p.M) {
                    const int      owner = c / slice;
                    const uint32_t to    = smem_base + (uint32_t)lay.red() + (uint32_t)(((rank * slice + c - owner * slice) * kWRows + wrow) * 4);
                    st_cluster_f32(map_to_cta(to, (uint32_t)owner), acc[c]);
                }
            }
        }
    }
    tc_fence_before_sync();
    cluster_sync_all();   // all partials of this CTA's columns have arrived
    tc_fence_after_sync();
    if (warp == 1) {
        tmem_dealloc(tmem_base, kTmemCols);
    }
    if (warp >= 2 && *abort_flag == 0 && n0 + wrow < p.N) {
        const float* red = reinterpret_cast<const float*>(gen_base + lay.red());
        for (int c = 0; c < slice; ++c) {
            const int m = rank * slice + c;
            if (m >= p.M) {
                break;
            }
            float acc = red[c * kWRows + wrow];
            for (int s = 1; s < splits; ++s) {
                acc += red[(s * slice + c) * kWRows + wrow];
            }
            if (p.c_dtype == LYRAQ_BF16) {
                finish<__nv_bfloat16>(p, acc, m, n0 + wrow);
            } else if (p.c_dtype == LYRAQ_F16) {
                finish<__half>(p, acc, m, n0 + wrow);
            } else {
                finish<float>(p, acc, m, n0 + wrow);
            }
        }
    }
}

// Clusters of `size` CTAs that run at once, two CTAs to an SM (a cluster lies within one GPC, and clusters of 4 or 8 leave some of a GPC's
// SMs over: measured on a B200 with the FP8 kernel of the same shape, gemm_skinny.cu).
static long clusters_at_once(int size, int sms) { return size == 2 ? sms : size == 4 ? sms * 71l / 148 : sms * 33l / 148; }

// CTAs along K: as many (1, 2, 4 or 8) as keep the clusters within one wave, with at least two K blocks each, and what a CTA's shared memory wants.
static int pick_splits(long tiles, int num_kb, int sms)
{
    int s = 1;
    while (s < 8 && num_kb >= 2 * (2 * s) && (tiles <= clusters_at_once(2 * s, sms) || (num_kb + s - 1) / s > kMaxKb)) {
        s *= 2;
    }
    return s;
}
static int blocks_of_cta(int num_kb, int splits) { return (num_kb + splits - 1) / splits; }

// Test hook (lyraq_debug_fp8_block_rows_wait_test)
static int          g_stalled_rank  = -1;
static unsigned int g_wait_limit_ms = kWaitLimitNs / 1000000;

template<typename X> static int launch(const Input& in, const uint8_t* W, const GemmParams& p, int sms, cudaStream_t stream)
{
    const int   n_tiles = (int)(((long)p.N + kWRows - 1) / kWRows), num_kb = (p.K + kBlock - 1) / kBlock;
    const int   splits = pick_splits(n_tiles, num_kb, sms);
    const Layout lay = layout_of(p.M, blocks_of_cta(num_kb, splits));
    CUtensorMap tw, tx;
    int         st = make_tmap_bytes_2d(&tw, W, (uint64_t)p.N, (uint64_t)p.K, (uint64_t)p.K, kWRows, kBlock, true);
    tx             = tw;    // never used where the rows are quantized here
    if (st == LYRAQ_OK && std::is_void_v<X>) {
        st = make_tmap_bytes_2d(&tx, in.codes, (uint64_t)p.M, (uint64_t)p.K, (uint64_t)p.K, (uint32_t)(lay.x_tile / kBlock), kBlock, true);
    }
    static bool smem_raised[64] = {};
    if (st == LYRAQ_OK) {
        st = raise_dynamic_smem_once(gemm_fp8_block_rows_kernel<X>, Layout{kMaxStages, kMaxKb, kRows * kBlock}.bytes(), smem_raised, "cudaFuncSetAttribute(gemm_fp8_block_rows_kernel)");
    }
    if (st != LYRAQ_OK) {
        return st;
    }
    return cuda_status(launch_kernel(gemm_fp8_block_rows_kernel<X>, (unsigned)(n_tiles * splits), (unsigned)kThreads, (size_t)lay.bytes(), stream,
                                     (unsigned)splits, tw, tx, p, in, num_kb, splits, lay, g_stalled_rank, g_wait_limit_ms),
                       "cudaLaunchKernelEx(gemm_fp8_block_rows_kernel)");
}

}  // namespace rows

int launch_rows(const Input& X, const uint8_t* W, const GemmParams& p, int sms, cudaStream_t stream)
{
    if (X.codes != nullptr) {
        return rows::launch<void>(X, W, p, sms, stream);
    }
    return X.dtype == LYRAQ_BF16 ? rows::launch<__nv_bfloat16>(X, W, p, sms, stream)
           : X.dtype == LYRAQ_F16 ? rows::launch<__half>(X, W, p, sms, stream)
                                  : rows::launch<float>(X, W, p, sms, stream);
}

static int blocks_of_cta(int n, int k, int sms)
{
    const int num_kb = (k + kBlock - 1) / kBlock;
    return rows::blocks_of_cta(num_kb, rows::pick_splits(((long)n + rows::kWRows - 1) / rows::kWRows, num_kb, sms));
}

bool rows_fit(int n, int k, int sms) { return blocks_of_cta(n, k, sms) <= rows::kMaxKb; }

// Quantizing in the kernel saves a launch, and every CTA does it for the K blocks it reads, 32 blocks of rows at a time, while a launch of its own hides
// behind the weight stream where that is long.  In the kernel against apart, us: 1 row of [1280, 2048] (2 K blocks a CTA) 4.3 / 4.6, of [1280, 5120] (5) 5.4 / 5.9,
// 4 rows of it 5.9 / 6.3, 8 rows 7.3 / 6.6, 1 row of [5120, 5120] (10) 9.5 / 9.3, of [13824, 5120] (20) 16.5 / 16.3.
bool rows_quantize_pays(int m, int n, int k, int sms)
{
    const int kbs = blocks_of_cta(n, k, sms);
    return kbs <= 8 && m * kbs <= 24;
}

}  // namespace fp8b
}  // namespace lyraq

extern "C" int lyraq_debug_fp8_block_rows_wait_test(int stalled_rank, unsigned int wait_limit_ms)
{
    lyraq::fp8b::rows::g_stalled_rank  = stalled_rank;
    lyraq::fp8b::rows::g_wait_limit_ms = wait_limit_ms == 0 ? (unsigned int)(lyraq::sm100::kWaitLimitNs / 1000000) : wait_limit_ms;
    return LYRAQ_OK;
}
