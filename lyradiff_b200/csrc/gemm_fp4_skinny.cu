// FP4 linear for few tokens: Y[m,n] = T(epi(g_x g_w (X W^T) + beta R + bias)) with so few rows of X that the tiles of gemm_fp4_kernel leave
// most of the chip idle.
//
// What bounds it is the weight: every byte of it is read once (16 MB for [9216, 3072], 2.4 us of HBM; measured 5.1), the arithmetic is negligible.  So the
// operands change places, 128 rows of W on the M side of the MMA, the rows of X (padded to 16 by TMA) on its N side, and K is split over the
// CTAs of a cluster until all SMs stream.  The partial products meet through distributed shared memory: each CTA of the cluster owns a share of
// the token columns, receives the others' partials for them and adds them in rank order, so the result does not depend on timing.
//
//   warp 0   : TMA producer (W 128 x 128 B, X 16 x 128 B, the scale atoms of W, the first half of X's: rows 0 to 15).  Before it waits for the
//              kernels in front of it, it asks its share of W into L2: the weight stream starts while the quantize of X still runs.  A
//              prefetch is not a read: whatever that kernel writes is what the loads behind the wait see.
//   warp 1   : scales to tensor memory, MMAs; the warp owns tensor memory
//   warps 2-5: accumulator -> shared memory of the owning CTA -> sum, epilogue, store.  For rows of X that are not FP4 yet they fill the stages' X and its
//              scales before that, 32 values a thread (fp4_deal.h has the order): every CTA quantizes what it reads, behind the weight stream, which saves a launch
//              and the way through memory
// All waits are bounded.  A timeout sets the status word and the abort flag of every CTA of the cluster: the sums a CTA stores need the partial
// products of all of them, so when one gives up none of the cluster stores anything.
#include "fp4_deal.h"
#include "gemm_fp4.cuh"

namespace lyraq {

using namespace sm100;

int make_tmap_bytes_2d(CUtensorMap* map, const void* base, uint64_t rows, uint64_t k_bytes, uint64_t row_stride_bytes,    // gemm_dense.cu
                       uint32_t box_rows, uint32_t box_bytes, bool swizzle128);
int make_tmap_atoms(CUtensorMap* map, const void* base, uint64_t row_blocks, uint64_t atoms, uint32_t box_blocks, uint32_t box_atoms,  // gemm_dense.cu
                    uint32_t box_words);

namespace fp4 {
namespace skinny {

constexpr int kWRows    = 128;
constexpr int kRows     = kFp4SkinnyRows;
constexpr int kRowBytes = 128;
constexpr int kBlockK   = 256;
constexpr int kThreads  = 192;
constexpr int kStages   = kDealStages;   // two CTAs share an SM

template<int FORMAT> struct Smem {
    static constexpr int kAtoms     = kBlockK / fp4_atom_k(FORMAT);
    static constexpr int kW         = kWRows * kRowBytes;
    static constexpr int kX         = kRows * kRowBytes;
    static constexpr int kSw        = kAtoms * 512;
    static constexpr int kSx        = kAtoms * 256;      // rows 0 to 15 of an atom are its first 256 bytes
    // an atom's copy reads 512 bytes: the last half atom is followed by the next stage or the sums, which only reach lanes that nobody reads
    static constexpr int kBytes     = kW + kX + kSw + kSx;
    static constexpr int kStage     = (kBytes + 1023) / 1024 * 1024;
    static constexpr int kRedOffset = kStages * kStage;
    static constexpr int kRedBytes  = kRows * kWRows * 4;
    static constexpr int kBarOffset = kRedOffset + kRedBytes;
    static constexpr int kTotal     = kBarOffset + 256 + 1024;
    static constexpr int kSlotCols  = kAtoms * 8;
    static_assert(kTotal <= 115000, "two CTAs share an SM");
    static_assert(16 + kStages * kSlotCols <= 256, "and its tensor memory");
};

__device__ __forceinline__ void tma_prefetch_2d(const CUtensorMap* m, int x, int y)
{
    asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global [%0, {%1, %2}];" ::"l"(reinterpret_cast<uint64_t>(m)), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ void tma_prefetch_3d(const CUtensorMap* m, int x, int y, int z)
{
    asm volatile("cp.async.bulk.prefetch.tensor.3d.L2.global [%0, {%1, %2, %3}];" ::"l"(reinterpret_cast<uint64_t>(m)), "r"(x), "r"(y), "r"(z)
                 : "memory");
}
__device__ __forceinline__ void st_cluster_f32(uint32_t cluster_addr, float v)
{
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(cluster_addr), "f"(v) : "memory");
}
__device__ __forceinline__ void st_cluster_u32(uint32_t cluster_addr, uint32_t v)
{
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(cluster_addr), "r"(v) : "memory");
}

template<typename T> __device__ __forceinline__ void finish(const Fp4GemmParams& p, float acc, float scale, int m, int n)
{
    const size_t at = (size_t)m * (size_t)p.N + (size_t)n;
    float        t  = acc * scale;
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

// X: the type of the rows, or void where they are FP4
template<int FORMAT, typename X>
__global__ void __launch_bounds__(kThreads, 2)
gemm_fp4_skinny_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_sw,
                       const __grid_constant__ CUtensorMap tmap_sx, const Fp4GemmParams p, const void* rows, const size_t ldx, const int num_kb,
                       const int splits, const int stalled_rank, const unsigned wait_limit_ms)
{
    using S = Smem<FORMAT>;
    constexpr bool kQuantize = !std::is_void_v<X>;
    extern __shared__ uint8_t smem_raw[];
    // the dynamic shared window starts at the same offset in every CTA of the kernel, so the layout is that of the peers too
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t*       gen_base  = smem_raw + (smem_base - smem_u32(smem_raw));
    const uint32_t bars      = smem_base + S::kBarOffset;
    auto full_bar  = [&](int s) { return bars + 8u * s; };
    auto empty_bar = [&](int s) { return bars + 8u * (kStages + s); };
    const uint32_t acc_bar    = bars + 8u * (2 * kStages);
    uint32_t*      tmem_slot  = reinterpret_cast<uint32_t*>(gen_base + S::kBarOffset + 8 * (2 * kStages + 1));
    volatile int*  abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int      warp = warp_index();
    const int      lane = threadIdx.x & 31;
    const int      rank = (int)cluster_ctarank();
    const int      tile = (int)blockIdx.x / splits;
    const int      n0   = tile * kWRows;
    const int      kb0  = (int)((long long)num_kb * rank / splits);
    const int      kb1  = (int)((long long)num_kb * (rank + 1) / splits);
    const uint64_t wait_limit_ns = (uint64_t)wait_limit_ms * 1000000u;
    const FewRowsDeal deal = few_rows_deal(p.M);   // which K blocks a quantizing warp takes
    // records a wait that ran out and stops the whole cluster; its writes are visible to the peers behind the barrier in front of the sums
    auto give_up = [&](unsigned code) {
        report_timeout(p.status, code);
        for (int r = 0; r < splits; ++r) {
            st_cluster_u32(map_to_cta(smem_u32(const_cast<int*>(abort_flag)), (uint32_t)r), 1u);
        }
    };

    grid_launch_dependents();
    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(full_bar(s), 1u + (kQuantize ? (uint32_t)deal.warps_per_kb : 0u));
            mbar_init(empty_bar(s), 1);
        }
        mbar_init(acc_bar, 1);
        *abort_flag = 0;
        fence_barrier_init();
        for (int kb = kb0; kb < kb1; ++kb) {
            tma_prefetch_2d(&tmap_w, kb * kRowBytes, n0);
            tma_prefetch_3d(&tmap_sw, 0, kb * S::kAtoms, tile);
        }
        prefetch_tensormap(&tmap_x);
        prefetch_tensormap(&tmap_sx);
    }
    if (warp == 1) {
        tmem_alloc(smem_u32(tmem_slot), 256);
        tmem_relinquish();
    }
    tc_fence_before_sync();
    cluster_sync_all();   // every CTA of the cluster runs before a peer writes to its shared memory
    tc_fence_after_sync();
    const uint32_t tmem_base = *tmem_slot;
    grid_dependency_wait();

    if (warp == 0) {
        int      stage = 0, issued = 0;
        uint32_t phase = 0;
        for (int kb = kb0; kb < kb1 && rank != stalled_rank; ++kb) {
            if (!mbar_wait_warp(empty_bar(stage), phase ^ 1u, abort_flag, wait_limit_ns)) {
                if (lane == 0) {
                    give_up(0x6100u | (unsigned)stage);
                }
                break;
            }
            if (elect_one()) {
                const uint32_t w = smem_base + stage * S::kStage, x = w + S::kW, sw = x + S::kX, sx = sw + S::kSw;
                mbar_arrive_expect_tx(full_bar(stage), (uint32_t)(kQuantize ? S::kW + S::kSw : S::kBytes));
                tma_load_2d(w, &tmap_w, full_bar(stage), kb * kRowBytes, n0);
                tma_load_3d(sw, &tmap_sw, full_bar(stage), 0, kb * S::kAtoms, tile);
                if (!kQuantize) {
                    tma_load_2d(x, &tmap_x, full_bar(stage), kb * kRowBytes, 0);
                    tma_load_3d(sx, &tmap_sx, full_bar(stage), 0, kb * S::kAtoms, 0);
                }
            }
            ++issued;
            if (++stage == kStages) {
                stage = 0;
                phase ^= 1u;
            }
        }
        // no copy may be in flight when the block leaves
        int      s  = stage;
        uint32_t ph = phase;
        for (int i = 0; i < kStages && i < issued; ++i) {
            if (s == 0) {
                s = kStages;
                ph ^= 1u;
            }
            --s;
            const uint64_t t0 = global_timer_ns();
            while (!mbar_try_wait(full_bar(s), ph)) {
                if (global_timer_ns() - t0 > wait_limit_ns) {
                    report_timeout(p.status, 0x6500u | (unsigned)s);
                    break;
                }
            }
        }
    } else if (warp == 1) {
        int      stage = 0;
        uint32_t phase = 0;
        for (int kb = kb0; kb < kb1; ++kb) {
            if (!mbar_wait_warp(full_bar(stage), phase, abort_flag, wait_limit_ns)) {
                if (lane == 0) {
                    give_up(0x6200u | (unsigned)stage);
                }
                break;
            }
            tc_fence_after_sync();
            const uint32_t w      = smem_base + stage * S::kStage;
            const uint64_t adesc  = umma_desc_k_sw128(w), bdesc = umma_desc_k_sw128(w + S::kW);
            const uint64_t swdesc = umma_desc_scales(w + S::kW + S::kX), sxdesc = umma_desc_scales(w + S::kW + S::kX + S::kSw);
            const uint32_t sfw    = tmem_base + 16u + (uint32_t)(stage * S::kSlotCols), sfx = sfw + S::kAtoms * 4;
            const int      steps  = min(kBlockK, p.K - kb * kBlockK + 63) / 64;
            if (elect_one()) {
#pragma unroll
                for (int a = 0; a < S::kAtoms; ++a) {
                    if (a * (4 / S::kAtoms) < steps) {
                        tmem_copy_scales<1>(sfw + a * 4, swdesc + (uint64_t)(a * 32));
                        tmem_copy_scales<1>(sfx + a * 4, sxdesc + (uint64_t)(a * 16));
#pragma unroll
                        for (int h = 0; h < 4 / S::kAtoms; ++h) {
                            const int k = a * (4 / S::kAtoms) + h;
                            if (k < steps) {
                                mma_fp4<FORMAT, 1>(tmem_base, adesc + (uint64_t)(2 * k), bdesc + (uint64_t)(2 * k),
                                                   umma_idesc_fp4(FORMAT, kWRows, kRows, 2u * h), sfw + a * 4, sfx + a * 4, (kb > kb0 || k > 0) ? 1u : 0u);
                            }
                        }
                    }
                }
                tc_commit(empty_bar(stage));
                if (kb + 1 == kb1) {
                    tc_commit(acc_bar);
                }
            }
            if (++stage == kStages) {
                stage = 0;
                phase ^= 1u;
            }
        }
    } else if constexpr (kQuantize) {
        constexpr int kPer  = 16 / (int)sizeof(X);
        constexpr int kVecs = 32 / kPer;
        // eight lanes have 256 values of a row; up to four rows, the quarters beyond them have further K blocks
        const int qw = warp - 2, j = lane & 7, quarter = lane >> 3;
        const int row   = deal.rows_log2 <= 2 ? quarter & ((1 << deal.rows_log2) - 1) : (qw & (deal.warps_per_kb - 1)) * 4 + quarter;
        const int piece = deal.rows_log2 <= 2 ? quarter >> deal.rows_log2 : 0;
        const X*  src   = reinterpret_cast<const X*>(rows) + (size_t)row * ldx;
        auto load = [&](int visit, Vec16* v) {
            const int kb = kb0 + few_rows_block(deal, qw, visit, piece);
#pragma unroll
            for (int a = 0; a < kVecs; ++a) {
                v[a] = Vec16{};
                if (row < p.M && kb < kb1 && kb * kBlockK + j * 32 < p.K) {   // K is a multiple of 32; zeros have zero codes and scales
                    v[a] = ld_nc_16(src + (size_t)kb * kBlockK + j * 32 + a * kPer);
                }
            }
        };
        Vec16 v[kVecs], ahead[kVecs];
        load(0, v);
        const Fp4Tensor tensor = fp4_tensor<FORMAT>(p.s_x);
        bool            ok     = true;
        for (int visit = 0; ok && few_rows_block(deal, qw, visit, 0) < kb1 - kb0; ++visit) {
            load(visit + 1, ahead);
            Vec16          o{};
            const uint32_t code = fp4_encode32<X, FORMAT, true>(v, tensor, o);
            // one K block after the other: each is written once its stage's last contents have been multiplied
            for (int t = 0; t < deal.per_visit; ++t) {
                const int i = few_rows_block(deal, qw, visit, t);
                if (i >= kb1 - kb0) {
                    break;
                }
                const int stage = i % kStages;
                ok = mbar_wait_warp(empty_bar(stage), (uint32_t)(i / kStages & 1) ^ 1u, abort_flag, wait_limit_ns);
                if (!ok) {
                    if (lane == 0) {
                        give_up(0x6400u | (unsigned)stage);
                    }
                    break;
                }
                if (piece == t && row < p.M) {
                    uint8_t* x  = gen_base + stage * S::kStage + S::kW;
                    uint8_t* sx = x + S::kX + S::kSw;
                    *reinterpret_cast<Vec16*>(x + row * kRowBytes + ((j ^ (row & 7)) << 4)) = o;    // the 128-byte swizzle
                    if (FORMAT == LYRAQ_NVFP4) {
                        *reinterpret_cast<uint16_t*>(sx + (j >> 1) * 256 + row * 16 + (j & 1) * 2) = (uint16_t)code;
                    } else {
                        sx[(j >> 2) * 256 + row * 16 + (j & 3)] = (uint8_t)code;
                    }
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(full_bar(stage));
                }
            }
#pragma unroll
            for (int a = 0; a < kVecs; ++a) {
                v[a] = ahead[a];
            }
        }
    }
    float scale = 0.0f;
    if (warp >= 2) {
        scale = fp4_tensor_scale(p);   // asked for before the accumulator is waited for
    }
    // ---- accumulator lane = row of W; the CTA of rank r owns the token columns [r kRows / S, (r + 1) kRows / S)
    const int slice = kRows / splits;
    const int wrow  = (warp & 3) * 32 + lane;
    if (warp >= 2) {
        if (!mbar_wait_warp(acc_bar, 0u, abort_flag, wait_limit_ns)) {
            if (lane == 0) {
                give_up(0x6300u);
            }
        } else {
            tc_fence_after_sync();
            uint32_t v[kRows];
            tmem_ld_32x16(tmem_base + ((uint32_t)((warp & 3) * 32) << 16), v);
            tmem_ld_wait();
#pragma unroll
            for (int c = 0; c < kRows; ++c) {
                if (c < p.M) {
                    const int      owner = c / slice;
                    const uint32_t at    = smem_base + S::kRedOffset + (uint32_t)(((rank * slice + c - owner * slice) * kWRows + wrow) * 4);
                    st_cluster_f32(map_to_cta(at, (uint32_t)owner), __uint_as_float(v[c]));
                }
            }
        }
    }
    tc_fence_before_sync();
    cluster_sync_all();   // all partials of this CTA's columns have arrived
    tc_fence_after_sync();
    if (warp == 1) {
        tmem_dealloc(tmem_base, 256);
    }
    if (warp >= 2 && *abort_flag == 0 && n0 + wrow < p.N) {
        const float* red = reinterpret_cast<const float*>(gen_base + S::kRedOffset);
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
                finish<__nv_bfloat16>(p, acc, scale, m, n0 + wrow);
            } else if (p.c_dtype == LYRAQ_F16) {
                finish<__half>(p, acc, scale, m, n0 + wrow);
            } else {
                finish<float>(p, acc, scale, m, n0 + wrow);
            }
        }
    }
}

// Clusters of `size` CTAs that run at once, two CTAs to an SM (a cluster lies within one GPC, and clusters of 4 or 8 leave some of a GPC's
// SMs over: measured on a B200 with the FP8 kernel of the same shape, gemm_skinny.cu).
static long clusters_at_once(int size, int sms) { return size == 2 ? sms : size == 4 ? sms * 71l / 148 : sms * 33l / 148; }

// CTAs along K: as many (1, 2, 4 or 8) as keep the clusters within one wave, with at least two K blocks each.
static int pick_splits(long tiles, int num_kb, int sms)
{
    int s = 1;
    while (s < 8 && num_kb >= 2 * (2 * s) && tiles <= clusters_at_once(2 * s, sms)) {
        s *= 2;
    }
    return s;
}

// Quantizing in the kernel saves a launch, and every CTA does it for the K blocks it reads: it pays up to 64 rows times K blocks of a CTA, rows in powers of
// two.  In the kernel against a launch of its own, nvfp4 / mxfp4, us: 1 row of [1280, 1280] 3.8 and 4.7 / 3.3 and 4.2, of [9216, 3072] (6) 6.2 and 6.4 / 5.3 and
// 5.8, 16 rows of [1280, 2048] (32) 6.1 and 6.6 / 5.3 and 6.2, of [3072, 3072] (48) 7.1 and 7.2 / 6.2 and 6.8, of [9216, 3072] (96) 11.1 and
// 9.6 / 9.6 and 8.8, of [3072, 12288] (96) 11.4 and 9.7 / 9.8 and 9.1.  Few rows over deep K: 1 row of [21504, 3072] (12) 8.3 and 9.2 / 7.6 and
// 8.2, of [28672, 8192] (32) 24.4 and 24.4 / 22.9 and 22.8, of [19072, 16128] (63) 35.3 and 34.8 / 32.3 and 32.5.
static bool quantize_pays(int m, int n, int k, int sms)
{
    const int num_kb = (k + kBlockK - 1) / kBlockK, splits = pick_splits(((long)n + kWRows - 1) / kWRows, num_kb, sms);
    int       rows   = 1;
    while (rows < m) {
        rows *= 2;
    }
    return (long long)rows * ((num_kb + splits - 1) / splits) <= 64;
}

// Test hook (lyraq_debug_fp4_skinny_wait_test)
static int          g_stalled_rank  = -1;
static unsigned int g_wait_limit_ms = kWaitLimitNs / 1000000;

template<int FORMAT, typename X>
static int launch(const Fp4Input& in, const uint8_t* W, const uint8_t* ws, const Fp4GemmParams& p, int sms, cudaStream_t stream)
{
    using S = Smem<FORMAT>;
    const int      n_tiles = (int)(((long)p.N + kWRows - 1) / kWRows);
    const int      num_kb  = (p.K + kBlockK - 1) / kBlockK;
    const int      splits  = pick_splits(n_tiles, num_kb, sms);
    const uint64_t kb = (uint64_t)p.K / 2, atoms = fp4_atoms((size_t)p.K, FORMAT);
    CUtensorMap    tw, tx, tsw, tsx;
    int            st = make_tmap_bytes_2d(&tw, W, (uint64_t)p.N, kb, kb, kWRows, kRowBytes, true);
    if (st == LYRAQ_OK) {
        st = make_tmap_atoms(&tsw, ws, ((uint64_t)p.N + 127) / 128, atoms, 1, S::kAtoms, 128);
    }
    if (!std::is_void_v<X>) {
        tx  = tw;    // never used
        tsx = tsw;
    } else {
        if (st == LYRAQ_OK) {
            st = make_tmap_bytes_2d(&tx, in.codes, (uint64_t)p.M, kb, kb, kRows, kRowBytes, true);
        }
        if (st == LYRAQ_OK) {
            st = make_tmap_atoms(&tsx, in.scales, 1, atoms, 1, S::kAtoms, 64);
        }
    }
    static bool smem_raised[64] = {};
    if (st == LYRAQ_OK) {
        st = raise_dynamic_smem_once(gemm_fp4_skinny_kernel<FORMAT, X>, S::kTotal, smem_raised, "cudaFuncSetAttribute(gemm_fp4_skinny_kernel)");
    }
    if (st != LYRAQ_OK) {
        return st;
    }
    return cuda_status(launch_kernel(gemm_fp4_skinny_kernel<FORMAT, X>, (unsigned)(n_tiles * splits), (unsigned)kThreads, (size_t)S::kTotal, stream,
                                     (unsigned)splits, tw, tx, tsw, tsx, p, in.x, in.ldx, num_kb, splits, g_stalled_rank, g_wait_limit_ms),
                       "cudaLaunchKernelEx(gemm_fp4_skinny_kernel)");
}

template<int FORMAT>
static int launch_of(const Fp4Input& in, const uint8_t* W, const uint8_t* ws, const Fp4GemmParams& p, int sms, cudaStream_t stream)
{
    return in.codes != nullptr        ? launch<FORMAT, void>(in, W, ws, p, sms, stream)
           : in.dtype == LYRAQ_BF16   ? launch<FORMAT, __nv_bfloat16>(in, W, ws, p, sms, stream)
           : in.dtype == LYRAQ_F16    ? launch<FORMAT, __half>(in, W, ws, p, sms, stream)
                                      : launch<FORMAT, float>(in, W, ws, p, sms, stream);
}

}  // namespace skinny

bool skinny_quantize_pays(int m, int n, int k, int sms) { return skinny::quantize_pays(m, n, k, sms); }

int launch_skinny(const Fp4Input& X, const uint8_t* W, const uint8_t* ws, int format, const Fp4GemmParams& p, int sms, cudaStream_t stream)
{
    return format == LYRAQ_NVFP4 ? skinny::launch_of<LYRAQ_NVFP4>(X, W, ws, p, sms, stream) : skinny::launch_of<LYRAQ_MXFP4>(X, W, ws, p, sms, stream);
}

}  // namespace fp4
}  // namespace lyraq

extern "C" int lyraq_debug_fp4_skinny_wait_test(int stalled_rank, unsigned int wait_limit_ms)
{
    lyraq::fp4::skinny::g_stalled_rank  = stalled_rank;
    lyraq::fp4::skinny::g_wait_limit_ms = wait_limit_ms == 0 ? (unsigned int)(lyraq::sm100::kWaitLimitNs / 1000000) : wait_limit_ms;
    return LYRAQ_OK;
}
