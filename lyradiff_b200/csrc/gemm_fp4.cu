// FP4 x FP4 GEMM with block scales for sm_100a:
//
//   Y[M,N] = T( epi( g_x g_w sum_blocks s_x s_w sum_k X[M,k] W[N,k]  + beta R + bias ) )
//
// tcgen05.mma kind::mxf4nvf4 (nvfp4) and kind::mxf4 (mxfp4): packed e2m1 operands from shared memory, block scales from tensor memory, fp32
// accumulation; one instruction covers 64 values of K.  Four times the rate of 16-bit operands, so what surrounds the tensor pipe decides:
// a K block of 256 values (128 bytes a row) is 512 clocks of MMA for a pair's 256 x 256 tile and 38 KB of loads per CTA.
//
// Persistent, 384 threads, warp-specialised, as a CTA pair (256 x 256 tile, cta_group::2) or one CTA (128 x 128):
//   warp 0    : TMA producer   - operand tiles (128-byte swizzle) and scale atoms (fp4.cuh) into a ring of stages, one K block each.  Each
//                                CTA of a pair loads its own A rows and scales, its half of the B rows, and the scales of ALL B rows:
//                                both halves of the accumulator need them.
//   warp 1    : MMA issuer     - copies a stage's scale atoms to tensor memory (tcgen05.cp runs in order before the MMAs behind it), issues the
//                                MMAs, commits the stage.  Scale columns belong to the stage, so they are overwritten only after the MMAs
//                                that read them have completed.
//   warp 2    : allocates / frees tensor memory (all 512 columns: 256 of accumulators, the rest scales).
//   warps 4-11: epilogue       - a pair's accumulator fills the 256 columns, so there is one of it: the warps first bring their whole share
//                                into registers (128 per thread) and give the columns back, then scale, add, store while the next tile's MMAs run.
// Every mbarrier wait is bounded; on a timeout the role records it in the status word, raises the block's abort flag and all roles fall
// through to the common exit, where tensor memory is freed.
#include "gemm_fp4.cuh"

namespace lyraq {

using namespace sm100;

int device_sm_count();                                                                                                    // gemm_dense.cu
int make_tmap_bytes_2d(CUtensorMap* map, const void* base, uint64_t rows, uint64_t k_bytes, uint64_t row_stride_bytes,    // gemm_dense.cu
                       uint32_t box_rows, uint32_t box_bytes, bool swizzle128);
int make_tmap_store(CUtensorMap* map, const void* base, uint64_t rows, uint64_t cols, uint64_t ld, int elem_bytes, bool wide);  // gemm_dense.cu
int make_tmap_atoms(CUtensorMap* map, const void* base, uint64_t row_blocks, uint64_t atoms, uint32_t box_blocks, uint32_t box_atoms,  // gemm_dense.cu
                    uint32_t box_words);

namespace fp4 {

using namespace tiles;

constexpr int kBlockM    = 128;
constexpr int kRowBytes  = 128;          // a K block: 256 values, 128 bytes of every row
constexpr int kBlockK    = 256;
constexpr int kThreads   = 384;
constexpr int kEpiWarp0  = 4;
constexpr int kEpiWarps  = 8;
constexpr int kBox       = 32 * 64;      // one warp's staging box: 32 rows x 32 columns of a 16-bit type
constexpr int kBoxes     = 2;            // the store of one chunk drains its box while the next chunk is computed and fills the other
constexpr int kBiasBytes = 128 * 2;      // one warp's bias: up to 128 columns of a 16-bit type (fp32, which uses no boxes, keeps its there)
constexpr int kBarBytes  = 256;
constexpr int kOtherRegs = 72;
constexpr int kEpiRegs   = 216;
static_assert(128 * kOtherRegs + 256 * kEpiRegs <= kThreads * 168, "the split draws on what the block was launched with");

template<int FORMAT, int BLOCK_N, int CTAS> struct Smem {
    static constexpr int kAtoms      = kBlockK / fp4_atom_k(FORMAT);    // scale atoms of 128 rows in a K block: 4 or 2
    static constexpr int kSbBlocks   = BLOCK_N / 128;                   // row blocks of 128 in a tile's B rows
    static constexpr int kABytes     = kBlockM * kRowBytes;
    static constexpr int kBBytes     = BLOCK_N / CTAS * kRowBytes;
    static constexpr int kSfaBytes   = kAtoms * 512;
    static constexpr int kSfbBytes   = kSbBlocks * kAtoms * 512;
    static constexpr int kStageBytes = kABytes + kBBytes + kSfaBytes + kSfbBytes;
    static constexpr int kEpiBytes   = kEpiWarps * (kBoxes * kBox + kBiasBytes);
    static constexpr int kStages     = (227 * 1024 - 1024 - kBarBytes - kEpiBytes) / kStageBytes;
    static constexpr int kEpiOffset  = kStages * kStageBytes;
    static constexpr int kBarOffset  = kEpiOffset + kEpiBytes;
    static constexpr int kTotal      = kBarOffset + kBarBytes + 1024;   // + alignment slack
    // tensor memory: accumulators, then each stage's scales
    static constexpr int kAccBufs    = BLOCK_N == 256 ? 1 : 2;
    static constexpr int kAccCols    = kAccBufs * BLOCK_N;
    static constexpr int kScaleCols  = kAtoms * 4 * (1 + kSbBlocks);
    static_assert(kStageBytes % 1024 == 0, "the swizzle pattern is anchored to 1024 bytes");
    static_assert(8 * (2 * kStages + 4) + 8 <= kBarBytes, "");
    static_assert(kAccCols + kStages * kScaleCols <= 512, "");
};

template<int FORMAT, int BLOCK_N, int CTAS, bool RES>
__global__ void __launch_bounds__(kThreads, 1)
gemm_fp4_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b, const __grid_constant__ CUtensorMap tmap_sa,
                const __grid_constant__ CUtensorMap tmap_sb, const __grid_constant__ CUtensorMap tmap_c, const Fp4GemmParams p)
{
    using S = Smem<FORMAT, BLOCK_N, CTAS>;
    constexpr int kStages = S::kStages;
    constexpr int kTileM  = kBlockM * CTAS;
    constexpr int kHalfN  = BLOCK_N / 2;      // columns per epilogue warp

    extern __shared__ uint8_t smem_raw[];
    // the dynamic shared window starts at the same offset in every CTA of the kernel, so both CTAs of a pair get the same layout
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t*       gen_base  = smem_raw + (smem_base - smem_u32(smem_raw));
    const uint32_t bars      = smem_base + S::kBarOffset;
    auto full_bar       = [&](int s) { return bars + 8u * s; };
    auto empty_bar      = [&](int s) { return bars + 8u * (kStages + s); };
    auto tmem_full_bar  = [&](int b) { return bars + 8u * (2 * kStages + b); };
    auto tmem_empty_bar = [&](int b) { return bars + 8u * (2 * kStages + 2 + b); };
    uint32_t*      tmem_slot  = reinterpret_cast<uint32_t*>(gen_base + S::kBarOffset + 8 * (2 * kStages + 4));
    volatile int*  abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int      warp    = warp_index();
    const int      lane    = threadIdx.x & 31;
    const uint32_t rank    = (CTAS == 2) ? cluster_ctarank() : 0u;  // position in the pair; 0 = leader
    const bool     leader  = (rank == 0);
    const int      unit    = (CTAS == 2) ? (int)(blockIdx.x >> 1) : (int)blockIdx.x;
    const int      n_units = (CTAS == 2) ? (int)(gridDim.x >> 1) : (int)gridDim.x;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(full_bar(s), 1);
            mbar_init(empty_bar(s), 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(tmem_full_bar(b), 1);
            mbar_init(tmem_empty_bar(b), kEpiWarps * CTAS);
        }
        *abort_flag = 0;
        fence_barrier_init();
        prefetch_tensormap(&tmap_a);
        prefetch_tensormap(&tmap_b);
        prefetch_tensormap(&tmap_sa);
        prefetch_tensormap(&tmap_sb);
        prefetch_tensormap(&tmap_c);
    }
    if (warp == 2) {
        if (CTAS == 2) {
            tmem_alloc_pair(smem_u32(tmem_slot), 512);
            tmem_relinquish_pair();
        } else {
            tmem_alloc(smem_u32(tmem_slot), 512);
            tmem_relinquish();
        }
    }
    tc_fence_before_sync();
    if (CTAS == 2) {
        cluster_sync_all();
    } else {
        __syncthreads();
    }
    tc_fence_after_sync();
    const uint32_t tmem_base = *tmem_slot;
    grid_dependency_wait();

    const int num_tiles = p.m_tiles * p.n_tiles;
    const int num_kb    = (p.K + kBlockK - 1) / kBlockK;

    if (warp < kEpiWarp0) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
        if (warp == 0) {
            // -------------------------------------------------------------- TMA producer
            int      stage = 0, issued = 0;
            uint32_t phase = 0;
            bool     ok = true;
            for (int tile = unit; ok && tile < num_tiles; tile += n_units) {
                int m_blk, n_blk;
                tile_coords(tile, p.m_tiles, p.n_tiles, m_blk, n_blk);
                const int a_row = m_blk * kTileM + (int)rank * kBlockM;
                const int b_row = n_blk * BLOCK_N + (int)rank * (BLOCK_N / CTAS);
                for (int kb = 0; kb < num_kb; ++kb) {
                    if (!mbar_wait_warp(empty_bar(stage), phase ^ 1u, abort_flag)) {
                        report_timeout(p.status, 0x5100u | (unsigned)stage);
                        *abort_flag = 1;
                        ok = false;
                        break;
                    }
                    if (elect_one()) {
                        const uint32_t sa = smem_base + stage * S::kStageBytes;
                        const uint32_t sb = sa + S::kABytes, ssa = sb + S::kBBytes, ssb = ssa + S::kSfaBytes;
                        if (CTAS == 2) {
                            // both CTAs' bytes are counted on the leader's barrier, which the leader arms for the pair
                            const uint32_t lbar = map_to_cta(full_bar(stage), 0u);
                            if (leader) {
                                mbar_arrive_expect_tx(full_bar(stage), 2u * (uint32_t)S::kStageBytes);
                            }
                            tma_load_2d_pair(sa, &tmap_a, lbar, kb * kRowBytes, a_row);
                            tma_load_2d_pair(sb, &tmap_b, lbar, kb * kRowBytes, b_row);
                            tma_load_3d_pair(ssa, &tmap_sa, lbar, 0, kb * S::kAtoms, a_row >> 7);
                            tma_load_3d_pair(ssb, &tmap_sb, lbar, 0, kb * S::kAtoms, (n_blk * BLOCK_N) >> 7);
                        } else {
                            mbar_arrive_expect_tx(full_bar(stage), (uint32_t)S::kStageBytes);
                            tma_load_2d(sa, &tmap_a, full_bar(stage), kb * kRowBytes, a_row);
                            tma_load_2d(sb, &tmap_b, full_bar(stage), kb * kRowBytes, b_row);
                            tma_load_3d(ssa, &tmap_sa, full_bar(stage), 0, kb * S::kAtoms, a_row >> 7);
                            tma_load_3d(ssb, &tmap_sb, full_bar(stage), 0, kb * S::kAtoms, (n_blk * BLOCK_N) >> 7);
                        }
                    }
                    ++issued;
                    if (++stage == kStages) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
            }
            if (CTAS == 1 || leader) {
                // every load counted on this CTA's barriers must have landed before the block may leave
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
                        if (global_timer_ns() - t0 > kWaitLimitNs) {
                            report_timeout(p.status, 0x5500u | (unsigned)s);
                            break;
                        }
                    }
                }
            }
        } else if (warp == 1 && leader) {
            // -------------------------------------------------------------- MMA issuer (the leader CTA only)
            int      stage = 0;
            uint32_t phase = 0;
            int      local = 0;
            bool     ok = true;
            for (int tile = unit; ok && tile < num_tiles; tile += n_units, ++local) {
                const int      buf       = S::kAccBufs == 2 ? (local & 1) : 0;
                const uint32_t acc_phase = (uint32_t)(S::kAccBufs == 2 ? local >> 1 : local) & 1u;
                const uint32_t d_tmem = tmem_base + (uint32_t)(buf * BLOCK_N);
                for (int kb = 0; kb < num_kb; ++kb) {
                    if (!mbar_wait_warp(full_bar(stage), phase, abort_flag)) {
                        report_timeout(p.status, 0x5300u | (unsigned)stage);
                        *abort_flag = 1;
                        ok = false;
                        break;
                    }
                    tc_fence_after_sync();
                    const uint32_t sa     = smem_base + stage * S::kStageBytes;
                    const uint64_t adesc  = umma_desc_k_sw128(sa);
                    const uint64_t bdesc  = umma_desc_k_sw128(sa + S::kABytes);
                    const uint64_t sadesc = umma_desc_scales(sa + S::kABytes + S::kBBytes);
                    const uint64_t sbdesc = umma_desc_scales(sa + S::kABytes + S::kBBytes + S::kSfaBytes);
                    const uint32_t sfa    = tmem_base + (uint32_t)(S::kAccCols + stage * S::kScaleCols);
                    const uint32_t sfb    = sfa + S::kAtoms * 4;
                    const int      steps  = min(kBlockK, p.K - kb * kBlockK + 63) / 64;   // MMAs of this K block
                    const bool     last   = kb + 1 == num_kb;
                    auto copy_scales = [&]() {
#pragma unroll
                        for (int a = 0; a < S::kAtoms; ++a) {
                            tmem_copy_scales<CTAS>(sfa + a * 4, sadesc + (uint64_t)(a * 32));
                            // in tensor memory the row blocks of an atom stand side by side
#pragma unroll
                            for (int rb = 0; rb < S::kSbBlocks; ++rb) {
                                tmem_copy_scales<CTAS>(sfb + a * (4 * S::kSbBlocks) + rb * 4, sbdesc + (uint64_t)((rb * S::kAtoms + a) * 32));
                            }
                        }
                    };
                    if (kb == 0) {
                        // the scales of a tile's first K block are on their way while the epilogue still has the accumulator
                        if (elect_one()) {
                            copy_scales();
                        }
                        if (!mbar_wait_warp(tmem_empty_bar(buf), acc_phase ^ 1u, abort_flag)) {
                            report_timeout(p.status, 0x5200u | (unsigned)buf);
                            *abort_flag = 1;
                            ok = false;
                            break;
                        }
                        tc_fence_after_sync();
                    }
                    if (elect_one()) {
                        if (kb > 0) {
                            copy_scales();
                        }
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            constexpr int kPer = 4 / S::kAtoms;   // MMAs of one atom
                            if (k < steps) {
                                mma_fp4<FORMAT, CTAS>(d_tmem, adesc + (uint64_t)(2 * k), bdesc + (uint64_t)(2 * k),
                                                      umma_idesc_fp4(FORMAT, kTileM, BLOCK_N, 2u * (k % kPer)), sfa + k / kPer * 4,
                                                      sfb + k / kPer * (4 * S::kSbBlocks), (kb > 0 || k > 0) ? 1u : 0u);
                            }
                        }
                        if (CTAS == 2) {
                            tc_commit_both(empty_bar(stage));
                            if (last) {
                                tc_commit_both(tmem_full_bar(buf));
                            }
                        } else {
                            tc_commit(empty_bar(stage));
                            if (last) {
                                tc_commit(tmem_full_bar(buf));
                            }
                        }
                    }
                    if (++stage == kStages) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
            }
        }
    } else {
        // ------------------------------------------------------------------ epilogue (warps 4..11)
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kEpiRegs));
        const int      quad      = warp & 3;                 // the TMEM lane quadrant this warp may read
        const int      half      = (warp - kEpiWarp0) >> 2;  // which half of the tile's columns
        const uint32_t lane_addr = (uint32_t)(quad * 32) << 16;
        uint8_t*       boxes     = gen_base + S::kEpiOffset + (warp - kEpiWarp0) * kBoxes * kBox;
        const uint32_t boxes_at  = smem_base + S::kEpiOffset + (warp - kEpiWarp0) * kBoxes * kBox;
        uint8_t*       bias      = p.c_dtype == LYRAQ_F32 ? boxes : gen_base + S::kEpiOffset + kEpiWarps * kBoxes * kBox + (warp - kEpiWarp0) * kBiasBytes;
        // the bias of this warp's columns of a tile, one column in 32 per lane; fetched a tile ahead
        uint32_t bias_ahead[kHalfN / 32];
        auto fetch_bias = [&](int tile) {
            int m_blk, n_blk;
            tile_coords(tile, p.m_tiles, p.n_tiles, m_blk, n_blk);
#pragma unroll
            for (int i = 0; i < kHalfN / 32; ++i) {
                const int col = n_blk * BLOCK_N + half * kHalfN + lane + 32 * i;
                bias_ahead[i] = 0;
                if (p.bias != nullptr && col < p.N) {
                    bias_ahead[i] = p.c_dtype == LYRAQ_F32 ? reinterpret_cast<const uint32_t*>(p.bias)[col]
                                                           : (uint32_t)reinterpret_cast<const uint16_t*>(p.bias)[col];
                }
            }
        };
        if (unit < num_tiles) {
            fetch_bias(unit);
        }
        const float    scale     = fp4_tensor_scale(p);
        const bool     vec_ok    = p.c_dtype == LYRAQ_F32 ? (p.N & 3) == 0 : (p.N & 7) == 0;
        int            local     = 0;
        for (int tile = unit; tile < num_tiles; tile += n_units, ++local) {
            const int      buf       = S::kAccBufs == 2 ? (local & 1) : 0;
            const uint32_t acc_phase = (uint32_t)(S::kAccBufs == 2 ? local >> 1 : local) & 1u;
            int m_blk, n_blk;
            tile_coords(tile, p.m_tiles, p.n_tiles, m_blk, n_blk);
            const int row0  = m_blk * kTileM + (int)rank * kBlockM + quad * 32;  // first row of this warp
            const int row   = row0 + lane;
            const int ncol0 = n_blk * BLOCK_N + half * kHalfN;
            if (p.bias != nullptr) {
                // the warp's own piece of shared memory, so no other warp is waited for
                __syncwarp();
#pragma unroll
                for (int i = 0; i < kHalfN / 32; ++i) {
                    if (p.c_dtype == LYRAQ_F32) {
                        reinterpret_cast<uint32_t*>(bias)[lane + 32 * i] = bias_ahead[i];
                    } else {
                        reinterpret_cast<uint16_t*>(bias)[lane + 32 * i] = (uint16_t)bias_ahead[i];
                    }
                }
                __syncwarp();
                if (tile + n_units < num_tiles) {
                    fetch_bias(tile + n_units);
                }
            }
            const uint32_t t_addr = tmem_base + lane_addr + (uint32_t)(buf * BLOCK_N + half * kHalfN);
            auto release = [&]() {   // this warp's share of the accumulator is in registers: the next tile may have its columns
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) {
                    if (CTAS == 2 && !leader) {
                        mbar_arrive_cluster_relaxed(map_to_cta(tmem_empty_bar(buf), 0u));
                    } else {
                        mbar_arrive(tmem_empty_bar(buf));
                    }
                }
            };
            constexpr int kChunks = kHalfN / 32;
            // Residual of a 16-bit output: a lane that fetched its own row would touch 32 lines an instruction and use half a sector of each
            // ([4608, 12288, 3072]: 191 us against 72 without a residual).  Instead four lanes fetch the 64 bytes of a row, eight rows an instruction, two chunks
            // ahead (the first brings all 256 bytes of the row's share into L2), and hand them over through the box that the result leaves by.
            const bool staged = RES && p.residual != nullptr && p.tma_store;
            Vec16      rr[2][RES ? 4 : 1];
            auto fetch = [&](int c, Vec16* dst) {
                const int col = ncol0 + c * 32 + (lane & 3) * 8;
#pragma unroll
                for (int i = 0; i < (RES ? 4 : 1); ++i) {
                    const int rw = row0 + i * 8 + (lane >> 2);
                    dst[i]       = Vec16{};
                    if (rw < p.M && col < p.N) {   // N is a multiple of 8
                        dst[i] = ld_16_l2_256(reinterpret_cast<const uint16_t*>(p.residual) + (size_t)rw * (size_t)p.N + (size_t)col);
                    }
                }
            };
            if (staged) {
                fetch(0, rr[0]);
                fetch(1, rr[1]);
            }
            constexpr int kAhead  = S::kAccBufs == 1 ? kChunks : 2;   // chunks in registers: all of a lone accumulator
            uint32_t acc[kAhead][32];
            if (!mbar_wait_warp(tmem_full_bar(buf), acc_phase, abort_flag)) {
                if (lane == 0) {
                    report_timeout(p.status, 0x5400u | (unsigned)buf);
                }
                *abort_flag = 1;
                break;
            }
            tc_fence_after_sync();
            if (S::kAccBufs == 1) {
#pragma unroll
                for (int c = 0; c < kChunks; ++c) {
                    tmem_ld_32x32(t_addr + (uint32_t)(c * 32), acc[c % kAhead]);
                }
                tmem_ld_wait();
                release();
            } else {
                tmem_ld_32x32(t_addr, acc[0]);
            }
#pragma unroll
            for (int c = 0; c < kChunks; ++c) {
                if (S::kAccBufs == 2) {
                    tmem_ld_wait();
                    if (c + 1 < kChunks) {
                        tmem_ld_32x32(t_addr + (uint32_t)((c + 1) * 32), acc[(c + 1) % kAhead]);
                    } else {
                        release();
                    }
                }
                const int col0  = ncol0 + c * 32;
                const int valid = p.N - col0;
                if (valid <= 0) {
                    continue;
                }
                float     v[32];
                uint8_t*  box  = boxes + (c % kBoxes) * kBox;
                uint8_t*  brow = box + lane * 64;
                const int sw   = (lane >> 1) & 3;
                if (p.tma_store) {
                    if (lane == 0) {
                        // the store before the last has drained this box; the tile before may have ended with either box
                        if (c == 0) {
                            tma_store_wait_read();
                        } else {
                            tma_store_wait_read_but_one();
                        }
                    }
                    __syncwarp();
                }
                if (staged) {
#pragma unroll
                    for (int i = 0; i < (RES ? 4 : 1); ++i) {
                        const int r = i * 8 + (lane >> 2);
                        *reinterpret_cast<Vec16*>(box + r * 64 + (((lane & 3) ^ ((r >> 1) & 3)) << 4)) = rr[c & 1][i];
                    }
                    __syncwarp();
                    if (c + 2 < kChunks) {
                        fetch(c + 2, rr[c & 1]);
                    }
                }
                if (p.c_dtype == LYRAQ_F32) {
                    if (row < p.M) {
                        finish32<float, RES>(p, acc[c % kAhead], bias + c * 128, nullptr, 0, scale, row, col0, valid, vec_ok, v);
                        store32<float>(reinterpret_cast<float*>(p.C) + (size_t)row * (size_t)p.N + (size_t)col0, valid, vec_ok, v);
                    }
                    continue;
                }
                const bool bf16 = p.c_dtype == LYRAQ_BF16;
                if (bf16) {
                    finish32<__nv_bfloat16, RES>(p, acc[c % kAhead], bias + c * 64, RES && staged ? brow : nullptr, sw, scale, row, col0, valid, vec_ok, v);
                } else {
                    finish32<__half, RES>(p, acc[c % kAhead], bias + c * 64, RES && staged ? brow : nullptr, sw, scale, row, col0, valid, vec_ok, v);
                }
                if (!p.tma_store) {
                    if (row < p.M) {
                        uint16_t* crow = reinterpret_cast<uint16_t*>(p.C) + (size_t)row * (size_t)p.N + (size_t)col0;
                        if (bf16) {
                            store32<__nv_bfloat16>(reinterpret_cast<__nv_bfloat16*>(crow), valid, vec_ok, v);
                        } else {
                            store32<__half>(reinterpret_cast<__half*>(crow), valid, vec_ok, v);
                        }
                    }
                    continue;
                }
                // 32 rows x 64 bytes through this warp's box in the 64-byte swizzle, one TMA store; rows and columns beyond the matrix are clipped
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    *reinterpret_cast<Vec16*>(brow + ((q ^ sw) << 4)) = bf16 ? pack8<__nv_bfloat16>(v + 8 * q) : pack8<__half>(v + 8 * q);
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0 && row0 < p.M) {
                    tma_store_2d(&tmap_c, boxes_at + (uint32_t)((c % kBoxes) * kBox), col0, row0);
                    tma_store_commit();
                }
            }
        }
        if (lane == 0) {
            tma_store_wait_read();  // shared memory must outlive the last store's read of it
        }
    }

    // ---------------------------------------------------------------------- common exit
    tc_fence_before_sync();
    if (CTAS == 2) {
        cluster_sync_all();  // neither CTA may leave while its peer can still touch its shared or tensor memory
    } else {
        __syncthreads();
    }
    // The kernel behind may begin only now: quantizers that were let in at the start and waited beside the GEMM made a chain of
    // linears 10 to 25 % slower ([1317, 3072, 12288] 40 us a linear against 31, [4608, 12288, 3072] 86 against 81).
    grid_launch_dependents();
    if (warp == 2) {
        tc_fence_after_sync();
        if (CTAS == 2) {
            tmem_dealloc_pair(tmem_base, 512);
        } else {
            tmem_dealloc(tmem_base, 512);
        }
    }
}

template<int FORMAT, int BLOCK_N, int CTAS, bool RES>
static int launch(const uint8_t* X, const uint8_t* xs, const uint8_t* W, const uint8_t* ws, Fp4GemmParams p, int sms, cudaStream_t stream)
{
    using S = Smem<FORMAT, BLOCK_N, CTAS>;
    const uint64_t kb = (uint64_t)p.K / 2, atoms = fp4_atoms((size_t)p.K, FORMAT);
    CUtensorMap ta, tb, tsa, tsb;
    int st = make_tmap_bytes_2d(&ta, X, (uint64_t)p.M, kb, kb, kBlockM, kRowBytes, true);
    if (st == LYRAQ_OK) {
        st = make_tmap_bytes_2d(&tb, W, (uint64_t)p.N, kb, kb, BLOCK_N / CTAS, kRowBytes, true);
    }
    if (st == LYRAQ_OK) {
        st = make_tmap_atoms(&tsa, xs, ((uint64_t)p.M + 127) / 128, atoms, 1, S::kAtoms, 128);
    }
    if (st == LYRAQ_OK) {
        st = make_tmap_atoms(&tsb, ws, ((uint64_t)p.N + 127) / 128, atoms, S::kSbBlocks, S::kAtoms, 128);
    }
    CUtensorMap tc = ta;   // never used where the output is stored directly
    p.tma_store    = p.c_dtype != LYRAQ_F32 && (p.N & 7) == 0;
    if (st == LYRAQ_OK && p.tma_store) {
        st = make_tmap_store(&tc, p.C, (uint64_t)p.M, (uint64_t)p.N, (uint64_t)p.N, 2, false);
    }
    if (st != LYRAQ_OK) {
        return st;
    }
    p.m_tiles = (int)(((long)p.M + kBlockM * CTAS - 1) / (kBlockM * CTAS));
    p.n_tiles = (int)(((long)p.N + BLOCK_N - 1) / BLOCK_N);
    const long long tiles = (long long)p.m_tiles * p.n_tiles;
    if (tiles > 0x40000000ll) {
        return LYRAQ_ERR_UNSUPPORTED;
    }
    const long long units = sms / CTAS;
    const int       grid  = (int)(tiles < units ? tiles : units) * CTAS;
    auto            kern  = gemm_fp4_kernel<FORMAT, BLOCK_N, CTAS, RES>;
    static bool     smem_raised[64] = {};
    st = raise_dynamic_smem_once(kern, (int)S::kTotal, smem_raised, "cudaFuncSetAttribute(gemm_fp4_kernel, dynamic shared memory)");
    if (st != LYRAQ_OK) {
        return st;
    }
    return cuda_status(launch_kernel(kern, (unsigned)grid, (unsigned)kThreads, (size_t)S::kTotal, stream, (unsigned)CTAS, ta, tb, tsa, tsb, tc, p),
                       "cudaLaunchKernelEx(gemm_fp4_kernel)");
}

// forced kernel for tests and sweeps: 0 = automatic, 16 = the few-row kernel (up to 16 rows), 2562 = CTA pair with 256 x 256, 1281 = one CTA with 128 x 128
static int g_forced_tile = 0;

bool few_rows(int m, int k)
{
    // The few-row kernel's time grows with the rows (their partial sums cross shared memory and leave row by row), the other's does not; what it
    // gains grows with K.  Dense against few-row, us: 4 rows of [256, 256] 2.8 / 3.1, of [1280, 1280] 4.3 / 4.1, 8 rows of it 4.3 / 5.2; 16
    // rows of [1280, 2048] 5.1 / 4.7, of [3072, 3072] 6.4 / 5.6, of [3072, 12288] 17.4 / 8.2; one row of [9216, 3072] 8.3 / 5.4.
    const int num_kb = (k + kBlockK - 1) / kBlockK;
    return m <= kFp4SkinnyRows && (g_forced_tile == 16 || (g_forced_tile == 0 && (num_kb >= 8 || m <= 2 + num_kb / 2)));
}

bool few_rows_quantize(int m, int n, int k) { return few_rows(m, k) && (g_forced_tile == 16 || skinny_quantize_pays(m, n, k, device_sm_count())); }

static int run(const Fp4Input& X, const uint8_t* W, const uint8_t* ws, int format, const Fp4GemmParams& p, int sms, cudaStream_t stream)
{
    const long m128 = ((long)p.M + 127) / 128, n128 = ((long)p.N + 127) / 128, m256 = ((long)p.M + 255) / 256, n256 = ((long)p.N + 255) / 256;
    const long pairs = sms / 2;
    const int num_kb = (p.K + kBlockK - 1) / kBlockK;
    if (few_rows(p.M, p.K)) {
        return launch_skinny(X, W, ws, format, p, sms, stream);
    }
    // Rounds of each tile times what one takes, us: 0.2 + 0.323 a K block for 128 x 128, 1.3 + 0.39 for a pair's 256 x 256, from [4608, 12288, 3072]
    // (98 / 72), [4608, 3072, 12288] (94 / 60), [4608, 3072, 3072] (29 / 19), [1155, 9216, 3072] (24 / 18), [512, 3072, 3072] (7.8 / 9.7).
    const double c1   = (double)((m128 * n128 + sms - 1) / sms) * (0.2 + 0.323 * num_kb);
    const double c2   = pairs > 0 ? (double)((m256 * n256 + pairs - 1) / pairs) * (1.3 + 0.39 * num_kb) : 1e30;
    const int    tile = g_forced_tile > 16 ? g_forced_tile : c2 <= c1 ? 2562 : 1281;
    auto pick = [&](auto fmt, auto res) {
        constexpr int  kFmt = decltype(fmt)::value;
        constexpr bool kRes = decltype(res)::value;
        return tile == 2562 ? launch<kFmt, 256, 2, kRes>(X.codes, X.scales, W, ws, p, sms, stream)
                            : launch<kFmt, 128, 1, kRes>(X.codes, X.scales, W, ws, p, sms, stream);
    };
    auto pick_res = [&](auto fmt) {
        return p.residual != nullptr ? pick(fmt, std::integral_constant<bool, true>{}) : pick(fmt, std::integral_constant<bool, false>{});
    };
    return format == LYRAQ_NVFP4 ? pick_res(std::integral_constant<int, LYRAQ_NVFP4>{}) : pick_res(std::integral_constant<int, LYRAQ_MXFP4>{});
}

int product(const Fp4Input& X, const float* g_x, const uint8_t* W, const uint8_t* ws, const float* g_w, int format, void* Y, int c_dtype, const void* bias,
            const void* residual, float beta, int epilogue, int m, int n, int k, cudaStream_t stream)
{
    Fp4GemmParams p{};
    p.M        = m;
    p.N        = n;
    p.K        = k;
    p.C        = Y;
    p.c_dtype  = c_dtype;
    p.s_x      = g_x;
    p.s_w      = g_w;
    p.bias     = bias;
    p.residual = residual;
    p.beta     = beta;
    p.gelu     = epilogue == LYRAQ_EPI_GELU_TANH;
    p.status   = status_word_ptr();
    const int sms = device_sm_count();
    if (p.status == nullptr || sms <= 0) {
        return LYRAQ_ERR_CUDA;
    }
    return run(X, W, ws, format, p, sms, stream);
}

}  // namespace fp4
}  // namespace lyraq

using namespace lyraq;

extern "C" {

int lyraq_debug_force_fp4_tile(int code)
{
    if (code != 0 && code != 16 && code != 1281 && code != 2562) {
        return LYRAQ_ERR_INVALID_ARG;
    }
    fp4::g_forced_tile = code;
    return LYRAQ_OK;
}

int lyraq_gemm_fp4(const uint8_t* X, const uint8_t* x_scale, const float* x_tensor_scale, const uint8_t* W, const uint8_t* w_scale,
                   const float* w_tensor_scale, int format, void* Y, int c_dtype, const void* bias, const void* residual, float beta,
                   int epilogue, int m, int n, int k, void* stream)
{
    if (m < 0 || n < 0 || k < 0 || (format != LYRAQ_NVFP4 && format != LYRAQ_MXFP4) ||
        (epilogue != LYRAQ_EPI_NONE && epilogue != LYRAQ_EPI_GELU_TANH) ||
        (c_dtype != LYRAQ_F16 && c_dtype != LYRAQ_BF16 && c_dtype != LYRAQ_F32)) {
        return LYRAQ_ERR_INVALID_ARG;
    }
    if (m == 0 || n == 0) {
        return LYRAQ_OK;
    }
    if (k == 0 || (k & 31) != 0 || m > fp4::kMaxSize || n > fp4::kMaxSize || k > fp4::kMaxSize) {
        return LYRAQ_ERR_UNSUPPORTED;
    }
    if (X == nullptr || x_scale == nullptr || W == nullptr || w_scale == nullptr || Y == nullptr || !aligned16(X) || !aligned16(x_scale) ||
        !aligned16(W) || !aligned16(w_scale) || !aligned16(Y) || (bias != nullptr && !aligned16(bias)) ||
        (residual != nullptr && !aligned16(residual))) {
        return LYRAQ_ERR_INVALID_ARG;
    }
    const size_t rows = (size_t)m, cols = (size_t)n, depth = (size_t)k, bytes = c_dtype == LYRAQ_F32 ? 4 : 2;
    if (result_clashes(view_of(Y, rows * cols * bytes), residual,
                            {view_of(X, rows * depth / 2), view_of(x_scale, lyraq_fp4_scale_bytes(rows, depth, format)), view_of(W, cols * depth / 2),
                             view_of(w_scale, lyraq_fp4_scale_bytes(cols, depth, format)), view_of(bias, cols * bytes)})) {
        return LYRAQ_ERR_INVALID_ARG;
    }
    return fp4::product({X, x_scale, nullptr, 0, 0}, x_tensor_scale, W, w_scale, w_tensor_scale, format, Y, c_dtype, bias, residual, beta, epilogue, m, n, k,
                        (cudaStream_t)stream);
}

}  // extern "C"
