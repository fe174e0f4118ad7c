// FP8 x FP8 GEMM with a scale for each block of 128 for sm_100a:
//
//   Y[M,N] = T( epi( sum_kb s_x[m,kb] s_w[n/128,kb] sum_{k in kb} X[m,k] W[n,k]  + beta R + bias ) )
//
// The scales are any fp32 numbers, so the tensor cores cannot apply them: a K block of 128 is one product of its own in tensor memory, and the
// epilogue warps add it, times its factor, to fp32 sums that they hold in registers for the whole tile (64 a thread).  Tensor memory holds two products of a
// pair's tile (four of a lone CTA's), so that the next is formed while one is taken.
//
// Persistent, 640 threads, warp-specialised, as a CTA pair (256 x 256 tile, cta_group::2) or one CTA (128 x 128):
//   warp 0    : TMA producer   - operand tiles (128-byte swizzle) into a ring of stages, one K block each; each CTA of a pair loads its own A rows
//                                and its half of the B rows.
//   warp 1    : MMA issuer     - four MMAs a K block into the product buffer that is free; commits the stage and the product.
//   warp 2    : allocates / frees tensor memory.
//   warps 4-19: epilogue       - per K block: products -> sums; at the end of a tile residual, bias, GELU, store.  A lane owns a row, so its factor is
//                                one number per K block: its row's scale times the scale of the warp's columns, which lie in one block of W.
//
// What bounds it: the way of a product from its last MMA to the next one in its place (completion, loads out of tensor memory, the word back to the issuer, about
// 1400 clocks with two in flight), against 512 of MMAs for a pair's K block, which take about 600 beside the loads into shared memory; 1000 measured.
// [4680, 13824, 5120]: 311 us in a burst (2.1 PFLOP/s), [4608, 3072, 12288] 155; the framework's FP8 product with one scale takes 117 for the latter.
// Measured on the way: eight epilogue warps with 128 sums a thread 360 and 180 (two a scheduler do not hide the loads' latency).  Not kept: products in pieces
// of 128 columns (an A tile read twice bounds the MMAs: 180), a pair's tile of 256 x 128 (198), the next product's loads ahead of the additions (229).
// Where few tiles have many K blocks, a cluster of 2, 4 or 8 CTAs shares out the K blocks of a tile.
// Every mbarrier wait is bounded; on a timeout the role records it in the status word, raises the block's abort flag and all roles fall
// through to the common exit, where tensor memory is freed.
#include "fp8_block.cuh"
#include "gemm_tiles.cuh"

namespace lyraq {

using namespace sm100;

int device_sm_count();                                                                                                    // gemm_dense.cu
int make_tmap_bytes_2d(CUtensorMap* map, const void* base, uint64_t rows, uint64_t k_bytes, uint64_t row_stride_bytes,    // gemm_dense.cu
                       uint32_t box_rows, uint32_t box_bytes, bool swizzle128);
int make_tmap_store(CUtensorMap* map, const void* base, uint64_t rows, uint64_t cols, uint64_t ld, int elem_bytes, bool wide);  // gemm_dense.cu

namespace fp8b {

using namespace tiles;

constexpr int kBlockM    = 128;
constexpr int kThreads   = 640;
constexpr int kEpiWarp0  = 4;
constexpr int kEpiWarps  = 16;
constexpr int kBox       = 32 * 64;      // one warp's staging box: 32 rows x 32 columns of a 16-bit type
constexpr int kBiasBytes = 64 * 2;       // one warp's bias: up to 64 columns of a 16-bit type (fp32, which uses no boxes, keeps its there)
constexpr int kBarBytes  = 256;
constexpr int kPartBytes = 32 * 32 * 4;  // one warp's sums of one CTA along K, [column][row]
constexpr int kOtherRegs = 32;
constexpr int kEpiRegs   = 112;
static_assert(128 * kOtherRegs + 512 * kEpiRegs <= kThreads * 96, "the split draws on what the block was launched with");

template<int BLOCK_N, int CTAS> struct Smem {
    static constexpr int kABytes     = kBlockM * kBlock;
    static constexpr int kBBytes     = BLOCK_N / CTAS * kBlock;
    static constexpr int kStageBytes = kABytes + kBBytes;
    static constexpr int kEpiBytes   = kEpiWarps * (kBox + kBiasBytes);
    static constexpr int kStages     = (227 * 1024 - 1024 - kBarBytes - kEpiBytes) / kStageBytes;
    static constexpr int kEpiOffset  = kStages * kStageBytes;
    static constexpr int kBarOffset  = kEpiOffset + kEpiBytes;
    static constexpr int kTotal      = kBarOffset + kBarBytes + 1024;   // + alignment slack
    static constexpr int kBufs       = 512 / BLOCK_N;                   // products in tensor memory: 2 or 4
    static_assert(kStageBytes % 1024 == 0, "the swizzle pattern is anchored to 1024 bytes");
    static_assert(8 * (2 * kStages + 2 * kBufs) + 8 <= kBarBytes, "");
};

// A warp's box of 32 rows x 32 columns of a 16-bit type against rows of memory that no 16-byte access fits (N no multiple of 8): a lane that wrote its own row
// would touch 32 lines an instruction, so a row's columns go beside each other, two rows an instruction where N is even and one where it is odd.
// IN: memory -> box, else box -> memory.  The box is in the 64-byte swizzle.
template<bool IN> __device__ __forceinline__ void move_box(uint8_t* box, uint16_t* mem, const GemmParams& p, int row0, int col0, int lane)
{
    const bool two  = (p.N & 1) == 0;
    const int  sub  = two ? lane >> 4 : 0;
    const int  col  = two ? (lane & 15) * 2 : lane;
    const int  step = two ? 2 : 1;
    const bool in   = col0 + col < p.N;
#pragma unroll 1
    for (int r0 = 0; r0 < 32 && row0 + r0 < p.M; r0 += 8) {
        uint32_t held[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int      r     = r0 + i * step + sub;
            uint8_t*       here  = box + r * 64 + ((((col >> 3) ^ (r >> 1)) & 3) << 4) + (col & 7) * 2;
            uint16_t*      there = mem + (size_t)(row0 + r) * (size_t)p.N + (size_t)(col0 + col);
            const bool     moves = in && i * step < 8 && row0 + r < p.M;
            held[i] = 0;
            if (moves) {
                if (two) {
                    held[i] = IN ? *reinterpret_cast<const uint32_t*>(there) : *reinterpret_cast<const uint32_t*>(here);
                } else {
                    held[i] = IN ? (uint32_t)*there : (uint32_t)*reinterpret_cast<const uint16_t*>(here);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int      r     = r0 + i * step + sub;
            uint8_t*       here  = box + r * 64 + ((((col >> 3) ^ (r >> 1)) & 3) << 4) + (col & 7) * 2;
            uint16_t*      there = mem + (size_t)(row0 + r) * (size_t)p.N + (size_t)(col0 + col);
            if (in && i * step < 8 && row0 + r < p.M) {
                if (two) {
                    *reinterpret_cast<uint32_t*>(IN ? here : reinterpret_cast<uint8_t*>(there)) = held[i];
                } else {
                    *reinterpret_cast<uint16_t*>(IN ? here : reinterpret_cast<uint8_t*>(there)) = (uint16_t)held[i];
                }
            }
        }
    }
}

__device__ __forceinline__ void st_cluster_u32(uint32_t cluster_addr, uint32_t v)
{
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(cluster_addr), "r"(v) : "memory");
}

// NARROW: 16-bit rows that start on less than 16 bytes, which no TMA store takes.  A kernel of its own: its stores beside the others cost 340 us for 318 with
// [4680, 13824, 5120].
// SPLIT: a tile is a cluster's, its K blocks shared out among the CTAs.  Each warp sends its sums to the CTA that owns its part of the tile, which adds them in
// rank order and finishes that part.
template<int BLOCK_N, int CTAS, bool RES, bool NARROW, bool SPLIT>
__global__ void __launch_bounds__(kThreads, 1)
gemm_fp8_block_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b, const __grid_constant__ CUtensorMap tmap_c,
                      const GemmParams p)
{
    using S = Smem<BLOCK_N, CTAS>;
    constexpr int kStages = S::kStages;
    constexpr int kBufs   = S::kBufs;
    constexpr int kTileM  = kBlockM * CTAS;
    constexpr int kCols   = BLOCK_N / 4;      // columns per epilogue warp: 64 or 32, all of one block of W
    constexpr int kChunks = kCols / 32;
    constexpr int kAhead  = 2;                // K blocks whose scales are fetched together
    static_assert(!SPLIT || (CTAS == 1 && kChunks == 1 && S::kEpiOffset >= kEpiWarps * kPartBytes), "the partial sums take the operands' place");

    extern __shared__ uint8_t smem_raw[];
    // the dynamic shared window starts at the same offset in every CTA of the kernel, so both CTAs of a pair get the same layout
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t*       gen_base  = smem_raw + (smem_base - smem_u32(smem_raw));
    const uint32_t bars      = smem_base + S::kBarOffset;
    auto full_bar       = [&](int s) { return bars + 8u * s; };
    auto empty_bar      = [&](int s) { return bars + 8u * (kStages + s); };
    auto tmem_full_bar  = [&](int b) { return bars + 8u * (2 * kStages + b); };
    auto tmem_empty_bar = [&](int b) { return bars + 8u * (2 * kStages + kBufs + b); };
    uint32_t*      tmem_slot  = reinterpret_cast<uint32_t*>(gen_base + S::kBarOffset + 8 * (2 * kStages + 2 * kBufs));
    volatile int*  abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int      warp    = warp_index();
    const int      lane    = threadIdx.x & 31;
    const uint32_t rank    = (CTAS == 2) ? cluster_ctarank() : 0u;  // position in the pair; 0 = leader
    const bool     leader  = (rank == 0);
    const int      splits  = SPLIT ? p.splits : 1;                  // CTAs along K
    const int      unit    = SPLIT ? (int)blockIdx.x / splits : (CTAS == 2) ? (int)(blockIdx.x >> 1) : (int)blockIdx.x;
    const int      n_units = SPLIT ? (int)gridDim.x / splits : (CTAS == 2) ? (int)(gridDim.x >> 1) : (int)gridDim.x;   // SPLIT: one for each tile
    const int      part    = SPLIT ? (int)cluster_ctarank() : 0;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(full_bar(s), 1);
            mbar_init(empty_bar(s), 1);
        }
        for (int b = 0; b < kBufs; ++b) {
            mbar_init(tmem_full_bar(b), 1);
            mbar_init(tmem_empty_bar(b), kEpiWarps * CTAS);
        }
        *abort_flag = 0;
        fence_barrier_init();
        prefetch_tensormap(&tmap_a);
        prefetch_tensormap(&tmap_b);
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
    const int num_kb    = (p.K + kBlock - 1) / kBlock;
    const int kb_first  = SPLIT ? num_kb * part / splits : 0;        // this CTA's K blocks
    const int kb_end    = SPLIT ? num_kb * (part + 1) / splits : num_kb;

    if (warp < kEpiWarp0) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
        if (warp == 0) {
            // -------------------------------------------------------------- TMA producer
            int      stage = 0, issued = 0;
            uint32_t phase = 0;
            bool     ok = (SPLIT ? part : (int)rank) != p.stalled_rank;
            for (int tile = unit; ok && tile < num_tiles; tile += n_units) {
                int m_blk, n_blk;
                tile_coords(tile, p.m_tiles, p.n_tiles, m_blk, n_blk);
                const int a_row = m_blk * kTileM + (int)rank * kBlockM;
                const int b_row = n_blk * BLOCK_N + (int)rank * (BLOCK_N / CTAS);
                for (int kb = kb_first; kb < kb_end; ++kb) {
                    if (!mbar_wait_warp(empty_bar(stage), phase ^ 1u, abort_flag, p.wait_limit_ns)) {
                        report_timeout(p.status, 0x7100u | (unsigned)stage);
                        *abort_flag = 1;
                        ok = false;
                        break;
                    }
                    if (elect_one()) {
                        const uint32_t sa = smem_base + stage * S::kStageBytes, sb = sa + S::kABytes;
                        if (CTAS == 2) {
                            // both CTAs' bytes are counted on the leader's barrier, which the leader arms for the pair
                            const uint32_t lbar = map_to_cta(full_bar(stage), 0u);
                            if (leader) {
                                mbar_arrive_expect_tx(full_bar(stage), 2u * (uint32_t)S::kStageBytes);
                            }
                            tma_load_2d_pair(sa, &tmap_a, lbar, kb * kBlock, a_row);
                            tma_load_2d_pair(sb, &tmap_b, lbar, kb * kBlock, b_row);
                        } else {
                            mbar_arrive_expect_tx(full_bar(stage), (uint32_t)S::kStageBytes);
                            tma_load_2d(sa, &tmap_a, full_bar(stage), kb * kBlock, a_row);
                            tma_load_2d(sb, &tmap_b, full_bar(stage), kb * kBlock, b_row);
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
                        if (global_timer_ns() - t0 > p.wait_limit_ns) {
                            report_timeout(p.status, 0x7500u | (unsigned)s);
                            break;
                        }
                    }
                }
            }
        } else if (warp == 1 && leader) {
            // -------------------------------------------------------------- MMA issuer (the leader CTA only)
            constexpr uint32_t kIdesc = umma_idesc(1u, 0u, kTileM, BLOCK_N);
            int       stage = 0, buf = 0, kb = kb_first;
            uint32_t  phase = 0, buf_phase = 0;
            long long left  = (long long)((num_tiles - unit + n_units - 1) / n_units) * (kb_end - kb_first);   // K blocks of all its tiles
            // The waits for the next K block stand between the MMAs of this one: the pipe has work while they pass (a passed wait costs about 100 clocks,
            // as much as two MMAs; [1317, 1280, 5120] 18.1 -> 16.2 us).  With two products in tensor memory the one before is still being taken then, and
            // they stand in front of them (388 us against 315 for [4680, 13824, 5120]).
            constexpr bool kEarly = kBufs > 2;
            bool           ok     = !kEarly || mbar_wait_warp2(full_bar(0), 0u, tmem_empty_bar(0), 1u, abort_flag, p.wait_limit_ns);
            for (; ok && left > 0; --left) {
                if (!kEarly && !(ok = mbar_wait_warp2(full_bar(stage), phase, tmem_empty_bar(buf), buf_phase ^ 1u, abort_flag, p.wait_limit_ns))) {
                    break;
                }
                const uint32_t sa     = smem_base + stage * S::kStageBytes;
                const uint64_t adesc  = umma_desc_k_sw128(sa);
                const uint64_t bdesc  = umma_desc_k_sw128(sa + S::kABytes);
                const uint32_t d_tmem = tmem_base + (uint32_t)(buf * BLOCK_N);
                const int      steps  = min(kBlock, p.K - kb * kBlock + 31) / 32;   // MMAs of this K block; TMA fills its end with zeros
                const int      was_stage = stage, was_buf = buf;
                auto mma = [&](int k) {
                    if (k < steps) {
                        if (CTAS == 2) {
                            mma_f8f6f4_pair(d_tmem, adesc + (uint64_t)(2 * k), bdesc + (uint64_t)(2 * k), kIdesc, k > 0 ? 1u : 0u);
                        } else {
                            mma_f8f6f4(d_tmem, adesc + (uint64_t)(2 * k), bdesc + (uint64_t)(2 * k), kIdesc, k > 0 ? 1u : 0u);
                        }
                    }
                };
                tc_fence_after_sync();
                if (elect_one()) {
                    mma(0);
                    mma(1);
                }
                kb = kb + 1 == kb_end ? kb_first : kb + 1;
                if (++stage == kStages) {
                    stage = 0;
                    phase ^= 1u;
                }
                if (++buf == kBufs) {
                    buf = 0;
                    buf_phase ^= 1u;
                }
                if (kEarly && left > 1) {
                    ok = mbar_wait_warp2(full_bar(stage), phase, tmem_empty_bar(buf), buf_phase ^ 1u, abort_flag, p.wait_limit_ns);
                }
                if (elect_one()) {
                    mma(2);
                    mma(3);
                    if (CTAS == 2) {
                        tc_commit_both(empty_bar(was_stage));
                        tc_commit_both(tmem_full_bar(was_buf));
                    } else {
                        tc_commit(empty_bar(was_stage));
                        tc_commit(tmem_full_bar(was_buf));
                    }
                }
            }
            if (!ok) {
                report_timeout(p.status, 0x7200u | (unsigned)(stage << 4) | (unsigned)buf);
                *abort_flag = 1;
            }
        }
        if constexpr (SPLIT) {
            cluster_sync_all();   // the two around the partial sums
            cluster_sync_all();
        }
    } else {
        // ------------------------------------------------------------------ epilogue (warps 4..19)
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kEpiRegs));
        const int      quad      = warp & 3;                 // the TMEM lane quadrant this warp may read
        const int      quarter   = (warp - kEpiWarp0) >> 2;  // which quarter of the tile's columns
        const uint32_t lane_addr = (uint32_t)(quad * 32) << 16;
        uint8_t*       boxes     = gen_base + S::kEpiOffset + (warp - kEpiWarp0) * kBox;
        const uint32_t boxes_at  = smem_base + S::kEpiOffset + (warp - kEpiWarp0) * kBox;
        uint8_t*       bias      = p.c_dtype == LYRAQ_F32 ? boxes : gen_base + S::kEpiOffset + kEpiWarps * kBox + (warp - kEpiWarp0) * kBiasBytes;
        const bool     vec_ok    = p.c_dtype == LYRAQ_F32 ? (p.N & 3) == 0 : (p.N & 7) == 0;
        int            buf       = 0;
        uint32_t       buf_phase = 0;
        bool           ok        = true;
        for (int tile = unit; ok && tile < num_tiles; tile += n_units) {
            int m_blk, n_blk;
            tile_coords(tile, p.m_tiles, p.n_tiles, m_blk, n_blk);
            const int row0  = m_blk * kTileM + (int)rank * kBlockM + quad * 32;  // first row of this warp
            const int row   = row0 + lane;
            const int ncol0 = n_blk * BLOCK_N + quarter * kCols;
            // factors: a row or columns beyond the matrix take part with 0
            const bool   there = row < p.M && ncol0 < p.N;
            const float* xs    = p.xs.p + (there ? (size_t)row * p.xs.row_step : 0);
            const float* ws    = p.ws + (there ? (size_t)(ncol0 / kBlock) * (size_t)num_kb : 0);
            auto fetch = [&](int kb, float* sx, float* sw) {
#pragma unroll
                for (int i = 0; i < kAhead; ++i) {
                    const bool in = there && kb + i < kb_end;
                    sx[i] = in ? ld_f32(xs + (size_t)(kb + i) * p.xs.block_step) : 0.0f;
                    sw[i] = in ? ld_f32(ws + kb + i) : 0.0f;
                }
            };
            float sx[kAhead], sw[kAhead];
            fetch(kb_first, sx, sw);
            uint32_t bias_here[kChunks];
#pragma unroll
            for (int i = 0; i < kChunks; ++i) {
                const int col = ncol0 + lane + 32 * i;
                bias_here[i] = 0;
                if (p.bias != nullptr && col < p.N) {
                    bias_here[i] = p.c_dtype == LYRAQ_F32 ? reinterpret_cast<const uint32_t*>(p.bias)[col]
                                                          : (uint32_t)reinterpret_cast<const uint16_t*>(p.bias)[col];
                }
            }
            uint32_t acc[kChunks][32];
#pragma unroll
            for (int c = 0; c < kChunks; ++c) {
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    acc[c][i] = 0u;
                }
            }
            for (int kb0 = kb_first; ok && kb0 < kb_end; kb0 += kAhead) {
                float f[kAhead];
#pragma unroll
                for (int i = 0; i < kAhead; ++i) {
                    f[i] = sx[i] * sw[i];
                }
                if (kb0 + kAhead < kb_end) {
                    fetch(kb0 + kAhead, sx, sw);
                }
#pragma unroll
                for (int i = 0; i < kAhead; ++i) {
                    if (kb0 + i < kb_end && ok) {
                        if (!mbar_wait_warp(tmem_full_bar(buf), buf_phase, abort_flag, p.wait_limit_ns)) {
                            if (lane == 0) {
                                report_timeout(p.status, 0x7400u | (unsigned)buf);
                            }
                            *abort_flag = 1;
                            ok = false;
                        } else {
                            tc_fence_after_sync();
                            const uint32_t t_addr = tmem_base + lane_addr + (uint32_t)(buf * BLOCK_N + quarter * kCols);
                            const float2   f2     = make_float2(f[i], f[i]);
#pragma unroll
                            for (int c = 0; c < kChunks; ++c) {
                                uint32_t part[32];
                                tmem_ld_32x32(t_addr + (uint32_t)(c * 32), part);
                                tmem_ld_wait();
                                if (c + 1 == kChunks) {
                                    // this warp's share of the product is in registers: its buffer may be overwritten
                                    tc_fence_before_sync();
                                    __syncwarp();
                                    if (lane == 0) {
                                        if (CTAS == 2 && !leader) {
                                            mbar_arrive_cluster_relaxed(map_to_cta(tmem_empty_bar(buf), 0u));
                                        } else {
                                            mbar_arrive(tmem_empty_bar(buf));
                                        }
                                    }
                                }
#pragma unroll
                                for (int e = 0; e < 16; ++e) {
                                    const float2 a = fma_f32x2(f2, make_float2(__uint_as_float(part[2 * e]), __uint_as_float(part[2 * e + 1])),
                                                               make_float2(__uint_as_float(acc[c][2 * e]), __uint_as_float(acc[c][2 * e + 1])));
                                    acc[c][2 * e]     = __float_as_uint(a.x);
                                    acc[c][2 * e + 1] = __float_as_uint(a.y);
                                }
                            }
                            if (++buf == kBufs) {
                                buf = 0;
                                buf_phase ^= 1u;
                            }
                        }
                    }
                }
            }
            if constexpr (SPLIT) {
                cluster_sync_all();   // every CTA has taken its last product: the operands' stages are free
                const int w = warp - kEpiWarp0, own = kEpiWarps / splits, owner = w / own;
                const uint32_t to = smem_base + (uint32_t)((w % own * splits + part) * kPartBytes + lane * 4);
                if (ok) {
                    const uint32_t there_at = map_to_cta(to, (uint32_t)owner);
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        st_cluster_u32(there_at + (uint32_t)i * 128u, acc[0][i]);
                    }
                } else if (lane == 0) {
                    // one CTA that gave up leaves every part of the tile without its sums, so none of the cluster stores anything
                    for (int r = 0; r < splits; ++r) {
                        st_cluster_u32(map_to_cta(smem_u32(const_cast<int*>(abort_flag)), (uint32_t)r), 1u);
                    }
                }
                cluster_sync_all();
                if (owner != part || *abort_flag != 0) {
                    break;
                }
                const float* from = reinterpret_cast<const float*>(gen_base + (w % own * splits) * kPartBytes) + lane;
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    acc[0][i] = __float_as_uint(from[i * 32]);
                }
                for (int r = 1; r < splits; ++r) {
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        acc[0][i] = __float_as_uint(__uint_as_float(acc[0][i]) + from[r * (kPartBytes / 4) + i * 32]);
                    }
                }
            } else if (!ok) {
                break;
            }
            if (p.bias != nullptr) {
                // the warp's own piece of shared memory, so no other warp is waited for
                __syncwarp();
#pragma unroll
                for (int i = 0; i < kChunks; ++i) {
                    if (p.c_dtype == LYRAQ_F32) {
                        reinterpret_cast<uint32_t*>(bias)[lane + 32 * i] = bias_here[i];
                    } else {
                        reinterpret_cast<uint16_t*>(bias)[lane + 32 * i] = (uint16_t)bias_here[i];
                    }
                }
                __syncwarp();
            }
            // Residual of a 16-bit output: a lane that fetched its own row would touch 32 lines an instruction and use half a sector of each.
            // Instead four lanes fetch the 64 bytes of a row, eight rows an instruction, and hand them over through the box that the result leaves by.
            const bool staged = RES && !NARROW && p.residual != nullptr && p.tma_store;
            Vec16      rr[RES ? 4 : 1];
            auto fetch_residual = [&](int c, Vec16* dst) {
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
                fetch_residual(0, rr);
            }
#pragma unroll
            for (int c = 0; c < kChunks; ++c) {
                const int col0  = ncol0 + c * 32;
                const int valid = p.N - col0;
                if (valid <= 0) {
                    continue;
                }
                float     v[32];
                uint8_t*  box  = boxes;
                uint8_t*  brow = box + lane * 64;
                const int sw_  = (lane >> 1) & 3;
                if (!NARROW && p.tma_store) {
                    if (lane == 0) {
                        tma_store_wait_read();   // the last store has drained the box
                    }
                    __syncwarp();
                }
                if (staged) {
#pragma unroll
                    for (int i = 0; i < (RES ? 4 : 1); ++i) {
                        const int r = i * 8 + (lane >> 2);
                        *reinterpret_cast<Vec16*>(box + r * 64 + (((lane & 3) ^ ((r >> 1) & 3)) << 4)) = rr[i];
                    }
                    __syncwarp();
                    if (c + 1 < kChunks) {
                        fetch_residual(c + 1, rr);
                    }
                }
                const bool moved = RES && NARROW && p.residual != nullptr;
                if (moved) {
                    __syncwarp();   // the last piece has left the box
                    move_box<true>(box, const_cast<uint16_t*>(reinterpret_cast<const uint16_t*>(p.residual)), p, row0, col0, lane);
                    __syncwarp();
                }
                if (!NARROW && p.c_dtype == LYRAQ_F32) {
                    if (row < p.M) {
                        finish32<float, RES, false>(p, acc[c], bias + c * 128, nullptr, 0, 1.0f, row, col0, valid, vec_ok, v);
                        store32<float>(reinterpret_cast<float*>(p.C) + (size_t)row * (size_t)p.N + (size_t)col0, valid, vec_ok, v);
                    }
                    continue;
                }
                const bool bf16 = p.c_dtype == LYRAQ_BF16;
                if (bf16) {
                    finish32<__nv_bfloat16, RES, false>(p, acc[c], bias + c * 64, staged || moved ? brow : nullptr, sw_, 1.0f, row, col0, valid, vec_ok, v);
                } else {
                    finish32<__half, RES, false>(p, acc[c], bias + c * 64, staged || moved ? brow : nullptr, sw_, 1.0f, row, col0, valid, vec_ok, v);
                }
                if (NARROW) {
                    __syncwarp();
                }
                // 32 rows x 64 bytes through this warp's box in the 64-byte swizzle, one TMA store where rows start on 16 bytes; rows and columns beyond the matrix are clipped
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    *reinterpret_cast<Vec16*>(brow + ((q ^ sw_) << 4)) = bf16 ? pack8<__nv_bfloat16>(v + 8 * q) : pack8<__half>(v + 8 * q);
                }
                if (NARROW) {
                    __syncwarp();
                    move_box<false>(box, reinterpret_cast<uint16_t*>(p.C), p, row0, col0, lane);
                    continue;
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0 && row0 < p.M) {
                    tma_store_2d(&tmap_c, boxes_at, col0, row0);
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
    grid_launch_dependents();   // not before: a kernel behind that waits beside this one takes its slots
    if (warp == 2) {
        tc_fence_after_sync();
        if (CTAS == 2) {
            tmem_dealloc_pair(tmem_base, 512);
        } else {
            tmem_dealloc(tmem_base, 512);
        }
    }
}

template<int BLOCK_N, int CTAS, bool RES, bool NARROW, bool SPLIT> static int launch(const uint8_t* X, const uint8_t* W, GemmParams p, int sms, cudaStream_t stream)
{
    using S = Smem<BLOCK_N, CTAS>;
    CUtensorMap ta, tb;
    int         st = make_tmap_bytes_2d(&ta, X, (uint64_t)p.M, (uint64_t)p.K, (uint64_t)p.K, kBlockM, kBlock, true);
    if (st == LYRAQ_OK) {
        st = make_tmap_bytes_2d(&tb, W, (uint64_t)p.N, (uint64_t)p.K, (uint64_t)p.K, BLOCK_N / CTAS, kBlock, true);
    }
    CUtensorMap tc = ta;   // never used where the output is stored directly
    p.tma_store    = !NARROW && p.c_dtype != LYRAQ_F32;
    if (st == LYRAQ_OK && p.tma_store) {
        st = make_tmap_store(&tc, p.C, (uint64_t)p.M, (uint64_t)p.N, (uint64_t)p.N, 2, false);
    }
    if (st != LYRAQ_OK) {
        return st;
    }
    p.m_tiles = (int)(((long)p.M + kBlockM * CTAS - 1) / (kBlockM * CTAS));
    p.n_tiles = (int)(((long)p.N + BLOCK_N - 1) / BLOCK_N);
    const long long tiles = (long long)p.m_tiles * p.n_tiles;
    if (tiles > (SPLIT ? 0x1000000ll : 0x40000000ll)) {
        return LYRAQ_ERR_UNSUPPORTED;
    }
    const long long units = sms / CTAS;
    const int       grid  = SPLIT ? (int)tiles * p.splits : (int)(tiles < units ? tiles : units) * CTAS;
    auto            kern  = gemm_fp8_block_kernel<BLOCK_N, CTAS, RES, NARROW, SPLIT>;
    static bool     smem_raised[64] = {};
    st = raise_dynamic_smem_once(kern, (int)S::kTotal, smem_raised, "cudaFuncSetAttribute(gemm_fp8_block_kernel, dynamic shared memory)");
    if (st != LYRAQ_OK) {
        return st;
    }
    return cuda_status(launch_kernel(kern, (unsigned)grid, (unsigned)kThreads, (size_t)S::kTotal, stream, (unsigned)(SPLIT ? p.splits : CTAS), ta, tb, tc, p),
                       "cudaLaunchKernelEx(gemm_fp8_block_kernel)");
}

// forced kernel for tests and sweeps: 0 = automatic, 16 = the few-row kernel (up to 16 rows), 2562 = CTA pair with 256 x 256, 1281 = one CTA with 128 x 128,
// 1282, 1284, 1288 = that with 2, 4 or 8 CTAs along K
static int g_forced_tile = 0;
// Test hook (lyraq_debug_fp8_block_wait_test)
static int                g_stalled_rank  = -1;
static unsigned long long g_wait_limit_ns = kWaitLimitNs;

bool few_rows(int m, int n, int k)
{
    // The few-row kernel's time grows with the rows (their partial sums cross shared memory and leave row by row), the other's does not; what it gains
    // grows with K.  Dense against few-row, a linear, us: 6 rows of [256, 256] 4.7 / 4.6, of [1280, 768] 5.9 / 5.8, 8 rows of it 5.9 / 6.2, 16 rows of [1280, 1024] 6.5 /
    // 6.5, of [1280, 5120] 16.2 / 7.4, of [13824, 5120] 25 / 20; one row of [5120, 5120] 16.9 / 9.5.
    const bool pays = m <= 6 || k > 7 * kBlock;
    return m <= kFewRows && (g_forced_tile == 16 || (g_forced_tile == 0 && pays)) && rows_fit(n, k, device_sm_count());
}

bool few_rows_quantize(int m, int n, int k) { return few_rows(m, n, k) && (g_forced_tile == 16 || rows_quantize_pays(m, n, k, device_sm_count())); }

// What a split costs, us: the cluster's launch and the partial sums' way (2.5 with 2 CTAs, 3.2 with 4, 3.6 with 8).  One CTA / the split it picks, us:
// [64, 5120, 13824] 35.9 / 25.0, [300, 1280, 5120] 15.3 / 10.1, [28, 1290, 12480] 33.7 / 11.7, [154, 1280, 2048] 8.1 / 7.3; [17, 1280, 1280] 5.7 against 6.9 stays whole.
constexpr double kSplitCost = 3.2;

static int run(const Input& X, const uint8_t* W, GemmParams p, int sms, cudaStream_t stream)
{
    if (few_rows(p.M, p.N, p.K)) {
        return launch_rows(X, W, p, sms, stream);
    }
    const long m128 = ((long)p.M + 127) / 128, n128 = ((long)p.N + 127) / 128, m256 = ((long)p.M + 255) / 256, n256 = ((long)p.N + 255) / 256;
    const long pairs = sms / 2;
    const int  num_kb = (p.K + kBlock - 1) / kBlock;
    // Rounds of each tile times what one takes, us: 0.6 + 0.33 a K block for 128 x 128, 1.0 + 0.53 for a pair's 256 x 256, from [4608, 3072, 12288] (194 / 157),
    // [4608, 3072, 3072] (53 / 42), [512, 5120, 5120] (30 / 23), [1317, 5120, 1280] (15.0 / 16.6), [2309, 4808, 1136] (26.6 / 24.3).
    const double c1   = (double)((m128 * n128 + sms - 1) / sms) * (0.6 + 0.33 * num_kb);
    const double c2   = pairs > 0 ? (double)((m256 * n256 + pairs - 1) / pairs) * (1.0 + 0.53 * num_kb) : 1e30;
    int          tile = g_forced_tile > 16 ? g_forced_tile : c2 <= c1 ? 2562 : 1281;
    p.splits = 1;
    if (g_forced_tile > 1281 && g_forced_tile < 1289) {
        p.splits = g_forced_tile - 1280;
        while (p.splits > num_kb) {
            p.splits /= 2;
        }
    } else if (g_forced_tile == 0) {
        // CTAs along K where few tiles have many K blocks, in one wave of clusters (of 4 and 8 some SMs of a GPC are left over): kSplitCost more a call
        double best = c1 < c2 ? c1 : c2;
        for (int s = 2; s <= 8 && s <= num_kb; s *= 2) {
            const long   room = s == 2 ? sms / 2 : s == 4 ? sms * 35l / 148 : sms * 16l / 148;
            const double cost = kSplitCost + 0.6 + 0.33 * ((num_kb + s - 1) / s);
            if (m128 * n128 <= room && cost < best) {
                best     = cost;
                p.splits = s;
            }
        }
    }
    if (p.splits > 1) {
        tile = 1282;
    }
    const bool narrow = p.c_dtype != LYRAQ_F32 && (p.N & 7) != 0;
    auto pick = [&](auto res, auto nar) {
        constexpr bool kRes = decltype(res)::value, kNarrow = decltype(nar)::value;
        return tile == 2562   ? launch<256, 2, kRes, kNarrow, false>(X.codes, W, p, sms, stream)
               : tile == 1282 ? launch<128, 1, kRes, kNarrow, true>(X.codes, W, p, sms, stream)
                              : launch<128, 1, kRes, kNarrow, false>(X.codes, W, p, sms, stream);
    };
    using Yes = std::true_type;
    using No  = std::false_type;
    return p.residual != nullptr ? (narrow ? pick(Yes{}, Yes{}) : pick(Yes{}, No{})) : narrow ? pick(No{}, Yes{}) : pick(No{}, No{});
}

int product(const Input& X, const uint8_t* W, const float* ws, void* Y, int c_dtype, const void* bias, const void* residual, float beta, int epilogue, int m,
            int n, int k, cudaStream_t stream)
{
    GemmParams p{};
    p.M        = m;
    p.N        = n;
    p.K        = k;
    p.C        = Y;
    p.c_dtype  = c_dtype;
    p.xs       = X.scales;
    p.ws       = ws;
    p.bias     = bias;
    p.residual = residual;
    p.beta     = beta;
    p.gelu     = epilogue == LYRAQ_EPI_GELU_TANH;
    p.status   = status_word_ptr();
    p.wait_limit_ns = g_wait_limit_ns;
    p.stalled_rank  = g_stalled_rank;
    const int sms = device_sm_count();
    if (p.status == nullptr || sms <= 0) {
        return LYRAQ_ERR_CUDA;
    }
    return run(X, W, p, sms, stream);
}

}  // namespace fp8b
}  // namespace lyraq

using namespace lyraq;

extern "C" {

int lyraq_debug_force_fp8_block_tile(int code)
{
    if (code != 0 && code != 16 && code != 1281 && code != 1282 && code != 1284 && code != 1288 && code != 2562) {
        return LYRAQ_ERR_INVALID_ARG;
    }
    fp8b::g_forced_tile = code;
    return LYRAQ_OK;
}

int lyraq_debug_fp8_block_wait_test(int stalled_rank, unsigned int wait_limit_ms)
{
    fp8b::g_stalled_rank  = stalled_rank;
    fp8b::g_wait_limit_ns = wait_limit_ms == 0 ? kWaitLimitNs : (unsigned long long)wait_limit_ms * 1000000ull;
    return LYRAQ_OK;
}

int lyraq_gemm_fp8_block(const uint8_t* X, const float* x_scale, size_t x_scale_row, size_t x_scale_block, const uint8_t* W, const float* w_scale, void* Y,
                         int c_dtype, const void* bias, const void* residual, float beta, int epilogue, int m, int n, int k, void* stream)
{
    if (m < 0 || n < 0 || k < 0 || (epilogue != LYRAQ_EPI_NONE && epilogue != LYRAQ_EPI_GELU_TANH) ||
        (c_dtype != LYRAQ_F16 && c_dtype != LYRAQ_BF16 && c_dtype != LYRAQ_F32)) {
        return LYRAQ_ERR_INVALID_ARG;
    }
    if (m == 0 || n == 0) {
        return LYRAQ_OK;
    }
    if (k == 0 || (k & 15) != 0 || m > fp8b::kMaxSize || n > fp8b::kMaxSize || k > fp8b::kMaxSize) {
        return LYRAQ_ERR_UNSUPPORTED;
    }
    if (X == nullptr || x_scale == nullptr || W == nullptr || w_scale == nullptr || Y == nullptr || !aligned16(X) || !aligned16(W) || !aligned16(Y) ||
        ((reinterpret_cast<uintptr_t>(x_scale) | reinterpret_cast<uintptr_t>(w_scale)) & 3u) != 0 || (bias != nullptr && !aligned16(bias)) ||
        (residual != nullptr && !aligned16(residual))) {
        return LYRAQ_ERR_INVALID_ARG;
    }
    const size_t rows = (size_t)m, cols = (size_t)n, depth = (size_t)k, blocks = fp8b::blocks_of(depth), bytes = c_dtype == LYRAQ_F32 ? 4 : 2;
    if (result_clashes(view_of(Y, rows * cols * bytes), residual,
                       {view_of(X, rows * depth), view_of(x_scale, 4, rows, x_scale_row, blocks, x_scale_block, 1, 0, 1), view_of(W, cols * depth),
                        view_of(w_scale, fp8b::blocks_of(cols) * blocks * 4), view_of(bias, cols * bytes)})) {
        return LYRAQ_ERR_INVALID_ARG;
    }
    return fp8b::product({X, {x_scale, x_scale_row, x_scale_block}, nullptr, 0, 0}, W, w_scale, Y, c_dtype, bias, residual, beta, epilogue, m, n, k,
                         (cudaStream_t)stream);
}

}  // extern "C"
