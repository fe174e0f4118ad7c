// Block-sparse attention forward: out[b, i, h, :] = softmax over the keys of the blocks listed for query block i / 128 of (q k^T scale) v.
//
// The kernel of attention.cu with lists: a CTA runs two query tiles of 128 rows, which share the tensor pipe and the exponent unit but no operand,
// since each has its own list.  So each has its own producer and part of shared memory, and takes its own query blocks ("items") in turn:
//   warps 8, 10  TMA producers of tile 0, 1.  They find each item's list and length and tell the other roles through a ring of two; then Q, and K and V
//                of each step of 128 keys (two listed blocks of 64, or one of 128), as boxes of 64 keys x 64 columns.  One buffer for K (free as soon as
//                the scores are there, needed when P V of the step is under way) and a ring of half steps for V.
//   warp 9       MMA issuer of both tiles, a step of each in turn: O += P V (P from tensor memory, in two halves of 64 keys), then the next step's
//                S = Q K^T over it
//   warps 0-3    softmax and epilogue of tile 0, warps 4-7 of tile 1: a thread owns one query row.  Keys of a half step that a row does not see are a
//                tail of it (beyond the keys, or behind the row's place), so a mask is one number.
// V rows beyond a sequence's keys may hold anything: the softmax warps clear them in shared memory, since 0 * NaN is NaN.
// P is rounded to the tensors' type, which the MMAs ask for (both operands of one type); its sum l is of the numbers before.
// Every wait is bounded; on a timeout the role records it in the status word, raises the block's abort flag and all roles leave; tensor
// memory is freed at the common exit.
//
// What bounds it (32760 tokens, 12 heads of 128, 64 of 512 blocks: 98304 steps of one tile, 824 GFLOP): the chain of a tile's softmax and MMAs, as in
// the dense kernel; a step of both tiles is 2048 clocks of tensor pipe, 1792 of the exponent unit, 3500 measured for long lists, 2.1 us (the dense
// kernel, which reads K and V once for two tiles: 1.8), and an item costs 3 us beside its steps.  K and V of a step are 64 KB for one tile; without the loads it takes the same time.
// Measured, the clip: 908 us with an issuer for each tile (their instructions mix on the pipe and both products end late) -> 759 with one -> 745 with
// items handed over and keys looked up only where a mask may be (a look at each step's keys by the softmax warps: 6 to 12 %).
// Not kept: an epilogue in warps of its own, which wait for either tile (their polling and the registers they take from the softmax: 848 to 1030 us); items found by a
// warp of their own (the same time); a quarter of the exponentials on the FMA pipe (2 % slower than an eighth).
#include "sparse_attention.cuh"
#include "sm100_ptx.cuh"

namespace lyraq {

using namespace sm100;

typedef CUresult (*EncodeTiledFnSparse)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                        const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                        CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

int device_sm_count();  // gemm_dense.cu

namespace sattn {

using attn::ex2_approx;
using attn::ex2_poly;
using attn::max3;

constexpr int kTile    = 128;                       // rows of a query tile, keys of a step
constexpr int kHalf    = 64;
constexpr int kTiles   = 2;
constexpr int kThreads = 384;
constexpr int kRole0   = 8;                         // warps 8 and 10 producers, 9 issuer
// registers: 384 threads x 168 at launch = 64512 = 256 x 216 + 128 x 72
constexpr int kSoftmaxRegs = 216;
constexpr int kOtherRegs   = 72;
constexpr int kInfos       = 2;                     // items a producer may be ahead with
constexpr float kRescaleThreshold = 8.0f;           // in log2 units
constexpr int kPolyPairs = 2;                       // of 16 pairs of scores, how many take their exponentials from the FMA pipe

template<int D> struct Smem {
    static constexpr int kPanels  = D / 64;                       // boxes of 64 columns side by side
    static constexpr int kPanelQ  = kTile * 128;                  // a panel of 128 rows
    static constexpr int kPanelV  = kHalf * 128;
    static constexpr int kQBytes  = kPanels * kPanelQ;
    static constexpr int kKBytes  = kQBytes;
    static constexpr int kVBytes  = kPanels * kPanelV;            // half a step
    static constexpr int kKSlots  = D == 128 ? 1 : 2;
    static constexpr int kVSlots  = D == 128 ? 3 : 6;
    static constexpr int kKOffset = kQBytes;
    static constexpr int kVOffset = kKOffset + kKSlots * kKBytes;
    static constexpr int kPerTile = kVOffset + kVSlots * kVBytes;
    // barriers of a tile, by number
    static constexpr int kQFull = 0, kQEmpty = 1, kSFull = 2, kPHalf = 3, kOFull = 5, kInfoFull = 6,
                         kInfoEmpty = kInfoFull + kInfos, kKFull = kInfoEmpty + kInfos, kKEmpty = kKFull + kKSlots, kVFull = kKEmpty + kKSlots,
                         kVEmpty = kVFull + kVSlots, kBars = kVEmpty + kVSlots;
    static constexpr int kInfoOffset = kTiles * kPerTile;
    static constexpr int kBarOffset  = kInfoOffset + kTiles * kInfos * 48;
    static constexpr int kUsed    = kBarOffset + 8 * kBars * kTiles + 16;
    static constexpr int kTotal   = kUsed + 1024;                 // + alignment slack
    static_assert(kTotal <= 232448 && kPerTile % 1024 == 0, "");
};

__device__ __forceinline__ void tma_load_4d(uint32_t smem_dst, const CUtensorMap* m, uint32_t bar, int x, int y, int z, int w)
{
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
        ::"r"(smem_dst), "l"(m), "r"(bar), "r"(x), "r"(y), "r"(z), "r"(w)
        : "memory");
}

// What a producer tells the other roles of an item: query block `qb` of head `h` of sequence `b`, its steps (-1: no item any more), the row of its list, how
// much of the list counts, the keys that exist, the last key its row 0 sees, the first step in which a row may miss a key, the first keys of the
// halves of its first step.
struct alignas(16) Info {
    int qb, h, b, steps;
    int list, entries, len, place;
    int masked, key[2], spare;
};
static_assert(sizeof(Info) == 48, "");

template<typename T, int D>
__global__ void __launch_bounds__(kThreads, 1)
sparse_attention_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
                        const __grid_constant__ Params p)
{
    using S = Smem<D>;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t*       gen_base  = smem_raw + (smem_base - smem_u32(smem_raw));
    auto bars_of = [&](int t) { return smem_base + S::kBarOffset + 8u * (uint32_t)(t * S::kBars); };
    auto info_of = [&](int t, int slot) { return reinterpret_cast<Info*>(gen_base + S::kInfoOffset) + t * kInfos + slot; };
    uint32_t*     tmem_slot  = reinterpret_cast<uint32_t*>(gen_base + S::kBarOffset + 8 * S::kBars * kTiles);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int warp = warp_index();
    const int lane = threadIdx.x & 31;

    grid_launch_dependents();
    if (threadIdx.x == 0) {
        for (int t = 0; t < kTiles; ++t) {
            for (int i = 0; i < S::kBars; ++i) {
                // P comes from four warps, "item taken" from these and the issuer
                const bool four = i == S::kPHalf || i == S::kPHalf + 1, five = i >= S::kInfoEmpty && i < S::kInfoEmpty + kInfos;
                mbar_init(bars_of(t) + 8u * (uint32_t)i, four ? 4u : five ? 5u : 1u);
            }
        }
        *abort_flag = 0;
        fence_barrier_init();
        prefetch_tensormap(&tmap_q);
        prefetch_tensormap(&tmap_k);
        prefetch_tensormap(&tmap_v);
    }
    if (warp == kRole0 + 1) {
        tmem_alloc(smem_u32(tmem_slot), 512);
        tmem_relinquish();
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem_base = *tmem_slot;
    grid_dependency_wait();

    auto give_up = [&](unsigned code) {
        report_timeout(p.status, code);
        *abort_flag = 1;
    };
    auto wait = [&](uint32_t b, uint32_t parity, unsigned code) {
        const bool ok = mbar_wait_warp(b, parity, abort_flag, p.wait_limit_ns);
        if (!ok) {
            give_up(code);
        }
        return ok;
    };
    // first key of half s of step i of a list, or `keys` where there is none: a box there is filled with zeros and its keys are masked
    auto key_of = [&](int list, int entries, int i, int s) {
        const int e = p.block == kTile ? i : 2 * i + s;
        if (e >= entries) {
            return p.keys;
        }
        const int j = load_int(p.index + (size_t)list * (size_t)p.count + (size_t)e);
        return j >= 0 && j <= (p.keys - 1) / p.block ? min(j * p.block + (p.block == kTile ? s * kHalf : 0), p.keys) : p.keys;
    };

    if (warp >= kRole0) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
        if ((warp & 1) == 0) {
            // -------------------------------------------------------------- TMA producer
            const int      t    = (warp - kRole0) >> 1;
            const uint32_t bars = bars_of(t), smem = smem_base + (uint32_t)(t * S::kPerTile);
            int      k_slot = 0, v_slot = 0, k_issued = 0, v_issued = 0, q_issued = 0, infos = 0;
            uint32_t k_phase = 0, v_phase = 0;
            bool     ok = p.skip_loads == 0;
            // tile 0 of every CTA first: few items spread over all SMs
            auto look = [&](int i) {
                Info it{0, 0, 0, -1, 0, 0, 0, 0, 0, {p.keys, p.keys}, 0};
                if (i < p.items) {
                    it.qb      = i % p.q_blocks;
                    it.h       = i / p.q_blocks % p.q_heads;
                    it.b       = i / (p.q_blocks * p.q_heads);
                    it.list    = (it.b * p.lists + it.h / (p.q_heads / p.lists)) * p.q_blocks + it.qb;
                    it.entries = min(max(load_int(p.counts + it.list), 0), p.count);
                    it.steps   = p.block == kTile ? it.entries : (it.entries + 1) / 2;
                    it.len     = key_count(p, it.b);
                    it.place   = p.causal ? (int)min((long long)first_place(p, it.b) + it.qb * kTile, (long long)kMaxKeys) : p.keys;
                    // The lists as select_blocks leaves them ascend, so blocks that end behind the keys or a row's place are at their end; the softmax warps
                    // look at no list before the first of them (a look at each step's keys there took 6 to 12 % of the time).
                    const int least = min(it.len, p.causal ? it.place + 1 : it.len);     // keys that row 0 sees
                    int       first = it.entries;
                    for (int e = lane; e < it.entries; e += 32) {
                        const int j = load_int(p.index + (size_t)it.list * (size_t)p.count + (size_t)e);
                        if (j < 0 || j >= least / p.block) {
                            first = min(first, e);
                        }
                    }
                    first     = __reduce_min_sync(0xffffffffu, first);
                    it.masked = p.block == kTile ? first : first / 2;
                    it.key[0] = key_of(it.list, it.entries, 0, 0);
                    it.key[1] = key_of(it.list, it.entries, 0, 1);
                }
                return it;
            };
            const int stride = kTiles * (int)gridDim.x;
            int       i      = (int)blockIdx.x + t * (int)gridDim.x;
            Info      it     = look(i);
            while (ok) {
                const int slot = infos % kInfos;
                if (!(ok = wait(bars + 8u * (S::kInfoEmpty + slot), (uint32_t)(infos / kInfos & 1) ^ 1u, 0x8130u))) {
                    break;
                }
                if (lane == 0) {
                    *info_of(t, slot) = it;
                    mbar_arrive(bars + 8u * (S::kInfoFull + slot));
                }
                ++infos;
                if (it.steps < 0) {
                    break;
                }
                i += stride;
                if (it.steps == 0) {
                    it = look(i);
                    continue;
                }
                if (!(ok = wait(bars + 8u * S::kQEmpty, (uint32_t)(q_issued & 1) ^ 1u, 0x8110u))) {
                    break;
                }
                const int kh = it.h / (p.q_heads / p.k_heads);
                if (elect_one()) {
                    mbar_arrive_expect_tx(bars + 8u * S::kQFull, (uint32_t)S::kQBytes);
#pragma unroll
                    for (int c = 0; c < S::kPanels; ++c) {
                        tma_load_4d(smem + c * S::kPanelQ, &tmap_q, bars + 8u * S::kQFull, c * 64, it.qb * kTile, it.h, (p.fixed & 1) != 0 ? 0 : it.b);
                    }
                }
                ++q_issued;
                int key[2] = {it.key[0], it.key[1]};
                for (int s = 0; ok && s < it.steps; ++s) {
                    int ahead[2] = {p.keys, p.keys};
                    if (s + 1 < it.steps) {      // on their way while the buffers are waited for
                        ahead[0] = key_of(it.list, it.entries, s + 1, 0);
                        ahead[1] = key_of(it.list, it.entries, s + 1, 1);
                    }
                    if (!(ok = wait(bars + 8u * (S::kKEmpty + k_slot), k_phase ^ 1u, 0x8100u))) {
                        break;
                    }
                    if (elect_one()) {
                        const uint32_t dst = smem + S::kKOffset + k_slot * S::kKBytes, full = bars + 8u * (S::kKFull + k_slot);
                        mbar_arrive_expect_tx(full, (uint32_t)S::kKBytes);
#pragma unroll
                        for (int c = 0; c < S::kPanels; ++c) {
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                tma_load_4d(dst + c * S::kPanelQ + h * S::kPanelV, &tmap_k, full, c * 64, key[h], kh, (p.fixed & 2) != 0 ? 0 : it.b);
                            }
                        }
                    }
                    ++k_issued;
                    if (++k_slot == S::kKSlots) {
                        k_slot = 0;
                        k_phase ^= 1u;
                    }
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        if (!ok || !(ok = wait(bars + 8u * (S::kVEmpty + v_slot), v_phase ^ 1u, 0x8120u))) {
                            break;
                        }
                        if (elect_one()) {
                            const uint32_t dst = smem + S::kVOffset + v_slot * S::kVBytes, full = bars + 8u * (S::kVFull + v_slot);
                            mbar_arrive_expect_tx(full, (uint32_t)S::kVBytes);
#pragma unroll
                            for (int c = 0; c < S::kPanels; ++c) {
                                tma_load_4d(dst + c * S::kPanelV, &tmap_v, full, c * 64, key[h], kh, (p.fixed & 4) != 0 ? 0 : it.b);
                            }
                        }
                        ++v_issued;
                        if (++v_slot == S::kVSlots) {
                            v_slot = 0;
                            v_phase ^= 1u;
                        }
                    }
                    key[0] = ahead[0];
                    key[1] = ahead[1];
                }
                it = look(i);
            }
            // no copy may be in flight when the block leaves: wait (bounded) for the buffers filled last
            auto settle = [&](uint32_t b, uint32_t parity, unsigned code) {
                const uint64_t t0 = global_timer_ns();
                while (!mbar_try_wait(b, parity)) {
                    if (global_timer_ns() - t0 > p.wait_limit_ns) {
                        report_timeout(p.status, code);
                        break;
                    }
                }
            };
            for (int n = 0; n < S::kKSlots && n < k_issued; ++n) {
                if (k_slot == 0) {
                    k_slot = S::kKSlots;
                    k_phase ^= 1u;
                }
                --k_slot;
                settle(bars + 8u * (S::kKFull + k_slot), k_phase, 0x8400u);
            }
            for (int n = 0; n < S::kVSlots && n < v_issued; ++n) {
                if (v_slot == 0) {
                    v_slot = S::kVSlots;
                    v_phase ^= 1u;
                }
                --v_slot;
                settle(bars + 8u * (S::kVFull + v_slot), v_phase, 0x8420u);
            }
            if (q_issued > 0) {
                settle(bars + 8u * S::kQFull, (uint32_t)((q_issued - 1) & 1), 0x8410u);
            }
        } else if (warp == kRole0 + 1) {
            // -------------------------------------------------------------- MMA issuer of both tiles
            constexpr uint32_t kAb = TypeTag<T>::value == LYRAQ_BF16 ? 1u : 0u;
            constexpr uint32_t idesc_qk = umma_idesc(1u, kAb, 128, kTile);
            constexpr uint32_t idesc_pv = umma_idesc(1u, kAb, 128, D) | kIdescBMajorMN;
            // One copy of the code serves both tiles in turn, and a wait that runs out is reported behind the loop: what the issuer runs between two
            // MMAs is fetched anew every time, as the other warps run theirs in between.
            struct Tile {
                int      t, steps, step;         // steps of the item under way (0: none yet, -1: no item any more)
                int      infos, v_slot, k_slot;
                uint32_t v_phase, k_phase, parity, item_parity;   // parity: of the steps of all items; item_parity: of the items with steps
            };
            Tile     c{0, 0, 0, 0, 0, 0, 0u, 0u, 0u, 0u}, other{1, 0, 0, 0, 0, 0, 0u, 0u, 0u, 0u};
            unsigned bad = 0;
            auto wait_for = [&](uint32_t b, uint32_t parity, unsigned code) {
                if (!mbar_wait_warp(b, parity, abort_flag, p.wait_limit_ns)) {
                    bad = code;
                    return false;
                }
                return true;
            };
            while (bad == 0 && (c.steps >= 0 || other.steps >= 0)) {
                if (c.steps >= 0) {
                    const uint32_t smem = smem_base + (uint32_t)(c.t * S::kPerTile), bars = bars_of(c.t);
                    const uint32_t s_acc = tmem_base + (uint32_t)(c.t * 128), o_acc = tmem_base + (uint32_t)(256 + c.t * 128);
                    bool           ok = true;
                    if (c.steps > 0) {
                        // O += P V of the step
                        const bool last = c.step + 1 == c.steps;
#pragma unroll 1
                        for (int h = 0; h < 2 && ok; ++h) {
                            ok = wait_for(bars + 8u * (uint32_t)(S::kVFull + c.v_slot), c.v_phase, 0x8230u) &&
                                 wait_for(bars + 8u * (uint32_t)(S::kPHalf + h), c.parity, 0x8240u);
                            if (!ok) {
                                break;
                            }
                            tc_fence_after_sync();
                            if (elect_one()) {
                                const uint64_t vdesc = umma_desc_mn_sw128(smem + S::kVOffset + c.v_slot * S::kVBytes, (uint32_t)S::kPanelV);
                                const uint32_t acc = c.step > 0 || h > 0 ? 1u : 0u, p_in = s_acc + (uint32_t)(h * 32);
#pragma unroll
                                for (int k4 = 0; k4 < 4; ++k4) {   // 16 keys each: 8 columns of P, 2048 bytes of v
                                    mma_f16_ts(o_acc, p_in + (uint32_t)(k4 * 8), vdesc + (uint64_t)(k4 * 128), idesc_pv, k4 > 0 ? 1u : acc);
                                }
                                tc_commit(bars + 8u * (uint32_t)(S::kVEmpty + c.v_slot));
                                if (h == 1 && last) {
                                    tc_commit(bars + 8u * S::kOFull);
                                }
                            }
                            if (++c.v_slot == S::kVSlots) {
                                c.v_slot = 0;
                                c.v_phase ^= 1u;
                            }
                        }
                        c.parity ^= 1u;
                        ++c.step;
                        if (last) {
                            c.step = c.steps = 0;
                            c.item_parity ^= 1u;
                        }
                    }
                    // the next item that has steps
                    while (ok && c.steps == 0) {
                        const int slot = c.infos % kInfos;
                        ok = wait_for(bars + 8u * (uint32_t)(S::kInfoFull + slot), (uint32_t)(c.infos / kInfos & 1), 0x8250u);
                        if (ok) {
                            c.steps = info_of(c.t, slot)->steps;
                            __syncwarp();
                            if (lane == 0) {
                                mbar_arrive(bars + 8u * (uint32_t)(S::kInfoEmpty + slot));
                            }
                            ++c.infos;
                        }
                    }
                    // S = Q K^T of its next step, over P, which the MMAs before read, in order
                    if (ok && c.steps > 0) {
                        ok = (c.step > 0 || wait_for(bars + 8u * S::kQFull, c.item_parity, 0x8200u)) &&
                             wait_for(bars + 8u * (uint32_t)(S::kKFull + c.k_slot), c.k_phase, 0x8210u);
                        if (ok) {
                            tc_fence_after_sync();
                            if (elect_one()) {
                                const uint64_t qdesc = umma_desc_k_sw128(smem);
                                const uint64_t kdesc = umma_desc_k_sw128(smem + S::kKOffset + c.k_slot * S::kKBytes);
#pragma unroll
                                for (int ks = 0; ks < D / 16; ++ks) {
                                    const uint64_t off = (uint64_t)(((ks >> 2) * S::kPanelQ + (ks & 3) * 32) >> 4);
                                    mma_f16(s_acc, qdesc + off, kdesc + off, idesc_qk, ks > 0 ? 1u : 0u);
                                }
                                tc_commit(bars + 8u * S::kSFull);
                                tc_commit(bars + 8u * (uint32_t)(S::kKEmpty + c.k_slot));
                                if (c.step + 1 == c.steps) {
                                    tc_commit(bars + 8u * S::kQEmpty);
                                }
                            }
                            if (++c.k_slot == S::kKSlots) {
                                c.k_slot = 0;
                                c.k_phase ^= 1u;
                            }
                        }
                    }
                }
                const Tile was = c;
                c     = other;
                other = was;
            }
            if (bad != 0) {
                give_up(bad);
            }
        }
    } else {
        // ------------------------------------------------------------------ softmax, one thread per query row
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
        const int      t        = warp >> 2;
        const int      quadrant = warp & 3;                                    // tensor-memory lane quadrant of this warp
        const int      r        = quadrant * 32 + lane;                        // row of the tile
        const uint32_t bars     = bars_of(t);
        const uint32_t lanes    = tmem_base + ((uint32_t)(quadrant * 32) << 16);
        const uint32_t s_addr   = lanes + (uint32_t)(t * 128);
        const uint32_t o_addr   = lanes + (uint32_t)(256 + t * 128);
        const float    c        = p.scale_log2;
        const bool     wide     = (reinterpret_cast<uintptr_t>(p.out) & 31u) == 0 && ((p.os.batch | p.os.token | p.os.head) & 15) == 0;   // rows on 32 bytes
        bool           ok       = true;
        uint32_t       g        = 0;                                           // steps of all items
        int            infos = 0, done = 0;
        while (ok) {
            const int slot = infos % kInfos;
            if (!(ok = wait(bars + 8u * (S::kInfoFull + slot), (uint32_t)(infos / kInfos & 1), 0x8340u))) {
                break;
            }
            const Info it = *info_of(t, slot);
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(bars + 8u * (uint32_t)(S::kInfoEmpty + slot));
            }
            ++infos;
            const int steps = it.steps, row = it.qb * kTile + r;
            if (steps < 0) {
                break;
            }
            // O / l, rounded to T
            uint32_t w[D / 2];
            auto store = [&]() {
                if (row < p.queries) {
                    T* dst = reinterpret_cast<T*>(p.out) + (long long)it.b * p.os.batch + (long long)row * p.os.token + (long long)it.h * p.os.head;
                    if (wide) {
#pragma unroll
                        for (int k = 0; k < D / 16; ++k) {
                            const Vec16 x = {w[8 * k], w[8 * k + 1], w[8 * k + 2], w[8 * k + 3]}, y = {w[8 * k + 4], w[8 * k + 5], w[8 * k + 6], w[8 * k + 7]};
                            st_32(dst + 16 * k, x, y);
                        }
                    } else {
#pragma unroll
                        for (int k = 0; k < D / 8; ++k) {
                            reinterpret_cast<uint4*>(dst)[k] = make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
                        }
                    }
                }
            };
            if (steps == 0) {
#pragma unroll
                for (int k = 0; k < D / 2; ++k) {
                    w[k] = 0u;
                }
                store();
                continue;
            }
            float m = -INFINITY;                                               // reference maximum of this row's raw scores; -inf: no key seen
            float l = 0.0f;                                                    // sum of exp2((s - m) c)
#pragma unroll 1
            for (int s_i = 0; s_i < steps; ++s_i, ++g) {
                // Keys [0, see[h]) of a half are this row's.  V rows that do not exist but lie in the tensor are cleared before the issuer hears of P.
                int see[2] = {kHalf, kHalf};
                if (s_i >= it.masked) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int key = key_of(it.list, it.entries, s_i, h), exist = min(max(it.len - key, 0), kHalf);
                        see[h]        = p.causal ? min(max(it.place + r - key + 1, 0), exist) : exist;
                        if (exist < kHalf && key + exist < p.keys) {
                            const uint32_t n = 2u * g + (uint32_t)h, slot_v = n % (uint32_t)S::kVSlots;
                            ok = ok && wait(bars + 8u * (S::kVFull + slot_v), n / (uint32_t)S::kVSlots & 1u, 0x8310u | (unsigned)t);
                            // two threads a row, which is 128 bytes in every panel
                            if (ok && (r >> 1) >= exist) {
                                uint8_t* at = gen_base + t * S::kPerTile + S::kVOffset + (int)slot_v * S::kVBytes + (r >> 1) * 128 + (r & 1) * 64;
#pragma unroll
                                for (int cc = 0; cc < S::kPanels; ++cc) {
#pragma unroll
                                    for (int e = 0; e < 4; ++e) {
                                        *reinterpret_cast<uint4*>(at + cc * S::kPanelV + e * 16) = make_uint4(0u, 0u, 0u, 0u);
                                    }
                                }
                            }
                            fence_proxy_async_smem();
                        }
                    }
                }
                if (!ok) {
                    break;
                }
                if (!(ok = wait(bars + 8u * S::kSFull, g & 1u, 0x8300u | (unsigned)t))) {
                    break;
                }
                tc_fence_after_sync();
                uint32_t s[128];
#pragma unroll
                for (int cc = 0; cc < 4; ++cc) {
                    tmem_ld_32x32(s_addr + cc * 32, s + cc * 32);
                }
                tmem_ld_wait();
                if (s_i >= it.masked) {
#pragma unroll
                    for (int k = 0; k < 128; ++k) {
                        if ((k & 63) >= see[k >> 6]) {
                            s[k] = 0xff800000u;                                // -inf
                        }
                    }
                }
                float mx[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    mx[j] = max3(__uint_as_float(s[3 * j]), __uint_as_float(s[3 * j + 1]), __uint_as_float(s[3 * j + 2]));
                }
#pragma unroll
                for (int k = 12; k < 124; k += 8) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        mx[j] = max3(mx[j], __uint_as_float(s[k + 2 * j]), __uint_as_float(s[k + 2 * j + 1]));
                    }
                }
                mx[0] = max3(mx[0], __uint_as_float(s[124]), __uint_as_float(s[125]));
                mx[1] = max3(mx[1], __uint_as_float(s[126]), __uint_as_float(s[127]));
                const float mxx = max3(max3(mx[0], mx[1], mx[2]), mx[3], mx[3]);
                const bool bad  = !(mxx < INFINITY);                           // a NaN or an infinity: the row comes out as NaN
                // Raise the reference when the maximum has grown by more than the threshold, from "no key seen" at any number, and to 0 for a bad row.
                const bool raise = mxx != -INFINITY && !((mxx - m) * c <= kRescaleThreshold);
                if (__any_sync(0xffffffffu, raise)) {
                    const float f = raise ? (bad ? 1.0f : ex2_approx((m - mxx) * c)) : 1.0f;
                    if (raise) {
                        l = bad ? __uint_as_float(0x7fc00000u) : l * f;
                        m = bad ? 0.0f : mxx;
                    }
                    if (s_i > 0) {
                        // S of this step was issued behind the previous step's P V, so the accumulator is at rest; the next P V
                        // waits for this step's P
#pragma unroll
                        for (int cc = 0; cc < D / 16; ++cc) {                  // rare path: small pieces keep the registers free
                            uint32_t o[16];
                            tmem_ld_32x16(o_addr + cc * 16, o);
                            tmem_ld_wait();
#pragma unroll
                            for (int k = 0; k < 16; ++k) {
                                o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
                            }
                            tmem_st_32x16(o_addr + cc * 16, o);
                        }
                        tmem_st_wait();
                    }
                }
                const float2 c2   = make_float2(c, c);
                const float  nmc  = m == -INFINITY ? 0.0f : -m * c;            // no key seen: every weight is exp2(-inf)
                const float2 nmc2 = make_float2(nmc, nmc);
                float2 sum_a = make_float2(0.0f, 0.0f), sum_b = make_float2(0.0f, 0.0f);
#pragma unroll
                for (int cc = 0; cc < 4; ++cc) {
                    uint32_t w[16];
#pragma unroll
                    for (int k = 0; k < 16; ++k) {
                        const float2 x = fma_f32x2(make_float2(__uint_as_float(s[cc * 32 + 2 * k]), __uint_as_float(s[cc * 32 + 2 * k + 1])), c2, nmc2);
                        const bool   poly = (k + 1) * kPolyPairs / 16 != k * kPolyPairs / 16;
                        const float2 e = poly ? ex2_poly(x) : make_float2(ex2_approx(x.x), ex2_approx(x.y));
                        if (k & 1) {
                            sum_b = add_f32x2(sum_b, e);
                        } else {
                            sum_a = add_f32x2(sum_a, e);
                        }
                        w[k] = Pair<T>::from_f32(e.x, e.y);
                    }
                    // P over the start of S: columns [16 cc, 16 cc + 16) hold keys [32 cc, 32 cc + 32)
                    tmem_st_32x16(s_addr + (uint32_t)(cc * 16), w);
                    if (cc & 1) {
                        tmem_st_wait();
                        tc_fence_before_sync();
                        __syncwarp();
                        if (lane == 0) {
                            mbar_arrive(bars + 8u * (uint32_t)(S::kPHalf + (cc >> 1)));
                        }
                    }
                }
                const float2 sum = add_f32x2(sum_a, sum_b);
                l += sum.x + sum.y;
            }
            if (!ok) {
                break;
            }
            if (!(ok = wait(bars + 8u * S::kOFull, (uint32_t)(done & 1), 0x8320u))) {
                break;
            }
            ++done;
            tc_fence_after_sync();
            // a row that saw no key, or does not exist: zeros (its length is read here, as one more number kept through the steps cost up to 0.4 us a call)
            const bool  none  = m == -INFINITY || (p.q_lens != nullptr && row >= query_count(p, it.b));
            const float inv_l = 1.0f / l;
#pragma unroll
            for (int cc = 0; cc < D / 32; ++cc) {
                uint32_t o[32];
                tmem_ld_32x32(o_addr + cc * 32, o);
                tmem_ld_wait();
#pragma unroll
                for (int k = 0; k < 16; ++k) {
                    const float2 x = mul_f32x2(make_float2(__uint_as_float(o[2 * k]), __uint_as_float(o[2 * k + 1])), make_float2(inv_l, inv_l));
                    w[cc * 16 + k] = none ? 0u : Pair<T>::from_f32(x.x, x.y);
                }
            }
            tc_fence_before_sync();   // the next item's P lets the issuer overwrite it
            store();
        }
    }

    tc_fence_before_sync();
    __syncthreads();
    if (warp == kRole0 + 1) {
        tc_fence_after_sync();
        tmem_dealloc(tmem_base, 512);
    }
}

// [batch, heads, tokens, D] with any steps, boxes of `rows` tokens x 64 columns.  A dimension that does not move is one of size one.
int make_map(CUtensorMap* map, const void* base, const Steps& s, int batch, int heads, int tokens, int dim, int rows)
{
    static EncodeTiledFnSparse encode = nullptr;
    if (encode == nullptr) {
        void*                           fp = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fp, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) {
            return LYRAQ_ERR_CUDA;
        }
        encode = reinterpret_cast<EncodeTiledFnSparse>(fp);
    }
    const cuuint64_t n[3] = {(cuuint64_t)tokens, (cuuint64_t)heads, (cuuint64_t)(s.batch == 0 ? 1 : batch)};
    const long long  e[3] = {s.token, s.head, s.batch};
    cuuint64_t       dims[4] = {(cuuint64_t)dim, n[0], n[1], n[2]}, strides[3];
    for (int i = 0; i < 3; ++i) {
        strides[i] = n[i] > 1 ? (cuuint64_t)e[i] * 2 : (cuuint64_t)dim * 2;
    }
    const cuuint32_t box[4] = {64, (cuuint32_t)rows, 1, 1}, estr[4] = {1, 1, 1, 1};
    if (encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 4, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS) {
        record_cuda_error(cudaErrorInvalidValue, "cuTensorMapEncodeTiled refused a tensor map of q, k or v");
        return LYRAQ_ERR_CUDA;
    }
    return LYRAQ_OK;
}

template<typename T, int D> static int launch(Params p, int sms, cudaStream_t stream)
{
    using S = Smem<D>;
    CUtensorMap tq, tk, tv;
    int         st = make_map(&tq, p.q, p.qs, p.batch, p.q_heads, p.queries, D, kTile);
    tk = tv = tq;
    if (st == LYRAQ_OK && p.count > 0) {
        st = make_map(&tk, p.k, p.ks, p.batch, p.k_heads, p.keys, D, kHalf);
    }
    if (st == LYRAQ_OK && p.count > 0) {
        st = make_map(&tv, p.v, p.vs, p.batch, p.k_heads, p.keys, D, kHalf);
    }
    static bool smem_raised[64] = {};
    if (st == LYRAQ_OK) {
        st = raise_dynamic_smem_once(sparse_attention_kernel<T, D>, (int)S::kTotal, smem_raised, "cudaFuncSetAttribute(sparse_attention_kernel)");
    }
    if (st != LYRAQ_OK) {
        return st;
    }
    const unsigned grid = (unsigned)(p.items < sms ? p.items : sms);
    return cuda_status(launch_kernel(sparse_attention_kernel<T, D>, grid, (unsigned)kThreads, (size_t)S::kTotal, stream, 1u, tq, tk, tv, p),
                       "cudaLaunchKernelEx(sparse_attention_kernel)");
}

// Test hook (lyraq_debug_sparse_attention_wait_test): producers that never signal and a short wait limit.
static int                g_skip_loads    = 0;
static unsigned long long g_wait_limit_ns = kWaitLimitNs;

}  // namespace sattn
}  // namespace lyraq

using namespace lyraq;

extern "C" {

int lyraq_debug_sparse_attention_wait_test(int skip_loads, unsigned int wait_limit_ms)
{
    sattn::g_skip_loads    = skip_loads ? 1 : 0;
    sattn::g_wait_limit_ns = wait_limit_ms == 0 ? sm100::kWaitLimitNs : (unsigned long long)wait_limit_ms * 1000000ull;
    return LYRAQ_OK;
}

int lyraq_sparse_attention(const lyraq_sparse_attention_t* a, void* stream)
{
    if (a == nullptr || a->q_heads < 0 || a->k_heads < 0 || a->lists < 0 || a->head_dim < 0 || a->count < 0 || !(a->softmax_scale > 0.0f) ||
        !(a->softmax_scale * 1.4426950408889634f < INFINITY)) {
        return LYRAQ_ERR_INVALID_ARG;
    }
    if ((a->dtype != LYRAQ_F16 && a->dtype != LYRAQ_BF16) || (a->head_dim != 64 && a->head_dim != 128) || (a->block != 64 && a->block != 128)) {
        return LYRAQ_ERR_UNSUPPORTED;
    }
    if (a->batch == 0 || a->queries == 0 || a->q_heads == 0) {
        return LYRAQ_OK;
    }
    if (a->k_heads == 0 || a->q_heads % a->k_heads != 0 || (a->lists != a->q_heads && a->lists != a->k_heads)) {
        return LYRAQ_ERR_INVALID_ARG;
    }
    const size_t q_blocks = (a->queries + sattn::kQueryBlock - 1) / sattn::kQueryBlock, rows = a->batch * (size_t)a->lists * q_blocks;
    if (a->keys > (size_t)sattn::kMaxKeys || a->queries > (size_t)sattn::kMaxKeys || a->batch > 0xffffu || a->q_heads > 0xffff ||
        a->batch * (size_t)a->q_heads * q_blocks > 0x3fffffffu) {
        return LYRAQ_ERR_UNSUPPORTED;
    }
    const size_t steps[12] = {a->q_batch, a->q_token, a->q_head, a->k_batch, a->k_token, a->k_head, a->v_batch, a->v_token, a->v_head, a->o_batch, a->o_token, a->o_head};
    for (size_t s : steps) {
        if ((s & 7u) != 0 || s >= (size_t)1 << 38) {
            return LYRAQ_ERR_INVALID_ARG;
        }
    }
    const bool none = a->keys == 0 || a->count == 0;
    if (a->q == nullptr || a->out == nullptr || !aligned16(a->q) || !aligned16(a->k) || !aligned16(a->v) || !aligned16(a->out) ||
        (!none && (a->k == nullptr || a->v == nullptr || a->index == nullptr)) || a->counts == nullptr ||
        ((reinterpret_cast<uintptr_t>(a->index) | reinterpret_cast<uintptr_t>(a->counts) | reinterpret_cast<uintptr_t>(a->k_lens) |
          reinterpret_cast<uintptr_t>(a->q_lens) | reinterpret_cast<uintptr_t>(a->q_start)) & 3u) != 0) {
        return LYRAQ_ERR_INVALID_ARG;
    }
    // a step of 0 repeats a sequence; tokens and heads have places of their own
    if ((a->queries > 1 && a->q_token == 0) || (a->q_heads > 1 && a->q_head == 0) || (a->keys > 1 && (a->k_token == 0 || a->v_token == 0)) ||
        (a->k_heads > 1 && (a->k_head == 0 || a->v_head == 0))) {
        return LYRAQ_ERR_UNSUPPORTED;
    }
    if ((a->batch > 1 && a->o_batch == 0) || (a->queries > 1 && a->o_token == 0) || (a->q_heads > 1 && a->o_head == 0)) {
        return LYRAQ_ERR_INVALID_ARG;      // results in one place
    }
    const size_t dim = (size_t)a->head_dim;
    auto view = [&](const void* p, size_t sb, size_t n, size_t st, int heads, size_t sh) { return view_of(p, 2, a->batch, sb, n, st, (size_t)heads, sh, dim); };
    const View out = view(a->out, a->o_batch, a->queries, a->o_token, a->q_heads, a->o_head);
    if (result_clashes(out, nullptr,
                       {view(a->q, a->q_batch, a->queries, a->q_token, a->q_heads, a->q_head), view(a->k, a->k_batch, a->keys, a->k_token, a->k_heads, a->k_head),
                        view(a->v, a->v_batch, a->keys, a->v_token, a->k_heads, a->v_head), view_of(a->index, rows * (size_t)a->count * 4),
                        view_of(a->counts, rows * 4), view_of(a->k_lens, a->batch * 4), view_of(a->q_lens, a->batch * 4), view_of(a->q_start, a->batch * 4)})) {
        return LYRAQ_ERR_INVALID_ARG;
    }
    sattn::Params p{};
    p.q   = a->q;
    p.k   = a->k;
    p.v   = a->v;
    p.out = a->out;
    auto pick = [&](size_t n, size_t s) { return n > 1 ? (long long)s : 0ll; };
    p.qs  = {pick(a->batch, a->q_batch), pick(a->queries, a->q_token), pick((size_t)a->q_heads, a->q_head)};
    p.ks  = {pick(a->batch, a->k_batch), pick(a->keys, a->k_token), pick((size_t)a->k_heads, a->k_head)};
    p.vs  = {pick(a->batch, a->v_batch), pick(a->keys, a->v_token), pick((size_t)a->k_heads, a->v_head)};
    p.os  = {(long long)a->o_batch, (long long)a->o_token, (long long)a->o_head};
    p.index      = a->index;
    p.counts     = a->counts;
    p.k_lens     = a->k_lens;
    p.q_lens     = a->q_lens;
    p.q_start    = a->q_start;
    p.batch      = (int)a->batch;
    p.queries    = (int)a->queries;
    p.keys       = (int)a->keys;
    p.q_heads    = a->q_heads;
    p.k_heads    = a->k_heads;
    p.lists      = a->lists;
    p.q_blocks   = (int)q_blocks;
    p.block      = a->block;
    p.count      = none ? 0 : a->count;   // no list is read and no key: rows of zeros
    p.causal     = a->causal;
    p.items      = (int)(a->batch * (size_t)a->q_heads * q_blocks);
    p.fixed      = (p.qs.batch == 0 ? 1 : 0) | (p.ks.batch == 0 ? 2 : 0) | (p.vs.batch == 0 ? 4 : 0);
    p.scale_log2 = a->softmax_scale * 1.4426950408889634f;
    p.status     = status_word_ptr();
    p.wait_limit_ns = sattn::g_wait_limit_ns;
    p.skip_loads    = sattn::g_skip_loads;
    const int sms = device_sm_count();
    if (p.status == nullptr || sms <= 0) {
        return LYRAQ_ERR_CUDA;
    }
    cudaStream_t s = (cudaStream_t)stream;
    if (sattn::few_rows(p)) {
        return sattn::launch_rows(p, a->dtype, a->head_dim, s);
    }
    if (a->dtype == LYRAQ_BF16) {
        return dim == 128 ? sattn::launch<__nv_bfloat16, 128>(p, sms, s) : sattn::launch<__nv_bfloat16, 64>(p, sms, s);
    }
    return dim == 128 ? sattn::launch<__half, 128>(p, sms, s) : sattn::launch<__half, 64>(p, sms, s);
}

}  // extern "C"
