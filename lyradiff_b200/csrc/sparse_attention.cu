// Block-sparse attention forward: out[b, i, h, :] = softmax over the keys of the blocks listed for query block i / 128 of (q k^T scale) v.
//
// The kernel of attention.cu with lists: a CTA runs two query tiles of 128 rows, which share the tensor pipe and the exponent unit but nothing else,
// since each has its own list.  So each has its own producer, issuer and part of shared memory, and takes its own query blocks in turn:
//   warps 8, 10  TMA producers of tile 0, 1: per query block Q, then K and V of each step of 128 keys (two listed blocks of 64, or one of 128), as
//                boxes of 64 keys x 64 columns.  One buffer for K (free as soon as the scores are there, needed when P V of the step is under way) and
//                a ring of half steps for V.
//   warps 9, 11  MMA issuers: S = Q K^T (M 128, N 128), O += P V, P read from tensor memory, in two halves of 64 keys
//   warps 0-3    softmax and epilogue of tile 0, warps 4-7 of tile 1: a thread owns one query row.  Keys of a half step that a row does not see are a
//                tail of it (beyond the keys, or behind the row's place), so a mask is one number.
// K V of a step are 64 KB for one tile where the dense kernel reads them once for two: 43 bytes a clock and SM out of L2 at its pace.
// V rows beyond a sequence's keys may hold anything: the softmax warps clear them in shared memory, since 0 * NaN is NaN.
// Every wait is bounded; on a timeout the role records it in the status word, raises the block's abort flag and all roles leave; tensor
// memory is freed at the common exit.
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
constexpr int kRole0   = 8;                         // warps 8 .. 11
// registers: 384 threads x 168 at launch = 64512 = 256 x 216 + 128 x 72
constexpr int kSoftmaxRegs = 216;
constexpr int kOtherRegs   = 72;
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
    static constexpr int kBars    = 2 + 2 * kKSlots + 2 * kVSlots + 4;   // of a tile
    static constexpr int kBarOffset = kTiles * kPerTile;
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

// The work of one tile: query block `qb` of head `h` of sequence `b`, and its list.
struct Item {
    int        qb, h, b;
    const int* list;
    int        entries;
};

template<typename T, int D>
__global__ void __launch_bounds__(kThreads, 1)
sparse_attention_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
                        const __grid_constant__ Params p)
{
    using S = Smem<D>;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t*       gen_base  = smem_raw + (smem_base - smem_u32(smem_raw));
    auto bar       = [&](int t, int i) { return smem_base + S::kBarOffset + 8u * (uint32_t)(t * S::kBars + i); };
    auto q_full    = [&](int t) { return bar(t, 0); };
    auto q_empty   = [&](int t) { return bar(t, 1); };
    auto s_full    = [&](int t) { return bar(t, 2); };    // scores of a step
    auto p_first   = [&](int t) { return bar(t, 3); };    // P of the step's keys 0 .. 63 is in tensor memory
    auto p_second  = [&](int t) { return bar(t, 4); };    // ... and of keys 64 .. 127
    auto o_full    = [&](int t) { return bar(t, 5); };    // accumulator of a query block is final
    auto k_full    = [&](int t, int s) { return bar(t, 6 + s); };
    auto k_empty   = [&](int t, int s) { return bar(t, 6 + S::kKSlots + s); };
    auto v_full    = [&](int t, int s) { return bar(t, 6 + 2 * S::kKSlots + s); };
    auto v_empty   = [&](int t, int s) { return bar(t, 6 + 2 * S::kKSlots + S::kVSlots + s); };
    uint32_t*     tmem_slot  = reinterpret_cast<uint32_t*>(gen_base + S::kBarOffset + 8 * S::kBars * kTiles);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

    const int warp = warp_index();
    const int lane = threadIdx.x & 31;

    grid_launch_dependents();
    if (threadIdx.x == 0) {
        for (int t = 0; t < kTiles; ++t) {
            for (int i = 0; i < S::kBars; ++i) {
                mbar_init(bar(t, i), i == 3 || i == 4 ? 4u : 1u);   // P comes from four warps
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
    // tile 0 of every CTA first: few items spread over all SMs
    auto item_of = [&](int i) {
        Item it;
        it.qb      = i % p.q_blocks;
        it.h       = i / p.q_blocks % p.q_heads;
        it.b       = i / (p.q_blocks * p.q_heads);
        const size_t row = ((size_t)it.b * (size_t)p.lists + (size_t)(it.h / (p.q_heads / p.lists))) * (size_t)p.q_blocks + (size_t)it.qb;
        it.list    = p.index + row * (size_t)p.count;
        it.entries = min(max(load_int(p.counts + row), 0), p.count);
        return it;
    };
    auto steps_of = [&](const Item& it) { return p.block == kTile ? it.entries : (it.entries + 1) / 2; };
    // first key of half s of step i, or `keys` where there is none: a box there is filled with zeros and its keys are masked
    auto key_of = [&](const Item& it, int i, int s) {
        const int e = p.block == kTile ? i : 2 * i + s;
        if (e >= it.entries) {
            return p.keys;
        }
        const int j = load_int(it.list + e);
        return j >= 0 && j <= (p.keys - 1) / p.block ? min(j * p.block + (p.block == kTile ? s * kHalf : 0), p.keys) : p.keys;
    };
    const int t     = warp < kRole0 ? warp >> 2 : (warp - kRole0) >> 1;
    const int first = (int)blockIdx.x + t * (int)gridDim.x, stride = kTiles * (int)gridDim.x;
    const uint32_t tile_smem = smem_base + (uint32_t)(t * S::kPerTile);

    if (warp >= kRole0) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
        if (((warp - kRole0) & 1) == 0) {
            // -------------------------------------------------------------- TMA producer
            int      k_slot = 0, v_slot = 0, k_issued = 0, v_issued = 0, q_issued = 0;
            uint32_t k_phase = 0, v_phase = 0;
            bool     ok = true;
            auto wait_for = [&](uint32_t b, uint32_t parity, unsigned code) {
                if (!mbar_wait_warp(b, parity, abort_flag, p.wait_limit_ns)) {
                    give_up(code);
                    ok = false;
                }
                return ok;
            };
            for (int i = first; ok && i < p.items && p.skip_loads == 0; i += stride) {
                const Item it    = item_of(i);
                const int  steps = steps_of(it), kh = it.h / (p.q_heads / p.k_heads);
                if (steps == 0) {
                    continue;
                }
                if (!wait_for(q_empty(t), (uint32_t)(q_issued & 1) ^ 1u, 0x8110u)) {
                    break;
                }
                if (elect_one()) {
                    mbar_arrive_expect_tx(q_full(t), (uint32_t)S::kQBytes);
#pragma unroll
                    for (int c = 0; c < S::kPanels; ++c) {
                        tma_load_4d(tile_smem + c * S::kPanelQ, &tmap_q, q_full(t), c * 64, it.qb * kTile, it.h, (p.fixed & 1) != 0 ? 0 : it.b);
                    }
                }
                ++q_issued;
                int key[2] = {key_of(it, 0, 0), key_of(it, 0, 1)};
                for (int s = 0; ok && s < steps; ++s) {
                    int next[2] = {p.keys, p.keys};
                    if (s + 1 < steps) {      // on their way while the buffers are waited for
                        next[0] = key_of(it, s + 1, 0);
                        next[1] = key_of(it, s + 1, 1);
                    }
                    if (!wait_for(k_empty(t, k_slot), k_phase ^ 1u, 0x8100u)) {
                        break;
                    }
                    if (elect_one()) {
                        const uint32_t dst = tile_smem + S::kKOffset + k_slot * S::kKBytes;
                        mbar_arrive_expect_tx(k_full(t, k_slot), (uint32_t)S::kKBytes);
#pragma unroll
                        for (int c = 0; c < S::kPanels; ++c) {
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                tma_load_4d(dst + c * S::kPanelQ + h * S::kPanelV, &tmap_k, k_full(t, k_slot), c * 64, key[h], kh, (p.fixed & 2) != 0 ? 0 : it.b);
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
                        if (!ok || !wait_for(v_empty(t, v_slot), v_phase ^ 1u, 0x8120u)) {
                            break;
                        }
                        if (elect_one()) {
                            const uint32_t dst = tile_smem + S::kVOffset + v_slot * S::kVBytes;
                            mbar_arrive_expect_tx(v_full(t, v_slot), (uint32_t)S::kVBytes);
#pragma unroll
                            for (int c = 0; c < S::kPanels; ++c) {
                                tma_load_4d(dst + c * S::kPanelV, &tmap_v, v_full(t, v_slot), c * 64, key[h], kh, (p.fixed & 4) != 0 ? 0 : it.b);
                            }
                        }
                        ++v_issued;
                        if (++v_slot == S::kVSlots) {
                            v_slot = 0;
                            v_phase ^= 1u;
                        }
                    }
                    key[0] = next[0];
                    key[1] = next[1];
                }
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
            for (int i = 0; i < S::kKSlots && i < k_issued; ++i) {
                if (k_slot == 0) {
                    k_slot = S::kKSlots;
                    k_phase ^= 1u;
                }
                --k_slot;
                settle(k_full(t, k_slot), k_phase, 0x8400u);
            }
            for (int i = 0; i < S::kVSlots && i < v_issued; ++i) {
                if (v_slot == 0) {
                    v_slot = S::kVSlots;
                    v_phase ^= 1u;
                }
                --v_slot;
                settle(v_full(t, v_slot), v_phase, 0x8420u);
            }
            if (q_issued > 0) {
                settle(q_full(t), (uint32_t)((q_issued - 1) & 1), 0x8410u);
            }
        } else {
            // -------------------------------------------------------------- MMA issuer
            constexpr uint32_t kAb = TypeTag<T>::value == LYRAQ_BF16 ? 1u : 0u;
            constexpr uint32_t idesc_qk = umma_idesc(1u, kAb, 128, kTile);
            constexpr uint32_t idesc_pv = umma_idesc(1u, kAb, 128, D) | kIdescBMajorMN;
            const uint32_t s_acc = tmem_base + (uint32_t)(t * 128), o_acc = tmem_base + (uint32_t)(256 + t * 128);
            int      k_slot = 0, v_slot = 0;
            uint32_t k_phase = 0, v_phase = 0, step = 0, taken = 0;
            bool     ok = true;
            auto wait_for = [&](uint32_t b, uint32_t parity, unsigned code) {
                if (!mbar_wait_warp(b, parity, abort_flag, p.wait_limit_ns)) {
                    give_up(code);
                    ok = false;
                }
                return ok;
            };
            // S = Q K^T with the k tile in k_slot
            auto scores = [&](bool last) {
                if (!wait_for(k_full(t, k_slot), k_phase, 0x8210u)) {
                    return;
                }
                tc_fence_after_sync();
                if (elect_one()) {
                    const uint64_t qdesc = umma_desc_k_sw128(tile_smem);
                    const uint64_t kdesc = umma_desc_k_sw128(tile_smem + S::kKOffset + k_slot * S::kKBytes);
#pragma unroll
                    for (int ks = 0; ks < D / 16; ++ks) {
                        const uint64_t off = (uint64_t)(((ks >> 2) * S::kPanelQ + (ks & 3) * 32) >> 4);
                        mma_f16(s_acc, qdesc + off, kdesc + off, idesc_qk, ks > 0 ? 1u : 0u);
                    }
                    tc_commit(s_full(t));
                    tc_commit(k_empty(t, k_slot));
                    if (last) {
                        tc_commit(q_empty(t));
                    }
                }
                if (++k_slot == S::kKSlots) {
                    k_slot = 0;
                    k_phase ^= 1u;
                }
            };
            for (int i = first; ok && i < p.items; i += stride) {
                const int steps = steps_of(item_of(i));
                if (steps == 0) {
                    continue;
                }
                if (!wait_for(q_full(t), taken & 1u, 0x8200u)) {
                    break;
                }
                ++taken;
                scores(steps == 1);
#pragma unroll 1
                for (int s = 0; ok && s < steps; ++s, ++step) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        if (!ok || !wait_for(v_full(t, v_slot), v_phase, 0x8230u) || !wait_for(h == 0 ? p_first(t) : p_second(t), step & 1u, 0x8240u)) {
                            break;
                        }
                        tc_fence_after_sync();
                        if (elect_one()) {
                            const uint64_t vdesc = umma_desc_mn_sw128(tile_smem + S::kVOffset + v_slot * S::kVBytes, (uint32_t)S::kPanelV);
#pragma unroll
                            for (int k4 = 0; k4 < 4; ++k4) {   // 16 keys each: 8 columns of P, 2048 bytes of v
                                mma_f16_ts(o_acc, s_acc + (uint32_t)((4 * h + k4) * 8), vdesc + (uint64_t)(k4 * 128), idesc_pv, s > 0 || h > 0 || k4 > 0 ? 1u : 0u);
                            }
                            tc_commit(v_empty(t, v_slot));
                            if (h == 1 && s + 1 == steps) {
                                tc_commit(o_full(t));
                            }
                        }
                        if (++v_slot == S::kVSlots) {
                            v_slot = 0;
                            v_phase ^= 1u;
                        }
                    }
                    if (ok && s + 1 < steps) {
                        scores(s + 2 == steps);   // over P, which the MMAs before read, in order
                    }
                }
            }
        }
    } else {
        // ------------------------------------------------------------------ softmax and epilogue, one thread per query row
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
        const int      quadrant = warp & 3;                                    // tensor-memory lane quadrant of this warp
        const int      r        = quadrant * 32 + lane;                        // row of the tile
        const uint32_t lanes    = tmem_base + ((uint32_t)(quadrant * 32) << 16);
        const uint32_t s_addr   = lanes + (uint32_t)(t * 128);
        const uint32_t o_addr   = lanes + (uint32_t)(256 + t * 128);
        const float    c        = p.scale_log2;
        bool           ok       = true;
        uint32_t       g        = 0, done = 0;                                 // steps and query blocks of this tile
        for (int i = first; ok && i < p.items; i += stride) {
            const Item it    = item_of(i);
            const int  steps = steps_of(it);
            const int  row   = it.qb * kTile + r;
            const int  len   = key_count(p, it.b);
            // the last key this row sees
            const int  place = p.causal ? (int)min((long long)first_place(p, it.b) + row, (long long)p.keys) : p.keys;
            float m = -INFINITY;                                               // reference maximum of this row's raw scores; -inf: no key seen
            float l = 0.0f;                                                    // sum of exp2((s - m) c)
            int   key[2] = {p.keys, p.keys};
            if (steps > 0) {
                key[0] = key_of(it, 0, 0);
                key[1] = key_of(it, 0, 1);
            }
#pragma unroll 1
            for (int s_i = 0; s_i < steps; ++s_i, ++g) {
                // keys [0, see[h]) of a half are this row's, of which [0, full[h]) exist
                int see[2], exist[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    exist[h] = min(max(len - key[h], 0), kHalf);
                    see[h]   = min(max(place - key[h] + 1, 0), exist[h]);
                }
                const bool clear[2] = {exist[0] < kHalf && key[0] + exist[0] < p.keys, exist[1] < kHalf && key[1] + exist[1] < p.keys};
                if (s_i + 1 < steps) {
                    key[0] = key_of(it, s_i + 1, 0);
                    key[1] = key_of(it, s_i + 1, 1);
                }
                if (!mbar_wait_warp(s_full(t), g & 1u, abort_flag, p.wait_limit_ns)) {
                    give_up(0x8300u | (unsigned)t);
                    ok = false;
                    break;
                }
                tc_fence_after_sync();
                uint32_t s[128];
#pragma unroll
                for (int cc = 0; cc < 4; ++cc) {
                    tmem_ld_32x32(s_addr + cc * 32, s + cc * 32);
                }
                tmem_ld_wait();
                if (__any_sync(0xffffffffu, see[0] < kHalf || see[1] < kHalf)) {
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
                // V rows beyond the sequence's keys: cleared before the issuer hears of P
                if (clear[0] || clear[1]) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        if (clear[h]) {
                            const uint32_t n = 2u * g + (uint32_t)h, slot = n % (uint32_t)S::kVSlots;
                            if (ok && !mbar_wait_warp(v_full(t, (int)slot), n / (uint32_t)S::kVSlots & 1u, abort_flag, p.wait_limit_ns)) {
                                give_up(0x8310u | (unsigned)t);
                                ok = false;
                            }
                            // two threads a row, which is 128 bytes in every panel
                            const int key_row = r >> 1;
                            if (ok && key_row >= exist[h]) {
                                uint8_t* at = gen_base + t * S::kPerTile + S::kVOffset + (int)slot * S::kVBytes + key_row * 128 + (r & 1) * 64;
#pragma unroll
                                for (int cc = 0; cc < S::kPanels; ++cc) {
#pragma unroll
                                    for (int e = 0; e < 4; ++e) {
                                        *reinterpret_cast<uint4*>(at + cc * S::kPanelV + e * 16) = make_uint4(0u, 0u, 0u, 0u);
                                    }
                                }
                            }
                        }
                    }
                    if (!ok) {
                        break;
                    }
                    fence_proxy_async_smem();
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
                            mbar_arrive(cc == 1 ? p_first(t) : p_second(t));
                        }
                    }
                }
                const float2 sum = add_f32x2(sum_a, sum_b);
                l += sum.x + sum.y;
            }
            if (!ok) {
                break;
            }
            // O / l, rounded to T; a row that saw no key: zeros
            const bool none  = m == -INFINITY;
            const float inv_l = 1.0f / l;
            uint32_t w[D / 2];
#pragma unroll
            for (int k = 0; k < D / 2; ++k) {
                w[k] = 0u;
            }
            if (steps > 0) {
                if (!mbar_wait_warp(o_full(t), done & 1u, abort_flag, p.wait_limit_ns)) {
                    give_up(0x8320u | (unsigned)t);
                    ok = false;
                    break;
                }
                ++done;
                tc_fence_after_sync();
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
                tc_fence_before_sync();
            }
            if (row < p.queries) {
                T* dst = reinterpret_cast<T*>(p.out) + (long long)it.b * p.os.batch + (long long)row * p.os.token + (long long)it.h * p.os.head;
#pragma unroll
                for (int k = 0; k < D / 8; ++k) {
                    reinterpret_cast<uint4*>(dst)[k] = make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
                }
            }
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
static int make_map(CUtensorMap* map, const void* base, const Steps& s, int batch, int heads, int tokens, int dim, int rows)
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
        !(a->softmax_scale < INFINITY)) {
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
          reinterpret_cast<uintptr_t>(a->q_start)) & 3u) != 0) {
        return LYRAQ_ERR_INVALID_ARG;
    }
    // a step of 0 repeats a sequence; tokens and heads have places of their own
    if ((a->queries > 1 && a->q_token == 0) || (a->q_heads > 1 && a->q_head == 0) || (a->keys > 1 && (a->k_token == 0 || a->v_token == 0)) ||
        (a->k_heads > 1 && (a->k_head == 0 || a->v_head == 0))) {
        return LYRAQ_ERR_UNSUPPORTED;
    }
    const size_t dim = (size_t)a->head_dim;
    auto view = [&](const void* p, size_t sb, size_t n, size_t st, int heads, size_t sh) { return view_of(p, 2, a->batch, sb, n, st, (size_t)heads, sh, dim); };
    const View out = view(a->out, a->o_batch, a->queries, a->o_token, a->q_heads, a->o_head);
    if (result_clashes(out, nullptr,
                       {view(a->q, a->q_batch, a->queries, a->q_token, a->q_heads, a->q_head), view(a->k, a->k_batch, a->keys, a->k_token, a->k_heads, a->k_head),
                        view(a->v, a->v_batch, a->keys, a->v_token, a->k_heads, a->v_head), view_of(a->index, rows * (size_t)a->count * 4),
                        view_of(a->counts, rows * 4), view_of(a->k_lens, a->batch * 4), view_of(a->q_start, a->batch * 4)})) {
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
    if (a->dtype == LYRAQ_BF16) {
        return dim == 128 ? sattn::launch<__nv_bfloat16, 128>(p, sms, s) : sattn::launch<__nv_bfloat16, 64>(p, sms, s);
    }
    return dim == 128 ? sattn::launch<__half, 128>(p, sms, s) : sattn::launch<__half, 64>(p, sms, s);
}

}  // extern "C"
