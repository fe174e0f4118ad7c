// Block-sparse attention of few queries over a cache: at most 16 rows share a list (its query heads x the queries), each new token of a sequence being
// one row a head.
//
// What bounds it is the gather: the listed keys and values are read once (134 MB for eight sequences, eight key heads and 64 blocks of 64 tokens of
// 128: 20.6 us of HBM), the products are small enough for mma.sync (the rows on the M side, padded to 16).  A cluster of CTAs takes one list, half
// block by half block in turn (64 keys), as many CTAs as let all SMs read; their sums meet through distributed shared memory, in rank order.
//
//   warp 4     TMA producer: K and V of a half block (64 keys x 64 columns a box) into a ring of stages
//   warps 0-3  16 keys of each stage: S = Q K^T, running maximum and sum, O += P V; keys and values as they lie in shared memory by ldmatrix
// V rows beyond a sequence's keys may hold anything: their registers are cleared, since 0 * NaN is NaN.
// Weights are rounded to the tensors' type, as mma.sync asks for and as the kernel of many queries does; their sum is of the numbers before.
// All waits are bounded.  A timeout sets the status word and the abort flag of every CTA of the cluster, and none of them stores anything.
#include "sparse_attention.cuh"
#include "sm100_ptx.cuh"

namespace lyraq {

using namespace sm100;

int device_sm_count();  // gemm_dense.cu

namespace sattn {

using attn::ex2_approx;

int make_map(CUtensorMap* map, const void* base, const Steps& s, int batch, int heads, int tokens, int dim, int rows);   // sparse_attention.cu

namespace rows {

constexpr int kKeys    = 64;     // of a stage
constexpr int kWarps   = 4;
constexpr int kThreads = (kWarps + 1) * 32;
constexpr int kMaxRows = 16;
constexpr int kPanel   = kKeys * 128;

template<int D> struct Smem {
    static constexpr int kPanels  = D / 64;
    static constexpr int kTile    = kPanels * kPanel;
    static constexpr int kStage   = 2 * kTile;                     // K, V
    static constexpr int kStages  = D == 128 ? 3 : 6;
    static constexpr int kQPitch  = D * 2 + 16;
    static constexpr int kQOffset = kStages * kStage;
    static constexpr int kMlOffset = kQOffset + kMaxRows * kQPitch;        // maxima and sums: [warp][2][row], then of the CTA [2][row]
    static constexpr int kKeyOffset = kMlOffset + (kWarps + 1) * 2 * kMaxRows * 4;
    static constexpr int kBarOffset = kKeyOffset + 8 * 4;
    static constexpr int kTotal   = kBarOffset + 2 * kStages * 8 + 16 + 1024;
    // partial sums lie over the ring once it is empty: [warp][row][D], pitch D + 4; then of the CTA [row][D] in the place of warp 0's
    static constexpr int kPitch   = D + 4;
    static_assert(kWarps * kMaxRows * kPitch * 4 <= kStages * kStage && kStages <= 8 && kTotal <= 115000, "two CTAs share an SM");
};

__device__ __forceinline__ void ldmatrix4(uint32_t* r, uint32_t addr)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t* r, uint32_t addr)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
template<typename T> __device__ __forceinline__ void mma16(float* c, const uint32_t* a, uint32_t b0, uint32_t b1)
{
    if constexpr (TypeTag<T>::value == LYRAQ_BF16) {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    } else {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
}
__device__ __forceinline__ void tma_load_4d(uint32_t smem_dst, const CUtensorMap* m, uint32_t bar, int x, int y, int z, int w)
{
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
        ::"r"(smem_dst), "l"(m), "r"(bar), "r"(x), "r"(y), "r"(z), "r"(w)
        : "memory");
}
__device__ __forceinline__ float ld_cluster_f32(uint32_t addr)
{
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ float4 ld_cluster_f32x4(uint32_t addr)
{
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void st_cluster_u32(uint32_t cluster_addr, uint32_t v)
{
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(cluster_addr), "r"(v) : "memory");
}

template<typename T, int D>
__global__ void __launch_bounds__(kThreads, 2)
sparse_attention_rows_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v, const __grid_constant__ Params p,
                             const int splits)
{
    using S = Smem<D>;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    // the dynamic shared window starts at the same offset in every CTA of the kernel, so the layout is that of the peers too
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t*       gen_base  = smem_raw + (smem_base - smem_u32(smem_raw));
    const uint32_t bars      = smem_base + S::kBarOffset;
    auto full_bar  = [&](int s) { return bars + 8u * (uint32_t)s; };
    auto empty_bar = [&](int s) { return bars + 8u * (uint32_t)(S::kStages + s); };
    volatile int* abort_flag = reinterpret_cast<volatile int*>(gen_base + S::kBarOffset + 2 * S::kStages * 8);
    volatile int* stage_key  = reinterpret_cast<volatile int*>(gen_base + S::kKeyOffset);

    const int warp = warp_index(), lane = threadIdx.x & 31;
    const int rank = (int)cluster_ctarank();
    const int unit = (int)blockIdx.x / splits, list = unit % p.lists, b = unit / p.lists;
    const int heads = p.q_heads / p.lists, n_rows = heads * p.queries;
    auto give_up = [&](unsigned code) {
        report_timeout(p.status, code);
        for (int r = 0; r < splits; ++r) {
            st_cluster_u32(map_to_cta(smem_u32(const_cast<int*>(abort_flag)), (uint32_t)r), 1u);
        }
    };

    grid_launch_dependents();
    if (threadIdx.x == 0) {
        for (int s = 0; s < S::kStages; ++s) {
            mbar_init(full_bar(s), 1);
            mbar_init(empty_bar(s), kWarps);
        }
        *abort_flag = 0;
        fence_barrier_init();
        prefetch_tensormap(&tmap_k);
        prefetch_tensormap(&tmap_v);
    }
    grid_dependency_wait();
    const int halves_per = p.block / kKeys;
    const int entries    = min(max(load_int(p.counts + unit), 0), p.count);
    const int halves     = entries * halves_per;
    const int len        = key_count(p, b);
    if (warp < kWarps) {
        for (int i = (int)threadIdx.x; i < kMaxRows * (D / 8); i += kWarps * 32) {
            const int r = i / (D / 8), c = i % (D / 8);
            Vec16     v{};
            if (r < n_rows) {
                const int head = list * heads + r / p.queries, qi = r % p.queries;
                v = ld_nc_16(reinterpret_cast<const T*>(p.q) + (long long)b * p.qs.batch + (long long)qi * p.qs.token + (long long)head * p.qs.head + c * 8);
            }
            *reinterpret_cast<Vec16*>(gen_base + S::kQOffset + r * S::kQPitch + c * 16) = v;
        }
    }
    cluster_sync_all();   // barriers are set and every CTA of the cluster runs before a peer reads its shared memory

    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};      // rows lane / 4 and lane / 4 + 8
    float o[D / 8][4];
#pragma unroll
    for (int n = 0; n < D / 8; ++n) {
        o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.0f;
    }
    if (warp == kWarps) {
        // ------------------------------------------------------------------ producer
        const int kh = list / (p.lists / p.k_heads);
        int       issued = 0;
        bool      ok     = p.skip_loads == 0;
        // the first key of a half block, or `keys` for a place outside: zeros there, and masked
        auto key_of = [&](int i) {
            if (i >= halves) {
                return p.keys;
            }
            const int j = load_int(p.index + (size_t)unit * (size_t)p.count + (size_t)(i / halves_per));
            return j >= 0 && j <= (p.keys - 1) / p.block ? min(j * p.block + i % halves_per * kKeys, p.keys) : p.keys;
        };
        int key = key_of(rank);
        for (int i = rank; ok && i < halves; i += splits, ++issued) {
            const int ahead = key_of(i + splits), s = issued % S::kStages;
            if (!mbar_wait_warp(empty_bar(s), (uint32_t)(issued / S::kStages & 1) ^ 1u, abort_flag, p.wait_limit_ns)) {
                if (lane == 0) {
                    give_up(0x9100u | (unsigned)s);
                }
                ok = false;
                break;
            }
            if (elect_one()) {
                const uint32_t dst = smem_base + (uint32_t)(s * S::kStage);
                stage_key[s]       = key;
                mbar_arrive_expect_tx(full_bar(s), (uint32_t)S::kStage);
#pragma unroll
                for (int c = 0; c < S::kPanels; ++c) {
                    tma_load_4d(dst + c * kPanel, &tmap_k, full_bar(s), c * 64, key, kh, (p.fixed & 2) != 0 ? 0 : b);
                    tma_load_4d(dst + S::kTile + c * kPanel, &tmap_v, full_bar(s), c * 64, key, kh, (p.fixed & 4) != 0 ? 0 : b);
                }
            }
            key = ahead;
        }
        // no copy may be in flight when the block leaves
        for (int n = 0; n < S::kStages && n < issued; ++n) {
            const int      at = issued - 1 - n;
            const uint64_t t0 = global_timer_ns();
            while (!mbar_try_wait(full_bar(at % S::kStages), (uint32_t)(at / S::kStages & 1))) {
                if (global_timer_ns() - t0 > p.wait_limit_ns) {
                    report_timeout(p.status, 0x9400u);
                    break;
                }
            }
        }
    } else {
        // ------------------------------------------------------------------ 16 keys of every stage
        uint32_t q[D / 16][4];
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
            // rows 0-7 and 8-15 of columns 16 k .. 16 k + 7, then of the next eight
            ldmatrix4(q[k], smem_base + (uint32_t)(S::kQOffset + (lane & 15) * S::kQPitch + k * 32 + (lane >> 4) * 16));
        }
        const int   g = lane >> 2, t = lane & 3;
        const float c = p.scale_log2;
        // the last key a row sees
        int place[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const long long at = (long long)first_place(p, b) + (g + 8 * h) % p.queries;
            place[h]           = p.causal ? (int)min(max(at, -1ll), (long long)kMaxKeys) : kMaxKeys;
        }
        int taken = 0;
        for (int i = rank; i < halves; i += splits, ++taken) {
            const int s = taken % S::kStages;
            if (!mbar_wait_warp(full_bar(s), (uint32_t)(taken / S::kStages & 1), abort_flag, p.wait_limit_ns)) {
                if (lane == 0) {
                    give_up(0x9200u | (unsigned)s);
                }
                break;
            }
            const uint32_t kt  = smem_base + (uint32_t)(s * S::kStage), vt = kt + S::kTile;
            const int      key = stage_key[s] + warp * 16;      // of the warp's first
            float          sc[2][4] = {};
            // chunk: 8 columns of a row, at its place in the 128-byte swizzle
            auto at = [&](uint32_t tile, int row, int chunk) {
                return tile + (uint32_t)((chunk >> 3) * kPanel + row * 128 + (((chunk & 7) ^ (row & 7)) << 4));
            };
#pragma unroll
            for (int n = 0; n < 2; ++n) {
#pragma unroll
                for (int k2 = 0; k2 < D / 32; ++k2) {
                    uint32_t kf[4];
                    ldmatrix4(kf, at(kt, warp * 16 + n * 8 + (lane & 7), k2 * 4 + (lane >> 3)));
                    mma16<T>(sc[n], q[2 * k2], kf[0], kf[1]);
                    mma16<T>(sc[n], q[2 * k2 + 1], kf[2], kf[3]);
                }
            }
            const int exist = min(max(len - key, 0), 16);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int see = min(place[h] - key + 1, exist);
                float     top = -INFINITY;
#pragma unroll
                for (int n = 0; n < 2; ++n) {
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float& x = sc[n][2 * h + e];
                        x        = n * 8 + 2 * t + e < see ? x : -INFINITY;
                        top      = fmaxf(top, x);      // a NaN is not the maximum, but its weight is NaN and so is the row's sum
                    }
                }
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const float was = m[h], now = fmaxf(was, top);
                const float nmc = now == -INFINITY ? 0.0f : -now * c;      // no key seen: every weight is exp2(-inf)
                // From the difference of the maxima, so that one that stands gives exactly 1: was * c + nmc is the rounding of now * c then (2^-14 for |now * c| of
                // 1300), which every stage would multiply in anew; over 4096 stages of equal keys a result was off by 4 % of its values.
                const float f   = was == now ? 1.0f : ex2_approx((was - now) * c);
                m[h]            = now;
                float sum = 0.0f;
#pragma unroll
                for (int n = 0; n < 2; ++n) {
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float w    = ex2_approx(fmaf(sc[n][2 * h + e], c, nmc));
                        sc[n][2 * h + e] = w;
                        sum += w;
                    }
                }
                l[h] = l[h] * f + sum;      // of this lane's keys; the quad's are added at the end
                if (__any_sync(0xffffffffu, f != 1.0f)) {
#pragma unroll
                    for (int n = 0; n < D / 8; ++n) {
                        o[n][2 * h] *= f;
                        o[n][2 * h + 1] *= f;
                    }
                }
            }
            const uint32_t pf[4] = {Pair<T>::from_f32(sc[0][0], sc[0][1]), Pair<T>::from_f32(sc[0][2], sc[0][3]), Pair<T>::from_f32(sc[1][0], sc[1][1]),
                                    Pair<T>::from_f32(sc[1][2], sc[1][3])};
            auto keep = [&](int k) { return (k < exist ? 0xffffu : 0u) | (k + 1 < exist ? 0xffff0000u : 0u); };
            const uint32_t keep0 = keep(2 * t), keep1 = keep(2 * t + 8);
#pragma unroll
            for (int n2 = 0; n2 < D / 16; ++n2) {
                uint32_t vf[4];
                ldmatrix4_trans(vf, at(vt, warp * 16 + (lane & 15), n2 * 2 + (lane >> 4)));
                mma16<T>(o[2 * n2], pf, vf[0] & keep0, vf[1] & keep1);
                mma16<T>(o[2 * n2 + 1], pf, vf[2] & keep0, vf[3] & keep1);
            }
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(empty_bar(s));
            }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
            l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
        }
    }
    // ---------------------------------------------------------------------- the warps' sums meet, then the CTAs'
    float* const ml   = reinterpret_cast<float*>(gen_base + S::kMlOffset);
    float* const part = reinterpret_cast<float*>(gen_base);
    __syncthreads();      // the ring is empty
    if (warp < kWarps) {
        const int g = lane >> 2, t = lane & 3;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int r = g + 8 * h;
            if (t == 0) {
                ml[(warp * 2) * kMaxRows + r]     = m[h];
                ml[(warp * 2 + 1) * kMaxRows + r] = l[h];
            }
            if (r < n_rows) {
#pragma unroll
                for (int n = 0; n < D / 8; ++n) {
                    *reinterpret_cast<float2*>(part + (warp * kMaxRows + r) * S::kPitch + n * 8 + 2 * t) = make_float2(o[n][2 * h], o[n][2 * h + 1]);
                }
            }
        }
    }
    __syncthreads();
    const float c = p.scale_log2;
    // weight of a part whose maximum is `of` in a sum whose maximum is `top`
    auto weight = [&](float of, float top) { return of == -INFINITY ? 0.0f : ex2_approx((of - top) * c); };
    for (int i = (int)threadIdx.x; i < n_rows * (D / 4); i += kThreads) {
        const int r = i / (D / 4), d = i % (D / 4) * 4;
        float     top = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            top = fmaxf(top, ml[w * 2 * kMaxRows + r]);
        }
        float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const float  f = weight(ml[w * 2 * kMaxRows + r], top);
            const float4 v = *reinterpret_cast<const float4*>(part + (w * kMaxRows + r) * S::kPitch + d);
            sum += f * ml[(w * 2 + 1) * kMaxRows + r];
            a.x += f * v.x;
            a.y += f * v.y;
            a.z += f * v.z;
            a.w += f * v.w;
        }
        *reinterpret_cast<float4*>(part + r * S::kPitch + d) = a;      // in the place of warp 0's, which no other thread reads
        if (d == 0) {
            ml[kWarps * 2 * kMaxRows + r]       = top;
            ml[(kWarps * 2 + 1) * kMaxRows + r] = sum;
        }
    }
    cluster_sync_all();
    if (*abort_flag == 0) {
        const uint32_t ml_at = smem_base + (uint32_t)(S::kMlOffset + kWarps * 2 * kMaxRows * 4);
        for (int i = (int)threadIdx.x + rank * kThreads; i < n_rows * (D / 8); i += kThreads * splits) {
            const int r = i / (D / 8), d = i % (D / 8) * 8;
            float     top = -INFINITY, sum = 0.0f, a[8] = {};
            for (int s = 0; s < splits; ++s) {
                top = fmaxf(top, ld_cluster_f32(map_to_cta(ml_at + (uint32_t)(r * 4), (uint32_t)s)));
            }
            for (int s = 0; s < splits; ++s) {
                const uint32_t at = map_to_cta(ml_at + (uint32_t)(r * 4), (uint32_t)s), v = map_to_cta(smem_base + (uint32_t)((r * S::kPitch + d) * 4), (uint32_t)s);
                const float    f  = weight(ld_cluster_f32(at), top);
                const float4   x = ld_cluster_f32x4(v), y = ld_cluster_f32x4(v + 16u);
                sum += f * ld_cluster_f32(at + kMaxRows * 4u);
                a[0] += f * x.x;
                a[1] += f * x.y;
                a[2] += f * x.z;
                a[3] += f * x.w;
                a[4] += f * y.x;
                a[5] += f * y.y;
                a[6] += f * y.z;
                a[7] += f * y.w;
            }
            const int   head = list * heads + r / p.queries, qi = r % p.queries;
            const float inv  = sum == 0.0f ? 0.0f : 1.0f / sum;      // no key seen: zeros
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                a[e] *= inv;
            }
            const Vec16 y = p.q_lens == nullptr || qi < query_count(p, b) ? pack8<T>(a) : Vec16{};    // a row behind the sequence's queries: zeros too
            st_16(reinterpret_cast<T*>(p.out) + (long long)b * p.os.batch + (long long)qi * p.os.token + (long long)head * p.os.head + d, y);
        }
    }
    cluster_sync_all();   // no CTA leaves while a peer reads its shared memory
}

template<typename T, int D> static int launch(const Params& p, int sms, cudaStream_t stream)
{
    using S = Smem<D>;
    CUtensorMap tk, tv;
    int         st = make_map(&tk, p.k, p.ks, p.batch, p.k_heads, p.keys, D, kKeys);
    if (st == LYRAQ_OK) {
        st = make_map(&tv, p.v, p.vs, p.batch, p.k_heads, p.keys, D, kKeys);
    }
    static bool smem_raised[64] = {};
    if (st == LYRAQ_OK) {
        st = raise_dynamic_smem_once(sparse_attention_rows_kernel<T, D>, (int)S::kTotal, smem_raised, "cudaFuncSetAttribute(sparse_attention_rows_kernel)");
    }
    if (st != LYRAQ_OK) {
        return st;
    }
    // CTAs of a list: two an SM, but no more than there may be half blocks
    const int units = p.batch * p.lists, halves = p.count * (p.block / kKeys);
    int       splits = 1;
    while (splits < 8 && units * splits * 2 <= 2 * sms && splits * 2 <= halves) {
        splits *= 2;
    }
    return cuda_status(launch_kernel(sparse_attention_rows_kernel<T, D>, (unsigned)(units * splits), (unsigned)kThreads, (size_t)S::kTotal, stream,
                                     (unsigned)splits, tk, tv, p, splits),
                       "cudaLaunchKernelEx(sparse_attention_rows_kernel)");
}

}  // namespace rows

// Up to 16 rows share a list.  A tile of 128 queries with as few in it takes the time of a full one, and one CTA walks the whole list.
bool few_rows(const Params& p) { return p.count > 0 && (long long)(p.q_heads / p.lists) * p.queries <= rows::kMaxRows && p.batch * p.lists <= 0x0fffffff; }

int launch_rows(const Params& p, int dtype, int head_dim, cudaStream_t stream)
{
    const int sms = device_sm_count();
    if (sms <= 0) {
        return LYRAQ_ERR_CUDA;
    }
    if (dtype == LYRAQ_BF16) {
        return head_dim == 128 ? rows::launch<__nv_bfloat16, 128>(p, sms, stream) : rows::launch<__nv_bfloat16, 64>(p, sms, stream);
    }
    return head_dim == 128 ? rows::launch<__half, 128>(p, sms, stream) : rows::launch<__half, 64>(p, sms, stream);
}

}  // namespace sattn
}  // namespace lyraq
