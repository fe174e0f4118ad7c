// Selection of key blocks for block-sparse attention: means of blocks of tokens, their products, and the largest of them for each query block.
//
//   mean(block) = fl( sum of its existing tokens, in 64 bits, / their number )                     fl: rounding to fp32
//   score(i, j) = fl( sum over the head's channels of q_mean(i) k_mean(j), in 64 bits )            for a shared list q_mean is the sum over its heads
//
// What is selected jumps where two scores change places, so the scores must not depend on the order of a sum: in 64 bits two orders differ by 2^-50
// of a score, and both round to the same fp32 number but once in 2^26.  The means are held in 32 bits, which is part of the definition.
#include "common.cuh"
#include "views.h"

namespace lyraq {

int device_sm_count();  // gemm_dense.cu

namespace bsel {

constexpr int kQueryBlock  = 128;     // queries that share a list
constexpr int kMeanThreads = 128;
constexpr int kMaxHeadDim  = 256;
constexpr int kMaxKeys     = 1 << 30;
constexpr int kMaxBlocks   = 32768;   // key blocks: the keys of a row are held in the registers of one thread block

// ------------------------------------------------------------------------------- means
// A pass over memory.  A thread block takes one block of tokens of one head: D / 8 lanes a token, 16 bytes each, as many tokens at a time as the
// threads allow; their sums meet in shared memory.  Where only the newest tokens changed, only the blocks that hold them are taken.
struct MeansParams {
    float*      means;          // [batch][heads][blocks][head_dim]
    const void* x;
    size_t      batch_step, token_step, head_step;
    const int*  lens;           // tokens of each sequence, or null
    int         tokens, heads, head_dim, block, blocks;
    int         newest;         // 0: all blocks
    int         per_head;       // thread blocks of one head
};

template<typename T> __global__ void __launch_bounds__(kMeanThreads) block_means_kernel(const MeansParams p)
{
    __shared__ double part[kMeanThreads * 8];
    grid_launch_dependents();
    grid_dependency_wait();
    const int unit = (int)blockIdx.x / p.per_head, h = unit % p.heads, b = unit / p.heads;
    int       j    = (int)blockIdx.x % p.per_head;
    const int len  = p.lens == nullptr ? p.tokens : min(max(__ldg(p.lens + b), 0), p.tokens);
    if (p.newest > 0) {
        j += max(len - p.newest, 0) / p.block;
        if (len == 0 || j > (len - 1) / p.block) {
            return;
        }
    }
    const int lanes = p.head_dim / 8, slots = kMeanThreads / lanes;
    const int slot = (int)threadIdx.x / lanes, c = (int)threadIdx.x % lanes * 8;
    const int first = j * p.block, end = min(first + p.block, len);
    double    sum[8] = {};
    if (slot < slots) {
        const T* src = reinterpret_cast<const T*>(p.x) + (size_t)b * p.batch_step + (size_t)h * p.head_step + (size_t)c;
        for (int t0 = first + slot; t0 < end; t0 += 8 * slots) {
            Vec16 v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int t = t0 + i * slots;
                v[i]        = Vec16{};
                if (t < end) {
                    v[i] = ld_nc_16(src + (size_t)t * p.token_step);
                }
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float f[8];
                unpack8<T>(v[i], f);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    sum[e] += (double)f[e];
                }
            }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            part[slot * p.head_dim + c + e] = sum[e];
        }
    }
    __syncthreads();
    float* out = p.means + (((size_t)b * (size_t)p.heads + (size_t)h) * (size_t)p.blocks + (size_t)j) * (size_t)p.head_dim;
    for (int d = (int)threadIdx.x; d < p.head_dim; d += kMeanThreads) {
        double s = 0.0;
        for (int i = 0; i < slots; ++i) {
            s += part[i * p.head_dim + d];
        }
        out[d] = end > first ? (float)(s / (double)(end - first)) : 0.0f;
    }
}

// ------------------------------------------------------------------------------- scores
struct SelectParams {
    const float* q_means;      // [batch][q_heads][q_blocks][head_dim]
    const float* k_means;      // [batch][k_heads][k_blocks][head_dim]
    float*       scores;       // [batch][lists][q_blocks][k_blocks]
    int*         index;        // [batch][lists][q_blocks][count]
    int*         counts;       // [batch][lists][q_blocks]
    const int*   k_lens;       // keys of each sequence, or null
    const int*   q_start;      // place of each sequence's first query among the keys, or null
    int          batch, q_heads, k_heads, lists, head_dim, queries, keys, block, q_blocks, k_blocks;
    int          count, sink, window, causal;
    int          q_tiles, k_tiles;
};

// Products on the 64-bit tensor path (mma m8n8k4): QR x KT scores a thread block, a warp (QR / 2 or QR) x 16, K chunk by chunk through shared memory,
// queries already in 64 bits (they may be sums over heads), keys in 32.  201 million products of [256 x 512] blocks in 12 heads of 128 are 11.5 us at
// 64 a clock and SM.
constexpr int kScoreThreads = 256;
constexpr int kChunk        = 64;

template<int QR> __global__ void __launch_bounds__(kScoreThreads) block_scores_kernel(const SelectParams p)
{
    constexpr int kWarpsQ = QR == 32 ? 2 : 1, kWarpsK = 8 / kWarpsQ;
    constexpr int kMt = QR / kWarpsQ / 8;     // fragments of 8 queries a warp
    constexpr int KT  = kWarpsK * 16;
    __shared__ double qs[QR][kChunk + 4];     // pitches that spread a fragment's 8 x 4 values over all banks
    __shared__ float  ks[KT][kChunk + 4];
    grid_launch_dependents();
    grid_dependency_wait();
    const int kt = (int)blockIdx.x % p.k_tiles, qt = (int)blockIdx.x / p.k_tiles % p.q_tiles, unit = (int)blockIdx.x / (p.k_tiles * p.q_tiles);
    const int list = unit % p.lists, b = unit / p.lists;
    const int heads = p.q_heads / p.lists;                               // query heads of the list
    const int kh    = list / (p.lists / p.k_heads);
    const float* q  = p.q_means + ((size_t)b * (size_t)p.q_heads + (size_t)list * (size_t)heads) * (size_t)p.q_blocks * (size_t)p.head_dim;
    const float* k  = p.k_means + ((size_t)b * (size_t)p.k_heads + (size_t)kh) * (size_t)p.k_blocks * (size_t)p.head_dim;
    const int warp = (int)threadIdx.x >> 5, lane = (int)threadIdx.x & 31;
    const int wq = warp % kWarpsQ * (QR / kWarpsQ), wk = warp / kWarpsQ * 16;
    double    acc[kMt][2][2] = {};
    for (int d0 = 0; d0 < p.head_dim; d0 += kChunk) {
        const int width = min(kChunk, p.head_dim - d0);                  // a multiple of 8
        __syncthreads();
        for (int i = (int)threadIdx.x; i < QR * kChunk; i += kScoreThreads) {
            const int r = i / kChunk, d = i % kChunk, row = qt * QR + r;
            double    v = 0.0;
            if (row < p.q_blocks && d < width) {
                for (int h = 0; h < heads; ++h) {
                    v += (double)ld_f32(q + ((size_t)h * (size_t)p.q_blocks + (size_t)row) * (size_t)p.head_dim + (size_t)(d0 + d));
                }
            }
            qs[r][d] = v;
        }
        for (int i = (int)threadIdx.x; i < KT * (kChunk / 4); i += kScoreThreads) {
            const int r = i / (kChunk / 4), d = i % (kChunk / 4) * 4, row = kt * KT + r;
            float4    v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (row < p.k_blocks && d < width) {
                v = ld_f32x4(reinterpret_cast<const float4*>(k + (size_t)row * (size_t)p.head_dim + (size_t)(d0 + d)));
            }
            *reinterpret_cast<float4*>(&ks[r][d]) = v;
        }
        __syncthreads();
#pragma unroll 4
        for (int d = 0; d < width; d += 4) {
            double a[kMt], c[2];
#pragma unroll
            for (int m = 0; m < kMt; ++m) {
                a[m] = qs[wq + m * 8 + (lane >> 2)][d + (lane & 3)];
            }
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                c[n] = (double)ks[wk + n * 8 + (lane >> 2)][d + (lane & 3)];
            }
#pragma unroll
            for (int m = 0; m < kMt; ++m) {
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    asm("mma.sync.aligned.m8n8k4.row.col.f64.f64.f64.f64 {%0, %1}, {%2}, {%3}, {%0, %1};"
                        : "+d"(acc[m][n][0]), "+d"(acc[m][n][1])
                        : "d"(a[m]), "d"(c[n]));
                }
            }
        }
    }
    float* out = p.scores + (size_t)unit * (size_t)p.q_blocks * (size_t)p.k_blocks;
#pragma unroll
    for (int m = 0; m < kMt; ++m) {
#pragma unroll
        for (int n = 0; n < 2; ++n) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int row = qt * QR + wq + m * 8 + (lane >> 2), col = kt * KT + wk + n * 8 + (lane & 3) * 2 + e;
                if (row < p.q_blocks && col < p.k_blocks) {
                    out[(size_t)row * (size_t)p.k_blocks + (size_t)col] = (float)acc[m][n][e];
                }
            }
        }
    }
}

// ------------------------------------------------------------------------------- the largest
// A score as an unsigned number of the same order: 0 for a block that may not be taken, all ones for one that is taken in any case.
__device__ __forceinline__ uint32_t score_key(float s)
{
    s = s != s ? -INFINITY : s + 0.0f;                   // a score that is no number comes last; -0 is 0
    const uint32_t u = __float_as_uint(s);
    return u ^ ((u >> 31) != 0u ? 0xffffffffu : 0x80000000u);
}

// What a query block may take: allowed are the blocks below `end`, taken in any case those below `sink` and those from `low` to `high`.
struct Range {
    int end, sink, low, high;
    __device__ __forceinline__ Range(const SelectParams& p, int b, int i)
    {
        const int  len   = p.k_lens == nullptr ? p.keys : min(max(__ldg(p.k_lens + b), 0), p.keys);
        // places beyond the keys, on either side, are all alike
        const int  start = p.q_start == nullptr ? p.keys - p.queries : min(max(__ldg(p.q_start + b), -kMaxKeys), kMaxKeys);
        const long long first = (long long)start + (long long)i * kQueryBlock;
        const long long last  = first + min(kQueryBlock, p.queries - i * kQueryBlock) - 1;
        auto block_of = [&](long long t) { return (t >= 0 ? t : t - (p.block - 1)) / p.block; };   // downwards
        const long long e = (len + (long long)p.block - 1) / p.block;
        end  = (int)(p.causal ? min(e, max(block_of(last) + 1, 0ll)) : e);
        sink = p.sink;
        low  = p.window > 0 ? (int)max(block_of(first) - (p.window - 1), -1ll) : 0;
        high = p.window > 0 ? (int)max(min(block_of(last) + (p.window - 1), (long long)kMaxKeys), -1ll) : -1;
    }
    __device__ __forceinline__ uint32_t key(int j, float s) const { return j >= end ? 0u : j < sink || (j >= low && j <= high) ? 0xffffffffu : score_key(s); }
};

// WARPS warps take one row of scores, each a run of 32 * PER neighbouring key blocks, PER a lane, and find by halving
// the largest T for which `want` keys or more are T or larger.  All above T are taken, and of those equal to T the first.
template<int WARPS, int PER> __global__ void __launch_bounds__(WARPS == 1 ? 128 : WARPS * 32) block_top_kernel(const SelectParams p)
{
    constexpr int kRows = WARPS == 1 ? 4 : 1;      // rows of a thread block
    __shared__ int part[2][WARPS];
    grid_launch_dependents();
    grid_dependency_wait();
    const int       warp = WARPS == 1 ? 0 : (int)threadIdx.x >> 5, lane = (int)threadIdx.x & 31;
    const long long row  = (long long)blockIdx.x * kRows + (WARPS == 1 ? (int)(threadIdx.x >> 5) : 0);
    if (row >= (long long)p.batch * p.lists * p.q_blocks) {
        return;    // whole warps, and in the form of several warps never
    }
    const int    i    = (int)(row % p.q_blocks), b = (int)(row / p.q_blocks / p.lists);
    const Range  range(p, b, i);
    const float* src  = p.scores + (size_t)row * (size_t)p.k_blocks;
    const int    base = warp * 32 * PER;
    uint32_t     key[PER];
    uint32_t     most = 0u, least = 0xffffffffu;
#pragma unroll
    for (int e = 0; e < PER; ++e) {
        const int j = base + e * 32 + lane;
        key[e]      = j < p.k_blocks ? range.key(j, ld_f32(src + j)) : 0u;
        most        = max(most, key[e]);
        least       = key[e] != 0u ? min(least, key[e]) : least;
    }
    int flip = 0;
    auto total = [&](int n) {      // over the row
        n = __reduce_add_sync(0xffffffffu, n);
        if (WARPS > 1) {
            if (lane == 0) {
                part[flip][warp] = n;
            }
            __syncthreads();
            n = 0;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                n += part[flip][w];
            }
            flip ^= 1;
        }
        return n;
    };
    const int allowed = min(max(range.end, 0), p.k_blocks), want = min(p.count, allowed);
    // the bounds' common bits need no halving (several warps: the whole range)
    uint32_t lo = 1u, hi = 0xffffffffu;
    if (WARPS == 1) {
        hi = __reduce_max_sync(0xffffffffu, most);
        lo = __reduce_min_sync(0xffffffffu, least);
        lo = min(lo, hi);
    }
    if (want < allowed) {
        while (lo < hi) {          // invariant: `want` or more are lo or larger, fewer are larger than hi
            const uint32_t mid = lo + (hi - lo) / 2u + 1u;
            int            n   = 0;
#pragma unroll
            for (int e = 0; e < PER; ++e) {
                n += key[e] >= mid ? 1 : 0;
            }
            if (total(n) >= want) {
                lo = mid;
            } else {
                hi = mid - 1u;
            }
        }
    } else {
        lo = 0u;                   // all that are allowed
    }
    const uint32_t t     = lo;
    int            above = 0, equal = 0;
#pragma unroll
    for (int e = 0; e < PER; ++e) {
        above += key[e] > t ? 1 : 0;
        equal += key[e] == t ? 1 : 0;
    }
    int before = 0, same_before = 0;      // taken, and equal to t, in the warps in front
    int spare;                            // how many of those equal to t are taken
    if (WARPS == 1) {
        spare = want - total(above);
    } else {
        above = __reduce_add_sync(0xffffffffu, above);
        equal = __reduce_add_sync(0xffffffffu, equal);
        __syncthreads();
        if (lane == 0) {
            part[0][warp] = above;
            part[1][warp] = equal;
        }
        __syncthreads();
        int all = 0;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            all += part[0][w];
        }
        spare = want - all;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            if (w < warp) {
                before += part[0][w];
                same_before += part[1][w];
            }
        }
        before += min(same_before, spare);
    }
    int*           out  = p.index + (size_t)row * (size_t)p.count;
    const uint32_t left = (1u << lane) - 1u;
#pragma unroll
    for (int e = 0; e < PER; ++e) {
        const uint32_t same = __ballot_sync(0xffffffffu, key[e] == t);
        const bool     take = key[e] > t || (key[e] == t && same_before + __popc(same & left) < spare);
        const uint32_t all  = __ballot_sync(0xffffffffu, take);
        if (take) {
            out[before + __popc(all & left)] = base + e * 32 + lane;
        }
        before += __popc(all);
        same_before += __popc(same);
    }
    for (int s = want + (int)(WARPS == 1 ? lane : threadIdx.x); s < p.count; s += WARPS * 32) {
        out[s] = -1;
    }
    if (WARPS == 1 ? lane == 0 : threadIdx.x == 0) {
        p.counts[row] = want;
    }
}

}  // namespace bsel
}  // namespace lyraq

using namespace lyraq;

extern "C" {

int lyraq_block_means(float* means, const void* x, int dtype, size_t batch_step, size_t token_step, size_t head_step, const int* lens, int block, int newest,
                      size_t batch, size_t tokens, int heads, int head_dim, void* stream)
{
    if (block <= 0 || newest < 0 || heads < 0 || head_dim < 0) {
        return LYRAQ_ERR_INVALID_ARG;
    }
    if (batch == 0 || tokens == 0 || heads == 0 || head_dim == 0) {
        return LYRAQ_OK;
    }
    if ((dtype != LYRAQ_F16 && dtype != LYRAQ_BF16) || (head_dim & 7) != 0 || head_dim > bsel::kMaxHeadDim || tokens > (size_t)bsel::kMaxKeys ||
        block > bsel::kMaxKeys || batch > 0xffffu || heads > 0xffff) {
        return LYRAQ_ERR_UNSUPPORTED;
    }
    if (means == nullptr || x == nullptr || !aligned16(means) || !aligned16(x) || ((batch_step | token_step | head_step) & 7u) != 0 ||
        (reinterpret_cast<uintptr_t>(lens) & 3u) != 0) {
        return LYRAQ_ERR_INVALID_ARG;
    }
    const size_t blocks = (tokens + (size_t)block - 1) / (size_t)block;
    const View   vm = view_of(means, batch * (size_t)heads * blocks * (size_t)head_dim * 4);
    if (views_meet(vm, view_of(x, 2, batch, batch_step, tokens, token_step, (size_t)heads, head_step, (size_t)head_dim)) ||
        views_meet(vm, view_of(lens, batch * 4))) {
        return LYRAQ_ERR_INVALID_ARG;
    }
    // `newest` tokens touch one block more than they fill, at most
    const size_t touched  = newest == 0 ? blocks : ((size_t)newest + (size_t)block - 2) / (size_t)block + 1;
    const size_t per_head = touched < blocks ? touched : blocks, grid = per_head * batch * (size_t)heads;
    if (grid > 0x7fffffffu) {
        return LYRAQ_ERR_UNSUPPORTED;
    }
    const bsel::MeansParams p{means,       x,     batch_step, token_step, head_step, lens, (int)tokens, heads, head_dim, block, (int)blocks,
                              newest < bsel::kMaxKeys ? newest : bsel::kMaxKeys, (int)per_head};
    const cudaError_t e = dtype == LYRAQ_BF16
                              ? launch_kernel(bsel::block_means_kernel<__nv_bfloat16>, (unsigned)grid, (unsigned)bsel::kMeanThreads, (size_t)0, (cudaStream_t)stream, 1u, p)
                              : launch_kernel(bsel::block_means_kernel<__half>, (unsigned)grid, (unsigned)bsel::kMeanThreads, (size_t)0, (cudaStream_t)stream, 1u, p);
    return cuda_status(e, "cudaLaunchKernelEx(block_means_kernel)");
}

size_t lyraq_select_blocks_workspace(size_t batch, int lists, size_t queries, size_t keys, int block)
{
    if (lists <= 0 || block <= 0) {
        return 0;
    }
    return batch * (size_t)lists * ((queries + bsel::kQueryBlock - 1) / bsel::kQueryBlock) * ((keys + (size_t)block - 1) / (size_t)block) * 4;
}

int lyraq_select_blocks(const lyraq_select_blocks_t* s, void* workspace, size_t workspace_bytes, void* stream)
{
    if (s == nullptr || s->block <= 0 || s->count <= 0 || s->sink < 0 || s->window < 0 || s->q_heads < 0 || s->k_heads < 0 || s->lists < 0 || s->head_dim < 0) {
        return LYRAQ_ERR_INVALID_ARG;
    }
    if (s->batch == 0 || s->queries == 0 || s->q_heads == 0) {
        return LYRAQ_OK;
    }
    if (s->k_heads == 0 || s->q_heads % s->k_heads != 0 || (s->lists != s->q_heads && s->lists != s->k_heads)) {
        return LYRAQ_ERR_INVALID_ARG;
    }
    const size_t k_blocks = (s->keys + (size_t)s->block - 1) / (size_t)s->block, q_blocks = (s->queries + bsel::kQueryBlock - 1) / bsel::kQueryBlock;
    if (s->keys > (size_t)bsel::kMaxKeys || s->queries > (size_t)bsel::kMaxKeys || k_blocks > (size_t)bsel::kMaxBlocks || s->batch > 0xffffu ||
        s->q_heads > 0xffff || s->head_dim == 0 || (s->head_dim & 7) != 0 || s->head_dim > bsel::kMaxHeadDim || s->count > bsel::kMaxBlocks) {
        return LYRAQ_ERR_UNSUPPORTED;
    }
    const size_t rows = s->batch * (size_t)s->lists * q_blocks, need = rows * k_blocks * 4;
    if (rows > 0x7fffffffu) {
        return LYRAQ_ERR_UNSUPPORTED;
    }
    if (s->q_means == nullptr || s->index == nullptr || s->counts == nullptr || !aligned16(s->q_means) || (k_blocks > 0 && s->k_means == nullptr) ||
        !aligned16(s->k_means) ||
        ((reinterpret_cast<uintptr_t>(s->index) | reinterpret_cast<uintptr_t>(s->counts) | reinterpret_cast<uintptr_t>(s->k_lens) |
          reinterpret_cast<uintptr_t>(s->q_start)) & 3u) != 0) {
        return LYRAQ_ERR_INVALID_ARG;
    }
    if (need > 0 && (workspace == nullptr || workspace_bytes < need || !aligned16(workspace))) {
        return LYRAQ_ERR_WORKSPACE;
    }
    const size_t dim = (size_t)s->head_dim;
    const View   out[3] = {view_of(s->index, rows * (size_t)s->count * 4), view_of(s->counts, rows * 4), view_of(workspace, need)};
    const View   in[4]  = {view_of(s->q_means, s->batch * (size_t)s->q_heads * q_blocks * dim * 4), view_of(s->k_means, s->batch * (size_t)s->k_heads * k_blocks * dim * 4),
                           view_of(s->k_lens, s->batch * 4), view_of(s->q_start, s->batch * 4)};
    for (int i = 0; i < 3; ++i) {
        for (const View& v : in) {
            if (views_meet(out[i], v)) {
                return LYRAQ_ERR_INVALID_ARG;
            }
        }
        if (views_meet(out[i], out[(i + 1) % 3])) {
            return LYRAQ_ERR_INVALID_ARG;
        }
    }
    bsel::SelectParams p{};
    p.q_means  = s->q_means;
    p.k_means  = s->k_means;
    p.scores   = static_cast<float*>(workspace);
    p.index    = s->index;
    p.counts   = s->counts;
    p.k_lens   = s->k_lens;
    p.q_start  = s->q_start;
    p.batch    = (int)s->batch;
    p.q_heads  = s->q_heads;
    p.k_heads  = s->k_heads;
    p.lists    = s->lists;
    p.head_dim = s->head_dim;
    p.queries  = (int)s->queries;
    p.keys     = (int)s->keys;
    p.block    = s->block;
    p.q_blocks = (int)q_blocks;
    p.k_blocks = (int)k_blocks;
    p.count    = s->count;
    p.sink     = s->sink;
    p.window   = s->window;
    p.causal   = s->causal;
    cudaStream_t st = (cudaStream_t)stream;
    if (k_blocks > 0) {
        const bool   few = q_blocks <= 8;
        const size_t qr = few ? 8 : 32, kt = few ? 128 : 64;
        p.q_tiles = (int)((q_blocks + qr - 1) / qr);
        p.k_tiles = (int)((k_blocks + kt - 1) / kt);
        const size_t grid = s->batch * (size_t)s->lists * (size_t)p.q_tiles * (size_t)p.k_tiles;
        if (grid > 0x7fffffffu) {
            return LYRAQ_ERR_UNSUPPORTED;
        }
        const cudaError_t e = few ? launch_kernel(bsel::block_scores_kernel<8>, (unsigned)grid, (unsigned)bsel::kScoreThreads, (size_t)0, st, 1u, p)
                                  : launch_kernel(bsel::block_scores_kernel<32>, (unsigned)grid, (unsigned)bsel::kScoreThreads, (size_t)0, st, 1u, p);
        if (e != cudaSuccess) {
            return cuda_status(e, "cudaLaunchKernelEx(block_scores_kernel)");
        }
    }
    auto top = [&](auto* kernel, int warps) {
        return launch_kernel(kernel, (unsigned)(warps == 1 ? (rows + 3) / 4 : rows), warps == 1 ? 128u : (unsigned)(warps * 32), (size_t)0, st, 1u, p);
    };
    const cudaError_t e = k_blocks <= 128 ? top(bsel::block_top_kernel<1, 4>, 1)
                          : k_blocks <= 512 ? top(bsel::block_top_kernel<1, 16>, 1)
                          : k_blocks <= 2048 ? top(bsel::block_top_kernel<4, 16>, 4)
                          : k_blocks <= 8192 ? top(bsel::block_top_kernel<16, 16>, 16)
                                             : top(bsel::block_top_kernel<32, 32>, 32);
    return cuda_status(e, "cudaLaunchKernelEx(block_top_kernel)");
}

}  // extern "C"
