// Selection of key blocks for block-sparse attention: means of blocks of tokens, their products, and the largest of them for each query block.
//
//   mean(block) = fl( sum of its existing tokens, in 64 bits, / their number )                     fl: rounding to fp32
//   score(i, j) = fl( sum over the head's channels of q_mean(i) k_mean(j), in 64 bits )            for a shared list q_mean is the sum over its heads
//
// What is selected jumps where two scores change places, so the scores should not depend on the order of a sum.  In 64 bits two orders differ by some 2^-50 of
// the sum of |q_mean k_mean|, and round to the same fp32 score unless it lies that close to the border of two: once in 2^26 where its terms hardly cancel, more
// often the more they do.  The means are held in 32 bits, which is part of the definition.
#include "common.cuh"
#include "views.h"

#include <type_traits>

namespace lyraq {

int device_sm_count();  // gemm_dense.cu

namespace bsel {

constexpr int kQueryBlock  = 128;     // queries that share a list
constexpr int kMeanThreads = 128;
constexpr int kAtOnce      = 16;      // tokens of a thread on their way together
constexpr int kMaxHeadDim  = 256;
constexpr int kMaxKeys     = 1 << 30;
constexpr int kMaxBlocks   = 32768;   // key blocks: the keys of a row are held in the registers of one thread block

// A fp32 number in 64 bits by shifts: its bits, the exponent under a double's, read as the value times 2^-896, subnormals and zeros included (infinities and
// NaN do not: their users look for them).
__device__ __forceinline__ double widen_f32(uint32_t u) { return __hiloint2double(((int)u >> 3) & (int)0x8fffffffu, (int)(u << 29)); }

// ------------------------------------------------------------------------------- means
// A pass over memory: 100 MB, 15 us, for q of 32760 tokens in 12 heads of 128 (measured: 28, the additions).  WARPS warps take one block of tokens of one head: D / 8 lanes a token, 16 bytes
// each, as many tokens at a time as there are lanes for; their sums meet in shared memory.  One warp a block where there are many, which spares
// instructions (the sums' way through shared memory, a division a channel), four where there are few.
// An addition in 64 bits for every value took 35 us: B200 does six of them a clock and SM.  So 16 tokens at a time are added in fp32 with their
// rounding errors beside them (D. Knuth's two-sum), and the sum and the sum of errors then go to 64 bits.  Both are exact as long as
// the exponents of the values lie close enough: with the largest E (below 2^(E + 1)) a sum of 16 is below 2^(E + 5), an error at most 2^(E - 19) and 16 of them
// 2^(E - 15); with the smallest e all are multiples of 2^(e - M), M bits behind the point, so 24 bits hold them if E - e <= 39 - M.  Blocks whose values lie further
// apart, or that hold infinities or NaN, are added again in 64 bits.
// Where only the newest tokens changed, only the blocks that hold them are taken.
struct MeansParams {
    float*      means;          // [batch][heads][blocks][head_dim]
    const void* x;
    size_t      batch_step, token_step, head_step;
    const int*  lens;           // tokens of each sequence, or null
    int         tokens, heads, head_dim, block, blocks;
    int         newest;         // 0: all blocks
    int         per_head;       // blocks of one head that are taken
    int         heads_first;    // neighbouring blocks: those of the same tokens in all heads (which lie side by side), or of the same head
    int         units;
};

// LANES: D / 8 where it is 8 or 16, else 0 (any)
template<typename T, int WARPS, int LANES> __global__ void __launch_bounds__(kMeanThreads) block_means_kernel(const MeansParams p)
{
    constexpr int kUnits = kMeanThreads / (WARPS * 32), kLanes = WARPS * 32;
    __shared__ double part_all[kUnits][kLanes * 8];
    grid_launch_dependents();
    grid_dependency_wait();
    double* const   part = part_all[kUnits == 1 ? 0 : (int)threadIdx.x / kLanes];
    const int       me   = (int)threadIdx.x % kLanes;
    const int       unit = (int)blockIdx.x * kUnits + (int)threadIdx.x / kLanes;
    if (unit >= p.units) {
        return;    // whole warps, and with one unit a thread block never
    }
    auto meet = [] {
        if (kUnits == 1) {
            __syncthreads();
        } else {
            __syncwarp();
        }
    };
    const int inner = p.heads_first ? p.heads : p.per_head, outer = p.heads_first ? p.per_head : p.heads;
    const int whole = unit / inner, in = unit - whole * inner, b = whole / outer, out_of = whole - b * outer;
    const int h  = p.heads_first ? in : out_of;
    int       j  = p.heads_first ? out_of : in;
    const int len = p.lens == nullptr ? p.tokens : min(max(__ldg(p.lens + b), 0), p.tokens);
    if (p.newest > 0) {
        j += max(len - p.newest, 0) / p.block;
        if (len == 0 || j > (len - 1) / p.block) {
            return;
        }
    }
    const int  lanes = LANES > 0 ? LANES : p.head_dim / 8, slots = kLanes / lanes;
    const int  slot = me / lanes, c = me % lanes * 8;
    const int  first = j * p.block, count = max(min(p.block, len - first), 0);
    const T*   src  = reinterpret_cast<const T*>(p.x) + (size_t)b * p.batch_step + (size_t)h * p.head_step + (size_t)(first + slot) * p.token_step + (size_t)c;
    const size_t step = (size_t)slots * p.token_step;
    double     sum[8] = {};
    // this thread's tokens, 16 at a time, as words of two channels each; those that do not exist are zeros
    auto each = [&](auto take) {
        if (slot < slots) {
            const T* at = src;
            for (int t = slot; t < count; t += kAtOnce * slots) {
                Vec16 v[kAtOnce];
#pragma unroll
                for (int i = 0; i < kAtOnce; ++i) {
                    v[i] = Vec16{};
                    if (t + i * slots < count) {
                        v[i] = ld_nc_16(at);
                    }
                    at += step;
                }
                take(v);
            }
        }
    };
    uint32_t most = 0, least = 0xffffffffu;      // of both channels of a word: the largest magnitude, and the smallest that is not 0, less 1
    each([&](const Vec16* v) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float2 s = make_float2(0.0f, 0.0f), lost = s;
            auto minus = [](float2 x, float2 y) { return fma_f32x2(y, make_float2(-1.0f, -1.0f), x); };
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i) {
                const uint32_t w = v[i].w[e], m = w & 0x7fff7fffu;
                most  = __vmaxu2(most, m);
                least = __viaddmin_u16x2(m, 0xffffffffu, least);
                const float2 x = Pair<T>::to_f32(w);
                const float2 t = add_f32x2(s, x), y = minus(t, s);
                lost = add_f32x2(lost, add_f32x2(minus(s, minus(t, y)), minus(x, y)));
                s    = t;
            }
            sum[2 * e] += (double)s.x;
            sum[2 * e + 1] += (double)s.y;
            sum[2 * e] += (double)lost.x;
            sum[2 * e + 1] += (double)lost.y;
        }
    });
    // exponents as the type holds them (of a subnormal: the least normal number's); bf16 sums stay below fp32's largest
    constexpr bool kBf16 = TypeTag<T>::value == LYRAQ_BF16;
    constexpr int  kMantissa = kBf16 ? 7 : 10, kTop = kBf16 ? 0xff - 5 : 0x1f;
    const int  top   = (int)(max(most & 0xffffu, most >> 16) >> kMantissa), low = max((int)((min(least & 0xffffu, least >> 16) + 1u) >> kMantissa), 1);
    const bool exact = top < kTop && top - low <= 39 - kMantissa;
    if (kUnits == 1 ? __syncthreads_or(exact ? 0 : 1) != 0 : !__all_sync(0xffffffffu, exact)) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            sum[e] = 0.0;
        }
        each([&](const Vec16* v) {
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float2 f = Pair<T>::to_f32(v[i].w[e]);
                    sum[2 * e] += (double)f.x;
                    sum[2 * e + 1] += (double)f.y;
                }
            }
        });
    }
    float*       out  = p.means + (((size_t)b * (size_t)p.heads + (size_t)h) * (size_t)p.blocks + (size_t)j) * (size_t)p.head_dim;
    const bool   even = (count & (count - 1)) == 0;                   // a power of two: the product with its reciprocal is the quotient
    const double n    = (double)max(count, 1);
    const double inv  = __hiloint2double((1023 - (31 - __clz(max(count, 1)))) << 20, 0);   // 1 / n of a power of two, by its exponent
    auto mean = [&](double s) {
        return (float)(even ? s * inv : s / n);
    };
    if constexpr (LANES > 0 && kUnits > 1) {
#pragma unroll
        for (int d = LANES; d < 32; d *= 2) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                sum[e] += __shfl_xor_sync(0xffffffffu, sum[e], d);
            }
        }
        if (slot < 2) {      // half of the lane's channels each
            float4 v;
            v.x = mean(slot == 0 ? sum[0] : sum[4]);
            v.y = mean(slot == 0 ? sum[1] : sum[5]);
            v.z = mean(slot == 0 ? sum[2] : sum[6]);
            v.w = mean(slot == 0 ? sum[3] : sum[7]);
            *reinterpret_cast<float4*>(out + c + slot * 4) = v;
        }
    } else {
        if (slot < slots) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                part[slot * p.head_dim + e * lanes + c / 8] = sum[e];      // neighbouring threads beside each other
            }
        }
        meet();
        for (int d = me; d < p.head_dim; d += kLanes) {
            double s = 0.0;
            for (int i = 0; i < slots; ++i) {
                s += part[i * p.head_dim + d];
            }
            out[d % lanes * 8 + d / lanes] = mean(s);
        }
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
    const int*   q_lens;       // queries of each sequence, or null
    const int*   q_start;      // place of each sequence's first query among the keys, or null
    int          batch, q_heads, k_heads, lists, head_dim, queries, keys, block, q_blocks, k_blocks;
    int          count, sink, window, causal;
    int          q_tiles, k_tiles;
};

// Products on the 64-bit tensor path (mma m8n8k4): QR x KT scores a thread block, a warp (QR / 2 or QR) x 16, chunk by chunk through shared memory, already in
// 64 bits (the queries may be sums over heads), the next chunk on its way.  201 million products of [256 x 512] blocks in 12 heads of 128 take 26 us, 30 a clock
// and SM; the vector pipe does six.
constexpr int    kScoreThreads = 256;
constexpr int    kChunk        = 32;
constexpr double kDown         = 1.8928834978668395e-270;     // 2^-896
constexpr double kUp           = 5.282945311356653e269;       // 2^896

template<int QR> __global__ void __launch_bounds__(kScoreThreads, 4) block_scores_kernel(const SelectParams p)
{
    constexpr int kWarpsQ = QR == 32 ? 2 : 1, kWarpsK = 8 / kWarpsQ;
    constexpr int kMt = QR / kWarpsQ / 8;     // fragments of 8 queries a warp
    constexpr int KT  = kWarpsK * 16;
    constexpr int kQ  = QR * kChunk / kScoreThreads, kK = KT * kChunk / 4 / kScoreThreads;   // queries' values and keys' vectors of a thread
    __shared__ double qs[QR][kChunk + 4];     // pitches that spread a fragment's 8 x 4 values over all banks
    __shared__ double ks[KT][kChunk + 4];
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
    float     qv[kQ];
    float4    kv[kK];
    auto load = [&](int d0) {
#pragma unroll
        for (int u = 0; u < kQ; ++u) {
            const int i = u * kScoreThreads + (int)threadIdx.x, r = i / kChunk, d = d0 + i % kChunk, row = qt * QR + r;
            qv[u] = row < p.q_blocks && d < p.head_dim && heads == 1 ? ld_f32(q + (size_t)row * (size_t)p.head_dim + (size_t)d) : 0.0f;
        }
#pragma unroll
        for (int u = 0; u < kK; ++u) {
            const int i = u * kScoreThreads + (int)threadIdx.x, r = i / (kChunk / 4), d = d0 + i % (kChunk / 4) * 4, row = kt * KT + r;
            kv[u] = row < p.k_blocks && d < p.head_dim ? ld_f32x4(reinterpret_cast<const float4*>(k + (size_t)row * (size_t)p.head_dim + (size_t)d))
                                                       : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
    };
    load(0);
    for (int d0 = 0; d0 < p.head_dim; d0 += kChunk) {
        const int width = min(kChunk, p.head_dim - d0);                  // a multiple of 8
        __syncthreads();
#pragma unroll
        for (int u = 0; u < kQ; ++u) {
            const int i = u * kScoreThreads + (int)threadIdx.x, r = i / kChunk, d = i % kChunk, row = qt * QR + r;
            double    v = (double)qv[u];
            if (heads > 1 && row < p.q_blocks && d < width) {
                v = 0.0;
                for (int h = 0; h < heads; ++h) {
                    v += (double)ld_f32(q + ((size_t)h * (size_t)p.q_blocks + (size_t)row) * (size_t)p.head_dim + (size_t)(d0 + d));
                }
            }
            qs[r][d] = v;
        }
        // keys times 2^-896, and the scores times 2^896: exact but for what is far below the least fp32 number
#pragma unroll
        for (int u = 0; u < kK; ++u) {
            const int    i = u * kScoreThreads + (int)threadIdx.x, r = i / (kChunk / 4), d = i % (kChunk / 4) * 4;
            const float4 v = kv[u];
            const float  f[4] = {v.x, v.y, v.z, v.w};
            const bool   finite = fabsf(v.x) < INFINITY && fabsf(v.y) < INFINITY && fabsf(v.z) < INFINITY && fabsf(v.w) < INFINITY;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                ks[r][d + e] = finite ? widen_f32(__float_as_uint(f[e])) : (double)f[e] * kDown;
            }
        }
        __syncthreads();
        if (d0 + kChunk < p.head_dim) {
            load(d0 + kChunk);
        }
#pragma unroll 4
        for (int d = 0; d < width; d += 4) {
            double a[kMt], c[2];
#pragma unroll
            for (int m = 0; m < kMt; ++m) {
                a[m] = qs[wq + m * 8 + (lane >> 2)][d + (lane & 3)];
            }
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                c[n] = ks[wk + n * 8 + (lane >> 2)][d + (lane & 3)];
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
                    out[(size_t)row * (size_t)p.k_blocks + (size_t)col] = (float)(acc[m][n][e] * kUp);
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
        // in 32 bits: a place beyond the keys by 2^30 and more is as good as one there
        const int first = (int)min((long long)start + (long long)i * kQueryBlock, (long long)kMaxKeys);
        const int rows  = min(kQueryBlock, (p.q_lens == nullptr ? p.queries : min(max(__ldg(p.q_lens + b), 0), p.queries)) - i * kQueryBlock);
        const int last  = min(first + max(rows, 1) - 1, kMaxKeys);
        auto block_of = [&](int t) { return t >= 0 ? t / p.block : -((p.block - 1 - t) / p.block); };   // downwards
        const int e = (int)(((unsigned)len + (unsigned)p.block - 1u) / (unsigned)p.block);
        end  = rows <= 0 ? 0 : p.causal ? min(e, max(block_of(last) + 1, 0)) : e;      // no query: nothing
        sink = p.sink;
        // windows wider than the keys are as good as all of them
        const int w = min(p.window - 1, kMaxKeys / 2);
        low  = p.window > 0 ? max(block_of(first) - w, -1) : 0;
        high = p.window > 0 ? max(min(block_of(last) + w, kMaxKeys), -1) : -1;
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
            n = total(n);
            if (n == want) {       // they are the ones: as a rule long before the bounds meet
                lo = mid - 1u;
                break;
            }
            if (n > want) {
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
    const size_t per_head = touched < blocks ? touched : blocks, units = per_head * batch * (size_t)heads;
    if (units > 0x7ffffff0u) {
        return LYRAQ_ERR_UNSUPPORTED;
    }
    const int sms = device_sm_count();
    if (sms <= 0) {
        return LYRAQ_ERR_CUDA;
    }
    // Four warps a block of tokens where one each would leave schedulers of an SM without one.  Four / one, us, changing buffers: 144 blocks of 128 x 128 6.6 / 10.4,
    // 432 8.1 / 11.9, 580 13.4 / 12.0 (fp16: 13.1 / 14.7), 888 14.7 / 12.9; 144 of 64 x 128 4.4 / 6.3, 432 5.3 / 7.4, 588 7.6 / 7.2, 888 9.1 / 7.5.
    const bool   few  = units <= 4 * (size_t)sms;
    const size_t grid = few ? units : (units + 3) / 4;
    const bsel::MeansParams p{means,       x,     batch_step, token_step, head_step, lens, (int)tokens, heads, head_dim, block, (int)blocks,
                              newest < bsel::kMaxKeys ? newest : bsel::kMaxKeys, (int)per_head, head_step < token_step ? 1 : 0, (int)units};
    auto launch = [&](auto* kernel) {
        return launch_kernel(kernel, (unsigned)grid, (unsigned)bsel::kMeanThreads, (size_t)0, (cudaStream_t)stream, 1u, p);
    };
    auto pick = [&](auto type, auto lanes) {
        using T = decltype(type);
        constexpr int kLanes = decltype(lanes)::value;
        return few ? launch(bsel::block_means_kernel<T, 4, kLanes>) : launch(bsel::block_means_kernel<T, 1, kLanes>);
    };
    auto pick_lanes = [&](auto type) {
        return head_dim == 128 ? pick(type, std::integral_constant<int, 16>{})
               : head_dim == 64 ? pick(type, std::integral_constant<int, 8>{})
                                : pick(type, std::integral_constant<int, 0>{});
    };
    const cudaError_t e = dtype == LYRAQ_BF16 ? pick_lanes(__nv_bfloat16{}) : pick_lanes(__half{});
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
    // a longer block than 2^30: its end less a place in front of the keys (Range) would leave 32 bits
    if (s->block > bsel::kMaxKeys || s->keys > (size_t)bsel::kMaxKeys || s->queries > (size_t)bsel::kMaxKeys || k_blocks > (size_t)bsel::kMaxBlocks || s->batch > 0xffffu ||
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
          reinterpret_cast<uintptr_t>(s->q_lens) | reinterpret_cast<uintptr_t>(s->q_start)) & 3u) != 0) {
        return LYRAQ_ERR_INVALID_ARG;
    }
    if (need > 0 && (workspace == nullptr || workspace_bytes < need || !aligned16(workspace))) {
        return LYRAQ_ERR_WORKSPACE;
    }
    const size_t dim = (size_t)s->head_dim;
    const View   out[3] = {view_of(s->index, rows * (size_t)s->count * 4), view_of(s->counts, rows * 4), view_of(workspace, need)};
    const View   in[5]  = {view_of(s->q_means, s->batch * (size_t)s->q_heads * q_blocks * dim * 4), view_of(s->k_means, s->batch * (size_t)s->k_heads * k_blocks * dim * 4),
                           view_of(s->k_lens, s->batch * 4), view_of(s->q_lens, s->batch * 4), view_of(s->q_start, s->batch * 4)};
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
    p.q_lens   = s->q_lens;
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
    const int    sms = device_sm_count();
    if (sms <= 0) {
        return LYRAQ_ERR_CUDA;
    }
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
    // Few rows of many blocks are spread over eight warps each.  Eight warps / one, us, with the scores: 1 row of 128 7.8 / 6.6, of 129 6.7 / 8.5, of 512 7.5 / 11.9; 148 rows of
    // 128 9.6 / 8.6, of 129 11.1 / 12.9, of 512 14.9 / 15.2; 600 rows of 129 15.4 / 11.7, 3000 of 512 42 / 29.
    const cudaError_t e = k_blocks <= 128 ? top(bsel::block_top_kernel<1, 4>, 1)
                          : rows <= (size_t)sms && k_blocks <= 1024 ? top(bsel::block_top_kernel<8, 4>, 8)
                          : k_blocks <= 512 ? top(bsel::block_top_kernel<1, 16>, 1)
                          : k_blocks <= 2048 ? top(bsel::block_top_kernel<4, 16>, 4)
                          : k_blocks <= 8192 ? top(bsel::block_top_kernel<16, 16>, 16)
                                             : top(bsel::block_top_kernel<32, 32>, 32);
    return cuda_status(e, "cudaLaunchKernelEx(block_top_kernel)");
}

}  // extern "C"
