// What the two kernels of block-sparse attention share (sparse_attention.cu: tiles of 128 queries; sparse_attention_rows.cu: few queries).
#pragma once

#include "common.cuh"
#include "softmax.cuh"
#include "views.h"

namespace lyraq {
namespace sattn {

constexpr int kQueryBlock = 128;
constexpr int kMaxKeys    = 1 << 30;

struct Steps {
    long long batch, token, head;   // elements
};

struct Params {
    const void*   q;
    const void*   k;
    const void*   v;
    void*         out;
    Steps         qs, ks, vs, os;
    const int*    index;
    const int*    counts;
    const int*    k_lens;
    const int*    q_lens;
    const int*    q_start;
    int           batch, queries, keys;
    int           q_heads, k_heads, lists;
    int           q_blocks, block, count, causal;
    int           items;          // work units of the kernel
    int           fixed;          // bits 0, 1, 2: q, k, v lie at one place for all sequences (a batch step of 0)
    float         scale_log2;     // softmax scale * log2(e)
    unsigned int* status;
    unsigned long long wait_limit_ns;
    int           skip_loads;     // test hook: the producers issue no copy, so every consumer's wait runs out
};

__device__ __forceinline__ int load_int(const int* p)
{
    int v;
    asm volatile("ld.global.s32 %0, [%1];" : "=r"(v) : "l"(p));
    return v;
}
// keys of a sequence, and the place of its first query
__device__ __forceinline__ int key_count(const Params& p, int b) { return p.k_lens == nullptr ? p.keys : min(max(load_int(p.k_lens + b), 0), p.keys); }
// its queries
__device__ __forceinline__ int query_count(const Params& p, int b) { return p.q_lens == nullptr ? p.queries : min(max(load_int(p.q_lens + b), 0), p.queries); }
__device__ __forceinline__ int first_place(const Params& p, int b)
{
    return p.q_start == nullptr ? p.keys - p.queries : min(max(load_int(p.q_start + b), -kMaxKeys), kMaxKeys);
}

bool few_rows(const Params& p);   // whether the few-row kernel takes the call
int launch_rows(const Params& p, int dtype, int head_dim, cudaStream_t stream);   // sparse_attention_rows.cu

}  // namespace sattn
}  // namespace lyraq
