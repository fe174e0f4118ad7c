// Rotary embedding over several position axes, from the positions: no table is built, stored or read.
//
// Pair i of a head turns by pos[token, axis(i)] * f(i).  Angles are 64-bit fractions of a turn: F(i) = f(i) / 2 pi * 2^64, and the product of
// an integer position with it, kept to its low 64 bits, IS the angle modulo a turn, at position one as at a billion (in fp32, position 10^6
// times 1 rad would be off by 0.03 rad).  The top 32 bits go through sincospi.  A fractional position multiplies its 24-bit significand and
// shifts.
//
// q and k heads are normalised first where weights are given (RMS over the head, fp32), rotated in fp32 and rounded once; what lies behind the
// rotated part of a head is normalised and copied.
//
// Bound by memory: q and k in and out.  A block takes a few tokens; its threads first form the tokens' cosines and sines in shared memory, once for all
// heads, then a group of L lanes takes a head, every lane VEC pairs (16 bytes of either half, or 32 in a row), two heads of every
// thread in flight.  A lane's cosines stay in registers while it goes through the heads of a token.
#include "common.cuh"
#include "views.h"

namespace lyraq {

int device_sm_count();  // gemm_dense.cu

struct RopeAxesParams {
    const void*          src[2];      // q, k
    void*                dst[2];
    const void*          norm[2];
    size_t               src_batch[2], src_token[2], src_head[2], dst_batch[2], dst_token[2], dst_head[2];   // strides in elements
    const void*          pos;
    size_t               pos_batch, pos_token, pos_axis;
    const uint64_t*      turns;       // [pairs]
    const unsigned char* axis;        // [pairs]
    int                  pos_dtype;
    int                  heads[2];
    int                  head_dim, pairs, lanes_log2, groups, chunks, share, tokens_per_block;
    int                  beside;      // tokens that a block's groups take at a time
    int                  wide;        // interleaved pairs whose 16 neighbours lie on 32 bytes, in and out
    unsigned             tokens, seq;
    float                eps, inv_dim;
};

// Angle of one pair as a fraction of a turn, in 1 / 2^64.
__device__ __forceinline__ bool angle_of(const RopeAxesParams& p, size_t at, uint64_t turns, uint64_t& phase)
{
    if (p.pos_dtype == LYRAQ_S32) {
        phase = (uint64_t)(int64_t)reinterpret_cast<const int*>(p.pos)[at] * turns;
        return true;
    }
    if (p.pos_dtype == LYRAQ_S64) {
        phase = (uint64_t)reinterpret_cast<const int64_t*>(p.pos)[at] * turns;
        return true;
    }
    const uint32_t b = __float_as_uint(reinterpret_cast<const float*>(p.pos)[at]);
    const uint32_t e = (b >> 23) & 0xffu;
    if (e == 0xffu) {
        return false;
    }
    const uint64_t m  = (uint64_t)((b & 0x7fffffu) | (e != 0u ? 0x800000u : 0u));
    const int      sh = (int)(e != 0u ? e : 1u) - 150;       // position = m 2^sh
    const uint64_t lo = m * turns, hi = __umul64hi(m, turns);
    uint64_t       v;
    if (sh >= 0) {
        v = sh < 64 ? lo << sh : 0u;                         // whole turns beyond
    } else if (sh > -64) {
        v = (lo >> -sh) | (hi << (64 + sh));
    } else {
        v = sh > -128 ? hi >> (-sh - 64) : 0u;
    }
    phase = (b >> 31) != 0u ? 0u - v : v;
    return true;
}

template<typename T, int VEC> struct Piece;   // VEC values of T
template<typename T> struct Piece<T, 8> {
    Vec16 v;
    __device__ __forceinline__ void load(const T* p) { v = ld_16(p); }
    __device__ __forceinline__ void store(T* p) const { st_16(p, v); }
    __device__ __forceinline__ void get(float* f) const { unpack8<T>(v, f); }
    __device__ __forceinline__ void set(const float* f) { v = pack8<T>(f); }
};
template<typename T> struct Piece<T, 4> {
    uint32_t a, b;
    __device__ __forceinline__ void load(const T* p) { asm volatile("ld.global.v2.u32 {%0, %1}, [%2];" : "=r"(a), "=r"(b) : "l"(p)); }
    __device__ __forceinline__ void store(T* p) const { st_8(p, a, b); }
    __device__ __forceinline__ void get(float* f) const
    {
        const float2 x = Pair<T>::to_f32(a), y = Pair<T>::to_f32(b);
        f[0] = x.x; f[1] = x.y; f[2] = y.x; f[3] = y.y;
    }
    __device__ __forceinline__ void set(const float* f)
    {
        a = Pair<T>::from_f32(f[0], f[1]);
        b = Pair<T>::from_f32(f[2], f[3]);
    }
};
template<typename T> struct Piece<T, 2> {
    uint32_t a;
    __device__ __forceinline__ void load(const T* p) { asm volatile("ld.global.u32 %0, [%1];" : "=r"(a) : "l"(p)); }
    __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<uint32_t*>(p) = a; }
    __device__ __forceinline__ void get(float* f) const
    {
        const float2 x = Pair<T>::to_f32(a);
        f[0] = x.x; f[1] = x.y;
    }
    __device__ __forceinline__ void set(const float* f) { a = Pair<T>::from_f32(f[0], f[1]); }
};
template<typename T> struct Piece<T, 1> {
    T v;
    __device__ __forceinline__ void load(const T* p) { v = *reinterpret_cast<const volatile T*>(p); }
    __device__ __forceinline__ void store(T* p) const { *p = v; }
    __device__ __forceinline__ void get(float* f) const { f[0] = to_f32(v); }
    __device__ __forceinline__ void set(const float* f) { v = from_f32<T>(f[0]); }
};
template<> __device__ __forceinline__ void Piece<__half, 1>::load(const __half* p) { v = __ushort_as_half((unsigned short)ld_u16(p)); }
template<> __device__ __forceinline__ void Piece<__nv_bfloat16, 1>::load(const __nv_bfloat16* p) { v = __ushort_as_bfloat16((unsigned short)ld_u16(p)); }

// VEC floats of shared memory, on 16 bytes where VEC is a multiple of four
template<int VEC> __device__ __forceinline__ void load_floats(const float* p, float* f)
{
    if constexpr (VEC % 4 == 0) {
#pragma unroll
        for (int j = 0; j < VEC; j += 4) {
            const float4 v = *reinterpret_cast<const float4*>(p + j);
            f[j] = v.x; f[j + 1] = v.y; f[j + 2] = v.z; f[j + 3] = v.w;
        }
    } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            f[j] = p[j];
        }
    }
}

// VEC: pairs of a lane's unit; NU: units of a lane (more than one only where 32 lanes of small units do not span a head); HALVES: pair i is (x[i], x[i + pairs]), else
// (x[2 i], x[2 i + 1]); NORM: q or k is normalised; BESIDE: several tokens at a time (asking
// for it took a block of many heads 23.6 -> 29.5 us).
template<typename T, int VEC, int NU, bool HALVES, bool NORM, bool BESIDE>
__global__ void __launch_bounds__(256) rope_axes_kernel(const RopeAxesParams p)
{
    extern __shared__ __align__(16) float turn_c[];      // [2][tokens_per_block][pairs]: cosines, then sines
    grid_launch_dependents();
    grid_dependency_wait();
    const unsigned at    = blockIdx.x / (unsigned)p.chunks, chunk = blockIdx.x - at * (unsigned)p.chunks;
    const unsigned t0    = at * (unsigned)p.tokens_per_block;
    const int      n_tok = (int)min((unsigned)p.tokens_per_block, p.tokens - t0);
    for (int i = threadIdx.x; i < n_tok * p.pairs; i += blockDim.x) {
        const int      tk = i / p.pairs, pair = i - tk * p.pairs;
        const unsigned token = t0 + tk, b = token / p.seq, s = token - b * p.seq;
        uint64_t       phase = 0;
        float2         cs    = make_float2(__int_as_float(0x7fc00000), __int_as_float(0x7fc00000));
        if (angle_of(p, b * p.pos_batch + s * p.pos_token + (size_t)p.axis[pair] * p.pos_axis, p.turns[pair], phase)) {
            // half turns in [-1, 1)
            sincospif((float)(int)(uint32_t)(phase >> 32) * 4.656612873077393e-10f, &cs.y, &cs.x);
        }
        turn_c[i]                                = cs.x;
        turn_c[p.tokens_per_block * p.pairs + i] = cs.y;
    }
    __syncthreads();

    const int lanes = 1 << p.lanes_log2;
    const int lane = (int)threadIdx.x & (lanes - 1), any_group = (int)threadIdx.x >> p.lanes_log2;
    const int next = BESIDE ? any_group / p.groups : 0, group = any_group - next * p.groups;     // which of the tokens beside each other, group of it
    const int units = p.head_dim / (2 * VEC), turning = p.pairs / VEC;     // units of a head, those of them that turn
    // this block's share of the heads, dealt to groups
    const int h0 = (int)chunk * p.share, h1 = min(h0 + p.share, p.heads[0] + p.heads[1]);
    int  at_a[NU], at_b[NU];
    bool there[NU], turns[NU];
#pragma unroll
    for (int u = 0; u < NU; ++u) {
        const int unit = lane + u * lanes;
        there[u] = unit < units;
        turns[u] = unit < turning;
        at_a[u]  = HALVES && turns[u] ? unit * VEC : unit * 2 * VEC;
        at_b[u]  = HALVES && turns[u] ? p.pairs + unit * VEC : unit * 2 * VEC + VEC;
    }
    for (int t = 0; t < n_tok; t += BESIDE ? p.beside : 1) {
        const bool     here  = !BESIDE || (next < p.beside && t + next < n_tok);
        const int      tk    = BESIDE && here ? t + next : t;
        const unsigned token = t0 + tk, b = token / p.seq, s = token - b * p.seq;
        float          cosine[NU][VEC], sine[NU][VEC];
#pragma unroll
        for (int u = 0; u < NU; ++u) {
            if (turns[u]) {
                const float* c = turn_c + tk * p.pairs + (lane + u * lanes) * VEC;
                load_floats<VEC>(c, cosine[u]);
                load_floats<VEC>(c + p.tokens_per_block * p.pairs, sine[u]);
            }
        }
        const T* base_in[2];
        T*       base_out[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            base_in[k]  = reinterpret_cast<const T*>(p.src[k]) + b * p.src_batch[k] + s * p.src_token[k];
            base_out[k] = reinterpret_cast<T*>(p.dst[k]) + b * p.dst_batch[k] + s * p.dst_token[k];
        }
        for (int hb = h0; hb < h1; hb += 2 * p.groups) {
            Piece<T, VEC> a[2][NU], c[2][NU];
            T*            out[2];
            const T*      w[2];
            bool          on[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int  head = hb + group + i * p.groups;
                const bool is_k = head >= p.heads[0];
                on[i]           = (BESIDE ? here : group < p.groups) && head < h1;
                const T* in     = is_k ? base_in[1] + (size_t)(head - p.heads[0]) * p.src_head[1] : base_in[0] + (size_t)head * p.src_head[0];
                out[i]          = is_k ? base_out[1] + (size_t)(head - p.heads[0]) * p.dst_head[1] : base_out[0] + (size_t)head * p.dst_head[0];
                w[i]            = reinterpret_cast<const T*>(is_k ? p.norm[1] : p.norm[0]);
#pragma unroll
                for (int u = 0; u < NU; ++u) {
                    if (on[i] && there[u]) {
                        if constexpr (VEC == 8 && !HALVES) {
                            if (p.wide) {
                                ld_32(in + at_a[u], a[i][u].v, c[i][u].v);
                                continue;
                            }
                        }
                        a[i][u].load(in + at_a[u]);
                        c[i][u].load(in + at_b[u]);
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (!NORM && !on[i]) {
                    continue;
                }
                float x[NU][2 * VEC];
#pragma unroll
                for (int u = 0; u < NU; ++u) {
#pragma unroll
                    for (int j = 0; j < 2 * VEC; ++j) {
                        x[u][j] = 0.0f;
                    }
                    if (on[i] && there[u]) {
                        a[i][u].get(x[u]);
                        c[i][u].get(x[u] + VEC);
                    }
                }
                if (NORM) {
                    float2 sq2 = make_float2(0.0f, 0.0f);
#pragma unroll
                    for (int u = 0; u < NU; ++u) {
#pragma unroll
                        for (int j = 0; j < VEC; ++j) {
                            const float2 e = make_float2(x[u][2 * j], x[u][2 * j + 1]);
                            sq2            = fma_f32x2(e, e, sq2);
                        }
                    }
                    float sq = sq2.x + sq2.y;
                    for (int m = lanes >> 1; m > 0; m >>= 1) {
                        sq += __shfl_xor_sync(0xffffffffu, sq, m);
                    }
                    if (w[i] != nullptr) {
                        const float  inv = rsqrtf(sq * p.inv_dim + p.eps);
                        const float2 in2 = make_float2(inv, inv);
#pragma unroll
                        for (int u = 0; u < NU; ++u) {
                            if (on[i] && there[u]) {
                                Piece<T, VEC> wa, wc;   // from L1; in shared memory as fp32 their bank conflicts cost 5 us of 26
                                float         f[2 * VEC];
                                wa.load(w[i] + at_a[u]);
                                wc.load(w[i] + at_b[u]);
                                wa.get(f);
                                wc.get(f + VEC);
#pragma unroll
                                for (int j = 0; j < VEC; ++j) {
                                    const float2 e  = mul_f32x2(make_float2(x[u][2 * j], x[u][2 * j + 1]), mul_f32x2(in2, make_float2(f[2 * j], f[2 * j + 1])));
                                    x[u][2 * j]     = e.x;
                                    x[u][2 * j + 1] = e.y;
                                }
                            }
                        }
                    }
                }
#pragma unroll
                for (int u = 0; u < NU; ++u) {
                    if (on[i] && there[u]) {
                        if (turns[u]) {
#pragma unroll
                            for (int j = 0; j < VEC; ++j) {
                                const int   p0 = HALVES ? j : 2 * j, p1 = HALVES ? VEC + j : 2 * j + 1;
                                const float v0 = x[u][p0], v1 = x[u][p1];
                                x[u][p0]       = fmaf(v0, cosine[u][j], -v1 * sine[u][j]);
                                x[u][p1]       = fmaf(v0, sine[u][j], v1 * cosine[u][j]);
                            }
                        }
                        a[i][u].set(x[u]);
                        c[i][u].set(x[u] + VEC);
                        if constexpr (VEC == 8 && !HALVES) {
                            if (p.wide) {
                                st_32(out[i] + at_a[u], a[i][u].v, c[i][u].v);
                                continue;
                            }
                        }
                        a[i][u].store(out[i] + at_a[u]);
                        c[i][u].store(out[i] + at_b[u]);
                    }
                }
            }
        }
    }
}

static bool even_strides(const void* p, size_t batch, size_t token, size_t head, unsigned vec)
{
    return (reinterpret_cast<uintptr_t>(p) & (2 * vec - 1)) == 0 && ((batch | token | head) & (vec - 1)) == 0;
}

// A head is written while others are read: an output is its input, element for element, or apart from it, and apart from the rest.
static bool outputs_clash(const lyraq_rope_axes_t& a)
{
    auto view = [&](const void* p, int heads, size_t batch, size_t token, size_t head) {
        return view_of(p, 2, a.batch, batch, a.seq_len, token, (size_t)heads, head, (size_t)a.head_dim);
    };
    const View q = view(a.q, a.q_heads, a.q_batch, a.q_token, a.q_head), qo = view(a.q_out, a.q_heads, a.q_out_batch, a.q_out_token, a.q_out_head);
    const View k = view(a.k, a.k_heads, a.k_batch, a.k_token, a.k_head), ko = view(a.k_out, a.k_heads, a.k_out_batch, a.k_out_token, a.k_out_head);
    return (!views_same(q, qo) && views_meet(q, qo)) || (!views_same(k, ko) && views_meet(k, ko)) || views_meet(qo, k) || views_meet(ko, q) || views_meet(qo, ko);
}

}  // namespace lyraq

using namespace lyraq;

extern "C" int lyraq_rope_axes(const lyraq_rope_axes_t* a, void* stream)
{
    if (a == nullptr || (a->pos_dtype != LYRAQ_S32 && a->pos_dtype != LYRAQ_S64 && a->pos_dtype != LYRAQ_F32) || a->q_heads < 0 || a->k_heads < 0 ||
        a->head_dim <= 0 || a->pairs < 0) {
        return LYRAQ_ERR_INVALID_ARG;
    }
    if ((a->dtype != LYRAQ_F16 && a->dtype != LYRAQ_BF16) || a->head_dim > 256 || (a->head_dim & 1) != 0 || a->pairs > a->head_dim / 2 ||
        a->q_heads > 65536 || a->k_heads > 65536 || a->batch > 0x7fffffffu || a->seq_len > 0x7fffffffu || a->batch * a->seq_len > 0x7fffffffu) {
        return LYRAQ_ERR_UNSUPPORTED;
    }
    const int heads = a->q_heads + a->k_heads;
    if (a->batch * a->seq_len == 0 || heads == 0) {
        return LYRAQ_OK;
    }
    if ((a->q_heads > 0 && (a->q == nullptr || a->q_out == nullptr)) || (a->k_heads > 0 && (a->k == nullptr || a->k_out == nullptr)) ||
        (a->pairs > 0 && (a->positions == nullptr || a->turns == nullptr || a->axis == nullptr))) {
        return LYRAQ_ERR_INVALID_ARG;
    }
    const uintptr_t pos_align = a->pos_dtype == LYRAQ_S64 ? 7u : 3u;
    if ((reinterpret_cast<uintptr_t>(a->positions) & pos_align) != 0 || (reinterpret_cast<uintptr_t>(a->turns) & 7u) != 0) {
        return LYRAQ_ERR_INVALID_ARG;
    }
    if (((reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->q_out) | reinterpret_cast<uintptr_t>(a->k) |
          reinterpret_cast<uintptr_t>(a->k_out) | reinterpret_cast<uintptr_t>(a->q_norm) | reinterpret_cast<uintptr_t>(a->k_norm)) & 1u) != 0) {
        return LYRAQ_ERR_INVALID_ARG;
    }
    if (outputs_clash(*a)) {
        return LYRAQ_ERR_INVALID_ARG;
    }
    const int sms = device_sm_count();
    if (sms <= 0) {
        return LYRAQ_ERR_CUDA;
    }
    RopeAxesParams p{};
    p.src[0] = a->q; p.src[1] = a->k; p.dst[0] = a->q_out; p.dst[1] = a->k_out; p.norm[0] = a->q_norm; p.norm[1] = a->k_norm;
    p.src_batch[0] = a->q_batch; p.src_token[0] = a->q_token; p.src_head[0] = a->q_head;
    p.src_batch[1] = a->k_batch; p.src_token[1] = a->k_token; p.src_head[1] = a->k_head;
    p.dst_batch[0] = a->q_out_batch; p.dst_token[0] = a->q_out_token; p.dst_head[0] = a->q_out_head;
    p.dst_batch[1] = a->k_out_batch; p.dst_token[1] = a->k_out_token; p.dst_head[1] = a->k_out_head;
    p.pos = a->positions; p.pos_batch = a->pos_batch; p.pos_token = a->pos_token; p.pos_axis = a->pos_axis; p.pos_dtype = a->pos_dtype;
    p.turns = a->turns; p.axis = a->axis; p.heads[0] = a->q_heads; p.heads[1] = a->k_heads; p.head_dim = a->head_dim; p.pairs = a->pairs;
    p.tokens = (unsigned)(a->batch * a->seq_len); p.seq = (unsigned)a->seq_len; p.eps = a->eps; p.inv_dim = 1.0f / (float)a->head_dim;
    // the widest pieces that sizes, strides and addresses allow
    auto fits = [&](int vec) {
        const int  rest = a->head_dim - 2 * a->pairs;
        const bool size = a->pairs % vec == 0 && rest % (2 * vec) == 0;
        const bool q = a->q_heads == 0 || (even_strides(a->q, a->q_batch, a->q_token, a->q_head, vec) &&
                                           even_strides(a->q_out, a->q_out_batch, a->q_out_token, a->q_out_head, vec) && even_strides(a->q_norm, 0, 0, 0, vec));
        const bool k = a->k_heads == 0 || (even_strides(a->k, a->k_batch, a->k_token, a->k_head, vec) &&
                                           even_strides(a->k_out, a->k_out_batch, a->k_out_token, a->k_out_head, vec) && even_strides(a->k_norm, 0, 0, 0, vec));
        return size && q && k;
    };
    const int vec   = fits(8) ? 8 : fits(4) ? 4 : fits(2) ? 2 : 1;
    const int units = a->head_dim / (2 * vec);
    auto on_32 = [](const void* x, size_t batch, size_t token, size_t head) { return even_strides(x, batch, token, head, 16); };
    p.wide = vec == 8 && a->interleaved != 0 &&
             (a->q_heads == 0 || (on_32(a->q, a->q_batch, a->q_token, a->q_head) && on_32(a->q_out, a->q_out_batch, a->q_out_token, a->q_out_head))) &&
             (a->k_heads == 0 || (on_32(a->k, a->k_batch, a->k_token, a->k_head) && on_32(a->k_out, a->k_out_batch, a->k_out_token, a->k_out_head)));
    while ((1 << p.lanes_log2) < units && p.lanes_log2 < 5) {
        ++p.lanes_log2;
    }
    // Groups: two heads each at a time (24 heads as 12 groups of two take 65 us for 32760 tokens of 128, as 24 of one 83), all of a token in as few
    // rounds as 128 threads make of them, the rounds equally full (48 normalised heads with 192 threads 26.5 us, with 96 23.7).
    // Tokens: enough to share the cosines' cost, few enough to fill the chip; where there are few, a token's heads are dealt to several blocks.
    const int lanes  = 1 << p.lanes_log2;
    const int most   = 128 / lanes;
    p.chunks         = p.tokens >= (unsigned)sms * 2 ? 1 : (heads + most - 1) / most;
    p.share          = (heads + p.chunks - 1) / p.chunks;
    const int rounds = (p.share + 2 * most - 1) / (2 * most);
    p.groups         = (p.share + 2 * rounds - 1) / (2 * rounds);
    p.tokens_per_block = p.tokens >= (unsigned)sms * 32 ? 4 : p.tokens >= (unsigned)sms * 16 ? 2 : 1;
    // Heads that leave most of 128 threads idle: several tokens beside each other, as long as two blocks an SM are left.  One after the other / beside, us:
    // 8000 tokens of 1 + 1 heads of 128 11.2 / 6.6, of 4 + 4 11.2 / 7.8, of 8 + 2 11.6 / 9.9; 30000 tokens of 1 + 1 20.6 / 13.2, but of 4 + 4 24.8 / 29.7:
    // where there are many of both, a token a block at a time keeps more loads in flight.
    p.beside = 1;
    const bool few = p.groups * lanes <= 16 || p.tokens < (unsigned)sms * 100u;
    while (p.chunks == 1 && few && 2 * p.beside * p.groups * lanes <= 128 && (unsigned)(2 * p.beside) * (unsigned)sms * 2u <= p.tokens) {
        p.beside *= 2;
    }
    p.tokens_per_block     = p.tokens_per_block > p.beside ? p.tokens_per_block : p.beside;
    const unsigned threads = (unsigned)((p.beside * p.groups * lanes + 31) / 32 * 32);
    const size_t   blocks  = ((size_t)p.tokens + p.tokens_per_block - 1) / p.tokens_per_block * (size_t)p.chunks;
    if (blocks > 0x7fffffffu) {
        return LYRAQ_ERR_UNSUPPORTED;
    }
    const unsigned grid = (unsigned)blocks;
    const bool   norm = a->q_norm != nullptr || a->k_norm != nullptr;
    const size_t smem = 2 * sizeof(float) * (size_t)p.tokens_per_block * (size_t)p.pairs;
    auto launch = [&](auto* kernel) { return launch_kernel(kernel, grid, threads, smem, (cudaStream_t)stream, 1u, p); };
    auto pick = [&](auto type, auto halves, auto normed) {
        using T           = decltype(type);
        constexpr bool kH = decltype(halves)::value, kN = decltype(normed)::value;
        auto by_tokens = [&](auto many) {
            constexpr bool kB = decltype(many)::value;
            return vec == 8   ? launch(rope_axes_kernel<T, 8, 1, kH, kN, kB>)
                   : vec == 4 ? launch(rope_axes_kernel<T, 4, 1, kH, kN, kB>)
                   : vec == 2 ? launch(rope_axes_kernel<T, 2, 2, kH, kN, kB>)
                              : launch(rope_axes_kernel<T, 1, 4, kH, kN, kB>);
        };
        return p.beside > 1 ? by_tokens(std::integral_constant<bool, true>{}) : by_tokens(std::integral_constant<bool, false>{});
    };
    auto pick_norm = [&](auto type, auto halves) {
        return norm ? pick(type, halves, std::integral_constant<bool, true>{}) : pick(type, halves, std::integral_constant<bool, false>{});
    };
    auto pick_style = [&](auto type) {
        return a->interleaved ? pick_norm(type, std::integral_constant<bool, false>{}) : pick_norm(type, std::integral_constant<bool, true>{});
    };
    const cudaError_t e = a->dtype == LYRAQ_BF16 ? pick_style(__nv_bfloat16{}) : pick_style(__half{});
    return cuda_status(e, "cudaLaunchKernelEx(rope_axes_kernel)");
}
