// Whether two strided views share memory, decided on the host before a launch: an output that lies partly on what other blocks of the same kernel still
// read would come out by chance.  Plain C++, so that it can be checked without a GPU.
#pragma once

#include <cstddef>
#include <cstdint>
#include <initializer_list>

namespace lyraq {

// Up to three outer dimensions with strides in bytes, and a run of bytes in a row.  A dimension of one has no stride.
struct View {
    uintptr_t base, last;  // its first and its last byte
    size_t    count[4];    // the last: the run
    size_t    stride[4];
    bool      empty;
};

inline View view_of(const void* p, size_t elem_bytes, size_t n0, size_t s0, size_t n1, size_t s1, size_t n2, size_t s2, size_t run)
{
    View v{reinterpret_cast<uintptr_t>(p),
           0,
           {n0, n1, n2, run * elem_bytes},
           {n0 > 1 ? s0 * elem_bytes : 0, n1 > 1 ? s1 * elem_bytes : 0, n2 > 1 ? s2 * elem_bytes : 0, 1},
           p == nullptr || n0 == 0 || n1 == 0 || n2 == 0 || run == 0};
    v.last = v.base;
    for (int i = 0; i < 4 && !v.empty; ++i) {
        size_t step;
        if (__builtin_mul_overflow(v.count[i] - 1, v.stride[i], &step) || __builtin_add_overflow(v.last, step, &v.last)) {
            v.last = UINTPTR_MAX;   // strides that lead out of memory
            break;
        }
    }
    return v;
}
inline View view_of(const void* p, size_t bytes) { return view_of(p, 1, 1, 0, 1, 0, 1, 0, bytes); }

// Every element of one lies where the same element of the other does: a kernel whose threads write what they have read may have both.
inline bool views_same(const View& a, const View& b)
{
    bool same = a.base == b.base;
    for (int i = 0; i < 4; ++i) {
        same = same && a.count[i] == b.count[i] && a.stride[i] == b.stride[i];
    }
    return same;
}

namespace view_detail {

struct Term {
    __int128 stride, lo, hi;    // the sum of a term is stride * x, lo <= x <= hi
};

// Whether the terms can add up to `sum`.  Largest strides first, each tried where the rest can still make up the difference: in nested layouts that
// is one or two places.  looks: how many more may be tried; when they run out the answer is yes.
inline bool reach(const Term* t, int n, __int128 sum, int& looks)
{
    if (n == 0) {
        return sum == 0;
    }
    if (n == 1) {
        return sum % t->stride == 0 && sum / t->stride >= t->lo && sum / t->stride <= t->hi;
    }
    __int128 lo = 0, hi = 0;
    for (int i = 1; i < n; ++i) {
        lo += t[i].stride * t[i].lo;
        hi += t[i].stride * t[i].hi;
    }
    auto down = [](__int128 a, __int128 b) { return a >= 0 ? a / b : -((-a + b - 1) / b); };
    __int128 first = -down(-(sum - hi), t->stride), last = down(sum - lo, t->stride);
    first = first > t->lo ? first : t->lo;
    last  = last < t->hi ? last : t->hi;
    for (__int128 x = first; x <= last; ++x) {
        if (--looks < 0 || reach(t + 1, n - 1, sum - x * t->stride, looks)) {
            return true;
        }
    }
    return false;
}

}  // namespace view_detail

// Whether a byte belongs to both.  Exact, but for layouts so entangled that 4096 looks do not tell: those count as sharing.
inline bool views_meet(const View& a, const View& b)
{
    using view_detail::Term;
    if (a.empty || b.empty || a.last < b.base || b.last < a.base) {
        return false;
    }
    const __int128 apart = (__int128)b.base - (__int128)a.base;     // what the steps within a, less those within b, have to make up
    Term t[8];
    int  n = 0;
    auto add = [&](__int128 stride, __int128 lo, __int128 hi) {
        int i = 0;
        while (i < n && t[i].stride > stride) {
            ++i;
        }
        if (i < n && t[i].stride == stride) {
            t[i].lo += lo;
            t[i].hi += hi;
            return;
        }
        for (int j = n++; j > i; --j) {
            t[j] = t[j - 1];
        }
        t[i] = Term{stride, lo, hi};
    };
    for (int i = 0; i < 4; ++i) {
        if (a.count[i] > 1 && a.stride[i] != 0) {
            add((__int128)a.stride[i], 0, (__int128)a.count[i] - 1);
        }
        if (b.count[i] > 1 && b.stride[i] != 0) {
            add((__int128)b.stride[i], -((__int128)b.count[i] - 1), 0);
        }
    }
    int looks = 4096;
    return view_detail::reach(t, n, apart, looks);
}

// Whether a result lies on something that is still read while it is stored.  It may be the residual, element for element.
inline bool result_clashes(const View& y, const void* residual, std::initializer_list<View> read)
{
    for (const View& v : read) {
        if (views_meet(y, v)) {
            return true;
        }
    }
    return reinterpret_cast<uintptr_t>(residual) != y.base && views_meet(y, view_of(residual, y.count[3]));
}

}  // namespace lyraq
