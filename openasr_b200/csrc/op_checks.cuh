// op_checks.cuh -- argument checks that the operators of the paged cache and of sampled
// verification share (host side).
#pragma once

#include <stdlib.h>

#include <algorithm>
#include <string>

#include "common.cuh"

namespace oasr {

inline int fail_op(oasr_backend *be, const char *op, const char *what) {
    return oasr_internal_fail(be, OASR_STATUS_FAILED, std::string(op) + ": " + what);
}

inline int launched(oasr_backend *be, cudaError_t e, const char *what) {
    if (e != cudaSuccess) return oasr_internal_cuda_fail(be, e, what, __LINE__);
    return oasr_internal_launch_check(be, what);
}

// 4-byte values that are read and written as such
inline bool aligned4(const oasr_tensor *t) { return ((uintptr_t)t->data & 3) == 0; }

inline bool is_vec(const oasr_tensor *t, int type, int64_t n) {
    return t && t->type == type && t->data && aligned4(t) && t->ne[0] == n && t->ne[1] == 1 && t->ne[2] == 1 &&
           t->ne[3] == 1 && (t->nb[0] == 4 || n <= 1);
}

inline bool is_vec_i32(const oasr_tensor *t, int64_t n) { return is_vec(t, OASR_TYPE_I32, n); }

inline bool rows16(const oasr_tensor *t) {
    return ((uintptr_t)t->data & 15) == 0 && t->nb[1] % 16 == 0 && t->nb[2] % 16 == 0 && t->nb[3] % 16 == 0;
}

// 4-byte values [N, S] with contiguous rows
inline bool is_rows(const oasr_tensor *t, int type, int64_t N, int64_t S) {
    return t && t->type == type && t->data && aligned4(t) && t->ne[0] == N && t->ne[1] == S && t->ne[2] == 1 &&
           t->ne[3] == 1 && (t->nb[0] == 4 || N <= 1) && t->nb[1] % 4 == 0;
}

inline bool is_rows_i32(const oasr_tensor *t, int64_t N, int64_t S) { return is_rows(t, OASR_TYPE_I32, N, S); }

// Rows of 4-byte values on the device: `n` rows of `width` values, `ld` values apart.
struct IntRows {
    const int *at;
    int64_t n, width, ld;
};
inline IntRows int_rows(const oasr_tensor *t) { return {(const int *)t->data, t->ne[1], t->ne[0], t->ne[1] > 1 ? t->nb[1] / 4 : 0}; }

// Whether the two have a value in common (rows side by side in one buffer have none).
inline bool share_values(const IntRows &a, const IntRows &b) {
    auto row = [](const IntRows &r, int64_t i) { return r.at + (r.ld < 0 ? r.n - 1 - i : i) * r.ld; };  // ascending
    if (row(a, a.n - 1) + a.width <= row(b, 0) || row(b, b.n - 1) + b.width <= row(a, 0)) return false;
    for (int64_t i = 0, j = 0; i < a.n && j < b.n;) {
        const int *x = row(a, i), *y = row(b, j);
        if (x + a.width <= y) ++i;
        else if (y + b.width <= x) ++j;
        else return true;
    }
    return false;
}

// The bytes that a tensor covers: runs of `run` bytes from `at` on, `n` of them in each dimension at a stride,
// the greatest stride first; dimensions that continue a run are part of it.
struct Runs {
    const char *at;
    int64_t run, extent, n[4], stride[4], inner[4];  // inner: extent of what repeats in that dimension
    int dims = 0;

    explicit Runs(const oasr_tensor *t) : at((const char *)t->data), run(t->type == OASR_TYPE_F16 ? 2 : t->type == OASR_TYPE_I64 ? 8 : 4) {
        int order[4], k = 0;
        for (int i = 0; i < 4; ++i) {
            if (t->ne[i] <= 1 || t->nb[i] == 0) continue;
            if (t->nb[i] < 0) at += (t->ne[i] - 1) * t->nb[i];
            int j = k++;
            for (; j > 0 && llabs(t->nb[order[j - 1]]) > llabs(t->nb[i]); --j) order[j] = order[j - 1];
            order[j] = i;
        }
        int from = 0;
        for (; from < k && llabs(t->nb[order[from]]) <= run; ++from) run += (t->ne[order[from]] - 1) * llabs(t->nb[order[from]]);
        extent = run;
        dims = k - from;
        for (int j = 0; j < dims; ++j) {
            const int i = order[from + j], d = dims - 1 - j;
            n[d] = t->ne[i], stride[d] = llabs(t->nb[i]), inner[d] = extent;
            extent += (n[d] - 1) * stride[d];
        }
    }
    int64_t extent_of(int d) const { return d ? inner[d - 1] : extent; }  // of dimensions d, d + 1, ...
};

// Whether a's dimensions from da on meet b's from db on, `off` bytes further.  Equal strides go together, one step
// for the few places where the insides meet (views of one buffer); of others the greater is taken apart.
inline bool runs_meet(const Runs &a, int da, const Runs &b, int db, int64_t off) {
    if (off >= a.extent_of(da) || -off >= b.extent_of(db)) return false;
    auto up = [](int64_t x, int64_t y) { return x >= 0 ? (x + y - 1) / y : -(-x / y); };  // x / y rounded up
    const int64_t sa = da < a.dims ? a.stride[da] : 0, sb = db < b.dims ? b.stride[db] : 0;
    if (!sa && !sb) return true;
    if (sa == sb) {  // index of a minus index of b
        const int64_t lo = std::max(1 - b.n[db], up(off - a.inner[da] + 1, sa)), hi = std::min(a.n[da] - 1, -up(-off - b.inner[db] + 1, sa));
        for (int64_t c = lo; c <= hi; ++c)
            if (runs_meet(a, da + 1, b, db + 1, off - c * sa)) return true;
        return false;
    }
    if (sa < sb) return runs_meet(b, db, a, da, -off);
    const int64_t lo = std::max<int64_t>(0, up(off - a.inner[da] + 1, sa)), hi = std::min(a.n[da] - 1, -up(-off - b.extent_of(db) + 1, sa));
    for (int64_t c = lo; c <= hi; ++c)
        if (runs_meet(a, da + 1, b, db, off - c * sa)) return true;
    return false;
}

// Whether two tensors have a byte in common; either may be null or empty.
inline bool share_bytes(const oasr_tensor *x, const oasr_tensor *y) {
    for (const oasr_tensor *t : {x, y})
        if (!t || !t->data || !t->ne[0] || !t->ne[1] || !t->ne[2] || !t->ne[3]) return false;
    const Runs a(x), b(y);
    return runs_meet(a, 0, b, 0, b.at - a.at);
}

// Whether no two elements of a tensor lie in one place, its dimensions inside one another.
inline bool apart(const oasr_tensor *t) {
    const Runs r(t);
    int64_t count = r.run / (t->type == OASR_TYPE_F16 ? 2 : t->type == OASR_TYPE_I64 ? 8 : 4);
    for (int d = 0; d < r.dims; ++d) {
        if (r.stride[d] < r.inner[d]) return false;
        count *= r.n[d];
    }
    return count == t->ne[0] * t->ne[1] * t->ne[2] * t->ne[3];
}

// F32 [page, H_kv, n_pages] beside the pages
inline bool is_weights(const oasr_tensor *w, const oasr_tensor *k) {
    if (!w || w->type != OASR_TYPE_F32 || !w->data || !aligned4(w) || w->ne[0] != k->ne[1] || w->ne[1] != k->ne[2] ||
        w->ne[2] != k->ne[3] || w->ne[3] != 1 || w->nb[0] != 4 || w->nb[1] % 4 || w->nb[2] % 4)
        return false;
    // entries are read and written: no two of them in one place
    int64_t extent = 4 * w->ne[0];
    const bool pages_inside = w->nb[2] < w->nb[1];
    for (int i : {pages_inside ? 2 : 1, pages_inside ? 1 : 2}) {
        if (w->ne[i] == 1) continue;
        if (w->nb[i] < extent) return false;
        extent += (w->ne[i] - 1) * w->nb[i];
    }
    return true;
}

}  // namespace oasr
