// op_checks.cuh -- argument checks that the operators of the paged cache and of sampled
// verification share (host side).
#pragma once

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
