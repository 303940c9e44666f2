// tree_split.h -- how the tree attention's work is counted and shared out (fattn_tree.cuh): the
// arithmetic alone, for the kernels and for a host that checks it.
#pragma once

#include <stdint.h>

#include <algorithm>

#ifdef __CUDACC__
#define OASR_HD __host__ __device__ __forceinline__
#else
#define OASR_HD inline
#endif

namespace oasr {

constexpr int TREE_BKV = 128;  // positions per unit

// Whether a sequence's committed positions and live nodes fit its MP pages and the N rows of the
// tensors; positions are 32-bit numbers, also those at the end of the last unit.
OASR_HD bool kv_lengths_fit(int past, int n, int N, int MP, int page) {
    return past >= 0 && n >= 0 && n <= N && (int64_t)past + n <= (int64_t)MP * page && (int64_t)past + n <= INT32_MAX - TREE_BKV;
}

struct TreeSeg {
    int s, hk, rt;         // sequence, K/V head, row tile
    int past, n, T, kt;    // committed positions, live nodes, past + n, units of the item
    int k0, k1;            // units of this segment
    int first, per, next;  // the item's first step, its steps, and where this segment ends
    int lead;              // its steps without a unit
};

// The call's steps (units in runs, pieces otherwise) over the CTAs: the first `more` CTAs take
// q + 1, the others q.  Lane l keeps what sequence l has: lengths, steps, and the steps of the
// sequences up to it.
struct TreeUnits {
    int total, ctas, q, more;
    int piece;  // most units of a piece, or 0: runs
    int past, n, mine, run;
};

// What the start and the end of a segment cost, and the join of an item's parts, in units: measured
// best of 1, 3, 5, 7 for tiles up to 64 rows (69.6, 69.2, 69.1, 69.1 us for 16 x 16 rows, 16 x 64 86.8,
// 84.7, 84.0, 85.1), of 7, 9, 12, 16 for 128 (16 trees of 61 nodes 100.8, 100.3, 103.6, 109).  A join:
// 8 sequences of one token of 20 heads of 64 take 13.3, 13.8, 11.5, 11.5 us with 1, 2, 3, 5, one token
// alone 8.8, 8.8, 8.8, 9.9.  The segments' figures are of D = 128; a unit of D = 64 is half the bytes,
// for which no other values were measured.
OASR_HD constexpr int tree_segment(int R) { return R == 128 ? 9 : 5; }
constexpr int TREE_JOIN = 3;

OASR_HD int tree_units(int past, int n) { return (past + n + TREE_BKV - 1) / TREE_BKV; }

OASR_HD float tree_rcp(int t) {
#ifdef __CUDA_ARCH__
    return __frcp_rn((float)t);
#else
    return 1.0f / (float)t;
#endif
}
// ceil(kt / t) for kt, t < 32768 by a reciprocal r = 1 / t: (kt + t - 1/2) / t is 1 / (2 t) or more
// away from every integer, the product less than 2^-7 / t off.
OASR_HD int tree_pieces(int kt, int t, float r) { return (int)(((float)(kt + t) - 0.5f) * r); }

// Steps of the `items` items of a sequence.
OASR_HD int tree_steps(int items, int kt, int piece, int R) {
    return items * (piece ? tree_pieces(kt, piece, tree_rcp(piece)) : kt + tree_segment(R));
}

// The size of pieces that lane l tries: from an even share of all units to the longest item.
OASR_HD int tree_try(int even, int most, int l) { return std::max(1, even + (most - even) * l / 31); }
// When the last of `pieces` pieces of at most t units ends, in units; TREE_MISFIT if they are more
// than the CTAs.
constexpr unsigned TREE_MISFIT = 65535u;
OASR_HD unsigned tree_piece_cost(int pieces, int ctas, int t, int most) {
    return pieces <= ctas ? (unsigned)(t < most ? t + TREE_JOIN : t) : TREE_MISFIT;
}
// Whether the call goes in pieces: the best cost of the lanes against a run of `run` steps.  Runs have
// no upper bound, so a misfit has to be told from a cost.
OASR_HD bool tree_in_pieces(unsigned cost, int run) { return cost != TREE_MISFIT && (int)cost <= run + TREE_JOIN; }

OASR_HD void tree_set_pieces(TreeUnits &w) {  // one per CTA
    w.ctas = std::max(1, w.total);
    w.q = std::min(w.total, 1);
    w.more = 0;
}
OASR_HD void tree_set_runs(TreeUnits &w, int ctas) {
    w.ctas = std::max(1, std::min(ctas, w.total));
    w.q = w.total / w.ctas;
    w.more = w.total - w.q * w.ctas;
}

OASR_HD int tree_start(const TreeUnits &w, int c) { return c >= w.ctas ? w.total : c * w.q + std::min(c, w.more); }
// the CTA whose range holds step u
OASR_HD int tree_owner(const TreeUnits &w, int u) {
    const int big = w.more * (w.q + 1);
    return u < big ? u / (w.q + 1) : w.more + (u - big) / w.q;
}
// A CTA leaves at most two unfinished segments: its first (slot 2c) and its last (2c + 1).
OASR_HD int tree_slot(const TreeUnits &w, int c, int item_first) { return 2 * c + (item_first > tree_start(w, c) ? 1 : 0); }

// The segment that starts at step u and ends before `end`, in the sequence whose first step is
// g.first, of g.past positions, g.n nodes and tiles of R of its `rows` rows.
OASR_HD void tree_cut(TreeSeg &g, int piece, int rows, int R, int u, int end) {
    g.T = g.past + g.n;
    g.kt = tree_units(g.past, g.n);
    g.lead = piece ? 0 : tree_segment(R);
    g.per = piece ? tree_pieces(g.kt, piece, tree_rcp(piece)) : g.kt + tree_segment(R);
    const int rts = (rows + R - 1) / R;
    const int item = (u - g.first) / g.per;
    g.hk = item / rts;
    g.rt = item - g.hk * rts;
    g.first += item * g.per;
    g.next = std::min(g.first + g.per, end);
    const int p0 = u - g.first, p1 = g.next - g.first;
    g.k0 = piece ? p0 * g.kt / g.per : std::max(0, p0 - g.lead);
    g.k1 = piece ? p1 * g.kt / g.per : std::max(0, p1 - g.lead);
}

}  // namespace oasr
