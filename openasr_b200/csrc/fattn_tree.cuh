// fattn_tree.cuh -- around the tree attention's inner loop: how the work is split over the CTAs,
// which nodes a row sees, and where unfinished sums wait to be joined.
//
// Work is counted in units: 128 positions of one item, an item being (sequence, K/V head, tile of
// R rows) and a row one query head of one node (row = node * G + head in the group).  The lengths
// are in device memory, so every warp works the split out itself, one of two:
//   - pieces: each item in equal pieces of at most t units, one piece per CTA, with the t that ends
//     first (a short call: a CTA has one start and one end; two caches of 30000 positions take 36 us
//     this way, 43 in runs);
//   - runs: CTA c takes the c-th of equal runs of units, across items (a long call, or more items
//     than CTAs: ragged batches balance to the unit).  An item counts tree_segment units more than
//     it has, at its front, for the start and the end of the segment that it begins; where a run
//     ends among those, the next one begins the item (16 trees of 61 nodes: 112 us without, 100 with).
// A segment is what a CTA does of one item.  One that is not the whole item leaves (maximum, sum,
// output) in the scratch, and the parts are joined in the order of the positions, so the bits do
// not depend on which CTA came first.
#pragma once

#include <cfloat>

#include "pages.cuh"
#include "tc_common.cuh"

namespace oasr {

constexpr float TREE_NONE = -1.7e38f;  // maximum of a row that has seen nothing (finite: -inf minus it is -inf)

static __device__ __forceinline__ int tree_items(const TreeAttn &a, int n, int R) {
    return (n * a.group.d + R - 1) / R * a.HKV;
}

// Lane l of every warp: lengths of sequence s.
static __device__ __forceinline__ bool tree_lane_lengths(const TreeAttn &a, const KvSeqs &q, int page, int s, int &past,
                                                         int &n) {
    past = n = 0;
    return s >= a.S || seq_lengths(q, s, page, past, n);
}

// Its steps (below 2^31: the launch checks) and the sum of those of the lanes up to this one.
static __device__ __forceinline__ void tree_lane_steps(const TreeAttn &a, int piece, int R, int past, int n, int &mine, int &run) {
    const int lane = threadIdx.x & 31, kt = tree_units(past, n);
    mine = n == 0 ? 0 : tree_steps(tree_items(a, n, R), kt, piece, R);
    run = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, run, o);
        if (lane >= o) run += up;
    }
}

// All warps: the call's split.  A sequence with lengths out of range counts nothing (reported).
static __device__ __forceinline__ TreeUnits tree_count(const TreeAttn &a, const KvSeqs &q, int page, int R, int ctas, int *err) {
    const int lane = threadIdx.x & 31;
    TreeUnits w;
    bool ok = tree_lane_lengths(a, q, page, lane, w.past, w.n);
    w.piece = 0;
    tree_lane_steps(a, 0, R, w.past, w.n, w.mine, w.run);
    w.total = __shfl_sync(0xffffffffu, w.run, 31);
    const int most = __reduce_max_sync(0xffffffffu, w.n ? tree_units(w.past, w.n) : 0);
    if (a.S <= 32 && most < 32768) {  // (products of two unit counts fit 31 bits)
        const int kt = tree_units(w.past, w.n), items = w.n ? tree_items(a, w.n, R) : 0;
        const int units = w.total - tree_segment(R) * (int)__reduce_add_sync(0xffffffffu, (unsigned)items);
        const int run = (w.total + ctas - 1) / ctas, even = min(most, (units + ctas - 1) / ctas);
        const int t = tree_try(even, most, lane);
        const float r = tree_rcp(t);
        int pieces = 0;
#pragma unroll 4
        for (int s = 0; s < a.S; ++s)
            pieces += __shfl_sync(0xffffffffu, items, s) * tree_pieces(__shfl_sync(0xffffffffu, kt, s), t, r);
        const unsigned cost = tree_piece_cost(pieces, ctas, t, most);
        const unsigned least = __reduce_min_sync(0xffffffffu, cost << 16 | (unsigned)t);
        const int best = (int)(least & 65535u);
        if (tree_in_pieces(least >> 16, run)) {
            w.piece = best;
            tree_lane_steps(a, best, R, w.past, w.n, w.mine, w.run);
            w.total = __shfl_sync(0xffffffffu, w.run, 31);
            tree_set_pieces(w);
            if (!ok && err && blockIdx.x == 0 && threadIdx.x < 32) atomicOr(err, ERR_BAD_INDEX);
            return w;
        }
    }
    for (int s0 = 32; s0 < a.S; s0 += 32) {
        int past, n, mine, run;
        ok &= tree_lane_lengths(a, q, page, s0 + lane, past, n);
        tree_lane_steps(a, 0, R, past, n, mine, run);
        w.total += __shfl_sync(0xffffffffu, run, 31);
    }
    if (!ok && err && blockIdx.x == 0 && threadIdx.x < 32) atomicOr(err, ERR_BAD_INDEX);
    tree_set_runs(w, ctas);
    return w;
}

// All lanes: the segment that starts at step u (u < total) and ends before `end`; without units only
// if it is the last before `end`.
static __device__ __forceinline__ TreeSeg tree_locate(const TreeAttn &a, const KvSeqs &q, const TreeUnits &w, int page, int R,
                                                      int u, int end) {
    const int lane = threadIdx.x & 31;
    int base = 0, past = w.past, n = w.n, mine = w.mine, run = w.run;
    TreeSeg g = {};
    for (int s0 = 0;;) {
        const unsigned hit = __ballot_sync(0xffffffffu, u < base + run);
        if (hit) {
            const int l = __ffs(hit) - 1;
            g.first = __shfl_sync(0xffffffffu, base + run - mine, l);
            g.past = __shfl_sync(0xffffffffu, past, l);
            g.n = __shfl_sync(0xffffffffu, n, l);
            g.s = s0 + l;
            break;
        }
        base += __shfl_sync(0xffffffffu, run, 31);
        if ((s0 += 32) >= a.S) break;  // not for u < total
        tree_lane_lengths(a, q, page, s0 + lane, past, n);
        tree_lane_steps(a, w.piece, R, past, n, mine, run);
    }
    tree_cut(g, w.piece, g.n * a.group.d, R, u, end);
    return g;
}

// What is read through two more dependent loads starts on its way to L2 with the lengths: the page
// table and the queries, spread over the grid.
static __device__ __forceinline__ void tree_prefetch(const TreeAttn &a, const KvSeqs &q) {
    const int step = gridDim.x * blockDim.x, me = blockIdx.x * blockDim.x + threadIdx.x;
    const int lines = (q.MP + 31) / 32;  // of 128 bytes per row of the table
    for (int s = me / lines, l = me % lines; s < a.S; s += step / lines + 1)
        asm volatile("prefetch.global.L2 [%0];" ::"l"(q.table + s * q.table_ld + l * 32));
    const int bytes = a.D * (a.q_f16 ? 2 : 4);
    for (unsigned e = me; e < (unsigned)(a.S * q.N) * (unsigned)a.H; e += step) {
        const unsigned i = e / (unsigned)a.H, h = e % (unsigned)a.H, s = i / (unsigned)q.N;
        const char *row = a.q + (i - s * q.N) * a.q_nb1 + h * a.q_nb2 + s * a.q_nb3;
        for (int x = 0; x < bytes; x += 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(row + x));
    }
}

// Whether the row of a live node sees position t < T.
static __device__ __forceinline__ bool tree_sees(const TreeAttn &a, const TreeSeg &g, int node, int t) {
    const int j = t - g.past;
    if (j < 0) return true;
    return a.tree ? (uint32_t)__ldg(a.tree + g.s * a.t_nb2 + node * a.t_nb1 + (j >> 5)) >> (j & 31) & 1u : j <= node;
}

// Which of the positions t0 .. t0 + 31 it sees, as bits (positions past the end: none).
static __device__ __forceinline__ uint32_t tree_sees32(const TreeAttn &a, const TreeSeg &g, int node, int t0) {
    const int j = t0 - g.past, live = g.n - j;  // node number of bit 0, and where the nodes end
    if (j <= -32) return 0xffffffffu;
    if (live <= 0) return 0u;
    uint32_t w;
    if (!a.tree) {
        const int c = node + 1 - j;
        w = c >= 32 ? 0xffffffffu : c <= 0 ? 0u : (1u << c) - 1u;
    } else {
        const int *row = a.tree + g.s * a.t_nb2 + node * a.t_nb1;
        if (j < 0) {
            w = (uint32_t)__ldg(row) << -j;
        } else {
            const int i = j >> 5, sh = j & 31;
            w = (uint32_t)__ldg(row + i) >> sh;
            if (sh && i + 1 < a.W) w |= (uint32_t)__ldg(row + i + 1) << (32 - sh);
        }
    }
    if (live < 32) w &= (1u << live) - 1u;
    return j < 0 ? w | ((1u << -j) - 1u) : w;
}

// Rows of padding nodes of every sequence: zeros.  Each of the `warps` warps of the grid, this
// one being number w, takes every warps-th node.
static __device__ __forceinline__ void tree_zero_padding(const TreeAttn &a, const KvSeqs &q, int page, int w,
                                                         int warps) {
    if (!q.n_nodes) return;
    const int lane = threadIdx.x & 31;
    const int per = a.D * (a.d_f16 ? 2 : 4) / 16;  // 16-byte pieces of a row
    for (int e = w; e < a.S * q.N; e += warps) {
        const int s = e / q.N, i = e % q.N;
        int past, n;
        seq_lengths(q, s, page, past, n);
        if (i < n) continue;
        char *d = a.dst + i * a.d_nb2 + s * a.d_nb3;
        for (int x = lane; x < a.H * per; x += 32)
            *reinterpret_cast<uint4 *>(d + (x / per) * a.d_nb1 + (x % per) * 16) = make_uint4(0, 0, 0, 0);
    }
}

// Four values of an output row at column c (a multiple of 4).
static __device__ __forceinline__ void tree_store4(const TreeAttn &a, int s, int h, int i, int c, float4 v) {
    char *d = a.dst + h * a.d_nb1 + i * a.d_nb2 + s * a.d_nb3;
    if (a.d_f16) {
        const __half2 x = __floats2half2_rn(v.x, v.y), y = __floats2half2_rn(v.z, v.w);
        uint2 pk;
        pk.x = *reinterpret_cast<const uint32_t *>(&x);
        pk.y = *reinterpret_cast<const uint32_t *>(&y);
        *reinterpret_cast<uint2 *>(d + c * 2) = pk;
    } else {
        *reinterpret_cast<float4 *>(d + c * 4) = v;
    }
}

// What the finite arithmetic of the tensor cores leaves out: V values that are infinite or NaN
// in the units with nodes are taken as zero there (a zero weight would still make NaN of them)
// and come back here, for the rows that see them.
static __device__ __noinline__ float4 tree_nonfinite4(const TreeAttn &a, const KvPages &p, const KvSeqs &q, const TreeSeg &g,
                                                      int node, int c, float4 o) {
    for (int t = max(g.k0, g.past / TREE_BKV) * TREE_BKV; t < min(g.k1 * TREE_BKV, g.T); ++t) {
        if (!tree_sees(a, g, node, t)) continue;
        const int pg = q.table[g.s * q.table_ld + t / p.page];
        if (pg < 0 || pg >= p.n_pages) continue;
        const char *v = p.v + pg * p.v_nb3 + g.hk * p.v_nb2 + t % p.page * p.v_nb1;
        for (int x = 0; x < 4; ++x) {
            const float y = __half2float(reinterpret_cast<const __half *>(v)[c + x]);
            if (!isfinite(y)) (x == 0 ? o.x : x == 1 ? o.y : x == 2 ? o.z : o.w) += y;
        }
    }
    return o;
}

// Two f32 in one register pair: one instruction for both.
typedef unsigned long long f32x2;
static __device__ __forceinline__ f32x2 pack2(float x, float y) {
    f32x2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
static __device__ __forceinline__ float2 unpack2(f32x2 v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
static __device__ __forceinline__ f32x2 fma2(f32x2 x, f32x2 y, f32x2 z) {
    f32x2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(x), "l"(y), "l"(z));
    return r;
}
static __device__ __forceinline__ f32x2 add2(f32x2 x, f32x2 y) {
    f32x2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
    return r;
}
static __device__ __forceinline__ f32x2 mul2(f32x2 x, f32x2 y) {
    f32x2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
    return r;
}

// x = hi + lo, both f16: 22 bits of an f32
static __device__ __forceinline__ void tree_split2(float x, float y, uint32_t &hi, uint32_t &lo) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
    hi = *reinterpret_cast<const uint32_t *>(&h);
    lo = *reinterpret_cast<const uint32_t *>(&l);
}

// An item that CTAs c0 .. c1 share, left by c0 for the join: its rows from `row` on (`live` of
// them), and where c0's part is (the others are in slots 2 c).  live = 0: nothing to join.
struct TreeJoin {
    int c1, slot, s, hk, row, live;
};

// Its parts joined at row r and the four columns from 4 ch: a part is R rows of D sums, then R
// pairs (maximum, sum of weights).
template <int U>  // parts loaded before any is used
static __device__ __forceinline__ float4 tree_join4(const float *parts, int R, int D, int c0, int c1, int slot, int r, int ch) {
    float M = TREE_NONE, L = 0.0f;
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int x = c0; x <= c1; x += U) {
        float2 ml[U];
        float4 y[U];
#pragma unroll
        for (int i = 0; i < U; ++i) {
            ml[i] = make_float2(M, 0.0f);
            y[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (x + i <= c1) {
                const float *pt = parts + (int64_t)(x + i == c0 ? slot : 2 * (x + i)) * (R * (D + 2));
                ml[i] = __ldcg(reinterpret_cast<const float2 *>(pt + R * D) + r);
                y[i] = __ldcg(reinterpret_cast<const float4 *>(pt + r * D) + ch);
            }
        }
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const float m = fmaxf(M, ml[i].x), f = tree_exp2(M - m), k = tree_exp2(ml[i].x - m);
            L = fmaf(L, f, ml[i].y * k);
            v.x = fmaf(v.x, f, y[i].x * k); v.y = fmaf(v.y, f, y[i].y * k);
            v.z = fmaf(v.z, f, y[i].z * k); v.w = fmaf(v.w, f, y[i].w * k);
            M = m;
        }
    }
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    return make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
}

// The same for weights up to 2^15, the upper half cut at 11 bits instead of rounded (exact as f16
// from 2^-14 on; below that the halves keep 2^-25, against a largest weight of 2^7).
static __device__ __forceinline__ void tree_cut2(f32x2 w, uint32_t &hi, uint32_t &lo) {
    const f32x2 h = w & 0xFFFFE000FFFFE000ull;
    const float2 x = unpack2(h), y = unpack2(fma2(h, pack2(-1.0f, -1.0f), w));
    const __half2 a = __floats2half2_rn(x.x, x.y), b = __floats2half2_rn(y.x, y.y);
    hi = *reinterpret_cast<const uint32_t *>(&a);
    lo = *reinterpret_cast<const uint32_t *>(&b);
}

// 4-D tensor map over pages [D, page, H_kv, n_pages]: boxes of 64 values x `rows` positions,
// 128-byte swizzle (kernels read pages of id n_pages, all out of range, as zeros)
bool tree_page_map(CUtensorMap *map, const char *base, int64_t nb1, int64_t nb2, int64_t nb3, int D, int page, int HKV,
                   int n_pages, int rows);

static __device__ __forceinline__ void tma_load_4d(void *smem_dst, const CUtensorMap *map, uint64_t *bar, int x, int y, int z,
                                                   int w, uint64_t policy) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%3, %4, %5, "
        "%6}], [%2], %7;" ::"r"(smem_u32(smem_dst)),
        "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w), "l"(policy)
        : "memory");
}
// K and V that only one tile of rows reads go through L2 first out: what every call starts with --
// its code, lengths, page tables, queries -- stays (16 trees of 61 nodes 149 -> 112 us, two caches of
// 30000 positions 36 -> 32.7).  What several tiles read is kept as usual.
static __device__ __forceinline__ uint64_t tree_policy(bool once) {
    uint64_t p;
    if (once) asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
    else asm volatile("createpolicy.fractional.L2::evict_unchanged.b64 %0, 1.0;" : "=l"(p));
    return p;
}

constexpr float TREE_EXP = 7.0f;    // weight of the reference maximum: 2^7
constexpr float TREE_MOST = 15.0f;  // weights up to 2^15 stay below f16's 65504

// K-major operand, 128-byte swizzle: sw128_desc.  M- or N-major operand in the same swizzle
// (64 values of M contiguous per position): 8-position groups 1024 bytes apart, 64-value blocks
// `block` bytes apart.
static __device__ __forceinline__ uint64_t mn_sw128_desc(uint32_t addr, uint32_t block) {
    uint64_t d = 0;
    d |= (uint64_t)((addr >> 4) & 0x3FFFu);
    d |= (uint64_t)(block >> 4) << 16;
    d |= (uint64_t)(1024u >> 4) << 32;
    d |= (uint64_t)1u << 46;
    d |= (uint64_t)2u << 61;
    return d;
}
static __device__ __forceinline__ bool elect_one() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r != 0;
}
// N columns of this warp's 32 lanes (16 at a time, one wait)
template <int N>
static __device__ __forceinline__ void tmem_load(uint32_t addr, f32x2 (&v)[N / 2]) {
    uint32_t r[N / 16][16];
#pragma unroll
    for (int x = 0; x < N / 16; ++x) tmem_ld16(addr + 16 * x, r[x]);
    // the first wait is for all; the others keep the uses of their registers behind it
#pragma unroll
    for (int x = 0; x < N / 16; ++x) tmem_ld_wait(r[x]);
#pragma unroll
    for (int x = 0; x < N / 2; ++x) v[x] = pack2(__uint_as_float(r[x / 8][2 * (x % 8)]), __uint_as_float(r[x / 8][2 * (x % 8) + 1]));
}
// any of the group's 128 threads
static __device__ __forceinline__ bool group_any(int id, bool x) {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %2, 0;\n\t"
        "barrier.cta.red.or.pred q, %1, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(r)
        : "r"(id), "r"((uint32_t)x)
        : "memory");
    return r != 0;
}
static __device__ __forceinline__ void group_sync(int id, int threads) {
    asm volatile("barrier.cta.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}
static __device__ __forceinline__ float warp_max_f32(float x) {
    float r;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(x));
    return r;
}
// The TMA warp's work: per segment K0, then K(j+1) and V(j), tiles of 128 positions through a ring
// of NS slots.  A tile is one box per run of positions within a page and 64 values of D; lane =
// (box, half of D).  Then the padding rows, and the end of all copies.
template <int D, int NS>
static __device__ __forceinline__ void tree_stream(const CUtensorMap *tm_k, const CUtensorMap *tm_v, const TreeAttn &a,
                                                   const KvPages &p, const KvSeqs &sq, const TreeUnits &w, TreeSeg g, int R,
                                                   int u0, int u1, int box, uint8_t *ring, uint64_t *full, uint64_t *empty,
                                                   volatile int *abort_flag, int *err) {
    constexpr int HALVES = D / 64, HALF = TREE_BKV * 128, TILE = HALF * HALVES;
    const int lane = threadIdx.x & 31, b = lane / HALVES, half = lane % HALVES;
    const bool mine = b < TREE_BKV / box;
    const uint64_t policy = tree_policy((int64_t)sq.N * a.group.d <= R);
    int q = 0;  // tiles issued
    bool ok = true;
    for (int u = u0; u < u1;) {
        if (u != u0) g = tree_locate(a, sq, w, p.page, R, u, u1);
        if (g.k0 == g.k1) break;
        const int *row = sq.table + g.s * sq.table_ld;
        auto page_of = [&](int k) {  // positions past the end read page n_pages: zeros
            const int t = k * TREE_BKV + b * box;
            int pg = p.n_pages;
            if (mine && t < g.T) {
                pg = __ldg(row + a.page(t));
                if (pg < 0 || pg >= p.n_pages) {
                    atomicOr(err, ERR_BAD_INDEX);
                    pg = p.n_pages;
                }
            }
            return pg;
        };
        auto issue = [&](const CUtensorMap *map, int k, int pg) {
            const int slot = q % NS, t = k * TREE_BKV + b * box;
            ok = ok && mbar_wait(&empty[slot], (uint32_t)(q / NS & 1) ^ 1u, abort_flag, err);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) return;
            if (lane == 0) mbar_arrive_expect_tx(&full[slot], TILE);
            __syncwarp();
            if (mine)
                tma_load_4d(ring + slot * TILE + half * HALF + b * box * 128, map, &full[slot], 64 * half,
                            t - a.page(t) * p.page, g.hk, pg, policy);
            __syncwarp();
            ++q;
        };
        int pg = page_of(g.k0);
        issue(tm_k, g.k0, pg);
        for (int k = g.k0; k < g.k1; ++k) {
            const int next = k + 1 < g.k1 ? page_of(k + 1) : 0;
            if (k + 1 < g.k1) issue(tm_k, k + 1, next);
            issue(tm_v, k, pg);
            pg = next;
        }
        u = g.next;
    }
    tree_zero_padding(a, sq, p.page, blockIdx.x, gridDim.x);
    // every copy lands before the block ends, also when the others gave up
    for (int i = max(0, q - NS); i < q; ++i) {
        const long long t0 = clock64();
        while (!mbar_try_wait(&full[i % NS], (uint32_t)(i / NS & 1)) && clock64() - t0 < kMbarWaitLimit) {
        }
    }
}

// Row `r` (a position) of a V tile: values that are infinite or NaN would make NaN of zero weights,
// so they become zeros, and tree_nonfinite4 adds the visible ones at the end.  True if there were any.
template <int D>
static __device__ __forceinline__ bool tree_clean_v(uint8_t *tile, int r) {
    constexpr int HALF = TREE_BKV * 128;
    uint32_t any = 0;
#pragma unroll
    for (int ch = 0; ch < D / 8; ++ch) {
        const uint4 v = *reinterpret_cast<const uint4 *>(tile + (ch >> 3) * HALF + sw128_off(r, ch & 7));
        any |= ((v.x & 0x7C007C00u) + 0x04000400u) | ((v.y & 0x7C007C00u) + 0x04000400u) |
               ((v.z & 0x7C007C00u) + 0x04000400u) | ((v.w & 0x7C007C00u) + 0x04000400u);
    }
    if (!(any & 0x80008000u)) return false;  // no exponent of all ones
    for (int ch = 0; ch < D / 8; ++ch) {
        uint32_t *v = reinterpret_cast<uint32_t *>(tile + (ch >> 3) * HALF + sw128_off(r, ch & 7));
        for (int x = 0; x < 4; ++x) v[x] &= ~__vcmpeq2(v[x] & 0x7C007C00u, 0x7C007C00u);
    }
    return true;
}

// RW rows of a tile's queries (from row0 on, `live` of them real) as 16-bit K-major operands: f16
// queries as they are, f32 ones times the scale and cut into hi and lo, lo R rows after hi, each row
// times a power of two that brings its largest value to 2^8 (its own: a row of huge or infinite values
// is no other row's business).  One group of 128 threads.  The products times the returned factor
// (f16), or times the row's factor[] (f32: a power of two, so exactly), are scores in powers of two;
// neither is ever zero, so that -inf stays -inf.
template <int D, int RW, int R, bool QF16>
static __device__ __forceinline__ float tree_load_q(const TreeAttn &a, const TreeSeg &g, int row0, int live, float scale,
                                                    uint8_t *qs, int qhalf, float *factor) {
    const int tid = threadIdx.x & 127, lane = tid & 31, G = a.group.d;
    const float c = scale * 1.4426950408889634f;
    auto q_row = [&](int r) -> const char * {
        const int gr = g.rt * R + row0 + r, node = a.group(gr);
        return a.q + node * a.q_nb1 + (g.hk * G + gr - node * G) * a.q_nb2 + g.s * a.q_nb3;
    };
    // short loops: at the start of a call the code itself comes from far away
    if constexpr (QF16) {
        const uint32_t flip = scale < 0.0f ? 0x80008000u : 0u;  // a negative scale turns the queries
#pragma unroll 4
        for (int e = tid; e < RW * (D / 8); e += 128) {
            const int r = e / (D / 8), ch = e % (D / 8);
            uint4 v = make_uint4(0, 0, 0, 0);
            if (r < live) v = *reinterpret_cast<const uint4 *>(q_row(r) + 16 * ch);
            *reinterpret_cast<uint4 *>(qs + (ch >> 3) * qhalf + sw128_off(row0 + r, ch & 7)) =
                make_uint4(v.x ^ flip, v.y ^ flip, v.z ^ flip, v.w ^ flip);
        }
        return fmaxf(fabsf(c), FLT_MIN);
    } else {
        // rows of a lane under way at once (32 trees of 43 nodes, no committed positions, 38.5 us one after
        // the other, 32.1 with four, 31.0 with eight)
        constexpr int B = RW * (D / 4) / 128 < 8 ? RW * (D / 4) / 128 : 8;
        static_assert(RW * (D / 4) % (128 * B) == 0, "whole rounds");
#pragma unroll 1
        for (int e0 = tid; e0 < RW * (D / 4); e0 += 128 * B) {  // a warp has one row, or two of D = 64
            float4 v[B];
#pragma unroll
            for (int b = 0; b < B; ++b) {
                const int r = (e0 + 128 * b) / (D / 4), ch = e0 % (D / 4);
                v[b] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (r < live) v[b] = *reinterpret_cast<const float4 *>(q_row(r) + 16 * ch);
            }
#pragma unroll
            for (int b = 0; b < B; ++b) {
                const int r = (e0 + 128 * b) / (D / 4), ch = e0 % (D / 4);
                const float4 z = make_float4(v[b].x * c, v[b].y * c, v[b].z * c, v[b].w * c);
                float m = fmaxf(fmaxf(fabsf(z.x), fabsf(z.y)), fmaxf(fabsf(z.z), fabsf(z.w)));
                if (D == 128) {
                    m = warp_max_f32(m);
                } else {
                    const float m0 = warp_max_f32(lane < 16 ? m : 0.0f), m1 = warp_max_f32(lane < 16 ? 0.0f : m);
                    m = lane < 16 ? m0 : m1;
                }
                // 2^(8 - e2) and its inverse, both in the normal range
                const int e2 = min(max((int)(__float_as_uint(m) >> 23) - 127, -100), 127);
                const float up = __uint_as_float((uint32_t)(127 + 8 - e2) << 23);
                uint2 hi, lo;
                tree_split2(z.x * up, z.y * up, hi.x, lo.x);
                tree_split2(z.z * up, z.w * up, hi.y, lo.y);
                uint8_t *half = qs + (ch >> 4) * qhalf + 8 * (ch & 1);
                *reinterpret_cast<uint2 *>(half + sw128_off(row0 + r, ch >> 1 & 7)) = hi;
                *reinterpret_cast<uint2 *>(half + sw128_off(R + row0 + r, ch >> 1 & 7)) = lo;
                if (ch == 0) factor[r] = __uint_as_float((uint32_t)(127 + e2 - 8) << 23);
            }
        }
    }
    return 1.0f;
}

// host: the launch that the two kernels share (fattn_tree.cu)
struct TreeLaunch {
    CUtensorMap k, v;
    int box, grid;
    float *parts;
    TreeJoin *joins;
};
int tree_prepare(oasr_backend *be, TreeAttn &a, const KvPages &p, const KvSeqs &s, int R, int ctas_per_sm, TreeLaunch *out);
int tree_join(oasr_backend *be, const TreeAttn &a, const KvPages &p, const KvSeqs &s, int R, const TreeLaunch &l);
// tiles of 128 rows (fattn_tree_wide.cu)
int launch_tree_wide(oasr_backend *be, const TreeAttn &a, const KvPages &p, const KvSeqs &s);

}  // namespace oasr
