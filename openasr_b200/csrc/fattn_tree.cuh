// fattn_tree.cuh -- what the two tree-attention kernels share: how the work is split over the
// CTAs, which nodes a row sees, and where unfinished sums wait to be joined.
//
// Work is counted in units: 64 positions of one (sequence, K/V head, tile of M rows), a row
// being one query head of one node (row = node * G + head in the group).  The lengths are in
// device memory, so every warp counts the units itself and CTA c of C takes the units
// [c T / C, (c + 1) T / C): ragged batches balance without the host knowing them, and one long
// sequence spreads over all SMs.  A CTA's range is a list of segments, each within one
// (sequence, head, tile); a segment that is not the whole of it leaves (max, sum, output) in
// the scratch, and the CTA that arrives last joins the parts in the order of the positions, so
// the bits do not depend on the order of arrival.
#pragma once

#include "pages.cuh"
#include "tc_common.cuh"

namespace oasr {

constexpr int TREE_BKV = 64;  // positions per unit

struct TreeSeg {
    int s, hk, rt;         // sequence, K/V head, row tile
    int past, n, T, kt;    // committed positions, live nodes, past + n, units of the item
    int k0, k1;            // units of this segment
    int64_t first;         // the item's first unit, counted from the call's first
};

struct TreeUnits {
    int64_t total;  // T above
    int ctas;       // C above
};

// units of sequence s
static __device__ __forceinline__ int64_t tree_seq_units(const KvSeqs &q, int s, int page, int G, int HKV, int M,
                                                         bool &ok) {
    int past, n;
    ok = seq_lengths(q, s, page, past, n);
    if (n == 0) return 0;
    return (int64_t)((n * G + M - 1) / M) * HKV * ((past + n + TREE_BKV - 1) / TREE_BKV);
}

// All warps: the call's units.  A sequence with lengths out of range counts none (reported).
static __device__ __forceinline__ int64_t tree_count(const TreeAttn &a, const KvSeqs &q, int page, int M, int *err) {
    const int lane = threadIdx.x & 31, G = a.H / a.HKV;
    int64_t sum = 0;
    for (int s = lane; s < a.S; s += 32) {
        bool ok;
        sum += tree_seq_units(q, s, page, G, a.HKV, M, ok);
        if (!ok && blockIdx.x == 0 && threadIdx.x < 32) atomicOr(err, ERR_BAD_INDEX);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    return sum;
}

// All lanes: the segment that starts at unit u (u < total) and ends before `end`.
static __device__ __forceinline__ TreeSeg tree_locate(const TreeAttn &a, const KvSeqs &q, int page, int M, int64_t u,
                                                      int64_t end) {
    const int lane = threadIdx.x & 31, G = a.H / a.HKV;
    int64_t base = 0;
    TreeSeg g = {};
    for (int s0 = 0; s0 < a.S; s0 += 32) {
        bool ok;
        const int64_t mine = s0 + lane < a.S ? tree_seq_units(q, s0 + lane, page, G, a.HKV, M, ok) : 0;
        int64_t run = mine;  // inclusive prefix sum over the lanes
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t up = __shfl_up_sync(0xffffffffu, run, o);
            if (lane >= o) run += up;
        }
        const int64_t all = __shfl_sync(0xffffffffu, run, 31);
        if (u < base + all) {
            const int l = __ffs(__ballot_sync(0xffffffffu, u < base + run)) - 1;
            g.first = __shfl_sync(0xffffffffu, base + run - mine, l);
            g.s = s0 + l;
            break;
        }
        base += all;
    }
    seq_lengths(q, g.s, page, g.past, g.n);
    g.T = g.past + g.n;
    g.kt = (g.T + TREE_BKV - 1) / TREE_BKV;
    const int rts = (g.n * G + M - 1) / M;
    const int item = (int)((u - g.first) / g.kt);
    g.hk = item / rts;
    g.rt = item % rts;
    g.first += (int64_t)item * g.kt;
    g.k0 = (int)(u - g.first);
    g.k1 = (int)min((int64_t)g.kt, end - g.first);
    return g;
}

static __device__ __forceinline__ int64_t tree_start(const TreeUnits &w, int64_t c) { return c * w.total / w.ctas; }
// the CTA whose range holds unit u
static __device__ __forceinline__ int tree_owner(const TreeUnits &w, int64_t u) {
    return (int)(((u + 1) * w.ctas - 1) / w.total);
}
// A CTA leaves at most two unfinished segments: its first (slot 2c) and its last (2c + 1).
static __device__ __forceinline__ int64_t tree_slot(const TreeUnits &w, int c, int64_t item_first) {
    return 2 * (int64_t)c + (item_first > tree_start(w, c) ? 1 : 0);
}

// Which of the positions t0 .. t0 + 31 the row of node `node` sees, as bits: all committed
// positions, and the nodes of its words (or the nodes up to itself).
static __device__ __forceinline__ uint32_t tree_sees(const TreeAttn &a, const TreeSeg &g, int node, int t0) {
    const int j = t0 - g.past;  // node number of bit 0
    if (node >= g.n || j >= g.n) return j < 0 && node < g.n ? 0xffffffffu : 0u;
    uint32_t w;
    if (!a.tree) {
        const int c = node + 1 - j;
        w = c >= 32 ? 0xffffffffu : c <= 0 ? 0u : (1u << c) - 1u;
    } else {
        const int *row = a.tree + g.s * a.t_nb2 + node * a.t_nb1;
        if (j <= -32) {
            w = 0u;
        } else if (j < 0) {
            w = (uint32_t)__ldg(row) << -j;
        } else {
            const int i = j >> 5, sh = j & 31;
            w = (uint32_t)__ldg(row + i) >> sh;
            if (sh && i + 1 < a.W) w |= (uint32_t)__ldg(row + i + 1) << (32 - sh);
        }
    }
    const int live = g.n - j;  // nodes end here
    if (live < 32) w &= (1u << live) - 1u;
    if (j < 0) w |= j <= -32 ? 0xffffffffu : (1u << -j) - 1u;
    return w;
}

// Rows of padding nodes of every sequence: zeros.  Each of the `warps` warps of the grid, this
// one being number w, takes every warps-th node.
static __device__ __forceinline__ void tree_zero_padding(const TreeAttn &a, const KvSeqs &q, int page, int64_t w,
                                                         int64_t warps) {
    if (!q.n_nodes) return;
    const int lane = threadIdx.x & 31;
    const int per = a.D * (a.d_f16 ? 2 : 4) / 16;  // 16-byte pieces of a row
    for (int64_t e = w; e < (int64_t)a.S * q.N; e += warps) {
        const int s = (int)(e / q.N), i = (int)(e % q.N);
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
    float *f = reinterpret_cast<float *>(&o);
    for (int t = max(g.k0, g.past / TREE_BKV) * TREE_BKV; t < min(g.k1 * TREE_BKV, g.T); ++t) {
        if (!(tree_sees(a, g, node, t) & 1u)) continue;
        const int pg = q.table[g.s * q.table_ld + t / p.page];
        if (pg < 0 || pg >= p.n_pages) continue;
        const __half *v =
            reinterpret_cast<const __half *>(p.v + pg * p.v_nb3 + g.hk * p.v_nb2 + t % p.page * p.v_nb1) + c;
        for (int x = 0; x < 4; ++x) {
            const float y = __half2float(v[x]);
            if (!isfinite(y)) f[x] += y;
        }
    }
    return o;
}

// 2^x, and the power of two that the weights carry: 2^15 times the weight keeps both 16-bit
// halves of a weight of 2^-20 exact to 2^-22 (f16 ends at 65504 and thins out below 2^-14).
static __device__ __forceinline__ float tree_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
constexpr float TREE_WEIGHT_EXP = 15.0f;

// x = hi + lo, both f16: 22 bits of an f32
static __device__ __forceinline__ void tree_split2(float x, float y, uint32_t &hi, uint32_t &lo) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
    hi = *reinterpret_cast<const uint32_t *>(&h);
    lo = *reinterpret_cast<const uint32_t *>(&l);
}

// 4-D tensor map over pages [D, page, H_kv, n_pages]: boxes of 64 values x `rows` positions,
// 128-byte swizzle (kernels read pages of id n_pages, all out of range, as zeros)
bool tree_page_map(CUtensorMap *map, const char *base, int64_t nb1, int64_t nb2, int64_t nb3, int D, int page, int HKV,
                   int n_pages, int rows);

static __device__ __forceinline__ void tma_load_4d(void *smem_dst, const CUtensorMap *map, uint64_t *bar, int x, int y, int z,
                                                   int w) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(
            smem_u32(smem_dst)),
        "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
        : "memory");
}

}  // namespace oasr
