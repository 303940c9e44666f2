// attn_weights.cu -- the attention that every cached position gets, added up (for kv_evict.cu).
//
// With s_r(p) = scale q_r . k_p the score of query row r (a node and one of the query heads of the K/V head) at
// position p,
//   w(p) = decay w(p) + sum over the rows that see p of exp(s_r(p) - m_r) / l_r,
// m_r and l_r the maximum and the sum over what row r sees.
#include <cooperative_groups.h>

#include <algorithm>

#include "mma_frag.cuh"
#include "once_per_device.h"
#include "op_checks.cuh"
#include "pages.cuh"

using namespace oasr;

namespace {

struct Weights {
    const char *q;
    int64_t q_nb1, q_nb2, q_nb3;  // node, head, sequence
    char *w;                      // [page, H_kv, n_pages] f32
    int64_t w_nb1, w_nb2;         // head, page
    int S, HKV, G, cs;            // sequences, K/V heads, query heads of each, CTAs per cluster
    int cr, band;                 // of attn_weights_wide_kernel: CTAs over the rows, rows of a group
    int stretch;                  // positions whose scores shared memory holds at a time (a multiple of 16); of the
                                  // wide kernel the scores and sums that it holds
    int stride;                   // scores of a position there
    float scale, decay;
};

constexpr int WT = 256, WW = WT / 32;  // threads, warps
constexpr int WTILE = 16;              // positions of a warp's tile
constexpr int WEIGHTS_MOST = 1 << 30;  // positions of a sequence, so that steps past them stay in 32 bits
constexpr int WPAGES = 520;            // pages of a stretch: of 8 positions and more

__device__ __forceinline__ uint4 stream(const void *p) {
    const int4 v = ldg_stream(p);
    return make_uint4(v.x, v.y, v.z, v.w);
}

// (m, l) of two sets of positions to that of both; m = -inf: nothing seen
__device__ __forceinline__ void join(float &m, float &l, float om, float ol) {
    const float mm = fmaxf(m, om), z = mm == -INFINITY ? 0.0f : mm;
    l = l * tree_exp2(m - z) + ol * tree_exp2(om - z);
    m = mm;
}

// 8 rows of queries per block, in the layout of the product's second operand: lane (g, t) has of row g the
// values 32 c + 8 t .. + 7 of each run c of 32, the first four for one product of depth 16 and the others
// for the next; a K row is read the same way, 16 bytes per lane, so that it goes from memory to registers
// without shared memory.  f32 queries are scaled by a power of two per row and split into two f16 halves: 22 of
// the 24 bits of a row's greatest value, fewer of its small ones, in two products instead of three.
template <int D, bool QF16>
struct Block {
    static constexpr int C = D / 32;
    uint4 hi[C], lo[QF16 ? 1 : C];
    float factor;  // of row g's scores, with log2 e
};

template <int D, bool QF16>
__device__ __forceinline__ Block<D, QF16> load_block(const Weights &a, const FastDiv &group, int r, int rows, int hk, int s) {
    constexpr int C = D / 32;
    const int t = threadIdx.x & 3;
    const int i = group(min(r, rows - 1)), h = hk * a.G + min(r, rows - 1) - i * a.G;
    const char *row = a.q + i * a.q_nb1 + h * a.q_nb2 + s * a.q_nb3;
    Block<D, QF16> q;
    q.factor = a.scale * 1.4426950408889634f;
    if (QF16) {
#pragma unroll
        for (int c = 0; c < C; ++c)
            q.hi[c] = r < rows ? *reinterpret_cast<const uint4 *>(row + 64 * c + 16 * t) : make_uint4(0, 0, 0, 0);
        return q;
    }
    float v[C][8], most = 0.0f;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int e = 0; e < 8; e += 4) {
            const float4 x = r < rows ? *reinterpret_cast<const float4 *>(row + 128 * c + 32 * t + 4 * e) : make_float4(0, 0, 0, 0);
            v[c][e] = x.x, v[c][e + 1] = x.y, v[c][e + 2] = x.z, v[c][e + 3] = x.w;
#pragma unroll
            for (int k = e; k < e + 4; ++k) most = fmaxf(most, fabsf(v[c][k]));
        }
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
    // 2^up brings the greatest value to [2^9, 2^10): two halves of 11 bits have 22 of its bits
    const int up = most > 0.0f && most < INFINITY ? max(-120, min(100, 9 - ilogbf(most))) : 0;
    const float m = __int_as_float((127 + up) << 23);
    q.factor *= __int_as_float((127 - up) << 23);
#pragma unroll
    for (int c = 0; c < C; ++c) {
        __half2 hh[4], ll[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float x = v[c][2 * e] * m, y = v[c][2 * e + 1] * m;
            hh[e] = __floats2half2_rn(x, y);
            ll[e] = __floats2half2_rn(x - __low2float(hh[e]), y - __high2float(hh[e]));
        }
        q.hi[c] = *reinterpret_cast<uint4 *>(hh);
        q.lo[QF16 ? 0 : c] = *reinterpret_cast<uint4 *>(ll);
    }
    return q;
}

// Sequence o of the call, the longest first (up to 32 of them), so that none of them starts when the others end.
__device__ __forceinline__ int sequence_of(const Weights &a, const KvSeqs &sq, int o) {
    if (a.S == 1 || a.S > 32) return o;
    const int lane = threadIdx.x & 31, own = lane < a.S ? sq.n_past[lane] : INT32_MIN;
    int before = 0;
    for (int j = 0; j < a.S; ++j) {
        const int other = __shfl_sync(0xffffffffu, own, j);
        before += other > own || (other == own && j < lane);
    }
    return __ffs(__ballot_sync(0xffffffffu, lane < a.S && before == o)) - 1;
}

// One cluster per (sequence, K/V head); its CTAs share out the positions.  A CTA goes through its own in
// stretches whose scores its shared memory holds: a warp multiplies 16 positions at a time with the rows and
// keeps m and l of every row.  The CTAs exchange those; then a thread takes a position and turns its scores
// into a weight, first of the last stretch, whose scores are still there, then of the others, computed
// again.  Every position belongs to one thread: the sums have one order, and the call needs no workspace.
// For up to 16 rows, whose queries stay in registers (24 of 64 values; the kernel below takes 18.5 us where
// this one takes 24.6 with 20 rows of 128 values at 0 to 1490 positions, and 24.2 to 18.5 with 12 rows of 64
// at 3454 to 6908).  Long caches are bound by HBM while a CTA multiplies (27000 of the 40000 cycles of each of
// 512 CTAs, two per SM: 16 sequences of 4001 to 8190 positions take 47 to 49 us, 4.3 TB/s); the rest is the start,
// the exchange (2800) and the weights (4200).  Short calls are a chain of five round trips: 6.3 us for one
// token.  K fetched to L2 ahead took 56 us, three CTAs per SM 51, every warp's m and l sent to every CTA 68.
template <int D, int NB, bool QF16>
__global__ void __launch_bounds__(WT, 2) attn_weights_kernel(Weights a, KvPages p, KvSeqs sq, FastDiv page, FastDiv group, int *err) {
    namespace cg = cooperative_groups;
    constexpr int C = D / 32, RB = 8 * NB;
    extern __shared__ float s_scores[];  // [position][stride]
    __shared__ float2 s_ml[16][RB], s_warp[WW][RB], s_row[RB];
    __shared__ int s_page[WPAGES];
    griddep_launch_dependents();
    griddep_wait();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int item = blockIdx.x / a.cs, rank = blockIdx.x % a.cs, hk = item % a.HKV, s = sequence_of(a, sq, item / a.HKV);
    int past, n;
    const bool fits = seq_lengths(sq, s, p.page, past, n) && past <= WEIGHTS_MOST - n;
    if (!fits && rank == 0 && tid == 0) atomicOr(err, ERR_BAD_INDEX);
    if (n == 0 || !fits) return;
    if (a.cs > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    const int T = past + n, tiles = (T + WTILE - 1) / WTILE;
    const int per = (tiles + a.cs - 1) / a.cs * WTILE;  // positions of a CTA
    const int p0 = (int)min((int64_t)rank * per, (int64_t)T), p1 = min(p0 + per, T);
    const int stretches = max(1, (p1 - p0 + a.stretch - 1) / a.stretch);
    const int *table = sq.table + s * sq.table_ld;
    const char *kh = p.k + hk * p.k_nb2;
    char *wh = a.w + hk * a.w_nb1;
    const int rows = n * a.G;

    int first_page = 0;
    auto pages_of = [&](int b0, int b1) {  // the pages of positions [b0, b1), -1 for what is none
        if (b0 >= b1) return;
        first_page = page(b0);
        const int last = page(b1 - 1);
        for (int j = first_page + tid; j <= last; j += WT) {
            const int pg = table[j];
            const bool is = pg >= 0 && pg < p.n_pages;
            if (!is) atomicOr(err, ERR_BAD_INDEX);
            s_page[j - first_page] = is ? pg : -1;
        }
        __syncthreads();
    };
    auto load_k = [&](uint4 (&k)[2][C], int at, int end) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int p8 = min(at + 8 * h, end - 1), j = page(p8), pg = s_page[j - first_page];
            const bool there = pg >= 0 && at + 8 * h + g < end;
            const char *row = kh + pg * p.k_nb3 + (int64_t)(at + 8 * h + g - j * p.page) * p.k_nb1 + 16 * t;
#pragma unroll
            for (int c = 0; c < C; ++c)
                k[h][c] = there ? stream(row + 64 * c) : make_uint4(0, 0, 0, 0);
        }
    };
    Block<D, QF16> q[NB];
    float2 factor[NB];  // of this lane's columns of the product: rows 2 t, 2 t + 1 of the block
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        q[b] = load_block<D, QF16>(a, group, 8 * b + g, rows, hk, s);
        factor[b] = make_float2(__shfl_sync(0xffffffffu, q[b].factor, 8 * t), __shfl_sync(0xffffffffu, q[b].factor, 8 * t + 4));
    }
    float m[NB][2], l[NB][2];
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int e = 0; e < 2; ++e) m[b][e] = -INFINITY, l[b][e] = 0.0f;
    // a stretch: its scores, with what they do to m and l; then, from the last one back, its weights
    for (int step = 0; step < 2 * stretches - 1; ++step) {
        const bool stats = step < stretches;
        const int i = stats ? step : 2 * stretches - 2 - step;
        const int b0 = p0 + i * a.stretch, b1 = min(b0 + a.stretch, p1);
        if (stretches > 1 || step == 0) pages_of(b0, b1);
        uint4 next[2][C];
        if (b0 + warp * WTILE < b1) load_k(next, b0 + warp * WTILE, b1);
        for (int at = b0 + warp * WTILE; at < b1; at += WW * WTILE) {
            uint4 k[2][C];
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int c = 0; c < C; ++c) k[h][c] = next[h][c];
            if (at + WW * WTILE < b1) load_k(next, at + WW * WTILE, b1);
            const bool edge = at + WTILE - 1 > past;  // some rows do not see all of it
            float *to = s_scores + (at - b0 + g) * a.stride + 2 * t;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                float c4[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    if (!QF16) {
                        const uint4 lo = q[b].lo[QF16 ? 0 : c];
                        mma_f16_16816_add(c4, k[0][c].x, k[1][c].x, k[0][c].y, k[1][c].y, lo.x, lo.y);
                        mma_f16_16816_add(c4, k[0][c].z, k[1][c].z, k[0][c].w, k[1][c].w, lo.z, lo.w);
                    }
                    const uint4 hi = q[b].hi[c];
                    mma_f16_16816_add(c4, k[0][c].x, k[1][c].x, k[0][c].y, k[1][c].y, hi.x, hi.y);
                    mma_f16_16816_add(c4, k[0][c].z, k[1][c].z, k[0][c].w, k[1][c].w, hi.z, hi.w);
                }
                const float2 f = factor[b];
                c4[0] *= f.x, c4[1] *= f.y, c4[2] *= f.x, c4[3] *= f.y;
                if (edge) {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (at + g + 8 * (e >> 1) > past + group(min(8 * b + 2 * t + (e & 1), rows - 1))) c4[e] = -INFINITY;
                }
                if (8 * b + 2 * t < rows) {
                    *reinterpret_cast<float2 *>(to + 8 * b) = make_float2(c4[0], c4[1]);
                    *reinterpret_cast<float2 *>(to + 8 * b + 8 * a.stride) = make_float2(c4[2], c4[3]);
                }
                if (stats) {
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float mm = fmaxf(m[b][e], fmaxf(c4[e], c4[e + 2])), z = mm == -INFINITY ? 0.0f : mm;
                        l[b][e] = l[b][e] * tree_exp2(m[b][e] - z) + tree_exp2(c4[e] - z) + tree_exp2(c4[e + 2] - z);
                        m[b][e] = mm;
                    }
                }
            }
        }
        if (step == stretches - 1) {  // the rows' m and l: over the lanes, the warps, the CTAs
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
#pragma unroll
                    for (int o = 4; o < 32; o <<= 1)
                        join(m[b][e], l[b][e], __shfl_xor_sync(0xffffffffu, m[b][e], o), __shfl_xor_sync(0xffffffffu, l[b][e], o));
                    if (g == 0) s_warp[warp][8 * b + 2 * t + e] = make_float2(m[b][e], l[b][e]);
                }
            __syncthreads();
            if (a.cs > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // all CTAs have started
            if (tid < RB) {
                float2 x = s_warp[0][tid];
#pragma unroll
                for (int w = 1; w < WW; ++w) join(x.x, x.y, s_warp[w][tid].x, s_warp[w][tid].y);
                if (a.cs == 1) {
                    s_ml[0][tid] = x;
                } else {
                    cg::cluster_group cl = cg::this_cluster();
                    for (int c = 0; c < a.cs; ++c) *cl.map_shared_rank(&s_ml[rank][tid], c) = x;
                }
            }
            if (a.cs == 1) __syncthreads();
            else cg::this_cluster().sync();
            if (tid < RB) {
                float2 x = s_ml[0][tid];
                for (int c = 1; c < a.cs; ++c) join(x.x, x.y, s_ml[c][tid].x, s_ml[c][tid].y);
                // 1 / l: 0 where all scores are -inf; NaN stays
                const bool none = x.x == -INFINITY && x.y == x.y;
                s_row[tid] = make_float2(x.x == -INFINITY ? 0.0f : x.x, none ? 0.0f : 1.0f / x.y);
            }
        }
        __syncthreads();
        if (step < stretches - 1) continue;
        constexpr int U = 4;  // positions of a thread with their old weights under way
        for (int base = b0 + tid; base < b1; base += U * WT) {
            float *to[U], old[U], sum[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int at = base + u * WT;
                const int j = page(min(at, b1 - 1)), pg = s_page[j - first_page];
                to[u] = at < b1 && pg >= 0 ? reinterpret_cast<float *>(wh + pg * a.w_nb2) + (at - j * p.page) : nullptr;
                old[u] = to[u] && a.decay != 0.0f && at < past ? *to[u] : 0.0f;
                sum[u] = 0.0f;
            }
#pragma unroll 2
            for (int r = 0; r < rows; r += 2) {
                const float2 x = s_row[r], y = s_row[r + 1];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int at = min(base + u * WT, b1 - 1);
                    const float2 v = *reinterpret_cast<const float2 *>(s_scores + (at - b0) * a.stride + r);
                    // the first row that sees the position: what it does not see a row that is NaN does not reach
                    const int seen = at > past ? (at - past) * a.G : 0;
                    if (r >= seen) sum[u] += tree_exp2(v.x - x.x) * x.y;
                    if (r + 1 >= seen && r + 1 < rows) sum[u] += tree_exp2(v.y - y.x) * y.y;
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (to[u]) *to[u] = a.decay * old[u] + sum[u];
        }
        __syncthreads();  // the scores are written again
    }
}

// More rows: groups of up to 8 NB, their queries in shared memory.  A tile of K, in registers, is multiplied
// with the blocks of a group, two at a time, for m and l of the rows; then the warp that did so turns its scores
// into weights, which add up in registers.  The scores of as many tiles as there is room for stay in shared
// memory in between, those of the others are computed again.  The cluster's CTAs share out the positions (cp)
// and the groups (cr): rank = cp * its share of the groups + its share of the positions.  A CTA's weights add
// up in shared memory where they fit (always if cr > 1), and at the end those of the cr CTAs with the same
// positions are added in order, each by the CTA that has that part of the positions.
// Bound by the chain of barriers and short loops, not by a unit (issue slots 25%, the matrix and exponential
// units below 20%; 210 CTAs for 14 heads of 272 rows at 368 to 737 positions, f32: 27 us).  With
// the positions alone shared out it took 61 us there; without kept scores 32 rows of 64 values at 700 to 1468
// positions took 20.5 instead of 16.4.  The page of a tile read two tiles ahead changed nothing.
// On mma.sync, since a group has 64 rows at most and K goes to registers; hundreds of rows of long caches would
// want tiles of 128 rows on tcgen05 (four chunks of 512 rows behind 3500 positions, 16 / 8 heads of 128: f16 432 us, f32
// 653; the tree attention takes 133 for 4000).  The last 32 rows of eight such prompts, which score
// all of them, take 53 us.
template <int D, int NB, bool QF16>
__global__ void __launch_bounds__(WT, 2) attn_weights_wide_kernel(Weights a, KvPages p, KvSeqs sq, FastDiv page, FastDiv group, int *err) {
    namespace cg = cooperative_groups;
    constexpr int C = D / 32, RB = 8 * NB, PARTS = QF16 ? 1 : 2, HELD = NB * PARTS * C * 32;
    constexpr bool AHEAD = D == 64;  // the next tile of K under way
    extern __shared__ uint4 s_q[];  // the blocks [block][half][run][lane], the scores, the sums
    __shared__ float s_factor[RB];
    __shared__ int s_last[RB];  // the last position that a row sees; -1: no row
    __shared__ float2 s_ml[2][16][RB], s_warp[WW][RB];
    __shared__ float4 s_row[RB / 2];  // m and 1 / l of two rows
    griddep_launch_dependents();
    griddep_wait();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int item = blockIdx.x / a.cs, rank = blockIdx.x % a.cs, hk = item % a.HKV, s = sequence_of(a, sq, item / a.HKV);
    int past, n;
    const bool fits = seq_lengths(sq, s, p.page, past, n) && past <= WEIGHTS_MOST - n;
    if (!fits && rank == 0 && tid == 0) atomicOr(err, ERR_BAD_INDEX);
    if (n == 0 || !fits) return;
    if (a.cs > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    const int cp = a.cs / a.cr, pi = rank % cp, ri = rank / cp;
    const int T = past + n, tiles = (T + WTILE - 1) / WTILE;
    const int per = (tiles + cp - 1) / cp * WTILE;  // positions of a CTA
    const int p0 = (int)min((int64_t)pi * per, (int64_t)T), p1 = min(p0 + per, T);
    const bool held = per <= a.stretch;
    // the scores of [p0, keep) stay for the weights, the others are computed again
    const int kept = held ? (a.stretch - per) / (WTILE * RB) : 0, keep = p0 + min(kept * WTILE, per);
    float4 *s_scores = reinterpret_cast<float4 *>(s_q + HELD) + lane;  // [tile][block][lane]
    float *s_sum = reinterpret_cast<float *>(s_q + HELD) + (keep - p0) * RB;
    const int *table = sq.table + s * sq.table_ld;
    const char *kh = p.k + hk * p.k_nb2;
    char *wh = a.w + hk * a.w_nb1;
    const int rows = n * a.G, groups = (rows + a.band - 1) / a.band;

    auto page_of = [&](int at) {  // of the 8 positions from `at` on; -1: none, or not a page
        if (at >= p1) return -1;
        const int pg = table[page(at)];
        if (pg >= 0 && pg < p.n_pages) return pg;
        if (lane == 0) atomicOr(err, ERR_BAD_INDEX);
        return -1;
    };
    auto load_k = [&](uint4 (&k)[2][C], const int (&pg)[2], int at) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const bool there = pg[h] >= 0 && at + 8 * h + g < p1;
            const int off = at + 8 * h + g - page(min(at + 8 * h, T - 1)) * p.page;
            const char *row = kh + pg[h] * p.k_nb3 + off * p.k_nb1 + 16 * t;
#pragma unroll
            for (int c = 0; c < C; ++c) k[h][c] = there ? *reinterpret_cast<const uint4 *>(row + 64 * c) : make_uint4(0, 0, 0, 0);
        }
    };
    auto entry = [&](int at, int pg) {
        return reinterpret_cast<float *>(wh + pg * a.w_nb2) + (at - page(at) * p.page);
    };
    int live = 0, r0 = 0;
    // whether a tile has positions that some rows of blocks b and b + 1 do not see
    auto hides = [&](int at, int b) { return at + WTILE - 1 > past || 8 * b + 16 > live; };
    // scores of a tile with blocks b and b + 1: two chains of products (with f32 queries four)
    auto scores = [&](const uint4 (&k)[2][C], int b, int at, float (&x)[2][4]) {
        float lo[2][4];
#pragma unroll
        for (int i = 0; i < 2 && b + i < NB; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) x[i][e] = lo[i][e] = 0.0f;
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int i = 0; i < 2 && b + i < NB; ++i) {
                const uint4 hi = s_q[((b + i) * PARTS * C + c) * 32 + lane];
                mma_f16_16816_add(x[i], k[0][c].x, k[1][c].x, k[0][c].y, k[1][c].y, hi.x, hi.y);
                mma_f16_16816_add(x[i], k[0][c].z, k[1][c].z, k[0][c].w, k[1][c].w, hi.z, hi.w);
                if (!QF16) {
                    const uint4 rest = s_q[(((b + i) * PARTS + PARTS - 1) * C + c) * 32 + lane];
                    mma_f16_16816_add(lo[i], k[0][c].x, k[1][c].x, k[0][c].y, k[1][c].y, rest.x, rest.y);
                    mma_f16_16816_add(lo[i], k[0][c].z, k[1][c].z, k[0][c].w, k[1][c].w, rest.z, rest.w);
                }
            }
        const bool edge = hides(at, b);
#pragma unroll
        for (int i = 0; i < 2 && b + i < NB; ++i) {
            const int2 last = *reinterpret_cast<const int2 *>(s_last + 8 * (b + i) + 2 * t);
            const float2 f = *reinterpret_cast<const float2 *>(s_factor + 8 * (b + i) + 2 * t);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x[i][e] = (x[i][e] + lo[i][e]) * (e & 1 ? f.y : f.x);
                if (edge && at + g + 8 * (e >> 1) > (e & 1 ? last.y : last.x)) x[i][e] = -INFINITY;
            }
        }
    };
    // f(tile's first position, its pages, K) for the warp's tiles from one on
    auto each_tile = [&](int at, auto f) {
        int pg[2] = {page_of(at), page_of(at + 8)};
        uint4 next[2][C];
        if (AHEAD && at < p1) load_k(next, pg, at);
        for (; at < p1; at += WW * WTILE) {
            const int here[2] = {pg[0], pg[1]};
            uint4 k[2][C];
            if (AHEAD) {
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int c = 0; c < C; ++c) k[h][c] = next[h][c];
            } else {
                load_k(k, here, at);
            }
            pg[0] = page_of(at + WW * WTILE), pg[1] = page_of(at + WW * WTILE + 8);
            if (AHEAD && at + WW * WTILE < p1) load_k(next, pg, at + WW * WTILE);
            f(at, here, k);
        }
    };

    for (int turn = 0; turn * a.cr < groups; ++turn) {  // as often in every CTA of the cluster
        r0 = (turn * a.cr + ri) * a.band;
        live = max(0, min(a.band, rows - r0));
        for (int b = warp; 8 * b < (NB == 8 ? (live + 15) / 16 * 16 : RB); b += WW) {
            const Block<D, QF16> x = load_block<D, QF16>(a, group, r0 + 8 * b + g, rows, hk, s);
#pragma unroll
            for (int c = 0; c < C; ++c) {
                s_q[(b * PARTS * C + c) * 32 + lane] = x.hi[c];
                if (!QF16) s_q[((b * PARTS + PARTS - 1) * C + c) * 32 + lane] = x.lo[QF16 ? 0 : c];
            }
            if (t == 0) {
                const int row = 8 * b + g;
                s_factor[row] = x.factor, s_last[row] = row < live ? past + group(r0 + row) : -1;
            }
        }
        __syncthreads();
        float m[NB][2], l[NB][2];
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int e = 0; e < 2; ++e) m[b][e] = -INFINITY, l[b][e] = 0.0f;
        if (live)
            each_tile(p0 + warp * WTILE, [&](int at, const int (&)[2], const uint4 (&k)[2][C]) {
#pragma unroll
                for (int b = 0; b < NB; b += 2) {
                    if (NB == 8 && 8 * b >= live) break;
                    float x[2][4];
                    scores(k, b, at, x);
                    if (at < keep) {
#pragma unroll
                        for (int i = 0; i < 2 && b + i < NB; ++i)
                            s_scores[((at - p0) / WTILE * NB + b + i) * 32] = make_float4(x[i][0], x[i][1], x[i][2], x[i][3]);
                    }
#pragma unroll
                    for (int i = 0; i < 2 && b + i < NB; ++i)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            float &mm = m[b + i][e], &ll = l[b + i][e];
                            const float up = fmaxf(mm, fmaxf(x[i][e], x[i][e + 2])), z = up == -INFINITY ? 0.0f : up;
                            ll = ll * tree_exp2(mm - z) + tree_exp2(x[i][e] - z) + tree_exp2(x[i][e + 2] - z);
                            mm = up;
                        }
                }
            });
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            if (NB == 8 && 8 * b >= live) break;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
                for (int o = 4; o < 32; o <<= 1)
                    join(m[b][e], l[b][e], __shfl_xor_sync(0xffffffffu, m[b][e], o), __shfl_xor_sync(0xffffffffu, l[b][e], o));
                if (g == 0) s_warp[warp][8 * b + 2 * t + e] = make_float2(m[b][e], l[b][e]);
            }
        }
        __syncthreads();
        if (turn == 0 && a.cs > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // all CTAs have started
        if (tid < live) {
            float2 x = s_warp[0][tid];
#pragma unroll
            for (int w = 1; w < WW; ++w) join(x.x, x.y, s_warp[w][tid].x, s_warp[w][tid].y);
            for (int c = 0; c < cp; ++c)
                *(a.cs == 1 ? &s_ml[turn & 1][0][tid] : cg::this_cluster().map_shared_rank(&s_ml[turn & 1][pi][tid], ri * cp + c)) = x;
        }
        if (a.cs == 1) __syncthreads();
        else cg::this_cluster().sync();
        if (tid < RB) {
            float2 x = make_float2(-INFINITY, 0.0f);
            if (tid < live)
                for (int c = 0; c < cp; ++c) join(x.x, x.y, s_ml[turn & 1][c][tid].x, s_ml[turn & 1][c][tid].y);
            // 1 / l: 0 where all scores are -inf, and for rows of padding; NaN stays
            const bool none = x.x == -INFINITY && x.y == x.y;
            reinterpret_cast<float2 *>(s_row)[tid] = make_float2(x.x == -INFINITY ? 0.0f : x.x, none ? 0.0f : 1.0f / x.y);
        }
        __syncthreads();
        auto weigh = [&](int at, const int (&pg)[2], auto score) {
            float w[2] = {0.0f, 0.0f}, old[2];
            if (!held && t == 0) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int pos = at + 8 * h + g;
                    old[h] = pg[h] >= 0 && pos < p1 && (turn || (a.decay != 0.0f && pos < past)) ? *entry(pos, pg[h]) : 0.0f;
                }
            }
#pragma unroll
            for (int b = 0; b < NB; b += 2) {
                if (NB == 8 && 8 * b >= live) break;
                float x[2][4];
                score(b, x);
                const bool edge = hides(at, b);
#pragma unroll
                for (int i = 0; i < 2 && b + i < NB; ++i) {
                    const int2 last = *reinterpret_cast<const int2 *>(s_last + 8 * (b + i) + 2 * t);
                    const float4 y = s_row[4 * (b + i) + t];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float u = tree_exp2(x[i][2 * h] - y.x) * y.y, v = tree_exp2(x[i][2 * h + 1] - y.z) * y.w;
                        // what it does not see a row that is NaN does not reach
                        w[h] += edge && at + g + 8 * h > last.x ? 0.0f : u;
                        w[h] += edge && at + g + 8 * h > last.y ? 0.0f : v;
                    }
                }
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                w[h] += __shfl_xor_sync(0xffffffffu, w[h], 1);
                w[h] += __shfl_xor_sync(0xffffffffu, w[h], 2);
                const int pos = at + 8 * h + g;
                if (t || pos >= p1) continue;
                if (held) s_sum[pos - p0] = turn ? s_sum[pos - p0] + w[h] : w[h];
                else if (pg[h] >= 0) *entry(pos, pg[h]) = turn ? old[h] + w[h] : a.decay * old[h] + w[h];
            }
        };
        if (live) {
            int at = p0 + warp * WTILE;
            for (; at < min(keep, p1); at += WW * WTILE)
                weigh(at, {0, 0}, [&](int b, float (&x)[2][4]) {
#pragma unroll
                    for (int i = 0; i < 2 && b + i < NB; ++i) {
                        const float4 v = s_scores[((at - p0) / WTILE * NB + b + i) * 32];
                        x[i][0] = v.x, x[i][1] = v.y, x[i][2] = v.z, x[i][3] = v.w;
                    }
                });
            each_tile(at, [&](int at, const int (&pg)[2], const uint4 (&k)[2][C]) {
                weigh(at, pg, [&](int b, float (&x)[2][4]) { scores(k, b, at, x); });
            });
        }
        __syncthreads();  // the queries and the rows' m and l are written again
    }
    if (!held) return;  // (then a.cr is 1)
    if (a.cr > 1) cg::this_cluster().sync();
    // the sums of all groups to the entries: this CTA's part of the positions
    const int part = (p1 - p0 + a.cr - 1) / a.cr, s0 = min(ri * part, p1 - p0), s1 = min(s0 + part, p1 - p0);
    const int others = min(a.cr, groups);  // CTAs that had a group
    for (int i = s0 + tid; i < s1; i += WT) {
        const int pos = p0 + i, pg = table[page(pos)];
        if (pg < 0 || pg >= p.n_pages) continue;
        float *to = entry(pos, pg);
        const float old = a.decay != 0.0f && pos < past ? *to : 0.0f;
        float w = 0.0f;
        for (int c = 0; c < others; ++c) w += a.cr == 1 ? s_sum[i] : *cg::this_cluster().map_shared_rank(s_sum + i, c * cp + pi);
        *to = a.decay * old + w;
    }
    if (a.cr > 1) cg::this_cluster().sync();  // until then the others read this CTA's sums
}

template <typename Kernel>
int launch_cluster(oasr_backend *be, Kernel *kernel, int64_t items, size_t smem, const Weights &a, const KvPages &p, const KvSeqs &sq) {
    if (items * a.cs > INT32_MAX) return fail_op(be, "attn_weights", "too many sequences");
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(items * a.cs));
    cfg.blockDim = dim3(WT);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = be->stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = a.cs, attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = be->pdl ? 2 : 1;
    return launched(be, cudaLaunchKernelEx(&cfg, kernel, a, p, sq, FastDiv(p.page), FastDiv(a.G), be->err_word), "attn_weights");
}

template <int D, int NB, bool QF16>
int launch_weights(oasr_backend *be, Weights a, const KvPages &p, const KvSeqs &sq, int S) {
    constexpr int SMEM = 100 << 10;  // two CTAs per SM, with what is static
    const int rows = (int)std::min<int64_t>((int64_t)sq.N * a.G, 8 * NB);
    // 8-byte accesses of neighbouring positions fall on different banks if half the stride is odd
    a.stride = (rows + 1) / 2 * 2;
    if (a.stride % 4 == 0) a.stride += 2;
    a.stretch = std::min(SMEM / (4 * a.stride) / WTILE * WTILE, (WPAGES - 2) * 8 / WTILE * WTILE);
    static OncePerDevice smem;
    cudaError_t e = (cudaError_t)smem(be->device, [] {
        return cudaFuncSetAttribute(attn_weights_kernel<D, NB, QF16>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
    });
    static OncePerDevice wide;
    if (e == cudaSuccess)
        e = (cudaError_t)wide(be->device, [] {
            return cudaFuncSetAttribute(attn_weights_kernel<D, NB, QF16>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        });
    if (e != cudaSuccess) return oasr_internal_cuda_fail(be, e, "attn_weights attribute", __LINE__);
    const int64_t items = (int64_t)S * a.HKV, most = (int64_t)sq.MP * p.page;
    // two CTAs per SM, of 128 positions (a tile per warp) at least; more where shared memory would not hold a
    // CTA's scores, since those of all stretches but the last are computed twice (128 heads of 4001 to 8190
    // positions: 120, 78, 50, 56 us with 1, 2, 4, 8 CTAs each)
    const int64_t even = std::min(2 * be->sm_count / items, (most + 127) / 128), whole = (most + a.stretch - 1) / a.stretch;
    a.cs = (int)std::max<int64_t>(1, std::min<int64_t>(16, std::max(even, whole)));
    if (a.cs > 8 && a.cs < 16) a.cs = 8;  // 24 heads of 0 to 4661 positions: 16.5 us with 12, 12.4 with 8 (32 of 9755 to 19511: 35 with 9, 39)
    const int64_t held = std::min<int64_t>(a.stretch, ((most + a.cs - 1) / a.cs + WTILE) / WTILE * WTILE);
    return launch_cluster(be, attn_weights_kernel<D, NB, QF16>, items, (size_t)held * a.stride * 4, a, p, sq);
}

template <int D, int NB, bool QF16>
int launch_wide(oasr_backend *be, Weights a, const KvPages &p, const KvSeqs &sq, int S) {
    constexpr int HELD = NB * (QF16 ? 1 : 2) * (D / 32) * 32 * 16, SMEM = (NB == 8 ? 84 : 100) << 10;  // two CTAs per SM, with what is static
    static OncePerDevice smem;
    cudaError_t e = (cudaError_t)smem(be->device, [] {
        return cudaFuncSetAttribute(attn_weights_wide_kernel<D, NB, QF16>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
    });
    static OncePerDevice wide;
    if (e == cudaSuccess)
        e = (cudaError_t)wide(be->device, [] {
            return cudaFuncSetAttribute(attn_weights_wide_kernel<D, NB, QF16>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        });
    if (e != cudaSuccess) return oasr_internal_cuda_fail(be, e, "attn_weights attribute", __LINE__);
    // up to 16 CTAs per head, two per SM: over the positions (128 each at least) and over the groups of rows.  A
    // group costs what 4 tiles do besides its tiles (lengths, queries, the exchange).  14 heads of 272 rows
    // at 368 to 737 positions take 27 us so, with up to 8 CTAs 45.
    const int64_t items = (int64_t)S * a.HKV, most = (int64_t)sq.MP * p.page, groups = ((int64_t)sq.N * a.G + 8 * NB - 1) / (8 * NB);
    const int64_t budget = std::max<int64_t>(1, std::min<int64_t>(16, 2 * be->sm_count / items));
    int64_t least = INT64_MAX;
    a.band = (int)((((int64_t)sq.N * a.G + groups - 1) / groups + 15) / 16 * 16);  // equal groups of pairs of blocks
    if (a.band > 8 * NB) a.band = 8 * NB;
    a.stretch = (SMEM - HELD) / 4;
    for (int cr = 1; cr <= std::min(budget, groups); ++cr) {
        const int64_t cp = std::max<int64_t>(1, std::min(budget / cr, (most + 127) / 128));
        if (cr > 1 && most > cp * (a.stretch - WTILE)) continue;  // its sums have to fit
        const int64_t cost = (groups + cr - 1) / cr * (4 + (most + 128 * cp - 1) / (128 * cp));
        if (cost < least) least = cost, a.cr = cr, a.cs = (int)cp * cr;
    }
    const int64_t each = ((most + a.cs / a.cr - 1) / (a.cs / a.cr) + WTILE) / WTILE * WTILE;
    a.stretch = (int)std::min<int64_t>(a.stretch, each * (8 * NB + 1));
    return launch_cluster(be, attn_weights_wide_kernel<D, NB, QF16>, items, (size_t)HELD + a.stretch * 4, a, p, sq);
}

}  // namespace

extern "C" int oasr_b200_attn_weights(oasr_backend *be, const oasr_tensor *q, const oasr_tensor *k_pages, const oasr_tensor *page_table,
                           const oasr_tensor *n_past, const oasr_tensor *n_nodes, float scale, float decay, oasr_tensor *weights) {
    const char *op = "attn_weights";
    if (!be) return oasr_internal_precheck(be);
    int st;
    if (!q) return fail_op(be, op, "null argument");
    KvPages p;
    KvSeqs sq;
    st = pages_check(be, op, k_pages, k_pages, 1, &p);
    if (st) return st;
    const int64_t D = q->ne[0], N = q->ne[1], H = q->ne[2], S = q->ne[3], HKV = k_pages->ne[2];
    if ((q->type != OASR_TYPE_F32 && q->type != OASR_TYPE_F16) || D != k_pages->ne[0] || H < 1 || H % HKV || H > 65535)
        return fail_op(be, op, "q must be F32 or F16 [D, n, H, n_seq] with H a multiple of H_kv");
    const bool f16 = q->type == OASR_TYPE_F16;
    if (q->nb[0] != (f16 ? 2 : 4)) return fail_op(be, op, "rows must be contiguous");
    if (!is_weights(weights, k_pages)) return fail_op(be, op, "weights must be F32 [page, H_kv, n_pages], rows contiguous and apart");
    if (!(scale == scale)) return fail_op(be, op, "scale must be a number");
    if (!(decay >= 0.0f && decay < INFINITY)) return fail_op(be, op, "decay must not be negative, and finite");
    if (N == 0 || S == 0) return oasr_internal_precheck(be);
    st = seqs_check(be, op, page_table, n_past, n_nodes, S, N, &sq);
    if (st) return st;
    if (N * (H / HKV) > INT32_MAX / 2) return fail_op(be, op, "too many rows");
    if (!q->data) return fail_op(be, op, "null argument");
    if (!rows16(q)) return fail_op(be, op, "rows must be 16-byte aligned");
    for (const oasr_tensor *t : {q, k_pages, page_table, n_past, n_nodes})
        if (share_bytes(weights, t)) return fail_op(be, op, "weights must not overlap an input (it is still read while they are written)");
    st = oasr_internal_precheck(be);  // the arguments need no device
    if (st) return st;
    Weights a = {};
    a.q = (const char *)q->data;
    a.q_nb1 = q->nb[1], a.q_nb2 = q->nb[2], a.q_nb3 = q->nb[3];
    a.w = (char *)weights->data, a.w_nb1 = weights->nb[1], a.w_nb2 = weights->nb[2];
    a.S = (int)S, a.HKV = (int)HKV, a.G = (int)(H / HKV);
    a.scale = scale, a.decay = decay;
    const int64_t rows = N * a.G;
#define AW(DD, NB, LAUNCH) \
    if (D == DD && rows <= 8 * NB) return f16 ? LAUNCH<DD, NB, true>(be, a, p, sq, (int)S) : LAUNCH<DD, NB, false>(be, a, p, sq, (int)S)
    AW(64, 1, launch_weights);
    AW(64, 2, launch_weights);
    AW(64, 3, launch_weights);
    AW(64, 4, launch_wide);
    AW(128, 1, launch_weights);
    AW(128, 2, launch_weights);
    AW(128, 3, launch_wide);
    AW(128, 4, launch_wide);
#undef AW
    if (D == 64) return f16 ? launch_wide<64, 8, true>(be, a, p, sq, (int)S) : launch_wide<64, 8, false>(be, a, p, sq, (int)S);
    if (D == 128) return f16 ? launch_wide<128, 8, true>(be, a, p, sq, (int)S) : launch_wide<128, 8, false>(be, a, p, sq, (int)S);
    return fail_op(be, op, "head_dim must be 64 or 128");
}
