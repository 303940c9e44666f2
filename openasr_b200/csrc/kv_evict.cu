// kv_evict.cu -- which positions of a paged cache to keep, by the attention that they got (kv_evict), and
// that attention added up (attn_weights).
//
// attn_weights: with s_r(p) = scale q_r . k_p the score of query row r (a node and one of the query heads of
// the K/V head) at position p,
//   w(p) = decay w(p) + sum over the rows that see p of exp(s_r(p) - m_r) / l_r,
// m_r and l_r the maximum and the sum over what row r sees.
//
// kv_evict: of a sequence's positions the first n_sink, the last n_recent, and of the others those with the
// greatest w stay, n_keep in all; their rows move to the front in their order.
#include <cooperative_groups.h>

#include "once_per_device.h"
#include "op_checks.cuh"
#include "pages.cuh"

using namespace oasr;

namespace {

// ---- attention added up -----------------------------------------------------------------------
struct Weights {
    const char *q;
    int64_t q_nb1, q_nb2, q_nb3;  // node, head, sequence
    char *w;                      // [page, H_kv, n_pages] f32
    int64_t w_nb1, w_nb2;         // head, page
    int HKV, G, cs;               // K/V heads, query heads of each, CTAs per cluster
    int cap;                      // tiles of a warp whose scores stay in shared memory
    float scale, decay;
};

constexpr int WT = 256, WW = WT / 32;  // threads, warps
constexpr int WTILE = 16;              // positions of a warp's tile

__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// (m, l) of two sets of positions to that of both; m = -inf: nothing seen
__device__ __forceinline__ void join(float &m, float &l, float om, float ol) {
    const float mm = fmaxf(m, om), z = mm == -INFINITY ? 0.0f : mm;
    l = l * ex2(m - z) + ol * ex2(om - z);
    m = mm;
}

// 8 rows of queries per block, in the layout of the product's second operand: lane (g, t) has of row g the
// values 32 c + 8 t .. + 7 of each run c of 32, the first four for one product of depth 16 and the others
// for the next; a K row is read the same way, 16 bytes per lane, so that both go from memory to registers
// without shared memory.  f32 queries are scaled by a power of two per row and split into two f16 halves.
template <int D, int NB, bool QF16>
struct Queries {
    static constexpr int C = D / 32;
    uint4 hi[NB][C], lo[QF16 ? 1 : NB][QF16 ? 1 : C];
};

// One cluster per (sequence, K/V head); its CTAs share out the positions, in tiles of 16 per warp.  The
// first pass over the tiles takes m and l of every row, which the CTAs then exchange; the second turns the
// scores, kept in shared memory or computed again, into weights.  Every position belongs to one thread:
// the sums have one order, and the call needs no workspace.
template <int D, int NB, bool QF16>
__global__ void __launch_bounds__(WT) attn_weights_kernel(Weights a, KvPages p, KvSeqs sq, FastDiv page, FastDiv group, int *err) {
    namespace cg = cooperative_groups;
    constexpr int C = D / 32, RB = 8 * NB;
    extern __shared__ float4 s_scores[];  // [tile of the warp][warp][NB][lane]
    __shared__ float2 s_ml[2][16][RB], s_warp[WW][RB], s_row[RB];
    griddep_launch_dependents();
    griddep_wait();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int item = blockIdx.x / a.cs, rank = blockIdx.x % a.cs;
    const int s = item / a.HKV, hk = item - s * a.HKV;
    int past, n;
    if (!seq_lengths(sq, s, p.page, past, n) && rank == 0 && tid == 0) atomicOr(err, ERR_BAD_INDEX);
    if (n == 0) return;
    if (a.cs > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    const int T = past + n, tiles = (T + WTILE - 1) / WTILE;
    const int per = (tiles + a.cs - 1) / a.cs;
    const int t0 = min(rank * per, tiles), t1 = min(t0 + per, tiles);
    const int *table = sq.table + s * sq.table_ld;
    const char *kh = p.k + hk * p.k_nb2;
    char *wh = a.w + hk * a.w_nb1;
    const int rows = n * a.G;

    // page and offset of the 8 positions from p8 on (a multiple of 8); -1: none, or not a page
    auto locate = [&](int p8, int &off) {
        if (p8 >= T) return -1;
        const int j = page(p8), pg = table[j];
        off = p8 - j * p.page;
        if (pg >= 0 && pg < p.n_pages) return pg;
        if (lane == 0) atomicOr(err, ERR_BAD_INDEX);
        return -1;
    };
    auto load_k = [&](uint4 (&k)[2][C], int tile) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            int off;
            const int p8 = tile * WTILE + 8 * h, pg = locate(p8, off);
            const bool there = pg >= 0 && p8 + g < T;
            const char *row = kh + pg * p.k_nb3 + (off + g) * p.k_nb1 + 16 * t;
#pragma unroll
            for (int c = 0; c < C; ++c)
                k[h][c] = there ? *reinterpret_cast<const uint4 *>(row + 64 * c) : make_uint4(0, 0, 0, 0);
        }
    };

    int parity = 0;
    for (int r0 = 0; r0 < rows; r0 += RB, parity ^= 1) {
        // the block's queries, and what their scores are multiplied by (with log2 e)
        Queries<D, NB, QF16> q;
        float factor[NB][2];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const int r = r0 + 8 * b + g, i = group(min(r, rows - 1)), h = hk * a.G + min(r, rows - 1) - i * a.G;
            const char *row = a.q + i * a.q_nb1 + h * a.q_nb2 + s * a.q_nb3;
            float f = a.scale * 1.4426950408889634f;
            if (QF16) {
#pragma unroll
                for (int c = 0; c < C; ++c)
                    q.hi[b][c] = r < rows ? *reinterpret_cast<const uint4 *>(row + 64 * c + 16 * t) : make_uint4(0, 0, 0, 0);
            } else {
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
                f = f * __int_as_float((127 - up) << 23);
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    __half2 hh[4], ll[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float x = v[c][2 * e] * m, y = v[c][2 * e + 1] * m;
                        hh[e] = __floats2half2_rn(x, y);
                        ll[e] = __floats2half2_rn(x - __low2float(hh[e]), y - __high2float(hh[e]));
                    }
                    q.hi[b][c] = *reinterpret_cast<uint4 *>(hh);
                    q.lo[b][c] = *reinterpret_cast<uint4 *>(ll);
                }
            }
            // the factors of this lane's columns of the product: rows 2 t, 2 t + 1 of the block
#pragma unroll
            for (int e = 0; e < 2; ++e) factor[b][e] = __shfl_sync(0xffffffffu, f, 4 * (2 * t + e));
        }
        auto scores = [&](const uint4 (&k)[2][C], float (&c4)[NB][4]) {
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                c4[b][0] = c4[b][1] = c4[b][2] = c4[b][3] = 0.0f;
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    if (!QF16) {
                        mma_f16(c4[b], k[0][c].x, k[1][c].x, k[0][c].y, k[1][c].y, q.lo[b][c].x, q.lo[b][c].y);
                        mma_f16(c4[b], k[0][c].z, k[1][c].z, k[0][c].w, k[1][c].w, q.lo[b][c].z, q.lo[b][c].w);
                    }
                    mma_f16(c4[b], k[0][c].x, k[1][c].x, k[0][c].y, k[1][c].y, q.hi[b][c].x, q.hi[b][c].y);
                    mma_f16(c4[b], k[0][c].z, k[1][c].z, k[0][c].w, k[1][c].w, q.hi[b][c].z, q.hi[b][c].w);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) c4[b][e] *= factor[b][e & 1];
            }
        };
        // whether the tile has positions that some nodes do not see, and whether value e of block b is such a one
        auto edge = [&](int tile) { return tile * WTILE + WTILE - 1 > past; };
        auto hidden = [&](int tile, int b, int e) {
            return tile * WTILE + g + 8 * (e >> 1) > past + group(min(r0 + 8 * b + 2 * t + (e & 1), rows - 1));
        };

        // ---- m and l of the block's rows
        float m[NB][2], l[NB][2];
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int e = 0; e < 2; ++e) m[b][e] = -INFINITY, l[b][e] = 0.0f;
        uint4 next[2][C];
        if (t0 + warp < t1) load_k(next, t0 + warp);
        int kept = 0;
        for (int tile = t0 + warp; tile < t1; tile += WW, ++kept) {
            uint4 k[2][C];
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int c = 0; c < C; ++c) k[h][c] = next[h][c];
            if (tile + WW < t1) load_k(next, tile + WW);
            float c4[NB][4];
            scores(k, c4);
            if (edge(tile)) {
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (hidden(tile, b, e)) c4[b][e] = -INFINITY;
            }
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                if (kept < a.cap) s_scores[((kept * WW + warp) * NB + b) * 32 + lane] = make_float4(c4[b][0], c4[b][1], c4[b][2], c4[b][3]);
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float mm = fmaxf(m[b][e], fmaxf(c4[b][e], c4[b][e + 2])), z = mm == -INFINITY ? 0.0f : mm;
                    l[b][e] = l[b][e] * ex2(m[b][e] - z) + ex2(c4[b][e] - z) + ex2(c4[b][e + 2] - z);
                    m[b][e] = mm;
                }
            }
        }
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
        if (r0 == 0 && a.cs > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // all CTAs have started
        if (tid < RB) {
            float2 x = s_warp[0][tid];
            for (int w = 1; w < WW; ++w) join(x.x, x.y, s_warp[w][tid].x, s_warp[w][tid].y);
            if (a.cs == 1) {
                s_ml[parity][0][tid] = x;
            } else {
                cg::cluster_group cl = cg::this_cluster();
                for (int c = 0; c < a.cs; ++c) *cl.map_shared_rank(&s_ml[parity][rank][tid], c) = x;
            }
        }
        if (a.cs == 1) __syncthreads();
        else cg::this_cluster().sync();
        if (tid < RB) {
            float2 x = s_ml[parity][0][tid];
            for (int c = 1; c < a.cs; ++c) join(x.x, x.y, s_ml[parity][c][tid].x, s_ml[parity][c][tid].y);
            // 1 / l: 0 for rows of padding, and where all scores are -inf; NaN stays
            const bool none = r0 + tid >= rows || (x.x == -INFINITY && x.y == x.y);
            s_row[tid] = make_float2(x.x == -INFINITY ? 0.0f : x.x, none ? 0.0f : 1.0f / x.y);
        }
        __syncthreads();
        float2 ml[NB][2];
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int e = 0; e < 2; ++e) ml[b][e] = s_row[8 * b + 2 * t + e];

        // ---- weights
        kept = 0;
        for (int tile = t0 + warp; tile < t1; tile += WW, ++kept) {
            float c4[NB][4];
            if (kept < a.cap) {
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    const float4 x = s_scores[((kept * WW + warp) * NB + b) * 32 + lane];
                    c4[b][0] = x.x, c4[b][1] = x.y, c4[b][2] = x.z, c4[b][3] = x.w;
                }
            } else {
                uint4 k[2][C];
                load_k(k, tile);
                scores(k, c4);
            }
            const bool all = !edge(tile);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float w = 0.0f;
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float x = ex2(c4[b][2 * h + e] - ml[b][e].x) * ml[b][e].y;
                        w += all || !hidden(tile, b, 2 * h + e) ? x : 0.0f;  // also where the row is NaN
                    }
                w += __shfl_xor_sync(0xffffffffu, w, 1);
                w += __shfl_xor_sync(0xffffffffu, w, 2);
                int off;
                const int p8 = tile * WTILE + 8 * h, pg = locate(p8, off);
                if (t == 0 && pg >= 0 && p8 + g < T) {
                    float *at = reinterpret_cast<float *>(wh + pg * a.w_nb2) + off + g;
                    if (r0) w += *at;
                    else if (a.decay != 0.0f && p8 + g < past) w += a.decay * *at;
                    *at = w;
                }
            }
        }
        __syncthreads();  // s_warp and s_row are written again
    }
}

template <int D, int NB, bool QF16>
int launch_weights(oasr_backend *be, Weights a, const KvPages &p, const KvSeqs &sq, int S) {
    // scores of a warp's tiles in 96 KB: two CTAs per SM
    constexpr int SMEM = 96 << 10;
    a.cap = SMEM / (WW * NB * 32 * (int)sizeof(float4));
    static OncePerDevice once;
    cudaError_t e = (cudaError_t)once(be->device, [] {
        const cudaError_t x = cudaFuncSetAttribute(attn_weights_kernel<D, NB, QF16>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
        return x != cudaSuccess ? x : cudaFuncSetAttribute(attn_weights_kernel<D, NB, QF16>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    });
    if (e != cudaSuccess) return oasr_internal_cuda_fail(be, e, "attn_weights attribute", __LINE__);
    const int64_t items = (int64_t)S * a.HKV, tiles = ((int64_t)sq.MP * p.page + WTILE - 1) / WTILE;
    a.cs = 16;
    while (a.cs > 1 && (items * a.cs > 2 * be->sm_count || tiles < a.cs)) a.cs /= 2;
    if (items * a.cs > INT32_MAX) return fail_op(be, "attn_weights", "too many sequences");
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(items * a.cs));
    cfg.blockDim = dim3(WT);
    cfg.dynamicSmemBytes = SMEM;
    cfg.stream = be->stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = a.cs, attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = be->pdl ? 2 : 1;
    return launched(be, cudaLaunchKernelEx(&cfg, attn_weights_kernel<D, NB, QF16>, a, p, sq, FastDiv(p.page), FastDiv(a.G), be->err_word),
                    "attn_weights");
}

// ---- eviction ---------------------------------------------------------------------------------
struct Evict {
    char *w;
    int64_t w_nb1, w_nb2;  // head, page
    const int *n_keep;     // [S]
    int *n_past_out;       // [S]
    int S, HKV, D, sink, recent;
};

constexpr int ET = 256;

// Numbers that order as the values do; -0 is 0, and NaN comes before everything.
__device__ __forceinline__ uint32_t order_key(float v) {
    const uint32_t b = __float_as_uint(v + 0.0f);
    return v != v ? 0u : b & 0x80000000u ? ~b : b | 0x80000000u;
}

// One CTA per (layer, sequence, K/V head): the least key that stays, by four rounds of counting 8 bits;
// then all positions once, in order, 256 at a time.  A row's place is its rank among the kept ones, never
// behind its position, and the rows of a batch are loaded before any of them is stored: what is stored
// lies before the next batch's rows.
__global__ void __launch_bounds__(ET) kv_evict_kernel(Evict a, KvPages p, KvSeqs sq, FastDiv page, int *err) {
    __shared__ int s_count[256], s_warp[2][ET / 32];
    __shared__ int s_src[ET], s_dst[ET];  // the kept positions of the 256, and where they go
    __shared__ uint32_t s_prefix;
    __shared__ int s_need, s_bad;
    griddep_launch_dependents();
    griddep_wait();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int h = blockIdx.x % a.HKV, s = blockIdx.x / a.HKV % a.S, layer = blockIdx.x / a.HKV / a.S;
    int past, none;
    const bool fits = seq_lengths(sq, s, p.page, past, none);
    const int keep = a.n_keep[s];
    const bool ok = fits && (past <= keep || (keep >= a.sink && keep - a.sink >= a.recent));
    const bool full = ok && past > keep;
    if (layer == 0 && h == 0 && tid == 0) {
        if (!ok) atomicOr(err, ERR_BAD_INDEX);
        a.n_past_out[s] = full ? keep : past;
    }
    if (!full) return;
    const int *table = sq.table + s * sq.table_ld;
    if (tid == 0) s_bad = 0;
    __syncthreads();
    for (int j = tid; j <= page(past - 1); j += ET)
        if (table[j] < 0 || table[j] >= p.n_pages) s_bad = 1;
    __syncthreads();
    if (s_bad) {
        if (tid == 0) atomicOr(err, ERR_BAD_INDEX);
        return;
    }
    char *wh = a.w + (int64_t)layer * p.n_pages * a.w_nb2 + h * a.w_nb1;
    auto weight_at = [&](int pos) {
        const int j = page(pos);
        return reinterpret_cast<float *>(wh + table[j] * a.w_nb2) + (pos - j * p.page);
    };
    const int m0 = a.sink, m1 = past - a.recent;  // the positions that compete
    int need = keep - a.sink - a.recent;          // how many of them stay
    uint32_t prefix = 0;                          // high bits of the least key that stays
    if (need > 0)
        for (int shift = 24; shift >= 0; shift -= 8) {
            for (int c = tid; c < 256; c += ET) s_count[c] = 0;
            __syncthreads();
            for (int pos = m0 + tid; pos < m1; pos += ET) {
                const uint32_t k = order_key(*weight_at(pos));
                if (shift == 24 || k >> (shift + 8) == prefix >> (shift + 8)) atomicAdd(&s_count[k >> shift & 255], 1);
            }
            __syncthreads();
            if (warp == 0) {  // from the greatest digit down, 8 digits a lane
                int own = 0;
                for (int c = 0; c < 8; ++c) own += s_count[255 - 8 * lane - c];
                int run = own;
                for (int o = 1; o < 32; o <<= 1) {
                    const int v = __shfl_up_sync(0xffffffffu, run, o);
                    if (lane >= o) run += v;
                }
                int left = need - (run - own);
                if (left > 0 && run >= need) {
                    int c = 0;
                    while (left > s_count[255 - 8 * lane - c]) left -= s_count[255 - 8 * lane - c++];
                    s_prefix = prefix | (uint32_t)(255 - 8 * lane - c) << shift;
                    s_need = left;
                }
            }
            __syncthreads();
            prefix = s_prefix;
            need = s_need;
        }
    // need: how many of the positions with exactly that key stay, the first ones
    const bool any = keep > a.sink + a.recent;
    int kept = a.sink, ties = 0;
    const int cpr = a.D / 8, per = ET / cpr;  // 16-byte columns of a row, rows at a time
    const int c16 = tid % cpr, r16 = tid / cpr;
    char *kh = p.k + (int64_t)layer * p.n_pages * p.k_nb3 + h * p.k_nb2 + 16 * c16;
    char *vh = p.v + (int64_t)layer * p.n_pages * p.v_nb3 + h * p.v_nb2 + 16 * c16;
    for (int base = a.sink; base < past; base += ET) {
        const int pos = base + tid;
        float w = 0.0f;
        bool above = false, equal = false;
        if (pos < past) {
            w = *weight_at(pos);
            const uint32_t k = order_key(w);
            above = pos >= m1 || (any && k > prefix);
            equal = pos < m1 && any && k == prefix;
        }
        const unsigned eq = __ballot_sync(0xffffffffu, equal);
        if (lane == 0) s_warp[0][warp] = __popc(eq);
        __syncthreads();
        int tie = ties + __popc(eq & ((1u << lane) - 1)), all_ties = 0;
        for (int k = 0; k < ET / 32; ++k) {
            if (k < warp) tie += s_warp[0][k];
            all_ties += s_warp[0][k];
        }
        const bool stays = above || (equal && tie < need);
        const unsigned st = __ballot_sync(0xffffffffu, stays);
        if (lane == 0) s_warp[1][warp] = __popc(st);
        __syncthreads();
        int place = __popc(st & ((1u << lane) - 1)), all = 0;
        for (int k = 0; k < ET / 32; ++k) {
            if (k < warp) place += s_warp[1][k];
            all += s_warp[1][k];
        }
        if (stays) {
            s_src[place] = pos;
            s_dst[place] = kept + place;
            *weight_at(kept + place) = w;
        }
        ties += all_ties;
        __syncthreads();
        for (int b = 0; b < all; b += 4 * per) {
            uint4 k4[4], v4[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int r = b + u * per + r16;
                if (r < all && s_src[r] != s_dst[r]) {
                    const int j = page(s_src[r]), off = s_src[r] - j * p.page;
                    k4[u] = *reinterpret_cast<const uint4 *>(kh + table[j] * p.k_nb3 + off * p.k_nb1);
                    v4[u] = *reinterpret_cast<const uint4 *>(vh + table[j] * p.v_nb3 + off * p.v_nb1);
                }
            }
            __syncthreads();
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int r = b + u * per + r16;
                if (r < all && s_src[r] != s_dst[r]) {
                    const int j = page(s_dst[r]), off = s_dst[r] - j * p.page;
                    *reinterpret_cast<uint4 *>(kh + table[j] * p.k_nb3 + off * p.k_nb1) = k4[u];
                    *reinterpret_cast<uint4 *>(vh + table[j] * p.v_nb3 + off * p.v_nb1) = v4[u];
                }
            }
        }
        kept += all;
        __syncthreads();
    }
}

// F32 [page, H_kv, n_pages] beside the pages
bool is_weights(const oasr_tensor *w, const oasr_tensor *k) {
    return w && w->type == OASR_TYPE_F32 && w->data && aligned4(w) && w->ne[0] == k->ne[1] && w->ne[1] == k->ne[2] &&
           w->ne[2] == k->ne[3] && w->ne[3] == 1 && w->nb[0] == 4 && w->nb[1] % 4 == 0 && w->nb[2] % 4 == 0 && w->nb[1] >= 0 &&
           w->nb[2] >= 0;
}

}  // namespace

extern "C" {

int oasr_b200_attn_weights(oasr_backend *be, const oasr_tensor *q, const oasr_tensor *k_pages, const oasr_tensor *page_table,
                           const oasr_tensor *n_past, const oasr_tensor *n_nodes, float scale, float decay, oasr_tensor *weights) {
    int st = oasr_internal_precheck(be);
    if (st) return st;
    const char *op = "attn_weights";
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
    if (!is_weights(weights, k_pages)) return fail_op(be, op, "weights must be F32 [page, H_kv, n_pages] with contiguous rows");
    if (!(scale == scale)) return fail_op(be, op, "scale must be a number");
    if (!(decay >= 0.0f && decay < INFINITY)) return fail_op(be, op, "decay must not be negative, and finite");
    if (N == 0 || S == 0) return OASR_STATUS_SUCCESS;
    st = seqs_check(be, op, page_table, n_past, n_nodes, S, N, &sq);
    if (st) return st;
    if (N * (H / HKV) > INT32_MAX / 2) return fail_op(be, op, "too many rows");
    if (!q->data) return fail_op(be, op, "null argument");
    if (!rows16(q)) return fail_op(be, op, "rows must be 16-byte aligned");
    Weights a = {};
    a.q = (const char *)q->data;
    a.q_nb1 = q->nb[1], a.q_nb2 = q->nb[2], a.q_nb3 = q->nb[3];
    a.w = (char *)weights->data, a.w_nb1 = weights->nb[1], a.w_nb2 = weights->nb[2];
    a.HKV = (int)HKV, a.G = (int)(H / HKV);
    a.scale = scale, a.decay = decay;
    const bool two = N * a.G > 8;
#define AW(DD, NB, Q) \
    if (D == DD && two == (NB == 2) && f16 == Q) return launch_weights<DD, NB, Q>(be, a, p, sq, (int)S)
    AW(64, 1, false); AW(64, 1, true); AW(64, 2, false); AW(64, 2, true);
    AW(128, 1, false); AW(128, 1, true); AW(128, 2, false); AW(128, 2, true);
#undef AW
    return fail_op(be, op, "head_dim must be 64 or 128");
}

int oasr_b200_kv_evict(oasr_backend *be, oasr_tensor *weights, const oasr_tensor *page_table, const oasr_tensor *n_past,
                       const oasr_tensor *n_keep, int32_t n_sink, int32_t n_recent, oasr_tensor *k_pages, oasr_tensor *v_pages,
                       int32_t n_layers, oasr_tensor *n_past_out) {
    int st = oasr_internal_precheck(be);
    if (st) return st;
    const char *op = "kv_evict";
    if (!n_past) return fail_op(be, op, "null argument");
    KvPages p;
    KvSeqs sq;
    st = pages_check(be, op, k_pages, v_pages, n_layers, &p);
    if (st) return st;
    const int64_t S = n_past->ne[0], HKV = k_pages->ne[2];
    if (!is_weights(weights, k_pages)) return fail_op(be, op, "weights must be F32 [page, H_kv, n_pages] with contiguous rows");
    if (n_sink < 0 || n_recent < 0) return fail_op(be, op, "n_sink and n_recent must not be negative");
    if (S == 0) return OASR_STATUS_SUCCESS;
    st = seqs_check(be, op, page_table, n_past, nullptr, S, 0, &sq);
    if (st) return st;
    if (!is_vec_i32(n_keep, S) || !is_vec_i32(n_past_out, S)) return fail_op(be, op, "n_keep and n_past_out must be I32 [n_seq]");
    for (const oasr_tensor *t : {n_past, n_keep, page_table})
        if (share_values(int_rows(n_past_out), int_rows(t)))
            return fail_op(be, op, "n_past_out must not overlap an input (it is still read while it is written)");
    if (S * HKV * n_layers > INT32_MAX) return fail_op(be, op, "too many sequences");
    Evict a;
    a.w = (char *)weights->data, a.w_nb1 = weights->nb[1], a.w_nb2 = weights->nb[2];
    a.n_keep = (const int *)n_keep->data, a.n_past_out = (int *)n_past_out->data;
    a.S = (int)S, a.HKV = (int)HKV, a.D = (int)k_pages->ne[0], a.sink = n_sink, a.recent = n_recent;
    return launched(be, launch_k(be, kv_evict_kernel, dim3((unsigned)(S * HKV * n_layers)), dim3(ET), 0, a, p, sq, FastDiv(p.page),
                                 be->err_word), op);
}

}  // extern "C"
