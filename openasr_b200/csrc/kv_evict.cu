// kv_evict.cu -- eviction from a paged cache by accumulated attention: of a sequence's positions the first
// n_sink, the last n_recent, and of the others those with the greatest weights (attn_weights.cu) stay,
// n_keep in all; their rows move to the front in their order.
#include <cooperative_groups.h>

#include <algorithm>

#include "once_per_device.h"
#include "op_checks.cuh"
#include "pages.cuh"

using namespace oasr;

namespace {

struct Evict {
    char *w;
    int64_t w_nb1, w_nb2;  // head, page
    const int *n_keep;     // [S]
    int *n_past_out;       // [S]
    int S, HKV, sink, recent;
    int words;             // of 32 positions that shared memory holds the choice of
    int keys;              // keys that it holds besides
};

constexpr int ET = 256, EW = ET / 32;
constexpr int EVICT_MOST = 1 << 18;  // positions of a sequence

// Numbers that order as the values do; -0 is 0, and NaN comes before everything.
__device__ __forceinline__ uint32_t order_key(float v) {
    const uint32_t b = __float_as_uint(v + 0.0f);
    return v != v ? 0u : b & 0x80000000u ? ~b : b | 0x80000000u;
}

// inc[i] = f(0) + ... + f(i) for i < n, by the whole CTA
template <typename F>
__device__ __forceinline__ void running(int n, uint32_t *inc, int *s_warp, F f) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int per = (n + ET - 1) / ET, i0 = min(tid * per, n), i1 = min(i0 + per, n);
    int own = 0;
    for (int i = i0; i < i1; ++i) own += f(i);
    int up = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, up, o);
        if (lane >= o) up += v;
    }
    if (lane == 31) s_warp[warp] = up;
    __syncthreads();
    int sum = up - own;
    for (int w = 0; w < warp; ++w) sum += s_warp[w];
    for (int i = i0; i < i1; ++i) inc[i] = sum += f(i);
    __syncthreads();
}

// the lowest n set bits of a word
__device__ __forceinline__ uint32_t lowest(uint32_t word, int n) {
    if (n >= __popc(word)) return word;
    uint32_t out = 0;
    for (; n > 0; --n) out |= word & -word, word &= word - 1;
    return out;
}

// the place of set bit n of a word
__device__ __forceinline__ int nth_bit(uint32_t word, int n) {
    int at = 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const int c = __popc(word & ((1u << o) - 1));
        if (n >= c) n -= c, word >>= o, at += o;
    }
    return at;
}

// One cluster of CS CTAs per (layer, sequence, K/V head).  Which positions stay is worked out together: each
// CTA has a run of the positions; the least key that stays is found by counting 8 bits at a time, the
// counts going to every CTA; then every CTA gets the whole choice, one bit per position, and how many bits
// are set up to each word.  The rows are moved by columns, each CTA its own 16 LPR bytes of every K row or
// every V row, so that from here on no CTA waits for another: row g of the kept ones comes from the
// position of bit g, never before position g, in rounds of BATCH rows (256; 128 in columns of 256 bytes) that
// are all loaded before any of them is stored.  What is stored lies before all later rounds' rows.
template <int CS, int LPR>
__global__ void __launch_bounds__(ET) kv_evict_kernel(Evict a, KvPages p, KvSeqs sq, FastDiv page, int *err) {
    namespace cg = cooperative_groups;
    constexpr int ROWS = ET / LPR, U = LPR > 8 ? 8 : LPR, BATCH = ROWS * U;  // rows at a time, of a thread, of a round
    extern __shared__ uint32_t s_dyn[];
    uint32_t *s_mask = s_dyn, *s_inc = s_mask + a.words, *s_keys = s_inc + a.words;
    __shared__ int s_count[2][CS][256], s_own[256];
    __shared__ int s_warp[EW], s_digit, s_need, s_bad;
    __shared__ int4 s_at[2][BATCH];  // source page and offset, destination page and offset
    griddep_launch_dependents();
    griddep_wait();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int item = blockIdx.x / CS, rank = blockIdx.x % CS;
    const int h = item % a.HKV, s = item / a.HKV % a.S, layer = item / a.HKV / a.S;
    int past, none;
    const bool fits = seq_lengths(sq, s, p.page, past, none) && past <= EVICT_MOST;
    const int keep = a.n_keep[s];
    const bool ok = fits && (past <= keep || (keep >= a.sink && keep - a.sink >= a.recent));
    const bool full = ok && past > keep;
    const bool reports = layer == 0 && h == 0 && rank == 0 && tid == 0;
    if (!full) {
        if (!reports) return;
        if (!ok) atomicOr(err, ERR_BAD_INDEX);
        a.n_past_out[s] = sq.n_past[s];
        return;
    }
    const int *table = sq.table + s * sq.table_ld;
    if (tid == 0) s_bad = 0;
    __syncthreads();
    for (int j = tid; j <= page(past - 1); j += ET)
        if (table[j] < 0 || table[j] >= p.n_pages) s_bad = 1;
    __syncthreads();
    if (reports) a.n_past_out[s] = s_bad ? past : keep;
    if (s_bad) {  // in every CTA of all its clusters: nothing moves
        if (tid == 0) atomicOr(err, ERR_BAD_INDEX);
        return;
    }
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    char *wh = a.w + (int64_t)layer * p.n_pages * a.w_nb2 + h * a.w_nb1;
    auto weight_at = [&](int pos) {
        const int j = page(pos);
        return reinterpret_cast<float *>(wh + table[j] * a.w_nb2) + (pos - j * p.page);
    };
    const int words = (past + 31) / 32, slice = (words + CS - 1) / CS;
    const int w0 = min(rank * slice, words), w1 = min(w0 + slice, words);
    const int m0 = a.sink, m1 = past - a.recent;  // the positions that compete
    const int c0 = max(32 * w0, m0), c1 = min(32 * w1, m1);
    const bool held = 32 * slice <= a.keys;
    if (held)
        for (int first = c0 + tid; first < c1; first += 16 * ET) {  // sixteen loads under way
            float v[16];
#pragma unroll
            for (int u = 0; u < 16; ++u)
                if (first + u * ET < c1) v[u] = *weight_at(first + u * ET);
#pragma unroll
            for (int u = 0; u < 16; ++u)
                if (first + u * ET < c1) s_keys[first + u * ET - 32 * w0] = order_key(v[u]);
        }
    auto key = [&](int pos) { return held ? s_keys[pos - 32 * w0] : order_key(*weight_at(pos)); };
    int need = keep - a.sink - a.recent;  // how many of those that compete stay
    const bool any = need > 0;
    uint32_t least = 0;  // the least key that stays, digit by digit
    int before = 0;      // positions with exactly that key in the CTAs before this one
    int equal = 0;       // and in all of them
    cg::cluster_group cl = cg::this_cluster();
    if (!any) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    for (int shift = 24, turn = 0; any && shift >= 0; shift -= 8, turn ^= 1) {
        s_own[tid] = 0;
        __syncthreads();
        for (int pos = c0 + tid; pos < c1; pos += ET) {
            const uint32_t k = key(pos);
            if (shift == 24 || k >> (shift + 8) == least >> (shift + 8)) atomicAdd(&s_own[k >> shift & 255], 1);
        }
        if (shift == 24) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // all CTAs have started
        __syncthreads();
#pragma unroll
        for (int c = 0; c < CS; ++c) *cl.map_shared_rank(&s_count[turn][rank][tid], c) = s_own[tid];
        cl.sync();
        if (warp == 0) {  // from the greatest digit down, 8 digits a lane
            int n[8], own = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                n[i] = 0;
#pragma unroll
                for (int c = 0; c < CS; ++c) n[i] += s_count[turn][c][255 - 8 * lane - i];
                own += n[i];
            }
            int up = own;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, up, o);
                if (lane >= o) up += v;
            }
            int left = need - (up - own);
            if (left > 0 && up >= need) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    if (left > 0 && left <= n[i]) s_digit = 255 - 8 * lane - i, s_need = left;
                    left -= n[i];
                }
            }
        }
        __syncthreads();
        least |= (uint32_t)s_digit << shift;
        need = s_need;
        if (shift == 0)
            for (int c = 0; c < CS; ++c) {
                if (c < rank) before += s_count[turn][c][s_digit];
                equal += s_count[turn][c][s_digit];
            }
    }
    // `need` of the `equal` positions with the least key stay, the first ones
    const bool cut = any && need < equal;
    for (int w = w0 + warp; w < w1; w += EW) {
        const int pos = 32 * w + lane;
        const bool stays = pos < past && (pos < m0 || pos >= m1), competes = any && pos >= m0 && pos < m1;
        const uint32_t k = competes ? key(pos) : 0;
        const uint32_t above = __ballot_sync(0xffffffffu, stays || (competes && k > least));
        const uint32_t ties = __ballot_sync(0xffffffffu, competes && k == least);
        if (lane == 0) s_mask[w] = cut ? above : above | ties;
        if (cut && lane == 0) s_inc[w] = ties;
    }
    __syncthreads();
    if (cut) {  // how many ties there are before each word, and which of the word's stay
        const int per = (w1 - w0 + ET - 1) / ET, b0 = min(w0 + tid * per, w1), b1 = min(b0 + per, w1);
        int own = 0;
        for (int w = b0; w < b1; ++w) own += __popc(s_inc[w]);
        int up = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, up, o);
            if (lane >= o) up += v;
        }
        if (lane == 31) s_warp[warp] = up;
        __syncthreads();
        int sum = before + up - own;
        for (int w = 0; w < warp; ++w) sum += s_warp[w];
        for (int w = b0; w < b1; ++w) {
            s_mask[w] |= lowest(s_inc[w], max(need - sum, 0));
            sum += __popc(s_inc[w]);
        }
        __syncthreads();
    }
    for (int w = w0 + tid; w < w1; w += ET)
#pragma unroll
        for (int c = 0; c < CS; ++c)
            if (c != rank) *cl.map_shared_rank(&s_mask[w], c) = s_mask[w];
    cl.sync();
    running(words, s_inc, s_warp, [&](int i) { return __popc(s_mask[i]); });

    // ---- the rows
    int w_first = 0;  // the rows of the words that keep all 32 are in place
    {
        if (tid == 0) s_bad = words;
        __syncthreads();
        for (int w = tid; w < words; w += ET)
            if (s_mask[w] != 0xffffffffu) {
                atomicMin(&s_bad, w);
                break;
            }
        __syncthreads();
        w_first = s_bad;
    }
    const int g0 = 32 * w_first;
    auto source = [&](int g) {  // the position of kept row g
        int lo = w_first, hi = words - 1;
        while (lo < hi) {
            const int mid = (lo + hi) / 2;
            if ((int)s_inc[mid] > g) hi = mid;
            else lo = mid + 1;
        }
        return 32 * lo + nth_bit(s_mask[lo], g - (lo ? (int)s_inc[lo - 1] : 0));
    };
    auto locate = [&](int base, int turn) {
        for (int i = tid; i < BATCH; i += ET) {
            const int g = base + i;
            if (g >= keep) continue;
            const int from = source(g), fj = page(from), tj = page(g);
            s_at[turn][i] = make_int4(from == g ? -1 : table[fj], from - fj * p.page, table[tj], g - tj * p.page);
        }
    };
    const int kv = rank & 1, c16 = (rank >> 1) * LPR + tid % LPR, r = tid / LPR;
    const int64_t nb1 = kv ? p.v_nb1 : p.k_nb1, nb3 = kv ? p.v_nb3 : p.k_nb3;
    char *rows = (kv ? p.v : p.k) + (int64_t)layer * p.n_pages * nb3 + h * (kv ? p.v_nb2 : p.k_nb2) + 16 * c16;
    locate(g0, 0);
    __syncthreads();
    for (int base = g0, turn = 0; base < keep; base += BATCH, turn ^= 1) {
        uint4 v[U];
        float w[(BATCH + ET - 1) / ET];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = u * ROWS + r;
            if (base + i < keep && s_at[turn][i].x >= 0)
                v[u] = *reinterpret_cast<const uint4 *>(rows + s_at[turn][i].x * nb3 + s_at[turn][i].y * nb1);
        }
        if (rank == 0) {
#pragma unroll
            for (int u = 0; u < (BATCH + ET - 1) / ET; ++u) {
                const int i = u * ET + tid;
                if (i < BATCH && base + i < keep && s_at[turn][i].x >= 0)
                    w[u] = reinterpret_cast<const float *>(wh + s_at[turn][i].x * a.w_nb2)[s_at[turn][i].y];
            }
        }
        locate(base + BATCH, turn ^ 1);
        __syncthreads();
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = u * ROWS + r;
            if (base + i < keep && s_at[turn][i].x >= 0)
                *reinterpret_cast<uint4 *>(rows + s_at[turn][i].z * nb3 + s_at[turn][i].w * nb1) = v[u];
        }
        if (rank == 0) {
#pragma unroll
            for (int u = 0; u < (BATCH + ET - 1) / ET; ++u) {
                const int i = u * ET + tid;
                if (i < BATCH && base + i < keep && s_at[turn][i].x >= 0)
                    reinterpret_cast<float *>(wh + s_at[turn][i].z * a.w_nb2)[s_at[turn][i].w] = w[u];
            }
        }
        __syncthreads();  // the places of this round are written again
    }
}

template <int CS, int LPR>
int launch_evict(oasr_backend *be, Evict a, const KvPages &p, const KvSeqs &sq, int64_t items) {
    if (items * CS > INT32_MAX) return fail_op(be, "kv_evict", "too many sequences");
    const int64_t most = std::min<int64_t>((int64_t)sq.MP * p.page, EVICT_MOST);
    a.words = (int)((most + 31) / 32);
    a.keys = std::min(12288, (a.words + CS - 1) / CS * 32);
    constexpr int SMEM = (EVICT_MOST / 32 * 2 + 12288) * 4;
    static OncePerDevice once;
    const cudaError_t e = (cudaError_t)once(be->device, [] {
        return cudaFuncSetAttribute(kv_evict_kernel<CS, LPR>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
    });
    if (e != cudaSuccess) return oasr_internal_cuda_fail(be, e, "kv_evict attribute", __LINE__);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(items * CS));
    cfg.blockDim = dim3(ET);
    cfg.dynamicSmemBytes = (size_t)(2 * a.words + a.keys) * 4;
    cfg.stream = be->stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = CS, attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = be->pdl ? 2 : 1;
    return launched(be, cudaLaunchKernelEx(&cfg, kv_evict_kernel<CS, LPR>, a, p, sq, FastDiv(p.page), be->err_word), "kv_evict");
}

}  // namespace

extern "C" int oasr_b200_kv_evict(oasr_backend *be, oasr_tensor *weights, const oasr_tensor *page_table, const oasr_tensor *n_past,
                       const oasr_tensor *n_keep, int32_t n_sink, int32_t n_recent, oasr_tensor *k_pages, oasr_tensor *v_pages,
                       int32_t n_layers, oasr_tensor *n_past_out) {
    const char *op = "kv_evict";
    if (!be) return oasr_internal_precheck(be);
    int st;
    if (!n_past) return fail_op(be, op, "null argument");
    KvPages p;
    KvSeqs sq;
    st = pages_check(be, op, k_pages, v_pages, n_layers, &p);
    if (st) return st;
    const int64_t S = n_past->ne[0], HKV = k_pages->ne[2];
    if (!is_weights(weights, k_pages)) return fail_op(be, op, "weights must be F32 [page, H_kv, n_pages], rows contiguous and apart");
    if (n_sink < 0 || n_recent < 0) return fail_op(be, op, "n_sink and n_recent must not be negative");
    if (S == 0) return oasr_internal_precheck(be);
    st = seqs_check(be, op, page_table, n_past, nullptr, S, 0, &sq);
    if (st) return st;
    if (!is_vec_i32(n_keep, S) || !is_vec_i32(n_past_out, S)) return fail_op(be, op, "n_keep and n_past_out must be I32 [n_seq]");
    // all of them are read while others are written
    const oasr_tensor *moved[] = {weights, k_pages, v_pages}, *read[] = {n_past, n_keep, page_table};
    for (const oasr_tensor *pages : {k_pages, v_pages})
        if (!apart(pages)) return fail_op(be, op, "rows of the pages must not overlap");
    if (share_bytes(weights, k_pages) || share_bytes(weights, v_pages) || share_bytes(k_pages, v_pages))
        return fail_op(be, op, "weights, k_pages and v_pages must not overlap");
    for (const oasr_tensor *t : read) {
        if (share_bytes(n_past_out, t)) return fail_op(be, op, "n_past_out must not overlap an input (it is still read while it is written)");
        for (const oasr_tensor *m : moved)
            if (share_bytes(m, t)) return fail_op(be, op, "weights and pages must not overlap lengths or page table");
    }
    for (const oasr_tensor *m : moved)
        if (share_bytes(n_past_out, m)) return fail_op(be, op, "n_past_out must not overlap an input (it is still read while it is written)");
    st = oasr_internal_precheck(be);  // the arguments need no device
    if (st) return st;
    Evict a = {};
    a.w = (char *)weights->data, a.w_nb1 = weights->nb[1], a.w_nb2 = weights->nb[2];
    a.n_keep = (const int *)n_keep->data, a.n_past_out = (int *)n_past_out->data;
    a.S = (int)S, a.HKV = (int)HKV, a.sink = n_sink, a.recent = n_recent;
    const int64_t items = S * HKV * n_layers;
    // a K row and a V row for a CTA each; half a row where that leaves SMs without work (96 heads of 128 and
    // 32000 positions: 171 us in halves, 343 in rows; 224 of 512: 38 and 22, 1792 of 390 to 1990: 279 and 205)
    const bool halves = items <= be->sm_count;
    if (k_pages->ne[0] == 128) return halves ? launch_evict<4, 8>(be, a, p, sq, items) : launch_evict<2, 16>(be, a, p, sq, items);
    return halves ? launch_evict<4, 4>(be, a, p, sq, items) : launch_evict<2, 8>(be, a, p, sq, items);
}
