// kv_pages.cu -- the paged K/V cache around the tree attention: per-head norms, rotation
// and the cache write of new nodes (qk_norm_rope), acceptance of a drafted tree with the
// compaction of its rows (tree_commit), and page copies (kv_pages_copy).
//
// The cache of one layer is a pool of pages [D, page, n_kv_heads, n_pages] f16; a sequence
// owns positions through its row of the page table.  Node i of sequence s sits at position
// n_past[s] + i; lengths live in device memory, so a step can be captured once and replayed.
#include <stdlib.h>
#include <string.h>

#include <algorithm>

#include "pages.cuh"

using namespace oasr;

namespace oasr {

// 4-byte values that are read and written as such
static bool aligned4(const oasr_tensor *t) { return ((uintptr_t)t->data & 3) == 0; }

static bool is_vec_i32(const oasr_tensor *t, int64_t n) {
    return t && t->type == OASR_TYPE_I32 && t->data && aligned4(t) && t->ne[0] == n && t->ne[1] == 1 && t->ne[2] == 1 &&
           t->ne[3] == 1 && (t->nb[0] == 4 || n <= 1);
}

static int fail_op(oasr_backend *be, const char *op, const char *what) {
    return oasr_internal_fail(be, OASR_STATUS_FAILED, std::string(op) + ": " + what);
}

int pages_check(oasr_backend *be, const char *op, const oasr_tensor *k, const oasr_tensor *v, int layers, KvPages *out) {
    if (!k || !v) return fail_op(be, op, "null argument");
    if (k->type != OASR_TYPE_F16 || v->type != OASR_TYPE_F16) return fail_op(be, op, "k/v pages must be F16");
    for (int i = 0; i < 4; ++i)
        if (k->ne[i] != v->ne[i]) return fail_op(be, op, "k/v pages must have one shape");
    if (k->ne[0] != 64 && k->ne[0] != 128) return fail_op(be, op, "head_dim must be 64 or 128");
    if (k->ne[1] < 8 || k->ne[1] % 8 || k->ne[1] > (1 << 24))
        return fail_op(be, op, "positions per page must be a multiple of 8");
    if (k->ne[2] < 1 || k->ne[2] > 65535 || k->ne[3] < 1 || k->ne[3] > (1 << 30)) return fail_op(be, op, "bad page pool shape");
    if (layers < 1 || k->ne[3] % layers) return fail_op(be, op, "n_layers must divide the pages");
    if (!k->data || !v->data) return fail_op(be, op, "null argument");
    for (const oasr_tensor *t : {k, v}) {
        if (t->nb[0] != 2) return fail_op(be, op, "rows of the pages must be contiguous");
        if (((uintptr_t)t->data & 15) || t->nb[1] % 16 || t->nb[2] % 16 || t->nb[3] % 16 || t->nb[1] < 0 || t->nb[2] < 0 ||
            t->nb[3] < 0)
            return fail_op(be, op, "rows of the pages must be 16-byte aligned");
    }
    *out = KvPages{(char *)k->data, (char *)v->data, k->nb[1], k->nb[2], k->nb[3], v->nb[1], v->nb[2], v->nb[3],
                   (int)(k->ne[3] / layers), (int)k->ne[1]};
    return OASR_STATUS_SUCCESS;
}

int seqs_check(oasr_backend *be, const char *op, const oasr_tensor *table, const oasr_tensor *n_past,
               const oasr_tensor *n_nodes, int64_t S, int64_t N, KvSeqs *out) {
    if (!table || !n_past) return fail_op(be, op, "null argument");
    if (S > (1 << 20) || N > (1 << 24) || S * N > INT32_MAX) return fail_op(be, op, "too many sequences or nodes");
    if (table->type != OASR_TYPE_I32 || !table->data || !aligned4(table) || table->ne[1] != S || table->ne[2] != 1 ||
        table->ne[3] != 1 || table->ne[0] < 1 || table->ne[0] > (1 << 24) || (table->nb[0] != 4 && table->ne[0] > 1) || table->nb[1] % 4)
        return fail_op(be, op, "page_table must be I32 [max_pages, n_seq]");
    if (!is_vec_i32(n_past, S)) return fail_op(be, op, "n_past must be I32 [n_seq]");
    if (n_nodes && !is_vec_i32(n_nodes, S)) return fail_op(be, op, "n_nodes must be I32 [n_seq]");
    *out = KvSeqs{(const int *)table->data, table->nb[1] / 4, (int)table->ne[0], (const int *)n_past->data,
                  n_nodes ? (const int *)n_nodes->data : nullptr, (int)N};
    return OASR_STATUS_SUCCESS;
}

}  // namespace oasr

namespace {

// ---- norms, rotation and the cache write -------------------------------------------------
struct NormRope {
    const char *x;
    int64_t x_nb1, x_nb2, x_nb3;  // head, node, sequence
    char *q;
    int64_t q_nb1, q_nb2, q_nb3;
    const float *q_norm, *k_norm;  // [D], or null: no norm
    const float *rope;             // [n_pos][D / 2][2], or null: no rotation
    int n_pos;
    const int *pos;  // [S][N], or null: n_past[s] + i
    int64_t pos_ld;
    int S, H, HKV;
    float eps;
    bool gains8;  // both gains there, and 8-byte aligned
};

// y = x / sqrt(mean(x^2) + eps) * w, then pair (i, i + D/2) turned by the angle of the node's
// position: (a cos - b sin, b cos + a sin).  D / 4 lanes take a head, two neighbouring values and
// the two they turn with per lane, so that the rotation needs no other lane; a warp takes U rounds
// of heads of one node, and what depends on the node alone (lengths, page, angles, gains) is
// fetched once for all of them.  The squares are summed in 64 bits and every product is rounded as in
// the decoders' own norm (qwen_qkv_post_kernel), so that a verification pass writes the bits that a
// decode step writes; the sums of the U rounds share one butterfly (at each step a lane passes on the
// heads its partner keeps).  For prompts bound by HBM and the issue of some 140 instructions per head:
// eight prompts of 512 rows of 16 + 16 heads (97 MB) take 25.7 us, 3.8 TB/s, and eight trees of 61 nodes
// of D = 64 4.5 us.  Sums in 32 bits took 24.3 and 4.2 (with them, two rounds per warp took 30 us for the
// prompts; eight 24, but then the trees 6.4) and left one K value in some 200 heads a bit apart.  For a
// step's few rows by three dependent loads and the launch: 2.5 us.
template <int D, int U, bool QF16>
__global__ void __launch_bounds__(U == 1 ? 256 : 128)
    qk_norm_rope_kernel(NormRope a, KvPages p, KvSeqs sq, FastDiv nodes, FastDiv page, int groups, int *err) {
    constexpr int LPH = D / 4, HPW = 32 / LPH;  // lanes per head, heads per warp and round
    constexpr int W = (U == 1 ? 8 : 4) * HPW;   // heads per block and round
    griddep_launch_dependents();
    griddep_wait();
    const int lane = threadIdx.x & 31, l = lane % LPH;
    const int HH = a.H + 2 * a.HKV;
    const int token = blockIdx.x / groups, h0 = (blockIdx.x - token * groups) * (W * U) + threadIdx.x / LPH;
    const int s = nodes(token), i = token - s * sq.N;
    float2 lo[U], hi[U];  // values 2 l, 2 l + 1 and D / 2 further
    const char *x = a.x + i * a.x_nb2 + s * a.x_nb3 + h0 * a.x_nb1 + 8 * l;
    const int64_t x_step = W * a.x_nb1;
#pragma unroll
    for (int u = 0; u < U; ++u, x += x_step) {
        const int h = h0 + W * u;
        if (h < HH) {
            lo[u] = *reinterpret_cast<const float2 *>(x);
            hi[u] = *reinterpret_cast<const float2 *>(x + 2 * D);
        } else {
            lo[u] = hi[u] = make_float2(0.0f, 0.0f);
        }
    }
    int past, n;
    if (!seq_lengths(sq, s, p.page, past, n) && threadIdx.x == 0) atomicOr(err, ERR_BAD_INDEX);
    const bool live = i < n;
    char *q = a.q + i * a.q_nb2 + s * a.q_nb3 + (QF16 ? 4 : 8) * l;
    constexpr int HALF = QF16 ? D : 2 * D;  // bytes
    if (!live) {  // padding nodes leave zeros in q, nothing in the cache
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int h = h0 + W * u;
            if (h >= a.H) break;
            char *d = q + h * a.q_nb1;
            if (QF16) *reinterpret_cast<uint32_t *>(d) = 0, *reinterpret_cast<uint32_t *>(d + HALF) = 0;
            else *reinterpret_cast<uint2 *>(d) = make_uint2(0, 0), *reinterpret_cast<uint2 *>(d + HALF) = make_uint2(0, 0);
        }
        return;
    }
    // this lane's gains, and the two angles
    float2 wq[2], wk[2], cs[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int c = 2 * l + j * (D / 2);
        if (a.gains8) {
            wq[j] = *reinterpret_cast<const float2 *>(a.q_norm + c);
            wk[j] = *reinterpret_cast<const float2 *>(a.k_norm + c);
        } else {
            wq[j] = a.q_norm ? make_float2(a.q_norm[c], a.q_norm[c + 1]) : make_float2(1.0f, 1.0f);
            wk[j] = a.k_norm ? make_float2(a.k_norm[c], a.k_norm[c + 1]) : make_float2(1.0f, 1.0f);
        }
    }
    if (a.rope) {
        int t = a.pos ? a.pos[s * a.pos_ld + i] : past + i;
        if (t < 0 || t >= a.n_pos) {
            if (lane == 0) atomicOr(err, ERR_BAD_INDEX);
            t = 0;
        }
        const float2 *from = reinterpret_cast<const float2 *>(a.rope + (int64_t)t * D) + 2 * l;
        cs[0] = from[0], cs[1] = from[1];
    }
    const int at = past + i, pj = page(at);
    const int64_t off = at - pj * p.page;
    int pg = sq.table[s * sq.table_ld + pj];
    if (pg < 0 || pg >= p.n_pages) {
        if (lane == 0) atomicOr(err, ERR_BAD_INDEX);
        pg = -1;
    }
    char *k_row = p.k + pg * p.k_nb3 + off * p.k_nb1 + 4 * l, *v_row = p.v + pg * p.v_nb3 + off * p.v_nb1 + 4 * l;
    // sums of squares: lane LPH / U * u of a head's lanes ends with that of round u
    float scale = 0.0f;
    {
        double ss[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            ss[u] = 0.0;
            if (h0 + W * u < a.H + a.HKV)  // value heads have no norm
                ss[u] = ((double)__fmul_rn(lo[u].x, lo[u].x) + (double)__fmul_rn(lo[u].y, lo[u].y)) +
                        ((double)__fmul_rn(hi[u].x, hi[u].x) + (double)__fmul_rn(hi[u].y, hi[u].y));
        }
#pragma unroll
        for (int o = LPH / 2, m = U / 2; o > 0; o >>= 1, m >>= 1) {
            const bool up = lane & o;
            if (m == 0) ss[0] += __shfl_xor_sync(0xffffffffu, ss[0], o);
#pragma unroll
            for (int k = 0; k < m; ++k)
                ss[k] = (up ? ss[k + m] : ss[k]) + __shfl_xor_sync(0xffffffffu, up ? ss[k] : ss[k + m], o);
        }
        scale = __frcp_rn(__fsqrt_rn(__fadd_rn((float)(ss[0] / (double)D), a.eps)));
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int h = h0 + W * u;
        const bool isq = h < a.H, isk = !isq && h < a.H + a.HKV;
        const float sc = U == 1 ? scale : __shfl_sync(0xffffffffu, scale, LPH / U * u, LPH);
        if (h >= HH) continue;
        if (isq ? a.q_norm != nullptr : isk && a.k_norm) {
            const float2 w0 = isq ? wq[0] : wk[0], w1 = isq ? wq[1] : wk[1];
            lo[u] = make_float2(__fmul_rn(__fmul_rn(lo[u].x, sc), w0.x), __fmul_rn(__fmul_rn(lo[u].y, sc), w0.y));
            hi[u] = make_float2(__fmul_rn(__fmul_rn(hi[u].x, sc), w1.x), __fmul_rn(__fmul_rn(hi[u].y, sc), w1.y));
        }
        if (a.rope && (isq || isk)) {
            const float2 f = lo[u], g = hi[u];
            lo[u] = make_float2(__fsub_rn(__fmul_rn(f.x, cs[0].x), __fmul_rn(g.x, cs[0].y)),
                                __fsub_rn(__fmul_rn(f.y, cs[1].x), __fmul_rn(g.y, cs[1].y)));
            hi[u] = make_float2(__fadd_rn(__fmul_rn(f.x, cs[0].y), __fmul_rn(g.x, cs[0].x)),
                                __fadd_rn(__fmul_rn(f.y, cs[1].y), __fmul_rn(g.y, cs[1].x)));
        }
        char *dst = q + h * a.q_nb1;
        if (isq && !QF16) {
            *reinterpret_cast<float2 *>(dst) = lo[u];
            *reinterpret_cast<float2 *>(dst + HALF) = hi[u];
            continue;
        }
        if (!isq) {
            if (pg < 0) continue;
            dst = isk ? k_row + (h - a.H) * p.k_nb2 : v_row + (h - a.H - a.HKV) * p.v_nb2;
        }
        *reinterpret_cast<__half2 *>(dst) = __floats2half2_rn(lo[u].x, lo[u].y);
        *reinterpret_cast<__half2 *>(dst + D) = __floats2half2_rn(hi[u].x, hi[u].y);
    }
}

// ---- acceptance and compaction -------------------------------------------------------------
struct Commit {
    const int *tokens, *parents, *target;  // [S][N]
    int64_t tok_ld, par_ld, tgt_ld;
    int *path;  // [S][N]
    int64_t path_ld;
    int *n_accept, *next, *n_past_out;  // [S]
    int S, L, HKV, D;
    int groups;  // CTAs per sequence
};

// The walk: node 0 is accepted; after node c, the first node j > c with parents[j] = c and
// tokens[j] = target[c].  Every node votes for itself at its parent (atomicMin keeps the first),
// then one thread follows the links.  The accepted path is strictly increasing and path[i] >= i,
// so a thread that moves its 16 bytes of every row in path order, a few rows loaded before they
// are stored, never overwrites a row that it has still to read.  Each CTA repeats the walk and
// moves 256 columns of 16 bytes of (layer, K or V, head).  Bound by HBM's rate for 256-byte rows
// from all over the pages: 32 trees, 13 rows each, 28 layers of 8 heads of 128 (88 MB) take 22 us, 4.0
// TB/s; more CTAs per SM (5 to 7 in the place of 4) take 23 to 25 us, twelve rows at a time 25, four
// 22.  4 us of it, and all of a small call, are the dependent loads up to the first row; those 896 CTAs
// are one and a half waves, and the second wave has them once more.
__global__ void __launch_bounds__(256) tree_commit_kernel(Commit a, KvPages p, KvSeqs sq, FastDiv page, int *err) {
    griddep_launch_dependents();
    griddep_wait();
    __shared__ int s_next[TREE_MAX_NODES], s_path[TREE_MAX_NODES], s_tgt[TREE_MAX_NODES];
    __shared__ int s_len, s_bad;
    const int s = blockIdx.x / a.groups, g = blockIdx.x % a.groups;
    int past, n;
    const bool ok = seq_lengths(sq, s, p.page, past, n);
    if (!ok && threadIdx.x == 0) atomicOr(err, ERR_BAD_INDEX);
    if (threadIdx.x == 0) s_bad = 0;
    for (int c = threadIdx.x; c < n; c += blockDim.x) {
        s_next[c] = n;
        s_tgt[c] = a.target[s * a.tgt_ld + c];
    }
    __syncthreads();
    for (int c = threadIdx.x; c < n; c += blockDim.x) {
        const int up = a.parents[s * a.par_ld + c];
        if (up >= 0 && up < c && a.tokens[s * a.tok_ld + c] == s_tgt[up]) atomicMin(&s_next[up], c);
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        int len = 0;
        for (int c = 0; c < n; c = s_next[c]) s_path[len++] = c;  // links only go forward
        s_len = len;
    }
    __syncthreads();
    const int len = s_len;
    if (g == 0) {
        for (int c = threadIdx.x; c < sq.N; c += blockDim.x) a.path[s * a.path_ld + c] = c < len ? s_path[c] : -1;
        if (threadIdx.x == 0) {
            a.n_accept[s] = len;
            a.next[s] = len ? s_tgt[s_path[len - 1]] : -1;
            a.n_past_out[s] = sq.n_past[s] + len;
        }
        __syncthreads();
    }
    // page and offset of the rows: their sources, and where they go
    __shared__ int s_spg[TREE_MAX_NODES], s_soff[TREE_MAX_NODES], s_doff[TREE_MAX_NODES];
    for (int c = threadIdx.x; c < len; c += blockDim.x) {
        const int from = past + s_path[c], to = past + c;
        const int fj = page(from), tj = page(to);
        const int fp = sq.table[s * sq.table_ld + fj], tp = sq.table[s * sq.table_ld + tj];
        if (fp < 0 || fp >= p.n_pages || tp < 0 || tp >= p.n_pages) s_bad = 1;
        s_spg[c] = fp;
        s_soff[c] = from - fj * p.page;
        s_next[c] = tp;
        s_doff[c] = to - tj * p.page;
    }
    __syncthreads();
    if (s_bad) {
        if (threadIdx.x == 0) atomicOr(err, ERR_BAD_INDEX);
        return;
    }
    const int cpr = a.D / 8;  // 16-byte columns per row
    const int col = g * 256 + threadIdx.x;
    if (col >= a.L * 2 * a.HKV * cpr) return;
    const int c16 = col % cpr, h = col / cpr % a.HKV, kv = col / cpr / a.HKV % 2, l = col / cpr / a.HKV / 2;
    const int64_t nb1 = kv ? p.v_nb1 : p.k_nb1, nb3 = kv ? p.v_nb3 : p.k_nb3;
    char *base = (kv ? p.v : p.k) + (int64_t)l * p.n_pages * nb3 + h * (kv ? p.v_nb2 : p.k_nb2) + 16 * c16;
    constexpr int U = 8;
    for (int b = 1; b < len; b += U) {
        uint4 r[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (b + u < len && s_path[b + u] != b + u)
                r[u] = *reinterpret_cast<const uint4 *>(base + s_spg[b + u] * nb3 + s_soff[b + u] * nb1);
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (b + u < len && s_path[b + u] != b + u)
                *reinterpret_cast<uint4 *>(base + s_next[b + u] * nb3 + s_doff[b + u] * nb1) = r[u];
    }
}

// ---- page copies -------------------------------------------------------------------------
// pair j: page src[j] -> page dst[j] of every layer, K and V; a negative source or destination
// leaves the pair out.  16 bytes per thread and step; FLAT: a page is one run of bytes.  Bound by
// HBM: 64 pages of 64 positions in 28 layers (940 MB read and written) take 142 us, 6.6 TB/s.
template <bool FLAT>
__global__ void __launch_bounds__(256) kv_pages_copy_kernel(const int *pairs, int64_t pair_ld, KvPages p, int L, int HKV,
                                                            int cpr, int chunks, int *err) {
    griddep_launch_dependents();
    griddep_wait();
    constexpr int U = 4;
    const int64_t b = blockIdx.x;
    const int ch = (int)(b % chunks), kv = (int)(b / chunks % 2), l = (int)(b / chunks / 2 % L);
    const int64_t j = b / chunks / 2 / L;
    const int src = pairs[j * pair_ld], dst = pairs[j * pair_ld + 1];
    if (src < 0 || dst < 0) return;
    if (src >= p.n_pages || dst >= p.n_pages) {
        if (threadIdx.x == 0) atomicOr(err, ERR_BAD_INDEX);
        return;
    }
    const int64_t nb1 = kv ? p.v_nb1 : p.k_nb1, nb2 = kv ? p.v_nb2 : p.k_nb2, nb3 = kv ? p.v_nb3 : p.k_nb3;
    char *layer = (kv ? p.v : p.k) + (int64_t)l * p.n_pages * nb3;
    const int total = HKV * p.page * cpr;
    const int e0 = ch * (256 * U) + threadIdx.x;
    uint4 r[U];
    int64_t off[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int e = e0 + 256 * u;
        off[u] = FLAT ? (int64_t)e * 16 : (e / cpr / p.page) * nb2 + (e / cpr % p.page) * nb1 + (e % cpr) * 16;
        if (e < total) r[u] = *reinterpret_cast<const uint4 *>(layer + src * nb3 + off[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (e0 + 256 * u < total) *reinterpret_cast<uint4 *>(layer + dst * nb3 + off[u]) = r[u];
}

int launched(oasr_backend *be, cudaError_t e, const char *what) {
    if (e != cudaSuccess) return oasr_internal_cuda_fail(be, e, what, __LINE__);
    return oasr_internal_launch_check(be, what);
}

bool rows16(const oasr_tensor *t) {
    return ((uintptr_t)t->data & 15) == 0 && t->nb[1] % 16 == 0 && t->nb[2] % 16 == 0 && t->nb[3] % 16 == 0;
}

// I32 [N, S] with contiguous rows
bool is_rows_i32(const oasr_tensor *t, int64_t N, int64_t S) {
    return t && t->type == OASR_TYPE_I32 && t->data && aligned4(t) && t->ne[0] == N && t->ne[1] == S && t->ne[2] == 1 &&
           t->ne[3] == 1 && (t->nb[0] == 4 || N <= 1) && t->nb[1] % 4 == 0;
}

// Rows of I32 on the device: `n` rows of `width` values, `ld` values apart.
struct IntRows {
    const int *at;
    int64_t n, width, ld;
};
IntRows int_rows(const oasr_tensor *t) { return {(const int *)t->data, t->ne[1], t->ne[0], t->ne[1] > 1 ? t->nb[1] / 4 : 0}; }

// Whether the two have a value in common (rows side by side in one buffer have none).
bool share_values(const IntRows &a, const IntRows &b) {
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

}  // namespace

extern "C" {

int oasr_b200_qk_norm_rope(oasr_backend *be, const oasr_tensor *qkv, const oasr_tensor *q_norm, const oasr_tensor *k_norm,
                           float eps, const oasr_tensor *rope, const oasr_tensor *pos, const oasr_tensor *page_table,
                           const oasr_tensor *n_past, const oasr_tensor *n_nodes, oasr_tensor *q, oasr_tensor *k_pages,
                           oasr_tensor *v_pages) {
    int st = oasr_internal_precheck(be);
    if (st) return st;
    const char *op = "qk_norm_rope";
    if (!qkv || !q) return fail_op(be, op, "null argument");
    NormRope a = {};
    KvPages p;
    KvSeqs sq;
    st = pages_check(be, op, k_pages, v_pages, 1, &p);
    if (st) return st;
    const int64_t D = k_pages->ne[0], HKV = k_pages->ne[2], N = qkv->ne[2], S = qkv->ne[3], H = qkv->ne[1] - 2 * HKV;
    if (qkv->type != OASR_TYPE_F32 || qkv->ne[0] != D || H < 1 || H % HKV || H > 65535)
        return fail_op(be, op, "qkv must be F32 [D, H + 2 * H_kv, n, n_seq] with H a multiple of H_kv");
    if ((q->type != OASR_TYPE_F32 && q->type != OASR_TYPE_F16) || q->ne[0] != D || q->ne[1] != H || q->ne[2] != N || q->ne[3] != S)
        return fail_op(be, op, "q must be F32 or F16 [D, H, n, n_seq]");
    for (const oasr_tensor *w : {q_norm, k_norm})
        if (w && (w->type != OASR_TYPE_F32 || !w->data || !aligned4(w) || w->ne[0] != D || w->ne[1] != 1 || w->ne[2] != 1 ||
                  w->ne[3] != 1 || w->nb[0] != 4))
            return fail_op(be, op, "q_norm and k_norm must be F32 [D]");
    if ((q_norm || k_norm) && !(eps >= 0.0f)) return fail_op(be, op, "eps must not be negative");
    if (rope && (rope->type != OASR_TYPE_F32 || !rope->data || rope->ne[0] != 2 || rope->ne[1] != D / 2 || rope->ne[2] < 1 ||
                 rope->ne[2] > INT32_MAX || rope->ne[3] != 1 || rope->nb[0] != 4 || rope->nb[1] != 8 ||
                 (rope->nb[2] != 4 * D && rope->ne[2] > 1) || ((uintptr_t)rope->data & 7)))
        return fail_op(be, op, "rope must be contiguous F32 [2, D / 2, n_pos]");
    if (pos && !is_rows_i32(pos, N, S)) return fail_op(be, op, "pos must be I32 [n, n_seq]");
    if (qkv->nb[0] != 4 || q->nb[0] != (q->type == OASR_TYPE_F16 ? 2 : 4)) return fail_op(be, op, "rows must be contiguous");
    st = seqs_check(be, op, page_table, n_past, n_nodes, S, N, &sq);
    if (st) return st;
    const int64_t units = S * N * qkv->ne[1];
    if (units == 0) return OASR_STATUS_SUCCESS;
    if (!qkv->data || !q->data) return fail_op(be, op, "null argument");
    if (!rows16(qkv) || !rows16(q)) return fail_op(be, op, "rows must be 16-byte aligned");
    a.x = (const char *)qkv->data;
    a.x_nb1 = qkv->nb[1], a.x_nb2 = qkv->nb[2], a.x_nb3 = qkv->nb[3];
    a.q = (char *)q->data;
    a.q_nb1 = q->nb[1], a.q_nb2 = q->nb[2], a.q_nb3 = q->nb[3];
    a.q_norm = q_norm ? (const float *)q_norm->data : nullptr;
    a.k_norm = k_norm ? (const float *)k_norm->data : nullptr;
    a.rope = rope ? (const float *)rope->data : nullptr;
    a.n_pos = rope ? (int)rope->ne[2] : 0;
    a.pos = pos ? (const int *)pos->data : nullptr;
    a.pos_ld = pos ? pos->nb[1] / 4 : 0;
    a.S = (int)S, a.H = (int)H, a.HKV = (int)HKV;
    a.eps = eps;
    a.gains8 = a.q_norm && a.k_norm && (((uintptr_t)a.q_norm | (uintptr_t)a.k_norm) & 7) == 0;
    // four rounds of heads per warp share what belongs to the node (eight prompts of 512 rows: 26 us; 24
    // against 30 with two when the sums were in 32 bits), as long as that leaves every SM some blocks;
    // below that one round per warp, so that a step's few rows start at once
    const int64_t HH = qkv->ne[1], per = D == 64 ? 2 : 1, few = (HH + 8 * per - 1) / (8 * per),
                  many = (HH + 16 * per - 1) / (16 * per);
    const bool share = S * N * many >= 4 * be->sm_count;
    const int groups = (int)(share ? many : few);
    if (S * N * groups > INT32_MAX) return fail_op(be, op, "too many rows");
    const dim3 grid((unsigned)(S * N * groups));
    const FastDiv nodes((int)N), page(p.page);
    const bool f16 = q->type == OASR_TYPE_F16;
    cudaError_t e = cudaSuccess;
#define NR(DD, UU, F)                       \
    if (D == DD && share == (UU == 4) && f16 == F) \
    e = launch_k(be, qk_norm_rope_kernel<DD, UU, F>, grid, dim3(UU == 1 ? 256 : 128), 0, a, p, sq, nodes, page, groups, be->err_word)
    NR(64, 1, false); NR(64, 1, true); NR(64, 4, false); NR(64, 4, true);
    NR(128, 1, false); NR(128, 1, true); NR(128, 4, false); NR(128, 4, true);
#undef NR
    return launched(be, e, op);
}

int oasr_b200_flash_attn_tree(oasr_backend *be, const oasr_tensor *q, const oasr_tensor *k_pages, const oasr_tensor *v_pages,
                              const oasr_tensor *page_table, const oasr_tensor *n_past, const oasr_tensor *n_nodes,
                              const oasr_tensor *tree, float scale, oasr_tensor *dst) {
    int st = oasr_internal_precheck(be);
    if (st) return st;
    const char *op = "flash_attn_tree";
    if (!q || !dst) return fail_op(be, op, "null argument");
    KvPages p;
    KvSeqs sq;
    st = pages_check(be, op, k_pages, v_pages, 1, &p);
    if (st) return st;
    const int64_t D = q->ne[0], N = q->ne[1], H = q->ne[2], S = q->ne[3], HKV = k_pages->ne[2];
    if ((q->type != OASR_TYPE_F32 && q->type != OASR_TYPE_F16) || D != k_pages->ne[0] || H < 1 || H % HKV || H > 65535)
        return fail_op(be, op, "q must be F32 or F16 [D, n, H, n_seq] with H a multiple of H_kv");
    if ((dst->type != OASR_TYPE_F32 && dst->type != OASR_TYPE_F16) || dst->ne[0] != D || dst->ne[1] != H || dst->ne[2] != N ||
        dst->ne[3] != S)
        return fail_op(be, op, "dst must be F32 or F16 [D, H, n, n_seq]");
    if (q->nb[0] != (q->type == OASR_TYPE_F16 ? 2 : 4) || dst->nb[0] != (dst->type == OASR_TYPE_F16 ? 2 : 4))
        return fail_op(be, op, "rows must be contiguous");
    if (!(scale == scale)) return fail_op(be, op, "scale must be a number");
    st = seqs_check(be, op, page_table, n_past, n_nodes, S, N, &sq);
    if (st) return st;
    if (tree && (tree->type != OASR_TYPE_I32 || !aligned4(tree) || tree->ne[0] != (N + 31) / 32 || tree->ne[1] != N ||
                 tree->ne[2] != S || tree->ne[3] != 1 || (tree->nb[0] != 4 && tree->ne[0] > 1) || tree->nb[1] % 4 || tree->nb[2] % 4))
        return fail_op(be, op, "tree must be I32 [ceil(n / 32), n, n_seq]");
    if (tree && N > TREE_MAX_NODES) return fail_op(be, op, "a tree has at most 1024 nodes");
    if (N == 0 || S == 0) return OASR_STATUS_SUCCESS;
    if (!q->data || !dst->data || (tree && !tree->data)) return fail_op(be, op, "null argument");
    if (!rows16(q) || !rows16(dst)) return fail_op(be, op, "rows must be 16-byte aligned");
    TreeAttn a;
    a.q = (const char *)q->data;
    a.q_nb1 = q->nb[1], a.q_nb2 = q->nb[2], a.q_nb3 = q->nb[3];
    a.dst = (char *)dst->data;
    a.d_nb1 = dst->nb[1], a.d_nb2 = dst->nb[2], a.d_nb3 = dst->nb[3];
    a.tree = tree ? (const int *)tree->data : nullptr;
    a.t_nb1 = tree ? tree->nb[1] / 4 : 0, a.t_nb2 = tree ? tree->nb[2] / 4 : 0;
    a.S = (int)S, a.H = (int)H, a.HKV = (int)HKV, a.D = (int)D, a.W = (int)((N + 31) / 32);
    a.scale = scale;
    a.q_f16 = q->type == OASR_TYPE_F16, a.d_f16 = dst->type == OASR_TYPE_F16;
    return launch_flash_attn_tree(be, a, p, sq);
}

int oasr_b200_tree_commit(oasr_backend *be, const oasr_tensor *tokens, const oasr_tensor *parents, const oasr_tensor *target,
                          const oasr_tensor *n_nodes, const oasr_tensor *n_past, const oasr_tensor *page_table,
                          oasr_tensor *k_pages, oasr_tensor *v_pages, int32_t n_layers, oasr_tensor *path,
                          oasr_tensor *n_accept, oasr_tensor *next_token, oasr_tensor *n_past_out) {
    int st = oasr_internal_precheck(be);
    if (st) return st;
    const char *op = "tree_commit";
    if (!tokens || !n_past_out || !n_past) return fail_op(be, op, "null argument");
    KvPages p;
    KvSeqs sq;
    st = pages_check(be, op, k_pages, v_pages, n_layers, &p);
    if (st) return st;
    const int64_t N = tokens->ne[0], S = tokens->ne[1];
    if (N > TREE_MAX_NODES) return fail_op(be, op, "a tree has at most 1024 nodes");
    st = seqs_check(be, op, page_table, n_past, n_nodes, S, N, &sq);
    if (st) return st;
    if (S == 0) return OASR_STATUS_SUCCESS;
    if (N == 0) return fail_op(be, op, "a tree has at least one node");
    if (!is_rows_i32(tokens, N, S) || !is_rows_i32(parents, N, S) || !is_rows_i32(target, N, S) || !is_rows_i32(path, N, S))
        return fail_op(be, op, "tokens, parents, target and path must be I32 [n, n_seq]");
    if (!is_vec_i32(n_accept, S) || !is_vec_i32(next_token, S) || !is_vec_i32(n_past_out, S))
        return fail_op(be, op, "n_accept, next_token and n_past_out must be I32 [n_seq]");
    // every CTA of a sequence walks its tree, while the first of them writes the results
    const oasr_tensor *outs[] = {path, n_accept, next_token, n_past_out};
    const oasr_tensor *ins[] = {tokens, parents, target, n_past, page_table, n_nodes};
    if (S > 1 && llabs(path->nb[1] / 4) < N) return fail_op(be, op, "path's rows must not overlap");
    for (int i = 0; i < 4; ++i) {
        for (const oasr_tensor *t : ins)
            if (t && share_values(int_rows(outs[i]), int_rows(t)))
                return fail_op(be, op, "path, n_accept, next_token and n_past_out must not overlap an input (it is still read "
                                       "while they are written)");
        for (int j = 0; j < i; ++j)
            if (share_values(int_rows(outs[i]), int_rows(outs[j])))
                return fail_op(be, op, "path, n_accept, next_token and n_past_out must not overlap one another");
    }
    Commit a;
    a.tokens = (const int *)tokens->data, a.tok_ld = tokens->nb[1] / 4;
    a.parents = (const int *)parents->data, a.par_ld = parents->nb[1] / 4;
    a.target = (const int *)target->data, a.tgt_ld = target->nb[1] / 4;
    a.path = (int *)path->data, a.path_ld = path->nb[1] / 4;
    a.n_accept = (int *)n_accept->data;
    a.next = (int *)next_token->data;
    a.n_past_out = (int *)n_past_out->data;
    a.S = (int)S, a.L = n_layers, a.HKV = (int)k_pages->ne[2], a.D = (int)k_pages->ne[0];
    const int64_t cols = (int64_t)a.L * 2 * a.HKV * (a.D / 8);
    if (cols > INT32_MAX / 2) return fail_op(be, op, "too many layers");
    a.groups = (int)((cols + 255) / 256);
    if (S * a.groups > INT32_MAX) return fail_op(be, op, "too many sequences");
    return launched(be, launch_k(be, tree_commit_kernel, dim3((unsigned)(S * a.groups)), dim3(256), 0, a, p, sq, FastDiv(p.page),
                                 be->err_word), op);
}

int oasr_b200_kv_pages_copy(oasr_backend *be, oasr_tensor *k_pages, oasr_tensor *v_pages, int32_t n_layers,
                            const oasr_tensor *pairs) {
    int st = oasr_internal_precheck(be);
    if (st) return st;
    const char *op = "kv_pages_copy";
    KvPages p;
    st = pages_check(be, op, k_pages, v_pages, n_layers, &p);
    if (st) return st;
    if (!pairs || pairs->type != OASR_TYPE_I32 || !aligned4(pairs) || pairs->ne[0] != 2 || pairs->ne[2] != 1 ||
        pairs->ne[3] != 1 || pairs->nb[0] != 4 || pairs->nb[1] % 4)
        return fail_op(be, op, "pairs must be I32 [2, n]");
    if (pairs->ne[1] == 0) return OASR_STATUS_SUCCESS;
    if (!pairs->data) return fail_op(be, op, "null argument");
    const int HKV = (int)k_pages->ne[2], cpr = (int)k_pages->ne[0] / 8;
    const int64_t total = (int64_t)HKV * p.page * cpr;
    if (total > INT32_MAX / 2) return fail_op(be, op, "pages too large");
    const int64_t chunks = (total + 1023) / 1024, grid = pairs->ne[1] * n_layers * 2 * chunks;
    if (grid > INT32_MAX) return fail_op(be, op, "too many pages in one call");
    const int64_t row = k_pages->ne[0] * 2, head = row * p.page;
    const bool flat = p.k_nb1 == row && p.v_nb1 == row && (HKV == 1 || (p.k_nb2 == head && p.v_nb2 == head));
    cudaError_t e;
    if (flat) e = launch_k(be, kv_pages_copy_kernel<true>, dim3((unsigned)grid), dim3(256), 0, (const int *)pairs->data,
                           pairs->nb[1] / 4, p, n_layers, HKV, cpr, (int)chunks, be->err_word);
    else e = launch_k(be, kv_pages_copy_kernel<false>, dim3((unsigned)grid), dim3(256), 0, (const int *)pairs->data,
                      pairs->nb[1] / 4, p, n_layers, HKV, cpr, (int)chunks, be->err_word);
    return launched(be, e, op);
}

int oasr_b200_tree_mask(const int32_t *parents, int32_t n, int32_t *words) {
    if (!parents || !words || n < 0 || n > TREE_MAX_NODES) return OASR_STATUS_FAILED;
    const int W = (n + 31) / 32;
    for (int i = 0; i < n; ++i) {
        if (parents[i] >= i || parents[i] < -1) return OASR_STATUS_FAILED;  // a parent comes before its children
        int32_t *row = words + (int64_t)i * W;
        if (parents[i] >= 0) memcpy(row, words + (int64_t)parents[i] * W, W * 4);
        else memset(row, 0, W * 4);
        row[i / 32] = (int32_t)((uint32_t)row[i / 32] | 1u << (i % 32));
    }
    return OASR_STATUS_SUCCESS;
}

}  // extern "C"
