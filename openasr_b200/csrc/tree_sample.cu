// tree_sample.cu -- the token after each node of a drafted tree, drawn from the target's probabilities
// with given uniform numbers; where the draft gives the probabilities that it drew from, the drafted
// children are accepted by rejection first.
//
// Node c has logits l, p(x) = exp((l(x) - m) / T) / Z.  Its children j1 < j2 < ... were drawn from q (the
// draft's row of c).  With r0 = p: child j_k is taken if u0[j_k] q(t) < r_{k-1}(t), t its token; otherwise
// r_k = max(r_{k-1} - q, 0) over its sum.  When no child is left, the token is the first x whose running
// sum of r passes u1[c] times the whole sum.
//
// The borders of that running sum are V numbers in [0, 1): an error e of it gives another token once in
// 1 / (V e) draws, so that with V = 152k sums in 32 bits (e = 1e-7 to 1e-6) would miss in some percent of
// the draws.  Weights and sums are therefore 64-bit, from an exponential made for it (exp16).
#include <cooperative_groups.h>

#include "once_per_device.h"
#include "op_checks.cuh"
#include "pages.cuh"

using namespace oasr;

namespace {

constexpr int NT = 256, NW = NT / 32;

struct Sample {
    const char *x;  // logits [S][N][V]
    int64_t x_nb1, x_nb2;
    const char *q;  // the draft's probabilities, or null
    int64_t q_nb1, q_nb2;
    const float *temp;  // [S], or null: 1
    const float *u;     // [S][N][2]
    int64_t u_ld1, u_ld2;
    const int *tokens, *parents;  // [S][N], with q only
    int64_t tok_ld, par_ld;
    const int *n_nodes;  // [S], or null: N
    int *target;
    int64_t tgt_ld;
    float *logp;  // or null
    int64_t logp_ld;
    int N, V;
};

// ---- the exponential --------------------------------------------------------------------------
// 2^(t / 16) = 2^e 2^(j / 16) 2^(r / 16), k = 16 e + j the integer nearest to t, |r| <= 1/2: the Taylor
// polynomial of degree 5 of 2^(r / 16) (remainder (ln 2 / 32)^6 / 720 = 1.4e-13), 2^(j / 16) from a table
// of 16 (one 8-byte value per pair of banks: no conflicts), 2^e added to its exponent field.  Adding
// 1.5 * 2^52 leaves k in the low word.
constexpr double MAGIC = 6755399441055744.0;
constexpr double LN2_16 = 0.69314718055994530942 / 16, LOG2E_16 = 16 / 0.69314718055994530942;
constexpr double T_LOW = -16000.0;   // below: a weight under 2^-1000 of the reference's
constexpr double T_HIGH = 13000.0;   // above: a new reference is taken
constexpr double B_MOST = 131072.0;  // most |reference / T| (in 1/16 octaves) for l / T in one multiply-add

// 2^(j / 16) with j << 16 taken off its high word, so that adding k << 16 = (16 e + j) << 16 adds e alone
__device__ __forceinline__ double table_entry(int j) {
    const double v = exp2((double)j / 16.0);
    return __hiloint2double(__double2hiint(v) - (j << 16), __double2loint(v));
}

__device__ __forceinline__ void exp16_parts(double t, const double *tab, double &scale, double &poly) {
    const double z = t + MAGIC;
    const int k = __double2loint(z);
    const double r = t - (z - MAGIC);
    constexpr double A1 = LN2_16, A2 = A1 * LN2_16 / 2, A3 = A2 * LN2_16 / 3, A4 = A3 * LN2_16 / 4, A5 = A4 * LN2_16 / 5;
    poly = fma(fma(fma(fma(fma(A5, r, A4), r, A3), r, A2), r, A1), r, 1.0);
    const double v = tab[k & 15];
    scale = __hiloint2double(__double2hiint(v) + (k << 16), __double2loint(v));
}

// for T_LOW <= t <= 16000; 0 below
__device__ __forceinline__ double exp16(double t, const double *tab) {
    if (!(t >= T_LOW)) return 0.0;
    double scale, poly;
    exp16_parts(t, tab, scale, poly);
    return scale * poly;
}

__device__ __forceinline__ bool finite(float v) { return fabsf(v) <= 3.402823466e38f; }

__device__ __forceinline__ double weight(float v, float ref, double C, const double *tab) {
    return finite(v) ? exp16(((double)v - (double)ref) * C, tab) : 0.0;
}

// ---- a warp's share of a row ------------------------------------------------------------------
// The row as 16-byte vectors of the aligned memory that it lies in: element e of it is value e - off.
struct Row {
    const float *base;  // of element 0
    int off, end;       // elements of the row: [off, end)
    __device__ __forceinline__ Row(const char *p, int V) {
        off = (int)(((uintptr_t)p >> 2) & 3);
        base = reinterpret_cast<const float *>(p) - off;
        end = off + V;
    }
    __device__ __forceinline__ int vectors() const { return (end + 3) >> 2; }
    __device__ __forceinline__ float4 load(int j) const {
        if (4 * j >= off && 4 * j + 4 <= end) {
            const int4 r = ldg_stream(base + 4 * (int64_t)j);
            return make_float4(__int_as_float(r.x), __int_as_float(r.y), __int_as_float(r.z), __int_as_float(r.w));
        }
        float v[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) v[c] = 4 * j + c >= off && 4 * j + c < end ? __ldg(base + 4 * (int64_t)j + c) : -INFINITY;
        return make_float4(v[0], v[1], v[2], v[3]);
    }
};

// sum = sum of exp((l - ref) / T); at: of the first maximum (T = 0), ref the maximum
struct Part {
    double sum;
    float ref;
    int at;
};

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

constexpr int U = 4;  // vectors of a lane in flight

__device__ __forceinline__ void load_tile(float4 (&b)[U], const Row &row, int j0, int j1, int lane) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int j = j0 + 32 * u + lane;
        b[u] = j < j1 ? row.load(j) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
    }
}

// any values: the maximum first, then the sum, values that are not finite left out
__device__ __noinline__ Part range_sum_any(Row row, int j0, int j1, double C, const double *tab) {
    const int lane = threadIdx.x & 31;
    float m = -INFINITY;
    for (int j = j0 + lane; j < j1; j += 32) {
        const float4 v = row.load(j);
        for (float f : {v.x, v.y, v.z, v.w})
            if (finite(f)) m = fmaxf(m, f);
    }
    m = warp_max(m);
    double s = 0.0;
    if (m > -INFINITY)
        for (int j = j0 + lane; j < j1; j += 32) {
            const float4 v = row.load(j);
            for (float f : {v.x, v.y, v.z, v.w}) s += weight(f, m, C, tab);
        }
    return Part{warp_sum(s), m, 0};
}

// Vectors [j0, j1) by one warp in one pass.  The reference is the first tile's maximum; a value far above
// it (T_HIGH) makes a new one, so that no maximum has to be known first.  l / T - ref / T is one
// multiply-add of 64 bits.  -inf falls below T_LOW; +inf, NaN and a reference too large for that
// multiply-add (a temperature of some 1e-4 and less) are left to range_sum_any.
__device__ __forceinline__ Part range_sum(const Row &row, int j0, int j1, double C, const double *tab) {
    const int lane = threadIdx.x & 31;
    float ref = -INFINITY, high = -INFINITY;
    double B = 0.0, acc[4] = {0.0, 0.0, 0.0, 0.0};
    bool plain = true;
    float4 next[U];
    load_tile(next, row, j0, j1, lane);
    for (int j = j0; j < j1; j += 32 * U) {
        float4 cur[U];
#pragma unroll
        for (int u = 0; u < U; ++u) cur[u] = next[u];
        if (j + 32 * U < j1) load_tile(next, row, j + 32 * U, j1, lane);
        float m = -INFINITY;
#pragma unroll
        for (int u = 0; u < U; ++u) m = fmaxf(m, fmaxf(fmaxf(cur[u].x, cur[u].y), fmaxf(cur[u].z, cur[u].w)));
        if (__any_sync(0xffffffffu, m > high)) {
            m = warp_max(m);
            plain = finite(m) && fabs((double)m * C) <= B_MOST;
            if (!plain) break;
            const double f = exp16(((double)ref - (double)m) * C, tab);
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[c] *= f;
            ref = m;
            B = -(double)m * C;
            high = (float)((double)m + T_HIGH / C);
        }
        if (ref == -INFINITY) continue;  // nothing finite so far
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const float v[4] = {cur[u].x, cur[u].y, cur[u].z, cur[u].w};
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                double t = fma((double)v[c], C, B);
                // not below T_LOW: negative numbers order by the high word, read without sign, backwards
                t = __hiloint2double((int)min((unsigned)__double2hiint(t), (unsigned)0xC0CF4000u), __double2loint(t));
                double scale, poly;
                exp16_parts(t, tab, scale, poly);
                acc[c] = fma(scale, poly, acc[c]);
            }
        }
    }
    const double s = warp_sum((acc[0] + acc[1]) + (acc[2] + acc[3]));
    if (plain && isfinite(s)) return Part{s, ref, 0};
    return range_sum_any(row, j0, j1, C, tab);
}

// the first of the greatest finite values (argmax_first's choice)
__device__ __forceinline__ Part range_max(const Row &row, int j0, int j1) {
    const int lane = threadIdx.x & 31;
    float best = -INFINITY;
    int at = INT32_MAX;
    for (int j = j0; j < j1; j += 32 * U) {
        float4 b[U];
        load_tile(b, row, j, j1, lane);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const float v[4] = {b[u].x, b[u].y, b[u].z, b[u].w};
#pragma unroll
            for (int c = 0; c < 4; ++c)
                if (v[c] > best && finite(v[c])) best = v[c], at = 4 * (j + 32 * u + lane) + c - row.off;
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float ob = __shfl_xor_sync(0xffffffffu, best, o);
        const int oa = __shfl_xor_sync(0xffffffffu, at, o);
        if (ob > best || (ob == best && oa < at)) best = ob, at = oa;
    }
    return Part{0.0, best, at};
}

// r_k of value x before it is divided by its sum; inv[k]: 1 / the sum of r_{k + 1}, or 0 for one without
// mass (the target's own probabilities then)
__device__ __forceinline__ double residual(double p, float q, const double *inv, int k) {
    const double qq = fmax((double)q, 0.0);
    double r = p;
    for (int i = 0; i < k; ++i) {
        const double rest = fmax(r - qq, 0.0);
        if (i == k - 1) return rest;
        r = inv[i] > 0.0 ? rest * inv[i] : p;
    }
    return r;
}

// Running sums of the ranges' sums, lanes of one warp with W / 32 ranges each; the whole sum comes back.
template <int W>
__device__ __forceinline__ double scan_parts(double (&c)[(W + 31) / 32], double *inc) {
    constexpr int PER = (W + 31) / 32;
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int k = 1; k < PER; ++k) c[k] += c[k - 1];
    double run = c[PER - 1];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const double v = __shfl_up_sync(0xffffffffu, run, o);
        if (lane >= o) run += v;
    }
    double before = __shfl_up_sync(0xffffffffu, run, 1);
    if (lane == 0) before = 0.0;
#pragma unroll
    for (int k = 0; k < PER; ++k)
        if (lane * PER + k < W) inc[lane * PER + k] = k == PER - 1 ? run : before + c[k];
    return __shfl_sync(0xffffffffu, run, 31);
}

// One cluster of CS CTAs per node; every warp takes one run of the row's vectors.  The warps' sums go to
// every CTA of the cluster, which then all take the same decisions, so that the call needs no workspace
// and no second launch; the CTA that holds the drawn value's run reads that run once more.
template <int CS>
__global__ void __launch_bounds__(NT) tree_sample_kernel(Sample a, int *err) {
    namespace cg = cooperative_groups;
    constexpr int W = CS * NW, PER = (W + 31) / 32;
    __shared__ double s_tab[16], s_inc[W], s_rest[W], s_inv[TREE_MAX_NODES], s_warp[NW];
    __shared__ Part s_part[2][W];
    __shared__ double s_total, s_Z;
    __shared__ float s_ref;
    __shared__ int s_kid, s_take, s_at, s_found, s_last;
    griddep_launch_dependents();
    griddep_wait();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int row_id = blockIdx.x / CS, rank = blockIdx.x % CS;
    const int s = row_id / a.N, i = row_id - s * a.N;
    const int n = a.n_nodes ? a.n_nodes[s] : a.N;
    const float T = a.temp ? a.temp[s] : 1.0f;
    const float u1 = a.u[s * a.u_ld2 + i * a.u_ld1 + 1];
    const bool bad = n < 0 || n > a.N || !(T >= 0.0f && T < INFINITY) || (T > 0.0f && i < n && !(u1 >= 0.0f && u1 < 1.0f));
    if (bad || i >= n) {
        if (rank == 0 && tid == 0) {
            if (bad) atomicOr(err, ERR_BAD_INDEX);
            a.target[s * a.tgt_ld + i] = -1;
            if (a.logp) a.logp[s * a.logp_ld + i] = 0.0f;
        }
        return;
    }
    if (CS > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    if (tid < 16) s_tab[tid] = table_entry(tid);
    __syncthreads();
    const char *x = a.x + s * a.x_nb2 + i * a.x_nb1;
    const Row row(x, a.V);
    const int run = (row.vectors() + W - 1) / W;  // vectors of a warp
    const int j0 = min((rank * NW + warp) * run, row.vectors()), j1 = min(j0 + run, row.vectors());
    const double inv_T = T > 0.0f ? 1.0 / (double)T : 0.0, C = LOG2E_16 * inv_T;
    const Part mine = T > 0.0f ? range_sum(row, j0, j1, C, s_tab) : range_max(row, j0, j1);
    if (CS > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // all CTAs have started

    // a warp's part to every CTA of the cluster; then all parts are here
    int parity = 0;
    auto share = [&](const Part &p) {
        if (CS == 1) {
            if (lane == 0) s_part[parity][warp] = p;
            __syncthreads();
        } else {
            cg::cluster_group cl = cg::this_cluster();
            if (lane < CS) *cl.map_shared_rank(&s_part[parity][rank * NW + warp], lane) = p;
            cl.sync();
        }
    };
    auto put = [&](int token, double logp) {
        a.target[s * a.tgt_ld + i] = token;
        if (a.logp) a.logp[s * a.logp_ld + i] = (float)logp;
    };
    share(mine);
    if (T == 0.0f) {
        if (rank == 0 && tid == 0) {
            float best = -INFINITY;
            int at = -1;
            for (int k = 0; k < W; ++k)
                if (s_part[0][k].ref > best) best = s_part[0][k].ref, at = s_part[0][k].at;
            put(at, 0.0);
        }
        return;
    }
    if (warp == 0) {
        float m = -INFINITY;
#pragma unroll
        for (int k = 0; k < PER; ++k)
            if (lane * PER + k < W) m = fmaxf(m, s_part[0][lane * PER + k].ref);
        m = warp_max(m);
        double c[PER];
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            const Part p = lane * PER + k < W ? s_part[0][lane * PER + k] : Part{0.0, -INFINITY, 0};
            c[k] = p.ref > -INFINITY ? p.sum * exp16(((double)p.ref - (double)m) * C, s_tab) : 0.0;
        }
        const double z = scan_parts<W>(c, s_inc);
        if (lane == 0) s_Z = z, s_ref = m;
    }
    __syncthreads();
    const double Z = s_Z, inv_Z = 1.0 / Z;
    const float ref = s_ref;
    if (ref == -INFINITY) {  // no finite logit
        if (rank == 0 && tid == 0) put(-1, 0.0);
        return;
    }
    const float *logits = reinterpret_cast<const float *>(x);
    auto log_p = [&](int t) { return ((double)logits[t] - (double)ref) * inv_T - log(Z); };

    const float *q = reinterpret_cast<const float *>(a.q + s * a.q_nb2 + i * a.q_nb1);
    int rounds = 0;
    double rest = 0.0;  // the last residual's sum
    if (a.q) {
        for (int prev = i;; ) {
            if (tid == 0) s_kid = INT32_MAX;
            __syncthreads();
            for (int j = prev + 1 + tid; j < n; j += NT)
                if (a.parents[s * a.par_ld + j] == i) {
                    atomicMin(&s_kid, j);
                    break;
                }
            __syncthreads();
            const int kid = s_kid;
            if (kid == INT32_MAX) break;
            if (tid == 0) {
                const int t = a.tokens[s * a.tok_ld + kid];
                const float u0 = a.u[s * a.u_ld2 + kid * a.u_ld1];
                s_take = -1;
                if (t < 0 || t >= a.V || !(u0 >= 0.0f && u0 < 1.0f)) {
                    atomicOr(err, ERR_BAD_INDEX);
                } else {
                    const float qt = q[t];
                    double r = residual(weight(logits[t], ref, C, s_tab) * inv_Z, qt, s_inv, rounds);
                    if (rounds) r = s_inv[rounds - 1] > 0.0 ? r * s_inv[rounds - 1] : weight(logits[t], ref, C, s_tab) * inv_Z;
                    if ((double)u0 * (double)qt < r) s_take = t;
                }
            }
            __syncthreads();
            if (s_take >= 0) {
                if (rank == 0 && tid == 0) put(s_take, log_p(s_take));
                return;
            }
            prev = kid;
            ++rounds;
            double sum = 0.0;
            for (int j = j0 + lane; j < j1; j += 32) {
                const float4 v = row.load(j);
                const float w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const int e = 4 * j + c - row.off;
                    if (e >= 0 && e < a.V) sum += residual(weight(w[c], ref, C, s_tab) * inv_Z, __ldg(q + e), s_inv, rounds);
                }
            }
            parity ^= 1;
            share(Part{warp_sum(sum), 0.0f, 0});
            if (warp == 0) {
                double c[PER];
#pragma unroll
                for (int k = 0; k < PER; ++k) c[k] = lane * PER + k < W ? s_part[parity][lane * PER + k].sum : 0.0;
                const double all = scan_parts<W>(c, s_rest);
                if (lane == 0) s_total = all, s_inv[rounds - 1] = all > 0.0 ? 1.0 / all : 0.0;
            }
            __syncthreads();
            rest = s_total;
        }
    }
    // the run in which the running sum passes the drawn value, and the value's place in it
    const bool left = rounds > 0 && rest > 0.0;
    const double *inc = left ? s_rest : s_inc;
    const double drawn = (double)u1 * (left ? rest : Z);
    if (tid == 0) s_at = W - 1;
    if (tid == 0) s_found = INT32_MAX, s_last = -1;
    __syncthreads();
    if (tid < W && inc[tid] > drawn && (tid == 0 || inc[tid - 1] <= drawn)) s_at = tid;
    __syncthreads();
    const int at = s_at;
    if (at / NW != rank) return;
    const int e0 = max(4 * at * run - row.off, 0), e1 = min(4 * (at + 1) * run - row.off, a.V);
    const int per = (e1 - e0 + NT - 1) / NT;
    const int b0 = min(e0 + tid * per, e1), b1 = min(b0 + per, e1);
    auto value = [&](int e) {
        const double w = weight(__ldg(logits + e), ref, C, s_tab);
        return left ? residual(w * inv_Z, __ldg(q + e), s_inv, rounds) : w;
    };
    double own = 0.0;
    int last = -1;  // of the values with any mass
    for (int e = b0; e < b1; ++e) {
        const double v = value(e);
        own += v;
        if (v > 0.0) last = e;
    }
    double scan = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const double v = __shfl_up_sync(0xffffffffu, scan, o);
        if (lane >= o) scan += v;
    }
    if (lane == 31) s_warp[warp] = scan;
    if (last >= 0) atomicMax(&s_last, last);
    __syncthreads();
    double base = at ? inc[at - 1] : 0.0;
    for (int k = 0; k < warp; ++k) base += s_warp[k];
    double before = __shfl_up_sync(0xffffffffu, scan, 1);
    before = lane ? base + before : base;
    if (before <= drawn && base + scan > drawn) {
        int found = last;  // where roundings let the walk miss it
        double cum = before;
        for (int e = b0; e < b1; ++e) {
            cum += value(e);
            if (cum > drawn) {
                found = e;
                break;
            }
        }
        atomicMin(&s_found, found);
    }
    __syncthreads();
    if (tid == 0) {
        const int t = s_found != INT32_MAX ? s_found : s_last;
        put(t, t >= 0 ? log_p(t) : 0.0);
    }
}

// whether the values of out (4 bytes each) and those of a 4-byte tensor [.., n, n_seq] meet
bool meets(const IntRows &out, const oasr_tensor *t) {
    if (!t) return false;
    for (int64_t s = 0; s < t->ne[2]; ++s)
        if (share_values(out, IntRows{(const int *)((const char *)t->data + s * t->nb[2]), t->ne[1], t->ne[0],
                                      t->ne[1] > 1 ? t->nb[1] / 4 : 0}))
            return true;
    return false;
}

bool is_rows3_f32(const oasr_tensor *t, int64_t w, int64_t N, int64_t S) {
    return t && t->type == OASR_TYPE_F32 && t->data && aligned4(t) && t->ne[0] == w && t->ne[1] == N && t->ne[2] == S &&
           t->ne[3] == 1 && (t->nb[0] == 4 || w <= 1) && t->nb[1] % 4 == 0 && t->nb[2] % 4 == 0;
}

template <int CS>
int launch_sample(oasr_backend *be, const Sample &a, int64_t rows) {
    if (rows * CS > INT32_MAX) return fail_op(be, "tree_sample", "too many nodes");
    if (CS > 8) {
        static OncePerDevice wide;
        const cudaError_t e = (cudaError_t)wide(be->device, [] {
            return cudaFuncSetAttribute(tree_sample_kernel<CS>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        });
        if (e != cudaSuccess) return oasr_internal_cuda_fail(be, e, "tree_sample attribute", __LINE__);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(rows * CS));
    cfg.blockDim = dim3(NT);
    cfg.stream = be->stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = CS, attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = be->pdl ? 2 : 1;
    return launched(be, cudaLaunchKernelEx(&cfg, tree_sample_kernel<CS>, a, be->err_word), "tree_sample");
}

}  // namespace

extern "C" int oasr_b200_tree_sample(oasr_backend *be, const oasr_tensor *logits, const oasr_tensor *temperature,
                                     const oasr_tensor *uniforms, const oasr_tensor *tokens, const oasr_tensor *parents,
                                     const oasr_tensor *draft_probs, const oasr_tensor *n_nodes, oasr_tensor *target,
                                     oasr_tensor *logprob) {
    int st = oasr_internal_precheck(be);
    if (st) return st;
    const char *op = "tree_sample";
    if (!logits || !uniforms || !target) return fail_op(be, op, "null argument");
    if (!draft_probs != !tokens || !draft_probs != !parents)
        return fail_op(be, op, "tokens, parents and draft_probs come together");
    const int64_t V = logits->ne[0], N = logits->ne[1], S = logits->ne[2];
    if (S < 0 || N < 0 || S > (1 << 20) || N > (1 << 24) || S * N > INT32_MAX / 16) return fail_op(be, op, "too many nodes");
    if (S == 0 || N == 0) return OASR_STATUS_SUCCESS;
    if (V < 1 || V > (1 << 30)) return fail_op(be, op, "1 to 2^30 tokens");
    if (!is_rows3_f32(logits, V, N, S)) return fail_op(be, op, "logits must be F32 [n_vocab, n, n_seq] with contiguous rows");
    if (!is_rows3_f32(uniforms, 2, N, S)) return fail_op(be, op, "uniforms must be F32 [2, n, n_seq]");
    if (temperature && !is_vec(temperature, OASR_TYPE_F32, S)) return fail_op(be, op, "temperature must be F32 [n_seq]");
    if (n_nodes && !is_vec_i32(n_nodes, S)) return fail_op(be, op, "n_nodes must be I32 [n_seq]");
    if (draft_probs) {
        if (N > TREE_MAX_NODES) return fail_op(be, op, "a tree has at most 1024 nodes");
        if (!is_rows3_f32(draft_probs, V, N, S)) return fail_op(be, op, "draft_probs must be F32 [n_vocab, n, n_seq]");
        if (!is_rows_i32(tokens, N, S) || !is_rows_i32(parents, N, S)) return fail_op(be, op, "tokens and parents must be I32 [n, n_seq]");
    }
    if (!is_rows_i32(target, N, S)) return fail_op(be, op, "target must be I32 [n, n_seq]");
    if (logprob && !is_rows(logprob, OASR_TYPE_F32, N, S)) return fail_op(be, op, "logprob must be F32 [n, n_seq]");
    // a node's results are written while others still read their inputs
    const oasr_tensor *outs[] = {target, logprob}, *ins[] = {logits, uniforms, temperature, tokens, parents, draft_probs, n_nodes};
    for (const oasr_tensor *o : outs) {
        if (!o) continue;
        if (S > 1 && llabs(o->nb[1] / 4) < N) return fail_op(be, op, "rows of target and logprob must not overlap");
        for (const oasr_tensor *t : ins)
            if (meets(int_rows(o), t)) return fail_op(be, op, "target and logprob must not overlap an input");
    }
    if (logprob && share_values(int_rows(target), int_rows(logprob))) return fail_op(be, op, "target and logprob must not overlap");
    Sample a = {};
    a.x = (const char *)logits->data, a.x_nb1 = logits->nb[1], a.x_nb2 = logits->nb[2];
    if (draft_probs) {
        a.q = (const char *)draft_probs->data, a.q_nb1 = draft_probs->nb[1], a.q_nb2 = draft_probs->nb[2];
        a.tokens = (const int *)tokens->data, a.tok_ld = tokens->nb[1] / 4;
        a.parents = (const int *)parents->data, a.par_ld = parents->nb[1] / 4;
    }
    a.temp = temperature ? (const float *)temperature->data : nullptr;
    a.u = (const float *)uniforms->data, a.u_ld1 = uniforms->nb[1] / 4, a.u_ld2 = uniforms->nb[2] / 4;
    a.n_nodes = n_nodes ? (const int *)n_nodes->data : nullptr;
    a.target = (int *)target->data, a.tgt_ld = target->nb[1] / 4;
    if (logprob) a.logp = (float *)logprob->data, a.logp_ld = logprob->nb[1] / 4;
    a.N = (int)N, a.V = (int)V;
    const int64_t rows = S * N;
    // CTAs per node: enough of them for the SMs, of at least 2048 values each
    int cs = 16;
    while (cs > 1 && (rows * cs > 4 * be->sm_count || V < 2048 * cs)) cs /= 2;
    switch (cs) {
    case 16: return launch_sample<16>(be, a, rows);
    case 8: return launch_sample<8>(be, a, rows);
    case 4: return launch_sample<4>(be, a, rows);
    case 2: return launch_sample<2>(be, a, rows);
    default: return launch_sample<1>(be, a, rows);
    }
}
