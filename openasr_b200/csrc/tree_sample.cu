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
// the draws.  Weights and sums are therefore 64-bit, from an exponential made for it (exp_of).
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
// With t = (l - ref) 256 log2(e) / T, exp((l - ref) / T) = 2^(t / 256) = 2^e 2^(j / 256) 2^(r / 256), k = 256 e + j
// the integer nearest to t and |r| <= 1/2: the Taylor polynomial of degree 3 of 2^(r / 256) (remainder
// (ln 2 / 512)^4 / 24 = 1.4e-13), 2^(j / 256) from a table in shared memory, 2^e added to its exponent field.
// Adding 1.5 * 2^52 to t in one multiply-add rounds it and leaves k in the low word, another one gives r.  That
// is seven operations of 64 bits per value; a table of 16 takes two more terms (in a
// loop of nothing else 3.6 values per clock and SM instead of 4.4).
// The table has a copy for each pair of banks, so that the 16 lanes of an access never meet (32 KB).
constexpr double MAGIC = 6755399441055744.0;
constexpr int STEPS = 256, COPIES = 16;
constexpr double LN2 = 0.69314718055994530942;
constexpr double LOW = 1000 * STEPS;   // steps below the reference: a weight under 2^-1000, left out
constexpr double HIGH = 800 * STEPS;   // steps above it: a new reference is taken
constexpr double ROOM = 300 * STEPS;   // a maximum in steps up to which weights are taken relative to exp(0)
constexpr double MOST = 1e6 * STEPS;   // a reference in steps up to which 32 bits resolve what lies LOW below it

struct Table {
    double v[STEPS][COPIES];
    // 2^(j / 256) with j << 12 taken off its high word, so that adding k << 12 = (256 e + j) << 12 adds e alone
    __device__ __forceinline__ void fill() {
        for (int j = threadIdx.x; j < STEPS; j += blockDim.x) {
            const double x = exp2((double)j / STEPS), y = __hiloint2double(__double2hiint(x) - (j << 12), __double2loint(x));
#pragma unroll
            for (int c = 0; c < COPIES; ++c) v[j][(c + j) % COPIES] = y;
        }
    }
};

// acc[i] += 2^(d[i] C / 256), step by step for all N: each step waits for the one before
template <int N>
__device__ __forceinline__ void exp_add(const double (&d)[N], double C, uint32_t tab, double (&acc)[N]) {
    constexpr double A1 = LN2 / STEPS, A2 = A1 * A1 / 2, A3 = A2 * A1 / 3;
    double z[N], v[N], r[N];
#pragma unroll
    for (int i = 0; i < N; ++i) z[i] = fma(d[i], C, MAGIC);
#pragma unroll
    for (int i = 0; i < N; ++i)
        asm volatile("ld.shared.f64 %0, [%1];" : "=d"(v[i]) : "r"((__double2loint(z[i]) & (STEPS - 1)) * (COPIES * 8) + tab));
#pragma unroll
    for (int i = 0; i < N; ++i) r[i] = MAGIC - z[i];
#pragma unroll
    for (int i = 0; i < N; ++i) r[i] = fma(d[i], C, r[i]);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = __hiloint2double(__double2hiint(v[i]) + (__double2loint(z[i]) << 12), __double2loint(v[i]));
#pragma unroll
    for (int i = 0; i < N; ++i) z[i] = fma(A3, r[i], A2);
#pragma unroll
    for (int i = 0; i < N; ++i) z[i] = fma(z[i], r[i], A1);
#pragma unroll
    for (int i = 0; i < N; ++i) z[i] = fma(z[i], r[i], 1.0);
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] = fma(v[i], z[i], acc[i]);
}

// 2^(d C / 256), d C at most 1000 octaves; 0 from 1000 octaves under 1 on
__device__ __forceinline__ double exp_of(double d, double C, uint32_t tab) {
    if (!(d * C > -LOW)) return 0.0;
    const double x[1] = {d};
    double y[1] = {0.0};
    exp_add(x, C, tab, y);
    return y[0];
}

__device__ __forceinline__ bool finite(float v) { return fabsf(v) <= 3.402823466e38f; }

__device__ __forceinline__ double weight(float v, float ref, double C, uint32_t tab) {
    return finite(v) ? exp_of((double)v - (double)ref, C, tab) : 0.0;
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
    __device__ __forceinline__ float4 whole(int j) const {
        const int4 r = ldg_stream(base + 4 * (int64_t)j);
        return make_float4(__int_as_float(r.x), __int_as_float(r.y), __int_as_float(r.z), __int_as_float(r.w));
    }
    __device__ __forceinline__ float4 load(int j) const {  // -inf where the row has no value
        if (4 * j >= off && 4 * j + 4 <= end) return whole(j);
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

// a warp's tile: U vectors per lane
template <int U>
__device__ __forceinline__ void load_tile(float4 (&b)[U], const Row &row, int j, int j1, int lane) {
    if (4 * j >= row.off && j + 32 * U <= j1 && 4 * (j + 32 * U) <= row.end) {
#pragma unroll
        for (int u = 0; u < U; ++u) b[u] = row.whole(j + 32 * u + lane);
    } else {
#pragma unroll
        for (int u = 0; u < U; ++u)
            b[u] = j + 32 * u + lane < j1 ? row.load(j + 32 * u + lane) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
    }
}

// A warp's run of vectors [j0, j1) in at most 32 stretches of `step` vectors (a multiple of 256: whole
// pairs of tiles); lane i keeps the sum of stretch i, so that a drawn value is then looked for in one of
// them alone.
struct Run {
    int j0, j1, step;
    __device__ __forceinline__ int from(int i) const { return min(j0 + i * step, j1); }
};

__device__ __forceinline__ double scaled(double sum, float from, float to, double C, uint32_t tab) {
    return from == to ? sum : from == -INFINITY ? 0.0 : sum * exp_of((double)from - (double)to, C, tab);
}

// any values: the maximum first, then the sums, values that are not finite left out
__device__ __noinline__ Part run_sum_any(Row row, Run run, double C, uint32_t tab) {
    const int lane = threadIdx.x & 31;
    float m = -INFINITY;
    for (int j = run.j0 + lane; j < run.j1; j += 32) {
        const float4 v = row.load(j);
        for (float f : {v.x, v.y, v.z, v.w})
            if (finite(f)) m = fmaxf(m, f);
    }
    m = warp_max(m);
    Part mine{0.0, m, 0};
    if (m > -INFINITY)
        for (int i = 0; run.from(i) < run.j1; ++i) {
            double s = 0.0;
            for (int j = run.from(i) + lane; j < run.from(i + 1); j += 32) {
                const float4 v = row.load(j);
                for (float f : {v.x, v.y, v.z, v.w}) s += weight(f, m, C, tab);
            }
            s = warp_sum(s);
            if (lane == i) mine.sum = s;
        }
    return mine;
}

__device__ __forceinline__ float abs_max3(float a, float b, float c) {
    float m;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(fabsf(a)), "f"(fabsf(b)), "f"(fabsf(c)));
    return m;
}

// The run in one pass, relative to exp(ref / T); ref is 0 as long as the values are of the common size
// (ROOM), so that no maximum has to be known first, the runs' sums need no scaling to one another, and
// the subtraction is left out.  A value far above it makes the tile's maximum the reference.  Values
// 1000 octaves below it and -inf count as 2^-1000; +inf, NaN and a reference too large (a temperature of
// some 1e-5 and less) are left to run_sum_any.  The next tile is on its way while one is summed.
template <int U>
__device__ __forceinline__ Part run_sum(const Row &row, const Run &run, float4 (&a)[U], double C, uint32_t tab) {
    const int lane = threadIdx.x & 31;
    float ref = -INFINITY;  // the first tile's maximum, or 0 where that leaves room on both sides
#pragma unroll
    for (int u = 0; u < U; ++u) ref = fmaxf(ref, fmaxf(fmaxf(a[u].x, a[u].y), fmaxf(a[u].z, a[u].w)));
    ref = warp_max(ref);
    if (fabs((double)ref * C) <= ROOM) ref = 0.0f;
    constexpr int G = 4;    // values at a time
    float low, high, calm;  // between -calm and calm lies nothing under low or over high
    double acc[G] = {};
    auto refer = [&](float m) {
        ref = m;
        low = (float)((double)m - LOW / C);
        high = m == -INFINITY ? m : fminf((float)((double)m + HIGH / C), 3.402823466e38f);
        calm = fminf(high, -low);
    };
    refer(ref);
    bool plain = ref == -INFINITY || fabs((double)ref * C) <= MOST;
    auto add = [&](float4 (&b)[U]) {
        float m = 0.0f;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            m = abs_max3(m, b[u].x, b[u].y);
            m = abs_max3(m, b[u].z, b[u].w);
        }
        if (__any_sync(0xffffffffu, m > calm)) {
            m = -INFINITY;
#pragma unroll
            for (int u = 0; u < U; ++u) m = fmaxf(m, fmaxf(fmaxf(b[u].x, b[u].y), fmaxf(b[u].z, b[u].w)));
            m = warp_max(m);
            if (m > high) {
                plain = finite(m) && fabs((double)m * C) <= MOST;
                if (!plain) return;
                const double f = ref == -INFINITY ? 0.0 : exp_of((double)ref - (double)m, C, tab);
#pragma unroll
                for (int c = 0; c < G; ++c) acc[c] *= f;
                refer(m);
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
                b[u] = make_float4(fmaxf(b[u].x, low), fmaxf(b[u].y, low), fmaxf(b[u].z, low), fmaxf(b[u].w, low));
        }
        if (ref == -INFINITY) return;  // nothing finite so far
#pragma unroll
        for (int u = 0; u < U; ++u) {
            double d[G] = {(double)b[u].x, (double)b[u].y, (double)b[u].z, (double)b[u].w};
            if (ref != 0.0f) {
#pragma unroll
                for (int c = 0; c < G; ++c) d[c] -= (double)ref;
            }
            exp_add(d, C, tab, acc);
        }
    };
    Part mine{0.0, ref, 0};
    float4 b[U];
    constexpr int TILE = 32 * U;
    int done = 0, i = 0;  // vectors of the stretch, and which one
    for (int j = run.j0; j < run.j1 && plain; j += 2 * TILE) {
        if (j + TILE < run.j1) load_tile(b, row, j + TILE, run.j1, lane);
        add(a);
        if (!plain) break;
        if (j + TILE < run.j1) {
            if (j + 2 * TILE < run.j1) load_tile(a, row, j + 2 * TILE, run.j1, lane);
            add(b);
            if (!plain) break;
        }
        if ((done += 2 * TILE) == run.step || j + 2 * TILE >= run.j1) {
            double s = (acc[0] + acc[1]) + (acc[2] + acc[3]);
            s = warp_sum(s);
            plain = isfinite(s);
            if (lane == i) mine = Part{s, ref, 0};
#pragma unroll
            for (int c = 0; c < G; ++c) acc[c] = 0.0;
            done = 0, ++i;
        }
    }
    if (!plain) mine = run_sum_any(row, run, C, tab);
    const float m = warp_max(mine.ref);
    return Part{scaled(mine.sum, mine.ref, m, C, tab), m, 0};
}

// the first of the greatest finite values (argmax_first's choice)
template <int U>
__device__ __forceinline__ Part run_max(const Row &row, const Run &run, float4 (&a)[U]) {
    constexpr int TILE = 32 * U;
    const int lane = threadIdx.x & 31;
    float best = -INFINITY;
    int at = INT32_MAX;
    for (int j = run.j0; j < run.j1; j += TILE) {
        float4 b[U];
        if (j + TILE < run.j1) load_tile(b, row, j + TILE, run.j1, lane);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const float v[4] = {a[u].x, a[u].y, a[u].z, a[u].w};
#pragma unroll
            for (int c = 0; c < 4; ++c)
                if (v[c] > best && finite(v[c])) best = v[c], at = 4 * (j + 32 * u + lane) + c - row.off;
            a[u] = b[u];
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

// A weight is good to 2^-42: a difference from m, if it is more than such errors, above 2^-40 of m; else nothing.
__device__ __forceinline__ double left_of(double m, double difference) {
    return __double2hiint(difference) > max(__double2hiint(m) - (40 << 20), 0) ? difference : 0.0;
}

// r_k of values, k >= 1, from their weights w and q, before it is divided by its sum: r_1 = w - q Z, in units of
// Z, so that nothing is left where p = q = 1; r_{n + 1} = r_n inv[n - 1] - q, inv[n - 1] being 1 / the sum of r_n,
// or 0 for one without mass (then once more from p).  The sums and the draw both have their values from
// here: what has a sum has a value that it came from.
template <int N>
__device__ __forceinline__ void residual(double (&w)[N], double Z, const float (&q)[N], const double *inv, int k) {
    double r[N];
#pragma unroll
    for (int c = 0; c < N; ++c) r[c] = left_of(w[c], fma(-(double)q[c], Z, w[c]));
    for (int n = 1; n < k; ++n) {
        const double g = inv[n - 1];
#pragma unroll
        for (int c = 0; c < N; ++c)
            r[c] = g > 0.0 ? left_of(r[c] * g, fma(r[c], g, -(double)q[c])) : left_of(w[c], fma(-(double)q[c], Z, w[c]));
    }
#pragma unroll
    for (int c = 0; c < N; ++c) w[c] = r[c];
}

// The draft's probabilities of a row's vectors.
struct Draft {
    const float *q;  // of value 0
    bool same;       // lies in 16-byte vectors as the row does
    __device__ __forceinline__ float4 load(const Row &row, int j) const {
        const int e = 4 * j - row.off;
        if (same && 4 * j >= row.off && 4 * j + 4 <= row.end) {
            const int4 r = ldg_stream(q + e);
            return make_float4(__int_as_float(r.x), __int_as_float(r.y), __int_as_float(r.z), __int_as_float(r.w));
        }
        float v[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) v[c] = 4 * j + c >= row.off && 4 * j + c < row.end ? __ldg(q + e + c) : 0.0f;
        return make_float4(v[0], v[1], v[2], v[3]);
    }
};

// Weights of four values: 0 from 1000 octaves under the reference on, and for what is not finite; `plain`: there
// is nothing of the kind.
__device__ __forceinline__ void weights(const float4 &x, float ref, double C, uint32_t tab, double (&w)[4], bool plain = false) {
    const float v[4] = {x.x, x.y, x.z, x.w};
    double d[4];
    unsigned none = 0;
#pragma unroll
    for (int c = 0; c < 4; ++c) d[c] = (double)v[c] - (double)ref, w[c] = 0.0;
    if (!plain) {
#pragma unroll
        for (int c = 0; c < 4; ++c)
            if (!(d[c] * C > -LOW) || !finite(v[c])) d[c] = 0.0, none |= 1u << c;
    }
    exp_add(d, C, tab, w);
    if (!plain) {
#pragma unroll
        for (int c = 0; c < 4; ++c)
            if (none >> c & 1) w[c] = 0.0;
    }
}

// The sums over the run's stretches of r_k (residual), or of the weights for k = 0.  Where all of a tile lies
// between -calm and calm it is finite and less than 1000 octaves below the reference.
__device__ __forceinline__ Part run_rest(const Row &row, const Draft &q, const Run &run, float ref, float calm, double Z, double C,
                                         uint32_t tab, const double *inv, int k) {
    const int lane = threadIdx.x & 31;
    constexpr int U = 2;
    Part mine{0.0, ref, 0};
    float4 nx[U], ny[U];
    auto load = [&](int j) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int at = j + 32 * u + lane;
            nx[u] = at < run.j1 ? row.load(at) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
            ny[u] = at < run.j1 ? q.load(row, at) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
    };
    load(run.j0);
    double acc[4] = {};
    int done = 0, i = 0;
    for (int j = run.j0; j < run.j1; j += 32 * U) {
        const float4 x[U] = {nx[0], nx[1]}, y[U] = {ny[0], ny[1]};
        if (j + 32 * U < run.j1) load(j + 32 * U);
        const float m = abs_max3(abs_max3(x[0].x, x[0].y, x[0].z), abs_max3(x[0].w, x[1].x, x[1].y), fmaxf(fabsf(x[1].z), fabsf(x[1].w)));
        // the maximum leaves NaN out, the sum does not
        const bool all = __all_sync(0xffffffffu, m <= calm && x[0].x + x[0].y + x[0].z + x[0].w + x[1].x + x[1].y + x[1].z + x[1].w < INFINITY);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const float f[4] = {y[u].x, y[u].y, y[u].z, y[u].w};
            double w[4];
            weights(x[u], ref, C, tab, w, all);
            if (k) residual(w, Z, f, inv, k);
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[c] += w[c];
        }
        if ((done += 32 * U) == run.step || j + 32 * U >= run.j1) {
            const double s = warp_sum((acc[0] + acc[1]) + (acc[2] + acc[3]));
            if (lane == i) mine.sum = s;
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[c] = 0.0;
            done = 0, ++i;
        }
    }
    return mine;
}

// running sum over the first N lanes
template <int N = 32>
__device__ __forceinline__ double scan(double v) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 1; o < N; o <<= 1) {
        const double w = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += w;
    }
    return v;
}

// The sums of a row's weights by stretch, warp and CTA, and where a drawn value lies.
template <int CS>
struct Sums {
    double stretch[NW][32], stretch_to[NW][32];  // of a warp's stretches, and up to them, relative to the CTA's reference
    double warp[NW], warp_to[NW];                // of the warps
    double cta[2][CS];       // sums of the cluster's CTAs (two calls in turn), relative to
    float cta_ref[2][CS];    // their references
    float warp_ref[NW];
    int cta_at[2][CS];       // T = 0: of the maximum (cta_ref)
};

// A child's token (-1: none that is one), and what it is tried with: its uniform number, its token's
// probability in the draft, and its logit.
struct Try {
    int token;
    float u, q, l;
};

// Where a drawn value lies: CTA, warp, stretch, and the running sum up to there.
struct Place {
    int cta, warp, stretch;
    double before;
};

// `mine`: this lane's stretch, relative to the warp's reference.  Then the sums are everywhere, `all` is the
// whole row's and `ref` what it is relative to; f: what this lane's CTA's are to be multiplied by, `to` the
// running sum up to it.
template <int CS>
__device__ __forceinline__ void gather(Sums<CS> &s, int turn, int rank, const Part &mine, double C, uint32_t tab, double &all, float &ref,
                                       double &to, double &f) {
    namespace cg = cooperative_groups;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (lane == 0) s.warp_ref[warp] = mine.ref;
    __syncthreads();
    const float m = warp_max(lane < NW ? s.warp_ref[lane] : -INFINITY);
    const double own = scaled(mine.sum, mine.ref, m, C, tab), up = scan(own);
    s.stretch[warp][lane] = own, s.stretch_to[warp][lane] = up;
    __syncthreads();
    if (warp == 0) {
        const double of_warp = lane < NW ? s.stretch_to[lane][31] : 0.0, w = scan<NW>(of_warp);
        if (lane < NW) s.warp[lane] = of_warp, s.warp_to[lane] = w;
        const double total = __shfl_sync(0xffffffffu, w, NW - 1);
        if (CS == 1) {
            if (lane == 0) s.cta[turn][0] = total, s.cta_ref[turn][0] = m;
        } else if (lane < CS) {
            cg::cluster_group cl = cg::this_cluster();
            *cl.map_shared_rank(&s.cta[turn][rank], lane) = total;
            *cl.map_shared_rank(&s.cta_ref[turn][rank], lane) = m;
        }
    }
    if (CS == 1) __syncthreads();
    else cg::this_cluster().sync();
    const float r = lane < CS ? s.cta_ref[turn][lane] : -INFINITY;
    ref = warp_max(r);
    f = lane < CS ? scaled(1.0, r, ref, C, tab) : 0.0;
    to = scan<CS>(lane < CS ? s.cta[turn][lane] * f : 0.0);
    all = __shfl_sync(0xffffffffu, to, CS - 1);
}

// The first of N lanes with mass whose running sum `to` is greater than `drawn`, the last with mass if roundings
// leave none; `before` then is the running sum up to it.  Running sums of lanes next to one another are
// rounded differently, so that one may rise past `drawn` at a lane that adds nothing: mass is more than `least`.
template <int N>
__device__ __forceinline__ int first_past(double own, double to, double least, double drawn, double &before) {
    const int lane = threadIdx.x & 31;
    const unsigned mass = __ballot_sync(0xffffffffu, lane < N && own > least), past = __ballot_sync(0xffffffffu, to > drawn) & mass;
    const int at = past ? __ffs(past) - 1 : 31 - __clz(mass | 1u);
    const double up = __shfl_sync(0xffffffffu, to, max(at - 1, 0));
    if (at) before = up;
    return at;
}

// The place whose running sum is the first to pass `drawn`.  Its sum is more than 2^-210 of the whole (there is
// such a stretch in such a warp of such a CTA: the greatest of 16, 8 and 32 parts), far above what values
// without weight may have been counted as.
template <int CS>
__device__ __forceinline__ Place find(const Sums<CS> &s, int turn, double all, double to, double f, double drawn, int rank) {
    const int lane = threadIdx.x & 31;
    Place p;
    p.before = 0.0;
    p.cta = first_past<CS>(lane < CS ? s.cta[turn][lane] * f : 0.0, to, all * 0x1p-200, drawn, p.before);
    if (p.cta != rank) return p;
    f = __shfl_sync(0xffffffffu, f, p.cta);
    const int w = min(lane, NW - 1);
    p.warp = first_past<NW>(f * s.warp[w], p.before + f * s.warp_to[w], all * 0x1p-204, drawn, p.before);
    p.stretch = first_past<32>(f * s.stretch[p.warp][lane], p.before + f * s.stretch_to[p.warp][lane], all * 0x1p-210, drawn, p.before);
    return p;
}

// One cluster of CS CTAs per node; every warp takes one run of the row's vectors.  The CTAs' sums go to
// every CTA of the cluster, which then all take the same decisions, so that the call needs no workspace
// and no second launch; the CTA that holds the drawn value's stretch reads that stretch once more.
// Many nodes (1952 of 151936: 266 us, 4.1 TB/s) take 18.8 instructions a value, 7.7 of them of 64 bits, which keep
// the issue slot for a second cycle: with those, slots are taken 72% of the time a CTA runs.  A loop of nothing but
// loads, weights and sum takes 215 us; the other 50 are starts, gathers and draws, which one other CTA per SM
// (126 registers) hides in part, and in the loop a warp waits 2.2 of the 6.4 cycles between two of its instructions
// for its own results, 1.2 for memory.  CTAs that take one node after another with the next one's first tile
// ahead were slower (300 to 324: the nodes are then dealt out evenly, not as CTAs end), and so were three CTAs
// per SM (272).  A few nodes are a chain of latencies: 2500 cycles to the first values, 2600 for a warp's tile,
// 2400 to gather the sums over a cluster, 2400 for the drawn value (one token of 51866: 8.3 us).
template <int CS, int U, bool DRAFT>
__global__ void __launch_bounds__(NT, 2) tree_sample_kernel(Sample a, int *err) {
    namespace cg = cooperative_groups;
    constexpr int W = CS * NW;
    __shared__ Table s_table;
    __shared__ Sums<CS> s_sums;
    __shared__ double s_inv[DRAFT ? TREE_MAX_NODES : 1], s_warp[NW], s_log;
    __shared__ unsigned short s_kids[DRAFT ? TREE_MAX_NODES : 1];
    __shared__ int s_n_kids, s_last, s_first;
    __shared__ Try s_try[32];  // of the first children
    griddep_launch_dependents();
    griddep_wait();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int row_id = blockIdx.x / CS, rank = blockIdx.x % CS;
    const int s = row_id / a.N, i = row_id - s * a.N;
    const char *x = a.x + s * a.x_nb2 + i * a.x_nb1;
    const Row row(x, a.V);
    const int per = (row.vectors() + W - 1) / W, step = max((per + 32 * 64 * U - 1) / (32 * 64 * U), 1) * 64 * U;
    auto run_of = [&](int cta, int warp) {
        const int j0 = min((cta * NW + warp) * per, row.vectors());
        return Run{j0, min(j0 + per, row.vectors()), step};
    };
    const Run run = run_of(rank, warp);
    const float4 zero = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float4 first[U];
    load_tile(first, row, run.j0, run.j1, lane);
    const int n = a.n_nodes ? a.n_nodes[s] : a.N;
    const float T = a.temp ? a.temp[s] : 1.0f;
    const float u1 = a.u[s * a.u_ld2 + i * a.u_ld1 + 1];
    s_table.fill();
    if (tid == 0) s_last = -1, s_first = NT;
    const uint32_t tab = (uint32_t)__cvta_generic_to_shared(&s_table.v[0][tid % COPIES]);
    auto put = [&](int token, double logp) {
        a.target[s * a.tgt_ld + i] = token;
        if (a.logp) a.logp[s * a.logp_ld + i] = (float)logp;
    };
    const bool bad = n < 0 || n > a.N || !(T >= 0.0f && T < INFINITY) || (T > 0.0f && i < n && !(u1 >= 0.0f && u1 < 1.0f));
    if (bad || i >= n) {
        if (rank == 0 && tid == 0) {
            if (bad) atomicOr(err, ERR_BAD_INDEX);
            put(-1, 0.0);
        }
        return;
    }
    if (CS > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    const float *logits = reinterpret_cast<const float *>(x);
    const float *q = reinterpret_cast<const float *>(a.q + s * a.q_nb2 + i * a.q_nb1);
    auto child = [&](int j) {
        Try t{a.tokens[s * a.tok_ld + j], a.u[s * a.u_ld2 + j * a.u_ld1], 0.0f, 0.0f};
        if (t.token < 0 || t.token >= a.V || !(t.u >= 0.0f && t.u < 1.0f)) {
            if (rank == 0) atomicOr(err, ERR_BAD_INDEX);
            t.token = -1;
        } else {
            t.q = q[t.token], t.l = logits[t.token];
        }
        return t;
    };
    if (DRAFT && warp == 0 && T > 0.0f) {  // the node's children in order
        int count = 0;
        for (int j0 = i + 1; j0 < n; j0 += 32) {
            const int j = j0 + lane;
            const bool is = j < n && a.parents[s * a.par_ld + j] == i;
            const unsigned all = __ballot_sync(0xffffffffu, is);
            if (is) s_kids[count + __popc(all & ((1u << lane) - 1))] = (unsigned short)j;
            count += __popc(all);
        }
        if (lane == 0) s_n_kids = count;
        __syncwarp();
        if (lane < count) s_try[lane] = child(s_kids[lane]);
    }
    __syncthreads();
    if (T == 0.0f) {
        const Part best = run_max(row, run, first);
        if (lane == 0) s_sums.warp_ref[warp] = best.ref, s_sums.stretch[warp][0] = best.at;
        if (CS > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // all CTAs have started
        __syncthreads();
        auto most = [&](float v, int at) {  // the first of the greatest over the lanes
            const float m = warp_max(v);
            const unsigned is = __ballot_sync(0xffffffffu, v == m && m > -INFINITY);
            return Part{0.0, m, is ? __shfl_sync(0xffffffffu, at, __ffs(is) - 1) : -1};
        };
        if (warp == 0) {
            const Part p = most(lane < NW ? s_sums.warp_ref[lane] : -INFINITY, lane < NW ? (int)s_sums.stretch[lane][0] : 0);
            if (lane == 0) {
                int *at = &s_sums.cta_at[0][rank];
                float *ref = &s_sums.cta_ref[0][rank];
                if (CS > 1) at = cg::this_cluster().map_shared_rank(at, 0), ref = cg::this_cluster().map_shared_rank(ref, 0);
                *at = p.at, *ref = p.ref;
            }
        }
        if (CS == 1) __syncthreads();
        else cg::this_cluster().sync();
        if (rank == 0 && warp == 0) {
            const Part p = most(lane < CS ? s_sums.cta_ref[0][lane] : -INFINITY, lane < CS ? s_sums.cta_at[0][lane] : 0);
            if (lane == 0) put(p.at, 0.0);
        }
        return;
    }
    const double inv_T = 1.0 / (double)T, C = STEPS / LN2 * inv_T;
    const Part mine = run_sum(row, run, first, C, tab);
    if (CS > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // all CTAs have started
    double Z, to, f;
    float ref;
    int turn = 0;  // of the sums that the token is drawn from
    gather(s_sums, 0, rank, mine, C, tab, Z, ref, to, f);
    if (ref == -INFINITY) {  // no finite logit
        if (rank == 0 && tid == 0) put(-1, 0.0);
        return;
    }
    const Draft draft{q, (((uintptr_t)q ^ (uintptr_t)logits) & 15) == 0};
    int rounds = 0;
    bool left = false;  // something is left of p
    double total = Z;
    if (DRAFT) {
        const double inv_Z = 1.0 / Z;
        // 64 steps of the 1000 octaves are left for its rounding to 32 bits
        const float low = (float)((double)ref - (LOW - 64) / C), calm = fabs((double)ref * C) <= MOST ? fminf(-low, 3.402823466e38f) : -1.0f;
        auto rest = [&](int k) { return run_rest(row, draft, run, ref, calm, Z, C, tab, s_inv, k); };
        const int kids = s_n_kids;
        while (rounds < kids) {
            const Try t = rounds < 32 ? s_try[rounds] : child(s_kids[rounds]);
            if (t.token >= 0) {
                double w[1] = {weight(t.l, ref, C, tab)};
                const float f[1] = {t.q};
                if (left) residual(w, Z, f, s_inv, rounds);
                if ((double)t.u * (double)t.q < w[0] * (left ? s_inv[rounds - 1] : inv_Z)) {
                    if (rank == 0 && tid == 0) put(t.token, ((double)t.l - (double)ref) * inv_T - log(Z));
                    return;
                }
            }
            ++rounds;
            float same;
            turn ^= 1;
            gather(s_sums, turn, rank, rest(rounds), C, tab, total, same, to, f);
            left = total > 0x1p-1000 && total < INFINITY;  // (a draft's -inf or NaN leaves p, not a sum without a place)
            if (tid == 0) s_inv[rounds - 1] = left ? 1.0 / total : 0.0;
            __syncthreads();
        }
        if (rounds && !left) {  // p once more
            turn ^= 1;
            gather(s_sums, turn, rank, rest(0), C, tab, total, ref, to, f);
        }
    }
    // a number on a border belongs to the value behind it, however the sums up to there were rounded
    const double drawn = (double)u1 * total + total * 0x1p-44;
    const Place at = find(s_sums, turn, total, to, f, drawn, rank);
    if (at.cta != rank) return;
    if (tid == NT - 1) s_log = log(Z);
    // the value's place in its stretch: `each` vectors of a thread, one after the other
    const Run found = run_of(rank, at.warp);
    const int j0 = found.from(at.stretch), j1 = found.from(at.stretch + 1), each = (step + NT - 1) / NT;
    auto values = [&](int j, const float4 &v, double (&w)[4]) {
        weights(v, ref, C, tab, w);
        if (DRAFT && left) {
            const float4 y = j < j1 ? draft.load(row, j) : zero;
            const float g[4] = {y.x, y.y, y.z, y.w};
            residual(w, Z, g, s_inv, rounds);
        }
    };
    const int b0 = j0 + tid * each, b1 = min(b0 + each, j1);
    double own = 0.0, w[4];
    int last = -1;  // of the values with any mass
    for (int j = b0; j < b1; ++j) {
        values(j, row.load(j), w);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            own += w[c];
            if (w[c] > 0.0) last = 4 * j + c;
        }
    }
    const double up = scan(own);
    if (lane == 31) s_warp[warp] = up;
    if (last >= 0) atomicMax(&s_last, last);
    __syncthreads();
    double base = at.before;
    for (int k = 0; k < warp; ++k) base += s_warp[k];
    double before = __shfl_up_sync(0xffffffffu, up, 1);
    before = lane ? base + before : base;
    // the first thread with mass whose running sum passes `drawn`; where roundings leave none, the last value with mass
    const unsigned past = __ballot_sync(0xffffffffu, last >= 0 && base + up > drawn);
    if (past && lane == __ffs(past) - 1) atomicMin(&s_first, tid);
    __syncthreads();
    auto report = [&](int e) { put(e - row.off, ((double)row.base[e] - (double)ref) * inv_T - s_log); };
    if (tid == s_first) {
        int e = -1;
        double cum = before;
        for (int j = b0; j < b1; ++j) {
            if (each > 1) values(j, row.load(j), w);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                cum += w[c];
                if (e < 0 && w[c] > 0.0 && cum > drawn) e = 4 * j + c;
            }
        }
        report(e < 0 ? last : e);
    }
    if (s_first == NT && tid == 0) report(s_last);
}

bool is_rows3_f32(const oasr_tensor *t, int64_t w, int64_t N, int64_t S) {
    return t && t->type == OASR_TYPE_F32 && t->data && aligned4(t) && t->ne[0] == w && t->ne[1] == N && t->ne[2] == S &&
           t->ne[3] == 1 && (t->nb[0] == 4 || w <= 1) && t->nb[1] % 4 == 0 && t->nb[2] % 4 == 0;
}

template <int CS, int U, bool DRAFT>
int launch_sample(oasr_backend *be, const Sample &a, int64_t rows) {
    if (rows * CS > INT32_MAX) return fail_op(be, "tree_sample", "too many nodes");
    if (CS > 8) {
        static OncePerDevice wide;
        const cudaError_t e = (cudaError_t)wide(be->device, [] {
            return cudaFuncSetAttribute(tree_sample_kernel<CS, U, DRAFT>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
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
    return launched(be, cudaLaunchKernelEx(&cfg, tree_sample_kernel<CS, U, DRAFT>, a, be->err_word), "tree_sample");
}

}  // namespace

extern "C" int oasr_b200_tree_sample(oasr_backend *be, const oasr_tensor *logits, const oasr_tensor *temperature,
                                     const oasr_tensor *uniforms, const oasr_tensor *tokens, const oasr_tensor *parents,
                                     const oasr_tensor *draft_probs, const oasr_tensor *n_nodes, oasr_tensor *target,
                                     oasr_tensor *logprob) {
    const char *op = "tree_sample";
    if (!be) return oasr_internal_precheck(be);
    if (!logits || !uniforms || !target) return fail_op(be, op, "null argument");
    if (!draft_probs != !tokens || !draft_probs != !parents)
        return fail_op(be, op, "tokens, parents and draft_probs come together");
    const int64_t V = logits->ne[0], N = logits->ne[1], S = logits->ne[2];
    if (S < 0 || N < 0 || S > (1 << 20) || N > (1 << 24) || S * N > INT32_MAX / 16) return fail_op(be, op, "too many nodes");
    if (S == 0 || N == 0) return oasr_internal_precheck(be);
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
            if (share_bytes(o, t)) return fail_op(be, op, "target and logprob must not overlap an input");
    }
    if (share_bytes(target, logprob)) return fail_op(be, op, "target and logprob must not overlap");
    const int st = oasr_internal_precheck(be);  // the arguments need no device
    if (st) return st;
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
    // CTAs per node: enough of them for the SMs, of at least 2048 values each.  Without a draft two per SM (8
    // nodes of 151936: 10.3 us with 16 CTAs each, 12.4 with 8, 15.1 with 4; 1952 nodes: 266 us with one, 315
    // with two).  With one, nodes whose children are rejected take two to four times as long as the others, and
    // more and smaller CTAs even that out (64 nodes: 38.7 us with 4, 37.5 with 8, 49.5 with 16; 124 of 51866: 43,
    // 31.4, 30.8 and 47 us with 2, 4, 8 and 16).
    const int most = draft_probs ? 8 : 16, per_sm = draft_probs ? 8 : 2;
    int cs = most;
    while (cs > 1 && (rows * cs > per_sm * be->sm_count || V < 2048 * cs)) cs /= 2;
    switch (cs) {
    case 16: return launch_sample<16, 4, false>(be, a, rows);
    case 8: return draft_probs ? launch_sample<8, 4, true>(be, a, rows) : launch_sample<8, 4, false>(be, a, rows);
    case 4: return draft_probs ? launch_sample<4, 4, true>(be, a, rows) : launch_sample<4, 4, false>(be, a, rows);
    case 2: return draft_probs ? launch_sample<2, 8, true>(be, a, rows) : launch_sample<2, 8, false>(be, a, rows);
    default: return draft_probs ? launch_sample<1, 8, true>(be, a, rows) : launch_sample<1, 8, false>(be, a, rows);
    }
}
