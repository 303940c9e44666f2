// fattn_tree.cu -- attention for a tree of drafted tokens over the paged K/V cache.
//
//   o[i, h, s] = sum_p softmax_p(scale q[i, h, s] . k_p) v_p   over the visible positions p:
//   p < n_past[s], or p = n_past[s] + j with bit j of tree[s][i] set (no tree: j <= i);
// a node that sees nothing, or that is padding, gets zeros.
//
// K and V dominate the traffic, so the G query heads of a K/V head and the nodes of a sequence
// share a tile of R = 16, 32, 64 or 128 rows and one read of K and V.  The rows are few, the
// positions many: both products run on the tcgen05 tensor cores with the long side as M,
//   S^T (128 positions x R) = K (128 x D) . Q^T        both operands as they lie (K-major)
//   O^T (D x R)             = V^T (D x 128) . P^T      V as it lies (M-major), P as written
// so no row of the matrix unit is padding, K and V are used in the layout of the pages, and the
// work of the softmax threads -- one per position, R weights each -- shrinks with R.
//
// f32 accuracy from 16-bit operands: an f32 query (after a power of two that brings the row's
// largest value to 2^8) and every weight are two f16 halves, hi + lo, 22 bits; both go through
// the same product, added in the f32 accumulator.  A unit's O^T is added to the running output
// in registers, because the tensor cores cut off the bits below a large accumulator.
//
// Softmax: a weight is 2^(s - off), off = (a maximum seen before) - 7.  As long as no score
// exceeds off by more than 15, f16 holds the weight and nothing is rescaled; one vote of the 128
// threads per unit decides, and only then are the true maxima found and the sums rescaled.
//
// CTA: one group of 4 softmax warps for 16 rows, two for 32 or 64, one TMA warp that streams K and
// V tiles of 128 positions (boxes that end with the pages) through a ring, one MMA warp.  S^T of
// the next unit is computed while this one's weights are; every wait is bounded.
//
// Long calls are bound by HBM: sixteen sequences of 4001 to 8190 positions, 8 K/V heads of 128, 16 rows
// (402 MB), take 69 us, 5.8 TB/s, 90 % of a plain copy; 32 sequences of one token 76 us, 93 %.  Short
// ones by the start and the end of a CTA (code and lengths from far away, the first tiles, the join):
// 8.8 us for one token after 390 positions.  Warp-level matrix instructions took 94 us for the first,
// scores with rows as the long side 16 us for the last.
#include <cudaTypedefs.h>

#include <algorithm>

#include "fattn_tree.cuh"

namespace oasr {

template <int D_, int RW_, int NWG_, bool QF16_>
struct TreeTc {
    static constexpr int D = D_, RW = RW_, NWG = NWG_, R = RW * NWG;
    static constexpr bool QF16 = QF16_;
    // The halves of P are 2 RW columns of one product, and so are those of Q: K and V are fetched
    // from shared memory once for both.
    static constexpr int SCOLS = QF16 ? R : 2 * R;
    // A group has the weights of PB units under way: while one is multiplied the next one's are made.
    static constexpr int PB = NWG == 1 ? 1 : 2;
    static constexpr int HALF = TREE_BKV * 128;          // 128 positions x 64 values
    static constexpr int TILE = HALF * (D / 64);         // one K or V tile
    static constexpr int QROWS = QF16 ? R : 2 * R;       // rows of Q hi, then of Q lo
    static constexpr int QHALF = QROWS * 128;            // they x 64 values
    static constexpr int QBYTES = QHALF * (D / 64);
    static constexpr int PBYTES = TREE_BKV * RW * 2;     // a group's P hi, its P lo follows
    static constexpr int PGROUP = PB * 2 * PBYTES;       // a group's units
    static constexpr int CTAS = NWG == 1 ? 2 : 1;
    static constexpr int MISC = CTAS == 2 ? 1024 : 3072;
    static constexpr int FIXED = QBYTES + NWG * PGROUP + MISC;
    static constexpr int MOST = (CTAS == 2 ? 115712 : 232448) - FIXED;
    static constexpr int NS = MOST / TILE > 8 ? 8 : MOST / TILE;  // tiles in flight
    static_assert(NS >= 3, "K of the next unit and K, V of this one");
    static constexpr int OFF_Q = NS * TILE;
    static constexpr int OFF_P = OFF_Q + QBYTES;
    static constexpr int OFF_MISC = OFF_P + NWG * PGROUP;
    // misc: off[R], query factors [R], see[NWG][4][RW], barriers, flags
    static constexpr int OFF_FAC = OFF_MISC + 4 * R;
    static constexpr int OFF_SEE = OFF_FAC + 4 * R;
    static constexpr int OFF_BAR = OFF_SEE + 16 * R;
    static constexpr int NBAR = 2 * NS + 4 + 2 * NWG * PB;
    static constexpr int OFF_FLAG = OFF_BAR + 8 * NBAR;
    static constexpr int SMEM = OFF_MISC + MISC;
    static_assert(OFF_FLAG + 32 <= SMEM, "misc");
    static_assert(RW * D * 4 <= PGROUP, "a group's output rows fit its P");
    static constexpr int SW = 4 * NWG;                   // softmax warps
    static constexpr int NT = 32 * (SW + 2);
    static constexpr int COLS = 2 * SCOLS + NWG * PB * 2 * RW;  // S twice, O of the groups' units
    static constexpr int TMEM = COLS <= 32 ? 32 : COLS <= 64 ? 64 : COLS <= 128 ? 128 : COLS <= 256 ? 256 : 512;
    static constexpr int PART = R * (D + 2);             // floats of an unfinished segment
    static constexpr bool JOINS = R <= 32;               // the last CTA joins them (else fattn_tree_join_kernel)
};

// N-major operand without swizzle: 8 x 8 blocks of 128 bytes (8 values of N contiguous, 8
// positions), `kgroup` bytes to the next 8 positions, `nblock` to the next 8 values of N.
static __device__ __forceinline__ uint64_t mn_plain_desc(uint32_t addr, uint32_t kgroup, uint32_t nblock) {
    uint64_t d = 0;
    d |= (uint64_t)((addr >> 4) & 0x3FFFu);
    d |= (uint64_t)(kgroup >> 4) << 16;
    d |= (uint64_t)(nblock >> 4) << 32;
    d |= (uint64_t)1u << 46;
    return d;
}
// Lane l gets the sum (or maximum) over the lanes of v[l]: at each step a lane passes on the half
// that its partner keeps.  With 16 values lanes l and l + 16 get the same.
template <int N, bool MAX>
static __device__ __forceinline__ float lane_reduce(float (&v)[N]) {
    const int lane = threadIdx.x & 31;
    if (N == 16) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float x = __shfl_xor_sync(0xffffffffu, v[i], 16);
            v[i] = MAX ? fmaxf(v[i], x) : v[i] + x;
        }
    }
#pragma unroll
    for (int o = N / 2; o > 0; o >>= 1) {
        const bool up = lane & o;
#pragma unroll
        for (int i = 0; i < o; ++i) {
            const float keep = up ? v[i + o] : v[i], x = __shfl_xor_sync(0xffffffffu, up ? v[i] : v[i + o], o);
            v[i] = MAX ? fmaxf(keep, x) : keep + x;
        }
    }
    return v[0];
}

template <int D, int RW, int NWG, bool QF16>
__global__ void __launch_bounds__(TreeTc<D, RW, NWG, QF16>::NT, TreeTc<D, RW, NWG, QF16>::CTAS)
    fattn_tree_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                      const __grid_constant__ TreeAttn a, const __grid_constant__ KvPages p,
                      const __grid_constant__ KvSeqs sq, int box, float *parts, TreeJoin *joins, unsigned int *tickets, int *err) {
    using C = TreeTc<D, RW, NWG, QF16>;
    constexpr int R = C::R, NS = C::NS;
    extern __shared__ __align__(1024) uint8_t smem[];
    griddep_launch_dependents();
    griddep_wait();
    if (smem_u32(smem) & 1023u) {  // the swizzle needs it
        if (threadIdx.x == 0) atomicOr(err, ERR_BAD_SHAPE);
        return;
    }
    float *s_off = (float *)(smem + C::OFF_MISC);
    uint64_t *full = (uint64_t *)(smem + C::OFF_BAR), *empty = full + NS;
    uint64_t *s_full = empty + NS /* [2] */, *p_full = s_full + 2 /* [NWG][PB] */, *o_full = p_full + NWG * C::PB /* the same */,
             *q_full = o_full + NWG * C::PB,
             *done = q_full + 1;
    volatile int *abort_flag = (volatile int *)(smem + C::OFF_FLAG);
    uint32_t *tmem_slot = (uint32_t *)(smem + C::OFF_FLAG + 4);
    unsigned int *s_bad = (unsigned int *)(smem + C::OFF_FLAG + 8);
    int *s_last = (int *)(smem + C::OFF_FLAG + 12);
    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const int G = a.group.d;
    // Each role does what it can before the one block-wide barrier: the TMA warp makes the
    // mbarriers and starts the first K tile, the MMA warp gets TMEM, the others bring Q.
    if (warp == C::SW && lane < 2)
        asm volatile("prefetch.tensormap [%0];" ::"l"(lane ? &tm_v : &tm_k) : "memory");
    else if (warp < C::SW) tree_prefetch(a, sq);
    const TreeUnits w = tree_count(a, sq, p.page, R, gridDim.x, err);
    const int u0 = tree_start(w, blockIdx.x), u1 = tree_start(w, blockIdx.x + 1);
    TreeSeg g = {};
    if (u0 < u1) g = tree_locate(a, sq, w, p.page, R, u0, u1);
    bool begun = false;
    uint32_t tmem = 0, tm_s = 0, tm_o = 0;
    auto begin = [&]() {
        tc_fence_before();
        // not barrier 0: the TMA warp only arrives here, and may come to the last barrier first
        group_sync(4, C::NT);
        tc_fence_after();
        tmem = *(volatile uint32_t *)tmem_slot;
        tm_s = tmem, tm_o = tmem + 2 * C::SCOLS;
        begun = true;
    };

    if (warp >= C::SW) {
        if (warp == C::SW) {
            // ---- TMA: K0, then K(j+1), V(j) ----
            if (lane == 0) {
                for (int i = 0; i < NS; ++i) {
                    mbar_init(&full[i], 1);
                    mbar_init(&empty[i], 1);
                }
                mbar_init(&s_full[0], 1);
                mbar_init(&s_full[1], 1);
                for (int i = 0; i < NWG * C::PB; ++i) {
                    mbar_init(&p_full[i], 128);
                    mbar_init(&o_full[i], 1);
                }
                mbar_init(q_full, 128 * NWG);
                mbar_init(done, 1);
                *abort_flag = 0;
                *s_bad = 0;
                fence_mbar_init();
                fence_proxy_async_smem();
            }
            __syncwarp();
            asm volatile("barrier.cta.arrive 4, %0;" ::"n"(C::NT) : "memory");  // it waits for nothing itself
            begun = true;
            tree_stream<D, NS>(&tm_k, &tm_v, a, p, sq, w, g, R, u0, u1, box, smem, full, empty, abort_flag, err);
        } else {
            tmem_alloc(tmem_slot, C::TMEM);
            begin();
            // ---- MMA: the warp stays together, one elected lane issues ----
            constexpr uint32_t id_s = idesc_f16_f32(TREE_BKV, C::SCOLS);
            constexpr uint32_t id_o = idesc_f16_f32(D, 2 * RW) | 1u << 15 | 1u << 16;  // V^T and P^T: M- and N-major
            const uint64_t dk = sw128_desc(smem_u32(smem)), dq = sw128_desc(smem_u32(smem + C::OFF_Q));
            const uint64_t dv = mn_sw128_desc(smem_u32(smem), D == 128 ? C::HALF : 16);
            const uint64_t dp = mn_plain_desc(smem_u32(smem + C::OFF_P), 128, TREE_BKV * 16);
            int q = 0, it = 0, seg = 0;
            bool ok = true;
            for (int u = u0; u < u1; ++seg) {
                if (u != u0) g = tree_locate(a, sq, w, p.page, R, u, u1);
                const int n = g.k1 - g.k0;
                if (n == 0) break;
                auto scores = [&](int j) {
                    const int slot = q % NS;
                    ok = ok && mbar_wait(&full[slot], (uint32_t)(q / NS & 1), abort_flag, err);
                    ok = __all_sync(0xffffffffu, ok);
                    ++q;
                    if (!ok) return;
                    tc_fence_after();
                    if (elect_one()) {
                        const uint64_t k = dk + slot * (C::TILE >> 4);
                        const uint32_t to = tm_s + (uint32_t)(j & 1) * C::SCOLS;
#pragma unroll
                        for (int x = 0; x < D / 16; ++x)
                            umma_f16(to, k + (x >> 2) * (C::HALF >> 4) + 2 * (x & 3),
                                     dq + (x >> 2) * (C::QHALF >> 4) + 2 * (x & 3), id_s, x != 0);
                        umma_commit(&s_full[j & 1]);
                        umma_commit(&empty[slot]);
                    }
                    __syncwarp();
                };
                ok = ok && mbar_wait(q_full, (uint32_t)seg & 1u, abort_flag, err);
                scores(it);
                for (int j = it; j < it + n; ++j) {
                    // S buffer (j + 1) & 1 was read before the weights of unit j - 1 were complete
                    if (j + 1 < it + n) scores(j + 1);
                    const int slot = q % NS;
                    ok = ok && mbar_wait(&full[slot], (uint32_t)(q / NS & 1), abort_flag, err);
#pragma unroll
                    for (int i = 0; i < NWG; ++i) {
                        const int at = i * C::PB + j % C::PB;
                        ok = ok && mbar_wait(&p_full[at], (uint32_t)(j / C::PB) & 1u, abort_flag, err);
                        ok = __all_sync(0xffffffffu, ok);
                        if (!ok) break;
                        tc_fence_after();
                        if (elect_one()) {
                            const uint64_t v = dv + slot * (C::TILE >> 4), pg = dp + at * (2 * C::PBYTES >> 4);
#pragma unroll
                            for (int x = 0; x < TREE_BKV / 16; ++x)
                                umma_f16(tm_o + at * 2 * RW, v + x * (2048 >> 4), pg + x * (256 >> 4), id_o, x != 0);
                            umma_commit(&o_full[at]);
                            if (i == NWG - 1) umma_commit(&empty[slot]);
                        }
                        __syncwarp();
                    }
                    ++q;
                    if (!ok) break;
                }
                it += n;
                u = g.next;
            }
            if (elect_one()) {
                umma_commit(done);
                const long long t0 = clock64();
                while (!mbar_try_wait(done, 0) && clock64() - t0 < kMbarWaitLimit) {
                }
            }
            __syncwarp();
        }
    } else {
        // ---- softmax: thread = position for the weights, = value of D for the output ----
        const int wg = warp / 4, tid = threadIdx.x & 127;
        const int row0 = wg * RW;                                  // the group's first row of the tile
        const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
        // D = 64 products fill 16 of a warp's 32 lanes
        const int d = D == 128 ? tid : 16 * (warp & 3) + lane;
        const bool has_d = D == 128 || lane < 16;
        float *noff = s_off + row0;  // minus the offsets
        float *fac = (float *)(smem + C::OFF_FAC) + row0;
        uint32_t *see = (uint32_t *)(smem + C::OFF_SEE) + 4 * row0;  // [4][RW]: bits of the unit's positions, by row
        // the group's part of P; while it is free, maxima and sums, then its output rows
        uint8_t *own_p = smem + C::OFF_P + wg * C::PGROUP;
        if (!C::JOINS && threadIdx.x == 0) joins[blockIdx.x].live = 0;
        int it = 0, q = 0;
        for (int u = u0; u < u1;) {
            if (u != u0) g = tree_locate(a, sq, w, p.page, R, u, u1);
            if (g.k0 == g.k1) break;
            const int live = g.n * G - g.rt * R - row0;  // rows of the group below this are real
            const float c = tree_load_q<D, RW, R, QF16>(a, g, row0, live, a.scale, smem + C::OFF_Q, C::QHALF, fac);
            if (tid < RW) noff[tid] = -TREE_NONE;
            fence_proxy_async_smem();
            if (!begun) begin();
            else group_sync(1 + wg, 128);
            mbar_arrive(q_full);

            const f32x2 c2 = pack2(c, c);
            f32x2 o[RW / 2], l[RW / 2];
#pragma unroll
            for (int r = 0; r < RW / 2; ++r) o[r] = l[r] = 0ull;
            // O^T of unit j from TMEM to the running output: the products of both halves of P
            auto drain = [&](int j) {
                const int at = wg * C::PB + j % C::PB;
                mbar_wait(&o_full[at], (uint32_t)(j / C::PB) & 1u, abort_flag, err);
                tc_fence_after();
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    f32x2 v[RW / 2];
                    tmem_load<RW>(tm_o + lanes + (at * 2 + x) * RW, v);
#pragma unroll
                    for (int i = 0; i < RW / 2; ++i) o[i] = add2(o[i], v[i]);
                }
            };
            const int n = g.k1 - g.k0, it0 = it;
            int due = it;  // the first unit that is still to be drained
            for (int k = g.k0; k < g.k1; ++k, ++it) {
                const int t = k * TREE_BKV + tid;             // this thread's position
                const bool tail = (k + 1) * TREE_BKV > g.past;  // nodes among the positions, or the end
                if (tail) {
                    group_sync(1 + wg, 128);  // the last unit's bits have been read
                    for (int e = tid; e < 4 * RW; e += 128) {
                        const int r = e % RW, t0 = k * TREE_BKV + e / RW * 32;
                        see[e] = r < live ? tree_sees32(a, g, a.group(g.rt * R + row0 + r), t0) : 0u;
                    }
                    group_sync(1 + wg, 128);
                }
                const uint32_t *bits = see + (warp & 3) * RW;
                mbar_wait(&s_full[it & 1], (uint32_t)(it >> 1) & 1u, abort_flag, err);
                tc_fence_after();
                const uint32_t ts = tm_s + lanes + (uint32_t)(it & 1) * C::SCOLS + row0;
                uint8_t *p_at = own_p + it % C::PB * (2 * C::PBYTES);
                f32x2 y[RW / 2];  // scores in powers of two
                tmem_load<RW>(ts, y);
                if (C::SCOLS != R) {
                    f32x2 lo[RW / 2];
                    tmem_load<RW>(ts + R, lo);
#pragma unroll
                    for (int i = 0; i < RW / 2; ++i) y[i] = add2(y[i], lo[i]);
                }
#pragma unroll
                for (int i = 0; i < RW / 2; i += 2) {
                    const ulonglong2 f = QF16 ? make_ulonglong2(c2, c2) : *reinterpret_cast<const ulonglong2 *>(fac + 2 * i);
                    y[i] = mul2(y[i], f.x), y[i + 1] = mul2(y[i + 1], f.y);
                }
                if (tail) {
#pragma unroll
                    for (int i = 0; i < RW / 2; ++i) {
                        float2 x = unpack2(y[i]);
                        if (!(bits[2 * i] >> lane & 1u)) x.x = -INFINITY;
                        if (!(bits[2 * i + 1] >> lane & 1u)) x.y = -INFINITY;
                        y[i] = pack2(x.x, x.y);
                    }
                }
                const bool fresh = it == it0;
                float top = -INFINITY;
#pragma unroll
                for (int i = 0; i < RW / 2; i += 2) {
                    const ulonglong2 f = *reinterpret_cast<const ulonglong2 *>(noff + 2 * i);
                    const float2 x = unpack2(add2(y[i], f.x)), z = unpack2(add2(y[i + 1], f.y));
                    top = fmaxf(fmaxf(top, fmaxf(x.x, x.y)), fmaxf(z.x, z.y));
                }
                const bool rescale = group_any(1 + wg, top > TREE_MOST);
                // the unit that had this one's place; with it its part of P is free
                if (due <= it - C::PB) drain(due++);
                if (rescale) {
                    // -- new maxima: of the unit's 128 positions, then with what was --
                    if (due < it) drain(due++);  // the rows' sums are complete
                    float *red = (float *)p_at, *down = red;  // [4][RW]
                    float v[RW];
#pragma unroll
                    for (int i = 0; i < RW / 2; ++i) {
                        const float2 e = unpack2(y[i]);
                        v[2 * i] = e.x, v[2 * i + 1] = e.y;
                    }
                    const float most = lane_reduce<RW, true>(v);
                    if (lane < RW) red[(warp & 3) * RW + lane] = most;
                    group_sync(1 + wg, 128);
                    if (tid < RW) {
                        const float old = -noff[tid];
                        const float m = fmaxf(fmaxf(red[tid], red[RW + tid]), fmaxf(red[2 * RW + tid], red[3 * RW + tid]));
                        const float now = fmaxf(old, m - TREE_EXP);
                        noff[tid] = -now;
                        down[tid] = tree_exp2(old - now);
                    }
                    group_sync(1 + wg, 128);
                    if (!fresh) {
#pragma unroll
                        for (int r = 0; r < RW / 2; r += 2) {
                            const ulonglong2 f = *reinterpret_cast<const ulonglong2 *>(down + 2 * r);
                            o[r] = mul2(o[r], f.x), o[r + 1] = mul2(o[r + 1], f.y);
                            l[r] = mul2(l[r], f.x), l[r + 1] = mul2(l[r + 1], f.y);
                        }
                        group_sync(1 + wg, 128);  // the factors lie where the weights go
                    }
                }
                // -- weights: 16 bytes per 8 rows into the N-major P tiles --
#pragma unroll
                for (int x = 0; x < RW / 8; ++x) {
                    uint32_t hi[4], lo[4];
#pragma unroll
                    for (int i = 0; i < 4; i += 2) {
                        const ulonglong2 f = *reinterpret_cast<const ulonglong2 *>(noff + 8 * x + 2 * i);
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const float2 e = unpack2(add2(y[4 * x + i + h], h ? f.y : f.x));
                            const f32x2 wt = pack2(tree_exp2(e.x), tree_exp2(e.y));
                            f32x2 &sum = l[4 * x + i + h];
                            sum = add2(sum, wt);
                            tree_cut2(wt, hi[i + h], lo[i + h]);
                        }
                    }
                    uint8_t *dst = p_at + x * (TREE_BKV * 16) + tid * 16;
                    *reinterpret_cast<uint4 *>(dst) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                    *reinterpret_cast<uint4 *>(dst + C::PBYTES) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                }
                if (tail && wg == 0) {
                    const int j = it - it0, qi = q + (j + 1 < n ? 2 + 2 * j : 2 * n - 1);  // V's place in the ring
                    mbar_wait(&full[qi % NS], (uint32_t)(qi / NS & 1), abort_flag, err);
                    if (t >= g.past && tree_clean_v<D>(smem + qi % NS * C::TILE, tid) && t < g.T) *s_bad = 1u;
                }
                tc_fence_before();
                fence_proxy_async_smem();
                mbar_arrive(&p_full[wg * C::PB + it % C::PB]);
            }
#pragma unroll
            for (int x = 0; x < C::PB; ++x)
                if (due < it) drain(due++);
            tc_fence_before();
            q += 2 * n;

            // -- sums of the weights over the group's positions --
            {
                float *red = (float *)own_p;  // [4][RW]
                float v[RW];
#pragma unroll
                for (int i = 0; i < RW / 2; ++i) {
                    const float2 e = unpack2(l[i]);
                    v[2 * i] = e.x, v[2 * i + 1] = e.y;
                }
                const float sum = lane_reduce<RW, false>(v);
                if (lane < RW) red[(warp & 3) * RW + lane] = sum;
            }
            group_sync(1 + wg, 128);
            const bool whole = g.k0 == 0 && g.k1 == g.kt;
            float *part = parts + (int64_t)tree_slot(w, blockIdx.x, g.first) * C::PART;
            if (tid < RW) {
                const float *red = (const float *)own_p;
                const float L = (red[tid] + red[RW + tid]) + (red[2 * RW + tid] + red[3 * RW + tid]);
                if (!whole) reinterpret_cast<float2 *>(part + R * D)[row0 + tid] = make_float2(-noff[tid], L);
                noff[tid] = L == 0.0f ? 0.0f : 1.0f / L;  // the rows' factors from here on
            }
            // V was cleaned by the first group for both
            group_sync(NWG == 1 ? 1 : 3, 128 * NWG);
            const bool anybad = *(volatile unsigned int *)s_bad != 0;
            // -- the output through shared memory: rows in a loop, 16 bytes at a time --
            if (has_d) {
#pragma unroll
                for (int r = 0; r < RW; ++r) {
                    const float2 y = unpack2(o[r / 2]);
                    reinterpret_cast<float *>(own_p)[r * D + d] = r & 1 ? y.y : y.x;
                }
            }
            group_sync(1 + wg, 128);
            const int chunks = min(RW, live) * (D / 4);
            float4 *rows = reinterpret_cast<float4 *>(own_p);
            if (anybad) {
                for (int e = tid; e < chunks; e += 128)
                    rows[e] = tree_nonfinite4(a, p, sq, g, a.group(g.rt * R + row0 + e / (D / 4)), e % (D / 4) * 4, rows[e]);
            }
            if (whole) {
#pragma unroll 4
                for (int e = tid; e < chunks; e += 128) {
                    const int r = e / (D / 4), gr = g.rt * R + row0 + r, node = a.group(gr);
                    const float4 x = rows[e];
                    const float f = noff[r];
                    tree_store4(a, g.s, g.hk * G + gr - node * G, node, e % (D / 4) * 4, make_float4(x.x * f, x.y * f, x.z * f, x.w * f));
                }
            } else {
#pragma unroll 4
                for (int e = tid; e < chunks; e += 128) reinterpret_cast<float4 *>(part)[row0 * (D / 4) + e] = rows[e];
            }
            if (!C::JOINS && !whole && g.k0 == 0 && threadIdx.x == 0)
                joins[blockIdx.x] = TreeJoin{tree_owner(w, g.first + g.per - 1), tree_slot(w, blockIdx.x, g.first), g.s, g.hk,
                                             g.rt * R, min(R, live)};
            // -- small tiles: the last of the CTAs that share the item joins the parts here --
            if (C::JOINS && !whole) {
                const int c0 = tree_owner(w, g.first + g.lead), c1 = tree_owner(w, g.first + g.per - 1);
                group_sync(NWG == 1 ? 1 : 3, 128 * NWG);
                if (threadIdx.x == 0) {
                    const bool is_last = atom_add_acq_rel_gpu(tickets + c0, 1u) == (unsigned)(c1 - c0);
                    if (is_last) atomicExch(tickets + c0, 0u);
                    *s_last = is_last;
                }
                group_sync(NWG == 1 ? 1 : 3, 128 * NWG);
                if (*(volatile int *)s_last) {
                    for (int e = threadIdx.x; e < min(R, live + row0) * (D / 4); e += 128 * NWG) {
                        const int r = e / (D / 4), ch = e % (D / 4), gr = g.rt * R + r, node = a.group(gr);
                        tree_store4(a, g.s, g.hk * G + gr - node * G, node, 4 * ch,
                                    tree_join4<8>(parts, R, D, c0, c1, tree_slot(w, c0, g.first), r, ch));
                    }
                }
            }
            u = g.next;
            if (u < u1) {  // the next segment reuses the flag, the sums, P and Q
                group_sync(NWG == 1 ? 1 : 3, 128 * NWG);
                if (threadIdx.x == 0) *s_bad = 0;
                group_sync(NWG == 1 ? 1 : 3, 128 * NWG);
            }
        }
    }
    if (!begun) begin();
    tc_fence_before();
    __syncthreads();
    if (warp == C::SW + 1) {
        tc_fence_after();
        tmem_dealloc(tmem, C::TMEM);
    }
}

// Joins the items that several CTAs of fattn_tree_kernel shared: block (c, rows) takes 8 rows of
// the one that begins in CTA c, four columns per thread, six parts loaded at a time.  After runs of
// 16 wide trees (2 or 3 parts of 66 KB each) the join costs 4 us of 96, after the pieces of two long
// caches (37 parts of 21 KB) 4 us of 32, half of it the launch; with sixteen parts at a time 8 and 5,
// with four 4 and 5, by the last CTA alone 6 and 10.
template <int D, int R>
__global__ void __launch_bounds__(2 * D) fattn_tree_join_kernel(const __grid_constant__ TreeAttn a, const float *parts,
                                                                const TreeJoin *joins) {
    griddep_launch_dependents();
    griddep_wait();
    const int c0 = blockIdx.x / (R / 8), r = blockIdx.x % (R / 8) * 8 + threadIdx.x / (D / 4), ch = threadIdx.x % (D / 4);
    const TreeJoin g = joins[c0];
    if (r >= g.live) return;
    const int node = a.group(g.row + r);
    tree_store4(a, g.s, g.hk * a.group.d + g.row + r - node * a.group.d, node, 4 * ch,
                tree_join4<6>(parts, R, D, c0, g.c1, g.slot, r, ch));
}

bool tree_page_map(CUtensorMap *map, const char *base, int64_t nb1, int64_t nb2, int64_t nb3, int D, int page, int HKV,
                   int n_pages, int rows) {
    static PFN_cuTensorMapEncodeTiled_v12000 enc = [] {
        void *f = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            f = nullptr;
        return (PFN_cuTensorMapEncodeTiled_v12000)f;
    }();
    if (!enc) return false;
    const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)page, (cuuint64_t)HKV, (cuuint64_t)n_pages};
    // the stride of a dimension of one is never used, but has to be a valid one
    const cuuint64_t strides[3] = {(cuuint64_t)nb1, HKV == 1 ? (cuuint64_t)nb1 : (cuuint64_t)nb2,
                                   n_pages == 1 ? (cuuint64_t)nb1 : (cuuint64_t)nb3};
    const cuuint32_t boxd[4] = {64, (cuuint32_t)rows, 1, 1};
    const cuuint32_t estr[4] = {1, 1, 1, 1};
    return enc(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<char *>(base), dims, strides, boxd, estr,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int tree_prepare(oasr_backend *be, TreeAttn &a, const KvPages &p, const KvSeqs &s, int R, int ctas_per_sm, TreeLaunch *out) {
    // the longest run of positions, up to a unit, that never crosses a page
    out->box = std::min(TREE_BKV, p.page & -p.page);
    if (!tree_page_map(&out->k, p.k, p.k_nb1, p.k_nb2, p.k_nb3, a.D, p.page, a.HKV, p.n_pages, out->box) ||
        !tree_page_map(&out->v, p.v, p.v_nb1, p.v_nb2, p.v_nb3, a.D, p.page, a.HKV, p.n_pages, out->box))
        return oasr_internal_fail(be, OASR_STATUS_FAILED, "flash_attn_tree: the pages' strides make no tensor map");
    a.group = FastDiv(a.H / a.HKV);
    a.page = FastDiv(p.page);
    const int64_t tiles = ((int64_t)s.N * a.group.d + R - 1) / R;
    const int64_t items = tiles * a.HKV * a.S, most = items * (((int64_t)s.MP * p.page + TREE_BKV - 1) / TREE_BKV);
    // (rows are counted in steps of the grid's warps, which must not pass 31 bits either)
    if (most + items * tree_segment(R) > INT32_MAX / 2 || (int64_t)s.N * a.group.d > INT32_MAX / 2 ||
        (int64_t)a.S * s.N * a.H > INT32_MAX - 65536)
        return oasr_internal_fail(be, OASR_STATUS_FAILED, "flash_attn_tree: too many rows and positions");
    out->grid = (int)std::max<int64_t>(1, std::min<int64_t>(most, (int64_t)be->sm_count * ctas_per_sm));
    const size_t part = (size_t)R * (a.D + 2) * 4;
    int st = 0;
    out->parts = (float *)oasr_internal_scratch(be, out->grid * (2 * part + sizeof(TreeJoin)), &st);
    out->joins = (TreeJoin *)((char *)out->parts + out->grid * 2 * part);
    return st;
}

int tree_join(oasr_backend *be, const TreeAttn &a, const KvPages &p, const KvSeqs &s, int R, const TreeLaunch &l) {
    if (l.grid == 1 || (int64_t)s.MP * p.page <= TREE_BKV) return OASR_STATUS_SUCCESS;  // no item is shared
    const dim3 grid(l.grid * (R / 8)), block(2 * a.D);
    const float *parts = l.parts;
    const TreeJoin *joins = l.joins;
    cudaError_t e;
    if (R == 64) e = a.D == 64 ? launch_k(be, fattn_tree_join_kernel<64, 64>, grid, block, 0, a, parts, joins)
                               : launch_k(be, fattn_tree_join_kernel<128, 64>, grid, block, 0, a, parts, joins);
    else e = a.D == 64 ? launch_k(be, fattn_tree_join_kernel<64, 128>, grid, block, 0, a, parts, joins)
                       : launch_k(be, fattn_tree_join_kernel<128, 128>, grid, block, 0, a, parts, joins);
    if (e != cudaSuccess) return oasr_internal_cuda_fail(be, e, "flash_attn_tree join launch", __LINE__);
    return oasr_internal_launch_check(be, "flash_attn_tree join");
}

template <int D, int RW, int NWG, bool QF16>
static int launch_tree(oasr_backend *be, TreeAttn a, const KvPages &p, const KvSeqs &s) {
    using C = TreeTc<D, RW, NWG, QF16>;
    TreeLaunch l;
    const int st = tree_prepare(be, a, p, s, C::R, C::CTAS, &l);
    if (st) return st;
    static OncePerDevice smem;
    cudaError_t e = (cudaError_t)smem(be->device, [] {
        return cudaFuncSetAttribute(fattn_tree_kernel<D, RW, NWG, QF16>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
    });
    if (e != cudaSuccess) return oasr_internal_cuda_fail(be, e, "flash_attn_tree attribute", __LINE__);
    e = launch_k(be, fattn_tree_kernel<D, RW, NWG, QF16>, dim3(l.grid), dim3(C::NT), C::SMEM, l.k, l.v, a, p,
                                   s, l.box, l.parts, l.joins, be->counters, be->err_word);
    if (e != cudaSuccess) return oasr_internal_cuda_fail(be, e, "flash_attn_tree launch", __LINE__);
    if (!C::JOINS) return tree_join(be, a, p, s, C::R, l);
    return oasr_internal_launch_check(be, "flash_attn_tree");
}

int launch_flash_attn_tree(oasr_backend *be, const TreeAttn &a, const KvPages &p, const KvSeqs &s) {
    // the smallest tile that takes all rows of a K/V head, so that K and V are read once: sixteen
    // sequences of 4001 to 8190 positions take 69 us in tiles of 16 or 32 rows, 78 in one of 64 (f32);
    // past 64 rows, tiles of 64 read K and V twice (156 us for 16 trees of 61 nodes and two heads, when
    // the tile of 128 took 149)
    const int64_t rows = (int64_t)s.N * (a.H / a.HKV);
    if (rows > 64) return launch_tree_wide(be, a, p, s);
#define FT(DD, RW, NWG, Q) \
    if (a.D == DD && a.q_f16 == Q && rows <= RW * NWG) return launch_tree<DD, RW, NWG, Q>(be, a, p, s)
#define FTQ(DD, RW, NWG) FT(DD, RW, NWG, false); FT(DD, RW, NWG, true)
    FTQ(64, 16, 1); FTQ(64, 16, 2); FTQ(64, 32, 2);
    FTQ(128, 16, 1); FTQ(128, 16, 2); FTQ(128, 32, 2);
#undef FTQ
#undef FT
    return oasr_internal_fail(be, OASR_STATUS_FAILED, "flash_attn_tree: head_dim must be 64 or 128");
}

}  // namespace oasr
