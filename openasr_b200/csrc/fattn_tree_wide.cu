// fattn_tree_wide.cu -- the tree attention (fattn_tree.cu) for more than 64 rows of a K/V head.
//
// With 128 rows the matrix unit is full the plain way round,
//   S (128 rows x 128 positions) = Q . K^T      both K-major
//   O (128 rows x D)             = P . V        P from TMEM, V as it lies (N-major)
// and a softmax thread owns a row: its maximum, its sum and its output need no other thread, and P
// goes back into the columns of TMEM that its scores came from, never through shared memory.  Per
// unit of 128 positions the tensor cores take 16 products of 64 clocks for P V (both halves of P)
// and 8 (f16 queries) or 16 for Q K^T, 1536 to 2048 clocks; an SM's share of the HBM rate allows
// 2900 for D = 128.
//
// CTA: two groups of 4 softmax warps take every other unit, each with sums of its own that are
// joined at the end of a segment; one TMA warp, one MMA warp.  The queries of the groups' units are
// the same 128 rows.  Accuracy, offsets and the split over the CTAs are those of fattn_tree.cu.
// S(j + 2) overwrites P(j): the products of one thread run in the order of their issue.
//
// Sixteen trees of 61 nodes, 4001 to 8190 positions, 8 K/V heads of 128, f16 (411 MB): 97 us, 4.2 TB/s
// at 1965 MHz (112 us with equal runs that did not count the segments' ends); back to back for a third
// of a second the power cap holds the SM clock near 1650 MHz and a call takes 107 to 119 us.  A unit takes a CTA 2600 clocks, of
// which the weights are 2400 of a group's 5200 -- 32 columns at a time: a loop over 16 columns takes
// 101 us, two rounds in one body 104, all four unrolled 102 (code is fetched more slowly than run).
// P goes to the matrix unit by 32 positions; handed over whole it took 133 -> 141 us for four chunks of
// 512 rows over 4000 positions.  The rest is the segments: 14000 clocks from the launch to the first
// product, 10000 for the end of each, 4 us for the join.
#include <algorithm>

#include "fattn_tree.cuh"

namespace oasr {

template <int D_, bool QF16_>
struct TreeWide {
    static constexpr int D = D_, R = 128;
    static constexpr int HALF = TREE_BKV * 128, TILE = HALF * (D / 64);
    static constexpr int QROWS = QF16_ ? R : 2 * R, QHALF = QROWS * 128, QBYTES = QHALF * (D / 64);
    static constexpr int MISC = 3072;
    static constexpr int MOST = 232448 - QBYTES - MISC;
    static constexpr int NS = MOST / TILE > 8 ? 8 : MOST / TILE;
    static_assert(NS >= 4, "K of two units, K and V of the next");
    static constexpr int OFF_Q = NS * TILE, OFF_MISC = OFF_Q + QBYTES;
    // misc: (offset, sum) [2][R], query factors [R], barriers, flags
    static constexpr int OFF_C = OFF_MISC + 16 * R;
    static constexpr int OFF_BAR = OFF_C + 4 * R;
    static constexpr int SPLIT = 4;  // parts of a unit's weights that are handed over one by one
    static constexpr int OFF_FLAG = OFF_BAR + 8 * (2 * NS + 6 + 2 * SPLIT);
    static constexpr int SMEM = OFF_MISC + MISC;
    static_assert(OFF_FLAG + 32 <= SMEM, "misc");
    // 12 warps at 168 registers; the softmax warps, with a row of output each, take more
    static constexpr int NT = 384;
    static constexpr int TM_O = 2 * R, TMEM = 512;  // S / P twice, O twice
};

// D(tmem) (+)= A(tmem) . B(smem desc)
static __device__ __forceinline__ void umma_f16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
// 32 columns of this warp's 32 lanes
static __device__ __forceinline__ void tmem_store32(uint32_t addr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
        "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(addr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]),
        "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]),
        "r"(r[31])
        : "memory");
}

template <int D, bool QF16>
__global__ void __launch_bounds__(384, 1)
    fattn_tree_wide_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                           const __grid_constant__ TreeAttn a, const __grid_constant__ KvPages p,
                           const __grid_constant__ KvSeqs sq, int box, float *parts, TreeJoin *joins, int *err) {
    using C = TreeWide<D, QF16>;
    constexpr int R = C::R, NS = C::NS;
    extern __shared__ __align__(1024) uint8_t smem[];
    griddep_launch_dependents();
    griddep_wait();
    if (smem_u32(smem) & 1023u) {  // the swizzle needs it
        if (threadIdx.x == 0) atomicOr(err, ERR_BAD_SHAPE);
        return;
    }
    float2 *s_ml = (float2 *)(smem + C::OFF_MISC);
    float *s_c = (float *)(smem + C::OFF_C);
    uint64_t *full = (uint64_t *)(smem + C::OFF_BAR), *empty = full + NS;
    uint64_t *s_full = empty + NS, *p_full = s_full + 2, *o_full = p_full + 2 * C::SPLIT /* [2][SPLIT] before */, *q_full = o_full + 2, *done = q_full + 1;
    volatile int *abort_flag = (volatile int *)(smem + C::OFF_FLAG);
    uint32_t *tmem_slot = (uint32_t *)(smem + C::OFF_FLAG + 4);
    unsigned int *s_bad = (unsigned int *)(smem + C::OFF_FLAG + 8);
    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const int G = a.group.d;
    // as in fattn_tree_kernel: every role begins on its own, one block-wide barrier (4) after that
    if (warp == 8 && lane < 2) asm volatile("prefetch.tensormap [%0];" ::"l"(lane ? &tm_v : &tm_k) : "memory");
    else if (warp < 8) tree_prefetch(a, sq);
    const TreeUnits w = tree_count(a, sq, p.page, R, gridDim.x, err);
    const int u0 = tree_start(w, blockIdx.x), u1 = tree_start(w, blockIdx.x + 1);
    TreeSeg g = {};
    if (u0 < u1) g = tree_locate(a, sq, w, p.page, R, u0, u1);
    uint32_t tmem = 0;
    bool begun = false;
    auto begin = [&]() {
        tc_fence_before();
        group_sync(4, C::NT);
        tc_fence_after();
        tmem = *(volatile uint32_t *)tmem_slot;
        begun = true;
    };

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        if (warp == 8) {
            if (lane == 0) {
                for (int i = 0; i < NS; ++i) {
                    mbar_init(&full[i], 1);
                    mbar_init(&empty[i], 1);
                }
                for (int i = 0; i < 2; ++i) {
                    mbar_init(&s_full[i], 1);
                    for (int x = 0; x < C::SPLIT; ++x) mbar_init(&p_full[i * C::SPLIT + x], 128);
                    mbar_init(&o_full[i], 1);
                }
                mbar_init(q_full, 256);
                mbar_init(done, 1);
                *abort_flag = 0;
                *s_bad = 0;
                fence_mbar_init();
                fence_proxy_async_smem();
            }
            __syncwarp();
            asm volatile("barrier.cta.arrive 4, %0;" ::"n"(C::NT) : "memory");  // it waits for nothing itself
            tree_stream<D, NS>(&tm_k, &tm_v, a, p, sq, w, g, R, u0, u1, box, smem, full, empty, abort_flag, err);
        } else if (warp == 9) {
            tmem_alloc(tmem_slot, C::TMEM);
            begin();
            // ---- MMA: S(0), S(1), then P V(j) and S(j + 2), which takes the place of P(j) ----
            constexpr uint32_t id_s = idesc_f16_f32(R, TREE_BKV);
            constexpr uint32_t id_o = idesc_f16_f32(R, D) | 1u << 16;  // V: N-major
            const uint64_t dq = sw128_desc(smem_u32(smem + C::OFF_Q)), dk = sw128_desc(smem_u32(smem));
            const uint64_t dv = mn_sw128_desc(smem_u32(smem), D == 128 ? C::HALF : 16);
            int q = 0, it = 0, seg = 0;
            bool ok = true;
            auto arrived = [&](uint64_t *bar, uint32_t parity) {
                ok = ok && mbar_wait(bar, parity, abort_flag, err);
                ok = __all_sync(0xffffffffu, ok);
                tc_fence_after();
                return ok;
            };
            for (int u = u0; u < u1; ++seg) {
                if (u != u0) g = tree_locate(a, sq, w, p.page, R, u, u1);
                const int n = g.k1 - g.k0;
                if (n == 0) break;
                auto scores = [&](int j) {
                    const int slot = q % NS;
                    const uint32_t parity = (uint32_t)(q / NS & 1);
                    ++q;
                    if (!arrived(&full[slot], parity)) return;
                    if (elect_one()) {
                        const uint64_t k = dk + slot * (C::TILE >> 4);
#pragma unroll
                        for (int part = 0; part < (QF16 ? 1 : 2); ++part)
#pragma unroll
                            for (int x = 0; x < D / 16; ++x)
                                umma_f16(tmem + (uint32_t)(j & 1) * R,
                                         dq + part * (R * 128 >> 4) + (x >> 2) * (C::QHALF >> 4) + 2 * (x & 3),
                                         k + (x >> 2) * (C::HALF >> 4) + 2 * (x & 3), id_s, part + x != 0);
                        umma_commit(&s_full[j & 1]);
                        umma_commit(&empty[slot]);
                    }
                    __syncwarp();
                };
                arrived(q_full, (uint32_t)seg & 1u);
                scores(it);
                if (n > 1) scores(it + 1);
                for (int j = it; j < it + n && ok; ++j) {
                    const int slot = q % NS, b = j & 1;
                    const uint32_t parity = (uint32_t)(q / NS & 1);
                    ++q;
                    if (!arrived(&full[slot], parity)) break;
                    const uint64_t v = dv + slot * (C::TILE >> 4);
                    // as the weights come: per 32 positions 16 columns of high halves, then 16 of low ones
#pragma unroll
                    for (int h = 0; h < C::SPLIT; ++h) {
                        if (!arrived(&p_full[b * C::SPLIT + h], (uint32_t)(j >> 1) & 1u)) break;
                        if (elect_one()) {
#pragma unroll
                            for (int x = h * (8 / C::SPLIT); x < (h + 1) * (8 / C::SPLIT); ++x)
#pragma unroll
                                for (int part = 0; part < 2; ++part)
                                    umma_f16_ts(tmem + C::TM_O + (uint32_t)b * R,
                                                tmem + (uint32_t)(b * R + 32 * (x >> 1) + 8 * (x & 1) + 16 * part),
                                                v + x * (2048 >> 4), id_o, x + part != 0);
                            if (h == C::SPLIT - 1) {
                                umma_commit(&o_full[b]);
                                umma_commit(&empty[slot]);
                            }
                        }
                        __syncwarp();
                    }
                    if (!ok) break;
                    if (j + 2 < it + n) scores(j + 2);
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
        } else {
            begin();  // only there to hand its registers over
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
        // ---- softmax: thread = row; group wg takes the units of its parity ----
        const int wg = warp / 4, tid = threadIdx.x & 127;
        const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
        if (threadIdx.x == 0) joins[blockIdx.x].live = 0;
        int it = 0, q = 0;
        for (int u = u0; u < u1;) {
            if (u != u0) g = tree_locate(a, sq, w, p.page, R, u, u1);
            if (g.k0 == g.k1) break;
            const int live = g.n * G - g.rt * R;  // rows of the tile below this are real
            const float c16 = tree_load_q<D, 64, R, QF16>(a, g, 64 * wg, live - 64 * wg, a.scale, smem + C::OFF_Q, C::QHALF,
                                                          s_c + 64 * wg);
            fence_proxy_async_smem();
            if (!begun) begin();
            else group_sync(3, 256);
            mbar_arrive(q_full);
            const float c = QF16 ? c16 : s_c[tid];
            const f32x2 c2 = pack2(c, c);
            const int node = tid < live ? a.group(g.rt * R + tid) : -1;

            f32x2 o[D / 2], l0 = 0ull, l1 = 0ull;
            float off = TREE_NONE;
#pragma unroll
            for (int i = 0; i < D / 2; ++i) o[i] = 0ull;
            const int n = g.k1 - g.k0, it0 = it;
            for (int k = g.k0; k < g.k1; ++k, ++it) {
                if ((it & 1) != wg) continue;
                const uint32_t phase = (uint32_t)(it >> 1) & 1u, ts = tmem + lanes + (uint32_t)wg * R;
                const bool tail = (k + 1) * TREE_BKV > g.past;  // nodes among the positions, or the end
                mbar_wait(&s_full[wg], phase, abort_flag, err);
                tc_fence_after();
                auto masked = [&](int x, f32x2 (&y)[16]) {
                    tmem_load<32>(ts + 32 * x, y);
                    if (tail) {
                        const uint32_t see = node < 0 ? 0u : tree_sees32(a, g, node, k * TREE_BKV + 32 * x);
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            float2 e = unpack2(y[i]);
                            if (!(see >> (2 * i) & 1u)) e.x = -INFINITY;
                            if (!(see >> (2 * i + 1) & 1u)) e.y = -INFINITY;
                            y[i] = pack2(e.x, e.y);
                        }
                    }
                };
                f32x2 y[16];
                float top = -INFINITY, top2 = -INFINITY;
#pragma unroll 1
                for (int x = 0; x < 4; ++x) {
                    masked(x, y);
#pragma unroll
                    for (int i = 0; i < 16; i += 2) {
                        const float2 e = unpack2(y[i]), f = unpack2(y[i + 1]);
                        top = fmaxf(top, fmaxf(e.x, e.y));
                        top2 = fmaxf(top2, fmaxf(f.x, f.y));
                    }
                }
                top = fmaxf(top, top2) * c;  // (c is positive: the sign of the scale is in Q)
                const bool more = top - off > TREE_MOST;
                if (__any_sync(0xffffffffu, more)) {
                    const float now = more ? fmaxf(off, top - TREE_EXP) : off, f = tree_exp2(off - now);
                    const f32x2 f2 = pack2(f, f);
                    l0 = mul2(l0, f2), l1 = mul2(l1, f2);
#pragma unroll
                    for (int i = 0; i < D / 2; ++i) o[i] = mul2(o[i], f2);
                    off = now;
                }
                if (tail) {
                    const int j = it - it0, qi = q + (j + 1 < n ? 2 + 2 * j : 2 * n - 1), t = k * TREE_BKV + tid;  // V's place
                    mbar_wait(&full[qi % NS], (uint32_t)(qi / NS & 1), abort_flag, err);
                    if (t >= g.past && tree_clean_v<D>(smem + qi % NS * C::TILE, tid) && t < g.T) *s_bad = 1u;
                    fence_proxy_async_smem();
                }
                // -- weights, in place of the scores --
                const f32x2 n2 = pack2(-off, -off);
#pragma unroll 1
                for (int x = 0; x < 4; ++x) {
                    masked(x, y);
                    uint32_t h[32];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const float2 e = unpack2(fma2(y[i], c2, n2));
                        const f32x2 wt = pack2(tree_exp2(e.x), tree_exp2(e.y));
                        if (i & 1) l1 = add2(l1, wt);
                        else l0 = add2(l0, wt);
                        tree_cut2(wt, h[i], h[16 + i]);
                    }
                    tmem_store32(ts + 32 * x, h);
                    if ((x + 1) % (4 / C::SPLIT) == 0) {
                        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                        tc_fence_before();
                        mbar_arrive(&p_full[wg * C::SPLIT + x / (4 / C::SPLIT)]);
                    }
                }
                // -- the product, when it is there --
                mbar_wait(&o_full[wg], phase, abort_flag, err);
                tc_fence_after();
#pragma unroll
                for (int x = 0; x < D / 32; ++x) {
                    tmem_load<32>(tmem + lanes + C::TM_O + wg * R + 32 * x, y);
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[16 * x + i] = add2(o[16 * x + i], y[i]);
                }
                tc_fence_before();
            }
            q += 2 * n;

            // -- the two groups' sums: the second's output goes through the place of Q --
            const float2 la = unpack2(l0), lb = unpack2(l1);
            s_ml[wg * R + tid] = make_float2(off, (la.x + la.y) + (lb.x + lb.y));
            group_sync(3, 256);
            const bool whole = g.k0 == 0 && g.k1 == g.kt, anybad = *(volatile unsigned int *)s_bad != 0;
            float *part = parts + (int64_t)tree_slot(w, blockIdx.x, g.first) * (R * (D + 2));
            {
                const float2 x = s_ml[tid], z = s_ml[R + tid];
                const float M = fmaxf(x.x, z.x), fx = tree_exp2(x.x - M), fz = tree_exp2(z.x - M);
                const float L = fmaf(x.y, fx, z.y * fz);
                const float f = (wg ? fz : fx) * (!whole ? 1.0f : L == 0.0f ? 0.0f : 1.0f / L);
                const f32x2 f2 = pack2(f, f);
#pragma unroll
                for (int i = 0; i < D / 2; ++i) o[i] = mul2(o[i], f2);
                if (!whole && wg == 0) reinterpret_cast<float2 *>(part + R * D)[tid] = make_float2(M, L);
            }
            constexpr int HC = D / 8;  // 16-byte pieces of half a row
            float4 *stage = reinterpret_cast<float4 *>(smem + C::OFF_Q);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                float4 *mine = stage + tid * HC;  // pieces of a row in another order for every row: no bank twice
                if (wg == 1) {
#pragma unroll
                    for (int i = 0; i < HC; ++i) {
                        const float2 e = unpack2(o[half * (D / 4) + 2 * i]), f = unpack2(o[half * (D / 4) + 2 * i + 1]);
                        mine[i ^ (tid & (HC - 1))] = make_float4(e.x, e.y, f.x, f.y);
                    }
                }
                group_sync(3, 256);
                if (wg == 0) {
#pragma unroll
                    for (int i = 0; i < HC; ++i) {
                        const float2 e = unpack2(o[half * (D / 4) + 2 * i]), f = unpack2(o[half * (D / 4) + 2 * i + 1]);
                        float4 &x = mine[i ^ (tid & (HC - 1))];
                        x = make_float4(x.x + e.x, x.y + e.y, x.z + f.x, x.w + f.y);
                    }
                }
                group_sync(3, 256);
                if (anybad) {
                    for (int e = threadIdx.x; e < min(R, live) * HC; e += 256) {
                        const int r = e / HC, ch = e % HC;
                        float4 &x = stage[r * HC + (ch ^ (r & (HC - 1)))];
                        x = tree_nonfinite4(a, p, sq, g, a.group(g.rt * R + r), half * (D / 2) + 4 * ch, x);
                    }
                }
#pragma unroll 4
                for (int e = threadIdx.x; e < min(R, live) * HC; e += 256) {
                    const int r = e / HC, ch = e % HC, gr = g.rt * R + r, nd = a.group(gr), col = half * (D / 2) + 4 * ch;
                    const float4 x = stage[r * HC + (ch ^ (r & (HC - 1)))];
                    if (whole) tree_store4(a, g.s, g.hk * G + gr - nd * G, nd, col, x);
                    else *reinterpret_cast<float4 *>(part + r * D + col) = x;
                }
                group_sync(3, 256);
            }
            if (!whole && g.k0 == 0 && threadIdx.x == 0)
                joins[blockIdx.x] = TreeJoin{tree_owner(w, g.first + g.per - 1), tree_slot(w, blockIdx.x, g.first), g.s, g.hk,
                                             g.rt * R, min(R, live)};
            u = g.next;
            if (u < u1) {  // the next segment reuses the flag
                if (threadIdx.x == 0) *s_bad = 0;
                group_sync(3, 256);
            }
        }
        if (!begun) begin();
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 9) {
        tc_fence_after();
        tmem_dealloc(tmem, C::TMEM);
    }
}

template <int D, bool QF16>
static int launch_wide(oasr_backend *be, TreeAttn a, const KvPages &p, const KvSeqs &s) {
    using C = TreeWide<D, QF16>;
    TreeLaunch l;
    const int st = tree_prepare(be, a, p, s, C::R, 1, &l);
    if (st) return st;
    static OncePerDevice smem;
    cudaError_t e = (cudaError_t)smem(be->device, [] {
        return cudaFuncSetAttribute(fattn_tree_wide_kernel<D, QF16>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
    });
    if (e != cudaSuccess) return oasr_internal_cuda_fail(be, e, "flash_attn_tree attribute", __LINE__);
    e = launch_k(be, fattn_tree_wide_kernel<D, QF16>, dim3(l.grid), dim3(C::NT), C::SMEM, l.k, l.v, a, p, s, l.box,
                                   l.parts, l.joins, be->err_word);
    if (e != cudaSuccess) return oasr_internal_cuda_fail(be, e, "flash_attn_tree launch", __LINE__);
    return tree_join(be, a, p, s, C::R, l);
}

int launch_tree_wide(oasr_backend *be, const TreeAttn &a, const KvPages &p, const KvSeqs &s) {
    if (a.D == 64) return a.q_f16 ? launch_wide<64, true>(be, a, p, s) : launch_wide<64, false>(be, a, p, s);
    return a.q_f16 ? launch_wide<128, true>(be, a, p, s) : launch_wide<128, false>(be, a, p, s);
}

}  // namespace oasr
