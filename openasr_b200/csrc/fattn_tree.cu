// fattn_tree.cu -- attention for a tree of drafted tokens over the paged K/V cache.
//
//   o[i, h, s] = sum_p softmax_p(scale q[i, h, s] . k_p) v_p   over the visible positions p:
//   p < n_past[s], or p = n_past[s] + j with bit j of tree[s][i] set (no tree: j <= i);
// a node that sees nothing, or that is padding, gets zeros.
//
// K and V are read once per tile of rows and dominate the traffic, so the G query heads of a
// K/V head and all nodes of a sequence share a tile.  The kernel below takes tiles of 16 or 32
// rows with warp-level matrix instructions (m16n8k16): at 64 positions of D = 128 an SM's share
// of the HBM rate allows about 1400 clocks, and 16 rows need 256 instructions.
//
// A producer warp streams units of 64 positions of K and V into a ring by TMA (one box per run
// of positions within a page, 128-byte swizzle); of four consumer warps per 16 rows each takes
// 16 of the 64 positions with a running maximum, sum and output of its own, and the four are
// joined at the end of a segment.
#include <cudaTypedefs.h>

#include <algorithm>

#include "fattn_tree.cuh"

namespace oasr {

template <int D_, int RT_>
struct TreeMma {
    static constexpr int D = D_, RT = RT_;
    static constexpr int M = 16 * RT;             // rows per tile
    static constexpr int NS = 3;                  // units in flight
    static constexpr int HALF = TREE_BKV * 128;   // 64 positions x 64 values
    static constexpr int KBYTES = HALF * (D / 64);
    static constexpr int STAGE = 2 * KBYTES;      // K, then V
    static constexpr int CW = 4 * RT;             // consumer warps
    static constexpr int NT = 32 * (CW + 1);
    static constexpr int OFF_ML = NS * STAGE;     // [CW][16] (max, sum)
    static constexpr int OFF_BAR = OFF_ML + CW * 16 * 8;
    static constexpr int OFF_MISC = OFF_BAR + 2 * NS * 8;
    static constexpr int SMEM = OFF_MISC + 16;
    static constexpr int PART = M * (D + 2);      // floats of an unfinished segment
    static_assert(4 * 16 * D * 4 == STAGE, "the outputs of four warps fit the stage they were read from");
};

static __device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
static __device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
static __device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <int N>
static __device__ __forceinline__ void consumers_sync() {
    asm volatile("bar.sync 1, %0;" ::"n"(N) : "memory");
}
// halves that are infinite or NaN to zero; `bad` notes that there were some
static __device__ __forceinline__ uint32_t finite2(uint32_t x, uint32_t &bad) {
    const uint32_t m = __vcmpeq2(x & 0x7C007C00u, 0x7C007C00u);
    bad |= m;
    return x & ~m;
}

template <int D, int RT, bool QF16>
__global__ void __launch_bounds__(TreeMma<D, RT>::NT, RT == 1 ? 2 : 1)
    fattn_tree_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, TreeAttn a,
                      KvPages p, KvSeqs sq, int box, int least, float *parts, unsigned int *tickets, int *err) {
    using C = TreeMma<D, RT>;
    extern __shared__ __align__(1024) uint8_t smem[];
    griddep_launch_dependents();
    griddep_wait();
    if (smem_u32(smem) & 1023u) {  // the swizzle needs it
        if (threadIdx.x == 0) atomicOr(err, ERR_BAD_SHAPE);
        return;
    }
    uint64_t *full = (uint64_t *)(smem + C::OFF_BAR), *empty = full + C::NS;
    volatile int *abort_flag = (volatile int *)(smem + C::OFF_MISC);
    unsigned int *s_bad = (unsigned int *)(smem + C::OFF_MISC + 4);
    int *s_last = (int *)(smem + C::OFF_MISC + 8);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int G = a.H / a.HKV;
    if (threadIdx.x == 0) {
        for (int i = 0; i < C::NS; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], C::CW);
        }
        *abort_flag = 0;
        *s_bad = 0;
        fence_mbar_init();
    }
    TreeUnits w;
    w.total = tree_count(a, sq, p.page, C::M, err);
    w.ctas = (int)max((int64_t)1, min((int64_t)gridDim.x, w.total / least));
    const int64_t u0 = (int)blockIdx.x < w.ctas ? tree_start(w, blockIdx.x) : 0;
    const int64_t u1 = (int)blockIdx.x < w.ctas ? tree_start(w, blockIdx.x + 1) : 0;
    __syncthreads();

    if (warp == C::CW) {
        // ---- producer: lane = (box, half of D, K or V) ----
        constexpr int PER = 2 * (D / 64);  // copies per box
        const int boxes = TREE_BKV / box;
        const int b = lane / PER, half = lane / 2 % (D / 64), kv = lane & 1;
        const bool mine = b < boxes;
        const CUtensorMap *map = kv ? &tm_v : &tm_k;
        int64_t it = 0;
        for (int64_t u = u0; u < u1;) {
            const TreeSeg g = tree_locate(a, sq, p.page, C::M, u, u1);
            const int *row = sq.table + g.s * sq.table_ld;
            for (int k = g.k0; k < g.k1; ++k, ++it) {
                // positions past the end read page n_pages: zeros
                const int t = k * TREE_BKV + b * box;
                int pg = p.n_pages;
                if (mine && t < g.T) {
                    pg = __ldg(row + t / p.page);
                    if (pg < 0 || pg >= p.n_pages) {
                        atomicOr(err, ERR_BAD_INDEX);
                        pg = p.n_pages;
                    }
                }
                const int slot = (int)(it % C::NS);
                if (!mbar_wait(&empty[slot], (uint32_t)(it / C::NS & 1) ^ 1u, abort_flag, err)) continue;
                if (lane == 0) mbar_arrive_expect_tx(&full[slot], C::STAGE);
                __syncwarp();
                if (mine)
                    tma_load_4d(smem + slot * C::STAGE + kv * C::KBYTES + half * C::HALF + b * box * 128, map, &full[slot],
                                64 * half, t % p.page, g.hk, pg);
                __syncwarp();
            }
            u = g.first + g.k1;
        }
        // copies still in flight when the consumers gave up land before the block ends
        if (*abort_flag)
            for (int i = 0; i < C::NS; ++i) {
                const long long t0 = clock64();
                const uint32_t ph = (uint32_t)((it + C::NS - 1 - i) / C::NS & 1) ^ 1u;
                while (!mbar_try_wait(&full[i], ph) && clock64() - t0 < (1LL << 24)) {
                }
            }
        return;
    }

    // ---- consumers ----
    tree_zero_padding(a, sq, p.page, (int64_t)blockIdx.x * C::CW + warp, (int64_t)gridDim.x * C::CW);
    const int kg = warp & 3, rl = warp >> 2;  // 16 positions of the unit, 16 rows of the tile
    const int gr = lane >> 2, c = lane & 3;   // fragment row and column pair
    float2 *s_ml = (float2 *)(smem + C::OFF_ML);
    int64_t it = 0;
    for (int64_t u = u0; u < u1;) {
        const TreeSeg g = tree_locate(a, sq, p.page, C::M, u, u1);
        const int R = g.n * G;
        // Q fragments: rows r0 and r0 + 8; f32 queries as two f16 halves after a power of two
        // that brings the row's largest value to 2^8
        const int r0 = g.rt * C::M + 16 * rl + gr;
        uint32_t qh[D / 16][4], ql[QF16 ? 1 : D / 16][4];
        float sc[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const int r = r0 + 8 * x;
            const bool in = r < R;
            const char *qr = a.q + (in ? r / G : 0) * a.q_nb1 + (g.hk * G + (in ? r % G : 0)) * a.q_nb2 + g.s * a.q_nb3;
            sc[x] = a.scale * 1.4426950408889634f;
            if (QF16) {
#pragma unroll
                for (int k = 0; k < D / 16; ++k) {
                    qh[k][x] = in ? *reinterpret_cast<const uint32_t *>(qr + 2 * (16 * k + 2 * c)) : 0u;
                    qh[k][x + 2] = in ? *reinterpret_cast<const uint32_t *>(qr + 2 * (16 * k + 8 + 2 * c)) : 0u;
                }
            } else {
                float2 v[D / 8];
                float m = 0.0f;
#pragma unroll
                for (int k = 0; k < D / 8; ++k) {
                    v[k] = in ? *reinterpret_cast<const float2 *>(qr + 4 * (8 * k + 2 * c)) : make_float2(0.0f, 0.0f);
                    m = fmaxf(m, fmaxf(fabsf(v[k].x), fabsf(v[k].y)));
                }
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
                m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
                // exponents of the factor 2^(8 - e) and of its inverse, both in the normal range
                const int e = min(max((int)(__float_as_uint(m) >> 23) - 127, -100), 100);
                const float up = __uint_as_float((uint32_t)(127 + 8 - e) << 23);
                sc[x] *= __uint_as_float((uint32_t)(127 + e - 8) << 23);
#pragma unroll
                for (int k = 0; k < D / 16; ++k) {
                    tree_split2(v[2 * k].x * up, v[2 * k].y * up, qh[k][x], ql[k][x]);
                    tree_split2(v[2 * k + 1].x * up, v[2 * k + 1].y * up, qh[k][x + 2], ql[k][x + 2]);
                }
            }
        }
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
        float o[D / 8][4];
#pragma unroll
        for (int j = 0; j < D / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.0f;
        uint32_t bad = 0;

        for (int k = g.k0; k < g.k1; ++k, ++it) {
            const int slot = (int)(it % C::NS);
            const bool tail = (k + 1) * TREE_BKV > g.past;  // some of the positions are nodes, or past the end
            uint32_t see[2] = {0xffffu, 0xffffu};
            if (tail) {
                see[0] = tree_sees(a, g, r0 / G, k * TREE_BKV + 16 * kg);
                see[1] = tree_sees(a, g, (r0 + 8) / G, k * TREE_BKV + 16 * kg);
            }
            if (mbar_wait(&full[slot], (uint32_t)(it / C::NS & 1), abort_flag, err)) {
                const uint32_t kb = smem_u32(smem + slot * C::STAGE), vb = kb + C::KBYTES;
                // S = Q K^T: two 8-position tiles, the 16-bit halves of Q in accumulators of their own
                float s[2][2][4] = {};
                const int kr = 16 * kg + (lane & 7) + 8 * (lane >> 4);  // this lane's row of the K matrices
#pragma unroll
                for (int x = 0; x < D / 16; ++x) {
                    // matrices: positions 0-7 x values 0-7, 8-15; positions 8-15 x values 0-7, 8-15
                    uint32_t f[4];
                    ldsm4(f, kb + (x / 4) * C::HALF + sw128_off(kr, (x & 3) * 2 + (lane >> 3 & 1)));
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        mma16816(s[t][QF16 ? x & 1 : 0], qh[x], f[2 * t], f[2 * t + 1]);
                        if (!QF16) mma16816(s[t][1], ql[x], f[2 * t], f[2 * t + 1]);
                    }
                }
                float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int x = e >> 1;
                        float v = (s[t][0][e] + s[t][1][e]) * sc[x];
                        if (tail && !(see[x] >> (8 * t + 2 * c + (e & 1)) & 1u)) v = -INFINITY;
                        s[t][0][e] = v;
                        mx[x] = fmaxf(mx[x], v);
                    }
                float f[2], off[2];
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    mx[x] = fmaxf(mx[x], __shfl_xor_sync(0xffffffffu, mx[x], 1));
                    mx[x] = fmaxf(mx[x], __shfl_xor_sync(0xffffffffu, mx[x], 2));
                    mx[x] = fmaxf(mx[x], m[x]);
                    off[x] = mx[x] == -INFINITY ? 0.0f : mx[x] - TREE_WEIGHT_EXP;
                    f[x] = mx[x] == -INFINITY ? 1.0f : tree_exp2(m[x] - mx[x]);
                    m[x] = mx[x];
                    l[x] *= f[x];
                }
                uint32_t ph[4], pl[4];
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const float p0 = tree_exp2(s[t][0][2 * x] - off[x]), p1 = tree_exp2(s[t][0][2 * x + 1] - off[x]);
                        l[x] += p0 + p1;
                        tree_split2(p0, p1, ph[2 * t + x], pl[2 * t + x]);
                    }
                // O = f O + P V, the product of this unit in accumulators of its own: the tensor
                // cores cut the bits below a large running sum off, an f32 multiply-add rounds
                const int vr = 16 * kg + (lane & 15);
                uint32_t keep0 = 0xffffffffu, keep1 = 0xffffffffu;
                if (tail) {  // positions past the end hold anything
                    const int left = g.T - (k * TREE_BKV + 16 * kg + 2 * c);
                    keep0 = left >= 2 ? 0xffffffffu : left == 1 ? 0xffffu : 0u;
                    keep1 = left >= 10 ? 0xffffffffu : left == 9 ? 0xffffu : 0u;
                }
#pragma unroll
                for (int j = 0; j < D / 16; ++j) {
                    // matrices: positions 0-7, 8-15 x values 0-7; the same x values 8-15
                    uint32_t v[4];
                    ldsm4_t(v, vb + (j / 4) * C::HALF + sw128_off(vr, (j & 3) * 2 + (lane >> 4)));
                    if (tail) {
                        v[0] = finite2(v[0] & keep0, bad);
                        v[1] = finite2(v[1] & keep1, bad);
                        v[2] = finite2(v[2] & keep0, bad);
                        v[3] = finite2(v[3] & keep1, bad);
                    }
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        float d[4] = {};
                        mma16816(d, ph, v[2 * t], v[2 * t + 1]);
                        mma16816(d, pl, v[2 * t], v[2 * t + 1]);
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[2 * j + t][e] = fmaf(o[2 * j + t][e], f[e >> 1], d[e]);
                    }
                }
            }
            if (k + 1 < g.k1) {  // the last one is kept for the join below
                fence_proxy_async_smem();  // these reads before the copy that refills the stage
                __syncwarp();
                if (lane == 0) mbar_arrive(&empty[slot]);
            }
        }

        // ---- join the four warps of each 16 rows, 16 rows at a time through the last stage ----
        uint8_t *last = smem + (int)((it - 1) % C::NS) * C::STAGE;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
            l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
            if (c == 0) s_ml[warp * 16 + gr + 8 * x] = make_float2(m[x], l[x]);
        }
        if (bad) atomicOr(s_bad, 1u);
        consumers_sync<32 * C::CW>();
        const bool anybad = *s_bad != 0;
        const bool whole = g.k0 == 0 && g.k1 == g.kt;
        float *part = parts + tree_slot(w, blockIdx.x, g.first) * C::PART;
#pragma unroll
        for (int x = 0; x < 2; ++x) {  // this warp's factor for its rows
            const int r = gr + 8 * x;
            float M = -INFINITY;
#pragma unroll
            for (int i = 0; i < 4; ++i) M = fmaxf(M, s_ml[(rl * 4 + i) * 16 + r].x);
            const float f = m[x] == -INFINITY ? 0.0f : tree_exp2(m[x] - M);
#pragma unroll
            for (int j = 0; j < D / 8; ++j) {
                o[j][2 * x] *= f;
                o[j][2 * x + 1] *= f;
            }
        }
#pragma unroll
        for (int pass = 0; pass < RT; ++pass) {
            if (rl == pass) {
#pragma unroll
                for (int x = 0; x < 2; ++x)
#pragma unroll
                    for (int j = 0; j < D / 8; ++j) {
                        const int r = gr + 8 * x, ch = (2 * j + (c >> 1)) ^ gr;  // 16-byte pieces spread over the banks
                        *reinterpret_cast<float2 *>(last + (((kg * 16 + r) * D + 4 * ch) * 4 + 8 * (c & 1))) =
                            make_float2(o[j][2 * x], o[j][2 * x + 1]);
                    }
            }
            consumers_sync<32 * C::CW>();
            if (threadIdx.x == 0) *s_bad = 0;  // everybody has read it
            for (int e = threadIdx.x; e < 16 * (D / 4); e += 32 * C::CW) {
                const int r = e / (D / 4), ch = e % (D / 4);
                const int gl = g.rt * C::M + 16 * pass + r;
                float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                float M = -INFINITY, L = 0.0f;
#pragma unroll
                for (int i = 0; i < 4; ++i) M = fmaxf(M, s_ml[(pass * 4 + i) * 16 + r].x);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 ml = s_ml[(pass * 4 + i) * 16 + r];
                    L += ml.x == -INFINITY ? 0.0f : ml.y * tree_exp2(ml.x - M);
                    const float4 x = *reinterpret_cast<const float4 *>(last + ((i * 16 + r) * D + 4 * (ch ^ (r & 7))) * 4);
                    v.x += x.x; v.y += x.y; v.z += x.z; v.w += x.w;
                }
                if (anybad && gl < R) v = tree_nonfinite4(a, p, sq, g, gl / G, 4 * ch, v);
                if (whole) {
                    if (gl < R) {
                        const float inv = L == 0.0f ? 0.0f : 1.0f / L;
                        tree_store4(a, g.s, g.hk * G + gl % G, gl / G, 4 * ch, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
                    }
                } else {
                    *reinterpret_cast<float4 *>(part + (16 * pass + r) * D + 4 * ch) = v;
                    if (ch == 0) *reinterpret_cast<float2 *>(part + C::M * D + 2 * (16 * pass + r)) = make_float2(M, L);
                }
            }
            fence_proxy_async_smem();
            consumers_sync<32 * C::CW>();
        }
        if (lane == 0) mbar_arrive(&empty[(it - 1) % C::NS]);

        // ---- the last of the CTAs that share the item joins their parts in order ----
        if (!whole) {
            const int c0 = tree_owner(w, g.first), c1 = tree_owner(w, g.first + g.kt - 1);
            if (threadIdx.x == 0) {
                const bool is_last = atom_add_acq_rel_gpu(tickets + c0, 1u) == (unsigned)(c1 - c0);
                if (is_last) atomicExch(tickets + c0, 0u);
                *s_last = is_last;
            }
            consumers_sync<32 * C::CW>();
            if (*s_last) {
                for (int e = threadIdx.x; e < C::M * (D / 4); e += 32 * C::CW) {
                    const int r = e / (D / 4), ch = e % (D / 4), gl = g.rt * C::M + r;
                    if (gl >= R) continue;
                    float M = -INFINITY, L = 0.0f;
                    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    for (int x = c0; x <= c1; ++x)
                        M = fmaxf(M, __ldcg(reinterpret_cast<const float2 *>(parts + tree_slot(w, x, g.first) * C::PART + C::M * D) + r).x);
                    for (int x = c0; x <= c1; ++x) {
                        const float *pt = parts + tree_slot(w, x, g.first) * C::PART;
                        const float2 ml = __ldcg(reinterpret_cast<const float2 *>(pt + C::M * D) + r);
                        const float4 y = __ldcg(reinterpret_cast<const float4 *>(pt + r * D) + ch);
                        const float f = ml.x == -INFINITY ? 0.0f : tree_exp2(ml.x - M);
                        L = fmaf(ml.y, f, L);
                        v.x = fmaf(y.x, f, v.x); v.y = fmaf(y.y, f, v.y);
                        v.z = fmaf(y.z, f, v.z); v.w = fmaf(y.w, f, v.w);
                    }
                    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
                    tree_store4(a, g.s, g.hk * G + gl % G, gl / G, 4 * ch, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
                }
            }
        }
        u = g.first + g.k1;
    }
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

template <int D, int RT, bool QF16>
static int launch_tree_mma(oasr_backend *be, const TreeAttn &a, const KvPages &p, const KvSeqs &s, const CUtensorMap &mk,
                           const CUtensorMap &mv, int box) {
    using C = TreeMma<D, RT>;
    static std::atomic<bool> attr_set{false};
    if (!attr_set) {
        const cudaError_t e =
            cudaFuncSetAttribute(fattn_tree_kernel<D, RT, QF16>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
        if (e != cudaSuccess) return oasr_internal_cuda_fail(be, e, "flash_attn_tree attribute", __LINE__);
        attr_set = true;
    }
    const int64_t rts = ((int64_t)s.N * (a.H / a.HKV) + C::M - 1) / C::M;
    const int64_t most = rts * a.HKV * a.S * (((int64_t)s.MP * p.page + TREE_BKV - 1) / TREE_BKV);
    const int grid = (int)std::max<int64_t>(1, std::min<int64_t>(most, (int64_t)be->sm_count * (RT == 1 ? 2 : 1)));
    int st = 0;
    float *parts = (float *)oasr_internal_scratch(be, (size_t)grid * 2 * C::PART * 4, &st);
    if (st) return st;
    const cudaError_t e = launch_k(be, fattn_tree_kernel<D, RT, QF16>, dim3(grid), dim3(C::NT), C::SMEM, mk, mv, a, p, s, box,
                                   1, parts, be->counters, be->err_word);
    if (e != cudaSuccess) return oasr_internal_cuda_fail(be, e, "flash_attn_tree launch", __LINE__);
    return oasr_internal_launch_check(be, "flash_attn_tree");
}

int launch_flash_attn_tree(oasr_backend *be, const TreeAttn &a, const KvPages &p, const KvSeqs &s) {
    // the longest run of positions, up to a unit, that never crosses a page
    const int box = std::min(TREE_BKV, p.page & -p.page);
    CUtensorMap mk, mv;
    if (!tree_page_map(&mk, p.k, p.k_nb1, p.k_nb2, p.k_nb3, a.D, p.page, a.HKV, p.n_pages, box) ||
        !tree_page_map(&mv, p.v, p.v_nb1, p.v_nb2, p.v_nb3, a.D, p.page, a.HKV, p.n_pages, box))
        return oasr_internal_fail(be, OASR_STATUS_FAILED, "flash_attn_tree: the pages' strides make no tensor map");
    const bool two = (int64_t)s.N * (a.H / a.HKV) > 16;
#define FT(DD, RR, Q) \
    if (a.D == DD && two == (RR == 2) && a.q_f16 == Q) return launch_tree_mma<DD, RR, Q>(be, a, p, s, mk, mv, box)
    FT(64, 1, false); FT(64, 1, true); FT(64, 2, false); FT(64, 2, true);
    FT(128, 1, false); FT(128, 1, true); FT(128, 2, false); FT(128, 2, true);
#undef FT
    return oasr_internal_fail(be, OASR_STATUS_FAILED, "flash_attn_tree: head_dim must be 64 or 128");
}

}  // namespace oasr
