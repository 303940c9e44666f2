// fattn_tree.cu -- attention for a tree of drafted tokens over the paged K/V cache.
//
//   o[i, h, s] = sum_p softmax_p(scale q[i, h, s] . k_p) v_p   over the visible positions p:
//   p < n_past[s], or p = n_past[s] + j with bit j of tree[s][i] set (no tree: j <= i);
// a node that sees nothing, or that is padding, gets zeros.
//
// One CTA per (node, head, sequence); each of its 4 warps takes every fourth position, D / 32
// values per lane, with its own running maximum, sum and output; the four are joined at the end.
#include "pages.cuh"

namespace oasr {

template <int D, bool QF16, bool DF16>
__global__ void __launch_bounds__(128) fattn_tree_kernel(TreeAttn a, KvPages p, KvSeqs sq, int *err) {
    constexpr int V = D / 32;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int h = (int)(blockIdx.x % a.H);
    const int i = (int)(blockIdx.x / a.H % sq.N), s = (int)(blockIdx.x / a.H / sq.N);
    const int hk = h / (a.H / a.HKV);
    int past, n;
    if (!seq_lengths(sq, s, p.page, past, n) && threadIdx.x == 0) atomicOr(err, ERR_BAD_INDEX);
    float q[V], o[V];
    const char *qr = a.q + i * a.q_nb1 + h * a.q_nb2 + s * a.q_nb3;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        q[j] = QF16 ? __half2float(reinterpret_cast<const __half *>(qr)[V * lane + j]) : reinterpret_cast<const float *>(qr)[V * lane + j];
        o[j] = 0.0f;
    }
    float m = -INFINITY, l = 0.0f;
    const int T = i < n ? past + n : 0;
    for (int t = warp; t < T; t += 4) {
        const int node = t - past;
        if (node >= 0) {
            const bool see = a.tree ? (a.tree[s * a.t_nb2 + i * a.t_nb1 + node / 32] >> (node % 32)) & 1 : node <= i;
            if (!see) continue;
        }
        const int pg = sq.table[s * sq.table_ld + t / p.page];
        if (pg < 0 || pg >= p.n_pages) {
            if (lane == 0) atomicOr(err, ERR_BAD_INDEX);
            continue;
        }
        const int64_t off = t % p.page;
        const __half *k = reinterpret_cast<const __half *>(p.k + pg * p.k_nb3 + hk * p.k_nb2 + off * p.k_nb1) + V * lane;
        const __half *v = reinterpret_cast<const __half *>(p.v + pg * p.v_nb3 + hk * p.v_nb2 + off * p.v_nb1) + V * lane;
        float d = 0.0f;
#pragma unroll
        for (int j = 0; j < V; ++j) d = fmaf(q[j], __half2float(k[j]), d);
        const float x = warp_sum(d) * a.scale;
        const float mn = fmaxf(m, x);
        const float f = mn == -INFINITY ? 1.0f : expf(m - mn), w = mn == -INFINITY ? 0.0f : expf(x - mn);
        l = l * f + w;
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] = o[j] * f + w * __half2float(v[j]);
        m = mn;
    }
    __shared__ float sm[4], sl[4], so[4][D];
    if (lane == 0) { sm[warp] = m; sl[warp] = l; }
#pragma unroll
    for (int j = 0; j < V; ++j) so[warp][V * lane + j] = o[j];
    __syncthreads();
    const int e = threadIdx.x;
    if (e >= D) return;
    const float M = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
    float L = 0.0f, O = 0.0f;
    for (int w = 0; w < 4; ++w) {
        if (sm[w] == -INFINITY) continue;
        const float f = expf(sm[w] - M);
        L += sl[w] * f;
        O += so[w][e] * f;
    }
    const float r = L == 0.0f ? 0.0f : O / L;
    char *out = a.dst + h * a.d_nb1 + i * a.d_nb2 + s * a.d_nb3;
    if (DF16) reinterpret_cast<__half *>(out)[e] = __float2half_rn(r);
    else reinterpret_cast<float *>(out)[e] = r;
}

int launch_flash_attn_tree(oasr_backend *be, const TreeAttn &a, const KvPages &p, const KvSeqs &s) {
    const int64_t grid = (int64_t)a.S * s.N * a.H;
    if (grid > INT32_MAX) return oasr_internal_fail(be, OASR_STATUS_FAILED, "flash_attn_tree: too many rows");
    cudaError_t e = cudaSuccess;
#define FT(DD, Q, O)                                                  \
    if (a.D == DD && a.q_f16 == Q && a.d_f16 == O)                    \
    e = launch_k(be, fattn_tree_kernel<DD, Q, O>, dim3((unsigned)grid), dim3(128), 0, a, p, s, be->err_word)
    FT(64, false, false); FT(64, false, true); FT(64, true, false); FT(64, true, true);
    FT(128, false, false); FT(128, false, true); FT(128, true, false); FT(128, true, true);
#undef FT
    if (e != cudaSuccess) return oasr_internal_cuda_fail(be, e, "flash_attn_tree launch", __LINE__);
    return oasr_internal_launch_check(be, "flash_attn_tree");
}

}  // namespace oasr
