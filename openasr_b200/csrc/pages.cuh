// pages.cuh -- the paged K/V cache as the kernels see it (kv_pages.cu, fattn_tree.cu).
#pragma once

#include "kernels.cuh"
#include "tree_split.h"

namespace oasr {

// Most nodes per sequence that a drafted tree may have (mask words and the acceptance walk
// live in shared memory); a chain (no tree tensor) may be longer.
constexpr int TREE_MAX_NODES = 1024;

// K and V pages [D, page, n_kv_heads, n_pages] f16 with their byte strides.
struct KvPages {
    char *k, *v;
    int64_t k_nb1, k_nb2, k_nb3;  // position, head, page
    int64_t v_nb1, v_nb2, v_nb3;
    int n_pages;
    int page;  // positions per page
};

// Which page holds which positions, and how far each sequence is.
struct KvSeqs {
    const int *table;  // [S] rows of MP page ids, table_ld ints apart
    int64_t table_ld;
    int MP;
    const int *n_past;   // [S] committed positions
    const int *n_nodes;  // [S] live nodes, or null: N everywhere
    int N;               // nodes per sequence in the tensors
};

// Committed positions and live nodes of sequence s; a sequence whose lengths do not fit its
// page table or the tensors is taken as empty (the caller records ERR_BAD_INDEX).
static __device__ __forceinline__ bool seq_lengths(const KvSeqs &q, int s, int page, int &past, int &n) {
    past = q.n_past[s];
    n = q.n_nodes ? q.n_nodes[s] : q.N;
    if (!kv_lengths_fit(past, n, q.N, q.MP, page)) {
        past = n = 0;
        return false;
    }
    return true;
}

// Argument checks shared by the entry points of the paged cache: a status, and the structs.
// `layers` > 1: the pages of all layers follow each other along ne3, n_pages is per layer.
int pages_check(oasr_backend *be, const char *op, const oasr_tensor *k, const oasr_tensor *v, int layers, KvPages *out);
int seqs_check(oasr_backend *be, const char *op, const oasr_tensor *table, const oasr_tensor *n_past,
               const oasr_tensor *n_nodes, int64_t S, int64_t N, KvSeqs *out);

// n / d for 0 <= n < 2^31 by a multiplication (Granlund and Montgomery, 1994): with s =
// ceil(log2 d) and m = floor(2^32 (2^s - d) / d) + 1, n / d = (mulhi(n, m) + n) >> s.
struct FastDiv {
    uint32_t m;
    int s, d;
    FastDiv() = default;
    explicit FastDiv(int div) : d(div) {
        for (s = 0; (1ll << s) < div; ++s) {
        }
        m = (uint32_t)((((1ull << s) - (uint64_t)div) << 32) / (uint64_t)div + 1);
    }
    __device__ __forceinline__ int operator()(int n) const {
        return (int)((__umulhi((uint32_t)n, m) + (uint32_t)n) >> s);
    }
};

// attention of N nodes per sequence over the pages (fattn_tree.cu)
struct TreeAttn {
    const char *q;
    int64_t q_nb1, q_nb2, q_nb3;  // node, head, sequence
    char *dst;
    int64_t d_nb1, d_nb2, d_nb3;  // head, node, sequence
    const int *tree;              // [S][N] rows of W words, or null: node i sees nodes 0..i
    int64_t t_nb1, t_nb2;         // in ints: node, sequence
    int S, H, HKV, D, W;
    float scale;
    bool q_f16, d_f16;
    FastDiv group, page;          // H / HKV, positions per page
};
int launch_flash_attn_tree(oasr_backend *be, const TreeAttn &a, const KvPages &p, const KvSeqs &s);

}  // namespace oasr
