// What the kernels of tree attention share: which keys a node sees, how a launch's work is dealt out, and the merge of its parts.
//
// A sequence brings a tree of n nodes behind its pos0 cached tokens. Node i is a query row; its own key lies at place pos0 + i of the
// sequence's cache, its position is row_pos (pos0 + its depth). It sees the cached tokens (within the window, by position) and the
// nodes j whose bit is set in its row of the tree's bits (within the window too).
//
// Work is counted in units: one page of keys for one tile of rows, a tile being up to tile_nodes nodes x the G query heads of a kv
// head. The units of all sequences stand in one run (sequence, kv head, tile, page), and block b of nb takes the b-th of nb equal
// shares, so lengths that differ leave no block idle, and the lengths may change under a captured graph: only device arrays say them.
// A block that holds all pages of a tile writes the tile's rows; else it leaves a part (maximum, sum, sum of P.V) in one of its two
// slots: 2 b + 1 for the tile its share begins (and does not end), 2 b for one that began in an earlier block.
#pragma once
#include "common.cuh"

struct TreeArgs {
    const int *cu_q, *seq_pos0, *row_pos, *page_table;
    const uint32_t* tree;                  // [rows, words]
    int n_seq, words, pt_stride, n_pages, nh, nkv, window, tile_nodes;
    float sl2;                             // scale * log2(e)
};

// One sequence as the work is counted.
struct TreeSeq {
    int n, pos0, first_page, pages, tiles, flat0;
    __device__ __forceinline__ void load(const TreeArgs& a, int s) {
        flat0 = a.cu_q[s];
        n = max(0, a.cu_q[s + 1] - flat0);
        pos0 = max(0, a.seq_pos0[s]);
        tiles = (n + a.tile_nodes - 1) / a.tile_nodes;
        // pages that the table has no column for hold no keys; one page at least, so that rows without a key are written too
        const int end = min((pos0 + n + DK_PAGE - 1) / DK_PAGE, a.pt_stride);
        first_page = min((a.window > 0 ? max(0, pos0 - a.window + 1) : 0) / DK_PAGE, a.pt_stride - 1);
        pages = max(1, end - first_page);
    }
    __device__ __forceinline__ long long units(int nkv) const { return (long long)tiles * nkv * pages; }
};

__device__ __forceinline__ long long warp_scan(long long v) {          // inclusive
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
    }
    return v;
}

// Units before sequence `upto` (n_seq: all of them). A whole warp calls it.
__device__ __forceinline__ long long tree_units(const TreeArgs& a, int upto) {
    long long sum = 0;
    for (int s = threadIdx.x & 31; s < upto; s += 32) {
        TreeSeq q;
        q.load(a, s);
        sum += q.units(a.nkv);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    return sum;
}

// The sequence that unit u (below the total) belongs to, and the units before it. A whole warp calls it.
__device__ __forceinline__ int tree_find(const TreeArgs& a, long long u, long long& before) {
    const int lane = threadIdx.x & 31;
    before = 0;
    for (int s0 = 0; s0 < a.n_seq; s0 += 32) {
        long long mine = 0;
        if (s0 + lane < a.n_seq) {
            TreeSeq q;
            q.load(a, s0 + lane);
            mine = q.units(a.nkv);
        }
        const long long upto = warp_scan(mine);
        const unsigned past = __ballot_sync(0xffffffffu, before + upto > u);
        if (past) {
            const int l = __ffs(past) - 1;
            before += __shfl_sync(0xffffffffu, upto - mine, l);
            return s0 + l;
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
    }
    return a.n_seq;
}

// Shares of a launch of `blocks`.
__device__ __forceinline__ int share_count(long long total, int blocks) { return (int)min(total, (long long)blocks); }
// Block b's share begins at this unit; the share that unit u lies in.
__device__ __forceinline__ long long share_begin(long long total, int b, int nb) { return total * b / nb; }
__device__ __forceinline__ int share_of(long long total, long long u, int nb) { return (int)(((u + 1) * nb - 1) / total); }

// Bits of the places [key0, key0 + 64) that a node sees; `words`: its row of the tree's bits; `pos`: its position, < 0 for none.
__device__ __forceinline__ uint64_t tree_mask(const TreeArgs& a, const TreeSeq& q, const uint32_t* words, int pos, int key0) {
    if (pos < 0) return 0;
    auto low = [](int k) { return k <= 0 ? 0ull : k >= 64 ? ~0ull : (1ull << k) - 1; };   // the first k bits
    uint64_t m = low(q.pos0 - key0);
    if (a.window > 0) m &= ~low(max(0, pos - a.window + 1) - key0);
    const int j0 = key0 - q.pos0;                                       // the node at place key0
    if (j0 > -64 && j0 < q.n) {
        auto word = [&](int w) { return w >= 0 && w < a.words ? (uint64_t)words[w] : 0ull; };
        uint64_t t;
        if (j0 < 0) t = (word(0) | word(1) << 32) << -j0;
        else {
            const int w = j0 >> 5, sh = j0 & 31;
            t = (word(w) | word(w + 1) << 32) >> sh;
            if (sh) t |= word(w + 2) << (64 - sh);
        }
        t &= low(q.n - j0) & ~low(-j0);
        if (a.window > 0 && a.window < q.n)                            // a tree deeper than the window
            for (uint64_t left = t; left; left &= left - 1) {
                const int b = __ffsll((long long)left) - 1;
                if (pos - a.row_pos[q.flat0 + j0 + b] >= a.window) t &= ~(1ull << b);
            }
        m |= t;
    }
    return m;
}

// Merges the parts of the tiles that more than one block worked on; the others have been written. A warp a row of one query head,
// grid (ceil(max_nodes * nh / 8), n_seq), 256 threads. tile_rows: rows a slot has room for.
template <typename T, int D>
__global__ void __launch_bounds__(256)
tree_merge_kernel(TreeArgs a, const float* ws_acc, const float2* ws_ml, T* out, long long ldo, int tile_rows, int blocks) {
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31, s = blockIdx.y, G = a.nh / a.nkv;
    const int i = blockIdx.x * 8 + (threadIdx.x >> 5), node = i / a.nh, h = i % a.nh, kvh = h / G;
    TreeSeq q;
    q.load(a, s);
    if (node >= q.n) return;
    const long long total = tree_units(a, a.n_seq);
    const int tile = node / a.tile_nodes;
    const int nb = share_count(total, blocks);
    const long long u0 = tree_units(a, s) + ((long long)kvh * q.tiles + tile) * q.pages;
    const int b0 = share_of(total, u0, nb), b1 = share_of(total, u0 + q.pages - 1, nb);
    if (b0 == b1) return;
    const int row = (node - tile * a.tile_nodes) * G + h % G;
    constexpr int C = (D + 31) / 32;
    float m = -INFINITY, l = 0.f, acc[C];
#pragma unroll
    for (int c = 0; c < C; c++) acc[c] = 0.f;
    for (int b = b0; b <= b1; b++) {
        const size_t at = (size_t)(2 * b + (b == b0 ? 1 : 0)) * tile_rows + row;
        const float2 ml = ws_ml[at];
        const float mn = fmaxf(m, ml.x), ms = mn == -INFINITY ? 0.f : mn;
        const float fa = exp2f(m - ms), fb = exp2f(ml.x - ms);
        l = l * fa + ml.y * fb;
#pragma unroll
        for (int c = 0; c < C; c++) {
            const int d = c * 32 + lane;
            if (d < D) acc[c] = acc[c] * fa + ws_acc[at * D + d] * fb;
        }
        m = mn;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;                        // no key at all: a row of zeros
#pragma unroll
    for (int c = 0; c < C; c++) {
        const int d = c * 32 + lane;
        if (d < D) out[(size_t)(q.flat0 + node) * ldo + h * D + d] = from_f<T>(acc[c] * inv);
    }
}
