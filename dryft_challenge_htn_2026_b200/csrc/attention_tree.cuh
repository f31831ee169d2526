// What the kernels of tree attention share: which keys a node sees, how a launch's work is dealt out, and the merge of its parts.
//
// A sequence brings a tree of n nodes behind its pos0 cached tokens. Node i is a query row; its own key lies at place pos0 + i of the
// sequence's cache, its position is row_pos (pos0 + its depth). It sees the cached tokens (within the window, by position) and the
// nodes j whose bit is set in its row of the tree's bits (within the window too).
//
// Work is counted in units: one page of keys for one tile of rows, a tile being up to tile_nodes nodes x the G query heads of a kv
// head (laid out as halves of half_nodes nodes, each half_rows rows apart in a slot). The units of all sequences stand in one run (sequence, kv head, tile, page), and block b of nb takes the b-th of nb equal
// shares, so lengths that differ leave no block idle, and the lengths may change under a captured graph: only device arrays say them.
// A block that holds all pages of a tile writes the tile's rows; else it leaves a part (maximum, sum, sum of P.V) in one of its two
// slots: 2 b + 1 for the tile its share begins (and does not end), 2 b for one that began in an earlier block.
#pragma once
#include "common.cuh"

struct TreeArgs {
    const int *cu_q, *seq_pos0, *row_pos, *page_table;
    const uint32_t* tree;                  // [rows, words]
    int n_seq, words, pt_stride, n_pages, nh, nkv, window, tile_nodes, half_nodes, half_rows;
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
    __device__ __forceinline__ int units(int nkv) const { return tiles * nkv * pages; }
};

__device__ __forceinline__ int warp_scan(int v) {          // inclusive
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
    }
    return v;
}

// Units of all sequences (the launch has seen to it that they stay below 2^31), and of those before sequence `upto`. A whole warp
// calls it.
__device__ __forceinline__ int tree_units(const TreeArgs& a, int upto, int& before) {
    int sum = 0, first = 0;
    for (int s = threadIdx.x & 31; s < a.n_seq; s += 32) {
        TreeSeq q;
        q.load(a, s);
        sum += q.units(a.nkv);
        if (s < upto) first += q.units(a.nkv);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        sum += __shfl_xor_sync(0xffffffffu, sum, o);
        first += __shfl_xor_sync(0xffffffffu, first, o);
    }
    before = first;
    return sum;
}

// The sequence that unit u (below the total) belongs to, and the units before it. A whole warp calls it.
__device__ __forceinline__ int tree_find(const TreeArgs& a, int u, int& before) {
    const int lane = threadIdx.x & 31;
    before = 0;
    for (int s0 = 0; s0 < a.n_seq; s0 += 32) {
        int mine = 0;
        if (s0 + lane < a.n_seq) {
            TreeSeq q;
            q.load(a, s0 + lane);
            mine = q.units(a.nkv);
        }
        const int upto = warp_scan(mine);
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
__device__ __forceinline__ int share_count(int total, int blocks) { return min(total, blocks); }
// Block b's share begins at this unit; the share that unit u lies in.
__device__ __forceinline__ int share_begin(int total, int b, int nb) { return (int)((long long)total * b / nb); }
__device__ __forceinline__ int share_of(int total, int u, int nb) { return (int)(((long long)(u + 1) * nb - 1) / total); }

// Where column d of row `row` of a slot lies among its tile_rows * D numbers: four columns of a row side by side, then the next row's,
// so that threads with a row each write and read whole lines.
__device__ __forceinline__ size_t part_at(int tile_rows, int row, int d) { return ((size_t)(d >> 2) * tile_rows + row) * 4 + (d & 3); }

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

// Merges the parts of the tiles that more than one block worked on; the others have been written. Grid (row groups of the largest
// tree, nkv, n_seq), 256 threads: a block has 32 rows of a tile, lane k its k-th, each warp an eighth of the columns.
template <typename T, int D>
__global__ void __launch_bounds__(256)
tree_merge_kernel(TreeArgs a, const float* ws_acc, const float2* ws_ml, T* out, long long ldo, int tile_rows, int blocks) {
    constexpr int WARPS = 8, C = (D / 4 + WARPS - 1) / WARPS;         // fours of columns a warp has: w, w + 8, ..
    __shared__ __align__(16) T rows_s[32][D + 16 / sizeof(T)];
    pdl_wait();
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, s = blockIdx.z, kvh = blockIdx.y, G = a.nh / a.nkv;
    const int groups = (tile_rows + 31) / 32, tile = blockIdx.x / groups, row = blockIdx.x % groups * 32 + lane;
    TreeSeq q;
    q.load(a, s);
    if (tile >= q.tiles) return;
    int u0;
    const int total = tree_units(a, s, u0), nb = share_count(total, blocks);
    u0 += (kvh * q.tiles + tile) * q.pages;
    const int b0 = share_of(total, u0, nb), b1 = share_of(total, u0 + q.pages - 1, nb);
    if (b0 == b1) return;
    // the node of a row; -1: a row that is none, which has no parts
    auto node_of = [&](int r) {
        const int half = r / a.half_rows * a.half_nodes, in = r % a.half_rows, node = tile * a.tile_nodes + half + in / G;
        return in < a.half_nodes * G && half < a.tile_nodes && node < q.n ? node : -1;
    };
    const bool mine = node_of(row) >= 0;
    auto slot = [&](int b) { return (size_t)(2 * b + (b == b0 ? 1 : 0)) * tile_rows; };
    float m = -INFINITY, l = 0.f, acc[C][4] = {};
    if (mine)
        for (int b = b0; b <= b1; b += 2) {                            // two parts at a time
            const bool two = b < b1;
            const float2 none = make_float2(-INFINITY, 0.f), p = ws_ml[slot(b) + row], p2 = two ? ws_ml[slot(b + 1) + row] : none;
            float4 v[2][C];
#pragma unroll
            for (int c = 0; c < C; c++) {
                const int d = (c * WARPS + w) * 4;
                if (d < D) {
                    v[0][c] = *reinterpret_cast<const float4*>(ws_acc + slot(b) * D + part_at(tile_rows, row, d));
                    if (two) v[1][c] = *reinterpret_cast<const float4*>(ws_acc + slot(b + 1) * D + part_at(tile_rows, row, d));
                }
            }
            const float mn = fmaxf(m, fmaxf(p.x, p2.x)), ms = mn == -INFINITY ? 0.f : mn;
            const float old = exp2f(m - ms), f = exp2f(p.x - ms), f2 = exp2f(p2.x - ms);
            l = l * old + p.y * f + p2.y * f2;
            m = mn;
#pragma unroll
            for (int c = 0; c < C; c++) {
                const float* x = reinterpret_cast<const float*>(&v[0][c]);
                const float* x2 = reinterpret_cast<const float*>(&v[1][c]);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    acc[c][e] = acc[c][e] * old + x[e] * f;
                    if (two) acc[c][e] += x2[e] * f2;
                }
            }
        }
    const float inv = l == 0.f ? 0.f : 1.f / l;                        // no key at all: a row of zeros
#pragma unroll
    for (int c = 0; c < C; c++) {
        const int d = (c * WARPS + w) * 4;
        struct alignas(4 * sizeof(T)) Four { T x[4]; } r;
#pragma unroll
        for (int e = 0; e < 4; e++) r.x[e] = from_f<T>(acc[c][e] * inv);
        if (d < D) *reinterpret_cast<Four*>(&rows_s[lane][d]) = r;
    }
    __syncthreads();
    constexpr int PIECES = D * (int)sizeof(T) / 16, PER = 16 / (int)sizeof(T);     // 16 bytes a thread, the pieces of a row side by side
    for (int i = threadIdx.x; i < 32 * PIECES; i += 256) {
        const int k = i / PIECES, c = i % PIECES * PER, r = row - lane + k, node = node_of(r);
        if (node >= 0)
            *reinterpret_cast<uint4*>(out + (size_t)(q.flat0 + node) * ldo + (kvh * G + r % a.half_rows % G) * D + c) =
                *reinterpret_cast<const uint4*>(&rows_s[k][c]);
    }
}

// Launch of the merge, behind the kernel that leaves the parts (it may start under that one's end: it reads nothing before).
template <typename T, int D>
static int tree_merge(const TreeArgs& a, const float* ws_acc, const float* ws_ml, void* out, long long ldo, int tile_rows, int max_nodes,
                      int blocks, cudaStream_t st) {
    const int tiles = (max_nodes + a.tile_nodes - 1) / a.tile_nodes;
    return dk_launch_as(true, tree_merge_kernel<T, D>, dim3((tile_rows + 31) / 32 * tiles, a.nkv, a.n_seq), dim3(256), 0, st, a, ws_acc,
                        (const float2*)ws_ml, (T*)out, ldo, tile_rows, blocks);
}

// Whether the largest launch of these sizes has fewer than 2^31 units.
static inline bool tree_units_fit(const TreeArgs& a, int max_nodes) {
    return (double)a.n_seq * ((max_nodes + a.tile_nodes - 1) / a.tile_nodes) * a.nkv * a.pt_stride < 2147483647.0;
}
