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
// slots: 2 b + 1 for the tile whose first page it has, 2 b for one that began in an earlier block. Taking up a tile and writing its
// rows costs a block as much as some pages do: `extra` units that stand before a tile's pages and ask for no work.
// With tables of a few pages (`whole`) a tile is one unit: there are no parts and there is no merge.
#pragma once
#include "common.cuh"

// two numbers at a time: a * b + c, a + b
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{ .reg .b64 x, y, z; mov.b64 x, {%2, %3}; mov.b64 y, {%4, %5}; mov.b64 z, {%6, %7}; fma.rn.f32x2 x, x, y, z; mov.b64 {%0, %1}, x; }"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{ .reg .b64 x, y; mov.b64 x, {%2, %3}; mov.b64 y, {%4, %5}; add.rn.f32x2 x, x, y; mov.b64 {%0, %1}, x; }"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}

struct TreeArgs {
    const int *cu_q, *seq_pos0, *row_pos, *page_table;
    const uint32_t* tree;                  // [rows, words]
    int n_seq, words, pt_stride, n_pages, nh, nkv, window, max_nodes, tile_nodes, half_nodes, half_rows, whole, extra;
    float sl2;                             // scale * log2(e)
};

// One sequence as the work is counted.
struct TreeSeq {
    int n, pos0, first_page, pages, tiles, flat0;
    __device__ __forceinline__ void load(const TreeArgs& a, int s) {
        flat0 = a.cu_q[s];
        n = min(max(0, a.cu_q[s + 1] - flat0), a.max_nodes);
        pos0 = max(0, a.seq_pos0[s]);
        tiles = (n + a.tile_nodes - 1) / a.tile_nodes;
        // pages that the table has no column for hold no keys; one page at least, so that rows without a key are written too
        const int end = min((pos0 + n + DK_PAGE - 1) / DK_PAGE, a.pt_stride);
        first_page = min((a.window > 0 ? max(0, pos0 - a.window + 1) : 0) / DK_PAGE, a.pt_stride - 1);
        pages = max(1, end - first_page);
    }
    __device__ __forceinline__ int length(const TreeArgs& a) const { return a.whole ? 1 : pages + a.extra; }      // units of a tile
    __device__ __forceinline__ int units(const TreeArgs& a) const { return tiles * a.nkv * length(a); }
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

// The run of units as a warp sees it: the total, and sequence by sequence where it begins. Up to 32 sequences are read once and kept,
// one a lane; more are read again where they are asked for. A whole warp calls all of this.
struct TreeRun {
    TreeSeq mine;                          // of sequence `lane`
    int upto, total;                       // units of the sequences up to and including `lane`'s; of all
    __device__ __forceinline__ int load(const TreeArgs& a, int s0) {
        const int s = s0 + (threadIdx.x & 31);
        if (s < a.n_seq) mine.load(a, s);
        else mine.tiles = 0, mine.pages = 0;
        upto = warp_scan(mine.units(a));
        return __shfl_sync(0xffffffffu, upto, 31);
    }
    __device__ __forceinline__ void read(const TreeArgs& a) {
        total = 0;
        for (int s0 = 0; s0 < a.n_seq; s0 += 32) total += load(a, s0);
    }
    __device__ __forceinline__ TreeSeq seq_of_lane(int l) const {
        TreeSeq q;
        q.n = __shfl_sync(0xffffffffu, mine.n, l), q.pos0 = __shfl_sync(0xffffffffu, mine.pos0, l);
        q.first_page = __shfl_sync(0xffffffffu, mine.first_page, l), q.pages = __shfl_sync(0xffffffffu, mine.pages, l);
        q.tiles = __shfl_sync(0xffffffffu, mine.tiles, l), q.flat0 = __shfl_sync(0xffffffffu, mine.flat0, l);
        return q;
    }
    // The sequence that unit u (below the total) belongs to, and the units before it.
    __device__ __forceinline__ TreeSeq find(const TreeArgs& a, int u, int& s, int& before) {
        before = 0;
        for (int s0 = 0;; s0 += 32) {
            const int here = a.n_seq <= 32 ? total : load(a, s0);
            if (before + here > u || s0 + 32 >= a.n_seq) {
                const int l = __ffs(__ballot_sync(0xffffffffu, before + upto > u)) - 1;
                before += __shfl_sync(0xffffffffu, upto - mine.units(a), l);
                s = s0 + l;
                return seq_of_lane(l);
            }
            before += here;
        }
    }
    // Sequence s, and the units before it.
    __device__ __forceinline__ TreeSeq at(const TreeArgs& a, int s, int& before) {
        before = 0;
        if (a.n_seq > 32)
            for (int s0 = 0; s0 <= s; s0 += 32) {
                const int here = load(a, s0);
                if (s0 + 32 <= s) before += here;
            }
        before += __shfl_sync(0xffffffffu, upto - mine.units(a), s & 31);
        return seq_of_lane(s & 31);
    }
};

// Shares of a launch of `blocks`.
__device__ __forceinline__ int share_count(int total, int blocks) { return min(total, blocks); }
// Block b's share begins at this unit; the share that unit u lies in.
__device__ __forceinline__ int scaled(int x, int y, int by) {             // x * y / by; a 64-bit division only where it has to be
    const unsigned long long xy = (unsigned long long)x * (unsigned)y;
    return xy >> 32 ? (int)(xy / (unsigned)by) : (int)((unsigned)xy / (unsigned)by);
}
__device__ __forceinline__ int share_begin(int total, int b, int nb) { return scaled(total, b, nb); }
__device__ __forceinline__ int share_of(int total, int u, int nb) {
    const unsigned long long x = (unsigned long long)(u + 1) * (unsigned)nb - 1;
    return x >> 32 ? (int)(x / (unsigned)total) : (int)((unsigned)x / (unsigned)total);
}

// Where a block stands in its share; every role walks it for itself. A whole warp calls begin().
struct TreeWalk {
    TreeSeq sq;
    int u, u_end, before, s;
    // the tile at hand: its kv head, first node, nodes, pages [p0, p1) of the sequence's
    int kvh, node0, nodes, p0, p1;
    const int* pt;
    __device__ __forceinline__ void begin(const TreeArgs& a) {
        u = u_end = 0;
        TreeRun run;
        run.read(a);
        const int nb = share_count(run.total, gridDim.x);
        if ((int)blockIdx.x < nb) {
            u = share_begin(run.total, blockIdx.x, nb), u_end = share_begin(run.total, blockIdx.x + 1, nb);
            sq = run.find(a, u, s, before);
        }
    }
    __device__ __forceinline__ bool next(const TreeArgs& a) {
        for (;;) {
            if (u >= u_end) return false;
            while (u >= before + sq.units(a)) {
                before += sq.units(a);
                sq.load(a, ++s);
            }
            const int len = sq.length(a), at = u - before, item = at / len, v0 = at % len, v1 = min(len, v0 + u_end - u);
            u += v1 - v0;
            p0 = a.whole ? 0 : max(0, v0 - a.extra), p1 = a.whole ? sq.pages : max(0, v1 - a.extra);
            if (p0 >= p1) continue;
            kvh = item / sq.tiles, node0 = (item % sq.tiles) * a.tile_nodes;
            nodes = min(a.tile_nodes, sq.n - node0);
            pt = a.page_table + (size_t)s * a.pt_stride + sq.first_page;
            return true;
        }
    }
    __device__ __forceinline__ int pages() const { return p1 - p0; }
    __device__ __forceinline__ bool all() const { return p1 - p0 == sq.pages; }       // the tile's rows are complete here
    __device__ __forceinline__ int slot() const { return 2 * blockIdx.x + (p0 == 0 ? 1 : 0); }
};

// Where column d of row `row` of a slot lies among its tile_rows * D numbers: four columns of a row side by side, then the next row's,
// so that threads with a row each write and read whole lines.
__device__ __forceinline__ size_t part_at(int tile_rows, int row, int d) { return ((size_t)(d >> 2) * tile_rows + row) * 4 + (d & 3); }

// Bits of the places [key0, key0 + 64) that a node sees; `words`: its row of the tree's bits; `pos`: its position, < 0 for none.
// (Not inlined: the kernels are short, and code that runs once costs them more for being fetched than for being run.)
static __device__ __noinline__ uint64_t tree_mask(const TreeArgs& a, TreeSeq q, const uint32_t* words, int pos, int key0) {
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

// Pages from this place on, up to the cached tokens' end, are seen by every row: with a window, those behind where the last node's begins.
__device__ __forceinline__ int open_from(const TreeArgs& a, const TreeSeq& q) { return a.window > 0 ? max(0, q.pos0 + q.n - a.window) : 0; }

// Merges the parts of the tiles that more than one block worked on; the others have been written. Grid (row groups of the largest
// tree x column groups, nkv, n_seq), 256 threads: a block has 32 rows of a tile, lane k its k-th, and COLS columns, an eighth of them a
// warp. What four parts say of a row is asked for together, or eight where a block has 64 columns.
template <typename T, int D, int COLS>
__global__ void __launch_bounds__(256)
tree_merge_kernel(TreeArgs a, const float* ws_acc, const float2* ws_ml, T* out, long long ldo, int tile_rows, int blocks) {
    constexpr int WARPS = 8, C = (COLS / 4 + WARPS - 1) / WARPS;       // fours of columns a warp has: w, w + 8, ..
    __shared__ __align__(16) T rows_s[32][COLS + 16 / sizeof(T)];
    // which rows and parts these are hangs on what the kernel before has read as well: worked out before the wait for it
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, s = blockIdx.z, kvh = blockIdx.y, G = a.nh / a.nkv;
    const int groups = (tile_rows + 31) / 32, part = blockIdx.x / (D / COLS), d0 = blockIdx.x % (D / COLS) * COLS;
    const int tile = part / groups, row = part % groups * 32 + lane;
    TreeRun run;
    run.read(a);
    int u0;
    const TreeSeq q = run.at(a, s, u0);
    const int total = run.total, nb = share_count(total, blocks);
    // the node of a row; -1: a row that is none, which has no parts
    auto node_of = [&](int r) {
        const int half = r / a.half_rows * a.half_nodes, in = r % a.half_rows, node = tile * a.tile_nodes + half + in / G;
        return in < a.half_nodes * G && half < a.tile_nodes && node < q.n ? node : -1;
    };
    const bool mine = node_of(row) >= 0;
    u0 += (kvh * q.tiles + tile) * q.length(a);
    const int b0 = tile < q.tiles ? share_of(total, u0 + a.extra, nb) : 0, b1 = tile < q.tiles ? share_of(total, u0 + q.length(a) - 1, nb) : 0;
    pdl_wait();
    pdl_launch_dependents();
    if (b0 == b1 || !__any_sync(0xffffffffu, mine)) return;            // the same for all warps
    auto slot = [&](int b) { return (size_t)(2 * b + (b == b0 ? 1 : 0)) * tile_rows; };
    float m = -INFINITY, l = 0.f, acc[C][4] = {};
    constexpr int AT_ONCE = C <= 2 ? 8 : C <= 4 ? 4 : 2;
    if (mine)
        for (int b = b0; b <= b1; b += AT_ONCE) {
            float2 p[AT_ONCE];
            float4 v[AT_ONCE][C];
#pragma unroll
            for (int k = 0; k < AT_ONCE; k++) {
                p[k] = b + k <= b1 ? ws_ml[slot(b + k) + row] : make_float2(-INFINITY, 0.f);
#pragma unroll
                for (int c = 0; c < C; c++) {
                    const int d = (c * WARPS + w) * 4;
                    v[k][c] = d < COLS && b + k <= b1 ? *reinterpret_cast<const float4*>(ws_acc + slot(b + k) * D + part_at(tile_rows, row, d0 + d))
                                                   : make_float4(0.f, 0.f, 0.f, 0.f);
                }
            }
            float mn = m;
#pragma unroll
            for (int k = 0; k < AT_ONCE; k++) mn = fmaxf(mn, p[k].x);
            const float ms = mn == -INFINITY ? 0.f : mn, old = exp2f(m - ms);
            l *= old, m = mn;
#pragma unroll
            for (int c = 0; c < C; c++)
#pragma unroll
                for (int e = 0; e < 4; e++) acc[c][e] *= old;
#pragma unroll
            for (int k = 0; k < AT_ONCE; k++) {
                if (b + k > b1) break;
                const float f = exp2f(p[k].x - ms);
                l = fmaf(p[k].y, f, l);
#pragma unroll
                for (int c = 0; c < C; c++)
#pragma unroll
                    for (int e = 0; e < 4; e++) acc[c][e] = fmaf(reinterpret_cast<const float*>(&v[k][c])[e], f, acc[c][e]);
            }
        }
    const float inv = l == 0.f ? 0.f : 1.f / l;                        // no key at all: a row of zeros
#pragma unroll
    for (int c = 0; c < C; c++) {
        const int d = (c * WARPS + w) * 4;
        struct alignas(4 * sizeof(T)) Four { T x[4]; } r;
#pragma unroll
        for (int e = 0; e < 4; e++) r.x[e] = from_f<T>(acc[c][e] * inv);
        if (d < COLS) *reinterpret_cast<Four*>(&rows_s[lane][d]) = r;
    }
    __syncthreads();
    constexpr int PIECES = COLS * (int)sizeof(T) / 16, PER = 16 / (int)sizeof(T);     // 16 bytes a thread, the pieces of a row side by side
    for (int i = threadIdx.x; i < 32 * PIECES; i += 256) {
        const int k = i / PIECES, c = i % PIECES * PER, r = row - lane + k, node = node_of(r);
        if (node >= 0)
            *reinterpret_cast<uint4*>(out + (size_t)(q.flat0 + node) * ldo + (kvh * G + r % a.half_rows % G) * D + d0 + c) =
                *reinterpret_cast<const uint4*>(&rows_s[k][c]);
    }
}

// A kernel's permission to use more shared memory than usual, asked for once on each device.
struct SmemOnce {
    unsigned long long done[4] = {};
    int allow(const void* kernel, size_t bytes) {
        int dev = 0;
        cudaGetDevice(&dev);
        if (dev >= 0 && dev < 256 && done[dev >> 6] >> (dev & 63) & 1) return 0;
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
        if (e != cudaSuccess) return cudaGetLastError(), (int)e;
        if (dev >= 0 && dev < 256) done[dev >> 6] |= 1ull << (dev & 63);
        return 0;
    }
};

// Launch of the merge, behind the kernel that leaves the parts (it may start under that one's end: it reads nothing before).
template <typename T, int D>
static int tree_merge(const TreeArgs& a, const float* ws_acc, const float* ws_ml, void* out, long long ldo, int tile_rows, int blocks,
                      cudaStream_t st) {
    if (a.whole) return 0;
    const int tiles = (a.max_nodes + a.tile_nodes - 1) / a.tile_nodes, groups = (tile_rows + 31) / 32 * tiles;
    // Few tiles, so many parts each (six or more): the columns in halves, to have more of them on the way at once. The whole call, 32 heads on
    // 8 of 128, bfloat16, 148 blocks, all columns a block / halves: one tree of 24 behind 32,768 tokens (8 tiles) 43.7 / 40.8 us, two 61.5 / 60.5,
    // three 81.1 / 81.0, four 101.2 / 101.7; one tree of 64 behind 4,096 24.3 / 21.5, four (32 tiles) 34.0 / 36.7, eight 54.3 / 59.3. float32,
    // 296 blocks: trees of 16 behind 4,096, one (8 tiles) 52.1 / 49.7, six (48) 183.5 / 182.9, four of 40 (96) 344.3 / 345.2.
    constexpr int HALF = D % 128 == 0 ? D / 2 : D;
    if (HALF < D && 6LL * a.n_seq * tiles * a.nkv <= blocks)
        return dk_launch_as(true, tree_merge_kernel<T, D, HALF>, dim3(groups * (D / HALF), a.nkv, a.n_seq), dim3(256), 0, st, a, ws_acc,
                            (const float2*)ws_ml, (T*)out, ldo, tile_rows, blocks);
    return dk_launch_as(true, tree_merge_kernel<T, D, D>, dim3(groups, a.nkv, a.n_seq), dim3(256), 0, st, a, ws_acc, (const float2*)ws_ml,
                        (T*)out, ldo, tile_rows, blocks);
}

// Whether the largest launch of these sizes has fewer than 2^31 units.
static inline bool tree_units_fit(const TreeArgs& a) {
    return (double)a.n_seq * ((a.max_nodes + a.tile_nodes - 1) / a.tile_nodes) * a.nkv * (a.pt_stride + a.extra) < 2147483647.0;
}
