// Attention of trees of drafted tokens over the paged cache on the CUDA cores, float32 arithmetic, for float32 or bfloat16 storage.
// Built per head size with -DHD=<multiple of 16, at most 256>. Which keys a node sees and how the work is dealt out:
// attention_tree.cuh.
//
//   out[i, h] = sum_j w_j v_j / sum_j w_j,  w_j = exp2(scale * log2(e) * q[i, h].k_j - m),  j over the keys node i sees
//
// with the running maximum m and both sums in float32, one pass over the keys. A node that sees no key gives zeros. What lies at a
// key that a row does not see, be it NaN or infinite, does not reach the row. An infinite value that it does see gives NaN where its
// weight has become 0 in float32.
//
// What bounds a page step is what shared memory returns to registers, 128 bytes a clock: a thread with 4 rows reads 8 x 16 bytes for 64
// products of the scores and 12 for 128 of the values, 14,300 clocks (7.4 us of an SM) for 64 rows of 128 columns against 8,200 of
// products. Hence the tiles by rows (see Share): 16 rows 2.9 us instead of 5.4. Measured in float32, 32 heads on 8 of 128: four trees of
// 3 to 16 nodes, 300 to 1,500 tokens, a window of 1,024: 48.7 us (12 us of products at 72 TFLOP/s, 5.2 us of bytes); four trees of 4 behind
// 4,400 tokens 62 us (22 us of bytes). With keys and values asked for at the start of their own page step instead of a half step before
// it: 54.5 us in the first case.
#include "attention_tree.cuh"

#ifndef HD
#error "compile with -DHD=<head size>"
#endif
static_assert(HD % 16 == 0 && HD >= 16 && HD <= 256, "head size must be a multiple of 16 up to 256");

namespace {

constexpr int WHOLE_PAGES = 1;                    // tables up to here are not split (see attention_tree.cuh)
constexpr int THREADS = 256, LDQ = HD + 4, LDK = HD + 4;
constexpr int PK = DK_PAGE / 2, LDP = PK + 16;     // weights of half a page at a time: with all of it two blocks of 64 rows of 128 would not fit an SM
// columns of a row: in groups of VEC side by side, a group every 16 * VEC
constexpr int VEC = HD % 64 == 0 ? 4 : HD % 32 == 0 ? 2 : 1, CV = HD / (16 * VEC);

__device__ __forceinline__ void load4(float* dst, const float* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void load4(float* dst, const bf16* src) {
    const uint2 v = *reinterpret_cast<const uint2*>(src);
    const __nv_bfloat162 *a = reinterpret_cast<const __nv_bfloat162*>(&v.x), *b = reinterpret_cast<const __nv_bfloat162*>(&v.y);
    *reinterpret_cast<float4*>(dst) = make_float4(__low2float(*a), __high2float(*a), __low2float(*b), __high2float(*b));
}
__device__ __forceinline__ void copies_end() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void copied() { asm volatile("cp.async.wait_group 0;" ::: "memory"); }

// How a block's 16 half-warps share a page: with more than 32 rows in the tile a half-warp h has rows h + 16 i (i < 4), with all columns and
// all keys. With up to 32 (16) rows a warp w has rows 4 w + i (2 w + i, i < 2), its halves take half the columns of the scores, whose sums they
// exchange, and half the keys of the values, whose sums are added up at the tile's end: what bounds the page step is what shared memory
// returns to registers (128 bytes a clock), and a thread with four (two) rows reads each key and value for all of them. (With rows h +
// 16 i throughout a page of 16 rows of 128 columns took 5.4 us of an SM, of 64 rows 7.4.)
template <int R, bool SPLIT>
struct Share {
    static __device__ __forceinline__ int half() { return threadIdx.x >> 4 & 1; }
    static __device__ __forceinline__ int row(int i) { return SPLIT ? (threadIdx.x >> 5) * R + i : (threadIdx.x >> 4) + 16 * i; }
    // where the weights of the row that the half-warp reads lie
    static __device__ __forceinline__ int p_row(int i) { return SPLIT ? 2 * row(i) + half() : row(i); }
};

// The thread's rows against one page's keys: keys tx + 16 j, each score a sum over even and one over odd columns, side by side.
template <int R, bool SPLIT>
__device__ __forceinline__ void scores(const float* q_s, const float* k_s, float (&sc)[R][4]) {
    typedef Share<R, SPLIT> S;
    const int tx = threadIdx.x & 15, d0 = SPLIT ? S::half() * (HD / 2) : 0;
    float2 s2[R][4] = {};
#pragma unroll 2
    for (int dd = 0; dd < (SPLIT ? HD / 2 : HD); dd += 4) {
        const int d = d0 + dd;
        float4 qa[R], kb[4];
#pragma unroll
        for (int i = 0; i < R; i++) qa[i] = *reinterpret_cast<const float4*>(q_s + S::row(i) * LDQ + d);
#pragma unroll
        for (int j = 0; j < 4; j++) kb[j] = *reinterpret_cast<const float4*>(k_s + (tx + 16 * j) * LDK + d);
#pragma unroll
        for (int i = 0; i < R; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                s2[i][j] = fma2(make_float2(qa[i].x, qa[i].y), make_float2(kb[j].x, kb[j].y), s2[i][j]);
                s2[i][j] = fma2(make_float2(qa[i].z, qa[i].w), make_float2(kb[j].z, kb[j].w), s2[i][j]);
            }
    }
#pragma unroll
    for (int i = 0; i < R; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            sc[i][j] = s2[i][j].x + s2[i][j].y;
            if (SPLIT) sc[i][j] += __shfl_xor_sync(0xffffffffu, sc[i][j], 16);
        }
}

// The same rows' weights and the page's values into the running results: thread tx has VEC columns from VEC * tx + 16 VEC c on. The
// weights go through memory of the row's 16 threads (32 with SPLIT), which sit in one warp. odd: a value that is not finite lies in a page
// that some row does not see all of, and reaches the rows that see it only.
template <int R, bool SPLIT>
__device__ __forceinline__ void weigh(float (&wt)[R][4], const float* v_s, float* p_s, const uint64_t* mask_s, float sl2, bool odd,
                                      float (&m)[R], float (&l)[R], float (&acc)[R][CV * VEC]) {
    typedef Share<R, SPLIT> S;
    const int tx = threadIdx.x & 15;
#pragma unroll
    for (int i = 0; i < R; i++) {
        const uint64_t seen = mask_s[S::row(i)];
        float mx = -INFINITY;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if (!(seen >> (tx + 16 * j) & 1)) wt[i][j] = -INFINITY;
            mx = fmaxf(mx, wt[i][j]);
        }
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        const float mn = fmaxf(m[i], mx * sl2), ms = mn == -INFINITY ? 0.f : mn, alpha = exp2f(m[i] - ms);
        m[i] = mn;
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            wt[i][j] = exp2f(fmaf(wt[i][j], sl2, -ms));
            sum += wt[i][j];
        }
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        l[i] = l[i] * alpha + sum;
#pragma unroll
        for (int c = 0; c < CV * VEC; c++) acc[i][c] *= alpha;
    }
    struct alignas(4 * VEC) Group { float x[VEC]; };
#pragma unroll
    for (int turn = 0; turn < (SPLIT ? 1 : 2); turn++) {               // half a page of keys a turn, or a half-warp
        const int half = SPLIT ? S::half() : turn;
        __syncwarp();
#pragma unroll
        for (int i = 0; i < R; i++)
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const float first = wt[i][j], second = wt[i][2 + j];
                p_s[S::p_row(i) * LDP + tx + 16 * j] = half ? second : first;
            }
        __syncwarp();
        const float* v_h = v_s + half * PK * HD;
        if (!odd) {
#pragma unroll 2
            for (int k = 0; k < PK; k += 4) {
                float4 w4[R];
#pragma unroll
                for (int i = 0; i < R; i++) w4[i] = *reinterpret_cast<const float4*>(p_s + S::p_row(i) * LDP + k);
#pragma unroll
                for (int e = 0; e < 4; e++) {
#pragma unroll
                    for (int c = 0; c < CV; c++) {
                        const Group v = *reinterpret_cast<const Group*>(v_h + (k + e) * HD + (c * 16 + tx) * VEC);
#pragma unroll
                        for (int i = 0; i < R; i++) {
                            const float w = reinterpret_cast<const float*>(&w4[i])[e];
                            float* a = acc[i] + c * VEC;
                            if (VEC == 1) a[0] = fmaf(w, v.x[0], a[0]);
                            else
#pragma unroll
                                for (int u = 0; u + 1 < VEC; u += 2) {
                                    const float2 r = fma2(make_float2(w, w), make_float2(v.x[u], v.x[u + 1]), make_float2(a[u], a[u + 1]));
                                    a[u] = r.x, a[u + 1] = r.y;
                                }
                        }
                    }
                }
            }
        } else {
#pragma unroll 1
            for (int k = 0; k < PK; k++)
#pragma unroll
                for (int i = 0; i < R; i++)
                    if (mask_s[S::row(i)] >> (half * PK + k) & 1) {
                        const float w = p_s[S::p_row(i) * LDP + k];
#pragma unroll
                        for (int c = 0; c < CV; c++)
#pragma unroll
                            for (int u = 0; u < VEC; u++) acc[i][c * VEC + u] = fmaf(w, v_h[k * HD + (c * 16 + tx) * VEC + u], acc[i][c * VEC + u]);
                    }
        }
    }
}

// weights: half a page of 64 rows, or a page of up to 32
template <int NI> constexpr int P_FLOATS = (NI < 4 ? 32 * NI : 64) * LDP;
template <int NI>
constexpr size_t tree_smem() {
    return sizeof(float) * (16 * NI * LDQ + P_FLOATS<NI> + DK_PAGE * (LDK + HD)) + 2 * 16 * NI * sizeof(uint64_t);
}

template <int NI>
struct Block {                                     // a block's shared memory
    float *q, *k, *v, *p;
    uint64_t* masks;                               // [page & 1][row]
    __device__ __forceinline__ Block(float* smem) {
        q = smem, k = q + 16 * NI * LDQ, v = k + DK_PAGE * LDK, p = v + DK_PAGE * HD;
        masks = reinterpret_cast<uint64_t*>(p + P_FLOATS<NI>);
    }
};

// The pages of a tile that are the block's, and its rows or their part. turn: pages before.
template <int R, bool SPLIT, int NI, typename T>
__device__ __forceinline__ void run_tile(const TreeArgs& a, const TreeWalk& w, const Block<NI>& s, uint32_t& turn, const T* q, long long ldq, T* out,
                                         long long ldo, const T* k_store, const T* v_store, float* ws_acc, float2* ws_ml) {
    constexpr int TM = 16 * NI;
    typedef Share<R, SPLIT> S;
    const TreeSeq& sq = w.sq;
    const int tx = threadIdx.x & 15, G = a.nh / a.nkv, kvh = w.kvh, rows = w.nodes * G, flat0 = sq.flat0 + w.node0, open_lo = open_from(a, sq);
    auto held = [&](int page) { return page >= 0 && page < a.n_pages; };                 // a page that is none holds no keys
    auto load = [&](float* dst, int ld, const T* store, int page) {
        const T* src = store + kv_offset(held(page) ? page : 0, a.nkv, kvh, 0, HD);
        for (int i = threadIdx.x; i < DK_PAGE * (HD / 4); i += THREADS) load4(dst + i / (HD / 4) * ld + (i % (HD / 4)) * 4, src + (size_t)i * 4);
        copies_end();
    };
    const int pos = threadIdx.x < rows ? a.row_pos[flat0 + threadIdx.x / G] : -1;       // of row `thread`, whose masks the thread works out
    // -> whether there is a row that does not see all of page p
    auto mask = [&](int p, int page) {
        if (threadIdx.x >= TM) return false;
        const int key0 = (sq.first_page + p) * DK_PAGE;
        const bool open = key0 + DK_PAGE <= sq.pos0 && key0 >= open_lo;
        uint64_t seen = 0;
        if (pos >= 0 && held(page)) seen = open ? ~0ull : tree_mask(a, sq, a.tree + (size_t)(flat0 + threadIdx.x / G) * a.words, pos, key0);
        s.masks[(turn & 1) * TM + threadIdx.x] = seen;
        return threadIdx.x < rows && seen != ~0ull;
    };
    int page = w.pt[w.p0];
    for (int i = threadIdx.x; i < TM * (HD / 4); i += THREADS) {
        const int r = i / (HD / 4), c = (i % (HD / 4)) * 4;
        if (r < rows) load4(s.q + r * LDQ + c, q + (size_t)(flat0 + r / G) * ldq + (kvh * G + r % G) * HD + c);
        else *reinterpret_cast<float4*>(s.q + r * LDQ + c) = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    load(s.k, LDK, k_store, page);
    bool masked = mask(w.p0, page);
    float m[R], l[R], acc[R][CV * VEC];
#pragma unroll
    for (int i = 0; i < R; i++) {
        m[i] = -INFINITY, l[i] = 0.f;
#pragma unroll
        for (int c = 0; c < CV * VEC; c++) acc[i][c] = 0.f;
    }
    for (int p = w.p0; p < w.p1; p++) {
        copied();
        masked = __syncthreads_or(masked);                              // the keys are here, nobody reads the page before's values
        load(s.v, HD, v_store, page);
        const uint64_t* mask_s = s.masks + (turn++ & 1) * TM;
        page = p + 1 < w.p1 ? w.pt[p + 1] : -1;
        float sc[R][4];
        scores<R, SPLIT>(s.q, s.k, sc);
        copied();
        __syncthreads();                                                // the values are here, nobody reads the keys
        bool masked_next = false, odd = false;
        if (p + 1 < w.p1) {
            load(s.k, LDK, k_store, page);
            masked_next = mask(p + 1, page);
        }
        if (masked) {
            for (int i = threadIdx.x; i < DK_PAGE * HD; i += THREADS) odd |= !isfinite(s.v[i]);
            odd = __syncthreads_or(odd);
        }
        weigh<R, SPLIT>(sc, s.v, s.p, mask_s, a.sl2, odd, m, l, acc);
        masked = masked_next;
    }
    if (SPLIT)
#pragma unroll
        for (int i = 0; i < R; i++)
#pragma unroll
            for (int c = 0; c < CV * VEC; c++) acc[i][c] += __shfl_xor_sync(0xffffffffu, acc[i][c], 16);
    if (SPLIT && S::half()) return;                                     // both halves have the sums
    const bool whole = w.all();
    const size_t slot = (size_t)w.slot() * TM;
#pragma unroll
    for (int i = 0; i < R; i++) {
        const int r = S::row(i);
        if (r >= rows) continue;
        const float inv = l[i] == 0.f ? 0.f : 1.f / l[i];
        T* dst = out + (size_t)(flat0 + r / G) * ldo + (kvh * G + r % G) * HD;
        if (!whole && tx == 0) ws_ml[slot + r] = make_float2(m[i], l[i]);
#pragma unroll
        for (int c = 0; c < CV; c++) {
            const int d = (c * 16 + tx) * VEC;
            struct alignas(4 * VEC) Part { float x[VEC]; } part;
            struct alignas(sizeof(T) * VEC) Group { T x[VEC]; } group;
#pragma unroll
            for (int u = 0; u < VEC; u++) part.x[u] = acc[i][c * VEC + u], group.x[u] = from_f<T>(part.x[u] * inv);
            if (whole) *reinterpret_cast<Group*>(dst + d) = group;
            else *reinterpret_cast<Part*>(ws_acc + slot * HD + part_at(TM, r, d)) = part;
        }
    }
}

// 256 threads, two blocks an SM where their shared memory allows it (64 rows of 128 columns: 111 KB). Keys and values have one buffer each:
// a page's keys come in under the weights and values of the page before, its values under its own scores.
template <typename T, int NI>
__global__ void __launch_bounds__(THREADS, tree_smem<NI>() <= 113 * 1024 ? 2 : 1)
tree_kernel(TreeArgs a, const T* q, long long ldq, T* out, long long ldo, const T* k_store, const T* v_store, float* ws_acc, float2* ws_ml) {
    extern __shared__ __align__(16) float smem[];
    const Block<NI> s(smem);
    pdl_wait();
    pdl_launch_dependents();
    TreeWalk w;
    w.begin(a);
    uint32_t turn = 0;
    while (w.next(a)) {
        const int rows = w.nodes * (a.nh / a.nkv);
#define DK_RUN(R, SPLIT) run_tile<R, SPLIT, NI, T>(a, w, s, turn, q, ldq, out, ldo, k_store, v_store, ws_acc, ws_ml)
        if (NI == 1 || rows <= 16) DK_RUN(2, true);
        else if (NI == 2 || rows <= 32) DK_RUN(4, true);
        else DK_RUN(4, false);
#undef DK_RUN
    }
}

template <typename T, int NI>
int launch(const TreeArgs& a, const void* q, long long ldq, void* out, long long ldo, const void* k_store, const void* v_store, float* ws_acc,
           float* ws_ml, int blocks, cudaStream_t st) {
    static SmemOnce once;
    int r = once.allow((const void*)tree_kernel<T, NI>, tree_smem<NI>());
    if (r) return r;
    r = dk_launch(tree_kernel<T, NI>, dim3(blocks), dim3(THREADS), tree_smem<NI>(), st, a, (const T*)q, ldq, (T*)out, ldo,
                      (const T*)k_store, (const T*)v_store, ws_acc, (float2*)ws_ml);
    if (r) return r;
    return tree_merge<T, HD>(a, ws_acc, ws_ml, out, ldo, 16 * NI, blocks, st);
}

}  // namespace

// Rows a block's tile has: the smallest of 16, 32 and 64 that takes the largest tree's rows, 64 if none does.
DK_EXPORT int dk_tree_tile_rows(int max_nodes, int group) {
    const long long rows = (long long)max_nodes * group;
    return rows <= 16 ? 16 : rows <= 32 ? 32 : 64;
}

DK_EXPORT int dk_tree_whole_pages() { return WHOLE_PAGES; }

// Blocks of a launch: as many as the device holds at once.
DK_EXPORT int dk_attn_tree_blocks(int f32, int max_nodes, int group) {
    const int rows = dk_tree_tile_rows(max_nodes, group);
    int per_sm = 0, sms = 0, dev = 0;
#define DK_OCC(T, NI) \
    (cudaFuncSetAttribute(tree_kernel<T, NI>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)tree_smem<NI>()), \
     cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, tree_kernel<T, NI>, THREADS, tree_smem<NI>()))
    if (f32) rows == 16 ? DK_OCC(float, 1) : rows == 32 ? DK_OCC(float, 2) : DK_OCC(float, 4);
    else rows == 16 ? DK_OCC(bf16, 1) : rows == 32 ? DK_OCC(bf16, 2) : DK_OCC(bf16, 4);
#undef DK_OCC
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    return (per_sm > 0 ? per_sm : 1) * sms;
}

// q [rows, nh*HD] and out [rows, nh*HD], rows ldq / ldo elements apart; k_store, v_store [n_pages, nkv, 64, HD]; all on 16-byte
// boundaries, q's and out's rows too: what is read and written is 16 bytes (bfloat16: 8) at a time. ws_acc: 2 * blocks * tile rows * HD floats, ws_ml: 2 * blocks * tile rows * 2 floats. f32 != 0: float32 storage, else bfloat16.
DK_EXPORT int dk_attn_tree(int f32, const void* q, long long ldq, void* out, long long ldo, const void* k_store, const void* v_store,
                           int n_pages, const int* cu_q, const int* seq_pos0, const int* row_pos, const uint32_t* tree, int words,
                           const int* page_table, int pt_stride, int n_seq, int nh, int nkv, int window, float scale, int max_nodes,
                           float* ws_acc, float* ws_ml, int blocks, cudaStream_t st) {
    const int size = f32 ? 4 : 2;
    if (nkv < 1 || nh % nkv || nh / nkv > 64 || n_pages < 1 || pt_stride < 1 || words < 1 || blocks < 1 || max_nodes < 1 || n_seq > 65535 ||
        ldq * size % 16 || ldo * size % 16 || ((uintptr_t)q | (uintptr_t)out | (uintptr_t)k_store | (uintptr_t)v_store) % 16)
        return (int)cudaErrorInvalidValue;
    const int G = nh / nkv, rows = dk_tree_tile_rows(max_nodes, G);
    TreeArgs a = {cu_q, seq_pos0, row_pos, page_table, tree, n_seq, words, pt_stride, n_pages, nh, nkv, window, max_nodes, rows / G, rows / G, rows,
                  pt_stride <= WHOLE_PAGES, 0, scale * 1.4426950408889634f};
    if (!tree_units_fit(a) || nkv > 65535 || (!a.whole && (ws_acc == nullptr || ws_ml == nullptr))) return (int)cudaErrorInvalidValue;
#define DK_TREE(T, NI) launch<T, NI>(a, q, ldq, out, ldo, k_store, v_store, ws_acc, ws_ml, blocks, st)
    if (f32) return rows == 16 ? DK_TREE(float, 1) : rows == 32 ? DK_TREE(float, 2) : DK_TREE(float, 4);
    return rows == 16 ? DK_TREE(bf16, 1) : rows == 32 ? DK_TREE(bf16, 2) : DK_TREE(bf16, 4);
#undef DK_TREE
}
