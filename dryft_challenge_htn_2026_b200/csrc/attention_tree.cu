// Attention of trees of drafted tokens over the paged cache on the CUDA cores, float32 arithmetic, for float32 or bfloat16 storage.
// Built per head size with -DHD=<multiple of 16, at most 256>. Which keys a node sees and how the work is dealt out:
// attention_tree.cuh.
//
//   out[i, h] = sum_j w_j v_j / sum_j w_j,  w_j = exp2(scale * log2(e) * q[i, h].k_j - m),  j over the keys node i sees
//
// with the running maximum m and both sums in float32, one pass over the keys. A node that sees no key gives zeros. What lies at a
// key that a row does not see, be it NaN or infinite, does not reach the row.
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

// Rows ty + 16 i (i < N) of a tile against one page's keys. Thread (ty, tx) of 16 x 16 has keys tx + 16 j: each score a sum over even and
// one over odd columns, side by side.
template <int N, int NI>
__device__ __forceinline__ void scores(const float* q_s, const float* k_s, float2 (&s2)[NI][4]) {
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
#pragma unroll
    for (int i = 0; i < N; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) s2[i][j] = make_float2(0.f, 0.f);
#pragma unroll 4
    for (int d = 0; d < HD; d += 4) {
        float4 qa[N], kb[4];
#pragma unroll
        for (int i = 0; i < N; i++) qa[i] = *reinterpret_cast<const float4*>(q_s + (ty + 16 * i) * LDQ + d);
#pragma unroll
        for (int j = 0; j < 4; j++) kb[j] = *reinterpret_cast<const float4*>(k_s + (tx + 16 * j) * LDK + d);
#pragma unroll
        for (int i = 0; i < N; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                s2[i][j] = fma2(make_float2(qa[i].x, qa[i].y), make_float2(kb[j].x, kb[j].y), s2[i][j]);
                s2[i][j] = fma2(make_float2(qa[i].z, qa[i].w), make_float2(kb[j].z, kb[j].w), s2[i][j]);
            }
    }
}

// The same rows' weights and the page's values into the running results: thread (ty, tx) has VEC columns from VEC * tx + 16 VEC c on. The
// weights go through memory of the row's 16 threads, which sit in one warp. odd: a value that is not finite lies in a page that some row
// does not see all of, and reaches the rows that see it only.
template <int N, int NI>
__device__ __forceinline__ void weigh(const float2 (&s2)[NI][4], const float* v_s, float* p_s, const uint64_t* mask_s, float sl2, bool odd,
                                      float (&m)[NI], float (&l)[NI], float (&acc)[NI][CV * VEC]) {
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    float wt[N][4];
#pragma unroll
    for (int i = 0; i < N; i++) {
        const uint64_t seen = mask_s[ty + 16 * i];
        float mx = -INFINITY;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            wt[i][j] = seen >> (tx + 16 * j) & 1 ? s2[i][j].x + s2[i][j].y : -INFINITY;
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
    for (int half = 0; half < 2; half++) {
        __syncwarp();
#pragma unroll
        for (int i = 0; i < N; i++)
#pragma unroll
            for (int j = 0; j < 2; j++) p_s[(ty + 16 * i) * LDP + tx + 16 * j] = wt[i][2 * half + j];
        __syncwarp();
        const float* v_h = v_s + half * PK * HD;
        if (!odd) {
#pragma unroll 2
            for (int k = 0; k < PK; k += 4) {
                float4 w4[N];
#pragma unroll
                for (int i = 0; i < N; i++) w4[i] = *reinterpret_cast<const float4*>(p_s + (ty + 16 * i) * LDP + k);
#pragma unroll
                for (int e = 0; e < 4; e++) {
#pragma unroll
                    for (int c = 0; c < CV; c++) {
                        const Group v = *reinterpret_cast<const Group*>(v_h + (k + e) * HD + (c * 16 + tx) * VEC);
#pragma unroll
                        for (int i = 0; i < N; i++) {
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
                for (int i = 0; i < N; i++)
                    if (mask_s[ty + 16 * i] >> (half * PK + k) & 1) {
                        const float w = p_s[(ty + 16 * i) * LDP + k];
#pragma unroll
                        for (int c = 0; c < CV; c++)
#pragma unroll
                            for (int u = 0; u < VEC; u++) acc[i][c * VEC + u] = fmaf(w, v_h[k * HD + (c * 16 + tx) * VEC + u], acc[i][c * VEC + u]);
                    }
        }
    }
}

template <int NI>
constexpr size_t tree_smem() {
    return sizeof(float) * (16 * NI * (LDQ + LDP) + DK_PAGE * (LDK + HD)) + 2 * 16 * NI * sizeof(uint64_t);
}

// 256 threads, two blocks an SM where their shared memory allows it (64 rows of 128 columns: 111 KB). Keys and values have one buffer each:
// a page's keys come in under the weights and values of the page before, its values under its own scores.
template <typename T, int NI>
__global__ void __launch_bounds__(THREADS, tree_smem<NI>() <= 113 * 1024 ? 2 : 1)
tree_kernel(TreeArgs a, const T* q, long long ldq, T* out, long long ldo, const T* k_store, const T* v_store, float* ws_acc, float2* ws_ml) {
    constexpr int TM = 16 * NI;
    extern __shared__ __align__(16) float smem[];
    float *q_s = smem, *k_s = q_s + TM * LDQ, *v_s = k_s + DK_PAGE * LDK, *p_s = v_s + DK_PAGE * HD;
    uint64_t* masks = reinterpret_cast<uint64_t*>(p_s + TM * LDP);      // [page & 1][row]
    pdl_wait();
    pdl_launch_dependents();
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4, G = a.nh / a.nkv;
    TreeWalk w;
    w.begin(a);
    const TreeSeq& sq = w.sq;
    uint32_t turn = 0;                                                  // pages before
    while (w.next(a)) {
        const int p0 = w.p0, p1 = w.p1, kvh = w.kvh, rows = w.nodes * G, flat0 = sq.flat0 + w.node0, open_lo = open_from(a, sq);
        const int* pt = w.pt;
        auto held = [&](int page) { return page >= 0 && page < a.n_pages; };             // a page that is none holds no keys
        auto load = [&](float* dst, int ld, const T* store, int page) {
            const T* src = store + kv_offset(held(page) ? page : 0, a.nkv, kvh, 0, HD);
            for (int i = threadIdx.x; i < DK_PAGE * (HD / 4); i += THREADS) load4(dst + i / (HD / 4) * ld + (i % (HD / 4)) * 4, src + (size_t)i * 4);
            copies_end();
        };
        const int pos = threadIdx.x < rows ? a.row_pos[flat0 + threadIdx.x / G] : -1;   // of row `thread`, whose masks the thread works out
        // -> whether there is a row that does not see all of page p
        auto mask = [&](int p, int page) {
            if (threadIdx.x >= TM) return false;
            const int key0 = (sq.first_page + p) * DK_PAGE;
            const bool open = key0 + DK_PAGE <= sq.pos0 && key0 >= open_lo;
            uint64_t seen = 0;
            if (pos >= 0 && held(page)) seen = open ? ~0ull : tree_mask(a, sq, a.tree + (size_t)(flat0 + threadIdx.x / G) * a.words, pos, key0);
            masks[(turn & 1) * TM + threadIdx.x] = seen;
            return threadIdx.x < rows && seen != ~0ull;
        };
        int page = pt[p0];
        for (int i = threadIdx.x; i < TM * (HD / 4); i += THREADS) {
            const int r = i / (HD / 4), c = (i % (HD / 4)) * 4;
            if (r < rows) load4(q_s + r * LDQ + c, q + (size_t)(flat0 + r / G) * ldq + (kvh * G + r % G) * HD + c);
            else *reinterpret_cast<float4*>(q_s + r * LDQ + c) = make_float4(0.f, 0.f, 0.f, 0.f);
        }
        load(k_s, LDK, k_store, page);
        bool masked = mask(p0, page);
        float m[NI], l[NI], acc[NI][CV * VEC];
#pragma unroll
        for (int i = 0; i < NI; i++) {
            m[i] = -INFINITY, l[i] = 0.f;
#pragma unroll
            for (int c = 0; c < CV * VEC; c++) acc[i][c] = 0.f;
        }
        for (int p = p0; p < p1; p++) {
            copied();
            masked = __syncthreads_or(masked);                          // the keys are here, nobody reads the page before's values
            load(v_s, HD, v_store, page);
            const uint64_t* mask_s = masks + (turn++ & 1) * TM;
            page = p + 1 < p1 ? pt[p + 1] : -1;
            float2 s2[NI][4];
            if (NI >= 4 && rows > 32) scores<NI, NI>(q_s, k_s, s2);
            else if (NI >= 2 && rows > 16) scores<(NI < 2 ? NI : 2), NI>(q_s, k_s, s2);
            else scores<1, NI>(q_s, k_s, s2);
            copied();
            __syncthreads();                                            // the values are here, nobody reads the keys
            bool masked_next = false, odd = false;
            if (p + 1 < p1) {
                load(k_s, LDK, k_store, page);
                masked_next = mask(p + 1, page);
            }
            if (masked) {
                for (int i = threadIdx.x; i < DK_PAGE * HD; i += THREADS) odd |= !isfinite(v_s[i]);
                odd = __syncthreads_or(odd);
            }
            if (NI >= 4 && rows > 32) weigh<NI, NI>(s2, v_s, p_s, mask_s, a.sl2, odd, m, l, acc);
            else if (NI >= 2 && rows > 16) weigh<(NI < 2 ? NI : 2), NI>(s2, v_s, p_s, mask_s, a.sl2, odd, m, l, acc);
            else weigh<1, NI>(s2, v_s, p_s, mask_s, a.sl2, odd, m, l, acc);
            masked = masked_next;
        }
        const bool whole = w.all();
        const size_t slot = (size_t)w.slot() * TM;
#pragma unroll
        for (int i = 0; i < NI; i++) {
            const int r = ty + 16 * i;
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

// q [rows, nh*HD] and out [rows, nh*HD], rows ldq / ldo elements apart; k_store, v_store [n_pages, nkv, 64, HD]; ws_acc: 2 * blocks *
// tile rows * HD floats, ws_ml: 2 * blocks * tile rows * 2 floats. f32 != 0: float32 storage, else bfloat16.
DK_EXPORT int dk_attn_tree(int f32, const void* q, long long ldq, void* out, long long ldo, const void* k_store, const void* v_store,
                           int n_pages, const int* cu_q, const int* seq_pos0, const int* row_pos, const uint32_t* tree, int words,
                           const int* page_table, int pt_stride, int n_seq, int nh, int nkv, int window, float scale, int max_nodes,
                           float* ws_acc, float* ws_ml, int blocks, cudaStream_t st) {
    if (nkv < 1 || nh % nkv || nh / nkv > 64 || n_pages < 1 || pt_stride < 1 || words < 1 || blocks < 1 || max_nodes < 1 || n_seq > 65535)
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
