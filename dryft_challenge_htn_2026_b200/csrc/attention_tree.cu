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
constexpr int THREADS = 256, LDQ = HD + 4, LDK = HD + 4, LDP = DK_PAGE + 4;
// columns of a row: in groups of VEC side by side, a group every 16 * VEC
constexpr int VEC = HD % 64 == 0 ? 4 : HD % 32 == 0 ? 2 : 1, CV = HD / (16 * VEC);
template <int NI> constexpr int P_FLOATS = 16 * NI * LDP;
template <int NI> constexpr int K_FLOATS = DK_PAGE * LDK > P_FLOATS<NI> ? DK_PAGE * LDK : P_FLOATS<NI>;          // P goes where K was

__device__ __forceinline__ void load4(float* dst, const float* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void load4(float* dst, const bf16* src) {
    const uint2 v = *reinterpret_cast<const uint2*>(src);
    const __nv_bfloat162 *a = reinterpret_cast<const __nv_bfloat162*>(&v.x), *b = reinterpret_cast<const __nv_bfloat162*>(&v.y);
    *reinterpret_cast<float4*>(dst) = make_float4(__low2float(*a), __high2float(*a), __low2float(*b), __high2float(*b));
}
__device__ __forceinline__ void copies_end() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT> __device__ __forceinline__ void copied() { asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory"); }

// Rows ty + 16 i (i < N) of a tile against one page, whose keys and values lie in shared memory. Thread (ty, tx) of 16 x 16 has keys tx +
// 16 j for the scores (each a sum over even and one over odd columns, side by side), then VEC columns from VEC * tx + 16 VEC c on.
template <int N, int NI>
__device__ __forceinline__ void page_step(const float* q_s, const float* k_s, const float* v_s, float* p_s, const uint64_t* mask_s, float sl2,
                                          bool masked, float (&m)[NI], float (&l)[NI], float (&acc)[NI][CV * VEC]) {
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    float2 s2[N][4] = {};
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
    copied<0>();                                                        // the values
    __syncthreads();                                                    // P goes where K was
    bool odd = false;
    if (masked) {       // some row does not see all of the page: is there a value in it that is not finite?
        for (int i = threadIdx.x; i < DK_PAGE * HD; i += THREADS) odd |= !isfinite(v_s[i]);
        odd = __syncthreads_or(odd);
    }
#pragma unroll
    for (int i = 0; i < N; i++) {
        const uint64_t seen = mask_s[ty + 16 * i];
        float sc[4], mx = -INFINITY;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            sc[j] = seen >> (tx + 16 * j) & 1 ? s2[i][j].x + s2[i][j].y : -INFINITY;
            mx = fmaxf(mx, sc[j]);
        }
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        const float mn = fmaxf(m[i], mx * sl2), ms = mn == -INFINITY ? 0.f : mn, alpha = exp2f(m[i] - ms);
        m[i] = mn;
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float w = exp2f(fmaf(sc[j], sl2, -ms));
            sum += w;
            p_s[(ty + 16 * i) * LDP + tx + 16 * j] = w;
        }
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        l[i] = l[i] * alpha + sum;
#pragma unroll
        for (int c = 0; c < CV * VEC; c++) acc[i][c] *= alpha;
    }
    __syncwarp();                                                       // a row's 16 threads sit in one warp
    struct alignas(4 * VEC) Group { float x[VEC]; };
    if (!odd) {
#pragma unroll 2
        for (int k = 0; k < DK_PAGE; k += 4) {
            float4 w4[N];
#pragma unroll
            for (int i = 0; i < N; i++) w4[i] = *reinterpret_cast<const float4*>(p_s + (ty + 16 * i) * LDP + k);
#pragma unroll
            for (int e = 0; e < 4; e++) {
#pragma unroll
                for (int c = 0; c < CV; c++) {
                    const Group v = *reinterpret_cast<const Group*>(v_s + (k + e) * HD + (c * 16 + tx) * VEC);
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
    } else {                                                            // a value that is not finite reaches the rows that see it only
        for (int k = 0; k < DK_PAGE; k++)
#pragma unroll
            for (int i = 0; i < N; i++)
                if (mask_s[ty + 16 * i] >> k & 1) {
                    const float w = p_s[(ty + 16 * i) * LDP + k];
#pragma unroll
                    for (int c = 0; c < CV; c++)
#pragma unroll
                        for (int u = 0; u < VEC; u++) acc[i][c * VEC + u] = fmaf(w, v_s[k * HD + (c * 16 + tx) * VEC + u], acc[i][c * VEC + u]);
                }
    }
}

// 256 threads, two blocks an SM where their shared memory allows it (64 rows of 128 columns: 97 KB): one block's products run beside the
// other's loads and exponentials.
template <typename T, int NI>
__global__ void __launch_bounds__(THREADS, 2)
tree_kernel(TreeArgs a, const T* q, long long ldq, T* out, long long ldo, const T* k_store, const T* v_store, float* ws_acc, float2* ws_ml) {
    constexpr int TM = 16 * NI;
    extern __shared__ __align__(16) float smem[];
    float *q_s = smem, *k_s = q_s + TM * LDQ, *v_s = k_s + K_FLOATS<NI>, *p_s = k_s;
    uint64_t* mask_s = reinterpret_cast<uint64_t*>(v_s + DK_PAGE * HD);
    pdl_wait();
    pdl_launch_dependents();
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4, G = a.nh / a.nkv;
    TreeWalk w;
    w.begin(a);
    const TreeSeq& sq = w.sq;
    while (w.next(a)) {
        const int p0 = w.p0, p1 = w.p1, kvh = w.kvh, rows = w.nodes * G, flat0 = sq.flat0 + w.node0;
        const int* pt = w.pt;
        for (int i = threadIdx.x; i < TM * (HD / 4); i += THREADS) {
            const int r = i / (HD / 4), c = (i % (HD / 4)) * 4;
            if (r < rows) load4(q_s + r * LDQ + c, q + (size_t)(flat0 + r / G) * ldq + (kvh * G + r % G) * HD + c);
            else *reinterpret_cast<float4*>(q_s + r * LDQ + c) = make_float4(0.f, 0.f, 0.f, 0.f);
        }
        float m[NI], l[NI], acc[NI][CV * VEC];
#pragma unroll
        for (int i = 0; i < NI; i++) {
            m[i] = -INFINITY, l[i] = 0.f;
#pragma unroll
            for (int c = 0; c < CV * VEC; c++) acc[i][c] = 0.f;
        }
        for (int p = p0; p < p1; p++) {
            const int key0 = (sq.first_page + p) * DK_PAGE;
            int page = pt[p];
            const bool held = page >= 0 && page < a.n_pages;           // a page that is none holds no keys
            if (!held) page = 0;
            const size_t off = kv_offset(page, a.nkv, kvh, 0, HD);
            for (int i = threadIdx.x; i < DK_PAGE * (HD / 4); i += THREADS) load4(k_s + i / (HD / 4) * LDK + (i % (HD / 4)) * 4, k_store + off + (size_t)i * 4);
            copies_end();                                              // the scores wait for the keys (and the tile's queries) alone
            for (int i = threadIdx.x; i < DK_PAGE * (HD / 4); i += THREADS) load4(v_s + i * 4, v_store + off + (size_t)i * 4);
            copies_end();
            bool masked = false;
            if (threadIdx.x < TM) {
                const int r = threadIdx.x, row = flat0 + r / G;
                const uint64_t seen = held && r < rows ? tree_mask(a, sq, a.tree + (size_t)row * a.words, a.row_pos[row], key0) : 0ull;
                mask_s[r] = seen;
                masked = r < rows && seen != ~0ull;
            }
            copied<1>();
            masked = __syncthreads_or(masked);
            if (NI >= 4 && rows > 32) page_step<NI, NI>(q_s, k_s, v_s, p_s, mask_s, a.sl2, masked, m, l, acc);
            else if (NI >= 2 && rows > 16) page_step<(NI < 2 ? NI : 2), NI>(q_s, k_s, v_s, p_s, mask_s, a.sl2, masked, m, l, acc);
            else page_step<1, NI>(q_s, k_s, v_s, p_s, mask_s, a.sl2, masked, m, l, acc);
            __syncthreads();
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
            for (int c = 0; c < CV * VEC; c++) {
                const int d = (c / VEC * 16 + tx) * VEC + c % VEC;
                if (whole) dst[d] = from_f<T>(acc[i][c] * inv);
                else ws_acc[slot * HD + part_at(TM, r, d)] = acc[i][c];
            }
        }
    }
}

template <int NI>
constexpr size_t tree_smem() {
    return sizeof(float) * (16 * NI * LDQ + K_FLOATS<NI> + DK_PAGE * HD) + 16 * NI * sizeof(uint64_t);
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
