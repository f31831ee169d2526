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
constexpr int THREADS = 256, LDK = HD + 4, LDP = DK_PAGE + 4, CV = HD / 16;

__device__ __forceinline__ void load4(float* dst, const float* src) { *reinterpret_cast<float4*>(dst) = *reinterpret_cast<const float4*>(src); }
__device__ __forceinline__ void load4(float* dst, const bf16* src) {
    const uint2 v = *reinterpret_cast<const uint2*>(src);
    const __nv_bfloat162 *a = reinterpret_cast<const __nv_bfloat162*>(&v.x), *b = reinterpret_cast<const __nv_bfloat162*>(&v.y);
    *reinterpret_cast<float4*>(dst) = make_float4(__low2float(*a), __high2float(*a), __low2float(*b), __high2float(*b));
}

// 256 threads: thread (ty, tx) of 16 x 16 has rows ty + 16 i of the tile (i < NI), keys tx + 16 j of the page, columns tx + 16 c.
template <typename T, int NI>
__global__ void __launch_bounds__(THREADS)
tree_kernel(TreeArgs a, const T* q, long long ldq, T* out, long long ldo, const T* k_store, const T* v_store, float* ws_acc, float2* ws_ml) {
    constexpr int TM = 16 * NI;
    extern __shared__ __align__(16) float smem[];
    float *q_s = smem, *k_s = q_s + TM * HD, *v_s = k_s + DK_PAGE * LDK, *p_s = v_s + DK_PAGE * HD;
    uint64_t* mask_s = reinterpret_cast<uint64_t*>(p_s + TM * LDP);
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
            if (r < rows) load4(q_s + r * HD + c, q + (size_t)(flat0 + r / G) * ldq + (kvh * G + r % G) * HD + c);
            else *reinterpret_cast<float4*>(q_s + r * HD + c) = make_float4(0.f, 0.f, 0.f, 0.f);
        }
        float m[NI], l[NI], acc[NI][CV];
#pragma unroll
        for (int i = 0; i < NI; i++) {
            m[i] = -INFINITY, l[i] = 0.f;
#pragma unroll
            for (int c = 0; c < CV; c++) acc[i][c] = 0.f;
        }
        for (int p = p0; p < p1; p++) {
            const int key0 = (sq.first_page + p) * DK_PAGE;
            int page = pt[p];
            const bool held = page >= 0 && page < a.n_pages;           // a page that is none holds no keys
            if (!held) page = 0;
            const size_t off = kv_offset(page, a.nkv, kvh, 0, HD);
            bool odd = false;                                           // an infinite or undefined value in this page
            for (int i = threadIdx.x; i < DK_PAGE * (HD / 4); i += THREADS) {
                const int r = i / (HD / 4), c = (i % (HD / 4)) * 4;
                load4(k_s + r * LDK + c, k_store + off + (size_t)i * 4);
                float* v = v_s + r * HD + c;
                load4(v, v_store + off + (size_t)i * 4);
                odd |= !isfinite(v[0]) || !isfinite(v[1]) || !isfinite(v[2]) || !isfinite(v[3]);
            }
            if (threadIdx.x < TM) {
                const int r = threadIdx.x, row = flat0 + r / G;
                mask_s[r] = held && r < rows ? tree_mask(a, sq, a.tree + (size_t)row * a.words, a.row_pos[row], key0) : 0ull;
            }
            odd = __syncthreads_or(odd);
            float sc[NI][4];
#pragma unroll
            for (int i = 0; i < NI; i++) sc[i][0] = sc[i][1] = sc[i][2] = sc[i][3] = 0.f;
#pragma unroll 4
            for (int d = 0; d < HD; d += 4) {
                float4 qa[NI], kb[4];
#pragma unroll
                for (int i = 0; i < NI; i++) qa[i] = *reinterpret_cast<const float4*>(q_s + (ty + 16 * i) * HD + d);
#pragma unroll
                for (int j = 0; j < 4; j++) kb[j] = *reinterpret_cast<const float4*>(k_s + (tx + 16 * j) * LDK + d);
#pragma unroll
                for (int i = 0; i < NI; i++)
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        sc[i][j] = fmaf(qa[i].x, kb[j].x, sc[i][j]);
                        sc[i][j] = fmaf(qa[i].y, kb[j].y, sc[i][j]);
                        sc[i][j] = fmaf(qa[i].z, kb[j].z, sc[i][j]);
                        sc[i][j] = fmaf(qa[i].w, kb[j].w, sc[i][j]);
                    }
            }
            float alpha[NI];
#pragma unroll
            for (int i = 0; i < NI; i++) {
                const uint64_t seen = mask_s[ty + 16 * i];
                float mx = -INFINITY;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    if (!(seen >> (tx + 16 * j) & 1)) sc[i][j] = -INFINITY;
                    mx = fmaxf(mx, sc[i][j]);
                }
#pragma unroll
                for (int o = 8; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
                const float mn = fmaxf(m[i], mx * a.sl2), ms = mn == -INFINITY ? 0.f : mn;
                alpha[i] = exp2f(m[i] - ms);
                m[i] = mn;
                float sum = 0.f;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float pw = exp2f(fmaf(sc[i][j], a.sl2, -ms));
                    sum += pw;
                    p_s[(ty + 16 * i) * LDP + tx + 16 * j] = pw;
                }
#pragma unroll
                for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                l[i] = l[i] * alpha[i] + sum;
#pragma unroll
                for (int c = 0; c < CV; c++) acc[i][c] *= alpha[i];
            }
            __syncwarp();                                               // a row's 16 threads sit in one warp
            if (!odd) {
#pragma unroll 4
                for (int k = 0; k < DK_PAGE; k++) {
                    float pw[NI];
#pragma unroll
                    for (int i = 0; i < NI; i++) pw[i] = p_s[(ty + 16 * i) * LDP + k];
#pragma unroll
                    for (int c = 0; c < CV; c++) {
                        const float v = v_s[k * HD + tx + 16 * c];
#pragma unroll
                        for (int i = 0; i < NI; i++) acc[i][c] = fmaf(pw[i], v, acc[i][c]);
                    }
                }
            } else {
                for (int k = 0; k < DK_PAGE; k++)
#pragma unroll
                    for (int i = 0; i < NI; i++)
                        if (mask_s[ty + 16 * i] >> k & 1) {
                            const float pw = p_s[(ty + 16 * i) * LDP + k];
#pragma unroll
                            for (int c = 0; c < CV; c++) acc[i][c] = fmaf(pw, v_s[k * HD + tx + 16 * c], acc[i][c]);
                        }
            }
            __syncthreads();
        }
        const bool whole = w.all();
        const size_t slot = (size_t)w.slot() * TM;
#pragma unroll
        for (int i = 0; i < NI; i++) {
            const int r = ty + 16 * i;
            if (r >= rows) continue;
            if (whole) {
                const float inv = l[i] == 0.f ? 0.f : 1.f / l[i];
                T* dst = out + (size_t)(flat0 + r / G) * ldo + (kvh * G + r % G) * HD;
#pragma unroll
                for (int c = 0; c < CV; c++) dst[tx + 16 * c] = from_f<T>(acc[i][c] * inv);
            } else {
                if (tx == 0) ws_ml[slot + r] = make_float2(m[i], l[i]);
#pragma unroll
                for (int c = 0; c < CV; c++) ws_acc[slot * HD + part_at(TM, r, tx + 16 * c)] = acc[i][c];
            }
        }
    }
}

template <int NI>
constexpr size_t tree_smem() {
    return sizeof(float) * (16 * NI * HD + DK_PAGE * LDK + DK_PAGE * HD + 16 * NI * LDP) + 16 * NI * sizeof(uint64_t);
}

template <typename T, int NI>
int launch(const TreeArgs& a, const void* q, long long ldq, void* out, long long ldo, const void* k_store, const void* v_store, float* ws_acc,
           float* ws_ml, int max_nodes, int blocks, cudaStream_t st) {
    static SmemOnce once;
    int r = once.allow((const void*)tree_kernel<T, NI>, tree_smem<NI>());
    if (r) return r;
    r = dk_launch(tree_kernel<T, NI>, dim3(blocks), dim3(THREADS), tree_smem<NI>(), st, a, (const T*)q, ldq, (T*)out, ldo,
                      (const T*)k_store, (const T*)v_store, ws_acc, (float2*)ws_ml);
    if (r) return r;
    return tree_merge<T, HD>(a, ws_acc, ws_ml, out, ldo, 16 * NI, max_nodes, blocks, st);
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
    TreeArgs a = {cu_q, seq_pos0, row_pos, page_table, tree, n_seq, words, pt_stride, n_pages, nh, nkv, window, rows / G, rows / G, rows,
                  pt_stride <= WHOLE_PAGES, 0, scale * 1.4426950408889634f};
    if (!tree_units_fit(a, max_nodes) || nkv > 65535) return (int)cudaErrorInvalidValue;
#define DK_TREE(T, NI) launch<T, NI>(a, q, ldq, out, ldo, k_store, v_store, ws_acc, ws_ml, max_nodes, blocks, st)
    if (f32) return rows == 16 ? DK_TREE(float, 1) : rows == 32 ? DK_TREE(float, 2) : DK_TREE(float, 4);
    return rows == 16 ? DK_TREE(bf16, 1) : rows == 32 ? DK_TREE(bf16, 2) : DK_TREE(bf16, 4);
#undef DK_TREE
}
