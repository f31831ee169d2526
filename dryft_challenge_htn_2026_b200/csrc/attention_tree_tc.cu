// bfloat16 attention of trees of drafted tokens over the paged cache on the 5th-generation tensor cores, for head sizes 64 and 128
// (built per head size with -DHD=64 or -DHD=128). Which keys a node sees and how the work is dealt out: attention_tree.cuh.
//
// A tile is 128 rows, nodes x the query heads of one kv head (four heads a kv head: 32 nodes), so that a page of keys is read once for
// all of them. A block walks the pages of its share:
//   warp 5, one thread: TMA loads. Q once a tile, as boxes [tile nodes][heads of the kv head][64 columns]; K and V of each page as
//       [64 keys x 64 columns], 128-byte swizzle, two stages each.
//   warp 4, one thread: all tcgen05.mma. S[128 x 64] = Q.K^T into one of two buffers, O[128 x HD] += P.V with P from tensor memory. S
//       runs two pages ahead of P.V.
//   warps 0-3: softmax, a thread a row: its row of S from tensor memory, running maximum and sum in float32, P as bfloat16 (rounded
//       once, to be the product's operand; the sum takes the unrounded weights) over its S buffer, and at the end the row of O.
// Pages of cached tokens that every row sees need no mask. In the others (the tree's own, the first of a window) a row's 64 visible
// places are one word of bits. P.V adds up 0 * v for what a row does not see: where such a page holds a value that is not finite it is
// set to zero in shared memory, and at the end the rows that do see it take it up from the cache.
// Tensor memory: S0 | S1 | O = 64 + 64 + 128 columns; two blocks an SM (96 KB of shared memory each at head size 128).
// Every mbarrier wait is bounded; a wait that runs out stores a code in *err, and the block still frees its tensor memory and returns.
#include <cuda.h>

#include "attention_tree.cuh"

#ifndef HD
#error "compile with -DHD=64 or -DHD=128"
#endif
static_assert(HD == 64 || HD == 128, "built for head sizes 64 and 128");

namespace {

constexpr int BM = 128, BN = DK_PAGE;             // rows a tile, keys a step (one page)
constexpr int SOFT = 128;                         // softmax threads, one a row; then the mma warp, then the loader warp
constexpr int THREADS = SOFT + 64;
constexpr int BLOCKS_PER_SM = 2;
constexpr int TMEM_ALLOC = 256;                   // S0 | S1 | O
constexpr int OC = 32;                            // columns of O a thread handles at a time
constexpr int HALVES = HD / 64;                   // 64-column swizzle atoms across the head
constexpr int Q_BYTES = BM * HD * 2, KV_BYTES = BN * HD * 2;
constexpr int Q_ATOM_BYTES = BM * 128, KV_ATOM_BYTES = BN * 128;
constexpr size_t SMEM_BYTES = 1024 + Q_BYTES + 4 * KV_BYTES + 14 * sizeof(uint64_t);
#ifndef DK_WAIT_CYCLES
#define DK_WAIT_CYCLES 2000000000LL               // about a second: a wait this long has failed
#endif
constexpr long long WAIT_CYCLES = DK_WAIT_CYCLES;
#ifdef DK_TEST_STALL
// Test build only: with the flag set the loader thread requests nothing, so the other waits run out and the error path runs.
__device__ int dk_stall_flag;
DK_EXPORT int dk_test_stall(int on) { return (int)cudaMemcpyToSymbol(dk_stall_flag, &on, sizeof(int)); }
#define DK_STALLED (dk_stall_flag != 0)
#else
#define DK_STALLED false
#endif
constexpr uint32_t IDESC_S = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(BM >> 4) << 24);
constexpr uint32_t IDESC_PV = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((uint32_t)(HD >> 3) << 17) | ((uint32_t)(BM >> 4) << 24);

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mbar_init(uint64_t* bar, int count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count));
}
__device__ __forceinline__ void mbar_expect_tx(uint64_t* bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{ .reg .pred p; mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return ok != 0;
}
// the clock is read only when the barrier is not through yet (most waits of the mma thread find it through)
// try_wait lets the hardware suspend the thread for a while instead of having it poll: a polling
// thread takes issue slots from the softmax warps of the other block on its scheduler
__device__ __forceinline__ bool mbar_try(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return ok != 0;
}
__device__ __forceinline__ bool mbar_wait(uint64_t* bar, uint32_t parity) {
    if (mbar_test(bar, parity)) return true;
    const long long t0 = clock64();
    for (;;) {
        if (mbar_try(bar, parity)) return true;
        if (clock64() - t0 > WAIT_CYCLES) return false;
    }
}
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
                 "l"((uint64_t)map), "r"(smem_u32(bar)), "r"(x), "r"(y)
                 : "memory");
}
// K-major operand, 128-byte swizzle: rows 128 bytes apart, groups of 8 rows 1024 bytes apart.
__device__ __forceinline__ uint64_t desc_k_major(uint32_t addr) {
    return (uint64_t)((addr & 0x3FFFF) >> 4) | ((uint64_t)1 << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) |
           ((uint64_t)2 << 61);
}
// N-major operand (V: keys are the rows in shared memory, the head columns are contiguous),
// 128-byte swizzle: the next 64 columns are KV_ATOM_BYTES away, the next 8 keys 1024 bytes.
__device__ __forceinline__ uint64_t desc_n_major(uint32_t addr) {
    return (uint64_t)((addr & 0x3FFFF) >> 4) | ((uint64_t)(KV_ATOM_BYTES >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
           ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
__device__ __forceinline__ void umma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile("{ .reg .pred p; setp.ne.b32 p, %4, 0; tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p; }" ::"r"(d),
                 "l"(a), "l"(b), "r"(idesc), "r"(acc)
                 : "memory");
}
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a_tmem, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile("{ .reg .pred p; setp.ne.b32 p, %4, 0; tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p; }" ::"r"(d),
                 "r"(a_tmem), "l"(b), "r"(idesc), "r"(acc)
                 : "memory");
}
__device__ __forceinline__ void umma_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// (no wait inside: call tmem_wait_ld() before the registers are used)
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,"
        "%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,"
        "%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]),
        "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]),
        "r"(r[31])
        : "memory");
}
// 2^x, one MUFU instruction (-inf gives 0)
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
                 "l"((uint64_t)map), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
                 : "memory");
}
// maximum of three, one instruction
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// grid min(units, 2 * SMs), 192 threads. q as [rows][heads][HD] (map_q), map_k / map_v over one layer's store as [pages * nkv * 64, HD].
// The per-step barriers (K, V, S, P, O) complete once a step and bar_q once a tile: their phases run on over the tiles.
__global__ void __launch_bounds__(THREADS, BLOCKS_PER_SM)
tree_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
               const __grid_constant__ TreeArgs a, bf16* out, long long ldo, const bf16* v_store, float* ws_acc, float2* ws_ml, int* err) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
    const uint32_t q_s = smem_u32(smem), k_s = q_s + Q_BYTES, v_s = k_s + 2 * KV_BYTES;   // Q, K stages 0 1, V stages 0 1
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Q_BYTES + 4 * KV_BYTES);
    uint64_t *bar_q = bars, *bar_k = bars + 1, *bar_v = bars + 3, *bar_s = bars + 5, *bar_p = bars + 7, *bar_o = bars + 9;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 11);
    volatile int* failed = reinterpret_cast<volatile int*>(bars + 12);     // [0] a wait ran out; [1] the last tile with a value that is not finite
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, G = a.nh / a.nkv;
    constexpr int MMA_WARP = SOFT / 32, LOAD_WARP = MMA_WARP + 1;

    pdl_wait();
    if (threadIdx.x == 0) {
        mbar_init(bar_q, 1);
        for (int b = 0; b < 2; b++)
            mbar_init(bar_k + b, 1), mbar_init(bar_v + b, 1), mbar_init(bar_s + b, 1), mbar_init(bar_o + b, 1), mbar_init(bar_p + b, SOFT);
        failed[0] = 0, failed[1] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == MMA_WARP) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(TMEM_ALLOC)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // where the block's share begins; every warp finds it for itself
    const long long total = tree_units(a, a.n_seq);
    const int nb = share_count(total, gridDim.x);
    const bool busy = (int)blockIdx.x < nb;
    long long u = busy ? share_begin(total, blockIdx.x, nb) : 0, before = 0;
    const long long u_end = busy ? share_begin(total, blockIdx.x + 1, nb) : 0;
    int s = busy ? tree_find(a, u, before) : 0;
    fence_before();
    __syncthreads();
    fence_after();
    pdl_launch_dependents();       // not before every block holds its tensor memory: the next kernel's blocks may want some too
    const uint32_t tmem = *tmem_slot;
    const uint32_t t_s = tmem, t_o = tmem + 2 * BN;        // S buffers (and P over them) of BN columns each, then O of HD columns

    TreeSeq sq;
    if (busy) sq.load(a, s);
    uint32_t step = 0;
    int tiles_done = 0;
    while (u < u_end && !failed[0]) {
        while (u >= before + sq.units(a.nkv)) {
            before += sq.units(a.nkv);
            sq.load(a, ++s);
        }
        const long long at = u - before;
        const int item = (int)(at / sq.pages), p0 = (int)(at % sq.pages), p1 = (int)min((long long)sq.pages, p0 + (u_end - u));
        const int kvh = item / sq.tiles, node0 = (item % sq.tiles) * a.tile_nodes;
        const int rows = min(a.tile_nodes, sq.n - node0) * G, flat0 = sq.flat0 + node0;
        const int* pt = a.page_table + (size_t)s * a.pt_stride + sq.first_page;
        const int n_blk = p1 - p0;

        // Step j of the tile is step t = step + j of the block; it uses stage / buffer / barrier t & 1, whose barriers are then in
        // their phase (t >> 1) & 1.
        if (warp == LOAD_WARP) {
            if (lane == 0 && DK_STALLED) failed[0] = 1;
            if (lane == 0 && !DK_STALLED) {  // --------------------------------------------------- every TMA
                auto load_kv = [&](const CUtensorMap* map, uint32_t stages, uint64_t* bar, int j) {
                    const uint32_t b = (step + j) & 1;
                    mbar_expect_tx(bar + b, KV_BYTES);
                    int page = pt[p0 + j];
                    if (page < 0 || page >= a.n_pages) page = 0;       // any page will do: its keys are masked
                    const int row = (page * a.nkv + kvh) * DK_PAGE;
                    for (int hh = 0; hh < HALVES; hh++)
                        tma_load_2d(stages + b * KV_BYTES + hh * KV_ATOM_BYTES, map, hh * 64, row, bar + b);
                };
                mbar_expect_tx(bar_q, HALVES * a.tile_nodes * G * 128);
                for (int hh = 0; hh < HALVES; hh++) tma_load_3d(q_s + hh * Q_ATOM_BYTES, &map_q, hh * 64, kvh * G, flat0, bar_q);
                load_kv(&map_k, k_s, bar_k, 0);
                load_kv(&map_v, v_s, bar_v, 0);
                if (n_blk > 1) load_kv(&map_k, k_s, bar_k, 1), load_kv(&map_v, v_s, bar_v, 1);
                bool ok = true;
                // in the order in which the stages come free: S(j) is done with K(j), then P.V(j-1) with V(j-1)
                for (int j = 0; j + 2 < n_blk && ok; j++) {
                    const uint32_t t = step + j;
                    if (!mbar_wait(bar_s + (t & 1), (t >> 1) & 1)) { ok = false; break; }
                    load_kv(&map_k, k_s, bar_k, j + 2);
                    if (j >= 1) {
                        if (!mbar_wait(bar_o + ((t - 1) & 1), ((t - 1) >> 1) & 1)) { ok = false; break; }
                        load_kv(&map_v, v_s, bar_v, j + 1);
                    }
                }
                if (ok && n_blk > 2) {                                 // the last page's values: after P.V(n - 3)
                    const uint32_t t = step + n_blk - 3;
                    ok = mbar_wait(bar_o + (t & 1), (t >> 1) & 1);
                    if (ok) load_kv(&map_v, v_s, bar_v, n_blk - 1);
                }
                if (!ok) atomicExch(err, 23), failed[0] = 1;
            }
        } else if (warp == MMA_WARP) {
            if (lane == 0) {  // ------------------------------------------------------------ every tcgen05.mma
                const uint64_t dq = desc_k_major(q_s), dk = desc_k_major(k_s), dv = desc_n_major(v_s);
                auto issue_s = [&](int j) {
                    const uint32_t b = (step + j) & 1;
                    const uint64_t dkb = dk + (uint64_t)((b * KV_BYTES) >> 4);
#pragma unroll
                    for (int hh = 0; hh < HALVES; hh++)
#pragma unroll
                        for (int k = 0; k < 4; k++)
                            umma_ss(t_s + b * BN, dq + (uint64_t)((hh * Q_ATOM_BYTES + k * 32) >> 4),
                                    dkb + (uint64_t)((hh * KV_ATOM_BYTES + k * 32) >> 4), IDESC_S, (hh | k) != 0);
                    umma_commit(bar_s + b);
                };
                bool ok = mbar_wait(bar_q, tiles_done & 1);
                for (int j = 0; j < 2 && j < n_blk && ok; j++) {
                    const uint32_t t = step + j;
                    ok = mbar_wait(bar_k + (t & 1), (t >> 1) & 1);
                    if (ok) fence_after(), issue_s(j);
                }
                for (int i = 0; i < n_blk && ok; i++) {
                    const uint32_t t = step + i, b = t & 1, ph = (t >> 1) & 1;
                    if (!mbar_wait(bar_p + b, ph)) { ok = false; break; }
                    if (!mbar_wait(bar_v + b, ph)) { ok = false; break; }
                    fence_after();
#pragma unroll
                    for (int k = 0; k < BN / 16; k++)
                        umma_ts(t_o, t_s + b * BN + k * 8, dv + (uint64_t)((b * KV_BYTES + k * 16 * 128) >> 4), IDESC_PV, (i | k) != 0);
                    umma_commit(bar_o + b);
                    if (i + 2 < n_blk) {       // into the buffer whose P was just used: products of one thread run in order
                        const uint32_t t2 = t + 2;
                        if (!mbar_wait(bar_k + (t2 & 1), (t2 >> 1) & 1)) { ok = false; break; }
                        fence_after();
                        issue_s(i + 2);
                    }
                }
                if (!ok) atomicExch(err, 21), failed[0] = 1;
            }
        } else {  // ------------------------------------------------------------------ softmax, a thread a row
            const int r = threadIdx.x, node = flat0 + r / G, mark = tiles_done + 1;
            const int qpos = r < rows ? a.row_pos[node] : -1;
            const bool valid = qpos >= 0;
            const uint32_t* words = a.tree + (size_t)(r < rows ? node : flat0) * a.words;
            const bool any_row = warp * 32 < rows;                     // else the warp has no row of the tile
            const uint32_t lane_off = (uint32_t)(warp * 32) << 16;
            // pages that every row sees: the cached tokens' and, with a window, none that the last node's begins in
            const int open_lo = a.window > 0 ? max(0, sq.pos0 + sq.n - a.window) : 0;
            float m = -INFINITY, l = 0.f;
            bool ok = true;
            for (int i = 0; i < n_blk && ok; i++) {
                const uint32_t t = step + i, b = t & 1, ph = (t >> 1) & 1;
                const int key0 = (sq.first_page + p0 + i) * BN, page = pt[p0 + i];
                const bool held = page >= 0 && page < a.n_pages;
                const bool open = held && key0 + BN <= sq.pos0 && key0 >= open_lo;
                uint64_t seen = ~0ull;
                if (!open) {
                    seen = held && valid ? tree_mask(a, sq, words, qpos, key0) : 0ull;
                    if (!mbar_wait(bar_v + b, ph)) { ok = false; break; }
                    // 16 bytes each of the page's values at a time
                    uint4* vs = reinterpret_cast<uint4*>(smem + Q_BYTES + 2 * KV_BYTES + b * KV_BYTES);
                    bool odd = false;
#pragma unroll
                    for (int k = 0; k < KV_BYTES / 16 / SOFT; k++) {
                        uint4 x = vs[k * SOFT + r];
                        uint32_t* w = reinterpret_cast<uint32_t*>(&x);
                        bool mine = false;
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            if ((w[e] & 0x7f80u) == 0x7f80u) w[e] &= 0xffff0000u, mine = true;
                            if ((w[e] & 0x7f800000u) == 0x7f800000u) w[e] &= 0xffffu, mine = true;
                        }
                        if (mine) vs[k * SOFT + r] = x, odd = true;
                    }
                    if (odd) {
                        failed[1] = mark;
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    }
                }
                if (!mbar_wait(bar_s + b, ph)) { ok = false; break; }
                if (any_row) {
                    __syncwarp();
                    fence_after();
                    uint32_t v[BN];
#pragma unroll
                    for (int c = 0; c < BN; c += 32) tmem_ld32(t_s + lane_off + b * BN + c, *reinterpret_cast<uint32_t(*)[32]>(v + c));
                    tmem_wait_ld();
                    float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                    if (!open) {
                        const uint32_t half[2] = {(uint32_t)seen, (uint32_t)(seen >> 32)};
#pragma unroll
                        for (int j = 0; j < BN; j++)
                            if (!(half[j / 32] >> (j % 32) & 1)) v[j] = 0xff800000u;           // -infinity
                    }
#pragma unroll
                    for (int j = 0; j < BN; j += 2) mx4[(j >> 1) & 3] = max3(mx4[(j >> 1) & 3], __uint_as_float(v[j]), __uint_as_float(v[j + 1]));
                    const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * a.sl2;   // sl2 > 0: scaling keeps the order
                    float m_new = fmaxf(m, mx);
                    // a maximum that moved by less than 8 (a factor 256) keeps the old reference: O need not be rescaled
                    if (m != -INFINITY && m_new - m < 8.f) m_new = m;
                    const float ms = m_new == -INFINITY ? 0.f : m_new;
                    const float alpha = m_new == m ? 1.f : ex2(m - ms);
                    if (i > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
                        if (!mbar_wait(bar_o + (b ^ 1), ((t - 1) >> 1) & 1)) { ok = false; break; }
                        fence_after();
#pragma unroll 1
                        for (int c = 0; c < HD; c += OC) {
                            uint32_t o[OC];
                            tmem_ld32(t_o + lane_off + c, o);
                            tmem_wait_ld();
#pragma unroll
                            for (int j = 0; j < OC; j++) o[j] = __float_as_uint(__uint_as_float(o[j]) * alpha);
                            tmem_st32(t_o + lane_off + c, o);
                        }
                    }
                    float sum4[4] = {0.f, 0.f, 0.f, 0.f};
                    uint32_t p[BN / 2];
#pragma unroll
                    for (int j = 0; j < BN; j += 2) {
                        const float e0 = ex2(fmaf(__uint_as_float(v[j]), a.sl2, -ms)), e1 = ex2(fmaf(__uint_as_float(v[j + 1]), a.sl2, -ms));
                        sum4[(j >> 1) & 3] += e0 + e1;
                        __nv_bfloat162 pk = __floats2bfloat162_rn(e0, e1);
                        p[j / 2] = *reinterpret_cast<uint32_t*>(&pk);
                    }
                    tmem_st32(t_s + lane_off + b * BN, p);
                    l = l * alpha + (sum4[0] + sum4[1]) + (sum4[2] + sum4[3]);
                    m = m_new;
                    tmem_wait_st();
                    fence_before();
                }
                mbar_arrive(bar_p + b);
            }
            if (ok) ok = mbar_wait(bar_o + ((step + n_blk - 1) & 1), ((step + n_blk - 1) >> 1) & 1);
            if (ok && any_row) {
                fence_after();
                const bool whole = n_blk == sq.pages, mend = failed[1] == mark;
                if (!valid) m = -INFINITY, l = 0.f;
                const float inv = l == 0.f ? 0.f : 1.f / l;
                const size_t slot = (size_t)(2 * blockIdx.x + (p0 == 0 ? 1 : 0)) * BM + r;
                bf16* dst = out + (size_t)(flat0 + r / G) * ldo + (size_t)(kvh * G + r % G) * HD;
                if (!whole && r < rows) ws_ml[slot] = make_float2(m, l);
#pragma unroll 1
                for (int c = 0; c < HD; c += OC) {
                    uint32_t o[OC];
                    __syncwarp();
                    tmem_ld32(t_o + lane_off + c, o);
                    tmem_wait_ld();
                    if (r >= rows) continue;
                    if (!valid || l == 0.f) {
#pragma unroll
                        for (int j = 0; j < OC; j++) o[j] = 0;
                    } else if (mend) {         // values that are not finite, for the rows that see them
                        for (int i = 0; i < n_blk; i++) {
                            const int key0 = (sq.first_page + p0 + i) * BN, page = pt[p0 + i];
                            if (page < 0 || page >= a.n_pages || (key0 + BN <= sq.pos0 && key0 >= open_lo)) continue;
                            for (uint64_t left = tree_mask(a, sq, words, qpos, key0); left; left &= left - 1) {
                                const bf16* val = v_store + kv_offset(page, a.nkv, kvh, __ffsll((long long)left) - 1, HD) + c;
#pragma unroll
                                for (int j = 0; j < OC; j++) {
                                    const float x = __bfloat162float(val[j]);
                                    if (!isfinite(x)) o[j] = __float_as_uint(__uint_as_float(o[j]) + x);
                                }
                            }
                        }
                    }
                    if (whole) {
#pragma unroll
                        for (int j = 0; j < OC; j += 8) {
                            uint4 pk;
                            __nv_bfloat162* pp = reinterpret_cast<__nv_bfloat162*>(&pk);
#pragma unroll
                            for (int e = 0; e < 4; e++)
                                pp[e] = __floats2bfloat162_rn(__uint_as_float(o[j + 2 * e]) * inv, __uint_as_float(o[j + 2 * e + 1]) * inv);
                            *reinterpret_cast<uint4*>(dst + c + j) = pk;
                        }
                    } else {
#pragma unroll
                        for (int j = 0; j < OC; j += 4) *reinterpret_cast<uint4*>(ws_acc + slot * HD + c + j) = make_uint4(o[j], o[j + 1], o[j + 2], o[j + 3]);
                    }
                }
            } else if (!ok && lane == 0) {
                atomicExch(err, 22), failed[0] = 1;
            }
        }
        // everyone is done with the tile: O has been read out of tensor memory
        step += n_blk, tiles_done++, u += n_blk;
        fence_before();
        __syncthreads();
        fence_after();
    }
    if (warp == MMA_WARP) {
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_ALLOC) : "memory");
    }
}

typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encoder() {
    static EncodeTiled fn = nullptr;
    if (!fn) {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = (EncodeTiled)p;
    }
    return fn;
}

// bf16 tensor of up to three dimensions (innermost first), 128-byte swizzle, zero fill; strides in bytes of all but the innermost
int make_map(CUtensorMap* map, const void* base, int rank, const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box) {
    EncodeTiled enc = encoder();
    if (!enc) return (int)cudaErrorNotSupported;
    cuuint32_t elem[3] = {1, 1, 1};
    CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank, const_cast<void*>(base), dims, strides, box, elem,
                     CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? 0 : (int)cudaErrorInvalidValue;
}

}  // namespace

DK_EXPORT int dk_tree_tc_tile_rows() { return BM; }
DK_EXPORT int dk_tree_tc_blocks_per_sm() { return BLOCKS_PER_SM; }

// q [n_rows, nh*HD] and out, bf16, rows ldq / ldo elements apart (multiples of 8, 16-byte boundaries); k_store, v_store [n_pages, nkv, 64,
// HD]; ws_acc: 2 * blocks * 128 * HD floats, ws_ml: 2 * blocks * 128 * 2 floats; err: device int for a wait that ran out.
DK_EXPORT int dk_attn_tree_tc(const void* q, long long ldq, void* out, long long ldo, long long n_rows, const void* k_store,
                              const void* v_store, int n_pages, const int* cu_q, const int* seq_pos0, const int* row_pos,
                              const uint32_t* tree, int words, const int* page_table, int pt_stride, int n_seq, int nh, int nkv, int window,
                              float scale, int max_nodes, float* ws_acc, float* ws_ml, int blocks, int* err, cudaStream_t st) {
    if (nkv < 1 || nh % nkv || nh / nkv > 64 || n_pages < 1 || pt_stride < 1 || words < 1 || blocks < 1 || max_nodes < 1 || n_seq > 65535 ||
        err == nullptr || ldq % 8 || ldo % 8 || ((uintptr_t)q | (uintptr_t)out) % 16 || (long long)n_pages * nkv * DK_PAGE > 0x7fffffffLL)
        return (int)cudaErrorInvalidValue;
    const int G = nh / nkv;
    TreeArgs a = {cu_q, seq_pos0, row_pos, page_table, tree, n_seq, words, pt_stride, n_pages, nh, nkv, window, BM / G,
                  scale * 1.4426950408889634f};
    cudaError_t ce = cudaFuncSetAttribute(tree_tc_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SMEM_BYTES);
    if (ce != cudaSuccess) {
        cudaGetLastError();
        return (int)ce;
    }
    CUtensorMap mq, mk, mv;
    const cuuint64_t q_dims[3] = {HD, (cuuint64_t)nh, (cuuint64_t)n_rows}, q_strides[2] = {HD * 2, (cuuint64_t)ldq * 2};
    const cuuint32_t q_box[3] = {64, (cuuint32_t)G, (cuuint32_t)(BM / G)};
    const cuuint64_t kv_dims[2] = {HD, (cuuint64_t)n_pages * nkv * DK_PAGE}, kv_strides[1] = {HD * 2};
    const cuuint32_t kv_box[2] = {64, DK_PAGE};
    int e = make_map(&mq, q, 3, q_dims, q_strides, q_box);
    if (!e) e = make_map(&mk, k_store, 2, kv_dims, kv_strides, kv_box);
    if (!e) e = make_map(&mv, v_store, 2, kv_dims, kv_strides, kv_box);
    if (e) return e;
    e = dk_launch(tree_tc_kernel, dim3(blocks), dim3(THREADS), SMEM_BYTES, st, mq, mk, mv, a, (bf16*)out, ldo, (const bf16*)v_store, ws_acc,
                  (float2*)ws_ml, err);
    if (e) return e;
    return dk_launch(tree_merge_kernel<bf16, HD>, dim3((unsigned)(((long long)max_nodes * nh + 7) / 8), n_seq), dim3(256), 0, st, a,
                     (const float*)ws_acc, (const float2*)ws_ml, (bf16*)out, ldo, BM, blocks);
}
