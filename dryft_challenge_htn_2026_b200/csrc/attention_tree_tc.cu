// bfloat16 attention of trees of drafted tokens over the paged cache on the 5th-generation tensor cores, for head sizes 64 and 128
// (built per head size with -DHD=64 or -DHD=128). Which keys a node sees and how the work is dealt out: attention_tree.cuh.
//
// A block, one an SM, has two streams A and B of softmax warps, score buffers and accumulators, which share the tensor core and the
// pages that one thread loads:
//   a tile of up to 256 rows (nodes x the query heads of one kv head; four heads a kv head: 64 nodes) goes with its first 128 rows to
//   A and the rest to B, and every page is read once for both;
//   a tile of up to 128 rows goes to both, A takes the even pages of the block's share and B the odd ones, and their results are put
//   together from tensor memory (a row has the same lane in both accumulators).
// Roles:
//   warp 10, one thread: TMA loads. Q once a tile, as boxes [nodes][heads of the kv head][64 columns]; K and V of each page as [64 keys x
//       64 columns], 128-byte swizzle, into rings of their own (a key page is free once S is computed, its values after P.V), K two
//       pages ahead of V.
//   warps 8 (A) and 9 (B), one thread each: the stream's tcgen05.mma. S[128 x 64] = Q.K^T into one of the stream's two buffers, O[128 x HD] += P.V with P from tensor
//       memory. S runs two pages ahead of P.V.
//   warps 0-3 (A), 4-7 (B): softmax, a thread a row: its row of S from tensor memory, running maximum and sum in float32, P as bfloat16
//       (rounded once, to be the product's operand; the sum takes the unrounded weights) over its S buffer, at the end the row of O.
// Nobody waits for a tile's end but for what it leaves: the loader runs on into the next tile's pages, S of the next tile starts while
// the rows of the last one are written, only P.V into O waits until they are read.
// Pages of cached tokens that every row sees need no mask. In the others (the tree's own, the first of a window) a row's 64 visible
// places are one word of bits. P.V adds up 0 * v for what a row does not see: where such a page holds a value that is not finite, warp 11
// sets it to zero in shared memory before the products may have the page, and at the end the rows that do see it take it up from the
// cache. (Softmax warps that looked the page over themselves took 1.3 us for it, at the end of every tile.)
// Tensor memory: S of A 0 | 1, S of B 0 | 1, O of A, O of B = 4 x 64 + 2 x 128 columns.
//
// Measured (32 heads on 8 of 128): eight trees of 40 to 64 nodes behind 1,400 to 4,096 tokens 47.6 us (17.5 us of bytes, 13.8 us of
// products at the measured peaks), two trees of 13 to 24 behind 30,000 to 32,768 tokens 60 us (4.5 TB/s, 68 % of the copy rate). With 256
// rows a page step takes 1.2 us whatever the softmax does: S, P.V and the next S of a stream are chains of 8 + 4 tcgen05.mma that one
// thread issues, 60 to 100 clocks each, and both streams run in step. With up to 128 rows a step is two pages, 0.72 to 0.84 us a page
// against 0.74 us that its 32 KB take at the copy rate. Around the pages: about 4 us until the first products, 2 us to leave the parts, 6 us for
// the merge. One block an SM with two streams instead of two blocks an SM: 51.7 us for 55.6 in the first case, as a page is read once for
// 256 rows. The rings are as deep as shared memory allows, so that both streams can be a page apart.
// Every mbarrier wait is bounded; a wait that runs out stores a code in *err, and the block still frees its tensor memory and returns.
#include <cuda.h>

#include "attention_tree.cuh"

#ifndef HD
#error "compile with -DHD=64 or -DHD=128"
#endif
static_assert(HD == 64 || HD == 128, "built for head sizes 64 and 128");

namespace {

constexpr int BM = 128, BN = DK_PAGE;             // rows of a stream, keys a step (one page)
constexpr int SOFT = 2 * BM;                      // softmax threads, one a row of each stream; two mma warps, the loader's, the one that looks values over
constexpr int THREADS = SOFT + 128, MMA_WARP = SOFT / 32, LOAD_WARP = MMA_WARP + 2, CHECK_WARP = MMA_WARP + 3;
constexpr int TMEM_ALLOC = 512;
constexpr int OC = 16;                            // columns of a row's result a thread handles at a time
constexpr int HALVES = HD / 64;                   // 64-column swizzle atoms across the head
constexpr int Q_BYTES = BM * HD * 2, KV_BYTES = BN * HD * 2;
constexpr int Q_ATOM_BYTES = BM * 128, KV_ATOM_BYTES = BN * 128;
constexpr int WHOLE_PAGES = 8;                    // tables up to here are not split (see attention_tree.cuh)
constexpr int EXTRA = 5;                          // pages that a tile's beginning and end take as long as
constexpr int NK = HD == 128 ? 5 : 9, NV = HD == 128 ? 4 : 8;          // pages in the rings
constexpr int RING = 2 * Q_BYTES, V_RING = RING + NK * KV_BYTES, BARS = V_RING + NV * KV_BYTES;
constexpr int N_BARS = 2 * NK + 3 * NV + 12 + 4;
constexpr int MARKS = 16;                         // tiles that the warp that looks values over may be ahead of the softmax warps: a page each at least, so no more than NV + 1
static_assert(MARKS > NV + 1, "marks of tiles");
constexpr int ML = BARS + (N_BARS + 1 + MARKS / 2) * 8;       // [2][2][BM] pairs (maximum, sum) that the streams exchange
constexpr size_t SMEM_BYTES = 1024 + ML + 4 * BM * 8;
static_assert(SMEM_BYTES <= 227 * 1024, "shared memory of a block");
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
// the clock is read only when the barrier is not through yet (most waits of the mma threads find it through)
// try_wait lets the hardware suspend the thread for a while instead of having it poll: a polling thread takes
// issue slots from the softmax warps on its scheduler
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
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
                   "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
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

// Whether one of two bfloat16 numbers is infinite or none; the two with 0 in the place of such a one.
__device__ __forceinline__ bool no_number(uint32_t x) { return (x & 0x7f80u) == 0x7f80u || (x & 0x7f800000u) == 0x7f800000u; }
__device__ __forceinline__ uint32_t numbers_of(uint32_t x) {
    if ((x & 0x7f80u) == 0x7f80u) x &= 0xffff0000u;
    return (x & 0x7f800000u) == 0x7f800000u ? x & 0xffffu : x;
}

struct Walk : TreeWalk {
    bool pair;                                             // two streams of rows; else two streams of pages
    __device__ __forceinline__ bool next(const TreeArgs& a) {
        if (!TreeWalk::next(a)) return false;
        pair = nodes > a.half_nodes;
        return true;
    }
    // steps of stream x, and the page of its step i, counted from p0
    __device__ __forceinline__ int steps(int x) const { return pair ? pages() : (pages() + 1 - x) / 2; }
    __device__ __forceinline__ int page_of(int x, int i) const { return pair ? i : 2 * i + x; }
};

// Values that are not finite were left out of the products: the columns [c0, c1) of a row that sees some become their sum, which the
// rest of the row's sum does not change, be their weights ever so small. (In pages that every row sees they go through the products, and
// an infinite one gives NaN where its weight has become 0.) To dst (the row's result) or, if that is null, to its part.
__device__ __noinline__ void mend_row(const TreeArgs& a, const Walk& w, const uint32_t* words, int pos, int open_lo, const bf16* v_store,
                                      int c0, int c1, bf16* dst, float* part, int row) {
    for (int c = c0; c < c1; c++) {
        float sum = 0.f;
        for (int j = w.p0; j < w.p1; j++) {
            const int key0 = (w.sq.first_page + j) * BN, page = w.pt[j];
            if (page < 0 || page >= a.n_pages || (key0 + BN <= w.sq.pos0 && key0 >= open_lo)) continue;
            for (uint64_t left = tree_mask(a, w.sq, words, pos, key0); left; left &= left - 1) {
                const float x = __bfloat162float(v_store[kv_offset(page, a.nkv, w.kvh, __ffsll((long long)left) - 1, HD) + c]);
                if (!isfinite(x)) sum += x;
            }
        }
        if (sum == 0.f) continue;
        if (dst != nullptr) dst[c] = __float2bfloat16_rn(sum);
        else part[part_at(2 * BM, row, c)] = sum;
    }
}

// A place in a ring of N barriers, whose slots complete a phase at every turn.
template <int N>
struct Ring {
    uint32_t slot = 0, phase = 0;
    __device__ __forceinline__ void advance(uint32_t by = 1) {
        slot += by;
        while (slot >= N) slot -= N, phase ^= 1;
    }
    __device__ __forceinline__ uint32_t ahead(uint32_t by) const { return (slot + by) % N; }
};

// grid SMs, 384 threads. q as [rows][heads][HD] (map_q), map_k / map_v over one layer's store as [pages * nkv * 64, HD].
__global__ void __launch_bounds__(THREADS, 1)
tree_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
               const __grid_constant__ TreeArgs a, bf16* out, long long ldo, const bf16* v_store, float* ws_acc, float2* ws_ml, int* err) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
    const uint32_t q_s = smem_u32(smem), k_s = q_s + RING, v_s = q_s + V_RING;
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + BARS);
    uint64_t *k_full = bars, *k_free = k_full + NK, *v_full = k_free + NK, *v_free = v_full + NV;
    uint64_t *v_fine = v_free + NV;                                                          // looked over
    uint64_t *s_full = v_fine + NV, *p_full = s_full + 4, *o_full = p_full + 4;              // [stream][step & 1]
    uint64_t *q_full = o_full + 4, *q_free = q_full + 1, *o_free = q_full + 2, *both = q_full + 3;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + N_BARS);
    volatile int* odd_tile = reinterpret_cast<volatile int*>(bars + N_BARS + 1);       // [tile % MARKS]: the last one with a value that is not finite
    float2* ml_s = reinterpret_cast<float2*>(smem + ML);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, G = a.nh / a.nkv;

    pdl_wait();
    if (threadIdx.x < N_BARS) {
        uint64_t* b = bars + threadIdx.x;
        const bool two = (b >= k_free && b < v_full) || (b >= v_free && b < v_fine) || b == q_free;     // both streams say so
        mbar_init(b, b >= p_full && b < o_full ? BM : b == o_free ? SOFT + 2 : b == both ? SOFT : two ? 2 : 1);
        if (threadIdx.x < MARKS) odd_tile[threadIdx.x] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == MMA_WARP) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(TMEM_ALLOC)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    Walk w;
    w.begin(a);
    fence_before();
    __syncthreads();
    fence_after();
    pdl_launch_dependents();       // not before every block holds its tensor memory: the next kernel's blocks may want some too
    const uint32_t tmem = *tmem_slot;
    const uint32_t t_s = tmem, t_o = tmem + 4 * BN;        // S (and P over it) of [stream][step & 1], BN columns each; O of [stream], 128 each

    if (warp == LOAD_WARP) {
        if (lane == 0 && !DK_STALLED) {  // --------------------------------------------------- every TMA
            uint32_t tile = 0, laps_k = 0, laps_v = 0;     // tiles before; pages asked for, up to a ring's length
            Ring<NK> rk;
            Ring<NV> rv;
            bool ok = true;
            auto load = [&](const CUtensorMap* map, uint32_t dst, uint64_t* bar, int j) {
                mbar_expect_tx(bar, KV_BYTES);
                int page = w.pt[w.p0 + j];
                if (page < 0 || page >= a.n_pages) page = 0;           // any page will do: its keys are masked
                const int row = (page * a.nkv + w.kvh) * DK_PAGE;
                for (int hh = 0; hh < HALVES; hh++) tma_load_2d(dst + hh * KV_ATOM_BYTES, map, hh * 64, row, bar);
            };
            for (; ok && w.next(a); tile++) {
                const int n = w.pages(), boxes = w.pair ? 2 : 1;
                if (tile > 0 && !mbar_wait(q_free, (tile - 1) & 1)) { ok = false; break; }
                mbar_expect_tx(q_full, boxes * HALVES * a.half_nodes * G * 128);
                for (int x = 0; x < boxes; x++)
                    for (int hh = 0; hh < HALVES; hh++)
                        tma_load_3d(q_s + x * Q_BYTES + hh * Q_ATOM_BYTES, &map_q, hh * 64, w.kvh * G, w.sq.flat0 + w.node0 + x * a.half_nodes, q_full);
                for (int j = 0; j < n + 2 && ok; j++) {
                    if (j < n) {
                        if (laps_k == NK && !mbar_wait(k_free + rk.slot, rk.phase ^ 1)) { ok = false; break; }
                        laps_k = min(laps_k + 1, (uint32_t)NK);
                        load(&map_k, k_s + rk.slot * KV_BYTES, k_full + rk.slot, j);
                        rk.advance();
                    }
                    if (j >= 2) {
                        if (laps_v == NV && !mbar_wait(v_free + rv.slot, rv.phase ^ 1)) { ok = false; break; }
                        laps_v = min(laps_v + 1, (uint32_t)NV);
                        load(&map_v, v_s + rv.slot * KV_BYTES, v_full + rv.slot, j - 2);
                        rv.advance();
                    }
                }
            }
            if (!ok) atomicExch(err, 23);
        }
    } else if (warp == CHECK_WARP) {  // ----------------------------------------------- pages that some row does not see all of
        uint32_t tile = 0;
        Ring<NV> rv;
        bool ok = !DK_STALLED;
        for (; ok && w.next(a); tile++) {
            const int open_lo = open_from(a, w.sq);
            for (int j = w.p0; j < w.p1 && ok; j++, rv.advance()) {
                const int key0 = (w.sq.first_page + j) * BN, page = w.pt[j];
                ok = __all_sync(0xffffffffu, mbar_wait(v_full + rv.slot, rv.phase));
                if (!ok) break;
                if (!(key0 + BN <= w.sq.pos0 && key0 >= open_lo && page >= 0 && page < a.n_pages)) {
                    uint4* vs = reinterpret_cast<uint4*>(smem + V_RING + rv.slot * KV_BYTES);
                    bool odd = false;
#pragma unroll 4
                    for (int k = lane; k < KV_BYTES / 16; k += 32) {
                        uint4 val = vs[k];
                        if (no_number(val.x) | no_number(val.y) | no_number(val.z) | no_number(val.w)) {
                            vs[k] = make_uint4(numbers_of(val.x), numbers_of(val.y), numbers_of(val.z), numbers_of(val.w));
                            odd = true;
                        }
                    }
                    if (odd) {
                        odd_tile[tile % MARKS] = (int)tile + 1;
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    }
                    __syncwarp();
                }
                if (lane == 0) mbar_arrive(v_fine + rv.slot);
            }
        }
        if (!ok && lane == 0) atomicExch(err, 23);
    } else if (warp >= MMA_WARP) {
        if (lane == 0) {  // ------------------------------------------------------------ a stream's tcgen05.mma
            // (One thread for both streams: a step of the two took 3,300 clocks, of which it was busy issuing for 2,100.)
            const int x = warp - MMA_WARP;
            const uint64_t dq = desc_k_major(q_s), dk = desc_k_major(k_s), dv = desc_n_major(v_s);
            uint64_t *bar_s = s_full + 2 * x, *bar_p = p_full + 2 * x, *bar_o = o_full + 2 * x;
            const uint32_t t_sx = t_s + 2 * x * BN, t_ox = t_o + x * 128;
            uint32_t tile = 0, done = 0;                   // tiles and steps before
            Ring<NK> rk;                                   // the next page to be seen
            Ring<NV> rv;
            bool ok = true;
            for (; ok && w.next(a); tile++) {
                const int n = w.steps(x);
                const uint64_t dqx = dq + (uint64_t)((w.pair ? x * Q_BYTES : 0) >> 4);
                // Both streams see every page come in, one after the other: a wait tells its phase from the one before by a bit alone,
                // so no phase may be left out. A page that only the other stream reads is given back as soon as it has come.
                int k_next = 0, v_next = 0;
                auto see = [&](uint64_t* full, uint64_t* free, auto& ring, int& next, int upto) {
                    for (; next < upto; next++) {
                        if (!mbar_wait(full + ring.slot, ring.phase)) return false;
                        mbar_arrive(free + ring.slot);
                        ring.advance();
                    }
                    return true;
                };
                auto have_k = [&](int i) {                 // the keys of step i are here
                    return see(k_full, k_free, rk, k_next, w.page_of(x, i)) && mbar_wait(k_full + rk.slot, rk.phase);
                };
                auto issue_s = [&](int i) {
                    const uint32_t b = (done + i) & 1;
                    const uint64_t dkt = dk + (uint64_t)((rk.slot * KV_BYTES) >> 4);
#pragma unroll
                    for (int hh = 0; hh < HALVES; hh++)
#pragma unroll
                        for (int k = 0; k < 4; k++)
                            umma_ss(t_sx + b * BN, dqx + (uint64_t)((hh * Q_ATOM_BYTES + k * 32) >> 4),
                                    dkt + (uint64_t)((hh * KV_ATOM_BYTES + k * 32) >> 4), IDESC_S, (hh | k) != 0);
                    umma_commit(bar_s + b);
                    umma_commit(k_free + rk.slot);
                    if (i + 1 == n) umma_commit(q_free);
                    rk.advance(), k_next++;
                };
                ok = mbar_wait(q_full, tile & 1);
                if (ok && n == 0) umma_commit(q_free);     // one page only: nothing for B
                for (int i = 0; i < min(n, 2) && ok; i++) {
                    ok = have_k(i);
                    if (ok) fence_after(), issue_s(i);
                }
                // the rows of the tile before have been read out of O
                if (ok && tile > 0) ok = mbar_wait(o_free, (tile - 1) & 1);
                for (int i = 0; i < n && ok; i++) {
                    const uint32_t step = done + i, b = step & 1;
                    if (!see(v_fine, v_free, rv, v_next, w.page_of(x, i)) || !mbar_wait(v_fine + rv.slot, rv.phase)) { ok = false; break; }
                    // all that both products wait for, so that they go out in one run
                    if (i + 2 < n && !have_k(i + 2)) { ok = false; break; }
                    if (!mbar_wait(bar_p + b, (step >> 1) & 1)) { ok = false; break; }
                    fence_after();
                    const uint64_t dvt = dv + (uint64_t)((rv.slot * KV_BYTES) >> 4);
#pragma unroll
                    for (int k = 0; k < BN / 16; k++)
                        umma_ts(t_ox, t_sx + b * BN + k * 8, dvt + (uint64_t)((k * 16 * 128) >> 4), IDESC_PV, (i | k) != 0);   // the first overwrites O
                    umma_commit(bar_o + b);
                    umma_commit(v_free + rv.slot);
                    rv.advance(), v_next++;
                    // into the buffer whose P was just used: products of one thread run in order
                    if (i + 2 < n) issue_s(i + 2);
                }
                if (ok) ok = see(k_full, k_free, rk, k_next, w.pages()) && see(v_fine, v_free, rv, v_next, w.pages());
                mbar_arrive(o_free);                       // the tile is not over before this thread has seen the last one's end
                done += n;
            }
            if (!ok) atomicExch(err, 21);
        }
    } else {  // ------------------------------------------------------------------ softmax, a thread a row of a stream
        const int x = warp >> 2, r = threadIdx.x & (BM - 1);
        const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16, t_sx = t_s + lane_off + 2 * x * BN, t_ox = t_o + lane_off + x * 128;
        uint64_t *bar_s = s_full + 2 * x, *bar_p = p_full + 2 * x, *bar_o = o_full + 2 * x;
        uint32_t tile = 0, done = 0, shared_tiles = 0;
        bool ok = true;
        for (; ok && w.next(a); tile++) {
            const TreeSeq& sq = w.sq;
            const int n = w.steps(x), first = w.node0 + (w.pair && x ? a.half_nodes : 0);
            const int rows = min(w.node0 + w.nodes - first, a.half_nodes) * G, node = sq.flat0 + first + r / G, mark = (int)tile + 1;
            const int qpos = r < rows ? a.row_pos[node] : -1;
            const bool valid = qpos >= 0;
            const uint32_t* words = a.tree + (size_t)(r < rows ? node : sq.flat0) * a.words;
            const bool any_row = (warp & 3) * 32 < rows;               // else the warp has no row of the tile
            const int open_lo = open_from(a, sq);
            // the places that the row sees in its sequence's last two pages, worked out while the first scores are on their way
            const int tail = max(w.p0, min(w.p1, sq.pages - 2));
            uint64_t seen_tail[2] = {0, 0};
#pragma unroll
            for (int k = 0; k < 2; k++)
                if (tail + k < w.p1 && valid) seen_tail[k] = tree_mask(a, sq, words, qpos, (sq.first_page + tail + k) * BN);
            float m = -INFINITY, l = 0.f;
            int next_page = n > 0 ? w.pt[w.p0 + w.page_of(x, 0)] : 0;
            for (int i = 0; i < n && ok; i++) {
                const uint32_t step = done + i, b = step & 1, ph = (step >> 1) & 1;
                const int j = w.p0 + w.page_of(x, i), key0 = (sq.first_page + j) * BN, page = next_page;
                if (i + 1 < n) next_page = w.pt[w.p0 + w.page_of(x, i + 1)];
                const bool held = page >= 0 && page < a.n_pages;
                const bool open = held && key0 + BN <= sq.pos0 && key0 >= open_lo;
                uint64_t seen = ~0ull;
                if (!open) seen = !held || !valid ? 0ull : j >= tail ? seen_tail[j - tail ? 1 : 0] : tree_mask(a, sq, words, qpos, key0);
                if (!mbar_wait(bar_s + b, ph)) { ok = false; break; }
                if (any_row) {
                    __syncwarp();
                    fence_after();
                    uint32_t v[BN];
#pragma unroll
                    for (int c = 0; c < BN; c += 32) tmem_ld32(t_sx + b * BN + c, *reinterpret_cast<uint32_t(*)[32]>(v + c));
                    tmem_wait_ld();
                    float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                    if (!open) {
                        const uint32_t half[2] = {(uint32_t)seen, (uint32_t)(seen >> 32)};
#pragma unroll
                        for (int k = 0; k < BN; k++)
                            if (!(half[k / 32] >> (k % 32) & 1)) v[k] = 0xff800000u;           // -infinity
                    }
#pragma unroll
                    for (int k = 0; k < BN; k += 2) mx4[(k >> 1) & 3] = max3(mx4[(k >> 1) & 3], __uint_as_float(v[k]), __uint_as_float(v[k + 1]));
                    const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * a.sl2;   // sl2 > 0: scaling keeps the order
                    float m_new = fmaxf(m, mx);
                    // a maximum that moved by less than 8 (a factor 256) keeps the old reference: O need not be rescaled
                    if (m != -INFINITY && m_new - m < 8.f) m_new = m;
                    const float ms = m_new == -INFINITY ? 0.f : m_new;
                    const float alpha = m_new == m ? 1.f : ex2(m - ms);
                    if (i > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
                        if (!mbar_wait(bar_o + (b ^ 1), ((step - 1) >> 1) & 1)) { ok = false; break; }
                        __syncwarp();
                        fence_after();
#pragma unroll 1
                        for (int c = 0; c < HD; c += 32) {
                            uint32_t o[32];
                            tmem_ld32(t_ox + c, o);
                            tmem_wait_ld();
#pragma unroll
                            for (int k = 0; k < 32; k++) o[k] = __float_as_uint(__uint_as_float(o[k]) * alpha);
                            tmem_st32(t_ox + c, o);
                        }
                    }
                    float2 sum2[2] = {};
                    uint32_t p[BN / 2];
                    const float2 scale2 = make_float2(a.sl2, a.sl2), minus = make_float2(-ms, -ms);
#pragma unroll
                    for (int k = 0; k < BN; k += 2) {
                        float2 e = fma2(make_float2(__uint_as_float(v[k]), __uint_as_float(v[k + 1])), scale2, minus);
                        e.x = ex2(e.x), e.y = ex2(e.y);
                        sum2[(k >> 1) & 1] = add2(sum2[(k >> 1) & 1], e);
                        __nv_bfloat162 pk = __floats2bfloat162_rn(e.x, e.y);
                        p[k / 2] = *reinterpret_cast<uint32_t*>(&pk);
                    }
                    tmem_st32(t_sx + b * BN, p);
                    l = l * alpha + (sum2[0].x + sum2[0].y) + (sum2[1].x + sum2[1].y);
                    m = m_new;
                    tmem_wait_st();
                    fence_before();
                }
                mbar_arrive(bar_p + b);
            }
            if (ok && n > 0) ok = mbar_wait(bar_o + ((done + n - 1) & 1), ((done + n - 1) >> 1) & 1);
            if (!ok) break;
            if (!valid) m = -INFINITY, l = 0.f;
            // the factors of the two streams' rows: with rows in both, the own one alone
            float mine = 1.f, other = 0.f;
            int c0 = 0, c1 = HD;
            if (!w.pair) {
                float2* ml = ml_s + (shared_tiles & 1) * 2 * BM;
                ml[x * BM + r] = make_float2(m, l);
                mbar_arrive(both);
                if (!mbar_wait(both, shared_tiles & 1)) { ok = false; break; }
                shared_tiles++;
                const float2 o = ml[(1 - x) * BM + r];
                const float mn = fmaxf(m, o.x), ms = mn == -INFINITY ? 0.f : mn;
                mine = ex2(m - ms), other = ex2(o.x - ms);
                l = l * mine + o.y * other, m = mn;
                c0 = x * (HD / 2), c1 = c0 + HD / 2;                   // each stream's thread writes half the row
            }
            if (any_row) {
                __syncwarp();
                fence_after();
                const bool whole = w.all(), mend = odd_tile[tile % MARKS] == mark, has = n > 0, has_other = !w.pair && w.steps(1 - x) > 0;
                const float inv = l == 0.f ? 0.f : 1.f / l;
                const size_t slot = (size_t)w.slot() * 2 * BM;
                const int row = (w.pair ? x * BM : 0) + r;
                bf16* dst = out + (size_t)node * ldo + (size_t)(w.kvh * G + r % G) * HD;
                if (!whole && r < rows && c0 == 0) ws_ml[slot + row] = make_float2(m, l);
#pragma unroll 1
                for (int c = c0; c < c1; c += OC) {
                    uint32_t o[OC], o2[OC];
                    __syncwarp();
                    if (has) tmem_ld16(t_ox + c, o);
                    if (has_other) tmem_ld16(t_o + lane_off + (1 - x) * 128 + c, o2);
                    tmem_wait_ld();
#pragma unroll
                    for (int k = 0; k < OC; k++)
                        o[k] = __float_as_uint((has ? __uint_as_float(o[k]) * mine : 0.f) + (has_other ? __uint_as_float(o2[k]) * other : 0.f));
                    if (r < rows) {
                        if (!valid || l == 0.f)
#pragma unroll
                            for (int k = 0; k < OC; k++) o[k] = 0;
                        if (whole) {
#pragma unroll
                            for (int k = 0; k < OC; k += 8) {
                                uint4 pk;
                                __nv_bfloat162* pp = reinterpret_cast<__nv_bfloat162*>(&pk);
#pragma unroll
                                for (int e = 0; e < 4; e++)
                                    pp[e] = __floats2bfloat162_rn(__uint_as_float(o[k + 2 * e]) * inv, __uint_as_float(o[k + 2 * e + 1]) * inv);
                                *reinterpret_cast<uint4*>(dst + c + k) = pk;
                            }
                        } else {
#pragma unroll
                            for (int k = 0; k < OC; k += 4)
                                *reinterpret_cast<uint4*>(ws_acc + slot * HD + part_at(2 * BM, row, c + k)) = make_uint4(o[k], o[k + 1], o[k + 2], o[k + 3]);
                        }
                    }
                }
                fence_before();
                if (mend && valid && l != 0.f)
                    mend_row(a, w, words, qpos, open_lo, v_store, c0, c1, whole ? dst : nullptr, ws_acc + slot * HD, row);
            }
            mbar_arrive(o_free);
            done += n;
        }
        if (!ok && lane == 0) atomicExch(err, 22);
    }
    fence_before();
    __syncthreads();
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

DK_EXPORT int dk_tree_tc_tile_rows() { return 2 * BM; }
DK_EXPORT int dk_tree_tc_whole_pages() { return WHOLE_PAGES; }

// q [n_rows, nh*HD] and out, bf16, rows ldq / ldo elements apart (multiples of 8); k_store, v_store [n_pages, nkv, 64, HD]; all on 16-byte
// boundaries; ws_acc: 2 * blocks * 256 * HD floats, ws_ml: 2 * blocks * 256 * 2 floats; err: device int for a wait that ran out.
DK_EXPORT int dk_attn_tree_tc(const void* q, long long ldq, void* out, long long ldo, long long n_rows, const void* k_store,
                              const void* v_store, int n_pages, const int* cu_q, const int* seq_pos0, const int* row_pos,
                              const uint32_t* tree, int words, const int* page_table, int pt_stride, int n_seq, int nh, int nkv, int window,
                              float scale, int max_nodes, float* ws_acc, float* ws_ml, int blocks, int* err, cudaStream_t st) {
    if (nkv < 1 || nh % nkv || nh / nkv > 64 || n_pages < 1 || pt_stride < 1 || words < 1 || blocks < 1 || max_nodes < 1 || n_seq > 65535 ||
        err == nullptr || ldq % 8 || ldo % 8 || ((uintptr_t)q | (uintptr_t)out | (uintptr_t)k_store | (uintptr_t)v_store) % 16 || (long long)n_pages * nkv * DK_PAGE > 0x7fffffffLL)
        return (int)cudaErrorInvalidValue;
    const int G = nh / nkv;
    TreeArgs a = {cu_q, seq_pos0, row_pos, page_table, tree, n_seq, words, pt_stride, n_pages, nh, nkv, window, max_nodes, 2 * (BM / G), BM / G, BM,
                  pt_stride <= WHOLE_PAGES, EXTRA, scale * 1.4426950408889634f};
    if (!tree_units_fit(a) || nkv > 65535 || (!a.whole && (ws_acc == nullptr || ws_ml == nullptr))) return (int)cudaErrorInvalidValue;
    static SmemOnce once;
    int e = once.allow((const void*)tree_tc_kernel, SMEM_BYTES);
    if (e) return e;
    CUtensorMap mq, mk, mv;
    const cuuint64_t q_dims[3] = {HD, (cuuint64_t)nh, (cuuint64_t)n_rows}, q_strides[2] = {HD * 2, (cuuint64_t)ldq * 2};
    const cuuint32_t q_box[3] = {64, (cuuint32_t)G, (cuuint32_t)(BM / G)};
    const cuuint64_t kv_dims[2] = {HD, (cuuint64_t)n_pages * nkv * DK_PAGE}, kv_strides[1] = {HD * 2};
    const cuuint32_t kv_box[2] = {64, DK_PAGE};
    e = make_map(&mq, q, 3, q_dims, q_strides, q_box);
    if (!e) e = make_map(&mk, k_store, 2, kv_dims, kv_strides, kv_box);
    if (!e) e = make_map(&mv, v_store, 2, kv_dims, kv_strides, kv_box);
    if (e) return e;
    e = dk_launch(tree_tc_kernel, dim3(blocks), dim3(THREADS), SMEM_BYTES, st, mq, mk, mv, a, (bf16*)out, ldo, (const bf16*)v_store, ws_acc,
                  (float2*)ws_ml, err);
    if (e) return e;
    return tree_merge<bf16, HD>(a, ws_acc, ws_ml, out, ldo, 2 * BM, blocks, st);
}
