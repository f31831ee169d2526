// Rows of the paged cache and fixed-size states that follow a choice among branches, in place.
//
//   kv_keep        a sequence's accepted nodes close up: row pos0 + path[k] goes to pos0 + k. The path rises, so path[k] >= k: a row
//                  goes down or stays, and whoever takes the rows in rising order has read a row before it writes over it.
//   kv_reorder     every beam of a request takes the rows [first, last) of its parent beam (parents may be one another's: a swap).
//   state_reorder  the same for the states of its parent's slot.
//
// Every thread owns a piece (16 bytes; 4 or 2 where sizes or addresses allow no more) of what it moves, at all rows of a path or in
// all beams of a request: it reads what its writes go over into registers first, so the moves need no second copy of the cache and no
// order among threads. Bound by reading and writing each moved byte once; a row that stays is not touched. A place outside the table,
// a page or slot outside the store, and a parent that is none are left out.
// Measured: four searches of four beams, 20 to 120 rows of 36 layers (8 heads of 128, bfloat16) 52.6 us (290 MB, 5.5 TB/s, 84 % of the
// copy rate); the states of 2 x 8 beams, 4 layers of 16 x 128 x 128 floats, 21.3 us (117 MB, 84 %); the paths of eight trees in 36 layers 3.7 us.
#include "common.cuh"

namespace {

constexpr int THREADS = 256, MAX_PATH = 1024, AHEAD = 8, MAX_BEAMS = 32;

// offset of a place's row within one [pages, nkv, 64, units] store, of kv head 0; -1: not held
__device__ __forceinline__ long long row_of(const int* pt, int pt_stride, int n_pages, int place, int nkv, int units) {
    if (place < 0 || place / DK_PAGE >= pt_stride) return -1;
    const int page = pt[place / DK_PAGE];
    if (page < 0 || page >= n_pages) return -1;
    return (long long)kv_offset(page, nkv, 0, place % DK_PAGE, units);
}

// grid (pieces of outer * nkv * units, sequences); a thread moves one piece at every row of its sequence's path. U: the type of a
// piece, units: pieces in a row. outer: stores one behind the other, n_pages * nkv * 64 rows each.
template <typename U>
__global__ void __launch_bounds__(THREADS)
kv_keep_kernel(U* store, int outer, int n_pages, int nkv, int units, const int* page_table, int pt_stride, const int* seq_pos0,
               const int* path, int path_stride, const int* n_path) {
    __shared__ long long from[MAX_PATH], to[MAX_PATH];
    __shared__ int moves;
    pdl_wait();
    pdl_launch_dependents();
    const int s = blockIdx.y, n = min(n_path[s], path_stride), pos0 = seq_pos0[s];
    const int* pt = page_table + (size_t)s * pt_stride;
    if (threadIdx.x < 32) {                                            // the rows that move, in order
        int k0 = 0;
        for (int b = 0; b < n; b += 32) {
            const int k = b + threadIdx.x, at = k < n ? path[(size_t)s * path_stride + k] : -1;
            const long long src = at > k ? row_of(pt, pt_stride, n_pages, pos0 + at, nkv, units) : -1;
            const long long dst = at > k ? row_of(pt, pt_stride, n_pages, pos0 + k, nkv, units) : -1;
            const bool on = src >= 0 && dst >= 0;
            const unsigned mask = __ballot_sync(0xffffffffu, on);
            const int i = k0 + __popc(mask & ((1u << threadIdx.x) - 1));
            if (on) from[i] = src, to[i] = dst;
            k0 += __popc(mask);
        }
        if (threadIdx.x == 0) moves = k0;
    }
    __syncthreads();
    const long long piece = (long long)blockIdx.x * THREADS + threadIdx.x;
    if (piece >= (long long)outer * nkv * units) return;
    const int c = (int)(piece % units), h = (int)(piece / units % nkv);
    U* base = store + (size_t)(piece / units / nkv) * n_pages * nkv * DK_PAGE * units + (size_t)h * DK_PAGE * units + c;
    const int m = moves;
    for (int k = 0; k < m; k += AHEAD) {
        U v[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; i++)
            if (k + i < m) v[i] = base[from[k + i]];
#pragma unroll
        for (int i = 0; i < AHEAD; i++)
            if (k + i < m) base[to[k + i]] = v[i];
    }
}

// grid (blocks, outer, requests): a thread moves one piece of one row in all beams
template <typename U, int NB>
__global__ void __launch_bounds__(THREADS)
kv_reorder_kernel(U* store, int n_pages, int nkv, int units, const int* page_table, int pt_stride, const int* parent, int beams,
                  const int* first, const int* last) {
    __shared__ int par[MAX_BEAMS];
    pdl_wait();
    pdl_launch_dependents();
    const int r = blockIdx.z;
    if (threadIdx.x < beams) {
        const int p = parent[r * beams + threadIdx.x];
        par[threadIdx.x] = p >= 0 && p < beams ? p : threadIdx.x;
    }
    __syncthreads();
    const int lo = max(0, first[r]);
    const long long hi = min((long long)last[r], (long long)pt_stride * DK_PAGE);
    const int* pt = page_table + (size_t)r * beams * pt_stride;
    U* base = store + (size_t)blockIdx.y * n_pages * nkv * DK_PAGE * units;
    const long long n = max(0ll, hi - lo) * nkv * units;
    for (long long i = (long long)blockIdx.x * THREADS + threadIdx.x; i < n; i += (long long)gridDim.x * THREADS) {
        // rows of one kv head one behind the other, as they lie in a page
        const int c = (int)(i % units), place = lo + (int)(i / units % (hi - lo)), h = (int)(i / units / (hi - lo));
        const size_t off = (size_t)h * DK_PAGE * units + c;
        U v[NB];
        long long at[NB];
        unsigned on = 0;
#pragma unroll
        for (int b = 0; b < NB; b++)
            if (b < beams && par[b] != b) {
                const long long src = row_of(pt + (size_t)par[b] * pt_stride, pt_stride, n_pages, place, nkv, units);
                at[b] = row_of(pt + (size_t)b * pt_stride, pt_stride, n_pages, place, nkv, units);
                if (src >= 0 && at[b] >= 0) {
                    v[b] = base[src + off];
                    on |= 1u << b;
                }
            }
#pragma unroll
        for (int b = 0; b < NB; b++)
            if (on >> b & 1) base[at[b] + off] = v[b];
    }
}

// store [entries, slots, units]; grid (blocks, entries, requests)
template <typename U, int NB>
__global__ void __launch_bounds__(THREADS)
state_reorder_kernel(U* store, int slots, long long units, const int* seq_slot, const int* parent, int beams) {
    __shared__ int src[MAX_BEAMS], dst[MAX_BEAMS];
    pdl_wait();
    pdl_launch_dependents();
    const int r = blockIdx.z;
    if (threadIdx.x < beams) {
        const int p = parent[r * beams + threadIdx.x], to = seq_slot[r * beams + threadIdx.x];
        const int of = p >= 0 && p < beams ? seq_slot[r * beams + p] : to;
        const bool on = of != to && of >= 0 && of < slots && to >= 0 && to < slots;
        src[threadIdx.x] = on ? of : -1, dst[threadIdx.x] = to;
    }
    __syncthreads();
    U* base = store + (size_t)blockIdx.y * slots * units;
    for (long long i = (long long)blockIdx.x * THREADS + threadIdx.x; i < units; i += (long long)gridDim.x * THREADS) {
        U v[NB];
#pragma unroll
        for (int b = 0; b < NB; b++)
            if (b < beams && src[b] >= 0) v[b] = base[(size_t)src[b] * units + i];
#pragma unroll
        for (int b = 0; b < NB; b++)
            if (b < beams && src[b] >= 0) base[(size_t)dst[b] * units + i] = v[b];
    }
}

int sm_count() {
    int sms = 0, dev = 0;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    return sms;
}

// Bytes of a piece: rows (or states) and the address are multiples of it
int piece_bytes(const void* p, long long bytes) {
    const uintptr_t x = (uintptr_t)p | (uintptr_t)bytes;
    return x % 16 == 0 ? 16 : x % 4 == 0 ? 4 : 2;
}

template <typename U>
int keep(void* store, int outer, int n_pages, int nkv, long long row_bytes, const int* page_table, int pt_stride, int n_seq,
         const int* seq_pos0, const int* path, int path_stride, const int* n_path, cudaStream_t st) {
    const long long units = row_bytes / (long long)sizeof(U);
    const long long blocks = ((long long)outer * nkv * units + THREADS - 1) / THREADS;
    return dk_launch(kv_keep_kernel<U>, dim3((unsigned)blocks, n_seq), dim3(THREADS), 0, st, (U*)store, outer, n_pages, nkv, (int)units,
                     page_table, pt_stride, seq_pos0, path, path_stride, n_path);
}

template <typename U, int NB>
int kv(void* store, int outer, int n_pages, int nkv, long long row_bytes, const int* page_table, int pt_stride, int requests, int beams,
       const int* parent, const int* first, const int* last, cudaStream_t st) {
    const int units = (int)(row_bytes / (long long)sizeof(U));
    // the rows' number is on the device: 16 blocks an SM over all stores and requests (52.4 us for 36 layers of four searches, 54.3 with 8, 55.0
    // with 64), no more than a page table can need
    const long long most = ((long long)pt_stride * DK_PAGE * nkv * units + THREADS - 1) / THREADS;
    long long blocks = (16LL * sm_count() + (long long)outer * requests - 1) / ((long long)outer * requests);
    blocks = blocks < most ? blocks : most;
    return dk_launch(kv_reorder_kernel<U, NB>, dim3((unsigned)blocks, outer, requests), dim3(THREADS), 0, st, (U*)store, n_pages, nkv, units,
                     page_table, pt_stride, parent, beams, first, last);
}

template <typename U, int NB>
int state(void* store, int entries, int slots, long long bytes, const int* seq_slot, int requests, int beams, const int* parent,
          cudaStream_t st) {
    const long long units = bytes / (long long)sizeof(U), most = (units + THREADS - 1) / THREADS;
    long long blocks = (16LL * sm_count() + (long long)entries * requests - 1) / ((long long)entries * requests);
    blocks = blocks < most ? blocks : most;
    return dk_launch(state_reorder_kernel<U, NB>, dim3((unsigned)blocks, entries, requests), dim3(THREADS), 0, st, (U*)store, slots, units,
                     seq_slot, parent, beams);
}

}  // namespace

// DK_BY_BEAMS(f<U>): the smallest of 4, 8, 16 and 32 registers of beams that holds them
#define DK_BY_BEAMS(F, U, ...) \
    (beams <= 4 ? F<U, 4>(__VA_ARGS__) : beams <= 8 ? F<U, 8>(__VA_ARGS__) : beams <= 16 ? F<U, 16>(__VA_ARGS__) : F<U, 32>(__VA_ARGS__))

// store: `outer` stores [n_pages, nkv, 64, row_bytes]; path [n_seq, path_stride], n_path [n_seq]
DK_EXPORT int dk_kv_keep(void* store, int outer, int n_pages, int nkv, long long row_bytes, const int* page_table, int pt_stride, int n_seq,
                         const int* seq_pos0, const int* path, int path_stride, const int* n_path, cudaStream_t st) {
    if (outer < 1 || n_pages < 1 || nkv < 1 || row_bytes < 2 || row_bytes % 2 || pt_stride < 1 || n_seq < 1 || n_seq > 65535 ||
        path_stride < 1 || path_stride > MAX_PATH)
        return (int)cudaErrorInvalidValue;
    const int p = piece_bytes(store, row_bytes);
#define DK_KEEP(U) keep<U>(store, outer, n_pages, nkv, row_bytes, page_table, pt_stride, n_seq, seq_pos0, path, path_stride, n_path, st)
    return p == 16 ? DK_KEEP(uint4) : p == 4 ? DK_KEEP(uint32_t) : DK_KEEP(uint16_t);
#undef DK_KEEP
}

// page_table [requests * beams, pt_stride], parent [requests, beams], first, last [requests]
DK_EXPORT int dk_kv_reorder(void* store, int outer, int n_pages, int nkv, long long row_bytes, const int* page_table, int pt_stride,
                            int requests, int beams, const int* parent, const int* first, const int* last, cudaStream_t st) {
    if (outer < 1 || outer > 65535 || n_pages < 1 || nkv < 1 || row_bytes < 2 || row_bytes % 2 || pt_stride < 1 || requests < 1 ||
        requests > 65535 || beams < 1 || beams > MAX_BEAMS)
        return (int)cudaErrorInvalidValue;
    const int p = piece_bytes(store, row_bytes);
#define DK_KV(U) DK_BY_BEAMS(kv, U, store, outer, n_pages, nkv, row_bytes, page_table, pt_stride, requests, beams, parent, first, last, st)
    return p == 16 ? DK_KV(uint4) : p == 4 ? DK_KV(uint32_t) : DK_KV(uint16_t);
#undef DK_KV
}

// store [entries, slots, bytes], seq_slot [requests * beams], parent [requests, beams]
DK_EXPORT int dk_state_reorder(void* store, int entries, int slots, long long bytes, const int* seq_slot, int requests, int beams,
                               const int* parent, cudaStream_t st) {
    if (entries < 1 || entries > 65535 || slots < 1 || bytes < 2 || bytes % 2 || requests < 1 || requests > 65535 || beams < 1 ||
        beams > MAX_BEAMS)
        return (int)cudaErrorInvalidValue;
    const int p = piece_bytes(store, bytes);
#define DK_STATE(U) DK_BY_BEAMS(state, U, store, entries, slots, bytes, seq_slot, requests, beams, parent, st)
    return p == 16 ? DK_STATE(uint4) : p == 4 ? DK_STATE(uint32_t) : DK_STATE(uint16_t);
#undef DK_STATE
}
