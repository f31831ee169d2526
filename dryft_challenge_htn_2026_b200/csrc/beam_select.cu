// The best continuations of a request's beams, over all beams and the whole vocabulary.
//
//   value(b, v) = score[b] + logit[b, v] - log(sum_u exp(logit[b, u]))
//
// and the `best` largest values, ties by the lower beam, then the lower token. A logit that is not finite is no candidate and weighs
// nothing; a beam whose score is not finite is not live and brings none; a beam at its end brings one, its own score with token 0.
// Where there are fewer candidates than asked for, the rest is (-infinity, 0, 0).
//
// Within a beam the order of the values is that of the logits, so a piece of a row can give up all but its `best` largest logits
// before the row's sum is known: one pass over the logits. Across beams the logarithms of the sums decide: exponentials in float32 of the
// logit's distance to the piece's maximum (subtracted before it is scaled: exact where the weight is, finite for every finite logit, and the
// same whatever is added to all logits of a row), added up in float32 within a thread and in double from there on, values compared in
// double, so that a rank does not hang on the rounding of the scores (float32 scores around -30 are 2^-19 apart).
//
// First launch, a block a piece of 8,192 logits of a row, which stay in registers. A floor under the `best`-th largest: of each warp
// the best / 8-th largest of its threads' own maxima, the least of these; few logits beside the ones looked for reach it, and these
// are ranked by counting. Where many do (equal logits, a warp without large ones), the exact `best`-th largest of the threads' maxima
// takes its place, above which `best` threads have all there is. (That one alone, 256 comparisons a thread, took two thirds of the
// kernel's time: 47 us for 128 rows of 100,003.) Second launch, a block a request: the same over the pieces' lists, which are in order.
//
// Measured: four beams over 151,936 tokens 8.7 us, 16 x 8 beams over 100,003 tokens 25.3 us (51 MB, 7.8 us at the copy rate), 16 x 8
// over 200,003 36.3: about 14 us of latency (a block's load, its rounds of barriers, the second launch) and 4.6 TB/s above that. Threads
// with 16 logits, twice as many a block, have looser floors (35 us, when this form took 24.8); 5 or 6 blocks an SM with fewer registers were
// no faster (25.3, 26.8).
#include "logit_rows.cuh"

namespace {

constexpr int THREADS = 256, WARPS = THREADS / 32, EACH = 32, MAX_BEST = 64, MAX_BEAMS = 32;
constexpr int ROOM = 512;                                               // logits that are ranked at once under the quick floor
typedef LogitPiece<THREADS, EACH> Piece;

// Larger key: larger logit, then lower index. 0: none.
__device__ __forceinline__ uint32_t order_of(float v) {
    const uint32_t b = __float_as_uint(v + 0.f);                         // -0 counts as 0
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ uint64_t key_of(float v, int i) { return isfinite(v) ? (uint64_t)order_of(v) << 32 | (uint32_t)~i : 0; }
__device__ __forceinline__ float value_of_order(uint32_t b) { return __uint_as_float(b & 0x80000000u ? b & 0x7fffffffu : ~b); }
__device__ __forceinline__ float logit_of(uint64_t key) { return value_of_order((uint32_t)(key >> 32)); }
__device__ __forceinline__ int index_of(uint64_t key) { return (int)~(uint32_t)key; }

constexpr float LOG2E = 1.4426950408889634f;
// 2^x, one instruction (-infinity gives 0)
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// grid (pieces, rows). ws_key [rows][pieces][best] in falling order (0: none), ws_sum [rows][pieces] = (maximum, sum).
__global__ void __launch_bounds__(THREADS)
beam_pieces_kernel(const float* logits, int V, int best, uint64_t* ws_key, double2* ws_sum) {
    __shared__ uint64_t tops[THREADS], exact_floor;
    __shared__ uint64_t found[MAX_BEST * EACH];
    __shared__ float red_m[WARPS], floors[WARPS];
    __shared__ double red_s[WARPS];
    __shared__ int count;
    pdl_wait();
    const int t = threadIdx.x, lane = t & 31, w = t >> 5;
    const float* z = logits + (size_t)blockIdx.y * V;
    const Piece piece(z, blockIdx.x);
    float v[EACH];
    piece.load(z, V, v);
    uint32_t bits = 0;                                                   // the thread's logits that reach the floor
    for (bool again = false;; again = true) {
        if (t == 0) count = 0, exact_floor = 1;
        float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int k = 0; k < EACH; k++) m4[k & 3] = fmaxf(m4[k & 3], v[k]);
        const float top = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
        // the warp's largest, and its floor: its threads' largest ones, one after the other
        uint32_t left = order_of(top), high = 0;
        float wm = 0.f;
        for (int r = 0; r < (best + WARPS - 1) / WARPS; r++) {
            high = __reduce_max_sync(0xffffffffu, left);
            if (r == 0) wm = value_of_order(high);
            if (lane == __ffs(__ballot_sync(0xffffffffu, left == high)) - 1) left = 0;
        }
        if (lane == 0) red_m[w] = wm, floors[w] = high ? value_of_order(high) : -INFINITY;
        __syncthreads();
        float bm = red_m[0], low = floors[0];
#pragma unroll
        for (int i = 1; i < WARPS; i++) bm = fmaxf(bm, red_m[i]), low = fminf(low, floors[i]);
        low = fmaxf(low, -3.402823466e38f);                             // -infinity is no candidate
        auto reach = [&](float least) {
            uint32_t b = 0;
#pragma unroll
            for (int k = 0; k < EACH; k++) b |= v[k] >= least ? 1u << k : 0u;
            return b;
        };
        bits = top >= low ? reach(low) : 0;
        if (bits) atomicAdd(&count, __popc(bits));
        float sum = 0.f;
        if (bm > -INFINITY)
#pragma unroll
            for (int k = 0; k < EACH; k++) sum += ex2((v[k] - bm) * LOG2E);
        double total = sum;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
        if (lane == 0) red_s[w] = total;
        __syncthreads();
        total = 0.;
#pragma unroll
        for (int i = 0; i < WARPS; i++) total += red_s[i];
        // an infinite logit, or one that is none, shows in the sum: once more without it
        if (!again && !(total < INFINITY)) {
#pragma unroll
            for (int k = 0; k < EACH; k++)
                if (!(fabsf(v[k]) < INFINITY)) v[k] = -INFINITY;
            __syncthreads();
            continue;
        }
        if (t == 0) ws_sum[(size_t)blockIdx.y * gridDim.x + blockIdx.x] = make_double2((double)bm, total);
        if (count > ROOM) {                                              // the best-th largest of the threads' largest, each the first of its kind
            int at = 0;
#pragma unroll
            for (int k = EACH - 1; k >= 0; k--)
                if (v[k] == top) at = k;
            const uint64_t key = key_of(top, piece.index(at));
            tops[t] = key;
            __syncthreads();
            int above = 0;
#pragma unroll 4
            for (int i = 0; i < THREADS; i++) above += tops[i] > key;
            if (key != 0 && above == best - 1) exact_floor = key;
            __syncthreads();
            bits = key >= exact_floor ? reach(exact_floor == 1 ? low : logit_of(exact_floor)) : 0;
        }
        break;
    }
    const uint64_t floor_key = exact_floor;                              // 1 without the exact one: all that `bits` says
    __syncthreads();
    if (t == 0) count = 0;
    __syncthreads();
    for (; bits; bits &= bits - 1) {                                     // few have any: they are read again
        const int i = piece.index(__ffs(bits) - 1);
        const uint64_t key = key_of(z[i], i);
        if (key >= floor_key) found[atomicAdd(&count, 1)] = key;
    }
    __syncthreads();
    const int n = count;
    uint64_t* out = ws_key + ((size_t)blockIdx.y * gridDim.x + blockIdx.x) * best;
    for (int i = t; i < n; i += THREADS) {
        const uint64_t key = found[i];
        int rank = 0;
#pragma unroll 4
        for (int j = 0; j < n; j++) rank += found[j] > key;
        if (rank < best) out[rank] = key;
    }
    for (int i = n + t; i < best; i += THREADS) out[i] = 0;
    // the second launch's blocks come in as these leave: called at the start, they stood in the way of blocks still to come (16 searches
    // of 8 beams: 33 us instead of 25)
    pdl_launch_dependents();
}

// A value in double, in the order of its bits, and its place among all beams' tokens; place -1: none.
struct Candidate {
    uint64_t order;
    int flat;
    // (without a branch: with two of them a comparison in the loops below took a hundred clocks)
    __device__ __forceinline__ bool before(const Candidate& o) const { return (order > o.order) | ((order == o.order) & ((unsigned)flat < (unsigned)o.flat)); }
};
__device__ __forceinline__ Candidate candidate(double value, int flat) {
    const uint64_t b = (uint64_t)__double_as_longlong(value + 0.);
    return Candidate{b >> 63 ? ~b : b | 1ull << 63, flat};
}
__device__ __forceinline__ double value_of(const Candidate& c) {
    return __longlong_as_double((long long)(c.order >> 63 ? c.order & ~(1ull << 63) : ~c.order));
}

constexpr int KEYS = 4096;                                              // keys that are brought into shared memory at once, if there are no more

// The sum of a block's numbers, in all threads. red: WARPS numbers of shared memory.
__device__ __forceinline__ int block_sum(int n, int* red) {
    n = __reduce_add_sync(0xffffffffu, n);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = n;
    __syncthreads();
    n = 0;
#pragma unroll
    for (int i = 0; i < WARPS; i++) n += red[i];
    return n;
}

// The best-th candidate of all lists (or one that all stand before, where there are fewer), found bit by bit: its value, then its place
// among those of that value. counted(c): how many stand before c or are it.
template <typename F>
__device__ __forceinline__ Candidate best_th(int best, const F& counted) {
    Candidate c = {0, 0x7fffffff};
    for (int bit = 63; bit >= 0; bit--) {
        const Candidate mid = {c.order | 1ull << bit, 0x7fffffff};
        const int n = counted(mid);
        if (n == best) return mid;
        if (n > best) c.order = mid.order;
    }
    if (c.order == 0) return c;                                          // fewer than asked for
    c.flat = 0;
    for (int bit = 30; bit >= 0; bit--)
        if (counted(Candidate{c.order, (c.flat | 1 << bit) - 1}) < best) c.flat |= 1 << bit;
    return c;
}

// grid (requests). Dynamic shared memory: best * best * ceil(lists / THREADS) candidates, then the keys where they are KEYS at most. MANY:
// where that is more than a block has (32 beams and 64 results from 25 pieces on): `best` candidates, which best_th has counted off before
// they are taken: up to 95 looks at the lists instead of one (32 beams over 200,003 tokens, 64 results: 137 us a call; over 190,000 27).
template <bool MANY>
__global__ void __launch_bounds__(THREADS)
beam_select_kernel(const uint64_t* ws_key, const double2* ws_sum, int pieces, int V, int beams, int best, const float* scores,
                   const int* ended, float* scores_out, int* beam_out, int* tok_out) {
    extern __shared__ __align__(16) unsigned char dyn[];
    Candidate* found = reinterpret_cast<Candidate*>(dyn);
    __shared__ Candidate tops[MANY ? 1 : THREADS], least;
    __shared__ int red[WARPS];
    __shared__ double highest[MAX_BEAMS], offset[MAX_BEAMS];            // a live beam: its largest logit, score - log(sum) against that
    __shared__ int kind[MAX_BEAMS];                                      // 0: not live, 1: live, 2: at its end
    __shared__ int count;
    const Candidate none = {0, -1};
    pdl_wait();
    pdl_launch_dependents();
    const int r = blockIdx.x, t = threadIdx.x, lane = t & 31, w = t >> 5;
    const int lists = beams * pieces;
    const uint64_t* keys = ws_key + (size_t)r * lists * best;
    if (!MANY && lists * best <= KEYS) {
        uint64_t* here = reinterpret_cast<uint64_t*>(found + best * best * ((lists + THREADS - 1) / THREADS));
#pragma unroll 8
        for (int i = t; i < lists * best; i += THREADS) here[i] = keys[i];
        keys = here;
    }
    for (int b = w; b < beams; b += WARPS) {
        const double2* part = ws_sum + (size_t)(r * beams + b) * pieces;
        const float score = scores[r * beams + b];
        const bool done = ended != nullptr && ended[r * beams + b] != 0;
        double m = -INFINITY, sum = 0.;
        for (int c0 = 0; c0 < pieces; c0 += 32) {                        // 32 pieces at a time, one after the other into (m, sum)
            const double2 p = c0 + lane < pieces ? part[c0 + lane] : make_double2(-INFINITY, 0.);
            double top = p.x;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) top = fmax(top, __shfl_xor_sync(0xffffffffu, top, o));
            const double mn = fmax(m, top);
            double add = p.y > 0. ? p.y * exp(p.x - mn) : 0.;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) add += __shfl_xor_sync(0xffffffffu, add, o);
            sum = (sum > 0. ? sum * exp(m - mn) : 0.) + add, m = mn;
        }
        if (lane == 0) {
            kind[b] = !isfinite(score) ? 0 : done ? 2 : sum > 0. ? 1 : 0;
            highest[b] = m, offset[b] = kind[b] == 1 ? (double)score - log(sum) : (double)score;
        }
    }
    if (t == 0) count = 0, least = none;
    __syncthreads();
    // list l: piece l % pieces of beam l / pieces, in falling order; a beam at its end has one candidate, in its first list
    auto item = [&](int l, int rank) {
        const int b = l / pieces;
        if (kind[b] == 2) return rank == 0 && l == b * pieces ? candidate(offset[b], b * V) : none;
        const uint64_t key = kind[b] == 1 ? keys[l * best + rank] : 0;
        return key ? candidate(((double)logit_of(key) - highest[b]) + offset[b], b * V + index_of(key)) : none;
    };
    Candidate low;
    bool some = true;                                                    // whether the thread's lists may hold one
    if (MANY) {
        low = best_th(best, [&](const Candidate& c) {
            int n = 0;
            for (int l = t; l < lists; l += THREADS) {
                int lo = 0, hi = best;                                   // the list's first `lo` stand before c or are it, those from hi on do not
                while (lo < hi) {
                    const int mid = lo == 0 ? 0 : (lo + hi) / 2;         // few lists hold any
                    const Candidate x = item(l, mid);
                    if (x.flat >= 0 && !c.before(x)) lo = mid + 1;
                    else hi = mid;
                }
                n += lo;
            }
            return block_sum(n, red);
        });
    } else {
        Candidate top = none;
        for (int l = t; l < lists; l += THREADS) {
            const Candidate c = item(l, 0);
            if (c.before(top)) top = c;
        }
        tops[t] = top;
        __syncthreads();
        int above = 0;
        const int n_tops = min(THREADS, lists);
#pragma unroll 8
        for (int i = 0; i < n_tops; i++) above += tops[i].before(top);
        if (top.flat >= 0 && above == best - 1) least = top;             // the best-th largest of the threads' largest
        __syncthreads();
        low = least;
        some = top.flat >= 0 && !low.before(top);
    }
    if (some)
        for (int l = t; l < lists; l += THREADS)
            for (int rank = 0; rank < best; rank++) {
                const Candidate c = item(l, rank);
                if (c.flat < 0 || low.before(c)) break;
                found[atomicAdd(&count, 1)] = c;
            }
    __syncthreads();
    const int n = count;
    for (int i = t; i < n; i += THREADS) {
        const Candidate c = found[i];
        int rank = 0;
#pragma unroll 8
        for (int j = 0; j < n; j++) rank += found[j].before(c);
        if (rank < best) {
            scores_out[(size_t)r * best + rank] = (float)value_of(c);
            beam_out[(size_t)r * best + rank] = c.flat / V;
            tok_out[(size_t)r * best + rank] = c.flat % V;
        }
    }
    for (int i = n + t; i < best; i += THREADS)
        scores_out[(size_t)r * best + i] = -INFINITY, beam_out[(size_t)r * best + i] = 0, tok_out[(size_t)r * best + i] = 0;
}

constexpr size_t SELECT_ROOM = 200 * 1024;

size_t select_smem(int beams, int pieces, int best) {
    const long long lists = (long long)beams * pieces;
    return (size_t)(best * best * ((lists + THREADS - 1) / THREADS)) * sizeof(Candidate) + (lists * best <= KEYS ? (size_t)(lists * best) * 8 : 0);
}

}  // namespace

DK_EXPORT int dk_beam_pieces(int V) { return logit_pieces(V, Piece::SIZE); }

// logits [requests * beams, V] float32, scores [requests, beams], ended [requests, beams] or null; ws_key: requests * beams * pieces *
// best 8-byte words, ws_sum: requests * beams * pieces pairs of doubles; results [requests, best].
DK_EXPORT int dk_beam_select(const float* logits, int V, int requests, int beams, int best, const float* scores, const int* ended,
                             uint64_t* ws_key, double* ws_sum, float* scores_out, int* beam_out, int* tok_out, cudaStream_t st) {
    if (V < 1 || beams < 1 || beams > MAX_BEAMS || best < 1 || best > MAX_BEST || requests < 1 || (long long)beams * V > 0x7fffffffLL ||
        (long long)requests * beams > 65535)
        return (int)cudaErrorInvalidValue;
    const int pieces = dk_beam_pieces(V);
    size_t smem = select_smem(beams, pieces, best);
    const bool many = smem > SELECT_ROOM;
    if (many) smem = best * sizeof(Candidate);
    if (smem > 32 * 1024) {
        cudaError_t ce = cudaFuncSetAttribute(beam_select_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SELECT_ROOM);
        if (ce != cudaSuccess) {
            cudaGetLastError();
            return (int)ce;
        }
    }
    int e = dk_launch(beam_pieces_kernel, dim3(pieces, requests * beams), dim3(THREADS), 0, st, logits, V, best, ws_key, (double2*)ws_sum);
    if (e) return e;
    // (may start under the end of the first: it reads nothing before)
    return dk_launch_as(true, many ? beam_select_kernel<true> : beam_select_kernel<false>, dim3(requests), dim3(THREADS), smem, st, (const uint64_t*)ws_key, (const double2*)ws_sum, pieces,
                        V, beams, best, scores, ended, scores_out, beam_out, tok_out);
}
