// The best continuations of a request's beams, over all beams and the whole vocabulary.
//
//   value(b, v) = score[b] + logit[b, v] - log(sum_u exp(logit[b, u]))
//
// and the `best` largest values, ties by the lower beam, then the lower token. A logit that is not finite is no candidate and weighs
// nothing; a beam whose score is not finite is not live and brings none; a beam at its end brings one, its own score with token 0.
// Where there are fewer candidates than asked for, the rest is (-infinity, 0, 0).
//
// Within a beam the order of the values is that of the logits, so a piece of a row can give up all but its `best` largest logits
// before the row's sum is known: one pass over the logits. Across beams the logarithms of the sums decide: exponentials in float32
// against the piece's maximum, added up in float32 within a thread and in double from there on, values compared in double, so that a
// rank does not hang on the rounding of the scores (float32 scores around -30 are 2^-19 apart).
//
// First launch, a block a piece of a row: the logits stay in registers; the block's `best`-th largest of the threads' own maxima is
// a floor under the `best`-th largest logit, few logits beside the ones looked for reach it, and these are ranked by counting. Second
// launch, a block a request: the same over what the pieces left. Bound by reading the logits where there are many rows, by the two
// launches' latency where there are few.
#include "common.cuh"

namespace {

constexpr int THREADS = 256, MAX_BEST = 64, MAX_BEAMS = 32;

// Larger key: larger logit, then lower index. 0: none.
__device__ __forceinline__ uint64_t key_of(float v, int i) {
    if (!isfinite(v)) return 0;
    const uint32_t b = __float_as_uint(v + 0.f);                         // -0 counts as 0
    return (uint64_t)(b & 0x80000000u ? ~b : b | 0x80000000u) << 32 | (uint32_t)~i;
}
__device__ __forceinline__ float logit_of(uint64_t key) {
    const uint32_t b = (uint32_t)(key >> 32);
    return __uint_as_float(b & 0x80000000u ? b & 0x7fffffffu : ~b);
}
__device__ __forceinline__ int index_of(uint64_t key) { return (int)~(uint32_t)key; }

// grid (pieces, rows). ws_key [rows][pieces][best] in falling order (0: none), ws_sum [rows][pieces] = (maximum, sum).
template <int EACH, bool WIDE>
__global__ void __launch_bounds__(THREADS)
beam_pieces_kernel(const float* logits, int V, int best, uint64_t* ws_key, double2* ws_sum) {
    __shared__ uint64_t tops[THREADS], floor_key;
    __shared__ uint64_t found[MAX_BEST * EACH];
    __shared__ float red_m[THREADS / 32];
    __shared__ double red_s[THREADS / 32];
    __shared__ int count;
    pdl_wait();
    pdl_launch_dependents();
    const int t = threadIdx.x, lane = t & 31, w = t >> 5;
    const float* z = logits + (size_t)blockIdx.y * V;
    const int begin = blockIdx.x * (THREADS * EACH), end = min(V, begin + THREADS * EACH);
    auto index = [&](int k) { return WIDE ? begin + ((k / 4) * THREADS + t) * 4 + k % 4 : begin + k * THREADS + t; };
    float v[EACH];
    if (WIDE) {
#pragma unroll
        for (int k = 0; k < EACH; k += 4)
            *reinterpret_cast<float4*>(v + k) = index(k) < end ? *reinterpret_cast<const float4*>(z + index(k))
                                                              : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
    } else {
#pragma unroll
        for (int k = 0; k < EACH; k++) v[k] = index(k) < end ? z[index(k)] : -INFINITY;
    }
    if (t == 0) count = 0, floor_key = 1;
    uint64_t top = 0;
    float m = -INFINITY;
#pragma unroll
    for (int k = 0; k < EACH; k++) {
        if (!isfinite(v[k])) v[k] = -INFINITY;
        m = fmaxf(m, v[k]);
    }
#pragma unroll
    for (int k = EACH - 1; k >= 0; k--)
        if (v[k] == m) top = key_of(v[k], index(k));                    // the lowest index of the thread's maximum
    tops[t] = top;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane == 0) red_m[w] = m;
    __syncthreads();
    m = red_m[0];
#pragma unroll
    for (int i = 1; i < THREADS / 32; i++) m = fmaxf(m, red_m[i]);
    // the best-th largest of the threads' maxima
    int above = 0;
#pragma unroll 8
    for (int i = 0; i < THREADS; i++) above += tops[i] > top;
    if (top != 0 && above == best - 1) floor_key = top;
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < EACH; k++) sum += v[k] == -INFINITY ? 0.f : expf(v[k] - m);
    double total = sum;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    if (lane == 0) red_s[w] = total;
    __syncthreads();
    if (t == 0) {
        total = 0.;
        for (int i = 0; i < THREADS / 32; i++) total += red_s[i];
        ws_sum[(size_t)blockIdx.y * gridDim.x + blockIdx.x] = make_double2((double)m, total);
    }
    const uint64_t least = floor_key;
    if (top >= least) {
#pragma unroll
        for (int k = 0; k < EACH; k++) {
            const uint64_t key = key_of(v[k], index(k));
            if (key >= least) found[atomicAdd(&count, 1)] = key;        // `best` threads at most have any
        }
    }
    __syncthreads();
    const int n = count;
    uint64_t* out = ws_key + ((size_t)blockIdx.y * gridDim.x + blockIdx.x) * best;
    for (int i = t; i < n; i += THREADS) {
        const uint64_t key = found[i];
        int rank = 0;
        for (int j = 0; j < n; j++) rank += found[j] > key;
        if (rank < best) out[rank] = key;
    }
    for (int i = n + t; i < best; i += THREADS) out[i] = 0;
}

struct Candidate {
    double value;
    int flat;                                                            // beam * V + token; -1: none
    __device__ __forceinline__ bool before(const Candidate& o) const {
        return flat >= 0 && (o.flat < 0 || value > o.value || (value == o.value && flat < o.flat));
    }
};

// grid (requests). Dynamic shared memory: best * ceil(beams * pieces * best / THREADS) candidates.
__global__ void __launch_bounds__(THREADS)
beam_select_kernel(const uint64_t* ws_key, const double2* ws_sum, int pieces, int V, int beams, int best, const float* scores,
                   const int* ended, float* scores_out, int* beam_out, int* tok_out) {
    extern __shared__ __align__(16) unsigned char dyn[];
    Candidate* found = reinterpret_cast<Candidate*>(dyn);
    __shared__ Candidate tops[THREADS], least;
    __shared__ double offset[MAX_BEAMS];
    __shared__ int kind[MAX_BEAMS];                                      // 0: not live, 1: live, 2: at its end
    __shared__ int count;
    pdl_wait();
    pdl_launch_dependents();
    const int r = blockIdx.x, t = threadIdx.x, lane = t & 31, w = t >> 5;
    for (int b = w; b < beams; b += THREADS / 32) {
        const double2* part = ws_sum + (size_t)(r * beams + b) * pieces;
        double m = -INFINITY, sum = 0.;
        for (int c = lane; c < pieces; c += 32) m = fmax(m, part[c].x);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = fmax(m, __shfl_xor_sync(0xffffffffu, m, o));
        for (int c = lane; c < pieces; c += 32) sum += part[c].y > 0. ? part[c].y * exp(part[c].x - m) : 0.;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) {
            const float score = scores[r * beams + b];
            const bool done = ended != nullptr && ended[r * beams + b] != 0;
            kind[b] = !isfinite(score) ? 0 : done ? 2 : sum > 0. ? 1 : 0;
            offset[b] = kind[b] == 1 ? (double)score - (m + log(sum)) : (double)score;
        }
    }
    if (t == 0) count = 0, least = Candidate{-INFINITY, -1};
    __syncthreads();
    // item i: the (i / lists)-th of list i % lists, so that the threads' first items are the lists' first
    const int lists = beams * pieces, items = lists * best;
    auto item = [&](int i) {
        const int list = i % lists, rank = i / lists, b = list / pieces;
        Candidate c = {-INFINITY, -1};
        if (kind[b] == 2) {
            if (rank == 0 && list == b * pieces) c = Candidate{offset[b], b * V};
        } else if (kind[b] == 1) {
            const uint64_t key = ws_key[((size_t)r * lists + list) * best + rank];
            if (key) c = Candidate{(double)logit_of(key) + offset[b], b * V + index_of(key)};
        }
        return c;
    };
    Candidate top = {-INFINITY, -1};
    for (int i = t; i < items; i += THREADS) {
        const Candidate c = item(i);
        if (c.before(top)) top = c;
    }
    tops[t] = top;
    __syncthreads();
    int above = 0;
#pragma unroll 8
    for (int i = 0; i < THREADS; i++) above += tops[i].before(top);
    if (top.flat >= 0 && above == best - 1) least = top;
    __syncthreads();
    if (top.flat >= 0 && !least.before(top))
        for (int i = t; i < items; i += THREADS) {
            const Candidate c = item(i);
            if (c.flat >= 0 && !least.before(c)) found[atomicAdd(&count, 1)] = c;
        }
    __syncthreads();
    const int n = count;
    for (int i = t; i < n; i += THREADS) {
        const Candidate c = found[i];
        int rank = 0;
        for (int j = 0; j < n; j++) rank += found[j].before(c);
        if (rank < best) {
            scores_out[(size_t)r * best + rank] = (float)c.value;
            beam_out[(size_t)r * best + rank] = c.flat / V;
            tok_out[(size_t)r * best + rank] = c.flat % V;
        }
    }
    for (int i = n + t; i < best; i += THREADS)
        scores_out[(size_t)r * best + i] = -INFINITY, beam_out[(size_t)r * best + i] = 0, tok_out[(size_t)r * best + i] = 0;
}

// Logits a block of the first launch takes
constexpr int EACH = 32;

size_t select_smem(int beams, int pieces, int best) {
    return (size_t)best * ((beams * pieces * best + THREADS - 1) / THREADS) * sizeof(Candidate);
}

}  // namespace

DK_EXPORT int dk_beam_pieces(int V) { return (V + THREADS * EACH - 1) / (THREADS * EACH); }

DK_EXPORT int dk_beam_select_takes(int V, int beams, int best) { return select_smem(beams, dk_beam_pieces(V), best) <= 200 * 1024; }

// logits [requests * beams, V] float32, scores [requests, beams], ended [requests, beams] or null; ws_key: requests * beams * pieces *
// best 8-byte words, ws_sum: requests * beams * pieces pairs of doubles; results [requests, best].
DK_EXPORT int dk_beam_select(const float* logits, int V, int requests, int beams, int best, const float* scores, const int* ended,
                             uint64_t* ws_key, double* ws_sum, float* scores_out, int* beam_out, int* tok_out, cudaStream_t st) {
    if (V < 1 || beams < 1 || beams > MAX_BEAMS || best < 1 || best > MAX_BEST || requests < 1 || (long long)beams * V > 0x7fffffffLL ||
        (long long)requests * beams > 65535)
        return (int)cudaErrorInvalidValue;
    const int pieces = dk_beam_pieces(V);
    const size_t smem = select_smem(beams, pieces, best);
    if (smem > 200 * 1024) return (int)cudaErrorInvalidValue;
    cudaError_t ce = cudaFuncSetAttribute(beam_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024);
    if (ce != cudaSuccess) {
        cudaGetLastError();
        return (int)ce;
    }
    const bool wide = V % 4 == 0 && ((uintptr_t)logits & 15) == 0;      // rows on 16-byte boundaries: 16 bytes a load
    int e = dk_launch(wide ? beam_pieces_kernel<EACH, true> : beam_pieces_kernel<EACH, false>, dim3(pieces, requests * beams), dim3(THREADS),
                      0, st, logits, V, best, ws_key, (double2*)ws_sum);
    if (e) return e;
    return dk_launch(beam_select_kernel, dim3(requests), dim3(THREADS), smem, st, (const uint64_t*)ws_key, (const double2*)ws_sum, pieces, V,
                     beams, best, scores, ended, scores_out, beam_out, tok_out);
}
