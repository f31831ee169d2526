// Which path of a tree of drafted tokens the model itself would have taken.
//
// Node i of a sequence's tree holds a drafted token tok[i], drafted to follow node parent[i] (< i; node 0 is the last token of the
// sequence, whose own place is settled). The model's token after node i is what the sampler (sampling.cu) draws from logits[i] at the
// position after the node's, with the sequence's temperature and seed: greedy, or argmax(logit / T + noise) with noise that hangs on
// seed, position and token alone. So the tokens that come out are those that one token a step would have drawn, and drafting changes
// how many steps they take, not which they are. From node 0 on the path goes to the child that holds the chosen token (the lowest
// one, if several do) until there is none; the token chosen there is the sequence's next.
//
// Two launches: the best token of each piece of 8,192 (or 2,048) logits, over all nodes and pieces side by side (one pass over the logits: bound
// by reading them where the choice is greedy); then a block a sequence puts the pieces together and walks the path. Drawing costs a
// hash and two logarithms a logit. Most logits are spared the logarithms: -log(u) >= 1 - u, so the noise is at most -log(1 - u), and
// what does not reach the thread's best so far with that much cannot win.
// Measured: eight trees of 40 to 64 nodes over 151,936 tokens, greedy, 42 us (252 MB, 6.0 TB/s, 92 % of the copy rate); five nodes, drawn, 8.7 us on
// the device, of which the logits are 0.5 and the two launches most; a call of this size takes the host 23 us.
#include "logit_rows.cuh"
#include "sampling_kernels.cuh"

namespace {

constexpr int THREADS = 256, MAX_NODES = 1024, PATH_THREADS = 1024;

template <int WIDTH>
__device__ __forceinline__ void best_of(float& bv, int& bi) {
#pragma unroll
    for (int o = WIDTH / 2; o > 0; o >>= 1) {
        const float ov = __shfl_xor_sync(0xffffffffu, bv, o);
        const int oi = __shfl_xor_sync(0xffffffffu, bi, o);
        better(bv, bi, ov, oi);
    }
}

// grid (pieces, max_nodes, sequences); EACH: logits a thread
template <int EACH>
__global__ void __launch_bounds__(THREADS)
accept_pieces_kernel(const float* logits, int V, const int* cu_q, const int* row_pos, const float* temperature, const uint32_t* seeds,
                     float* ws_val, int* ws_idx) {
    __shared__ float sv[THREADS / 32];
    __shared__ int si[THREADS / 32];
    pdl_wait();
    const int s = blockIdx.z, row = cu_q[s] + blockIdx.y;
    if (row >= cu_q[s + 1]) return;
    const float* z = logits + (size_t)row * V;
    const LogitPiece<THREADS, EACH> piece(z, blockIdx.x);
    const int pos = row_pos[row];
    const float temp = temperature[s];
    float bv = -INFINITY;
    int bi = 0x7fffffff;
    if (!(temp > 0.f)) {
        float v[EACH];
        piece.load(z, V, v);
#pragma unroll
        for (int k = 0; k < EACH; k++)
            if (v[k] > bv) bv = v[k], bi = piece.index(k);             // a thread's own numbers come with rising index
    } else {
        const float inv_t = 1.f / temp;
        const uint32_t lo = seeds[2 * s], hi = seeds[2 * s + 1], mid = lo + (uint32_t)(pos + 1) * 0x85EBCA6Bu;
#pragma unroll 2
        for (int q = 0; q < EACH / 4; q++) {
            const float4 four = piece.four(z, V, q);
            const float v[4] = {four.x, four.y, four.z, four.w};
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int i = piece.at(q) + e;
                const uint32_t x = mix32(mix32(mix32((uint32_t)i ^ 0x9E3779B9u) + mid) ^ hi) >> 8, d = max(0xffffffu - x, 1u);   // as gumbel() makes them
                // u is (x + 0.5) / 2^24 to the nearest float32, 1 - 2^-24 at most, so 1 - u is d / 2^24 at least
                const float most = 0.6931472f * (24.f - __log2f((float)d)) + 1e-3f;
                if (v[e] * inv_t + most >= bv) better(bv, bi, v[e] * inv_t + gumbel(lo, hi, (uint32_t)(pos + 1), (uint32_t)i), i);
            }
        }
    }
    if (pos < 0) bv = -INFINITY;                                       // a padding row
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    best_of<32>(bv, bi);
    if (lane == 0) sv[w] = bv, si[w] = bi;
    __syncthreads();
    if (w == 0) {
        bv = lane < THREADS / 32 ? sv[lane] : -INFINITY;
        bi = lane < THREADS / 32 ? si[lane] : 0x7fffffff;
        best_of<THREADS / 32>(bv, bi);
        if (lane == 0) {
            const size_t at = (size_t)row * gridDim.x + blockIdx.x;
            ws_val[at] = bv, ws_idx[at] = bi;
        }
    }
    pdl_launch_dependents();                                           // (at the start, the second launch's blocks would stand in the way)
}

// grid (sequences)
__global__ void __launch_bounds__(PATH_THREADS)
accept_path_kernel(const float* ws_val, const int* ws_idx, int pieces, const int* cu_q, const int* tok, const int* parent, int max_nodes,
                   int* path, int* n_path, int* next_tok) {
    __shared__ int choice[MAX_NODES], toks[MAX_NODES], up[MAX_NODES];
    pdl_wait();
    pdl_launch_dependents();
    const int s = blockIdx.x, row0 = cu_q[s], n = min(max_nodes, cu_q[s + 1] - row0);
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    for (int i = threadIdx.x; i < n; i += PATH_THREADS) toks[i] = tok[row0 + i], up[i] = parent[row0 + i];
    for (int i = w; i < n; i += PATH_THREADS / 32) {
        float bv = -INFINITY;
        int bi = 0x7fffffff;
        const size_t at = (size_t)(row0 + i) * pieces;
        for (int c = lane; c < pieces; c += 32) better(bv, bi, ws_val[at + c], ws_idx[at + c]);
        best_of<32>(bv, bi);
        if (lane == 0) choice[i] = bv == -INFINITY ? 0 : bi;
    }
    __syncthreads();
    if (w != 0) return;
    int at = 0, len = 0;
    int* out = path + (size_t)s * max_nodes;
    if (n > 0) {
        if (lane == 0) out[0] = 0;
        len = 1;
        for (int i0 = 1; i0 < n;) {                                    // a child stands behind its parent: one run over the nodes
            const int i = i0 + lane;
            const unsigned hit = __ballot_sync(0xffffffffu, i < n && up[i] == at && toks[i] == choice[at]);
            if (!hit) {
                i0 += 32;
                continue;
            }
            at = i0 + __ffs(hit) - 1;
            if (lane == 0) out[len] = at;
            len++;
            i0 = at + 1;
        }
    }
    for (int i = len + lane; i < max_nodes; i += 32) out[i] = -1;
    if (lane == 0) n_path[s] = len, next_tok[s] = n > 0 ? choice[at] : 0;
}

}  // namespace

// Logits a thread of the first launch takes: 32, or 8 where that leaves SMs without a block, as with a handful of nodes. With 8 / 32, nodes of
// 151,936 logits: drawn, 5 nodes 8.6 / 12.0 us, 16 15.2 / 18.0, 32 (where the rule changes) 24.6 / 26.5, 64 45.7 / 46.7, 8 x 64 305 / 281;
// greedy 5 nodes 5.3 / 4.8, 16 6.3 / 5.3, 32 8.0 / 6.5, 64 14.8 / 12.3.
static int each_for(int V, long long rows) {
    static int sms = 0;
    if (sms == 0) {
        int dev = 0;
        cudaGetDevice(&dev);
        cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    }
    return rows * logit_pieces(V, 32 * THREADS) >= 4 * sms ? 32 : 8;
}

DK_EXPORT int dk_tree_accept_pieces(int V, int n_seq, int max_nodes) { return logit_pieces(V, each_for(V, (long long)n_seq * max_nodes) * THREADS); }

// logits [rows, V] float32; temperature [n_seq], seeds [n_seq][2]; ws_val, ws_idx: rows * dk_tree_accept_pieces elements;
// path [n_seq, max_nodes], n_path [n_seq], next_tok [n_seq].
DK_EXPORT int dk_tree_accept(const float* logits, int V, const int* tok, const int* parent, const int* cu_q, const int* row_pos,
                             const float* temperature, const uint32_t* seeds, int n_seq, int max_nodes, float* ws_val, int* ws_idx,
                             int* path, int* n_path, int* next_tok, cudaStream_t st) {
    if (V < 1 || max_nodes < 1 || max_nodes > MAX_NODES || n_seq < 1 || n_seq > 65535) return (int)cudaErrorInvalidValue;
    const int each = each_for(V, (long long)n_seq * max_nodes), pieces = logit_pieces(V, each * THREADS);
    int e = dk_launch(each == 8 ? accept_pieces_kernel<8> : accept_pieces_kernel<32>, dim3(pieces, max_nodes, n_seq), dim3(THREADS), 0, st, logits,
                      V, cu_q, row_pos, temperature, seeds, ws_val, ws_idx);
    if (e) return e;
    // (may start under the end of the first: it reads nothing before)
    return dk_launch_as(true, accept_path_kernel, dim3(n_seq), dim3(PATH_THREADS), 0, st, (const float*)ws_val, (const int*)ws_idx, pieces, cu_q,
                        tok, parent, max_nodes, path, n_path, next_tok);
}
