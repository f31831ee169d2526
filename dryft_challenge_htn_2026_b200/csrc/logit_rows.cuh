// Reading rows of float32 logits in pieces, 16 bytes a load whatever a row's alignment.
#pragma once
#include "common.cuh"

// A block of THREADS threads takes piece `piece` of a row of V numbers at z: EACH numbers a thread, in fours. Fours start on 16-byte
// boundaries, so a row that begins within one has up to three places in front that are not its own; a four that is not wholly the
// row's is read one number at a time. Number 4 q + e of a thread has index at(q) + e; those outside [0, V) come as -infinity.
template <int THREADS, int EACH>
struct LogitPiece {
    static constexpr int SIZE = THREADS * EACH;
    int first;                              // index of the thread's first number
    __device__ __forceinline__ LogitPiece(const float* z, int piece) {
        first = piece * SIZE + (int)threadIdx.x * 4 - (int)(((uintptr_t)z >> 2) & 3);
    }
    __device__ __forceinline__ int at(int q) const { return first + q * THREADS * 4; }
    __device__ __forceinline__ int index(int k) const { return at(k / 4) + k % 4; }
    // whether all of the block's piece is the row's
    __device__ __forceinline__ bool inside(int V) const {
        const int begin = first - (int)threadIdx.x * 4;
        return begin >= 0 && begin + SIZE <= V;
    }
    __device__ __forceinline__ float one(const float* z, int V, int i) const { return i >= 0 && i < V ? z[i] : -INFINITY; }
    __device__ __forceinline__ float4 four(const float* z, int V, int q) const {
        const int i = at(q);
        if (i >= 0 && i + 4 <= V) return *reinterpret_cast<const float4*>(z + i);
        return make_float4(one(z, V, i), one(z, V, i + 1), one(z, V, i + 2), one(z, V, i + 3));
    }
    __device__ __forceinline__ void load(const float* z, int V, float (&v)[EACH]) const {
        if (inside(V)) {
#pragma unroll
            for (int q = 0; q < EACH / 4; q++) {
                const float4 x = *reinterpret_cast<const float4*>(z + at(q));
                v[4 * q] = x.x, v[4 * q + 1] = x.y, v[4 * q + 2] = x.z, v[4 * q + 3] = x.w;
            }
        } else {
#pragma unroll
            for (int k = 0; k < EACH; k++) v[k] = one(z, V, index(k));
        }
    }
};

// Pieces that a row of V numbers has at most.
static inline int logit_pieces(int V, int size) { return (int)(((long long)V + 3 + size - 1) / size); }
