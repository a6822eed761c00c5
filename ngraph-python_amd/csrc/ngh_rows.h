// Rows of fp32, fp16 or bf16 elements as fp32 registers: the loads and stores the row operators
// (embedding, block norms) share.  A lane holds C chunks of VEC consecutive elements, chunk c of
// lane l starting at element (c * lanes + l) * VEC, so that a wavefront's access is contiguous.
#pragma once
#include <hip/hip_runtime.h>

#include "ngraph_hip.h"

namespace ngh {

constexpr int kRowSumsMax = 4;          // values one reduction sums at most

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

// V consecutive elements: on a boundary of V of them, or on any boundary of one (the device takes
// such accesses; where a row's start allows no better, this costs a few per cent against 16-byte
// boundaries and an access for each element several times the loads).
template <class T, int V> struct VecOf {
    typedef T type __attribute__((ext_vector_type(V)));
    typedef T loose __attribute__((ext_vector_type(V), aligned(sizeof(T))));
};

// V consecutive elements as floats (conversion is exact) and back (round to nearest even, once).
template <class T, int V, bool LOOSE = false>
__device__ __forceinline__ void load_as_float(const T* p, float (&out)[V]) {
    typedef typename VecOf<T, V>::type vec;
    typedef typename VecOf<T, V>::loose loose;
    vec v;
    if constexpr (LOOSE) v = *reinterpret_cast<const loose*>(p);
    else v = *reinterpret_cast<const vec*>(p);
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = (float)v[i];
}

template <class T, int V, bool LOOSE = false>
__device__ __forceinline__ void store_from_float(T* p, const float (&in)[V]) {
    typedef typename VecOf<T, V>::type vec;
    typedef typename VecOf<T, V>::loose loose;
    vec v;
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = (T)in[i];
    if constexpr (LOOSE) *reinterpret_cast<loose*>(p) = v;
    else *reinterpret_cast<vec*>(p) = v;
}

// The first `count` (0 .. V) of V elements, zeros behind them.  RAGGED: rows start on any boundary
// and may end inside a piece; else count is 0 or V.
template <class T, int V, bool RAGGED>
__device__ __forceinline__ void load_piece(const T* p, int count, float (&out)[V]) {
    if (RAGGED ? count == V : count > 0) {
        load_as_float<T, V, RAGGED>(p, out);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            out[i] = 0.0f;
            if (RAGGED && i < count) out[i] = (float)p[i];
        }
    }
}

template <class T, int V, bool RAGGED>
__device__ __forceinline__ void store_piece(T* p, int count, const float (&in)[V]) {
    if (RAGGED ? count == V : count > 0) {
        store_from_float<T, V, RAGGED>(p, in);
    } else if (RAGGED) {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i < count) p[i] = (T)in[i];
    }
}

// Elements of the piece that starts at `col` that are in a row of `width`.
template <int V, bool RAGGED>
__device__ __forceinline__ int piece_count(unsigned col, unsigned width) {
    if constexpr (RAGGED) return col >= width ? 0 : (int)min((unsigned)V, width - col);
    else return col < width ? V : 0;
}

// The sum over the lanes of a row.  NW > 1: the row has NW whole wavefronts, which are the workgroup;
// `sh` holds 2 x kRowSumsMax x NW floats and `phase` alternates, so one barrier a reduction is enough (a
// wavefront that is a reduction ahead writes the other half).  NW == 1: `lanes` (a power of two up to
// 64) consecutive lanes of a wavefront, no barrier.
template <int N, int NW>
__device__ __forceinline__ void row_sums(float (&v)[N], int lanes, float* sh, int& phase) {
    if constexpr (NW == 1) {
        for (int m = lanes >> 1; m > 0; m >>= 1) {
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] += __shfl_xor(v[i], m, 64);
        }
    } else {
#pragma unroll
        for (int m = 32; m > 0; m >>= 1) {
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] += __shfl_xor(v[i], m, 64);
        }
        float* half = sh + phase * (kRowSumsMax * NW);
        phase ^= 1;
        if ((threadIdx.x & 63) == 0) {
#pragma unroll
            for (int i = 0; i < N; ++i) half[i * NW + (threadIdx.x >> 6)] = v[i];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float s = half[i * NW];
#pragma unroll
            for (int w = 1; w < NW; ++w) s += half[i * NW + w];
            v[i] = s;
        }
    }
}

}  // namespace ngh
