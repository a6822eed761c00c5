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

// The first `count` (0 .. V) of V elements as they lie in memory, zeros where count is 0; what lies behind
// them is undefined.  RAGGED: rows start on any boundary and may end inside a piece; else count is 0 or V.
// A piece that ends behind its row is still loaded whole where that stays inside the operand (`inside`:
// another row follows that is no shorter than a piece), and element by element only in the last row.
// Nothing here waits for the load: elements behind the row are masked where the piece is used (a mask
// right behind the load made every one wait for the one before it: 141 us, not 104, for the backward pass
// over [12000, 1027] fp32 rows).
template <class T, int V, bool RAGGED>
__device__ __forceinline__ typename VecOf<T, V>::type load_raw(const T* p, int count, bool inside) {
    typename VecOf<T, V>::type v = (T)0.0f;
    if constexpr (RAGGED) {
        if (count == V || (inside && count > 0)) {
            v = *reinterpret_cast<const typename VecOf<T, V>::loose*>(p);
        } else if (count > 0) {
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (i < count) v[i] = p[i];
        }
    } else {
        if (count > 0) v = *reinterpret_cast<const typename VecOf<T, V>::type*>(p);
    }
    return v;
}

// A piece as floats, zeros behind the first `count` elements.
template <class T, int V, bool RAGGED>
__device__ __forceinline__ void to_float(const typename VecOf<T, V>::type& v, int count, float (&out)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = !RAGGED || i < count ? (float)v[i] : 0.0f;
}

// The same, worked out here: loads that follow stay behind it and may fill v again.  Left to itself the compiler uses
// v only where the floats are needed, behind the loads of the next piece, and, since those are conditional,
// waits for them too, so that nothing is in flight meanwhile (the same rows: 104 us, 92 so).
template <class T, int V, bool RAGGED>
__device__ __forceinline__ void take_piece(const typename VecOf<T, V>::type& v, int count, float (&out)[V]) {
    to_float<T, V, RAGGED>(v, count, out);
#pragma unroll
    for (int i = 0; i < V; ++i) {
        if constexpr (sizeof(T) == 4 && !RAGGED) asm volatile("v_mov_b32 %0, %1" : "=v"(out[i]) : "v"((float)v[i]) : "memory");
        else asm volatile("" : "+v"(out[i])::"memory");
    }
}

template <class T, int V, bool RAGGED>
__device__ __forceinline__ void load_piece(const T* p, int count, bool inside, float (&out)[V]) {
    to_float<T, V, RAGGED>(load_raw<T, V, RAGGED>(p, count, inside), count, out);
}

// The piece of a vector on any boundary, zeros behind its end.  Nothing may be read behind the vector: its last
// piece is loaded from V elements before the end where there are as many (`behind_another`: it is not the first),
// and shifted (norms of [16384, 4095] with gains in bf16: 169 us, 146 so).
template <class T, int V>
__device__ __forceinline__ void load_end(const T* p, int count, bool behind_another, float (&out)[V]) {
    if (count == V) {
        load_piece<T, V, true>(p, V, false, out);
    } else if (count > 0 && behind_another) {
        const int shift = V - count;
        load_piece<T, V, true>(p - shift, V, false, out);
#pragma unroll
        for (int bit = V / 2; bit > 0; bit /= 2) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float further = i + bit < V ? out[i + bit < V ? i + bit : 0] : 0.0f;
                out[i] = shift & bit ? further : out[i];
            }
        }
    } else {
        load_piece<T, V, true>(p, count, false, out);
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

// The x of the lane's partner at distance 1, 2, 4, 8, 16 or 32 for reductions in which the lanes at smaller
// distances hold the same value already: one instruction within 16 lanes, mostly part of the one that
// uses it (the partner of a mirror is not the lane at that distance but one with the same value), and
// one for a pair of values beyond.
template <int CTRL>
__device__ __forceinline__ unsigned dpp(unsigned x) {
    return (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xf, 0xf, true);
}

template <int DISTANCE, class F>
__device__ __forceinline__ unsigned with_partner(unsigned x, F f) {
    if constexpr (DISTANCE == 1) return f(x, dpp<0xB1>(x));          // quad_perm 1,0,3,2
    else if constexpr (DISTANCE == 2) return f(x, dpp<0x4E>(x));     // quad_perm 2,3,0,1
    else if constexpr (DISTANCE == 4) return f(x, dpp<0x141>(x));    // row_half_mirror
    else if constexpr (DISTANCE == 8) return f(x, dpp<0x140>(x));    // row_mirror
    else if constexpr (DISTANCE == 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
        return f(r[0], r[1]);
    } else {
        const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
        return f(r[0], r[1]);
    }
}

template <int DISTANCE>
__device__ __forceinline__ float add_partner(float x) {
    return __uint_as_float(with_partner<DISTANCE>(
        __float_as_uint(x), [](unsigned a, unsigned b) { return __float_as_uint(__uint_as_float(a) + __uint_as_float(b)); }));
}

__device__ __forceinline__ unsigned wave_max(unsigned x) {
    const auto f = [](unsigned a, unsigned b) { return max(a, b); };
    return with_partner<32>(with_partner<16>(with_partner<8>(with_partner<4>(with_partner<2>(with_partner<1>(x, f), f), f), f), f), f);
}

// The sums over the lanes of a row of up to kRowSumsMax values.  SEVERAL: the row has several wavefronts
// (up to 16), which are the workgroup; `sh` holds 2 x 16 entries that were cleared before the first
// reduction (clear_row_sums) and `phase` alternates, so one barrier a reduction is enough (a wavefront that
// is a reduction ahead writes the other half).  Else `lanes` (a power of two up to 64) consecutive lanes
// of a wavefront, no barrier.  A value costs 8 vector instructions within a wavefront and 5 across them;
// with a permutation through LDS for every step they were a fifth of the backward kernel.
struct alignas(16) RowSums {
    float v[kRowSumsMax];
};

template <bool SEVERAL>
__device__ __forceinline__ void clear_row_sums(RowSums* sh) {
    if constexpr (SEVERAL) {
        if (threadIdx.x < 2 * 16 * kRowSumsMax) reinterpret_cast<float*>(sh)[threadIdx.x] = 0.0f;
        if (blockDim.x < 2 * 16 * kRowSumsMax && threadIdx.x + blockDim.x < 2 * 16 * kRowSumsMax)
            reinterpret_cast<float*>(sh)[threadIdx.x + blockDim.x] = 0.0f;
        __syncthreads();
    }
}

template <int N, bool SEVERAL>
__device__ __forceinline__ void row_sums(float (&v)[N], int lanes, RowSums* sh, int& phase) {
#define NGH_ROW_SUMS_STEP(DISTANCE)          \
    if (SEVERAL || lanes > DISTANCE) {       \
        _Pragma("unroll") for (int i = 0; i < N; ++i) v[i] = add_partner<DISTANCE>(v[i]); \
    }
    NGH_ROW_SUMS_STEP(1)
    NGH_ROW_SUMS_STEP(2)
    NGH_ROW_SUMS_STEP(4)
    NGH_ROW_SUMS_STEP(8)
    NGH_ROW_SUMS_STEP(16)
    NGH_ROW_SUMS_STEP(32)
#undef NGH_ROW_SUMS_STEP
    if constexpr (SEVERAL) {
        RowSums* half = sh + phase * 16;
        phase ^= 1;
        if ((threadIdx.x & 63) == 0) {
#pragma unroll
            for (int i = 0; i < N; ++i) half[threadIdx.x >> 6].v[i] = v[i];
        }
        __syncthreads();
        const RowSums all = half[threadIdx.x & 15];
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = add_partner<8>(add_partner<4>(add_partner<2>(add_partner<1>(all.v[i]))));
    }
}

}  // namespace ngh
