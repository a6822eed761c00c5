// Kernels of ngh_block_norm / ngh_block_norm_grad: the norms before and after a block fused with its
// gate and residual.  For a row, with bh = N(b):
//     u = bh p + q;   h = alpha x + g u;   y = N(h) w + z
// and backward, with T the transpose of N's Jacobian, T(t; x) = r (t - xh mean(t xh) [- mean(t)]):
//     d = dh + T(dy w; h);   dx = alpha d;   dg += d u;   e = d g;   dp += e bh;   dq += e;
//     db = T(e p; b);   dw += dy hh;   dz += dy
// A row is held in registers from its one load on (C pieces of VEC elements a lane, a row on as many
// wavefronts as it fills or, not SEVERAL, on a power of two of lanes), so the forward pass reads x and
// b and writes h and y once, the backward pass reads dh, dy, h and b and writes dx and db: both are
// bound by memory (16384 rows of 4096 bf16 elements with a gate: forward 99 us, 5.4 TB/s; backward 177,
// 4.5).  The variance of the layer norm is taken around the mean, in registers.  The statistics are
// computed again in the backward pass: a reduction that is there anyway, and no operand.
#pragma once
#include <hip/hip_runtime.h>

#include "ngh_internal.h"
#include "ngh_rows.h"

// Products and sums contract to fused multiply-adds here: one rounding less each, and the backward kernel is
// as near to its vector instructions as to memory.
#pragma clang fp contract(fast)

namespace ngh {

struct NormArgs {
    const void *x, *b, *gain, *bias, *post_gain, *post_bias, *gate, *dy, *dh;
    void *h, *y, *dx, *db, *dgate;
    float* parts;                  // backward: [part][vector][part_stride] sums of a part's rows
    long long x_stride, b_stride, gate_stride, h_stride, y_stride, dy_stride, dh_stride, dx_stride, db_stride, dgate_stride, part_stride;
    unsigned rows, width, gate_rows;
    unsigned first_row;            // forward: of this launch
    int lanes;                     // along a row: whole wavefronts, or a power of two up to 64
    int post, param_f32;
    float eps, alpha, inv_width, width_f;      // (a mean is a quotient: a row of equal elements is all zeros behind it)
    // backward: a part (a workgroup) has rows [part * per_part, ...) of a span of consecutive rows, those of one
    // gate row or all; a group of lanes that makes up a row has per_group of them
    unsigned span_rows, parts_per_span, per_part, per_group;
    int vectors;                   // sums a part writes: gain, bias, post gain, post bias, gate (bits), in this order
    int gate_whole;                // a group has whole gate rows and writes their gradients itself
    int in_lds;                    // vectors that the workgroup keeps in LDS (bits, kVec*)
    unsigned lds_stride;           // floats from one of them to the next
};

constexpr int kVecGain = 1, kVecBias = 2, kVecPostGain = 4, kVecPostBias = 8, kVecGate = 16;

// VEC elements of a gain, bias or gate; `other` where there is none.
template <class T, int VEC, bool RAGGED, bool FORWARD>
__device__ __forceinline__ void load_param(const void* p, long long at, unsigned col, int count, bool f32, float other, float (&out)[VEC]) {
    if (!p) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) out[i] = other;
    } else if (f32) {
        load_piece<float, VEC, RAGGED>((const float*)p + at, count, false, out);
    } else {
        // (in the forward pass, where every row loads them; vectors in fp32, and the backward pass, lost by it)
        if constexpr (RAGGED && FORWARD) load_end<T, VEC>((const T*)p + at, count, col > 0, out);
        else load_piece<T, VEC, RAGGED>((const T*)p + at, count, false, out);
    }
}

template <class T, int VEC, int C, int THREADS, bool SEVERAL, bool RAGGED, bool LAYER>
__global__ __launch_bounds__(THREADS) void block_norm_kernel(NormArgs a) {
    __shared__ RowSums sh[SEVERAL ? 32 : 1];
    int phase = 0;
    clear_row_sums<SEVERAL>(sh);
    const unsigned lanes = a.lanes;
    const unsigned lane = SEVERAL ? threadIdx.x : threadIdx.x & (lanes - 1);
    const unsigned row = a.first_row + (SEVERAL ? blockIdx.x : blockIdx.x * (THREADS / lanes) + threadIdx.x / lanes);
    const bool live = row < a.rows;                      // (idle lanes still take part in the reductions)
    const unsigned n = live ? row : 0;
    const bool inside = n + 1 < a.rows && a.width >= VEC;
    typename VecOf<T, VEC>::type rx[C], rb[C];
    int in[C];                                           // elements of each piece
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const unsigned col = (c * lanes + lane) * VEC;
        in[c] = live ? piece_count<VEC, RAGGED>(col, a.width) : 0;
        rx[c] = load_raw<T, VEC, RAGGED>((const T*)a.x + (long long)n * a.x_stride + col, in[c], inside);
        rb[c] = load_raw<T, VEC, RAGGED>((const T*)a.b + (long long)n * a.b_stride + col, a.b ? in[c] : 0, inside);
    }
    // Gains, biases and gate are asked for with the rows rather than behind the reductions, where each costs its
    // latency again: 16384 rows of 4096 bf16 elements 98 us, 103 then.
    // Not where a workgroup has more than 512 lanes: without their registers two such workgroups fit a compute unit
    // (8192 rows of 8192 bf16 elements 145 us, 102 so); nor on any boundary, where their masks wait for them
    // ([16384, 4095] 152 us, 147 so).
    constexpr bool kEarly = THREADS <= 512 && !RAGGED;
    float p[C][VEC], q[C][VEC], g[C][VEC], w[C][VEC], z[C][VEC];
    auto load_post = [&](int c) {
        const unsigned col = (c * lanes + lane) * VEC;
        load_param<T, VEC, RAGGED, true>(a.post_gain, col, col, in[c], a.param_f32, 1.0f, p[c]);
        load_param<T, VEC, RAGGED, true>(a.post_bias, col, col, in[c], a.param_f32, 0.0f, q[c]);
    };
    auto load_gate = [&](int c) {
        const unsigned col = (c * lanes + lane) * VEC;
        load_param<T, VEC, RAGGED, true>(a.gate, a.gate ? (long long)(n / a.gate_rows) * a.gate_stride + col : 0, col, in[c], a.param_f32, 1.0f, g[c]);
    };
    auto load_gain = [&](int c) {
        const unsigned col = (c * lanes + lane) * VEC;
        load_param<T, VEC, RAGGED, true>(a.gain, col, col, in[c], a.param_f32, 1.0f, w[c]);
        load_param<T, VEC, RAGGED, true>(a.bias, col, col, in[c], a.param_f32, 0.0f, z[c]);
    };
    if constexpr (kEarly) {
#pragma unroll
        for (int c = 0; c < C; ++c) {
            if (!in[c]) continue;
            if (a.post) load_post(c);
            load_gate(c);
            if (a.y) load_gain(c);
        }
    }
    float v[C][VEC], x[C][VEC];
#pragma unroll
    for (int c = 0; c < C; ++c) {
        to_float<T, VEC, RAGGED>(rx[c], in[c], x[c]);
        to_float<T, VEC, RAGGED>(rb[c], in[c], v[c]);
    }
    if (a.post) {
        float mean = 0.0f;
        if (LAYER) {
            float s[1] = {0.0f};
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int i = 0; i < VEC; ++i) s[0] += v[c][i];
            row_sums<1, SEVERAL>(s, lanes, sh, phase);
            mean = s[0] / a.width_f;
        }
        float s[1] = {0.0f};
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                v[c][i] = (RAGGED ? i < in[c] : in[c] > 0) ? v[c][i] - mean : 0.0f;
                s[0] += v[c][i] * v[c][i];
            }
        row_sums<1, SEVERAL>(s, lanes, sh, phase);
        const float r = 1.0f / sqrtf(s[0] * a.inv_width + a.eps);
#pragma unroll
        for (int c = 0; c < C; ++c) {
            if (in[c]) {
                if constexpr (!kEarly) load_post(c);
#pragma unroll
                for (int i = 0; i < VEC; ++i) v[c][i] = v[c][i] * r * p[c][i] + q[c][i];
            }
        }
    }
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const unsigned col = (c * lanes + lane) * VEC;
        if (in[c]) {
            if constexpr (!kEarly) load_gate(c);
#pragma unroll
            for (int i = 0; i < VEC; ++i) v[c][i] = a.alpha * x[c][i] + v[c][i] * g[c][i];
            if (a.h) store_piece<T, VEC, RAGGED>((T*)a.h + (long long)n * a.h_stride + col, in[c], v[c]);
        }
    }
    if (!a.y) return;
    float mean = 0.0f;
    if (LAYER) {
        float s[1] = {0.0f};
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int i = 0; i < VEC; ++i) s[0] += v[c][i];
        row_sums<1, SEVERAL>(s, lanes, sh, phase);
        mean = s[0] / a.width_f;
    }
    float s[1] = {0.0f};
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            v[c][i] = (RAGGED ? i < in[c] : in[c] > 0) ? v[c][i] - mean : 0.0f;
            s[0] += v[c][i] * v[c][i];
        }
    row_sums<1, SEVERAL>(s, lanes, sh, phase);
    const float r = 1.0f / sqrtf(s[0] * a.inv_width + a.eps);
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const unsigned col = (c * lanes + lane) * VEC;
        if (in[c]) {
            if constexpr (!kEarly) load_gain(c);
#pragma unroll
            for (int i = 0; i < VEC; ++i) v[c][i] = v[c][i] * r * w[c][i] + z[c][i];
            store_piece<T, VEC, RAGGED>((T*)a.y + (long long)n * a.y_stride + col, in[c], v[c]);
        }
    }
}

// Backward.  A workgroup (not SEVERAL: each group of lanes of it) takes the rows of a part one after the
// other, the next row in flight while one is worked on, and keeps the part's sums over rows in registers;
// they go to a.parts at its end (of the groups of a workgroup joined in LDS, in order), and
// block_norm_merge_kernel adds the parts in order.  BIAS: the sums of dz and dq are wanted.
template <class T, int VEC, int C, int THREADS, bool SEVERAL, bool RAGGED, bool LAYER, bool BIAS>
__global__ __launch_bounds__(THREADS) __attribute__((amdgpu_waves_per_eu(4))) void block_norm_grad_kernel(NormArgs a) {
    typedef typename VecOf<T, VEC>::type Raw;
    __shared__ RowSums sh[SEVERAL ? 32 : 1];
    extern __shared__ float4 lds4[];
    float* lds = reinterpret_cast<float*>(lds4);
    int phase = 0;
    clear_row_sums<SEVERAL>(sh);
    const unsigned lanes = a.lanes;
    const unsigned lane = SEVERAL ? threadIdx.x : threadIdx.x & (lanes - 1);
    const unsigned part = blockIdx.x, group = SEVERAL ? 0 : threadIdx.x / lanes;
    const unsigned span = part / a.parts_per_span;
    const unsigned part_first = span * a.span_rows + (part - span * a.parts_per_span) * a.per_part;
    const unsigned part_end = min(min(a.rows, (span + 1) * a.span_rows), part_first + a.per_part);
    const unsigned first = part_first + group * a.per_group;
    const unsigned last = max(first, min(part_end, first + a.per_group));
    float sw[C][VEC], sp[C][VEC], sg[C][VEC], sz[BIAS ? C : 1][VEC], sq[BIAS ? C : 1][VEC];
    int in[C];                                           // elements of each piece
#pragma unroll
    for (int c = 0; c < C; ++c) {
        in[c] = piece_count<VEC, RAGGED>((c * lanes + lane) * VEC, a.width);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            sw[c][i] = sp[c][i] = sg[c][i] = 0.0f;
            if constexpr (BIAS) sz[c][i] = sq[c][i] = 0.0f;
        }
    }
    Raw rh[C], rt[C], rb[C], rd[C];
    auto fetch = [&](unsigned n, bool live) {
        const bool inside = n + 1 < a.rows && a.width >= VEC;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const unsigned col = (c * lanes + lane) * VEC;
            const int count = live ? in[c] : 0;
            rh[c] = load_raw<T, VEC, RAGGED>((const T*)a.h + (long long)n * a.h_stride + col, a.dy ? count : 0, inside);
            rt[c] = load_raw<T, VEC, RAGGED>((const T*)a.dy + (long long)n * a.dy_stride + col, a.dy ? count : 0, inside);
            rb[c] = load_raw<T, VEC, RAGGED>((const T*)a.b + (long long)n * a.b_stride + col, a.b ? count : 0, inside);
            rd[c] = load_raw<T, VEC, RAGGED>((const T*)a.dh + (long long)n * a.dh_stride + col, a.dh ? count : 0, inside);
        }
    };
    fetch(first, first < last);
    float* lds_post_gain = lds + (a.in_lds & kVecGain ? a.lds_stride : 0);
    float* lds_post_bias = lds_post_gain + (a.in_lds & kVecPostGain ? a.lds_stride : 0);
    float* lds_gate = lds_post_bias + (a.in_lds & kVecPostBias ? a.lds_stride : 0);
    // Gains, bias and gate are needed right behind the reductions, several times a row: a lane keeps its pieces of
    // them in LDS (where registers are short; every lane reads back what it wrote, so there is no barrier).  A
    // row of 4096 bf16 elements, 16384 of them: 299 us with loads from the second-level cache each time, 202 so.
    if (a.in_lds) {
#pragma unroll
        for (int c = 0; c < C; ++c) {
            if (!in[c]) continue;
            const unsigned col = (c * lanes + lane) * VEC;
            float w[VEC], p[VEC], q[VEC], g[VEC];
            if (a.in_lds & kVecGain) load_param<T, VEC, RAGGED, false>(a.gain, col, col, in[c], a.param_f32, 1.0f, w);
            if (a.in_lds & kVecPostGain) load_param<T, VEC, RAGGED, false>(a.post_gain, col, col, in[c], a.param_f32, 1.0f, p);
            if (a.in_lds & kVecPostBias) load_param<T, VEC, RAGGED, false>(a.post_bias, col, col, in[c], a.param_f32, 0.0f, q);
            if (a.in_lds & kVecGate)                     // (a part's rows share a gate row where the gate is copied)
                load_param<T, VEC, RAGGED, false>(a.gate, (long long)(part_first / a.gate_rows) * a.gate_stride + col, col, in[c], a.param_f32, 1.0f, g);
            if (a.in_lds & kVecGain) store_from_float<float, VEC>(lds + col, w);
            if (a.in_lds & kVecPostGain) store_from_float<float, VEC>(lds_post_gain + col, p);
            if (a.in_lds & kVecPostBias) store_from_float<float, VEC>(lds_post_bias + col, q);
            if (a.in_lds & kVecGate) store_from_float<float, VEC>(lds_gate + col, g);
        }
    }
    auto param = [&](int bit, const float* copy, const void* p, long long at, unsigned col, int count, float other, float (&out)[VEC]) {
        if (a.in_lds & bit) load_as_float<float, VEC>(copy + col, out);
        else load_param<T, VEC, RAGGED, false>(p, at, col, count, a.param_f32, other, out);
    };
    // (every group of lanes of a workgroup makes the same number of turns)
    for (unsigned turn = 0; turn < a.per_group; ++turn) {
        const bool live = first + turn < last;
        if constexpr (SEVERAL) {
            if (!live) break;
        }
        const unsigned n = first + turn;
        float h[C][VEC], t[C][VEC], b[C][VEC], d[C][VEC];
#pragma unroll
        for (int c = 0; c < C; ++c) {
            take_piece<T, VEC, RAGGED>(rh[c], in[c], h[c]);
            take_piece<T, VEC, RAGGED>(rt[c], in[c], t[c]);
            take_piece<T, VEC, RAGGED>(rb[c], in[c], b[c]);
            take_piece<T, VEC, RAGGED>(rd[c], in[c], d[c]);
        }
        fetch(n + 1, n + 1 < last);
        float brs = 1.0f;
        if (LAYER) {
            float s[2] = {0.0f, 0.0f};
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    s[0] += h[c][i];
                    s[1] += b[c][i];
                }
            row_sums<2, SEVERAL>(s, lanes, sh, phase);
            const float hmean = s[0] / a.width_f, bmean = a.post ? s[1] / a.width_f : 0.0f;
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    h[c][i] = (RAGGED ? i < in[c] : in[c] > 0) ? h[c][i] - hmean : 0.0f;
                    b[c][i] = (RAGGED ? i < in[c] : in[c] > 0) ? b[c][i] - bmean : 0.0f;
                }
        }
        {
            // sums of h^2, t h (t = dy w), b^2 and, for the layer norm, t
            float s[LAYER ? 4 : 3] = {};
#pragma unroll
            for (int c = 0; c < C; ++c) {
                float w[VEC];
                const unsigned col = (c * lanes + lane) * VEC;
                if (in[c]) {
                    param(kVecGain, lds, a.gain, col, col, in[c], 1.0f, w);
                } else {
#pragma unroll
                    for (int i = 0; i < VEC; ++i) w[i] = 0.0f;
                }
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    const float tw = t[c][i] * w[i];
                    s[0] += h[c][i] * h[c][i];
                    s[1] += tw * h[c][i];
                    s[2] += b[c][i] * b[c][i];
                    if constexpr (LAYER) s[3] += tw;
                }
            }
            row_sums<LAYER ? 4 : 3, SEVERAL>(s, lanes, sh, phase);
            const float r = 1.0f / sqrtf(s[0] * a.inv_width + a.eps);
            if (a.post) brs = 1.0f / sqrtf(s[2] * a.inv_width + a.eps);
            if (a.dy && live) {
                const float along = s[1] * r * a.inv_width;              // mean(t hh)
                const float level = LAYER ? s[LAYER ? 3 : 0] * a.inv_width : 0.0f;
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    float w[VEC];
                    const unsigned col = (c * lanes + lane) * VEC;
                    if (in[c]) {
                        param(kVecGain, lds, a.gain, col, col, in[c], 1.0f, w);
#pragma unroll
                        for (int i = 0; i < VEC; ++i) {
                            const float hh = h[c][i] * r;
                            sw[c][i] += t[c][i] * hh;
                            if constexpr (BIAS) sz[c][i] += t[c][i];
                            if (!RAGGED || i < in[c]) d[c][i] += r * (t[c][i] * w[i] - hh * along - (LAYER ? level : 0.0f));
                        }
                    }
                }
            }
        }
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const unsigned col = (c * lanes + lane) * VEC;
            if (live && in[c] && a.dx) {
                float o[VEC];
#pragma unroll
                for (int i = 0; i < VEC; ++i) o[i] = a.alpha * d[c][i];
                store_piece<T, VEC, RAGGED>((T*)a.dx + (long long)n * a.dx_stride + col, in[c], o);
            }
        }
        if (!a.db) continue;
        const unsigned gate_row = a.gate && live ? n / a.gate_rows : 0;
        float s[LAYER ? 2 : 1] = {};
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const unsigned col = (c * lanes + lane) * VEC;
            if (live && in[c]) {
                float g[VEC], p[VEC], q[VEC];
                param(kVecGate, lds_gate, a.gate, a.gate ? (long long)gate_row * a.gate_stride + col : 0, col, in[c], 1.0f, g);
                param(kVecPostGain, lds_post_gain, a.post_gain, col, col, in[c], 1.0f, p);
                param(kVecPostBias, lds_post_bias, a.post_bias, col, col, in[c], 0.0f, q);
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    const float bh = b[c][i] * brs;
                    b[c][i] = bh;
                    sg[c][i] += d[c][i] * (bh * p[i] + q[i]);
                    const float e = d[c][i] * g[i];
                    sp[c][i] += e * bh;
                    if constexpr (BIAS) sq[c][i] += e;
                    d[c][i] = e * p[i];
                    s[0] += d[c][i] * bh;
                    if constexpr (LAYER) s[LAYER ? 1 : 0] += d[c][i];
                }
            }
        }
        if (a.post) {
            row_sums<LAYER ? 2 : 1, SEVERAL>(s, lanes, sh, phase);
            const float along = s[0] * a.inv_width, level = LAYER ? s[LAYER ? 1 : 0] * a.inv_width : 0.0f;
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int i = 0; i < VEC; ++i) d[c][i] = brs * (d[c][i] - b[c][i] * along - (LAYER ? level : 0.0f));
        }
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const unsigned col = (c * lanes + lane) * VEC;
            if (live && in[c]) store_piece<T, VEC, RAGGED>((T*)a.db + (long long)n * a.db_stride + col, in[c], d[c]);
        }
        if (a.gate_whole && a.dgate && (n + 1) % a.gate_rows == 0) {
            // the last row of a gate row: its gradient is complete
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const unsigned col = (c * lanes + lane) * VEC;
                if (live && in[c]) {
                    const long long at = (long long)gate_row * a.dgate_stride + col;
                    if (a.param_f32) store_piece<float, VEC, RAGGED>((float*)a.dgate + at, in[c], sg[c]);
                    else store_piece<T, VEC, RAGGED>((T*)a.dgate + at, in[c], sg[c]);
                }
#pragma unroll
                for (int i = 0; i < VEC; ++i) sg[c][i] = live ? 0.0f : sg[c][i];
            }
        }
    }
    if (!a.vectors) return;
    float* out = a.parts + (size_t)part * __popc(a.vectors) * a.part_stride;
    if constexpr (SEVERAL) {
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const unsigned col = (c * lanes + lane) * VEC;
            if (!in[c]) continue;
            float* to = out + col;
            if (a.vectors & kVecGain) store_from_float<float, VEC>(to, sw[c]), to += a.part_stride;
            if constexpr (BIAS) {
                if (a.vectors & kVecBias) store_from_float<float, VEC>(to, sz[c]), to += a.part_stride;
            }
            if (a.vectors & kVecPostGain) store_from_float<float, VEC>(to, sp[c]), to += a.part_stride;
            if constexpr (BIAS) {
                if (a.vectors & kVecPostBias) store_from_float<float, VEC>(to, sq[c]), to += a.part_stride;
            }
            if (a.vectors & kVecGate) store_from_float<float, VEC>(to, sg[c]);
        }
    } else {
        static_assert(C == 1, "a group of lanes holds one piece a lane");
        __shared__ float joined[THREADS * VEC];              // [VEC][groups][lanes]
        auto join = [&](const float (&v)[VEC]) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < VEC; ++i) joined[i * THREADS + threadIdx.x] = v[i];
            __syncthreads();
            if (group == 0 && in[0]) {
                float o[VEC];
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    o[i] = v[i];
                    for (unsigned g = lane + lanes; g < THREADS; g += lanes) o[i] += joined[i * THREADS + g];
                }
                store_from_float<float, VEC>(out + lane * VEC, o);
            }
            out += a.part_stride;
        };
        if (a.vectors & kVecGain) join(sw[0]);
        if constexpr (BIAS) {
            if (a.vectors & kVecBias) join(sz[0]);
        }
        if (a.vectors & kVecPostGain) join(sp[0]);
        if constexpr (BIAS) {
            if (a.vectors & kVecPostBias) join(sq[0]);
        }
        if (a.vectors & kVecGate) join(sg[0]);
    }
}

struct NormMergeArgs {
    const float* parts;
    long long part_stride;
    unsigned width, per_part_vectors, n_parts, parts_per_span, gates;            // gates: 1 when the last vector is the gate's
    unsigned first;                // of the sums this launch makes (its grid's second axis is limited)
    void* out[4];                  // of the vectors other than the gate
    void* dgate;
    long long dgate_stride;
};

// Sums the parts of a vector (over all of them) or of a gate row (over those of its span): 16 columns a
// workgroup, 64 lanes a column each adding every 64th part, joined in LDS in order.
constexpr int kMergeCols = 16;

template <class T>
__global__ __launch_bounds__(1024) void block_norm_merge_kernel(NormMergeArgs a) {
    __shared__ float sh[64][kMergeCols + 1];
    const unsigned x = threadIdx.x % kMergeCols, y = threadIdx.x / kMergeCols;
    const unsigned col = blockIdx.x * kMergeCols + x;
    const unsigned plain = a.per_part_vectors - a.gates;
    const unsigned which = a.first + blockIdx.y;
    const bool gate = which >= plain;
    const unsigned vec = gate ? plain : which, span = gate ? which - plain : 0;
    const unsigned begin = gate ? span * a.parts_per_span : 0;
    const unsigned count = gate ? a.parts_per_span : a.n_parts;
    const float* from = a.parts + ((size_t)begin * a.per_part_vectors + vec) * a.part_stride + col;
    const size_t step = (size_t)a.per_part_vectors * a.part_stride;
    float acc = 0.0f;
    if (col < a.width)
        for (unsigned p = y; p < count; p += 64 * 8) {
            float v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = p + 64 * k < count ? from[(p + 64 * k) * step] : 0.0f;
#pragma unroll
            for (int k = 0; k < 8; ++k) acc += v[k];
        }
    sh[y][x] = acc;
    __syncthreads();
    if (y < 8) {
        acc = 0.0f;
#pragma unroll
        for (int k = 0; k < 8; ++k) acc += sh[y * 8 + k][x];
    }
    __syncthreads();
    if (y < 8) sh[y][x] = acc;
    __syncthreads();
    if (y != 0 || col >= a.width) return;
    acc = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; ++k) acc += sh[k][x];
    if (gate) ((T*)a.dgate)[(long long)span * a.dgate_stride + col] = (T)acc;
    else ((T*)a.out[vec])[col] = (T)acc;
}

// The shape of the kernel that a row takes: `pieces` pieces of `vec` elements a lane on `lanes` lanes (whole
// wavefronts, or a power of two up to 64).  ragged: rows that do not start, or end, on 16-byte boundaries.
struct NormShape {
    int vec, pieces, lanes;
    bool ragged;
    bool several() const { return lanes > 64; }
    unsigned threads() const { return several() ? (unsigned)lanes : 256u; }
    unsigned rows_a_workgroup() const { return several() ? 1u : 256u / (unsigned)lanes; }
};

// One translation unit for each storage type.
enum NormPass { kNormForward, kNormBackward, kNormBackwardBias };
NGH_INTERNAL int launch_norm_f32(const NormShape& s, const NormArgs& a, NormPass pass, bool layer, unsigned grid, hipStream_t stream);
NGH_INTERNAL int launch_norm_f16(const NormShape& s, const NormArgs& a, NormPass pass, bool layer, unsigned grid, hipStream_t stream);
NGH_INTERNAL int launch_norm_bf16(const NormShape& s, const NormArgs& a, NormPass pass, bool layer, unsigned grid, hipStream_t stream);

template <class T, int VEC, int C, int THREADS, bool SEVERAL, bool RAGGED, bool LAYER>
void launch_norm_kernel(const NormShape& s, const NormArgs& a, NormPass pass, unsigned grid, hipStream_t stream) {
    const dim3 block(s.threads());
    const unsigned lds = (unsigned)__builtin_popcount((unsigned)a.in_lds) * a.lds_stride * 4;
    if (pass == kNormForward) hipLaunchKernelGGL((block_norm_kernel<T, VEC, C, THREADS, SEVERAL, RAGGED, LAYER>), dim3(grid), block, 0, stream, a);
    else if (pass == kNormBackward)
        hipLaunchKernelGGL((block_norm_grad_kernel<T, VEC, C, THREADS, SEVERAL, RAGGED, LAYER, false>), dim3(grid), block, lds, stream, a);
    else hipLaunchKernelGGL((block_norm_grad_kernel<T, VEC, C, THREADS, SEVERAL, RAGGED, LAYER, true>), dim3(grid), block, lds, stream, a);
}

// The pieces a lane may hold: one (rows of up to 16 KiB: at most 1024 lanes), two, and four of 4 elements.
// Pieces of 4 elements where 16 bytes are 8: only what shape_of asks for (ragged rows, backward).
template <class T, bool RAGGED, bool LAYER>
int launch_norm_shape(const NormShape& s, const NormArgs& a, NormPass pass, unsigned grid, hipStream_t stream) {
    constexpr int kVec = 16 / sizeof(T);
    if (s.vec != kVec) {
        if constexpr (RAGGED && kVec == 8) {
            const dim3 block(s.threads());
            const unsigned lds = (unsigned)__builtin_popcount((unsigned)a.in_lds) * a.lds_stride * 4;
            if (!s.several() && pass == kNormBackward)
                hipLaunchKernelGGL((block_norm_grad_kernel<T, 4, 1, 256, false, true, LAYER, false>), dim3(grid), block, lds, stream, a);
            else if (!s.several())
                hipLaunchKernelGGL((block_norm_grad_kernel<T, 4, 1, 256, false, true, LAYER, true>), dim3(grid), block, lds, stream, a);
            else if (s.lanes <= 512)
                hipLaunchKernelGGL((block_norm_grad_kernel<T, 4, 1, 512, true, true, LAYER, true>), dim3(grid), block, lds, stream, a);
            else
                hipLaunchKernelGGL((block_norm_grad_kernel<T, 4, 1, 1024, true, true, LAYER, true>), dim3(grid), block, lds, stream, a);
        }
    } else if (s.pieces == 1) {
        if (!s.several()) launch_norm_kernel<T, kVec, 1, 256, false, RAGGED, LAYER>(s, a, pass, grid, stream);
        else if (s.lanes <= 256) launch_norm_kernel<T, kVec, 1, 256, true, RAGGED, LAYER>(s, a, pass, grid, stream);
        else if (s.lanes <= 512) launch_norm_kernel<T, kVec, 1, 512, true, RAGGED, LAYER>(s, a, pass, grid, stream);
        else launch_norm_kernel<T, kVec, 1, 1024, true, RAGGED, LAYER>(s, a, pass, grid, stream);
    } else if (s.pieces == 2) {
        launch_norm_kernel<T, kVec, 2, 1024, true, RAGGED, LAYER>(s, a, pass, grid, stream);
    } else {
        if constexpr (kVec == 4) launch_norm_kernel<T, kVec, 4, 1024, true, RAGGED, LAYER>(s, a, pass, grid, stream);
    }
    NGH_HIP_TRY(hipGetLastError());
    return NGH_OK;
}

template <class T>
int launch_norm(const NormShape& s, const NormArgs& a, NormPass pass, bool layer, unsigned grid, hipStream_t stream) {
    if (s.ragged)
        return layer ? launch_norm_shape<T, true, true>(s, a, pass, grid, stream) : launch_norm_shape<T, true, false>(s, a, pass, grid, stream);
    return layer ? launch_norm_shape<T, false, true>(s, a, pass, grid, stream) : launch_norm_shape<T, false, false>(s, a, pass, grid, stream);
}

}  // namespace ngh
