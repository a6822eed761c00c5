// ngh_block_norm, ngh_block_norm_grad: checks, the shape of the kernels and the launches.  The
// mathematics and the kernels are in ngh_block_norm.h.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "ngh_block_norm.h"

namespace ngh {
namespace {

int size_of(int dtype) { return dtype == NGH_F32 ? 4 : (dtype == NGH_F16 || dtype == NGH_BF16) ? 2 : 0; }

struct View {
    const char* name;
    const void* p;
    int64_t rows, stride;
    int item;
    bool written;
};

constexpr int kMostViews = 20;

struct Views {
    View v[kMostViews];
    int n = 0;
    int in_place = -1, over = -1;      // the output that may be the same view as an input, and that input
};

// Everything the call touches.
void views_of(const ngh_block_norm_spec* s, bool grad, Views& views) {
    View* v = views.v;
    const int e = size_of(s->dtype), q = size_of(s->param_dtype);
    const int64_t gates = s->gate_rows > 0 ? s->rows / s->gate_rows : 0;
    int n = 0;
    auto add = [&](const char* name, const void* p, int64_t rows, int64_t stride, int item, bool written) {
        if (p) v[n++] = View{name, p, rows, stride, item, written};
    };
    add("gain", s->gain, 1, s->width, q, false);
    add("post_gain", s->post_gain, 1, s->width, q, false);
    add("post_bias", s->post_bias, 1, s->width, q, false);
    add("gate", s->gate, gates, s->gate_stride, q, false);
    add("b", s->b, s->rows, s->b_stride, e, false);
    if (!grad && s->h) views.in_place = n;
    add("h", s->h, s->rows, s->h_stride, e, !grad);
    if (!grad) {
        add("bias", s->bias, 1, s->width, q, false);
        if (s->x) views.over = n;
        add("x", s->x, s->rows, s->x_stride, e, false);
        add("y", s->y, s->rows, s->y_stride, e, true);
    } else {
        add("dy", s->dy, s->rows, s->dy_stride, e, false);
        if (s->dh) views.over = n;
        add("dh", s->dh, s->rows, s->dh_stride, e, false);
        if (s->dx) views.in_place = n;
        add("dx", s->dx, s->rows, s->dx_stride, e, true);
        add("db", s->db, s->rows, s->db_stride, e, true);
        add("dgain", s->dgain, 1, s->width, q, true);
        add("dbias", s->dbias, 1, s->width, q, true);
        add("dpost_gain", s->dpost_gain, 1, s->width, q, true);
        add("dpost_bias", s->dpost_bias, 1, s->width, q, true);
        add("dgate", s->dgate, gates, s->dgate_stride, q, true);
        add("workspace", s->workspace, 1, (int64_t)s->workspace_bytes, 1, true);
    }
    views.n = n;
}

int check(const ngh_block_norm_spec* s, bool grad, const char* what, Views& views) {
    if (!s) return report(NGH_E_INVALID, "%s: spec is NULL", what);
    if (s->abi_version != NGH_ABI_VERSION)
        return report(NGH_E_INVALID, "%s: abi_version %d, this library is %d", what, s->abi_version, NGH_ABI_VERSION);
    if (s->kind != NGH_NORM_RMS && s->kind != NGH_NORM_LAYER) return report(NGH_E_INVALID, "%s: kind %d", what, s->kind);
    if (!size_of(s->dtype) || (s->param_dtype != s->dtype && s->param_dtype != NGH_F32))
        return report(NGH_E_INVALID, "%s: dtype %d with parameters of dtype %d (NGH_F32, NGH_F16, NGH_BF16; parameters the same or NGH_F32)", what,
                      s->dtype, s->param_dtype);
    if (s->rows < 0 || s->width < 1) return report(NGH_E_INVALID, "%s: rows %lld, width %lld", what, (long long)s->rows, (long long)s->width);
    if (s->width > NGH_BLOCK_NORM_MAX_WIDTH || s->rows >= (1LL << 31) - 65536)
        return report(NGH_E_UNSUPPORTED, "%s: %lld rows of %lld elements", what, (long long)s->rows, (long long)s->width);
    if (!(s->eps >= 0.0f) || !std::isfinite(s->eps) || !std::isfinite(s->residual_scale))
        return report(NGH_E_INVALID, "%s: eps %g, residual_scale %g", what, (double)s->eps, (double)s->residual_scale);
    const bool block = s->b != nullptr || (grad && s->db != nullptr);
    if (!block && (s->post_norm || s->post_gain || s->post_bias || s->gate))
        return report(NGH_E_INVALID, "%s: a norm, gain, bias or gate after the block, and no block output", what);
    if (!s->post_norm && (s->post_gain || s->post_bias))
        return report(NGH_E_INVALID, "%s: a gain or bias after the block without post_norm", what);
    if (s->gate) {
        if (s->gate_rows < 1 || s->gate_rows >= (1LL << 31) || s->rows % s->gate_rows) return report(NGH_E_INVALID, "%s: gate_rows %lld of %lld rows", what, (long long)s->gate_rows, (long long)s->rows);
    } else if (s->gate_rows) {
        return report(NGH_E_INVALID, "%s: gate_rows without a gate", what);
    }
    if (!grad) {
        if (!s->x && s->rows) return report(NGH_E_INVALID, "%s: x is NULL", what);
        if (!s->h && !s->y && s->rows) return report(NGH_E_INVALID, "%s: neither h nor y", what);
        if (!s->y && (s->gain || s->bias)) return report(NGH_E_INVALID, "%s: a gain or bias without y", what);
    } else if (s->rows) {
        if (!s->dy && !s->dh) return report(NGH_E_INVALID, "%s: neither dy nor dh", what);
        if (s->dy && !s->h) return report(NGH_E_INVALID, "%s: dy without h", what);
        if ((s->b != nullptr) != (s->db != nullptr)) return report(NGH_E_INVALID, "%s: b and db come together", what);
        if (!s->dx && !s->db) return report(NGH_E_INVALID, "%s: neither dx nor db", what);
        if (!s->dy && (s->gain || s->dgain || s->dbias)) return report(NGH_E_INVALID, "%s: the gain or its gradient without dy", what);
        if (!s->post_norm && (s->dpost_gain || s->dpost_bias)) return report(NGH_E_INVALID, "%s: a gradient of the norm after the block without post_norm", what);
        if (s->dgate && !s->gate) return report(NGH_E_INVALID, "%s: dgate without a gate", what);
    }
    views_of(s, grad, views);
    const View* v = views.v;
    const int n = views.n;
    for (int i = 0; i < n; ++i) {
        if ((uintptr_t)v[i].p % v[i].item) return report(NGH_E_INVALID, "%s: %s is not aligned to its elements", what, v[i].name);
        if (v[i].rows > 1 && v[i].stride < s->width) return report(NGH_E_INVALID, "%s: stride %lld of %s below the width", what, (long long)v[i].stride, v[i].name);
        if (v[i].stride >= (1LL << 40)) return report(NGH_E_UNSUPPORTED, "%s: stride of %s too large", what, v[i].name);
    }
    auto bytes = [&](const View& a) {
        return a.item == 1 ? (unsigned long long)a.stride : span_bytes(a.rows, s->width, a.stride, a.item);      // (item 1: the workspace)
    };
    for (int i = 0; i < n; ++i)
        for (int j = 0; j < n; ++j) {
            if (i == j || !v[i].written || (v[j].written && j < i)) continue;
            if (!spans_overlap(v[i].p, bytes(v[i]), v[j].p, bytes(v[j]))) continue;
            // a row is read whole before it is written: the stream and its gradient may be updated in place (these two
            // views and no others, whatever else has their address)
            const bool same = v[i].p == v[j].p && (v[i].stride == v[j].stride || s->rows == 1);
            if (same && i == views.in_place && j == views.over) continue;
            return report(NGH_E_INVALID, "%s: %s overlaps %s", what, v[i].name, v[j].name);
        }
    return NGH_OK;
}

NormShape shape_of(const ngh_block_norm_spec* s, const Views& views, NormPass pass) {
    NormShape f;
    const View* v = views.v;
    const int n = views.n;
    const int vec = 16 / size_of(s->dtype);
    bool whole = s->width % vec == 0;
    for (int i = 0; i < n; ++i) {
        if (v[i].item == 1) continue;
        const int piece = std::min(16, vec * v[i].item);
        whole = whole && (uintptr_t)v[i].p % piece == 0 && (v[i].rows <= 1 || v[i].stride * v[i].item % piece == 0);
    }
    f.ragged = !whole;
    // Backward, ragged rows of 16 bits: pieces of 8 elements do not fit the registers with the sums of the biases
    // (16384 layer norms of 2050 bf16 elements 302 us, 234 with pieces of 4; without those sums 158 and 235), nor
    // where rows share a wavefront (65536 rows of 100: 52 and 34 us; of 250: 71 and 63).
    f.vec = f.ragged && ((pass == kNormBackward && s->width <= 64 * 4) || (pass == kNormBackwardBias && s->width <= 1024 * 4)) ? 4 : vec;
    f.pieces = 1;
    while (1024 * f.vec * f.pieces < s->width) f.pieces *= 2;
    const int per_lane = f.vec * f.pieces;
    f.lanes = 1;
    while (f.lanes < 64 && f.lanes * per_lane < s->width) f.lanes *= 2;
    if (f.lanes * per_lane < s->width) f.lanes = (int)((s->width + per_lane * 64 - 1) / (per_lane * 64)) * 64;
    return f;
}

void fill_args(const ngh_block_norm_spec* s, const NormShape& f, NormArgs& a) {
    a = NormArgs{};
    a.x = s->x, a.b = s->b, a.gain = s->gain, a.bias = s->bias, a.post_gain = s->post_gain, a.post_bias = s->post_bias, a.gate = s->gate;
    a.dy = s->dy, a.dh = s->dh, a.h = s->h, a.y = s->y, a.dx = s->dx, a.db = s->db, a.dgate = s->dgate;
    a.x_stride = s->x_stride, a.b_stride = s->b_stride, a.gate_stride = s->gate_stride, a.h_stride = s->h_stride, a.y_stride = s->y_stride;
    a.dy_stride = s->dy_stride, a.dh_stride = s->dh_stride, a.dx_stride = s->dx_stride, a.db_stride = s->db_stride, a.dgate_stride = s->dgate_stride;
    a.rows = (unsigned)s->rows;
    a.width = (unsigned)s->width;
    a.gate_rows = (unsigned)std::max<int64_t>(1, s->gate_rows);
    a.lanes = f.lanes;
    a.post = s->post_norm != 0;
    a.param_f32 = s->param_dtype == NGH_F32;
    a.eps = s->eps;
    a.alpha = s->residual_scale;
    a.width_f = (float)s->width;
    a.inv_width = 1.0f / a.width_f;
}

int launch(const ngh_block_norm_spec* s, const NormShape& f, const NormArgs& a, NormPass pass, unsigned grid, hipStream_t stream) {
    const bool layer = s->kind == NGH_NORM_LAYER;
    if (s->dtype == NGH_F32) return launch_norm_f32(f, a, pass, layer, grid, stream);
    if (s->dtype == NGH_F16) return launch_norm_f16(f, a, pass, layer, grid, stream);
    return launch_norm_bf16(f, a, pass, layer, grid, stream);
}

// How the rows of the backward pass are dealt, and where the sums of the parts lie.
struct GradPlan {
    NormShape shape;
    unsigned span_rows, spans, parts_per_span, per_part, per_group, parts;
    int vectors, count;
    bool gate_whole, bias;
    size_t part_stride, bytes;
};

GradPlan plan_grad(const ngh_block_norm_spec* s, const Views& views, int cus) {
    GradPlan g;
    g.vectors = (s->dgain ? kVecGain : 0) | (s->dbias ? kVecBias : 0) | (s->dpost_gain ? kVecPostGain : 0) | (s->dpost_bias ? kVecPostBias : 0);
    g.bias = s->dbias || s->dpost_bias;
    g.shape = shape_of(s, views, g.bias ? kNormBackwardBias : kNormBackward);
    const unsigned rows = (unsigned)s->rows;
    // 16 wavefronts a compute unit (what the registers allow; a workgroup of 5 takes the room of 8), but at least
    // 8 rows a part, for a part's sums are written in fp32 and read once more; fewer, down to 1, where else
    // compute units would have no part.
    const unsigned groups = g.shape.rows_a_workgroup();
    const unsigned want = 1024u / ((g.shape.threads() + 255u) / 256u * 256u) * cus;
    const unsigned least = std::min(8u, std::max(1u, rows / (2u * cus)));
    g.per_part = std::max(least, (rows + want - 1) / want);
    g.per_group = (g.per_part + groups - 1) / groups;
    const unsigned gate_rows = (unsigned)std::max<int64_t>(1, s->gate_rows);
    g.gate_whole = !s->dgate || gate_rows < 2 * g.per_group;
    g.span_rows = g.gate_whole ? std::max(1u, rows) : gate_rows;
    if (!g.gate_whole) {
        // the rows of a gate row are shared by as many parts as they fill
        g.vectors |= kVecGate;
        const unsigned parts = std::max(1u, gate_rows / g.per_part);
        g.per_group = ((gate_rows + parts - 1) / parts + groups - 1) / groups;
    } else if (s->dgate) {
        g.per_group = std::max(1u, g.per_group / gate_rows) * gate_rows;                 // (whole gate rows)
    }
    g.per_part = g.per_group * groups;
    g.count = __builtin_popcount((unsigned)g.vectors);
    g.spans = g.gate_whole ? 1 : rows / g.span_rows;
    g.parts_per_span = (g.span_rows + g.per_part - 1) / g.per_part;
    g.parts = rows ? g.spans * g.parts_per_span : 0;                 // (no rows: the merge writes zeros)
    g.part_stride = ((size_t)s->width + 7) / 8 * 8;
    g.bytes = (size_t)g.parts * g.count * g.part_stride * 4;
    return g;
}

template <class T>
int launch_merge(NormMergeArgs m, unsigned spans, hipStream_t stream) {
    const unsigned sums = m.per_part_vectors - m.gates + (m.gates ? spans : 0);
    for (m.first = 0; m.first < sums; m.first += 65535u) {
        hipLaunchKernelGGL(block_norm_merge_kernel<T>, dim3((m.width + kMergeCols - 1) / kMergeCols, std::min(65535u, sums - m.first)), dim3(1024), 0, stream, m);
        NGH_HIP_TRY(hipGetLastError());
    }
    return NGH_OK;
}

}  // namespace
}  // namespace ngh

using namespace ngh;

extern "C" {

int ngh_validate_block_norm(const ngh_block_norm_spec* spec, int32_t gradient) {
    Views views;
    return check(spec, gradient != 0, gradient ? "ngh_block_norm_grad" : "ngh_block_norm", views);
}

int ngh_block_norm(ngh_context* ctx, const ngh_block_norm_spec* spec) {
    Views views;
    const int rc = ctx ? check(spec, false, "ngh_block_norm", views) : report(NGH_E_INVALID, "ctx is NULL");
    if (rc != NGH_OK || spec->rows == 0) return rc;
    const ContextView c = view_of(ctx);
    DeviceScope scope(c.device);
    if (!scope.ok()) return report(NGH_E_RUNTIME, "ngh_block_norm: the context's device cannot be made current");
    const NormShape f = shape_of(spec, views, kNormForward);
    NormArgs a;
    fill_args(spec, f, a);
    const unsigned per_wg = f.rows_a_workgroup();
    const unsigned slice = (unsigned)(kMostThreads / f.threads()) * per_wg;
    for (; a.first_row < a.rows; a.first_row += std::min(slice, a.rows - a.first_row)) {
        const int lrc = launch(spec, f, a, kNormForward, (std::min(slice, a.rows - a.first_row) + per_wg - 1) / per_wg, c.stream);
        if (lrc != NGH_OK) return lrc;
    }
    return NGH_OK;
}

int ngh_block_norm_grad_workspace(const ngh_block_norm_spec* spec, size_t* out_bytes) {
    if (!out_bytes) return report(NGH_E_INVALID, "ngh_block_norm_grad_workspace: out_bytes is NULL");
    *out_bytes = 0;
    Views views;
    const int rc = check(spec, true, "ngh_block_norm_grad_workspace", views);
    if (rc != NGH_OK) return rc;
    // (how the rows are dealt depends on the device's compute units; enough for any number of them)
    size_t most = 256;
    for (int cus = 1; spec->rows && cus <= 1024; cus *= 2) most = std::max(most, plan_grad(spec, views, cus).bytes);
    *out_bytes = most;
    return NGH_OK;
}

int ngh_block_norm_grad(ngh_context* ctx, const ngh_block_norm_spec* spec) {
    Views views;
    const int rc = ctx ? check(spec, true, "ngh_block_norm_grad", views) : report(NGH_E_INVALID, "ctx is NULL");
    if (rc != NGH_OK) return rc;
    const ContextView c = view_of(ctx);
    DeviceScope scope(c.device);
    if (!scope.ok()) return report(NGH_E_RUNTIME, "ngh_block_norm_grad: the context's device cannot be made current");
    const GradPlan g = plan_grad(spec, views, c.cus);
    if (spec->workspace_bytes < g.bytes || (g.bytes && !spec->workspace))
        return report(NGH_E_INVALID, "ngh_block_norm_grad: workspace of %zu bytes, %zu needed", spec->workspace_bytes, g.bytes);
    if ((uintptr_t)spec->workspace % 16) return report(NGH_E_INVALID, "ngh_block_norm_grad: misaligned workspace");
    NormArgs a;
    fill_args(spec, g.shape, a);
    a.parts = (float*)spec->workspace;
    a.part_stride = (long long)g.part_stride;
    a.span_rows = g.span_rows;
    a.parts_per_span = g.parts_per_span;
    a.per_part = g.per_part;
    a.per_group = g.per_group;
    a.vectors = g.vectors;
    a.gate_whole = g.gate_whole;
    // Vectors copied to LDS, as far as 48 KiB go (64 KiB a workgroup without further ado, the reductions' words
    // among it); the gate where a part's rows share one row of it.
    a.lds_stride = (a.width + 7) / 8 * 8;
    const int wanted[4][2] = {{kVecGain, spec->gain != nullptr},
                              {kVecPostGain, spec->post_gain != nullptr},
                              {kVecGate, spec->gate != nullptr && (spec->gate_rows == spec->rows || !g.gate_whole)},
                              {kVecPostBias, spec->post_bias != nullptr}};
    size_t room = 48u << 10;
    for (const auto& w : wanted)
        if (w[1] && a.lds_stride * 4 <= room) {
            a.in_lds |= w[0];
            room -= a.lds_stride * 4;
        }
    if (spec->rows) {
        const int lrc = launch(spec, g.shape, a, g.bias ? kNormBackwardBias : kNormBackward, g.parts, c.stream);
        if (lrc != NGH_OK) return lrc;
    }
    if (!g.vectors) return NGH_OK;
    NormMergeArgs m{};
    m.parts = a.parts;
    m.part_stride = a.part_stride;
    m.width = a.width;
    m.per_part_vectors = (unsigned)g.count;
    m.n_parts = g.parts;
    m.parts_per_span = g.parts_per_span;
    m.gates = g.vectors & kVecGate ? 1 : 0;
    int k = 0;
    if (spec->dgain) m.out[k++] = spec->dgain;
    if (spec->dbias) m.out[k++] = spec->dbias;
    if (spec->dpost_gain) m.out[k++] = spec->dpost_gain;
    if (spec->dpost_bias) m.out[k++] = spec->dpost_bias;
    m.dgate = spec->dgate;
    m.dgate_stride = spec->dgate_stride;
    if (spec->param_dtype == NGH_F32) return launch_merge<float>(m, g.spans, c.stream);
    if (spec->param_dtype == NGH_F16) return launch_merge<f16_t>(m, g.spans, c.stream);
    return launch_merge<bf16_t>(m, g.spans, c.stream);
}

}  // extern "C"
