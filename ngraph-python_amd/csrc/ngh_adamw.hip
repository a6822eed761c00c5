// AdamW over many tensors at once (ngh_adamw_* in ngraph_hip.h): one launch for all of them.
//
// The plan holds a record for each tensor and, for each workgroup, which tensor and which of its
// chunks it takes, so that one large matrix and a hundred short vectors keep the chip equally busy.
// With fp32 states and gradients an element moves 28 bytes (p, m, v in and out, g in), with 8-bit
// states and bf16 gradients 14: bound by memory either way (25.6 M elements 137 us, 5.2 TB/s; 152 M
// with 8 bits 400 us, 5.3), though 8-bit states need two quotients and three roots, correctly rounded,
// for the codes of an element (four_codes).
//
// 8-bit states.  256 consecutive elements share a scale.  A wavefront holds a block, 4 consecutive
// elements a lane: the largest |moment| is a butterfly over the lanes, on the bit patterns as unsigned
// integers, which order as magnitudes and put inf and NaN on top.  The codes are defined by fp32
// arithmetic in this order, every operation rounded (the build contracts nothing):
//     m: q = rint(sqrt(|m| / s) * 127), with m's sign         stands for ((q c) |q c|) s,  c = fp32(1/127)
//     v: q = rint(sqrt(sqrt(v / s)) * 255)                    stands for ((t t) (t t)) s,  t = q fp32(1/255)
// The roots make steps proportional to a power of the value: 1.6 % at the top of a block for both, while
// only a v below (0.5 / 255)^4 = 1.5e-11 of the block's largest rounds to 0.  After one gradient far above
// the block's others that happens beside first moments that are not 0, for the largest m decays by beta1 a
// step and the largest v by beta2: the step would be m over eps (gradients of 1e-5, one of 10 once: up to 765
// times the rate, where states in fp32 take 1).  So a step stores a v above 0 as code 1 at least, and where
// it meets code 0 beside an m that is not 0 (states encoded from fp32) it divides by the root of (0.5 / 255)^4 s
// at least, the most that the code was rounded from: fp32's root is at most sqrt(2) times the one used.
// What remains is the format's own: an increase of v by less than half a step of its code is lost, so that
// v may stay at (1 - beta2) g^2 / ((1.5^4 - 1) beta2) with gradients g, at code 1, and a step reach
// 1.9 / sqrt(1 - beta2) times the rate (8 with beta2 = 0.95, 60 with 0.999).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <new>
#include <vector>

#include "ngh_internal.h"
#include "ngh_rows.h"

namespace ngh {
namespace {

constexpr int kAdamBlock = 256;
constexpr int kPer = 4;                        // elements a lane takes at a time: a wavefront takes NGH_ADAMW_BLOCK
// A workgroup takes a chunk of TURNS * 1024 elements of one tensor, a lane's TURNS pieces of it in flight together.
constexpr int kPiece = kAdamBlock * kPer;
constexpr int kTurnsMany = 4, kTurnsFew = 1;
static_assert(64 * kPer == NGH_ADAMW_BLOCK, "a wavefront holds one block of 8-bit states");

struct Record {
    void* param;
    const void* grad;
    void* m;
    void* v;
    float* m_scale;
    float* v_scale;
    void* copy;
    long long n;
    float weight_decay;
    int aligned;               // every array starts on a boundary of 4 of its elements
};

struct Job {
    int tensor, chunk;
};

// What a step's scalars come to: by value, or from the words a device-side step counter was turned into.
struct Scalars {
    float lr, a, root2;        // a = lr / (1 - beta1^t), root2 = 1 / sqrt(1 - beta2^t)
};

struct StepArgs {
    const Record* records;
    const Job* jobs;
    const Scalars* dev;        // NULL: `by_value`
    const float* dev_grad_scale;
    Scalars by_value;
    float beta1, rest1, beta2, rest2, eps, grad_scale;
    int copy_dtype;
};

// The scale of a block from the bit patterns of its magnitudes.
__device__ __forceinline__ float scale_of(unsigned bits) {
    const unsigned top = wave_max(bits);
    return top >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : __uint_as_float(top);
}

__device__ __forceinline__ int first_code(float m, float s) {
    if (!(s > 0.0f)) return 0;
    const int q = (int)rintf(sqrtf(fabsf(m) / s) * 127.0f);
    return m < 0.0f ? -q : q;
}

__device__ __forceinline__ int second_code(float v, float s) {
    if (!(s > 0.0f)) return 0;
    return (int)rintf(sqrtf(sqrtf(v / s)) * 255.0f);
}

__device__ __forceinline__ float first_value(int q, float s) {
    const float t = (float)q * (float)(1.0 / 127.0);
    return (t * fabsf(t)) * s;
}

__device__ __forceinline__ float second_value(int q, float s) {
    const float t = (float)q * (float)(1.0 / 255.0);
    return ((t * t) * (t * t)) * s;
}

// The top bit of every byte of w that is 0.
__device__ __forceinline__ unsigned zero_bytes(unsigned w) {
    return ~(((w & 0x7f7f7f7fu) + 0x7f7f7f7fu) | w | 0x7f7f7f7fu);
}

constexpr float kLeastSecond = (float)((0.5 / 255.0) * (0.5 / 255.0) * (0.5 / 255.0) * (0.5 / 255.0));

// The codes of a lane's four moments of either kind, as a step stores them.  They are decided by the correctly rounded quotient and
// roots above, which take some 90 instructions an element for both; here approximate ones (v_rcp, v_sqrt: 1 ulp)
// place the root within 7.5 * 2^-24 * 255 = 1.2e-4 steps of the exact chain's, so that only a root that
// lies within 2^-12 of the border of two codes has to be worked out exactly, for the whole wavefront then (one
// in eight blocks).  Scales whose approximate reciprocal would be near overflow or below the normal numbers
// (flushed to 0) take that way too.
template <bool SECOND>
__device__ __forceinline__ unsigned four_codes(const float (&x)[kPer], float s) {
    unsigned w = 0;
    bool close = !(s >= 0x1p-100f && s <= 0x1p100f);
    const float r = __builtin_amdgcn_rcpf(s);
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        const float root = __builtin_amdgcn_sqrtf(fabsf(x[j]) * r);
        const float y = SECOND ? __builtin_amdgcn_sqrtf(root) * 255.0f : copysignf(root * 127.0f, x[j]);
        const float q = rintf(y);
        close = close || !(fabsf(y - q) <= 0.5f - 0x1p-12f);
        w |= ((unsigned)(int)q & 255u) << (8 * j);
    }
    if (__any(close)) {
        w = 0;
#pragma unroll
        for (int j = 0; j < kPer; ++j) w |= ((unsigned)(SECOND ? second_code(x[j], s) : first_code(x[j], s)) & 255u) << (8 * j);
    }
    // (looked for in whole words: 152 M elements 401 us a step, 411 with comparisons for each element)
    if (SECOND && __any(zero_bytes(w) != 0)) {
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            if (x[j] > 0.0f && s > 0.0f && ((w >> (8 * j)) & 255u) == 0) w |= 1u << (8 * j);
        }
    }
    return w;
}

template <class T>
__device__ __forceinline__ void load_four(const T* p, long long at, int count, bool whole, float (&out)[kPer]) {
    if (whole) {
        load_as_float<T, kPer>(p + at, out);
    } else {
#pragma unroll
        for (int j = 0; j < kPer; ++j) out[j] = j < count ? (float)p[at + j] : 0.0f;
    }
}

template <class T>
__device__ __forceinline__ void store_four(T* p, long long at, int count, bool whole, const float (&in)[kPer]) {
    if (whole) {
        store_from_float<T, kPer>(p + at, in);
    } else {
#pragma unroll
        for (int j = 0; j < kPer; ++j)
            if (j < count) p[at + j] = (T)in[j];
    }
}

__device__ __forceinline__ unsigned load_codes(const unsigned char* p, long long at, int count, bool whole) {
    if (whole) return *reinterpret_cast<const unsigned*>(p + at);
    unsigned w = 0;
#pragma unroll
    for (int j = 0; j < kPer; ++j)
        if (j < count) w |= (unsigned)p[at + j] << (8 * j);
    return w;
}

__device__ __forceinline__ void store_codes(unsigned char* p, long long at, int count, bool whole, unsigned w) {
    if (whole) {
        *reinterpret_cast<unsigned*>(p + at) = w;
        return;
    }
#pragma unroll
    for (int j = 0; j < kPer; ++j)
        if (j < count) p[at + j] = (unsigned char)(w >> (8 * j));
}

template <class P, class G, int BITS, int TURNS>
__global__ __launch_bounds__(kAdamBlock) void adamw_kernel(StepArgs a) {
    const Job job = a.jobs[blockIdx.x];
    const Record r = a.records[job.tensor];
    const Scalars k = a.dev ? *a.dev : a.by_value;
    const float gs = a.dev_grad_scale ? a.grad_scale * *a.dev_grad_scale : a.grad_scale;
    const float keep = 1.0f - k.lr * r.weight_decay;
    const long long first = (long long)job.chunk * (TURNS * kPiece) + threadIdx.x * kPer;
    float p[TURNS][kPer], g[TURNS][kPer], m[TURNS][kPer], v[TURNS][kPer];
    unsigned mq[TURNS], vq[TURNS];
    float ms[TURNS], vs[TURNS];
#pragma unroll
    for (int t = 0; t < TURNS; ++t) {
        const long long at = first + t * kPiece;
        const int count = (int)max(0ll, min((long long)kPer, r.n - at));
        const bool whole = r.aligned && count == kPer;
        load_four((const P*)r.param, at, count, whole, p[t]);
        load_four((const G*)r.grad, at, count, whole, g[t]);
        if constexpr (BITS == 32) {
            load_four((const float*)r.m, at, count, whole, m[t]);
            load_four((const float*)r.v, at, count, whole, v[t]);
        } else {
            mq[t] = load_codes((const unsigned char*)r.m, at, count, whole);
            vq[t] = load_codes((const unsigned char*)r.v, at, count, whole);
            ms[t] = count > 0 ? r.m_scale[at / NGH_ADAMW_BLOCK] : 0.0f;
            vs[t] = count > 0 ? r.v_scale[at / NGH_ADAMW_BLOCK] : 0.0f;
        }
    }
#pragma unroll
    for (int t = 0; t < TURNS; ++t) {
        const long long at = first + t * kPiece;
        const int count = (int)max(0ll, min((long long)kPer, r.n - at));
        const bool whole = r.aligned && count == kPer;
        if constexpr (BITS == 8) {
#pragma unroll
            for (int j = 0; j < kPer; ++j) {
                m[t][j] = first_value((int)(signed char)(mq[t] >> (8 * j)), ms[t]);
                v[t][j] = second_value((int)((vq[t] >> (8 * j)) & 255u), vs[t]);
            }
        }
        unsigned mtop = 0, vtop = 0;
        float counted[kPer];                   // the second moments as they count in the step
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            const float gj = g[t][j] * gs;
            m[t][j] = m[t][j] * a.beta1 + gj * a.rest1;
            counted[j] = v[t][j] = v[t][j] * a.beta2 + (gj * gj) * a.rest2;
        }
        if constexpr (BITS == 8) {
            const unsigned zeros = zero_bytes(vq[t]);
            if (__any(zeros != 0)) {
                const unsigned low = zeros & ~zero_bytes(mq[t]);
                const float least = kLeastSecond * vs[t];
#pragma unroll
                for (int j = 0; j < kPer; ++j)
                    if ((low >> (8 * j + 7)) & 1u && counted[j] < least) counted[j] = least;
            }
        }
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            // (the step itself to a few ulp: approximate root and reciprocal, unless eps is so small that
            // what they do to the smallest numbers would show)
            float step;
            if (a.eps >= 1e-12f) step = m[t][j] * __builtin_amdgcn_rcpf(__builtin_amdgcn_sqrtf(counted[j]) * k.root2 + a.eps) * k.a;
            else step = m[t][j] / (sqrtf(counted[j]) * k.root2 + a.eps) * k.a;
            p[t][j] = p[t][j] * keep - step;
            if (BITS == 8 && j < count) {
                mtop = max(mtop, __float_as_uint(m[t][j]) & 0x7fffffffu);
                vtop = max(vtop, __float_as_uint(v[t][j]) & 0x7fffffffu);
            }
        }
        store_four((P*)r.param, at, count, whole, p[t]);
        if (r.copy) {
            if (a.copy_dtype == NGH_BF16) store_four((bf16_t*)r.copy, at, count, whole, p[t]);
            else if (a.copy_dtype == NGH_F16) store_four((f16_t*)r.copy, at, count, whole, p[t]);
            else store_four((float*)r.copy, at, count, whole, p[t]);
        }
        if constexpr (BITS == 32) {
            store_four((float*)r.m, at, count, whole, m[t]);
            store_four((float*)r.v, at, count, whole, v[t]);
        } else {
            const float s1 = scale_of(mtop), s2 = scale_of(vtop);
            store_codes((unsigned char*)r.m, at, count, whole, four_codes<false>(m[t], s1));
            store_codes((unsigned char*)r.v, at, count, whole, four_codes<true>(v[t], s2));
            if ((threadIdx.x & 63) == 0 && count > 0) {
                r.m_scale[at / NGH_ADAMW_BLOCK] = s1;
                r.v_scale[at / NGH_ADAMW_BLOCK] = s2;
            }
        }
    }
}

// The scalars of a step whose number the device counts (an empty plan has no place for them and only counts).
__global__ void adamw_advance_kernel(int* step, const float* dev_lr, double lr, double beta1, double beta2, Scalars* out) {
    const int t = *step + 1;
    *step = t;
    if (!out) return;
    if (dev_lr) lr = (double)*dev_lr;
    out->lr = (float)lr;
    out->a = (float)(lr / (1.0 - pow(beta1, (double)t)));
    out->root2 = (float)(1.0 / sqrt(1.0 - pow(beta2, (double)t)));
}

__global__ __launch_bounds__(kAdamBlock) void adamw_decode_kernel(float* out, const unsigned char* codes, const float* scales, long long n,
                                                                  int second, int aligned) {
    const long long step = (long long)gridDim.x * kAdamBlock * kPer;
    for (long long at = ((long long)blockIdx.x * kAdamBlock + threadIdx.x) * kPer; at < n; at += step) {
        const int count = (int)min((long long)kPer, n - at);
        const bool whole = aligned && count == kPer;
        const unsigned w = load_codes(codes, at, count, whole);
        const float s = scales[at / NGH_ADAMW_BLOCK];
        float v[kPer];
#pragma unroll
        for (int j = 0; j < kPer; ++j)
            v[j] = second ? second_value((int)((w >> (8 * j)) & 255u), s) : first_value((int)(signed char)(w >> (8 * j)), s);
        store_four(out, at, count, whole, v);
    }
}

// A wavefront for each block of NGH_ADAMW_BLOCK values (all of it makes the same turns).
__global__ __launch_bounds__(kAdamBlock) void adamw_encode_kernel(unsigned char* codes, float* scales, const float* in, long long n, int second,
                                                                  int aligned) {
    const long long step = (long long)gridDim.x * kAdamBlock * kPer;
    for (long long base = ((long long)blockIdx.x * kAdamBlock + (threadIdx.x & ~63u)) * kPer; base < n; base += step) {
        const long long at = base + (threadIdx.x & 63) * kPer;
        const int count = (int)max(0ll, min((long long)kPer, n - at));
        const bool whole = aligned && count == kPer;
        float v[kPer];
        load_four(in, at, count, whole, v);
        unsigned top = 0;
#pragma unroll
        for (int j = 0; j < kPer; ++j) top = max(top, __float_as_uint(v[j]) & 0x7fffffffu);
        const float s = scale_of(top);
        unsigned w = 0;
#pragma unroll
        for (int j = 0; j < kPer; ++j)
            w |= ((unsigned)(second ? second_code(v[j], s) : first_code(v[j], s)) & 255u) << (8 * j);
        store_codes(codes, at, count, whole, w);
        if ((threadIdx.x & 63) == 0) scales[base / NGH_ADAMW_BLOCK] = s;
    }
}

int size_of(int dtype) { return dtype == NGH_F32 ? 4 : (dtype == NGH_F16 || dtype == NGH_BF16) ? 2 : 0; }

struct Span {
    uintptr_t begin, end;
    int tensor;
    bool written;
};

}  // namespace
}  // namespace ngh

using namespace ngh;

struct ngh_adamw_plan {
    int device = 0;
    int param_dtype = 0, grad_dtype = 0, copy_dtype = -1, bits = 32;
    unsigned jobs = 0;
    int turns = kTurnsMany;
    void* memory = nullptr;            // scalars, records, jobs
    const Record* dev_records = nullptr;
    const Job* dev_jobs = nullptr;
    Scalars* dev_scalars = nullptr;
};

namespace ngh {
namespace {

// Checks the tensors and works out the plan's records and jobs; touches no device.
int lay_out(const ngh_adamw_tensor* tensors, int32_t n_tensors, int cus, ngh_adamw_plan& plan, std::vector<Record>& records, std::vector<Job>& jobs) {
    if (n_tensors < 0 || (n_tensors > 0 && !tensors)) return report(NGH_E_INVALID, "ngh_adamw: %d tensors", n_tensors);
    if (!size_of(plan.param_dtype) || !size_of(plan.grad_dtype) || (plan.copy_dtype != -1 && !size_of(plan.copy_dtype)))
        return report(NGH_E_INVALID, "ngh_adamw: dtypes %d, %d, %d (NGH_F32, NGH_F16, NGH_BF16; no copy: -1)", plan.param_dtype, plan.grad_dtype,
                      plan.copy_dtype);
    if (plan.bits != 8 && plan.bits != 32) return report(NGH_E_INVALID, "ngh_adamw: states of %d bits (8 or 32)", plan.bits);
    const int pe = size_of(plan.param_dtype), ge = size_of(plan.grad_dtype), ce = plan.copy_dtype < 0 ? 0 : size_of(plan.copy_dtype);
    const int se = plan.bits / 8;
    records.resize(n_tensors);
    std::vector<Span> spans;
    for (int i = 0; i < n_tensors; ++i) {
        const ngh_adamw_tensor& t = tensors[i];
        if (t.n < 0) return report(NGH_E_INVALID, "ngh_adamw: tensor %d has length %lld", i, (long long)t.n);
        if (t.n >= (1LL << 42)) return report(NGH_E_UNSUPPORTED, "ngh_adamw: tensor %d is too long", i);
        if (!std::isfinite(t.weight_decay)) return report(NGH_E_INVALID, "ngh_adamw: tensor %d: weight_decay is not finite", i);
        if (t.copy && !ce) return report(NGH_E_INVALID, "ngh_adamw: tensor %d has a copy and the plan no copy_dtype", i);
        if (t.n > 0) {
            if (!t.param || !t.grad || !t.m || !t.v || (plan.bits == 8 && (!t.m_scale || !t.v_scale)))
                return report(NGH_E_INVALID, "ngh_adamw: tensor %d: NULL device pointer", i);
            if ((uintptr_t)t.param % pe || (uintptr_t)t.grad % ge || (uintptr_t)t.m % se || (uintptr_t)t.v % se ||
                (t.copy && (uintptr_t)t.copy % ce) || (uintptr_t)t.m_scale % 4 || (uintptr_t)t.v_scale % 4)
                return report(NGH_E_INVALID, "ngh_adamw: tensor %d: misaligned pointer", i);
        }
        Record& r = records[i];
        r.param = t.param;
        r.grad = t.grad;
        r.m = t.m;
        r.v = t.v;
        r.m_scale = t.m_scale;
        r.v_scale = t.v_scale;
        r.copy = t.copy;
        r.n = t.n;
        r.weight_decay = t.weight_decay;
        r.aligned = (uintptr_t)t.param % (kPer * pe) == 0 && (uintptr_t)t.grad % (kPer * ge) == 0 && (uintptr_t)t.m % (kPer * se) == 0 &&
                    (uintptr_t)t.v % (kPer * se) == 0 && (!t.copy || (uintptr_t)t.copy % (kPer * ce) == 0);
        auto span = [&](const void* p, unsigned long long bytes, bool written) {
            if (p && bytes) spans.push_back(Span{(uintptr_t)p, (uintptr_t)p + bytes, i, written});
        };
        const unsigned long long n = t.n, blocks = (n + NGH_ADAMW_BLOCK - 1) / NGH_ADAMW_BLOCK;
        span(t.param, n * pe, true);
        span(t.grad, n * ge, false);
        span(t.m, n * se, true);
        span(t.v, n * se, true);
        span(t.copy, n * ce, true);
        if (plan.bits == 8) {
            span(t.m_scale, blocks * 4, true);
            span(t.v_scale, blocks * 4, true);
        }
    }
    // Chunks of 4096 elements, of 1024 where else compute units would have fewer than four workgroups (1.3 M
    // parameters in 69 tensors: 8.4 -> 7.6 us, with 8-bit states 10.2 -> 7.5; 82 thousand 5.7 -> 3.5)
    long long pieces = 0;
    for (int i = 0; i < n_tensors; ++i) pieces += (tensors[i].n + kPiece - 1) / kPiece;
    plan.turns = pieces >= 4ll * kTurnsMany * cus ? kTurnsMany : kTurnsFew;
    const long long chunk = (long long)plan.turns * kPiece;
    if (pieces / plan.turns + n_tensors >= 2 * kMostThreads / kAdamBlock) return report(NGH_E_UNSUPPORTED, "ngh_adamw: too many elements for one plan");
    for (int i = 0; i < n_tensors; ++i)
        for (long long c = 0; c * chunk < tensors[i].n; ++c) jobs.push_back(Job{i, (int)c});
    // nothing that is written may be anything else of the plan
    std::sort(spans.begin(), spans.end(), [](const Span& x, const Span& y) { return x.begin < y.begin; });
    uintptr_t end = 0, end_written = 0;
    int by = -1, by_written = -1;
    for (const Span& s : spans) {
        if (s.begin < end_written || (s.written && s.begin < end))
            return report(NGH_E_INVALID, "ngh_adamw: tensors %d and %d share memory that is written", s.begin < end_written ? by_written : by,
                          s.tensor);
        if (s.end > end) end = s.end, by = s.tensor;
        if (s.written && s.end > end_written) end_written = s.end, by_written = s.tensor;
    }
    return NGH_OK;
}

int make_plan(ngh_context* ctx, const ngh_adamw_tensor* tensors, int32_t n_tensors, ngh_adamw_plan& plan) {
    std::vector<Record> records;
    std::vector<Job> jobs;
    const int rc = lay_out(tensors, n_tensors, view_of(ctx).cus, plan, records, jobs);
    if (rc != NGH_OK) return rc;
    plan.jobs = (unsigned)jobs.size();
    if (jobs.empty()) return NGH_OK;
    const size_t head = 256, rec = (records.size() * sizeof(Record) + 255) / 256 * 256;
    DeviceScope scope(plan.device);
    if (!scope.ok()) return report(NGH_E_RUNTIME, "ngh_adamw: the context's device cannot be made current");
    NGH_HIP_TRY(hipMalloc(&plan.memory, head + rec + jobs.size() * sizeof(Job)));
    char* at = (char*)plan.memory;
    plan.dev_scalars = (Scalars*)at;
    plan.dev_records = (const Record*)(at + head);
    plan.dev_jobs = (const Job*)(at + head + rec);
    const hipStream_t stream = view_of(ctx).stream;
    NGH_HIP_TRY(hipMemcpyAsync(at + head, records.data(), records.size() * sizeof(Record), hipMemcpyHostToDevice, stream));
    NGH_HIP_TRY(hipMemcpyAsync(at + head + rec, jobs.data(), jobs.size() * sizeof(Job), hipMemcpyHostToDevice, stream));
    NGH_HIP_TRY(hipStreamSynchronize(stream));
    return NGH_OK;
}

template <class P, class G, int BITS>
void launch_step(const ngh_adamw_plan& plan, const StepArgs& a, hipStream_t stream) {
    if (plan.turns == kTurnsMany) hipLaunchKernelGGL((adamw_kernel<P, G, BITS, kTurnsMany>), dim3(plan.jobs), dim3(kAdamBlock), 0, stream, a);
    else hipLaunchKernelGGL((adamw_kernel<P, G, BITS, kTurnsFew>), dim3(plan.jobs), dim3(kAdamBlock), 0, stream, a);
}

template <class P, class G>
void launch_step(const ngh_adamw_plan& plan, const StepArgs& a, hipStream_t stream) {
    if (plan.bits == 8) launch_step<P, G, 8>(plan, a, stream);
    else launch_step<P, G, 32>(plan, a, stream);
}

template <class P>
void launch_step(const ngh_adamw_plan& plan, const StepArgs& a, hipStream_t stream) {
    if (plan.grad_dtype == NGH_F32) launch_step<P, float>(plan, a, stream);
    else if (plan.grad_dtype == NGH_BF16) launch_step<P, bf16_t>(plan, a, stream);
    else launch_step<P, f16_t>(plan, a, stream);
}

int check_codes(ngh_context* ctx, const void* codes, const float* scales, const float* values, int64_t n, const char* what) {
    if (!ctx) return report(NGH_E_INVALID, "ctx is NULL");
    if (n < 0) return report(NGH_E_INVALID, "%s: n %lld", what, (long long)n);
    if (n >= (1LL << 40)) return report(NGH_E_UNSUPPORTED, "%s: too many values", what);
    if (n == 0) return NGH_OK;
    if (!codes || !scales || !values) return report(NGH_E_INVALID, "%s: NULL device pointer", what);
    if ((uintptr_t)scales % 4 || (uintptr_t)values % 4) return report(NGH_E_INVALID, "%s: misaligned pointer", what);
    const unsigned long long blocks = ((unsigned long long)n + NGH_ADAMW_BLOCK - 1) / NGH_ADAMW_BLOCK;
    if (spans_overlap(codes, n, values, n * 4ull) || spans_overlap(scales, blocks * 4, values, n * 4ull) ||
        spans_overlap(codes, n, scales, blocks * 4))
        return report(NGH_E_INVALID, "%s: the operands overlap", what);
    return NGH_OK;
}

}  // namespace
}  // namespace ngh

extern "C" {

int ngh_validate_adamw(const ngh_adamw_tensor* tensors, int32_t n_tensors, int32_t param_dtype, int32_t grad_dtype, int32_t copy_dtype,
                       int32_t state_bits) {
    ngh_adamw_plan plan;
    plan.param_dtype = param_dtype;
    plan.grad_dtype = grad_dtype;
    plan.copy_dtype = copy_dtype;
    plan.bits = state_bits;
    try {
        std::vector<Record> records;
        std::vector<Job> jobs;
        return lay_out(tensors, n_tensors, 256, plan, records, jobs);
    } catch (const std::exception&) {
        return report(NGH_E_NOMEM, "ngh_validate_adamw: out of host memory");
    }
}

int ngh_adamw_plan_create(ngh_context* ctx, const ngh_adamw_tensor* tensors, int32_t n_tensors, int32_t param_dtype, int32_t grad_dtype,
                          int32_t copy_dtype, int32_t state_bits, ngh_adamw_plan** out) {
    if (!ctx) return report(NGH_E_INVALID, "ctx is NULL");
    if (!out) return report(NGH_E_INVALID, "ngh_adamw_plan_create: out is NULL");
    *out = nullptr;
    const ContextView c = view_of(ctx);
    if (c.capturing) return report(NGH_E_INVALID, "ngh_adamw_plan_create: a graph is being recorded: make the plan before ngh_graph_begin");
    ngh_adamw_plan* plan = new (std::nothrow) ngh_adamw_plan();
    if (!plan) return report(NGH_E_NOMEM, "ngh_adamw_plan_create: out of host memory");
    plan->device = c.device;
    plan->param_dtype = param_dtype;
    plan->grad_dtype = grad_dtype;
    plan->copy_dtype = copy_dtype;
    plan->bits = state_bits;
    int rc;
    try {
        rc = make_plan(ctx, tensors, n_tensors, *plan);
    } catch (const std::exception&) {
        rc = report(NGH_E_NOMEM, "ngh_adamw_plan_create: out of host memory");
    }
    if (rc != NGH_OK) {
        if (plan->memory) (void)hipFree(plan->memory);
        delete plan;
        return rc;
    }
    *out = plan;
    return NGH_OK;
}

int ngh_adamw_step(ngh_context* ctx, ngh_adamw_plan* plan, const ngh_adamw_hyper* h) {
    if (!ctx) return report(NGH_E_INVALID, "ctx is NULL");
    if (!plan || !h) return report(NGH_E_INVALID, "ngh_adamw_step: NULL argument");
    const ContextView c = view_of(ctx);
    if (plan->device != c.device) return report(NGH_E_INVALID, "ngh_adamw_step: the plan is for device %d, the context for %d", plan->device, c.device);
    if (!(h->beta1 >= 0.0 && h->beta1 < 1.0) || !(h->beta2 >= 0.0 && h->beta2 < 1.0))
        return report(NGH_E_INVALID, "ngh_adamw_step: beta1 %g, beta2 %g (0 <= beta < 1)", h->beta1, h->beta2);
    if (!(h->eps >= 0.0) || !std::isfinite(h->lr) || std::isnan(h->grad_scale))
        return report(NGH_E_INVALID, "ngh_adamw_step: lr %g, eps %g, grad_scale %g", h->lr, h->eps, (double)h->grad_scale);
    if (!h->dev_step && h->step < 1) return report(NGH_E_INVALID, "ngh_adamw_step: step %d (steps count from 1)", h->step);
    if ((uintptr_t)h->dev_step % 4 || (uintptr_t)h->dev_lr % 4 || (uintptr_t)h->dev_grad_scale % 4)
        return report(NGH_E_INVALID, "ngh_adamw_step: misaligned pointer");
    if (h->dev_lr && !h->dev_step) return report(NGH_E_INVALID, "ngh_adamw_step: dev_lr without dev_step");
    DeviceScope scope(c.device);
    if (!scope.ok()) return report(NGH_E_RUNTIME, "ngh_adamw_step: the context's device cannot be made current");
    if (plan->jobs == 0 && !h->dev_step) return NGH_OK;
    StepArgs a;
    a.records = plan->dev_records;
    a.jobs = plan->dev_jobs;
    a.dev = nullptr;
    a.dev_grad_scale = h->dev_grad_scale;
    a.beta1 = (float)h->beta1;
    a.rest1 = (float)(1.0 - h->beta1);
    a.beta2 = (float)h->beta2;
    a.rest2 = (float)(1.0 - h->beta2);
    a.eps = (float)h->eps;
    a.grad_scale = h->grad_scale;
    a.copy_dtype = plan->copy_dtype;
    a.by_value = Scalars{0.0f, 0.0f, 0.0f};
    if (h->dev_step) {
        hipLaunchKernelGGL(adamw_advance_kernel, dim3(1), dim3(1), 0, c.stream, h->dev_step, h->dev_lr, h->lr, h->beta1, h->beta2,
                           plan->dev_scalars);
        NGH_HIP_TRY(hipGetLastError());
        if (plan->jobs == 0) return NGH_OK;
        a.dev = plan->dev_scalars;
    } else {
        a.by_value.lr = (float)h->lr;
        a.by_value.a = (float)(h->lr / (1.0 - std::pow(h->beta1, (double)h->step)));
        a.by_value.root2 = (float)(1.0 / std::sqrt(1.0 - std::pow(h->beta2, (double)h->step)));
    }
    if (plan->param_dtype == NGH_F32) launch_step<float>(*plan, a, c.stream);
    else if (plan->param_dtype == NGH_BF16) launch_step<bf16_t>(*plan, a, c.stream);
    else launch_step<f16_t>(*plan, a, c.stream);
    NGH_HIP_TRY(hipGetLastError());
    return NGH_OK;
}

int ngh_adamw_plan_free(ngh_context* ctx, ngh_adamw_plan* plan) {
    if (!plan) return NGH_OK;
    if (ctx && view_of(ctx).capturing) return report(NGH_E_INVALID, "ngh_adamw_plan_free: a graph is being recorded");
    if (ctx && plan->memory) (void)hipStreamSynchronize(view_of(ctx).stream);
    if (plan->memory) (void)hipFree(plan->memory);
    delete plan;
    return NGH_OK;
}

int ngh_adamw_decode(ngh_context* ctx, float* dev_out, const void* dev_codes, const float* dev_scales, int64_t n, int32_t second) {
    const int rc = check_codes(ctx, dev_codes, dev_scales, dev_out, n, "ngh_adamw_decode");
    if (rc != NGH_OK || n == 0) return rc;
    const ContextView c = view_of(ctx);
    DeviceScope scope(c.device);
    if (!scope.ok()) return report(NGH_E_RUNTIME, "ngh_adamw_decode: the context's device cannot be made current");
    const long long wgs = (n + kAdamBlock * kPer - 1) / (kAdamBlock * kPer);
    const int aligned = (uintptr_t)dev_out % 16 == 0 && (uintptr_t)dev_codes % 4 == 0;
    hipLaunchKernelGGL(adamw_decode_kernel, dim3((unsigned)std::min<long long>(wgs, 64ll * c.cus)), dim3(kAdamBlock), 0, c.stream, dev_out,
                       (const unsigned char*)dev_codes, dev_scales, (long long)n, (int)second, aligned);
    NGH_HIP_TRY(hipGetLastError());
    return NGH_OK;
}

int ngh_adamw_encode(ngh_context* ctx, void* dev_codes, float* dev_scales, const float* dev_in, int64_t n, int32_t second) {
    const int rc = check_codes(ctx, dev_codes, dev_scales, dev_in, n, "ngh_adamw_encode");
    if (rc != NGH_OK || n == 0) return rc;
    const ContextView c = view_of(ctx);
    DeviceScope scope(c.device);
    if (!scope.ok()) return report(NGH_E_RUNTIME, "ngh_adamw_encode: the context's device cannot be made current");
    const long long wgs = (n + kAdamBlock * kPer - 1) / (kAdamBlock * kPer);
    const int aligned = (uintptr_t)dev_in % 16 == 0 && (uintptr_t)dev_codes % 4 == 0;
    hipLaunchKernelGGL(adamw_encode_kernel, dim3((unsigned)std::min<long long>(wgs, 64ll * c.cus)), dim3(kAdamBlock), 0, c.stream,
                       (unsigned char*)dev_codes, dev_scales, dev_in, (long long)n, (int)second, aligned);
    NGH_HIP_TRY(hipGetLastError());
    return NGH_OK;
}

}  // extern "C"
