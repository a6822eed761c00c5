// Embedding lookup with scaling and its gradient by sorted tokens (ngh_embedding,
// ngh_embedding_grad in ngraph_hip.h).
//
// Lookup: y[n, :] = scale * table[tokens[n], :].  Two streams, nothing else: bound by memory.
//
// Gradient: table[v, :] (+)= scale * sum of dy[n, :] over the n with tokens[n] == v.  The order of
// the sum must not depend on the schedule, so the places n are sorted by (token, n) first:
//   1. sort.  The token's bits as digits, least significant first, each pass stable.  Up to
//      kOneSortMax places one workgroup sorts in LDS (one launch); more are dealt in tiles of
//      kTile places, a pass being one launch that ranks and scatters (the digit counts of the next
//      pass are taken while scattering).  In the first launch all other workgroups fill the table
//      with zeros, which is most of the traffic of an ordinary step and hides the sort.
//   2. sums.  The sorted list is cut into units of equal length, whatever the tokens are: a unit is
//      summed by a wavefront for each block of columns, row after row in fp32.  A token all of whose
//      rows lie in one unit is finished there; parts of a token that crosses units go to the
//      workspace, so that one frequent token is spread over as many wavefronts as many rare ones.
//   3. merge.  A workgroup for each unit in which a crossing token begins adds its parts in order.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "ngh_internal.h"
#include "ngh_rows.h"

namespace ngh {
namespace {

constexpr int kEmbBlock = 256;
constexpr int kSortThreads = 1024;
constexpr int kSortWaves = kSortThreads / 64;
constexpr int kItems = 16;                               // places a lane of the one-workgroup sort holds
constexpr int kOneSortMax = kSortThreads * kItems;       // 16384: keys and places take 96 KiB of LDS
constexpr int kOneDigitBits = 6;
constexpr int kTileItems = 4;
constexpr int kTile = kSortThreads * kTileItems;
constexpr int kTileDigitBits = 9;
constexpr int kTileDigits = 1 << kTileDigitBits;

// ---- lookup ----------------------------------------------------------------------------------
struct LookupArgs {
    const int32_t* tokens;
    const void* table;
    void* y;
    long long table_stride, y_stride;
    unsigned rows, vocab, width, chunks;   // chunks of VEC elements a row
    unsigned lanes;                        // lanes along a row, a power of two up to the workgroup
    float scale;
    int pad;
};

// `lanes` lanes lie along a row; a group of lanes takes kLookupRows rows, whose tokens and then
// whose chunks are in flight together.
constexpr int kLookupRows = 4;

template <class TIn, class TOut, int VEC, bool RAGGED>
__global__ __launch_bounds__(kEmbBlock) void embedding_kernel(LookupArgs a) {
    const unsigned group = threadIdx.x / a.lanes, lane = threadIdx.x & (a.lanes - 1);
    const unsigned per_wg = kEmbBlock / a.lanes;
    const unsigned first = (blockIdx.x * per_wg + group) * kLookupRows;
    const TIn* src[kLookupRows];
    bool live[kLookupRows], has[kLookupRows];
#pragma unroll
    for (int r = 0; r < kLookupRows; ++r) {
        const unsigned n = first + r;
        live[r] = n < a.rows;
        const int t = live[r] ? a.tokens[n] : -1;
        has[r] = live[r] && (unsigned)t < a.vocab && t != a.pad;
        src[r] = (const TIn*)a.table + (has[r] ? (long long)t * a.table_stride : 0);
    }
    for (unsigned c = lane; c < a.chunks; c += a.lanes) {
        const int in = piece_count<VEC, RAGGED>(c * VEC, a.width);
        float v[kLookupRows][VEC];
#pragma unroll
        for (int r = 0; r < kLookupRows; ++r) {
            if (has[r]) {
                load_piece<TIn, VEC, RAGGED>(src[r] + (size_t)c * VEC, in, v[r]);
            } else {
#pragma unroll
                for (int i = 0; i < VEC; ++i) v[r][i] = 0.0f;
            }
        }
#pragma unroll
        for (int r = 0; r < kLookupRows; ++r) {
            if (!live[r]) continue;
            if (has[r]) {
#pragma unroll
                for (int i = 0; i < VEC; ++i) v[r][i] *= a.scale;
            }
            store_piece<TOut, VEC, RAGGED>((TOut*)a.y + (long long)(first + r) * a.y_stride + (size_t)c * VEC, in, v[r]);
        }
    }
}

// ---- sort ------------------------------------------------------------------------------------
struct SortArgs {
    const int32_t* tokens;
    unsigned n, vocab;
    int pad;
    unsigned* key_in;      // sorted so far (tiles, passes after the first)
    unsigned* place_in;
    unsigned* key_out;
    unsigned* place_out;
    unsigned* table;       // [tiles][kTileDigits] counts of this pass
    unsigned* next;        // ... of the next pass; NULL in the last
    unsigned tiles;
    int shift, bits, next_shift, next_bits;
};

// A token that takes part in no sum sorts behind all others.
__device__ __forceinline__ unsigned key_of(int t, unsigned vocab, int pad) {
    return ((unsigned)t < vocab && t != pad) ? (unsigned)t : vocab;
}

// Lanes of the wavefront whose `digit` is this lane's (only lanes with `live`).
__device__ __forceinline__ unsigned long long same_digit(unsigned digit, int bits, bool live) {
    unsigned long long m = __ballot(live);
    for (int b = 0; b < bits; ++b) {
        const bool one = (digit >> b) & 1u;
        const unsigned long long with = __ballot(one);
        m &= one ? with : ~with;
    }
    return m;
}

// Exclusive scan of one value a lane over the workgroup of kSortThreads; `sh` holds kSortWaves words.
__device__ __forceinline__ unsigned scan_exclusive(unsigned v, unsigned* sh) {
    unsigned s = v;
    const unsigned lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const unsigned o = __shfl_up(s, d, 64);
        if (lane >= (unsigned)d) s += o;
    }
    if (lane == 63) sh[wave] = s;
    __syncthreads();
    unsigned before = 0;
    for (unsigned w = 0; w < wave; ++w) before += sh[w];
    __syncthreads();
    return before + s - v;
}

// The part of the table that workgroup `part` of `parts` clears.
struct FillArgs {
    void* table;
    unsigned long long row_bytes, stride_bytes;
    unsigned rows;
    int flat;              // rows follow each other without gaps, from a 16-byte boundary
};

__device__ __forceinline__ void clear_table(const FillArgs& f, unsigned part, unsigned parts) {
    if (f.flat) {
        const unsigned long long bytes = f.row_bytes * f.rows, pieces = bytes / 16;
        uint4* p = (uint4*)f.table;
        const uint4 zero = make_uint4(0, 0, 0, 0);
        for (unsigned long long i = (unsigned long long)part * blockDim.x + threadIdx.x; i < pieces;
             i += (unsigned long long)parts * blockDim.x)
            p[i] = zero;
        if (part == 0)
            for (unsigned long long i = pieces * 16 + threadIdx.x * 2; i < bytes; i += blockDim.x * 2)
                *(unsigned short*)((char*)f.table + i) = 0;
    } else {
        const unsigned wave = part * (blockDim.x >> 6) + (threadIdx.x >> 6), waves = parts * (blockDim.x >> 6);
        for (unsigned r = wave; r < f.rows; r += waves) {
            unsigned short* row = (unsigned short*)((char*)f.table + (unsigned long long)r * f.stride_bytes);
            for (unsigned long long i = threadIdx.x & 63; i < f.row_bytes / 2; i += 64) row[i] = 0;
        }
    }
}

// All places in one workgroup (n <= kOneSortMax); the others of the grid clear the table.
__global__ __launch_bounds__(kSortThreads) void sort_one_kernel(SortArgs a, FillArgs f, int total_bits) {
    __shared__ unsigned keys[kOneSortMax];
    __shared__ unsigned short places[kOneSortMax];
    __shared__ unsigned hist[kSortWaves << kOneDigitBits];
    __shared__ unsigned sh[kSortWaves];
    if (blockIdx.x > 0) {
        clear_table(f, blockIdx.x - 1, gridDim.x - 1);
        return;
    }
    const unsigned lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    // wavefront w owns items [w * per, (w + 1) * per) of the list in its present order
    const unsigned rounds = (a.n + kSortThreads - 1) / kSortThreads;      // 64-item rounds a wavefront
    const unsigned base = wave * rounds * 64;
    unsigned key[kItems], place[kItems], rank[kItems];
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
        const unsigned i = base + k * 64 + lane;
        const bool in = (unsigned)k < rounds && i < a.n;
        key[k] = in ? key_of(a.tokens[i], a.vocab, a.pad) : 0u;
        place[k] = i;
    }
    const int passes = (total_bits + kOneDigitBits - 1) / kOneDigitBits;
    const int bits = (total_bits + passes - 1) / passes;
    const unsigned digits = 1u << bits;
    for (int p = 0; p < passes; ++p) {
        for (unsigned i = threadIdx.x; i < kSortWaves * digits; i += kSortThreads) hist[i] = 0;
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kItems; ++k) {
            if ((unsigned)k < rounds) {
                const bool in = base + k * 64 + lane < a.n;
                const unsigned d = (key[k] >> (p * bits)) & (digits - 1);
                const unsigned long long m = same_digit(d, bits, in);
                const unsigned before = __popcll(m & ((1ull << lane) - 1));
                unsigned* h = hist + wave * digits + d;
                // (a wavefront's LDS operations are carried out in order: every lane reads the count
                // before the first lane of its digit raises it)
                const unsigned seen = in ? *(volatile unsigned*)h : 0u;
                if (in && before == 0) *(volatile unsigned*)h = seen + __popcll(m);
                rank[k] = seen + before;
            }
        }
        __syncthreads();
        // where each wavefront's items of a digit start: digits first, wavefronts within a digit
        const unsigned e = threadIdx.x;
        const bool mine = e < kSortWaves * digits;
        const unsigned w = e % kSortWaves, d = e / kSortWaves;
        const unsigned start = scan_exclusive(mine ? hist[w * digits + d] : 0u, sh);
        if (mine) hist[w * digits + d] = start;
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kItems; ++k) {
            if ((unsigned)k < rounds && base + k * 64 + lane < a.n) {
                const unsigned dk = (key[k] >> (p * bits)) & (digits - 1);
                const unsigned to = hist[wave * digits + dk] + rank[k];
                keys[to] = key[k];
                places[to] = (unsigned short)place[k];
            }
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kItems; ++k) {
            const unsigned i = base + k * 64 + lane;
            if ((unsigned)k < rounds && i < a.n) {
                key[k] = keys[i];
                place[k] = places[i];
            }
        }
        __syncthreads();
    }
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
        const unsigned i = base + k * 64 + lane;
        if ((unsigned)k < rounds && i < a.n) {
            a.key_out[i] = key[k];
            a.place_out[i] = place[k];
        }
    }
}

// Tiles, first launch: the counts of the first digit of every tile, the counters of the second pass
// cleared; the other workgroups clear the table.
__global__ __launch_bounds__(kSortThreads) void sort_count_kernel(SortArgs a, FillArgs f) {
    __shared__ unsigned hist[kTileDigits];
    if (blockIdx.x >= a.tiles) {
        clear_table(f, blockIdx.x - a.tiles, gridDim.x - a.tiles);
        return;
    }
    for (unsigned i = threadIdx.x; i < kTileDigits; i += kSortThreads) {
        hist[i] = 0;
        if (a.next) a.next[blockIdx.x * kTileDigits + i] = 0;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kTileItems; ++k) {
        const unsigned i = blockIdx.x * kTile + k * kSortThreads + threadIdx.x;
        if (i < a.n) atomicAdd(&hist[(key_of(a.tokens[i], a.vocab, a.pad) >> a.shift) & ((1u << a.bits) - 1)], 1u);
    }
    __syncthreads();
    for (unsigned i = threadIdx.x; i < kTileDigits; i += kSortThreads) a.table[blockIdx.x * kTileDigits + i] = hist[i];
}

// Clears the counters of the pass after the next (three passes or more).
__global__ __launch_bounds__(kEmbBlock) void sort_clear_kernel(unsigned* p, unsigned n) {
    const unsigned i = blockIdx.x * kEmbBlock + threadIdx.x;
    if (i < n) p[i] = 0;
}

// Tiles, a pass: ranks within the tile, offset by the counts of the tiles before it and of the
// smaller digits; counts the next digit of every item at the tile it goes to.
template <bool FIRST>
__global__ __launch_bounds__(kSortThreads) void sort_scatter_kernel(SortArgs a) {
    __shared__ unsigned hist[kSortWaves * kTileDigits];
    __shared__ unsigned start[kTileDigits];
    __shared__ unsigned sh[kSortWaves];
    const unsigned lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const unsigned digits = 1u << a.bits;
    for (unsigned i = threadIdx.x; i < kSortWaves * digits; i += kSortThreads) hist[i] = 0;
    // digit `threadIdx.x`: items of smaller tiles, and of all
    unsigned before_me = 0, all = 0;
    if (threadIdx.x < digits)
        for (unsigned t = 0; t < a.tiles; ++t) {
            const unsigned c = a.table[t * kTileDigits + threadIdx.x];
            all += c;
            if (t < blockIdx.x) before_me += c;
        }
    const unsigned smaller = scan_exclusive(threadIdx.x < digits ? all : 0u, sh);      // (ends with a barrier)
    if (threadIdx.x < digits) start[threadIdx.x] = smaller + before_me;
    unsigned key[kTileItems], place[kTileItems], rank[kTileItems];
    const unsigned base = blockIdx.x * kTile + wave * (kTileItems * 64);
#pragma unroll
    for (int k = 0; k < kTileItems; ++k) {
        const unsigned i = base + k * 64 + lane;
        const bool in = i < a.n;
        if constexpr (FIRST) {
            key[k] = in ? key_of(a.tokens[i], a.vocab, a.pad) : 0u;
            place[k] = i;
        } else {
            key[k] = in ? a.key_in[i] : 0u;
            place[k] = in ? a.place_in[i] : 0u;
        }
    }
#pragma unroll
    for (int k = 0; k < kTileItems; ++k) {
        const bool in = base + k * 64 + lane < a.n;
        const unsigned d = (key[k] >> a.shift) & (digits - 1);
        const unsigned long long m = same_digit(d, a.bits, in);
        const unsigned before = __popcll(m & ((1ull << lane) - 1));
        unsigned* h = hist + wave * digits + d;
        const unsigned seen = in ? *(volatile unsigned*)h : 0u;
        if (in && before == 0) *(volatile unsigned*)h = seen + __popcll(m);
        rank[k] = seen + before;
    }
    __syncthreads();
    if (threadIdx.x < digits) {
        unsigned s = start[threadIdx.x];
        for (int w = 0; w < kSortWaves; ++w) {
            const unsigned c = hist[w * digits + threadIdx.x];
            hist[w * digits + threadIdx.x] = s;
            s += c;
        }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kTileItems; ++k) {
        if (base + k * 64 + lane < a.n) {
            const unsigned to = hist[wave * digits + ((key[k] >> a.shift) & (digits - 1))] + rank[k];
            a.key_out[to] = key[k];
            a.place_out[to] = place[k];
            if (a.next) atomicAdd(&a.next[(to / kTile) * kTileDigits + ((key[k] >> a.next_shift) & ((1u << a.next_bits) - 1))], 1u);
        }
    }
}

// ---- sums ------------------------------------------------------------------------------------
struct SumArgs {
    const unsigned* keys;      // sorted
    const unsigned* places;
    const void* dy;
    void* table;
    float* parts;              // [units][2][part_stride]: the part of the token that began before the
                               // unit, the part of the one that goes on behind it
    long long dy_stride, table_stride, part_stride;
    unsigned n, vocab, width, units, unit;
    float scale;
    int accumulate;
};

template <class TOut, int VEC, bool RAGGED>
__device__ __forceinline__ void finish_row(const SumArgs& a, unsigned token, unsigned col, int in, const float (&acc)[VEC]) {
    TOut* to = (TOut*)a.table + (long long)token * a.table_stride + col;
    float v[VEC];
    if (a.accumulate) {
        load_piece<TOut, VEC, RAGGED>(to, in, v);
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] += a.scale * acc[i];
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] = a.scale * acc[i];
    }
    store_piece<TOut, VEC, RAGGED>(to, in, v);
}

constexpr int kSumAhead = 8;       // rows in flight

// A wavefront sums one unit over 64 * VEC columns.
template <class TIn, class TOut, int VEC, bool RAGGED>
__global__ __launch_bounds__(kEmbBlock) void embedding_sum_kernel(SumArgs a, unsigned col_blocks) {
    const unsigned job = blockIdx.x * (kEmbBlock / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const unsigned u = job / col_blocks, cb = job - u * col_blocks;
    if (u >= a.units) return;
    const unsigned col = (cb * 64 + (threadIdx.x & 63)) * VEC;
    const int in = piece_count<VEC, RAGGED>(col, a.width);
    const bool live = in > 0;
    const unsigned begin = u * a.unit, end = min(a.n, begin + a.unit);
    unsigned token = a.keys[begin];
    if (token >= a.vocab) return;
    const unsigned before = begin > 0 ? a.keys[begin - 1] : ~0u;
    bool from_before = before == token;
    float acc[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) acc[i] = 0.0f;
    const TIn* dy = (const TIn*)a.dy;
    for (unsigned i = begin; i < end; i += kSumAhead) {
        float v[kSumAhead][VEC];
        unsigned key[kSumAhead];
#pragma unroll
        for (int k = 0; k < kSumAhead; ++k) {
            const bool more = i + k < end;
            key[k] = more ? a.keys[i + k] : a.vocab;
            const unsigned place = more ? a.places[i + k] : 0u;
            if (live && key[k] < a.vocab) {
                load_piece<TIn, VEC, RAGGED>(dy + (long long)place * a.dy_stride + col, in, v[k]);
            } else {
#pragma unroll
                for (int j = 0; j < VEC; ++j) v[k][j] = 0.0f;
            }
        }
#pragma unroll
        for (int k = 0; k < kSumAhead; ++k) {
            if (i + k < end) {
                if (key[k] != token) {
                    if (live && token < a.vocab) {
                        if (from_before)
                            store_from_float<float, VEC>(a.parts + (size_t)u * 2 * a.part_stride + col, acc);
                        else
                            finish_row<TOut, VEC, RAGGED>(a, token, col, in, acc);
                    }
                    from_before = false;
                    token = key[k];
#pragma unroll
                    for (int j = 0; j < VEC; ++j) acc[j] = v[k][j];
                } else {
#pragma unroll
                    for (int j = 0; j < VEC; ++j) acc[j] += v[k][j];
                }
            }
        }
    }
    if (!live || token >= a.vocab) return;
    const bool goes_on = end < a.n && a.keys[end] == token;
    if (from_before)
        store_from_float<float, VEC>(a.parts + (size_t)u * 2 * a.part_stride + col, acc);
    else if (goes_on)
        store_from_float<float, VEC>(a.parts + ((size_t)u * 2 + 1) * a.part_stride + col, acc);
    else
        finish_row<TOut, VEC, RAGGED>(a, token, col, in, acc);
}

// The units in which a token that crosses their end begins: 4 wavefronts share the parts of 64 * VEC
// columns, each adding a run of them, and meet in LDS in that order.
template <class TOut, int VEC, bool RAGGED>
__global__ __launch_bounds__(kEmbBlock) void embedding_merge_kernel(SumArgs a, unsigned col_blocks) {
    const unsigned u = blockIdx.x / col_blocks, cb = blockIdx.x - u * col_blocks;
    const unsigned end = (u + 1) * a.unit;               // (the last unit has no workgroup here)
    const unsigned token = a.keys[end - 1];
    if (token >= a.vocab || a.keys[end] != token) return;
    const unsigned begin = u * a.unit;
    if (a.keys[begin] == token && begin > 0 && a.keys[begin - 1] == token) return;     // began earlier
    // units after u that begin with the token: the list is sorted
    unsigned low = u + 1, high = a.units;                // low does, high (or the end) does not
    while (high - low > 1) {
        const unsigned mid = (low + high) / 2;
        if (a.keys[mid * a.unit] == token) low = mid; else high = mid;
    }
    const unsigned parts = low - u + 1;
    const unsigned wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const unsigned col = (cb * 64 + lane) * VEC;
    const int in = piece_count<VEC, RAGGED>(col, a.width);
    const bool live = in > 0;
    const unsigned share = (parts + 3) / 4;
    const unsigned p0 = min(parts, wave * share), p1 = min(parts, p0 + share);
    float acc[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) acc[i] = 0.0f;
    if (live)
        for (unsigned p = p0; p < p1; p += 4) {
            float v[4][VEC];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if (p + k < p1) {
                    const unsigned q = u + p + k;         // part 0 is what unit u passed on
                    load_as_float<float, VEC>(a.parts + ((size_t)q * 2 + (p + k == 0 ? 1 : 0)) * a.part_stride + col, v[k]);
                } else {
#pragma unroll
                    for (int i = 0; i < VEC; ++i) v[k][i] = 0.0f;
                }
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
#pragma unroll
                for (int i = 0; i < VEC; ++i) acc[i] += v[k][i];
            }
        }
    __shared__ float sh[4][64 * VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) sh[wave][i * 64 + lane] = acc[i];
    __syncthreads();
    if (wave != 0 || !live) return;
#pragma unroll
    for (int i = 0; i < VEC; ++i)
        acc[i] = (sh[0][i * 64 + lane] + sh[1][i * 64 + lane]) + (sh[2][i * 64 + lane] + sh[3][i * 64 + lane]);
    finish_row<TOut, VEC, RAGGED>(a, token, col, in, acc);
}

// ---- host ------------------------------------------------------------------------------------
int size_of(int dtype) { return dtype == NGH_F32 ? 4 : (dtype == NGH_F16 || dtype == NGH_BF16) ? 2 : 0; }

int check(const ngh_embedding_spec* s, bool grad, const char* what) {
    if (!s) return report(NGH_E_INVALID, "%s: spec is NULL", what);
    if (s->abi_version != NGH_ABI_VERSION)
        return report(NGH_E_INVALID, "%s: abi_version %d, this library is %d", what, s->abi_version, NGH_ABI_VERSION);
    const int te = size_of(s->table_dtype), ye = size_of(s->y_dtype);
    if (!te || !ye) return report(NGH_E_INVALID, "%s: dtypes %d and %d (NGH_F32, NGH_F16, NGH_BF16)", what, s->table_dtype, s->y_dtype);
    if (s->table_dtype != s->y_dtype && s->table_dtype != NGH_F32)
        return report(NGH_E_UNSUPPORTED, "%s: a table of dtype %d with rows of dtype %d", what, s->table_dtype, s->y_dtype);
    if (s->rows < 0 || s->vocab < 0 || s->width < 0)
        return report(NGH_E_INVALID, "%s: rows %lld, vocab %lld, width %lld", what, (long long)s->rows, (long long)s->vocab,
                      (long long)s->width);
    if (s->rows >= (1LL << 31) - kTile || s->vocab >= (1LL << 31) - 1 || s->width >= (1LL << 31) - 4096)
        return report(NGH_E_UNSUPPORTED, "%s: extent too large", what);
    if (s->rows > 1 && s->y_stride < s->width) return report(NGH_E_INVALID, "%s: y_stride %lld below the width", what, (long long)s->y_stride);
    if (s->vocab > 1 && s->table_stride < s->width)
        return report(NGH_E_INVALID, "%s: table_stride %lld below the width", what, (long long)s->table_stride);
    if (s->y_stride >= (1LL << 40) || s->table_stride >= (1LL << 40)) return report(NGH_E_UNSUPPORTED, "%s: stride too large", what);
    if (s->rows && s->width) {
        if (!s->tokens || !s->y) return report(NGH_E_INVALID, "%s: NULL device pointer", what);
        if ((uintptr_t)s->tokens % 4 || (uintptr_t)s->y % ye) return report(NGH_E_INVALID, "%s: misaligned pointer", what);
    }
    if (s->vocab && s->width) {
        if (!s->table) return report(NGH_E_INVALID, "%s: NULL device pointer", what);
        if ((uintptr_t)s->table % te) return report(NGH_E_INVALID, "%s: misaligned pointer", what);
    }
    const unsigned long long tb = span_bytes(s->vocab, s->width, s->table_stride, te), yb = span_bytes(s->rows, s->width, s->y_stride, ye);
    const void* out = grad ? s->table : s->y;
    if (spans_overlap(s->table, tb, s->y, yb) || spans_overlap(out, grad ? tb : yb, s->tokens, s->rows * 4ull))
        return report(NGH_E_INVALID, "%s: the result overlaps an operand", what);
    return NGH_OK;
}

// Whether rows of both sides can be taken VEC elements (16 bytes of the narrower type) at a time.
bool whole_pieces(const ngh_embedding_spec* s, int vec) {
    const int te = size_of(s->table_dtype), ye = size_of(s->y_dtype);
    const int ta = std::min(16, vec * te), ya = std::min(16, vec * ye);
    return s->width % vec == 0 && s->table_stride * te % ta == 0 && s->y_stride * ye % ya == 0 &&
           (uintptr_t)s->table % ta == 0 && (uintptr_t)s->y % ya == 0;
}

template <class TIn, class TOut>
int launch_lookup(const ContextView& c, const ngh_embedding_spec* s) {
    constexpr int kVec = sizeof(TOut) == 2 ? 8 : 4;
    const bool vec = whole_pieces(s, kVec);
    LookupArgs a;
    a.tokens = s->tokens;
    a.table = s->table;
    a.y = s->y;
    a.table_stride = s->table_stride;
    a.y_stride = s->y_stride;
    a.rows = (unsigned)s->rows;
    a.vocab = (unsigned)s->vocab;
    a.width = (unsigned)s->width;
    a.chunks = (unsigned)((s->width + kVec - 1) / kVec);
    a.lanes = 1;
    while (a.lanes < kEmbBlock && a.lanes < a.chunks) a.lanes <<= 1;
    a.scale = s->scale;
    a.pad = s->pad_idx;
    const unsigned per_wg = kEmbBlock / a.lanes * kLookupRows;
    const dim3 grid((a.rows + per_wg - 1) / per_wg);
    if (vec) hipLaunchKernelGGL((embedding_kernel<TIn, TOut, kVec, false>), grid, dim3(kEmbBlock), 0, c.stream, a);
    else hipLaunchKernelGGL((embedding_kernel<TIn, TOut, kVec, true>), grid, dim3(kEmbBlock), 0, c.stream, a);
    NGH_HIP_TRY(hipGetLastError());
    return NGH_OK;
}

// How the gradient of n places is worked on, and where its parts lie in the workspace.
struct GradPlan {
    int bits, passes;          // of the key, tiles only
    unsigned tiles;            // 0: one workgroup sorts
    unsigned unit, units, col_blocks;
    bool ragged;
    size_t part_stride;
    size_t keys_a, places_a, keys_b, places_b, tables, parts, bytes;
};

GradPlan plan_grad(const ngh_embedding_spec* s, int cus) {
    GradPlan g;
    const unsigned n = (unsigned)s->rows;
    g.bits = 1;
    while ((1ull << g.bits) <= (unsigned long long)s->vocab) ++g.bits;           // keys 0 .. vocab
    g.tiles = n <= (unsigned)kOneSortMax ? 0 : (n + kTile - 1) / kTile;
    g.passes = (g.bits + kTileDigitBits - 1) / kTileDigitBits;
    const int vec = size_of(s->y_dtype) == 2 ? 8 : 4;
    g.ragged = !whole_pieces(s, vec);
    g.col_blocks = (unsigned)((s->width + 64 * vec - 1) / (64 * vec));
    // Units of 64 places while that gives every compute unit 8 wavefronts, shorter ones (down to 8)
    // for fewer: a unit's parts cost two fp32 rows where its tokens cross its ends.
    g.unit = 64;
    while (g.unit > 8 && (unsigned long long)((n + g.unit - 1) / g.unit) * g.col_blocks < 8ull * cus) g.unit /= 2;
    g.units = (n + g.unit - 1) / g.unit;
    g.part_stride = ((size_t)s->width + 7) / 8 * 8;
    auto room = [](size_t b) { return (b + 255) / 256 * 256; };
    size_t at = 0;
    g.keys_a = at, at += room(4ull * n);
    g.places_a = at, at += room(4ull * n);
    g.keys_b = at, at += g.tiles ? room(4ull * n) : 0;
    g.places_b = at, at += g.tiles ? room(4ull * n) : 0;
    g.tables = at, at += (size_t)g.tiles * 3 * kTileDigits * 4;
    g.parts = at, at += g.units > 1 ? (size_t)g.units * 2 * g.part_stride * 4 : 0;
    g.bytes = at;
    return g;
}

template <class TIn, class TOut, bool RAGGED>
int launch_sums(const ContextView& c, const SumArgs& a, unsigned col_blocks) {
    constexpr int kVec = 16 / sizeof(TIn);
    const unsigned long long jobs = (unsigned long long)a.units * col_blocks;
    if (jobs >= (1ull << 31)) return report(NGH_E_UNSUPPORTED, "ngh_embedding_grad: grid too large");
    hipLaunchKernelGGL((embedding_sum_kernel<TIn, TOut, kVec, RAGGED>), dim3((unsigned)((jobs + 3) / 4)), dim3(kEmbBlock), 0, c.stream, a,
                       col_blocks);
    NGH_HIP_TRY(hipGetLastError());
    if (a.units > 1) {
        hipLaunchKernelGGL((embedding_merge_kernel<TOut, kVec, RAGGED>), dim3((a.units - 1) * col_blocks), dim3(kEmbBlock), 0, c.stream, a,
                           col_blocks);
        NGH_HIP_TRY(hipGetLastError());
    }
    return NGH_OK;
}

template <class TIn, class TOut>
int launch_sums(const ContextView& c, const SumArgs& a, const GradPlan& g) {
    return g.ragged ? launch_sums<TIn, TOut, true>(c, a, g.col_blocks) : launch_sums<TIn, TOut, false>(c, a, g.col_blocks);
}

}  // namespace
}  // namespace ngh

using namespace ngh;

extern "C" {

int ngh_validate_embedding(const ngh_embedding_spec* spec, int32_t gradient) {
    return check(spec, gradient != 0, gradient ? "ngh_embedding_grad" : "ngh_embedding");
}

int ngh_embedding(ngh_context* ctx, const ngh_embedding_spec* spec) {
    const int rc = ctx ? check(spec, false, "ngh_embedding") : report(NGH_E_INVALID, "ctx is NULL");
    if (rc != NGH_OK) return rc;
    if (spec->rows == 0 || spec->width == 0) return NGH_OK;
    const ContextView c = view_of(ctx);
    DeviceScope scope(c.device);
    if (!scope.ok()) return report(NGH_E_RUNTIME, "ngh_embedding: the context's device cannot be made current");
    switch (spec->table_dtype * 16 + spec->y_dtype) {
        case NGH_F32 * 16 + NGH_F32: return launch_lookup<float, float>(c, spec);
        case NGH_F32 * 16 + NGH_BF16: return launch_lookup<float, bf16_t>(c, spec);
        case NGH_F32 * 16 + NGH_F16: return launch_lookup<float, f16_t>(c, spec);
        case NGH_BF16 * 16 + NGH_BF16: return launch_lookup<bf16_t, bf16_t>(c, spec);
        default: return launch_lookup<f16_t, f16_t>(c, spec);
    }
}

int ngh_embedding_grad_workspace(const ngh_embedding_spec* spec, size_t* out_bytes) {
    if (!spec || !out_bytes) return report(NGH_E_INVALID, "ngh_embedding_grad_workspace: NULL argument");
    if (spec->rows < 0 || spec->vocab < 0 || spec->width < 0 || spec->rows >= (1LL << 31) - kTile || spec->vocab >= (1LL << 31) - 1 ||
        spec->width >= (1LL << 31) - 4096 || !size_of(spec->y_dtype))
        return report(NGH_E_INVALID, "ngh_embedding_grad_workspace: rows %lld, vocab %lld, width %lld, dtype %d", (long long)spec->rows,
                      (long long)spec->vocab, (long long)spec->width, spec->y_dtype);
    // (the units depend on the device's compute units only through being shorter for small calls:
    // the shortest units need the most room)
    size_t most = 0;
    for (int cus = 1; cus <= 1024; cus *= 2) most = std::max(most, plan_grad(spec, cus).bytes);
    *out_bytes = std::max<size_t>(most, 256);
    return NGH_OK;
}

int ngh_embedding_grad(ngh_context* ctx, const ngh_embedding_spec* spec) {
    const int rc = ctx ? check(spec, true, "ngh_embedding_grad") : report(NGH_E_INVALID, "ctx is NULL");
    if (rc != NGH_OK) return rc;
    if (spec->vocab == 0 || spec->width == 0) return NGH_OK;
    if (spec->rows == 0 && spec->accumulate) return NGH_OK;
    const ContextView c = view_of(ctx);
    const GradPlan g = plan_grad(spec, c.cus);
    if (spec->workspace_bytes < g.bytes || (g.bytes && !spec->workspace))
        return report(NGH_E_INVALID, "ngh_embedding_grad: workspace of %zu bytes, %zu needed", spec->workspace_bytes, g.bytes);
    if ((uintptr_t)spec->workspace % 16) return report(NGH_E_INVALID, "ngh_embedding_grad: misaligned workspace");
    const int te = size_of(spec->table_dtype), ye = size_of(spec->y_dtype);
    if (spans_overlap(spec->workspace, g.bytes, spec->table, span_bytes(spec->vocab, spec->width, spec->table_stride, te)) ||
        spans_overlap(spec->workspace, g.bytes, spec->y, span_bytes(spec->rows, spec->width, spec->y_stride, ye)) ||
        spans_overlap(spec->workspace, g.bytes, spec->tokens, spec->rows * 4ull))
        return report(NGH_E_INVALID, "ngh_embedding_grad: the workspace overlaps an operand");
    DeviceScope scope(c.device);
    if (!scope.ok()) return report(NGH_E_RUNTIME, "ngh_embedding_grad: the context's device cannot be made current");

    FillArgs f;
    f.table = spec->table;
    f.row_bytes = (unsigned long long)spec->width * te;
    f.stride_bytes = (unsigned long long)spec->table_stride * te;
    f.rows = (unsigned)spec->vocab;
    f.flat = (spec->table_stride == spec->width || spec->vocab == 1) && (uintptr_t)spec->table % 16 == 0;
    unsigned fill_wgs = 0;
    if (!spec->accumulate) {
        // 64 KiB a workgroup at least, two workgroups a compute unit at most
        const unsigned long long bytes = f.row_bytes * f.rows;
        fill_wgs = (unsigned)std::max<unsigned long long>(1, std::min<unsigned long long>((bytes + 65535) / 65536, 2ull * c.cus));
    }
    char* ws = (char*)spec->workspace;
    SortArgs s;
    s.tokens = spec->tokens;
    s.n = (unsigned)spec->rows;
    s.vocab = (unsigned)spec->vocab;
    s.pad = spec->pad_idx;
    s.key_in = s.place_in = nullptr;
    s.key_out = (unsigned*)(ws + g.keys_a);
    s.place_out = (unsigned*)(ws + g.places_a);
    s.table = s.next = nullptr;
    s.tiles = g.tiles;
    s.shift = s.bits = s.next_shift = s.next_bits = 0;
    if (g.tiles == 0) {
        hipLaunchKernelGGL(sort_one_kernel, dim3(1 + fill_wgs), dim3(kSortThreads), 0, c.stream, s, f, g.bits);
        NGH_HIP_TRY(hipGetLastError());
    } else {
        unsigned* tables[3];
        for (int i = 0; i < 3; ++i) tables[i] = (unsigned*)(ws + g.tables) + (size_t)i * g.tiles * kTileDigits;
        const int digit = (g.bits + g.passes - 1) / g.passes;
        for (int p = 0; p < g.passes; ++p) {
            const bool last = p + 1 == g.passes;
            s.shift = p * digit;
            s.bits = std::min(digit, g.bits - s.shift);
            s.next_shift = s.shift + s.bits;
            s.next_bits = last ? 0 : std::min(digit, g.bits - s.next_shift);
            s.table = tables[p % 3];
            s.next = last ? nullptr : tables[(p + 1) % 3];
            const bool a_out = (g.passes - 1 - p) % 2 == 0;            // the last pass ends in the first pair
            s.key_out = (unsigned*)(ws + (a_out ? g.keys_a : g.keys_b));
            s.place_out = (unsigned*)(ws + (a_out ? g.places_a : g.places_b));
            s.key_in = (unsigned*)(ws + (a_out ? g.keys_b : g.keys_a));
            s.place_in = (unsigned*)(ws + (a_out ? g.places_b : g.places_a));
            if (p == 0) {
                hipLaunchKernelGGL(sort_count_kernel, dim3(g.tiles + fill_wgs), dim3(kSortThreads), 0, c.stream, s, f);
                NGH_HIP_TRY(hipGetLastError());
                hipLaunchKernelGGL(sort_scatter_kernel<true>, dim3(g.tiles), dim3(kSortThreads), 0, c.stream, s);
            } else {
                if (!last) {
                    const unsigned words = g.tiles * kTileDigits;
                    hipLaunchKernelGGL(sort_clear_kernel, dim3((words + kEmbBlock - 1) / kEmbBlock), dim3(kEmbBlock), 0, c.stream, s.next, words);
                    NGH_HIP_TRY(hipGetLastError());
                }
                hipLaunchKernelGGL(sort_scatter_kernel<false>, dim3(g.tiles), dim3(kSortThreads), 0, c.stream, s);
            }
            NGH_HIP_TRY(hipGetLastError());
        }
    }
    if (spec->rows == 0) return NGH_OK;
    SumArgs a;
    a.keys = (const unsigned*)(ws + g.keys_a);
    a.places = (const unsigned*)(ws + g.places_a);
    a.dy = spec->y;
    a.table = spec->table;
    a.parts = (float*)(ws + g.parts);
    a.dy_stride = spec->y_stride;
    a.table_stride = spec->table_stride;
    a.part_stride = (long long)g.part_stride;
    a.n = (unsigned)spec->rows;
    a.vocab = (unsigned)spec->vocab;
    a.width = (unsigned)spec->width;
    a.units = g.units;
    a.unit = g.unit;
    a.scale = spec->scale;
    a.accumulate = spec->accumulate;
    switch (spec->y_dtype * 16 + spec->table_dtype) {
        case NGH_F32 * 16 + NGH_F32: return launch_sums<float, float>(c, a, g);
        case NGH_BF16 * 16 + NGH_F32: return launch_sums<bf16_t, float>(c, a, g);
        case NGH_F16 * 16 + NGH_F32: return launch_sums<f16_t, float>(c, a, g);
        case NGH_BF16 * 16 + NGH_BF16: return launch_sums<bf16_t, bf16_t>(c, a, g);
        default: return launch_sums<f16_t, f16_t>(c, a, g);
    }
}

}  // extern "C"
