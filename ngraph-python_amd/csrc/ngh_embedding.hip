// Embedding lookup with scaling and its gradient by sorted tokens (ngh_embedding,
// ngh_embedding_grad in ngraph_hip.h).
//
// Lookup: y[n, :] = scale * table[tokens[n], :].  Two streams, nothing else: bound by memory (65536 rows
// of 2048 elements, fp32 to bf16: 93 us, 4.7 TB/s where a copy reaches 5.2; one row: 1.8 us, a launch).
//
// Gradient: table[v, :] (+)= scale * sum of dy[n, :] over the n with tokens[n] == v.  The order of
// the sum must not depend on the schedule.  Up to kFew places one launch does everything: a wavefront
// for each place looks through all tokens, goes on if none before it is the same, and adds the rows of
// its token in order of their places (its whole workgroup does where there are many); other workgroups
// clear the rows of the table whose token does not occur.  More places are sorted by (token, place) first:
//   1. sort.  Up to kRankMax places: chunks of kChunk are ranked by all pairs, then every place looks
//      its rank up in the other chunks.  More: tiles of kTile places, sorted by the token's bits as
//      digits, least significant first, each pass stable: a launch that counts a tile's digits, where
//      there are many tiles one that adds the counts up, and one that ranks and scatters.
//   2. sums.  The sorted list is cut into units of equal length, whatever the tokens are: a unit is
//      summed by a wavefront for each block of columns, row after row in fp32.  A token all of whose
//      rows lie in one unit is finished there; parts of a token that crosses units go to the
//      workspace, so that one frequent token is spread over as many wavefronts as many rare ones.
//      In the same launch other workgroups clear the rows whose token the sorted list does not hold; the
//      launches that rank chunks, which leave the memory idle, have cleared the table's first rows altogether.
//   3. merge.  A workgroup for each unit in which a crossing token begins adds its parts in order.
// Measured: 1999 places into [20011, 301] fp32 12.4 us (latency, and 24 MB to clear); 16384 bf16 rows into [65536, 1024]
// fp32 78 us (sort 33 with half of the table cleared beside it, sums and the other half 39, merge 5.5); 131072 rows
// of 2048 bf16, added: 218 us (sort 29, sums 178 = 4.5 TB/s, merge 14).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "ngh_internal.h"
#include "ngh_rows.h"

namespace ngh {
namespace {

constexpr int kEmbBlock = 256;
constexpr int kSortThreads = 1024;
constexpr int kSortWaves = kSortThreads / 64;
constexpr int kRankMax = 16384;                          // places sorted by chunks: 64 KiB of keys in LDS
constexpr int kChunk = 2048;
constexpr int kOneChunk = 4096;                          // up to here one chunk holds all places
constexpr int kFew = 2048;                               // places that need no sort
constexpr int kFewWaves = 8;
constexpr int kFewAlone = 16;                            // rows a wavefront adds by itself (one batch in flight)
constexpr int kFewRows = 4096;                           // rows of the table one workgroup clears at most
constexpr int kTileItems = 2;
constexpr int kTile = kSortThreads * kTileItems;
constexpr int kTileDigitBits = 9;
constexpr int kTileDigits = 1 << kTileDigitBits;
// Up to here every tile adds the counts of those before it itself (of 64 elements a row: 131072 places 60 us,
// 64 with a launch that does it for all; 1048576 places 204 and 177 us).
constexpr int kTilesUnscanned = 128;

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
    bool live[kLookupRows], has[kLookupRows], inside[kLookupRows];
#pragma unroll
    for (int r = 0; r < kLookupRows; ++r) {
        const unsigned n = first + r;
        live[r] = n < a.rows;
        const int t = live[r] ? a.tokens[n] : -1;
        has[r] = live[r] && (unsigned)t < a.vocab && t != a.pad;
        inside[r] = has[r] && (unsigned)t + 1 < a.vocab && a.width >= VEC;
        src[r] = (const TIn*)a.table + (has[r] ? (long long)t * a.table_stride : 0);
    }
    for (unsigned c = lane; c < a.chunks; c += a.lanes) {
        const int in = piece_count<VEC, RAGGED>(c * VEC, a.width);
        float v[kLookupRows][VEC];
#pragma unroll
        for (int r = 0; r < kLookupRows; ++r) {
            if (has[r]) {
                load_piece<TIn, VEC, RAGGED>(src[r] + (size_t)c * VEC, in, inside[r], v[r]);
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
    const unsigned* key_in;      // sorted so far (tiles, passes after the first)
    const unsigned* place_in;
    unsigned* key_out;
    unsigned* place_out;
    unsigned* table;             // [tiles][kTileDigits] counts of this pass; with `scanned` those of the tiles
                                 // before, and a row of all tiles'
    unsigned tiles, scanned;
    int shift, bits;
    // ranking launches: workgroups behind the first `workers` clear [clear, clear + clear_bytes), from a 16-byte boundary
    unsigned workers;
    char* clear;
    unsigned long long clear_bytes;
};

// Workgroups of a launch that ranks chunks which do not sort: each clears its share of a part of the table.
__device__ __forceinline__ bool clears(const SortArgs& a) {
    if (blockIdx.x < a.workers) return false;
    const uint4 zero = make_uint4(0, 0, 0, 0);
    uint4* p = reinterpret_cast<uint4*>(a.clear);
    for (unsigned long long i = (unsigned long long)(blockIdx.x - a.workers) * blockDim.x + threadIdx.x; i < a.clear_bytes / 16;
         i += (unsigned long long)(gridDim.x - a.workers) * blockDim.x)
        p[i] = zero;
    return true;
}

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

// All pairs within chunks of CHUNK places: a workgroup ranks 64 places, one a lane; its wavefronts share
// the places of the chunk they are compared with, which lie in LDS as keys.  Equal keys rank in order of
// their places.  Two to three instructions a pair: 2.5 us for chunks of 2048, whatever their number.
template <int CHUNK>
__global__ __launch_bounds__(kSortThreads) void rank_chunk_kernel(SortArgs a) {
    __shared__ uint4 keys4[CHUNK / 4];
    if (clears(a)) return;
    unsigned* keys = reinterpret_cast<unsigned*>(keys4);
    const unsigned first = blockIdx.x * 64 / CHUNK * CHUNK;        // of the chunk
    for (unsigned i = threadIdx.x; i < CHUNK; i += kSortThreads)
        keys[i] = first + i < a.n ? key_of(a.tokens[first + i], a.vocab, a.pad) : ~0u;
    __syncthreads();
    const unsigned lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const unsigned base = blockIdx.x * 64 - first, mine = keys[base + lane];
    constexpr unsigned kEach = CHUNK / kSortWaves;
    unsigned count = 0;
    for (unsigned c = wave * kEach; c < (wave + 1) * kEach; c += 64) {
        const uint4* k4 = keys4 + c / 4;
        if (c < base) {
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const uint4 k = k4[j];
                count += (k.x <= mine) + (k.y <= mine) + (k.z <= mine) + (k.w <= mine);
            }
        } else if (c > base) {
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const uint4 k = k4[j];
                count += (k.x < mine) + (k.y < mine) + (k.z < mine) + (k.w < mine);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 16; ++j) {                  // (keys are below 2^32 - 1: an equal one in front counts)
                const uint4 k = k4[j];
                count += (k.x < mine + (4 * j < lane)) + (k.y < mine + (4 * j + 1 < lane)) + (k.z < mine + (4 * j + 2 < lane)) +
                         (k.w < mine + (4 * j + 3 < lane));
            }
        }
    }
    __syncthreads();
    keys[wave * 64 + lane] = count;
    __syncthreads();
    if (wave != 0 || first + base + lane >= a.n) return;
    unsigned rank = 0;
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) rank += keys[w * 64 + lane];
    a.key_out[first + rank] = mine;
    a.place_out[first + rank] = first + base + lane;
}

// The rank among all chunks: a place's rank in its own, and in every other chunk the number of keys below
// it (chunks behind) or not above it (chunks in front), found by halving in all chunks at once.
__global__ __launch_bounds__(kEmbBlock) void rank_join_kernel(SortArgs a) {
    __shared__ unsigned keys[kRankMax];
    if (clears(a)) return;
    constexpr int kChunks = kRankMax / kChunk;
    const unsigned i = blockIdx.x * kEmbBlock + threadIdx.x;
    const unsigned place = i < a.n ? a.place_in[i] : 0u;
    const unsigned whole = a.n / 4;
    for (unsigned k = threadIdx.x; k < whole; k += kEmbBlock)
        reinterpret_cast<uint4*>(keys)[k] = reinterpret_cast<const uint4*>(a.key_in)[k];
    for (unsigned k = whole * 4 + threadIdx.x; k < kRankMax; k += kEmbBlock) keys[k] = k < a.n ? a.key_in[k] : ~0u;
    __syncthreads();
    if (i >= a.n) return;
    const unsigned mine = keys[i], own = i / kChunk;
    unsigned low[kChunks];                                          // keys in front of it are below the limit
#pragma unroll
    for (int c = 0; c < kChunks; ++c) low[c] = 0;
    // (keys are below 2^31, what lies behind the last is above every limit)
#pragma unroll
    for (unsigned step = kChunk / 2; step > 0; step /= 2) {
#pragma unroll
        for (int c = 0; c < kChunks; ++c) {
            const unsigned limit = (unsigned)c < own ? mine + 1 : mine;
            if (keys[c * kChunk + low[c] + step - 1] < limit) low[c] += step;
        }
    }
    unsigned rank = i - own * kChunk;
#pragma unroll
    for (int c = 0; c < kChunks; ++c) {
        // (kChunk - 1 keys have been told apart: the last one)
        const unsigned limit = (unsigned)c < own ? mine + 1 : mine;
        if (keys[c * kChunk + low[c]] < limit) ++low[c];
        if ((unsigned)c != own) rank += low[c];
    }
    a.key_out[rank] = mine;
    a.place_out[rank] = place;
}

template <bool FIRST>
__device__ __forceinline__ unsigned tile_key(const SortArgs& a, unsigned i) {
    if constexpr (FIRST) return key_of(a.tokens[i], a.vocab, a.pad);
    else return a.key_in[i];
}

// Tiles: the counts of a pass's digit in every tile.
template <bool FIRST>
__global__ __launch_bounds__(kSortThreads) void sort_count_kernel(SortArgs a) {
    __shared__ unsigned hist[kTileDigits];
    for (unsigned i = threadIdx.x; i < kTileDigits; i += kSortThreads) hist[i] = 0;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kTileItems; ++k) {
        const unsigned i = blockIdx.x * kTile + k * kSortThreads + threadIdx.x;
        if (i < a.n) atomicAdd(&hist[(tile_key<FIRST>(a, i) >> a.shift) & ((1u << a.bits) - 1)], 1u);
    }
    __syncthreads();
    for (unsigned i = threadIdx.x; i < kTileDigits; i += kSortThreads) a.table[blockIdx.x * kTileDigits + i] = hist[i];
}

// Many tiles: a digit's counts become those of the tiles before, and row `tiles` holds those of all.  A
// workgroup has 16 digits (a 64-byte piece of a row) and 64 lanes a digit, each with a run of tiles.
constexpr int kScanDigits = 16;

__global__ __launch_bounds__(kSortThreads) void sort_scan_kernel(SortArgs a) {
    constexpr unsigned kRuns = kSortThreads / kScanDigits;
    __shared__ unsigned sums[kRuns][kScanDigits + 1];
    const unsigned x = threadIdx.x % kScanDigits, y = threadIdx.x / kScanDigits;
    const unsigned each = (a.tiles + kRuns - 1) / kRuns, first = min(a.tiles, y * each), last = min(a.tiles, first + each);
    unsigned* column = a.table + blockIdx.x * kScanDigits + x;
    unsigned sum = 0;
    for (unsigned t = first; t < last; t += 8) {
        unsigned c[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) c[k] = t + k < last ? column[(size_t)(t + k) * kTileDigits] : 0u;
#pragma unroll
        for (int k = 0; k < 8; ++k) sum += c[k];
    }
    sums[y][x] = sum;
    __syncthreads();
    unsigned before = 0;
    for (unsigned r = 0; r < y; ++r) before += sums[r][x];
    for (unsigned t = first; t < last; t += 8) {
        unsigned c[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) c[k] = t + k < last ? column[(size_t)(t + k) * kTileDigits] : 0u;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            if (t + k < last) column[(size_t)(t + k) * kTileDigits] = before;
            before += c[k];
        }
    }
    if (y == kRuns - 1) column[(size_t)a.tiles * kTileDigits] = before;
}

// Tiles, a pass: ranks within the tile, offset by the counts of the tiles before it and of the
// smaller digits.
template <bool FIRST>
__global__ __launch_bounds__(kSortThreads) void sort_scatter_kernel(SortArgs a) {
    __shared__ unsigned hist[kSortWaves * kTileDigits];
    __shared__ unsigned start[kTileDigits];
    __shared__ unsigned part[kTileDigits];
    __shared__ unsigned sh[kSortWaves];
    const unsigned lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const unsigned digits = 1u << a.bits;
    unsigned key[kTileItems], place[kTileItems], rank[kTileItems];
    const unsigned base = blockIdx.x * kTile + wave * (kTileItems * 64);
#pragma unroll
    for (int k = 0; k < kTileItems; ++k) {
        const unsigned i = base + k * 64 + lane;
        const bool in = i < a.n;
        key[k] = in ? tile_key<FIRST>(a, i) : 0u;
        place[k] = FIRST ? i : in ? a.place_in[i] : 0u;
    }
    for (unsigned i = threadIdx.x; i < kSortWaves * digits; i += kSortThreads) hist[i] = 0;
    // a digit's items in smaller tiles, and in all: two lanes share a digit, each taking every other tile,
    // 16 counts in flight
    static_assert(kSortThreads == 2 * kTileDigits, "two lanes a digit");
    const unsigned digit = threadIdx.x & (kTileDigits - 1), half = threadIdx.x / kTileDigits;
    unsigned before_me = 0, all = 0;
    if (a.scanned) {
        if (digit < digits && !half) {
            before_me = a.table[(size_t)blockIdx.x * kTileDigits + digit];
            all = a.table[(size_t)a.tiles * kTileDigits + digit];
        }
    } else if (digit < digits) {
        for (unsigned t0 = half; t0 < a.tiles; t0 += 32) {
            unsigned c[16];
#pragma unroll
            for (int k = 0; k < 16; ++k) c[k] = t0 + 2 * k < a.tiles ? a.table[(t0 + 2 * k) * kTileDigits + digit] : 0u;
#pragma unroll
            for (int k = 0; k < 16; ++k) {
                all += c[k];
                if (t0 + 2 * k < blockIdx.x) before_me += c[k];
            }
        }
    }
    if (half) start[digit] = all, part[digit] = before_me;
    __syncthreads();
    if (!half) {
        all += start[digit];
        before_me += part[digit];
    }
    const unsigned smaller = scan_exclusive(half ? 0u : all, sh);          // (lanes of the second half lie behind)
    if (!half) start[digit] = smaller + before_me;
#pragma unroll
    for (int k = 0; k < kTileItems; ++k) {
        const bool in = base + k * 64 + lane < a.n;
        const unsigned d = (key[k] >> a.shift) & (digits - 1);
        const unsigned long long m = same_digit(d, a.bits, in);
        const unsigned before = __popcll(m & ((1ull << lane) - 1));
        unsigned* h = hist + wave * digits + d;
        // (a wavefront's LDS operations are carried out in order: every lane reads the count before
        // the first lane of its digit raises it)
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
    unsigned workers, slab;    // workgroups that add; behind them one for every `slab` rows of the table to clear
    unsigned cleared;          // rows of the table that are clear already
    float scale;
    int accumulate;
};

template <class TOut, int VEC, bool RAGGED>
__device__ __forceinline__ void finish_row(const SumArgs& a, unsigned token, unsigned col, int in, const float (&acc)[VEC]) {
    TOut* to = (TOut*)a.table + (long long)token * a.table_stride + col;
    float v[VEC];
    if (a.accumulate) {
        load_piece<TOut, VEC, RAGGED>(to, in, token + 1 < a.vocab && a.width >= VEC, v);
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] += a.scale * acc[i];
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] = a.scale * acc[i];
    }
    store_piece<TOut, VEC, RAGGED>(to, in, v);
}

constexpr int kUnitMax = 64;       // places of a unit: a lane holds one

// Writes zeros to the rows of lanes whose `clear` is set; lane l stands for row r0 + l.
template <class TOut, bool RAGGED>
__device__ __forceinline__ void clear_rows(const SumArgs& a, unsigned r0, bool clear) {
    constexpr int kPiece = 16 / sizeof(TOut);
    unsigned long long rows = __ballot(clear);
    const unsigned lane = threadIdx.x & 63, chunks = (a.width + kPiece - 1) / kPiece;
    float zero[kPiece];
#pragma unroll
    for (int j = 0; j < kPiece; ++j) zero[j] = 0.0f;
    while (rows) {
        const unsigned r = r0 + __builtin_ctzll(rows);
        rows &= rows - 1;
        TOut* row = (TOut*)a.table + (long long)r * a.table_stride;
        for (unsigned c = lane; c < chunks; c += 64)
            store_piece<TOut, kPiece, RAGGED>(row + (size_t)c * kPiece, piece_count<kPiece, RAGGED>(c * kPiece, a.width), zero);
    }
}

// A wavefront clears those of up to 64 rows that the sorted list does not hold: a lane looks one up.
template <class TOut, bool RAGGED>
__device__ __forceinline__ void clear_missing(const SumArgs& a, unsigned r0, unsigned count) {
    const unsigned lane = threadIdx.x & 63, row = r0 + lane;
    unsigned low = 0, high = a.n;                          // the first key not below `row` is in [low, high]
    while (low < high) {
        const unsigned mid = (low + high) / 2;
        if (a.keys[mid] < row) low = mid + 1; else high = mid;
    }
    const bool holds = low < a.n && a.keys[low] == row;
    clear_rows<TOut, RAGGED>(a, r0, lane < count && !holds);
}

// A wavefront sums one unit over 64 * VEC columns.  The unit's keys and places are one load a lane; the
// rows come in batches of AHEAD, the next batch in flight while one is added.  ADD: the sums are added to
// the table, whose rows are fetched with the batch in which their token ends.
template <class TIn, class TOut, int VEC, bool RAGGED, bool ADD>
__global__ __launch_bounds__(kEmbBlock) void embedding_sum_kernel(SumArgs a, unsigned col_blocks) {
    constexpr int kAhead = ADD ? 4 : 8;
    typedef typename VecOf<TIn, VEC>::type Raw;
    typedef typename VecOf<TOut, VEC>::type Old;
    if (!ADD && blockIdx.x >= a.workers) {
        const unsigned r0 = a.cleared + ((blockIdx.x - a.workers) * (kEmbBlock / 64) + (threadIdx.x >> 6)) * a.slab;
        if (r0 < a.vocab) clear_missing<TOut, RAGGED>(a, r0, min(a.slab, a.vocab - r0));
        return;
    }
    const unsigned job = blockIdx.x * (kEmbBlock / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const unsigned u = job / col_blocks, cb = job - u * col_blocks;
    if (u >= a.units) return;
    const unsigned lane = threadIdx.x & 63;
    const unsigned col = (cb * 64 + lane) * VEC;
    const int in = piece_count<VEC, RAGGED>(col, a.width);
    const unsigned begin = u * a.unit, end = min(a.n, begin + a.unit), count = end - begin;
    const unsigned my_key = lane < count ? a.keys[begin + lane] : a.vocab;
    const unsigned my_place = lane < count ? a.places[begin + lane] : 0u;
    const unsigned before = begin > 0 ? a.keys[begin - 1] : ~0u;
    const unsigned after = end < a.n ? a.keys[end] : ~0u;
    unsigned token = __builtin_amdgcn_readlane(my_key, 0);
    if (token >= a.vocab) return;
    // entries of tokens in the table lie in front of the others
    const unsigned valid = __popcll(__ballot(lane < count && my_key < a.vocab));
    const TIn* dy = (const TIn*)a.dy + col;
    TOut* table = (TOut*)a.table + col;
    float* part = a.parts + (size_t)u * 2 * a.part_stride + col;
    bool from_before = before == token;
    float acc[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) acc[i] = 0.0f;
    auto key_at = [&](unsigned e) { return e < valid ? (unsigned)__builtin_amdgcn_readlane(my_key, e) : e == count ? after : a.vocab; };
    Raw rows[kAhead], next[kAhead];
    Old olds[ADD ? kAhead : 1], next_olds[ADD ? kAhead : 1];
    auto fetch = [&](unsigned i, Raw (&to)[kAhead], Old (&old)[ADD ? kAhead : 1]) {
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            if (i + k < valid) {
                const unsigned place = __builtin_amdgcn_readlane(my_place, i + k);
                to[k] = load_raw<TIn, VEC, RAGGED>(dy + (long long)place * a.dy_stride, in, place + 1 < a.n && a.width >= VEC);
                if constexpr (ADD) {
                    const unsigned key = key_at(i + k);
                    if (key != key_at(i + k + 1)) old[k] = load_raw<TOut, VEC, RAGGED>(table + (long long)key * a.table_stride, in, key + 1 < a.vocab && a.width >= VEC);
                }
            }
        }
    };
    fetch(0, rows, olds);
    for (unsigned i = 0; i < valid; i += kAhead) {
        fetch(i + kAhead, next, next_olds);
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            if (i + k < valid) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) acc[j] += (float)rows[k][j];
                const unsigned following = key_at(i + k + 1);
                if (following != token || i + k + 1 == count) {
                    // the token ends here, or the unit does
                    if (in > 0) {
                        if (from_before) {
                            store_from_float<float, VEC>(part, acc);
                        } else if (following == token) {
                            store_from_float<float, VEC>(part + a.part_stride, acc);
                        } else {
                            float v[VEC];
#pragma unroll
                            for (int j = 0; j < VEC; ++j) {
                                v[j] = a.scale * acc[j];
                                if constexpr (ADD) v[j] += (float)olds[k][j];
                            }
                            store_piece<TOut, VEC, RAGGED>(table + (long long)token * a.table_stride, in, v);
                        }
                    }
                    from_before = false;
                    token = following;
#pragma unroll
                    for (int j = 0; j < VEC; ++j) acc[j] = 0.0f;
                }
            }
        }
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            rows[k] = next[k];
            if constexpr (ADD) olds[k] = next_olds[k];
        }
    }
}

// Few places, no sort.  A wavefront takes a place: it looks through the tokens for the other places of its
// token and goes on if its own is the first.  Up to kFewAlone rows it adds by itself,
// more are shared by the workgroup's wavefronts and their sums meet in LDS in order.  col_parts workgroups
// share the blocks of columns.  Behind these, workgroups clear the rows of a slab whose token does not occur.
template <class TIn, class TOut, int VEC, bool RAGGED>
__global__ __launch_bounds__(kFewWaves * 64) void embedding_few_kernel(SumArgs a, const int32_t* tokens, int pad, unsigned col_parts, unsigned col_blocks) {
    constexpr int kAhead = kFewAlone;
    typedef typename VecOf<TIn, VEC>::type Raw;
    __shared__ unsigned keys[kFew];
    __shared__ unsigned short found[kFewWaves][kFew];
    __shared__ float sums[kFewWaves][64 * VEC];
    __shared__ unsigned counts[kFewWaves], token_of[kFewWaves];
    const unsigned lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // (all tokens in flight at once: the last one again behind the end)
    constexpr int kEach = kFew / (kFewWaves * 64);
    unsigned token_key[kEach];
#pragma unroll
    for (int k = 0; k < kEach; ++k) token_key[k] = a.n ? (unsigned)tokens[min(threadIdx.x + k * kFewWaves * 64, a.n - 1)] : ~0u;
#pragma unroll
    for (int k = 0; k < kEach; ++k) token_key[k] = key_of((int)token_key[k], a.vocab, pad);
    if (blockIdx.x >= a.workers) {
        unsigned char* occurs = reinterpret_cast<unsigned char*>(found);
        static_assert(sizeof(found) >= kFewRows, "a slab's marks fit");
        const unsigned r0 = (blockIdx.x - a.workers) * a.slab, r1 = min(a.vocab, r0 + a.slab);
        for (unsigned r = threadIdx.x; r < r1 - r0; r += kFewWaves * 64) occurs[r] = 0;
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kEach; ++k)
            if (token_key[k] >= r0 && token_key[k] < r1) occurs[token_key[k] - r0] = 1;
        __syncthreads();
        const unsigned each = (r1 - r0 + kFewWaves - 1) / kFewWaves, last = min(r1, r0 + (wave + 1) * each);
        for (unsigned r = r0 + wave * each; r < last; r += 64)
            clear_rows<TOut, RAGGED>(a, r, r + lane < last && !occurs[r + lane - r0]);
        return;
    }
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
        const unsigned i = threadIdx.x + k * kFewWaves * 64;
        keys[i] = i < a.n ? token_key[k] : ~0u;
    }
    __syncthreads();
    const unsigned group = blockIdx.x / col_parts, cp = blockIdx.x - group * col_parts;
    // (frequent tokens have their first places near the front: a workgroup's places lie far apart)
    const unsigned mine = group + wave * (a.workers / col_parts);
    const unsigned token = mine < a.n ? (unsigned)__builtin_amdgcn_readfirstlane(keys[mine]) : ~0u;
    unsigned count = 0;
    if (token < a.vocab) {
        bool first = true;
        for (unsigned c = 0; c < a.n && first; c += 256) {             // (kFew keys, a multiple of 256)
            bool same[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) same[k] = keys[c + k * 64 + lane] == token;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const unsigned at = c + k * 64;
                const unsigned long long m = __ballot(same[k]);
                if (same[k]) found[wave][count + __popcll(m & ((1ull << lane) - 1))] = (unsigned short)(at + lane);
                first = first && (mine >= at + 64 ? m == 0 : mine < at || (m & ((1ull << (mine - at)) - 1)) == 0);
                count += __popcll(m);
            }
        }
        if (!first) count = 0;
    }
    if (lane == 0) {
        counts[wave] = count;
        token_of[wave] = token;
    }
    __syncthreads();
    // the sum of entries [e0, e1) of the list of wavefront w
    auto add = [&](unsigned w, unsigned e0, unsigned e1, unsigned col, int in, float (&acc)[VEC]) {
        const TIn* dy = (const TIn*)a.dy + col;
#pragma unroll
        for (int j = 0; j < VEC; ++j) acc[j] = 0.0f;
        for (unsigned e = e0; e < e1; e += kAhead) {
            Raw rows[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                if (e + k < e1) {
                    const unsigned place = __builtin_amdgcn_readfirstlane((unsigned)found[w][e + k]);
                    rows[k] = load_raw<TIn, VEC, RAGGED>(dy + (long long)place * a.dy_stride, in, place + 1 < a.n && a.width >= VEC);
                }
            }
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                if (e + k < e1) {
#pragma unroll
                    for (int j = 0; j < VEC; ++j) acc[j] += (float)rows[k][j];
                }
            }
        }
    };
    for (unsigned cb = cp; cb < col_blocks; cb += col_parts) {
        const unsigned col = (cb * 64 + lane) * VEC;
        const int in = piece_count<VEC, RAGGED>(col, a.width);
        float acc[VEC];
        if (count > 0 && count <= kFewAlone) {
            add(wave, 0, count, col, in, acc);
            if (in > 0) finish_row<TOut, VEC, RAGGED>(a, token, col, in, acc);
        }
        for (unsigned w = 0; w < kFewWaves; ++w) {
            const unsigned many = counts[w];
            if (many <= kFewAlone) continue;
            const unsigned share = (many + kFewWaves - 1) / kFewWaves;
            add(w, min(many, wave * share), min(many, (wave + 1) * share), col, in, acc);
#pragma unroll
            for (int j = 0; j < VEC; ++j) sums[wave][j * 64 + lane] = acc[j];
            __syncthreads();
            if (wave == w && in > 0) {
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    acc[j] = sums[0][j * 64 + lane];
#pragma unroll
                    for (int v = 1; v < kFewWaves; ++v) acc[j] += sums[v][j * 64 + lane];
                }
                finish_row<TOut, VEC, RAGGED>(a, token_of[w], col, in, acc);
            }
            __syncthreads();
        }
    }
}

// A workgroup for each unit but the last and each block of columns: if a token begins in the unit and goes on
// behind it, its parts are added in order, up to kMergeAlone by one wavefront, more in shares that meet
// in LDS.  (A workgroup for all columns of a unit took half as long again: the most frequent token's
// parts are what the launch waits for.)
constexpr int kMergeWaves = 4;
constexpr int kMergeAlone = 8;

template <class TOut, int VEC, bool RAGGED>
__global__ __launch_bounds__(kMergeWaves * 64) void embedding_merge_kernel(SumArgs a, unsigned col_blocks) {
    const unsigned u = blockIdx.x / col_blocks, cb = blockIdx.x - u * col_blocks;
    const unsigned wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const unsigned begin = u * a.unit, end = begin + a.unit;
    // lane l looks at the first key of unit u + 1 + l: the units behind u that begin with its last token
    const unsigned token = a.keys[end - 1];
    const unsigned here = a.keys[begin], before = begin > 0 ? a.keys[begin - 1] : ~0u;
    unsigned more = 0;
    for (unsigned v = u + 1; v < a.units; v += 64) {
        const bool same = v + lane < a.units && a.keys[(v + lane) * a.unit] == token;
        const unsigned long long m = __ballot(same);
        const unsigned run = ~m ? __builtin_ctzll(~m) : 64;
        more += run;
        if (run < 64) break;
    }
    if (token >= a.vocab || more == 0 || (here == token && before == token)) return;   // (the last: began earlier)
    const unsigned parts = more + 1;
    // the sum of parts [p0, p1) in a block of columns; part 0 is what unit u passed on
    auto add = [&](unsigned p0, unsigned p1, unsigned col, int in, float (&acc)[VEC]) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[i] = 0.0f;
        if (in <= 0) return;
        for (unsigned p = p0; p < p1; p += kMergeAlone) {
            float v[kMergeAlone][VEC];
#pragma unroll
            for (int k = 0; k < kMergeAlone; ++k) {
                if (p + k < p1)
                    load_as_float<float, VEC>(a.parts + ((size_t)(u + p + k) * 2 + (p + k == 0 ? 1 : 0)) * a.part_stride + col, v[k]);
            }
#pragma unroll
            for (int k = 0; k < kMergeAlone; ++k) {
                if (p + k < p1) {
#pragma unroll
                    for (int i = 0; i < VEC; ++i) acc[i] += v[k][i];
                }
            }
        }
    };
    float acc[VEC];
    const unsigned col = (cb * 64 + lane) * VEC;
    const int in = piece_count<VEC, RAGGED>(col, a.width);
    if (parts <= kMergeAlone) {
        if (wave != 0) return;
        add(0, parts, col, in, acc);
    } else {
        __shared__ float sh[kMergeWaves][64 * VEC];
        const unsigned share = (parts + kMergeWaves - 1) / kMergeWaves;
        add(min(parts, wave * share), min(parts, (wave + 1) * share), col, in, acc);
#pragma unroll
        for (int i = 0; i < VEC; ++i) sh[wave][i * 64 + lane] = acc[i];
        __syncthreads();
        if (wave != 0) return;
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
#pragma unroll
            for (int w = 1; w < kMergeWaves; ++w) acc[i] += sh[w][i * 64 + lane];
        }
    }
    if (in > 0) finish_row<TOut, VEC, RAGGED>(a, token, col, in, acc);
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
    a.vocab = (unsigned)s->vocab;
    a.width = (unsigned)s->width;
    a.chunks = (unsigned)((s->width + kVec - 1) / kVec);
    a.lanes = 1;
    while (a.lanes < kEmbBlock && a.lanes < a.chunks) a.lanes <<= 1;
    a.scale = s->scale;
    a.pad = s->pad_idx;
    const unsigned per_wg = kEmbBlock / a.lanes * kLookupRows;
    const int64_t slice = kMostThreads / kEmbBlock * per_wg;
    for (int64_t first = 0; first < s->rows; first += slice) {
        a.rows = (unsigned)std::min(slice, s->rows - first);
        const dim3 grid((a.rows + per_wg - 1) / per_wg);
        if (vec) hipLaunchKernelGGL((embedding_kernel<TIn, TOut, kVec, false>), grid, dim3(kEmbBlock), 0, c.stream, a);
        else hipLaunchKernelGGL((embedding_kernel<TIn, TOut, kVec, true>), grid, dim3(kEmbBlock), 0, c.stream, a);
        NGH_HIP_TRY(hipGetLastError());
        a.tokens += slice;
        a.y = (TOut*)a.y + slice * s->y_stride;
    }
    return NGH_OK;
}

// How the gradient of n places is worked on, and where its parts lie in the workspace.
struct GradPlan {
    int bits, passes;          // of the key, tiles only
    bool few;                  // no sort
    unsigned tiles;            // 0: ranked in chunks
    unsigned unit, units, col_blocks;
    bool ragged;
    size_t part_stride;
    size_t keys_a, places_a, keys_b, places_b, tables, parts, bytes;
};

GradPlan plan_grad(const ngh_embedding_spec* s, int cus) {
    GradPlan g{};
    const unsigned n = (unsigned)s->rows;
    g.bits = 1;
    while ((1ull << g.bits) <= (unsigned long long)s->vocab) ++g.bits;           // keys 0 .. vocab
    g.few = n <= (unsigned)kFew;
    g.tiles = n <= (unsigned)kRankMax ? 0 : (n + kTile - 1) / kTile;
    g.passes = (g.bits + kTileDigitBits - 1) / kTileDigitBits;
    const int vec = size_of(s->y_dtype) == 2 ? 8 : 4;
    g.ragged = !whole_pieces(s, vec);
    g.col_blocks = (unsigned)((s->width + 64 * vec - 1) / (64 * vec));
    // Units of 64 places while that gives every compute unit 8 wavefronts, shorter ones (down to 8)
    // for fewer: a unit's parts cost two fp32 rows where its tokens cross its ends.
    g.unit = kUnitMax;
    while (g.unit > 8 && (unsigned long long)((n + g.unit - 1) / g.unit) * g.col_blocks < 8ull * cus) g.unit /= 2;
    g.units = (n + g.unit - 1) / g.unit;
    g.part_stride = ((size_t)s->width + 7) / 8 * 8;
    auto room = [](size_t b) { return (b + 255) / 256 * 256; };
    size_t at = 0;
    if (!g.few) {
        g.keys_a = at, at += room(4ull * n);
        g.places_a = at, at += room(4ull * n);
        g.keys_b = at, at += room(4ull * n);
        g.places_b = at, at += room(4ull * n);
        g.tables = at, at += (size_t)(g.tiles + 1) * kTileDigits * 4;
        g.parts = at, at += g.units > 1 ? (size_t)g.units * 2 * g.part_stride * 4 : 0;
    }
    g.bytes = at;
    return g;
}

// Workgroups that clear the table, a.slab rows for each of `parts` parts of one: about `wgs` of them.
unsigned slabs_of(SumArgs& a, unsigned wgs, unsigned most, unsigned parts) {
    const unsigned rows = a.vocab - a.cleared;
    if (a.accumulate || rows == 0) return 0;
    a.slab = std::min(most, std::max(1u, (rows + wgs * parts - 1) / (wgs * parts)));
    const unsigned per = a.slab * parts;
    return (rows + per - 1) / per;
}

template <class TIn, class TOut, bool RAGGED>
int launch_sums(const ContextView& c, SumArgs a, unsigned col_blocks) {
    constexpr int kVec = 16 / sizeof(TIn);
    a.workers = (a.units * col_blocks + 3) / 4;
    const unsigned grid = a.workers + slabs_of(a, 16 * c.cus, 64, kEmbBlock / 64);
    if (a.accumulate) hipLaunchKernelGGL((embedding_sum_kernel<TIn, TOut, kVec, RAGGED, true>), dim3(grid), dim3(kEmbBlock), 0, c.stream, a, col_blocks);
    else hipLaunchKernelGGL((embedding_sum_kernel<TIn, TOut, kVec, RAGGED, false>), dim3(grid), dim3(kEmbBlock), 0, c.stream, a, col_blocks);
    NGH_HIP_TRY(hipGetLastError());
    if (a.units > 1) {
        hipLaunchKernelGGL((embedding_merge_kernel<TOut, kVec, RAGGED>), dim3((a.units - 1) * col_blocks), dim3(kMergeWaves * 64), 0, c.stream, a,
                           col_blocks);
        NGH_HIP_TRY(hipGetLastError());
    }
    return NGH_OK;
}

template <class TIn, class TOut, bool RAGGED>
int launch_few(const ContextView& c, SumArgs a, const ngh_embedding_spec* s, unsigned col_blocks) {
    constexpr int kVec = 16 / sizeof(TIn);
    // the columns are dealt out while that gives every compute unit no more than four workgroups
    const unsigned groups = (a.n + kFewWaves - 1) / kFewWaves;
    const unsigned col_parts = std::min(col_blocks, std::max(1u, 4u * c.cus / std::max(1u, groups)));
    a.workers = groups * col_parts;
    const unsigned grid = a.workers + slabs_of(a, 2 * c.cus, kFewRows, 1);
    if (!grid) return NGH_OK;
    hipLaunchKernelGGL((embedding_few_kernel<TIn, TOut, kVec, RAGGED>), dim3(grid), dim3(kFewWaves * 64), 0, c.stream, a, s->tokens, (int)s->pad_idx,
                       col_parts, col_blocks);
    NGH_HIP_TRY(hipGetLastError());
    return NGH_OK;
}

template <class TIn, class TOut>
int launch_sums(const ContextView& c, const SumArgs& a, const ngh_embedding_spec* s, const GradPlan& g) {
    if (g.few) return g.ragged ? launch_few<TIn, TOut, true>(c, a, s, g.col_blocks) : launch_few<TIn, TOut, false>(c, a, s, g.col_blocks);
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
    if (!g.few && (long long)g.units * g.col_blocks >= kMostThreads / (kMergeWaves * 64))
        return report(NGH_E_UNSUPPORTED, "ngh_embedding_grad: %lld rows of %lld elements", (long long)spec->rows, (long long)spec->width);
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

    char* ws = (char*)spec->workspace;
    SortArgs s{};
    s.tokens = spec->tokens;
    s.n = (unsigned)spec->rows;
    s.vocab = (unsigned)spec->vocab;
    s.pad = spec->pad_idx;
    s.tiles = g.tiles;
    s.table = (unsigned*)(ws + g.tables);
    // What a launch that ranks chunks clears beside it: 64 MiB at most, in whole rows, eight at a time so that the next
    // part starts on 16 bytes too ([65536, 1024] fp32: 82 -> 79 us with 16384 places, 69 -> 57 with 2100; beside the
    // longer sort by tiles it gained nothing).
    const unsigned long long row_bytes = (unsigned long long)spec->width * te;
    const bool dense = (spec->table_stride == spec->width || spec->vocab == 1) && (uintptr_t)spec->table % 16 == 0;
    const unsigned part_rows = spec->accumulate || !dense || g.tiles ? 0u : (unsigned)std::min<unsigned long long>((64ull << 20) / row_bytes / 8 * 8, spec->vocab);
    unsigned cleared = 0;
    auto launch_sort = [&](auto kernel, unsigned workers, unsigned threads) {
        const unsigned rows = std::min(part_rows, (s.vocab - cleared) / 8 * 8);
        s.workers = workers;
        s.clear = (char*)spec->table + cleared * row_bytes;
        s.clear_bytes = rows * row_bytes;
        cleared += rows;
        const unsigned extra = (unsigned)std::min<unsigned long long>((s.clear_bytes + 16 * threads - 1) / (16 * threads), 2u * c.cus);
        hipLaunchKernelGGL(kernel, dim3(workers + extra), dim3(threads), 0, c.stream, s);
        return hipGetLastError();
    };
    if (!g.few && g.tiles == 0) {
        // one launch while that is cheaper than a second one (4096 places: 8 us, 14 in two)
        const bool one = s.n <= (unsigned)kOneChunk;
        s.key_out = (unsigned*)(ws + (one ? g.keys_a : g.keys_b));
        s.place_out = (unsigned*)(ws + (one ? g.places_a : g.places_b));
        const unsigned workers = (s.n + 63) / 64;
        if (one) NGH_HIP_TRY(launch_sort(rank_chunk_kernel<kOneChunk>, workers, kSortThreads));
        else NGH_HIP_TRY(launch_sort(rank_chunk_kernel<kChunk>, workers, kSortThreads));
        if (!one) {
            s.key_in = s.key_out;
            s.place_in = s.place_out;
            s.key_out = (unsigned*)(ws + g.keys_a);
            s.place_out = (unsigned*)(ws + g.places_a);
            NGH_HIP_TRY(launch_sort(rank_join_kernel, (s.n + kEmbBlock - 1) / kEmbBlock, kEmbBlock));
        }
    } else if (!g.few) {
        const int digit = (g.bits + g.passes - 1) / g.passes;
        s.scanned = g.tiles > (unsigned)kTilesUnscanned;
        for (int p = 0; p < g.passes; ++p) {
            s.shift = p * digit;
            s.bits = std::min(digit, g.bits - s.shift);
            const bool a_out = (g.passes - 1 - p) % 2 == 0;            // the last pass ends in the first pair
            s.key_out = (unsigned*)(ws + (a_out ? g.keys_a : g.keys_b));
            s.place_out = (unsigned*)(ws + (a_out ? g.places_a : g.places_b));
            s.key_in = (const unsigned*)(ws + (a_out ? g.keys_b : g.keys_a));
            s.place_in = (const unsigned*)(ws + (a_out ? g.places_b : g.places_a));
            if (p == 0) NGH_HIP_TRY(launch_sort(sort_count_kernel<true>, g.tiles, kSortThreads));
            else NGH_HIP_TRY(launch_sort(sort_count_kernel<false>, g.tiles, kSortThreads));
            if (s.scanned) NGH_HIP_TRY(launch_sort(sort_scan_kernel, kTileDigits / kScanDigits, kSortThreads));
            if (p == 0) NGH_HIP_TRY(launch_sort(sort_scatter_kernel<true>, g.tiles, kSortThreads));
            else NGH_HIP_TRY(launch_sort(sort_scatter_kernel<false>, g.tiles, kSortThreads));
        }
    }
    SumArgs a{};
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
    a.cleared = cleared;
    a.units = g.units;
    a.unit = g.unit;
    a.scale = spec->scale;
    a.accumulate = spec->accumulate;
    switch (spec->y_dtype * 16 + spec->table_dtype) {
        case NGH_F32 * 16 + NGH_F32: return launch_sums<float, float>(c, a, spec, g);
        case NGH_BF16 * 16 + NGH_F32: return launch_sums<bf16_t, float>(c, a, spec, g);
        case NGH_F16 * 16 + NGH_F32: return launch_sums<f16_t, float>(c, a, spec, g);
        case NGH_BF16 * 16 + NGH_BF16: return launch_sums<bf16_t, bf16_t>(c, a, spec, g);
        default: return launch_sums<f16_t, f16_t>(c, a, spec, g);
    }
}

}  // extern "C"
