// radx_beam.hip — beam search beside the sort: selection over beams and vocabulary, reordering of
// the survivors' states, and the sequences out of the recorded choices (include/radx_hip.h).
//
// Selection is the sort's relative — the first k of a descending float order, ties by index — and
// reordering is radx_hip_permutation's: rows moved by an index.
#include <hip/hip_runtime.h>

#include <float.h>
#include <math.h>
#include <stdint.h>
#include <string.h>

#include <algorithm>
#include <new>

#include "engine_host.h"
#include "radx_hip.h"

using namespace radx_engine;

namespace {

constexpr int kThreads = 256;  // 4 waves
constexpr int kWaves = kThreads / 64;
constexpr uint32_t kMaxBeams = RADX_HIP_BEAM_MAX_BEAMS;
constexpr uint32_t kMaxK = RADX_HIP_BEAM_MAX_K;
constexpr uint32_t kMaxVocab = RADX_HIP_BEAM_MAX_VOCAB;

// ---------------------------------------------------------------------------------------------
// small device helpers
// ---------------------------------------------------------------------------------------------
// Sixteen bytes at any address: global memory takes wide accesses at every alignment, so rows of
// odd pitch need no variant of their own.
struct __attribute__((packed, aligned(1))) Bytes16 { uint32_t w[4]; };
struct __attribute__((packed, aligned(1))) Bytes8 { uint32_t w[2]; };
struct __attribute__((packed, aligned(1))) Bytes4 { uint32_t w; };
struct __attribute__((packed, aligned(1))) Bytes2 { uint16_t w; };

struct BF16 { uint16_t bits; };

// Unsigned integers in the order of the floats (-0 and +0 are made one value first).
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return b ^ (static_cast<uint32_t>(static_cast<int32_t>(b) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float from_ordered(uint32_t o) {
    return __uint_as_float(o ^ ((o >> 31) ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ uint64_t ordered64(double x) {
    const uint64_t b = static_cast<uint64_t>(__double_as_longlong(x + 0.0));
    return b ^ (static_cast<uint64_t>(static_cast<int64_t>(b) >> 63) | 0x8000000000000000ull);
}
__device__ __forceinline__ double from_ordered64(uint64_t o) {
    return __longlong_as_double(static_cast<int64_t>(o ^ ((o >> 63) ? 0x8000000000000000ull : 0xffffffffffffffffull)));
}
constexpr uint32_t kLowestFinite = 0x00800000u;  // ordered(-FLT_MAX): below it is -inf

// The largest of a wave's values, in every lane: within rows of 16 lanes, then across them.
__device__ __forceinline__ float wave_max(float v) {
#define RADX_DPP_MAX(ctrl) \
    v = fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(v), __float_as_int(v), ctrl, 0xf, 0xf, false)))
    RADX_DPP_MAX(0x111);  // row_shr:1
    RADX_DPP_MAX(0x112);
    RADX_DPP_MAX(0x114);
    RADX_DPP_MAX(0x118);
    RADX_DPP_MAX(0x142);  // row_bcast:15
    RADX_DPP_MAX(0x143);  // row_bcast:31
#undef RADX_DPP_MAX
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}
__device__ __forceinline__ uint32_t lanes_before(uint64_t mask) {
    return __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(mask >> 32), __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(mask), 0u));
}
// The sum of a wave's values, in every lane.
__device__ __forceinline__ double wave_sum(double v) {
#define RADX_DPP_SUM(ctrl, rows)                                                                                     \
    {                                                                                                                \
        const uint64_t u = static_cast<uint64_t>(__double_as_longlong(v));                                           \
        const uint32_t lo = static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(u), ctrl, rows, 0xf, false));         \
        const uint32_t hi = static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(u >> 32), ctrl, rows, 0xf, false));   \
        v += __longlong_as_double(static_cast<int64_t>(static_cast<uint64_t>(hi) << 32 | lo));                       \
    }
    RADX_DPP_SUM(0x111, 0xf)  // row_shr:1
    RADX_DPP_SUM(0x112, 0xf)
    RADX_DPP_SUM(0x114, 0xf)
    RADX_DPP_SUM(0x118, 0xf)
    RADX_DPP_SUM(0x142, 0xa)  // row_bcast:15 into rows 1 and 3
    RADX_DPP_SUM(0x143, 0xc)  // row_bcast:31 into rows 2 and 3
#undef RADX_DPP_SUM
    const uint64_t u = static_cast<uint64_t>(__double_as_longlong(v));
    const uint32_t lo = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(u), 63));
    const uint32_t hi = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(u >> 32), 63));
    return __longlong_as_double(static_cast<int64_t>(static_cast<uint64_t>(hi) << 32 | lo));
}
// A value that all lanes of a wave have, as the scalar that it is.
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(v))); }
__device__ __forceinline__ float uniform(float v) { return __uint_as_float(uniform(__float_as_uint(v))); }
__device__ __forceinline__ uint64_t uniform(uint64_t v) {
    return static_cast<uint64_t>(uniform(static_cast<uint32_t>(v >> 32))) << 32 | uniform(static_cast<uint32_t>(v));
}
// i / d by m = ceil(2^32 / d), for i * d < 2^32
__device__ __forceinline__ uint32_t divided(uint32_t i, uint32_t d, uint32_t m) { return d == 1 ? i : __umulhi(i, m); }

// Elements of one 16-byte vector as floats and back; tail(): the first n elements at p, -inf behind them; one(): the
// i-th element of an array of vectors.
template <typename T> struct Vec;
template <> struct Vec<float> {
    static constexpr int n = 4;
    static __device__ __forceinline__ void unpack(uint4 r, float* f) {
        f[0] = __uint_as_float(r.x);
        f[1] = __uint_as_float(r.y);
        f[2] = __uint_as_float(r.z);
        f[3] = __uint_as_float(r.w);
    }
    static __device__ __forceinline__ uint4 pack(const float* f) {
        return uint4{__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3])};
    }
    static __device__ __forceinline__ float one(const uint4* vectors, uint32_t i) { return reinterpret_cast<const float*>(vectors)[i]; }
    static __device__ __forceinline__ uint4 tail(const float* p, uint32_t n) {
        const uint32_t none = 0xff800000u;
        return uint4{n > 0 ? __float_as_uint(p[0]) : none, n > 1 ? __float_as_uint(p[1]) : none, n > 2 ? __float_as_uint(p[2]) : none, none};
    }
};
struct Half16 {  // the 16-bit types
    static constexpr int n = 8;
    static __device__ __forceinline__ uint4 tail16(const uint16_t* p, uint32_t n, uint32_t none) {
        uint32_t w[4];
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i)
            w[i] = (2 * i < n ? p[2 * i] : none) | (2 * i + 1 < n ? p[2 * i + 1] : none) << 16;
        return uint4{w[0], w[1], w[2], w[3]};
    }
};
template <> struct Vec<BF16> : Half16 {
    static __device__ __forceinline__ void unpack(uint4 r, float* f) {
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = __uint_as_float(w[i] << 16);
            f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
    static __device__ __forceinline__ uint4 pack(const float* f) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = __float_as_uint(f[2 * i]) >> 16 | (__float_as_uint(f[2 * i + 1]) & 0xffff0000u);
        return uint4{w[0], w[1], w[2], w[3]};
    }
    static __device__ __forceinline__ float one(const uint4* vectors, uint32_t i) {
        return __uint_as_float(static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(vectors)[i]) << 16);
    }
    static __device__ __forceinline__ uint4 tail(const BF16* p, uint32_t n) { return tail16(&p->bits, n, 0xff80u); }
};
template <> struct Vec<_Float16> : Half16 {
    static __device__ __forceinline__ void unpack(uint4 r, float* f) {
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(w[i])));
            f[2 * i + 1] = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(w[i] >> 16)));
            asm("" : "+v"(f[2 * i]), "+v"(f[2 * i + 1]));  // or the halves stay in registers beside them, and these spill
        }
    }
    static __device__ __forceinline__ uint4 pack(const float* f) {  // the values are float16's: nothing is rounded
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(f[2 * i], f[2 * i + 1]));
        return uint4{w[0], w[1], w[2], w[3]};
    }
    static __device__ __forceinline__ float one(const uint4* vectors, uint32_t i) {
        return static_cast<float>(reinterpret_cast<const _Float16*>(vectors)[i]);
    }
    static __device__ __forceinline__ uint4 tail(const _Float16* p, uint32_t n) { return tail16(reinterpret_cast<const uint16_t*>(p), n, 0xfc00u); }
};

// Counts by distance below the largest, in bins that grow by a sixteenth of an octave: whatever the scale of the
// values, the bins up to the k-th one's hold few more than k (with a quarter of an octave 290 for k = 64).
constexpr uint32_t kBins = 512;
// The first bin up to which there are k (the last bin if there are fewer), in every lane of a wave.
__device__ __forceinline__ uint32_t bin_with(const uint32_t* bins, uint32_t k) {
    const uint32_t lane = threadIdx.x & 63u;
    const uint4 lo = reinterpret_cast<const uint4*>(bins)[2 * lane], hi = reinterpret_cast<const uint4*>(bins)[2 * lane + 1];
    const uint32_t c[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
    uint32_t mine = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) mine += c[i];
    uint32_t upto = mine;
#define RADX_DPP_ADD(ctrl, rows) \
    upto += static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(upto), ctrl, rows, 0xf, false))
    RADX_DPP_ADD(0x111, 0xf);  // row_shr:1
    RADX_DPP_ADD(0x112, 0xf);
    RADX_DPP_ADD(0x114, 0xf);
    RADX_DPP_ADD(0x118, 0xf);
    RADX_DPP_ADD(0x142, 0xa);  // row_bcast:15 into rows 1 and 3
    RADX_DPP_ADD(0x143, 0xc);  // row_bcast:31 into rows 2 and 3
#undef RADX_DPP_ADD
    const uint64_t enough = __ballot(upto >= k);
    if (!enough) return kBins - 1;
    uint32_t before = upto - mine, at = 8 * lane;
#pragma unroll
    for (int i = 0; i < 7; ++i) {
        before += c[i];
        at += before < k;
    }
    return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(at), __ffsll(static_cast<unsigned long long>(enough)) - 1));
}
// Bins of whole-number distances: up to 15 one each, then sixteen for every power of two.
__device__ __forceinline__ uint32_t bin_of(uint32_t distance) {
    if (distance < 16) return distance;
    const uint32_t top = 31 - __clz(distance);
    return (top - 3) * 16 + ((distance >> (top - 4)) & 15u);
}
// The largest distance that a bin holds.
__device__ __forceinline__ uint32_t end_of_bin(uint32_t bin) {
    if (bin < 16) return bin;
    const uint32_t top = bin / 16 + 3;
    if (top > 31) return 0xffffffffu;
    const uint64_t end = (16ull + (bin & 15u) + 1) << (top - 4);
    return static_cast<uint32_t>(end - 1);
}

// The k-th largest (k <= 64 * N) of a wave's values, or a value that exactly k reach.
template <int N>
__device__ __forceinline__ uint32_t reached_by(const uint32_t (&v)[N], uint32_t k) {
    uint32_t t = 0;
#pragma unroll 1
    for (int bit = 31; bit >= 0; --bit) {
        const uint32_t c = t | (1u << bit);
        uint32_t n = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) n += __popcll(__ballot(v[i] >= c));
        if (n >= k) t = c;
        if (n == k) break;
    }
    return t;
}

// ---------------------------------------------------------------------------------------------
// selection
// ---------------------------------------------------------------------------------------------
// score(row, token) = cum[row] + ((x - M) - log sum exp(x - M)) with the row's maximum M: within a row the order of
// the scores is the order of the logits, so a part of a row can be searched for its k best before M and
// the sum are known, and the logits are read once.  A workgroup takes a slice of a row and leaves the
// slice's maximum, its sum of exponentials relative to that maximum and its k best logits; another joins the
// slices of an item.  What bounds it, large: reading, and the issue of about seven operations an element beside it
// (64 x 8 x 131072 bfloat16, k = 16: a call 34.9 us for 134 MB, 3.8 TB/s; the loads and maxima alone take 26).  Small: the
// latency of the two phases (1 x 4 x 32000 float32: 10 us).
// Exponentials are 32-bit, eight of them are added in 32 bits and from there on in 64; scores are 64-bit and rounded
// once, so that the order of two candidates of one row is exact, and of different rows hangs on the logs of their rows'
// sums alone.  These are within (3 ln n + 5) 2^-24 for n tokens; measured, 0.1e-8 to 2e-8 on average and 6e-8 at most for
// rows of normal logits (standard deviation 1 to 4, 32000 and 131072 tokens), 2.5e-7 where all terms but the first are alike.
struct SliceInfo {
    double sum;  // of exp(x - max)
    float max;
    uint32_t unused;
};

// Counters are lines of their own: slices of other items that count in the same line cost more than all of an item's
// (4 x 4 x 131072: 12.2 us a call with one line for all, 10.5 so).
constexpr uint32_t kCounterWords = 32;

struct SelectArgs {
    const void* logits;
    int64_t row_stride;         // elements
    const float* cum;
    const uint32_t* allowed;    // or null
    int64_t allowed_stride;     // words; 0: one mask for all rows
    const uint8_t* finished;    // or null
    int32_t end_token;
    int normalize;
    uint32_t beams, vocab, k;
    uint32_t slices, tiles_per_slice;
    uint32_t k_inverse, slices_inverse;  // ceil(2^32 / d), for divided()
    uint32_t merge_parts_log2;  // threads that the join gives a list
    SliceInfo* info;            // [row][slice]
    uint64_t* best;             // [row][slice][k], best first: ordered logit, then ~token; 0: none
    uint32_t* arrived;          // [batch][kCounterWords], the first of each: slices of an item that are done; 0 between calls
    float* scores;
    int32_t* parents;
    int32_t* tokens;
    uint8_t* out_finished;
};

__device__ __forceinline__ bool finite(float x) { return fabsf(x) < INFINITY; }

// ---------------------------------------------------------------------------------------------
// selection, the join: one workgroup takes one batch item
// ---------------------------------------------------------------------------------------------
// The rows' maxima and sums are joined from their slices, every slice's entries get their scores in
// 64 bits, and the k best come out in the order (score down, beam up, logit down, token up).
// Within a beam that is the slices' own order.
constexpr uint32_t kMergeStage = 512;      // entries that are ranked at once; more than k only by ties and the bins' width
constexpr uint32_t kMergeThreads = 1024;  // of the join as a kernel of its own
constexpr uint32_t kHeld = 2;             // entries of its first list that a thread fetches ahead

struct Entry {
    uint64_t score;  // ordered64
    uint64_t rest;   // beam, ~ordered logit, token: smaller is better
};
__device__ __forceinline__ bool better(const Entry& p, const Entry& q) {
    return p.score > q.score || (p.score == q.score && p.rest < q.rest);
}

struct RowBase {
    double top, log_sum, cum;
};

__device__ __forceinline__ double score_of(const RowBase& r, uint64_t key) {
    return r.cum + ((static_cast<double>(from_ordered(static_cast<uint32_t>(key >> 32))) - r.top) - r.log_sum);
}

// A float not below v.
__device__ __forceinline__ float rounded_up(double v) {
    const float f = static_cast<float>(v);
    return static_cast<double>(f) < v ? from_ordered(ordered(f) + 1u) : f;
}

__device__ __forceinline__ Entry entry_of(const RowBase& r, uint32_t beam, uint64_t key) {
    const uint32_t o = static_cast<uint32_t>(key >> 32), token = ~static_cast<uint32_t>(key);
    return Entry{ordered64(score_of(r, key)), static_cast<uint64_t>(beam) << 56 | static_cast<uint64_t>(~o) << 24 | token};
}
// The k best of from[0..n_from) and stage[0..n) into to[], sorted: an entry's place is the number of better ones.
// Arrays have room for kPad entries behind their last, which are made the worst there are.
constexpr uint32_t kPad = 64;
template <uint32_t THREADS>
__device__ __forceinline__ uint32_t prune(Entry* from, uint32_t n_from, Entry* stage, uint32_t n, Entry* to, uint32_t k) {
    const uint32_t all = n_from + n;
    if (threadIdx.x < kPad) {
        from[n_from + threadIdx.x] = Entry{0, 0};
        stage[n + threadIdx.x] = Entry{0, 0};
    }
    __syncthreads();
    // lanes an entry gets: up to eight, as long as each has eight entries to compare with
    uint32_t parts = 1;
    while (parts < 8 && parts * 8 < all && 2 * parts * all <= THREADS) parts <<= 1;
    const uint32_t part = threadIdx.x & (parts - 1u);
    auto count = [&](const Entry* list, uint32_t size, const Entry& e) {
        uint32_t above = 0;
        for (uint32_t j = part; j < size; j += parts * 8) {
            Entry other[8];
#pragma unroll
            for (uint32_t i = 0; i < 8; ++i) other[i] = list[j + i * parts];  // an entry's lanes read neighbours
#pragma unroll
            for (int i = 0; i < 8; ++i) above += better(other[i], e);
        }
        return above;
    };
    for (uint32_t i = threadIdx.x / parts; i < all; i += THREADS / parts) {
        const Entry e = i < n_from ? from[i] : stage[i - n_from];
        uint32_t above = count(from, n_from, e) + count(stage, n, e);
        for (uint32_t o = parts >> 1; o; o >>= 1) above += __shfl_xor(above, o);
        if (above < k) to[above] = e;  // from all of the entry's lanes
    }
    __syncthreads();
    return all < k ? all : k;
}

// Bins of scores by their distance below the best one, sixteen for every power of two from 2^-24 to 2^8.
__device__ __forceinline__ uint32_t bin_of(double best, double score) {
    const uint32_t b = __float_as_uint(static_cast<float>(best - score)) >> 19;  // exponent and four bits of the fraction
    constexpr uint32_t kLow = (127 - 24) * 16;
    return b <= kLow ? 0 : min(b - kLow, kBins - 1);
}

struct MergeLds {
    uint32_t bins[2][kBins];
    Entry kept[2][kMaxK + kPad];
    Entry stage[kMergeStage + kPad];
    RowBase base[kMaxBeams];
    float wave_best[16];
    uint32_t staged;
};

// What the slices of a launch hand to the one that joins them goes past the XCDs' L2s: stores of agent scope write
// through, and loads of that scope read behind them, so no L2 has to be written back or invalidated whole (8 x 4 x 32000, a
// call: 11.4 us with a release and an acquire, 10.5 so).
template <bool THROUGH, typename T>
__device__ __forceinline__ void put(T* p, T v) {
    if (THROUGH) __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    else *p = v;
}
template <bool THROUGH, typename T>
__device__ __forceinline__ T got(const T* p) {
    return THROUGH ? __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : *p;
}

// A list has merge_parts threads, and a thread every merge_parts-th entry of it.  Of its first list a thread fetches kHeld
// entries ahead; ALL: that is all there is, otherwise it may have more entries, and more lists.
template <uint32_t THREADS, bool ALL, bool THROUGH>
__device__ __forceinline__ void merge_item(const SelectArgs& a, uint32_t item, MergeLds& lds) {
    RowBase* const base = lds.base;
    Entry* const stage = lds.stage;
    uint32_t& staged = lds.staged;
    const uint32_t lane = threadIdx.x & 63u;
    const uint32_t lists = a.beams * a.slices;
    const SliceInfo* info = a.info + static_cast<size_t>(item) * lists;
    const uint64_t* best = a.best + static_cast<size_t>(item) * lists * a.k;
    const uint32_t parts = 1u << a.merge_parts_log2, part = threadIdx.x & (parts - 1u);
    const uint32_t first_list = threadIdx.x >> a.merge_parts_log2, list_step = THREADS >> a.merge_parts_log2;

    uint64_t held[kHeld];
#pragma unroll
    for (uint32_t r = 0; r < kHeld; ++r) {
        const uint32_t j = part + (r << a.merge_parts_log2);
        held[r] = first_list < lists && j < a.k ? got<THROUGH>(best + first_list * a.k + j) : 0;
    }
    if (threadIdx.x == 0) staged = 0;
    for (uint32_t i = threadIdx.x; i < kBins; i += THREADS) lds.bins[0][i] = lds.bins[1][i] = 0;
    __syncthreads();
    // rows: a group of lanes each, a power of two that covers the slices
    uint32_t group = 1;
    while (group < a.slices && group < 64) group <<= 1;
    const uint32_t first = threadIdx.x & (group - 1u);
    float most = -INFINITY;  // the best score among this thread's rows, rounded up
    for (uint32_t beam = threadIdx.x / group; beam < a.beams; beam += THREADS / group) {
        const uint32_t row = item * a.beams + beam;
        const float cum = a.cum[row];
        const bool ended = a.finished && a.finished[row];
        const SliceInfo* mine = info + beam * a.slices;
        // the first slice of every lane is fetched whole before any is looked at; most rows have no more
        const bool some = first < a.slices;
        const float m0 = some ? got<THROUGH>(&mine[first].max) : -INFINITY;
        const double s0 = some ? got<THROUGH>(&mine[first].sum) : 0.0;
        float m = m0;
        for (uint32_t s = first + group; s < a.slices; s += group) m = fmaxf(m, got<THROUGH>(&mine[s].max));
        for (uint32_t o = group >> 1; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
        auto scaled = [&](float ms, double p) {
            return ms > -INFINITY || !(p == 0.0) ? p * exp(static_cast<double>(ms) - static_cast<double>(m)) : 0.0;
        };
        double sum = scaled(m0, s0);
        for (uint32_t s = first + group; s < a.slices; s += group) sum += scaled(got<THROUGH>(&mine[s].max), got<THROUGH>(&mine[s].sum));
        for (uint32_t o = group >> 1; o; o >>= 1) sum += __shfl_xor(sum, o);
        // a NaN or +inf among the allowed logits has made the sum a NaN
        const bool live = !ended && finite(cum) && finite(m) && sum > 0.0 && sum < INFINITY;
        const RowBase r{a.normalize ? static_cast<double>(m) : 0.0, a.normalize ? log(sum) : 0.0, live ? static_cast<double>(cum) : -INFINITY};
        if (live) most = fmaxf(most, rounded_up(score_of(r, static_cast<uint64_t>(ordered(m)) << 32)));
        if (first == 0) {
            base[beam] = r;
            if (ended && finite(cum)) {
                stage[atomicAdd(&staged, 1u)] = Entry{ordered64(cum), static_cast<uint64_t>(beam) << 56 | static_cast<uint32_t>(a.end_token)};
                most = fmaxf(most, cum);
            }
        }
    }
    most = wave_max(most);
    if (lane == 0) lds.wave_best[threadIdx.x >> 6] = most;
    __syncthreads();
    for (uint32_t w = 0; w < THREADS / 64; ++w) most = fmaxf(most, lds.wave_best[w]);
    const double top = static_cast<double>(most);

    const uint32_t ended_beams = staged;
    // which entries: those in the bins up to the k-th best one's.  f(entry, its beam, its bin) is called for a list's
    // entries in the bins up to `last`; they come best first.
    auto in_list = [&](uint32_t l, uint32_t last, uint32_t most_of_it, auto&& f) {
        const uint32_t beam = divided(l, a.slices, a.slices_inverse);
        const RowBase r = base[beam];
        if (r.cum == -INFINITY) return;
        uint32_t from = part;
        if (ALL || l == first_list) {
            bool more = true;
#pragma unroll
            for (uint32_t i = 0; i < kHeld; ++i) {
                const uint32_t bin = held[i] && part + (i << a.merge_parts_log2) < most_of_it ? bin_of(top, score_of(r, held[i])) : kBins;
                more = bin <= last;
                if (more) f(held[i], beam, bin);
                if (!__any(more)) break;
            }
            if (ALL || !more) return;
            from += kHeld << a.merge_parts_log2;
        }
        for (uint32_t j = from; j < most_of_it; j += parts) {
            const uint64_t key = got<THROUGH>(best + static_cast<size_t>(l) * a.k + j);
            const uint32_t bin = key ? bin_of(top, score_of(r, key)) : kBins;
            if (bin > last) break;
            f(key, beam, bin);
        }
    };
    auto in_lists = [&](uint32_t last, uint32_t most_of_it, auto&& f) {
        for (uint32_t l = first_list; l < lists; l += list_step) in_list(l, last, most_of_it, f);
    };
    uint32_t* const bins = lds.bins[0];
    const uint32_t ended_bin = threadIdx.x < ended_beams ? bin_of(top, from_ordered64(stage[threadIdx.x].score)) : kBins;
    uint32_t limit = kBins - 1;
    if (lists * a.k > 2 * THREADS) {
        // first by the lists' best entries alone: most others are far away, in few bins, where their counts would queue
        uint32_t* const heads = lds.bins[1];
        in_lists(kBins - 1, 1, [&](uint64_t, uint32_t, uint32_t bin) { atomicAdd(&heads[bin], 1u); });
        if (ended_bin < kBins) atomicAdd(&heads[ended_bin], 1u);
        __syncthreads();
        limit = bin_with(heads, a.k);
    }
    in_lists(limit, a.k, [&](uint64_t, uint32_t, uint32_t bin) { atomicAdd(&bins[bin], 1u); });
    if (ended_bin < kBins) atomicAdd(&bins[ended_bin], 1u);
    __syncthreads();
    const uint32_t upto = min(bin_with(bins, a.k), limit);
    in_lists(upto, a.k, [&](uint64_t key, uint32_t beam, uint32_t) {
        const uint32_t at = atomicAdd(&staged, 1u);
        if (at < kMergeStage) stage[at] = entry_of(base[beam], beam, key);
    });
    __syncthreads();
    Entry* kept = lds.kept[0];
    uint32_t n_kept = 0;
    if (staged <= kMergeStage) {
        n_kept = prune<THREADS>(lds.kept[1], 0, stage, staged, kept, a.k);
    } else {
        // very many ties: the lists a few at a time
        n_kept = prune<THREADS>(lds.kept[1], 0, stage, ended_beams, kept, a.k);
        uint32_t turn = 1;
        const uint32_t step = kMergeStage / a.k;
        for (uint32_t l0 = 0; l0 < lists; l0 += step) {
            if (threadIdx.x == 0) staged = 0;
            __syncthreads();
            const uint32_t now = min(step, lists - l0) * a.k;
            for (uint32_t i = threadIdx.x; i < now; i += THREADS) {
                const uint32_t l = l0 + divided(i, a.k, a.k_inverse), beam = divided(l, a.slices, a.slices_inverse);
                const uint64_t key = got<THROUGH>(best + static_cast<size_t>(l0) * a.k + i);
                if (!key || base[beam].cum == -INFINITY || bin_of(top, score_of(base[beam], key)) > upto) continue;
                const Entry e = entry_of(base[beam], beam, key);
                if (n_kept == a.k && !better(e, kept[a.k - 1])) continue;
                stage[atomicAdd(&staged, 1u)] = e;
            }
            __syncthreads();
            n_kept = prune<THREADS>(kept, n_kept, stage, staged, lds.kept[turn], a.k);
            kept = lds.kept[turn];
            turn ^= 1;
        }
    }

    for (uint32_t i = threadIdx.x; i < a.k; i += THREADS) {
        const size_t at = static_cast<size_t>(item) * a.k + i;
        float score = -INFINITY;
        int32_t parent = -1, token = -1;
        if (i < n_kept) {
            score = static_cast<float>(from_ordered64(kept[i].score));  // the one rounding of a score
            parent = static_cast<int32_t>(kept[i].rest >> 56);
            token = static_cast<int32_t>(kept[i].rest & 0xffffffu);
        }
        a.scores[at] = score;
        a.parents[at] = parent;
        a.tokens[at] = token;
        // (lists that calls overlapping by mistake have mixed may hold an entry twice, and a place no parent of the item)
        if (a.out_finished)
            a.out_finished[at] = parent >= 0 && (token == a.end_token || a.finished[item * a.beams + min(static_cast<uint32_t>(parent), a.beams - 1u)]);
    }
}

template <bool ALL>
__global__ __launch_bounds__(kMergeThreads) void beam_merge_kernel(SelectArgs a) {
    __shared__ __attribute__((aligned(16))) MergeLds lds;
    merge_item<kMergeThreads, ALL, false>(a, blockIdx.x, lds);
}

// ---------------------------------------------------------------------------------------------
// selection, the slices
// ---------------------------------------------------------------------------------------------
// Orders a wave's LDS traffic between its lanes: the wave runs in step and its LDS operations are
// done in order, so only the compiler has to be held back.
__device__ __forceinline__ void wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

constexpr uint32_t kWaveList = 256;  // entries a wave's list holds; eight more are padding
constexpr uint32_t kQueue = 288;     // vectors a wave's queue holds: a tile's 256, and what was too few to look through

// The k-th largest of list[0..n), n >= k; the keys are unique and none is 0.  For lists that grew too long only.
__device__ __forceinline__ uint64_t kth_key(const uint64_t* list, uint32_t n, uint32_t k) {
    const uint32_t lane = threadIdx.x & 63u;
    uint64_t high = 0, low = ~0ull;
    for (uint32_t at = lane; at < n; at += 64) {
        high = max(high, list[at]);
        low = min(low, list[at]);
    }
    for (int o = 32; o; o >>= 1) {
        high = max(high, static_cast<uint64_t>(__shfl_xor(static_cast<unsigned long long>(high), o)));
        low = min(low, static_cast<uint64_t>(__shfl_xor(static_cast<unsigned long long>(low), o)));
    }
    if (high == low) return high;
    // bits in which all agree need no step
    const int alike = __clzll(static_cast<long long>(high ^ low));
    uint64_t t = alike ? high & ~(~0ull >> alike) : 0;
#pragma unroll 1
    for (int bit = 63 - alike; bit >= 0; --bit) {
        const uint64_t c = t | (1ull << bit);
        uint32_t m = 0;
#pragma unroll
        for (uint32_t r = 0; r < kWaveList / 64; ++r) {
            if (r * 64 >= n) break;
            m += __popcll(__ballot(r * 64 + lane < n && list[r * 64 + lane] >= c));
        }
        if (m >= k) t = c;
        if (m == k) break;
    }
    return t;
}

// Leaves the entries of list[0..n) that reach t, in front.
__device__ __forceinline__ uint32_t keep_from(uint64_t* list, uint32_t n, uint64_t t) {
    const uint32_t lane = threadIdx.x & 63u;
    uint32_t kept = 0;
    for (uint32_t at = 0; at < n; at += 64) {
        const uint64_t key = at + lane < n ? list[at + lane] : 0;
        const uint64_t mask = __ballot(key != 0 && key >= t);
        wave_fence();
        if (key != 0 && key >= t) list[kept + lanes_before(mask)] = key;
        wave_fence();
        kept += __popcll(mask);
    }
    return kept;
}

constexpr int kVecs = 4;  // 16-byte vectors a thread holds: a tile is 16 KiB of logits
template <typename T> constexpr uint32_t tile_of() { return kThreads * kVecs * Vec<T>::n; }

// A thread's part of a tile, as it came from memory.  What lies behind the row is -inf.
template <typename T, bool MASKED>
struct TilePart {
    uint4 raw[kVecs];
    uint8_t bits[kVecs];

    // `end`: behind the tile.  Full tiles are plain loads; in the last one the vectors that reach past the row are
    // fetched by elements.
    __device__ __forceinline__ void load(const T* x, const uint8_t* mask, uint32_t at, uint32_t end, uint32_t vocab) {
        constexpr uint32_t V = Vec<T>::n;
        const bool full = end <= vocab;
#pragma unroll
        for (uint32_t j = 0; j < kVecs; ++j) {
            const uint32_t from = at + j * 64 * V;
            raw[j] = Vec<T>::tail(x, 0);
            if (full || from + V <= vocab) {
                // read once: nontemporal (64 x 8 x 131072, logits not in any cache: 37 -> 35 us)
                typedef uint32_t Words __attribute__((ext_vector_type(4), aligned(1)));
                const Words w = __builtin_nontemporal_load(reinterpret_cast<const Words*>(x + from));
                raw[j] = uint4{w.x, w.y, w.z, w.w};
            }
            if (MASKED) {
                bits[j] = 0;
                if (full || from < vocab) bits[j] = mask[from >> 3];
            }
        }
        if (full) return;
#pragma unroll
        for (uint32_t j = 0; j < kVecs; ++j) {
            const uint32_t from = at + j * 64 * V;
            if (from < vocab && from + V > vocab) raw[j] = Vec<T>::tail(x + from, vocab - from);
        }
    }
    __device__ __forceinline__ void unpack(uint32_t at, float* f) const {
        constexpr uint32_t V = Vec<T>::n;
#pragma unroll
        for (uint32_t j = 0; j < kVecs; ++j) {
            Vec<T>::unpack(raw[j], f + j * V);
            if (MASKED) {
                const uint32_t b = static_cast<uint32_t>(bits[j]) >> (at & 7u);  // a wave's vectors are 64 V apart: at & 7 is the same in all
#pragma unroll
                for (uint32_t e = 0; e < V; ++e) {
                    const uint32_t keep = static_cast<uint32_t>(static_cast<int32_t>(b << (31 - e)) >> 31);
                    f[j * V + e] = __uint_as_float((__float_as_uint(f[j * V + e]) & keep) | (0xff800000u & ~keep));
                }
            }
        }
    }
};

// Zeros behind a list, so that it can be read in eights.
__device__ __forceinline__ void pad_list(uint64_t* list, uint32_t n) {
    const uint32_t lane = threadIdx.x & 63u;
    if (lane < 8) list[n + lane] = 0;
}
// The number of entries in a workgroup's padded lists that are larger than key.
__device__ __forceinline__ uint32_t larger(const uint64_t (*lists)[kWaveList + 8], const uint32_t (&listed)[kWaves], uint64_t key) {
    uint32_t above = 0;
    for (int w = 0; w < kWaves; ++w) {
        for (uint32_t j = 0; j < listed[w]; j += 8) {
            uint64_t other[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) other[e] = lists[w][j + e];
#pragma unroll
            for (int e = 0; e < 8; ++e) above += other[e] > key;
        }
    }
    return above;
}

// Candidates are the elements that reach a threshold which k elements are known to reach: in the first tile
// one that k of its 1024 vectors' maxima reach (few more do, by their counts), then the k-th best of that
// tile, in long slices later on one by the counts of all candidates.  Every wave collects its own in a list, so
// nothing waits inside the loop over the other tiles.  The few vectors that hold a candidate go through a queue, where a
// wave tests 64 of their elements at a time: a test and a branch for every element of a tile took 15 us
// of a call's (64 x 8 x 131072 bfloat16, k = 16).
// JOINED: the workgroup that finishes an item's last slice joins them.
template <typename T, bool MASKED, bool JOINED>
__global__ __launch_bounds__(kThreads, 4) void beam_slice_kernel(SelectArgs a) {
    struct SliceLds {
        uint4 queue[kWaves][kQueue];
        uint64_t lists[kWaves][kWaveList + 8];
        uint32_t queue_token[kWaves][kQueue];
    };
    union Lds {
        SliceLds slice;
        MergeLds merge;
    };
    __shared__ __attribute__((aligned(16))) char lds_bytes[JOINED ? sizeof(Lds) : sizeof(SliceLds)];
    Lds& lds = *reinterpret_cast<Lds*>(lds_bytes);
    auto& lists = lds.slice.lists;
    __shared__ uint32_t is_last;
    __shared__ uint64_t block_kth;
    __shared__ __attribute__((aligned(16))) uint32_t bins[kBins], end_bins[kBins], seen[kBins];  // of the first tile, of the lists, of candidates
    __shared__ uint32_t listed[kWaves], wave_top[kWaves], some_count;
    __shared__ float wave_ref[kWaves];
    __shared__ double wave_total[kWaves];
    constexpr int V = Vec<T>::n;
    constexpr uint32_t kTile = tile_of<T>();

    const uint32_t row = blockIdx.x / a.slices, slice = blockIdx.x - row * a.slices;
    const uint32_t lane = threadIdx.x & 63u, wave = uniform(threadIdx.x >> 6);
    const uint32_t k = a.k;
    SliceInfo* info = a.info + static_cast<size_t>(row) * a.slices + slice;
    if (!finite(a.cum[row]) || (a.finished && a.finished[row])) {
        // nothing is looked up in a row that offers nothing by its logits
        if (threadIdx.x == 0) {
            put<JOINED>(&info->sum, 0.0);
            put<JOINED>(&info->max, -INFINITY);
        }
        if (JOINED) goto done;
        return;
    }
    {
    const T* x = static_cast<const T*>(a.logits) + static_cast<int64_t>(row) * a.row_stride;
    const uint8_t* mask = MASKED ? reinterpret_cast<const uint8_t*>(a.allowed + static_cast<int64_t>(row) * a.allowed_stride) : nullptr;
    const uint32_t first = slice * a.tiles_per_slice * kTile;
    const uint32_t last = min(a.vocab, first + a.tiles_per_slice * kTile);
    const uint32_t mine = wave * (kTile / kWaves) + lane * V;

    // candidates are counted by their distance below the first tile's maximum, so that the threshold rises with the
    // tiles: after n of them a tile has k / n candidates, not k (64 x 8 x 131072 bfloat16, a call: k = 16 38 -> 35 us,
    // k = 64 52 -> 42).  Not in slices of few tiles (64 x 4 x 65536 float32, four tiles: 20.6 -> 21.2).
    const bool counted = last - first > 4 * kTile;
    uint64_t* list = lists[wave];
    uint4* queue = lds.slice.queue[wave];
    uint32_t* queue_token = lds.slice.queue_token[wave];
    uint32_t n = 0, q = 0;       // entries in the list, vectors in the queue
    uint64_t reach = static_cast<uint64_t>(kLowestFinite) << 32;  // what an entry has to reach
    float thr = -FLT_MAX;        // and so an element: the logit of `reach`
    double sum = 0.0;            // this lane's share, relative to ref
    float ref = -INFINITY;       // the wave's maximum so far (the workgroup's, in the first tile)
    uint32_t high = 0;           // the first tile's maximum, ordered

    // the queue's vectors in order of their tokens, 64 elements at a time; all of them, or whole rounds only
    constexpr uint32_t kRound = 64 / V;
    auto empty_queue = [&](bool all) {
        wave_fence();
        uint32_t done = 0;
        for (; done < q && (all || q - done >= kRound); done += kRound) {
            if (n > kWaveList - 64) {
                reach = uniform(kth_key(list, n, k));
                thr = from_ordered(static_cast<uint32_t>(reach >> 32));
                n = uniform(keep_from(list, n, reach));
            }
            const bool some = done * V + lane < q * V;
            const float v = Vec<T>::one(queue, done * V + lane);
            const uint64_t key = static_cast<uint64_t>(ordered(v)) << 32 | ~(queue_token[done + lane / V] + lane % V);
            const uint64_t who = __ballot(some && key >= reach);
            if (some && key >= reach) list[n + lanes_before(who)] = key;
            n += __popcll(who);
        }
        wave_fence();
        if (done < q && lane < kRound) {
            const uint4 v = queue[done + lane];
            const uint32_t token = queue_token[done + lane];
            wave_fence();
            queue[lane] = v;
            queue_token[lane] = token;
        }
        wave_fence();
        q = done < q ? q - done : 0;
    };

    TilePart<T, MASKED> next;
    next.load(x, mask, first + mine, first + kTile, a.vocab);
    for (uint32_t tile = first; tile < last; tile += kTile) {
        float f[kVecs * V];
        next.unpack(tile + mine, f);
        if (tile + kTile < last) next.load(x, mask, tile + kTile + mine, tile + 2 * kTile, a.vocab);
        float top[kVecs];
        float most = -INFINITY;
#pragma unroll
        for (int j = 0; j < kVecs; ++j) {
            top[j] = f[j * V];
#pragma unroll
            for (int e = 1; e < V; ++e) top[j] = fmaxf(top[j], f[j * V + e]);
            most = fmaxf(most, top[j]);
        }
        if (tile == first) {
            const float wave_high = wave_max(most);
            if (lane == 0) wave_top[wave] = ordered(wave_high);
            bins[threadIdx.x] = bins[threadIdx.x + kThreads] = 0;
            end_bins[threadIdx.x] = end_bins[threadIdx.x + kThreads] = 0;
            if (counted) seen[threadIdx.x] = seen[threadIdx.x + kThreads] = 0;
            __syncthreads();
            const uint32_t o = max(max(wave_top[0], wave_top[1]), max(wave_top[2], wave_top[3]));
#pragma unroll
            for (int j = 0; j < kVecs; ++j)
                if (top[j] >= thr) atomicAdd(&bins[bin_of(o - ordered(top[j]))], 1u);
            __syncthreads();
            high = uniform(o);
            ref = from_ordered(high);
            const uint32_t within = end_of_bin(bin_with(bins, k));
            if (o > kLowestFinite && o - kLowestFinite > within) {
                thr = uniform(from_ordered(o - within));
                reach = static_cast<uint64_t>(uniform(o - within)) << 32;
            }
        }

        // sum of exponentials relative to the maximum, as powers of two.  log2 e is in two parts: the rounded factor alone is
        // 1.3e-8 off, always to the same side, which moves the logarithm of the sum by that times the mean distance from the
        // maximum (for a leader over a flat row of 2^24 the sum's log was 1.66e-7 off, with both parts it is 4e-9; 64 x 8 x 131072
        // bfloat16, k = 16: 33.2 -> 34.9 us a call)
        if (__any(most > ref)) {
            const float new_ref = wave_max(most);
            sum *= exp(static_cast<double>(ref) - static_cast<double>(new_ref));
            ref = new_ref;
        }
        const float base = ref > -INFINITY ? ref : 0.0f;
        constexpr float kLog2eHi = 1.44269502162933349609375f, kLog2eLo = 1.92596298909109e-8f;
#pragma unroll
        for (int j = 0; j < kVecs * V; j += 8) {
            float e[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float d = f[j + i] - base;
                e[i] = __builtin_amdgcn_exp2f(fmaf(d, kLog2eHi, d * kLog2eLo));
            }
            sum += static_cast<double>(((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7])));
        }

        const bool final_tile = tile + kTile >= last;
        if (__any(most >= thr)) {
            uint64_t who[kVecs];
            uint32_t passing = 0;
#pragma unroll
            for (int j = 0; j < kVecs; ++j) {
                who[j] = __ballot(top[j] >= thr);
                passing += __popcll(who[j]);
            }
            if (passing > k + 32) {
                // a tile that is better than all before it: k of its own vectors set the threshold (a row that rises
                // with the token, 64 x 8 x 131072: 730 us without this, 158 with it)
                uint32_t o[kVecs];
#pragma unroll
                for (int j = 0; j < kVecs; ++j) o[j] = ordered(top[j]);
                const uint64_t floor = static_cast<uint64_t>(reached_by(o, k)) << 32;
                if (floor > reach) {
                    reach = floor;
                    thr = from_ordered(static_cast<uint32_t>(reach >> 32));
#pragma unroll
                    for (int j = 0; j < kVecs; ++j) who[j] = __ballot(top[j] >= thr);
                }
            }
#pragma unroll
            for (int j = 0; j < kVecs; ++j) {
                if (!who[j]) continue;
                if (top[j] >= thr) {
                    const uint32_t slot = q + lanes_before(who[j]);
                    queue[slot] = Vec<T>::pack(f + j * V);
                    queue_token[slot] = tile + mine + j * 64 * V;
                    if (counted && tile != first) atomicAdd(&seen[bin_of(high - min(high, ordered(top[j])))], 1u);
                }
                q += __popcll(who[j]);
            }
        }
        if (q >= 2 * kRound || (q && (tile == first || final_tile))) empty_queue(tile == first || final_tile);
        // later tiles' tokens are larger: an element that equals the entry to be reached would come behind it
        if (static_cast<uint32_t>(reach)) {
            reach = ((reach >> 32) + 1) << 32;
            thr = from_ordered(static_cast<uint32_t>(reach >> 32));
        }
        // after the second tile, the fourth, the eighth: what other waves have not counted yet leaves the threshold lower
        const uint32_t before = (tile - first) / kTile;
        if (counted && before && (before & (before + 1)) == 0 && !final_tile) {
            const uint32_t within = end_of_bin(bin_with(seen, k));
            if (high > within && high - within > static_cast<uint32_t>(reach >> 32)) {
                reach = static_cast<uint64_t>(uniform(high - within)) << 32;
                thr = from_ordered(static_cast<uint32_t>(reach >> 32));
            }
        }
        if (tile == first && tile + kTile < last) {
            if (threadIdx.x == 0) block_kth = 0;
            if (lane == 0) listed[wave] = n;
            pad_list(list, n);
            __syncthreads();
            const uint32_t has[kWaves] = {uniform(listed[0]), uniform(listed[1]), uniform(listed[2]), uniform(listed[3])};
            for (uint32_t i = lane; i < n; i += 64) {
                const uint32_t rank = larger(lists, has, list[i]);
                if (counted && rank < k) atomicAdd(&seen[bin_of(high - static_cast<uint32_t>(list[i] >> 32))], 1u);
                if (rank == k - 1) block_kth = list[i];
            }
            __syncthreads();
            const uint64_t beyond = ((uniform(block_kth) >> 32) + 1) << 32;
            if (block_kth && beyond > reach) {
                reach = beyond;
                thr = from_ordered(static_cast<uint32_t>(reach >> 32));
            }
        }
    }

    if (n > 2 * k + 32) n = uniform(keep_from(list, n, uniform(kth_key(list, n, k))));

    const double total = wave_sum(sum);
    pad_list(list, n);
    if (lane == 0) {
        listed[wave] = n;
        wave_ref[wave] = ref;
        wave_total[wave] = total;
    }
    __syncthreads();
    // the four lists as one, sorted: an entry's place is the number of larger ones
    uint64_t* best = a.best + (static_cast<size_t>(row) * a.slices + slice) * k;
    const uint32_t has[kWaves] = {uniform(listed[0]), uniform(listed[1]), uniform(listed[2]), uniform(listed[3])};
    const uint32_t all = has[0] + has[1] + has[2] + has[3];
    const float m = fmaxf(fmaxf(wave_ref[0], wave_ref[1]), fmaxf(wave_ref[2], wave_ref[3]));
    if (all <= 2 * k) {
        for (uint32_t i = lane; i < n; i += 64) {
            const uint32_t rank = larger(lists, has, list[i]);
            if (rank < k) put<JOINED>(best + rank, list[i]);
        }
    } else {
        // many more than k: first those that are near enough to the largest, by their counts
        uint64_t* const some = reinterpret_cast<uint64_t*>(lds.slice.queue);
        const uint32_t o = ordered(m);
        for (uint32_t i = lane; i < n; i += 64) atomicAdd(&end_bins[bin_of(o - static_cast<uint32_t>(list[i] >> 32))], 1u);
        if (threadIdx.x == 0) some_count = 0;
        __syncthreads();
        const uint32_t upto = bin_with(end_bins, k);
        for (uint32_t i = lane; i < n; i += 64)
            if (bin_of(o - static_cast<uint32_t>(list[i] >> 32)) <= upto) some[atomicAdd(&some_count, 1u)] = list[i];
        __syncthreads();
        const uint32_t count = uniform(some_count);
        for (uint32_t i = threadIdx.x; i < count; i += kThreads) {
            const uint64_t key = some[i];
            uint32_t rank = 0;
            for (uint32_t j = 0; j < count; j += 8) {
                uint64_t other[8];
#pragma unroll
                for (uint32_t e = 0; e < 8; ++e) other[e] = some[j + e];
#pragma unroll
                for (uint32_t e = 0; e < 8; ++e) rank += j + e < count && other[e] > key;
            }
            if (rank < k) put<JOINED>(best + rank, key);
        }
    }
    for (uint32_t i = all + threadIdx.x; i < k; i += kThreads) put<JOINED>(best + i, uint64_t{0});
    if (wave == 0) {
        double s = 0.0;
        if (lane < kWaves) {
            // a wave without a number above -inf has no maximum to scale by; its sum is 0, or a NaN to be passed on
            s = wave_total[lane];
            if (wave_ref[lane] > -INFINITY && wave_ref[lane] != m) s *= exp(static_cast<double>(wave_ref[lane]) - static_cast<double>(m));
        }
        s += __shfl_xor(s, 1);
        s += __shfl_xor(s, 2);
        if (lane == 0) {
            put<JOINED>(&info->sum, s);
            put<JOINED>(&info->max, m);
        }
    }
    }
done:
    if (!JOINED) return;
    const uint32_t item = row / a.beams, slices = a.beams * a.slices;
    // every wave's stores have gone through to where all XCDs see them (a barrier alone does not wait for that) before
    // one thread counts the slice, and whichever workgroup comes last, on whatever XCD, reads them there
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0) {
        const uint32_t before = __hip_atomic_fetch_add(&a.arrived[item * kCounterWords], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        is_last = before + 1 == slices;
        if (before + 1 == slices) a.arrived[item * kCounterWords] = 0;  // for the next call on the stream
    }
    __syncthreads();
    if (!is_last) return;
    merge_item<kThreads, false, true>(a, item, lds.merge);
}

// ---------------------------------------------------------------------------------------------
// reordering
// ---------------------------------------------------------------------------------------------
constexpr int kStatesPerLaunch = 24;
struct StateDesc {
    const char* src;
    char* dst;
    int64_t src_row, dst_row;            // bytes between rows
    int64_t src_outer[2], dst_outer[2];  // bytes between pieces, outermost first
    uint32_t outer[2];
    uint32_t threads_log2;               // threads a piece gets
    uint32_t chunks;                     // parts of a piece, 16 bytes a thread each
    uint64_t unit_bytes, units;
};
struct ReorderArgs {
    StateDesc state[kStatesPerLaunch];
    const int32_t* parents;
    const int32_t* lengths;  // or null
    uint32_t src_beams, dst_beams, k;
};

// Up to 16 bytes at p, n of them wanted.
__device__ __forceinline__ uint4 load_bytes(const char* p, uint32_t n) {
    uint4 v{0, 0, 0, 0};
    if (n >= 16) {
        const Bytes16 b = *reinterpret_cast<const Bytes16*>(p);
        return uint4{b.w[0], b.w[1], b.w[2], b.w[3]};
    }
    if (n & 8) { const Bytes8 b = *reinterpret_cast<const Bytes8*>(p); v.x = b.w[0]; v.y = b.w[1]; p += 8; }
    if (n & 4) { v.z = reinterpret_cast<const Bytes4*>(p)->w; p += 4; }
    if (n & 2) { v.w = reinterpret_cast<const Bytes2*>(p)->w; p += 2; }
    if (n & 1) v.w |= static_cast<uint32_t>(*reinterpret_cast<const uint8_t*>(p)) << 16;
    return v;
}
// Stores of whole vectors are nontemporal: the rows are larger than the L2s that would hold them to the kernel's end
// (934 MB: 181 -> 166 us, 2.8 GB: 547 -> 525, 252 MB: 45 -> 40).
__device__ __forceinline__ void store_bytes(char* p, uint4 v, uint32_t n) {
    if (n >= 16) {
        typedef uint32_t Words __attribute__((ext_vector_type(4), aligned(1)));
        __builtin_nontemporal_store(Words{v.x, v.y, v.z, v.w}, reinterpret_cast<Words*>(p));
        return;
    }
    if (n & 8) { *reinterpret_cast<Bytes8*>(p) = Bytes8{{v.x, v.y}}; p += 8; }
    if (n & 4) { *reinterpret_cast<Bytes4*>(p) = Bytes4{v.z}; p += 4; }
    if (n & 2) { *reinterpret_cast<Bytes2*>(p) = Bytes2{static_cast<uint16_t>(v.w)}; p += 2; }
    if (n & 1) *reinterpret_cast<uint8_t*>(p) = static_cast<uint8_t>(v.w >> 16);
}

// A thread holds the same 16 bytes of every row of its batch item: all of them are loaded, each from
// its parent's row, before any is stored, so a permutation with repeats works in place and reads
// and writes what changes once.  Nothing else touches those bytes.
template <int ROWS>
__global__ __launch_bounds__(kThreads) void beam_reorder_kernel(ReorderArgs a) {
    const StateDesc& s = a.state[blockIdx.y];
    const uint32_t per_block = kThreads >> s.threads_log2;
    const uint32_t pieces = s.outer[0] * s.outer[1];
    const uint32_t groups = (pieces + per_block - 1) / per_block;
    // every eighth workgroup goes to the same XCD: each gets a stretch of a row of its own, so that it walks few pages
    // (934 MB: 168 -> 135 us, 2.8 GB: 525 -> 512), and not the same stretch of every row, which may be the empty one
    uint32_t stretch = blockIdx.x & 7u;
    if ((gridDim.x & 7u) == 0) stretch = (stretch + blockIdx.y + blockIdx.z) & 7u;
    uint32_t b = stretch * (gridDim.x >> 3) + min(stretch, gridDim.x & 7u) + (blockIdx.x >> 3);
    const uint32_t chunk = b % s.chunks;
    b /= s.chunks;
    const uint32_t group = b % groups;
    if (b / groups) return;  // a state of smaller rows than the call's largest
    const uint32_t batch_item = blockIdx.z;
    const uint32_t piece = group * per_block + (threadIdx.x >> s.threads_log2);
    if (piece >= pieces) return;
    uint64_t units = s.units;
    if (a.lengths) {
        const int32_t len = a.lengths[batch_item];
        const uint64_t want = len < 0 ? 0 : static_cast<uint64_t>(len);
        units = want < units ? want : units;
    }
    const uint64_t bytes = units * s.unit_bytes;
    const uint64_t at = (static_cast<uint64_t>(chunk) * (1u << s.threads_log2) + (threadIdx.x & ((1u << s.threads_log2) - 1u))) * 16u;
    if (at >= bytes) return;
    const uint32_t n = bytes - at < 16 ? static_cast<uint32_t>(bytes - at) : 16u;
    const uint32_t o0 = s.outer[1] > 1 ? piece / s.outer[1] : piece, o1 = s.outer[1] > 1 ? piece - o0 * s.outer[1] : 0;
    const char* src = s.src + static_cast<int64_t>(batch_item) * a.src_beams * s.src_row + o0 * s.src_outer[0] + o1 * s.src_outer[1] + at;
    char* dst = s.dst + static_cast<int64_t>(batch_item) * a.dst_beams * s.dst_row + o0 * s.dst_outer[0] + o1 * s.dst_outer[1] + at;
    const bool in_place = s.src == s.dst;
    const int32_t* parents = a.parents + static_cast<size_t>(batch_item) * a.k;
    uint4 v[ROWS];
#pragma unroll
    for (int j = 0; j < ROWS; ++j) {
        if (j >= static_cast<int>(a.k)) continue;
        const uint32_t p = static_cast<uint32_t>(parents[j]);
        if (p < a.src_beams && !(in_place && p == static_cast<uint32_t>(j))) v[j] = load_bytes(src + p * s.src_row, n);
    }
#pragma unroll
    for (int j = 0; j < ROWS; ++j) {
        if (j >= static_cast<int>(a.k)) continue;
        const uint32_t p = static_cast<uint32_t>(parents[j]);
        if (p < a.src_beams && !(in_place && p == static_cast<uint32_t>(j))) store_bytes(dst + j * s.dst_row, v[j], n);
    }
}

// ---------------------------------------------------------------------------------------------
// backtrace
// ---------------------------------------------------------------------------------------------
struct BacktraceArgs {
    const int32_t* tokens;
    const int32_t* parents;
    const int32_t* steps;  // or null
    int32_t* out;          // [batch][k][out_stride]
    int64_t out_stride;
    uint32_t total, batch, k;
    uint32_t k_inverse, quads_inverse;  // for divided()
    uint32_t segments, segment;  // workgroups an item gets, and the steps that each writes
};

// A step's parents are a map of k places, and maps join in any grouping: a workgroup keeps a window of steps in
// LDS (a byte a place), its groups of threads each walk a chunk of it, a scan over the chunks' maps
// tells where every chunk is entered from, and a second walk writes down the way.  A window's chain of n
// dependent look-ups becomes one of 2 n / groups + log2(groups), all of them in LDS.  A segment's workgroup
// walks through everything behind it first, which needs no traffic between workgroups.
constexpr uint32_t kTraceThreads = 1024;
constexpr uint32_t kWindow = 32768;  // places in LDS at once, of steps that are only walked through
constexpr uint32_t kOwn = 8192;      // and of steps that are written, whose tokens follow the parents in the same LDS
constexpr uint32_t kOwnEach = kOwn / kTraceThreads;

__global__ __launch_bounds__(kTraceThreads) void beam_backtrace_kernel(BacktraceArgs a) {
    __shared__ __attribute__((aligned(16))) uint8_t parent_of[kWindow];
    __shared__ __attribute__((aligned(16))) uint8_t way[kOwn];
    __shared__ uint8_t maps[2][kTraceThreads];
    __shared__ uint8_t entry[2][kMaxK];
    // an XCD's workgroups (every eighth) take neighbouring items with all their segments: a line of a step's
    // row holds several items, and a segment reads what the later ones read, so its L2 serves them all
    const uint32_t xcd = blockIdx.x & 7u, share = gridDim.x >> 3, more = gridDim.x & 7u;
    const uint32_t place = xcd * share + min(xcd, more) + (blockIdx.x >> 3);
    const uint32_t item = place / a.segments, k = a.k;
    const uint32_t wide_log2 = k > 1 ? 32 - __clz(k - 1) : 0, wide = 1u << wide_log2;
    const uint32_t groups = kTraceThreads >> wide_log2, group = threadIdx.x >> wide_log2, j = threadIdx.x & (wide - 1u);
    uint32_t ends = a.total;
    if (a.steps) ends = min(a.total, static_cast<uint32_t>(max(0, a.steps[item])));
    const uint32_t s0 = (place - item * a.segments) * a.segment, s1 = min(ends, s0 + a.segment);
    if (s0 >= ends) return;
    const size_t step_places = static_cast<size_t>(a.batch) * k;
    uint32_t turn = 0;
    if (threadIdx.x < k) entry[0][threadIdx.x] = static_cast<uint8_t>(threadIdx.x);
    for (uint32_t w1 = ends; w1 > s0;) {
        const bool own = w1 <= s1;
        const uint32_t border = own ? s0 : s1;
        const uint32_t window = (own ? kOwn : kWindow) / k;
        const uint32_t w0 = w1 - border > window ? w1 - window : border, n = w1 - w0;
        const size_t origin = w0 * step_places + static_cast<size_t>(item) * k;
        const int32_t* from = a.parents + origin;
        __syncthreads();
        // the tokens are on their way while the parents are walked
        uint32_t token[kOwnEach];
        if (own) {
            const int32_t* tokens = a.tokens + origin;
            if ((k & 3u) == 0) {
                const uint32_t quads = k >> 2;
#pragma unroll
                for (uint32_t r = 0; r < kOwnEach / 4; ++r) {
                    const uint32_t i = threadIdx.x + r * kTraceThreads;
                    if (i >= n * quads) continue;
                    const uint32_t t = divided(i, quads, a.quads_inverse), p = (i - t * quads) * 4;
                    const Bytes16 v = *reinterpret_cast<const Bytes16*>(tokens + t * step_places + p);
#pragma unroll
                    for (uint32_t e = 0; e < 4; ++e) token[4 * r + e] = v.w[e];
                }
            } else {
#pragma unroll
                for (uint32_t r = 0; r < kOwnEach; ++r) {
                    const uint32_t i = threadIdx.x + r * kTraceThreads;
                    if (i >= n * k) continue;
                    const uint32_t t = divided(i, k, a.k_inverse);
                    token[r] = static_cast<uint32_t>(tokens[t * step_places + (i - t * k)]);
                }
            }
        }
        if ((k & 3u) == 0) {
            // four places at a time; a step's row is whole fours
            const uint32_t quads = k >> 2;
#pragma unroll 4
            for (uint32_t i = threadIdx.x; i < n * quads; i += kTraceThreads) {
                const uint32_t t = divided(i, quads, a.quads_inverse), p = (i - t * quads) * 4;
                const Bytes16 v = *reinterpret_cast<const Bytes16*>(from + t * step_places + p);
                uint32_t packed = 0;
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e) packed |= (v.w[e] < k ? v.w[e] : p + e) << (8 * e);
                reinterpret_cast<uint32_t*>(parent_of)[i] = packed;
            }
        } else {
#pragma unroll 4
            for (uint32_t i = threadIdx.x; i < n * k; i += kTraceThreads) {
                const uint32_t t = divided(i, k, a.k_inverse), p = i - t * k;
                const uint32_t v = static_cast<uint32_t>(from[t * step_places + p]);
                parent_of[i] = static_cast<uint8_t>(v < k ? v : p);
            }
        }
        __syncthreads();
        const uint32_t chunk = (n + groups - 1) / groups;
        const uint32_t c0 = min(n, group * chunk), c1 = min(n, c0 + chunk);
        uint32_t at = j;
        if (j < k)
            for (uint32_t t = c1; t-- > c0;) at = parent_of[t * k + at];
        uint32_t side = 0;
        maps[0][threadIdx.x] = static_cast<uint8_t>(at);
        __syncthreads();
        // maps[group]: from behind the window to before this chunk
        for (uint32_t d = 1; d < groups; d <<= 1, side ^= 1) {
            uint32_t v = j;
            if (j < k) {
                if (group + d < groups) v = maps[side][(group + d) * wide + j];
                v = maps[side][group * wide + v];
            }
            maps[side ^ 1][threadIdx.x] = static_cast<uint8_t>(v);
            __syncthreads();
        }
        if (j < k) {
            at = entry[turn][j];
            if (group == 0) entry[turn ^ 1][j] = maps[side][at];
            if (own) {
                if (group + 1 < groups) at = maps[side][(group + 1) * wide + at];
                for (uint32_t t = c1; t-- > c0;) {
                    way[t * k + j] = static_cast<uint8_t>(at);
                    at = parent_of[t * k + at];
                }
            }
        }
        turn ^= 1;
        __syncthreads();
        if (own) {
            uint32_t* const tokens = reinterpret_cast<uint32_t*>(parent_of);
            if ((k & 3u) == 0) {
#pragma unroll
                for (uint32_t r = 0; r < kOwnEach / 4; ++r) {
                    const uint32_t i = threadIdx.x + r * kTraceThreads;
                    if (i < n * (k >> 2)) reinterpret_cast<uint4*>(tokens)[i] = uint4{token[4 * r], token[4 * r + 1], token[4 * r + 2], token[4 * r + 3]};
                }
            } else {
#pragma unroll
                for (uint32_t r = 0; r < kOwnEach; ++r)
                    if (threadIdx.x + r * kTraceThreads < n * k) tokens[threadIdx.x + r * kTraceThreads] = token[r];
            }
            __syncthreads();
            int32_t* out = a.out + static_cast<int64_t>(item) * k * a.out_stride + w0;
            // sequences are written along their length
            for (uint32_t t = threadIdx.x; t < n; t += kTraceThreads)
#pragma unroll 4
                for (uint32_t p = 0; p < k; ++p) out[p * a.out_stride + t] = static_cast<int32_t>(tokens[t * k + way[t * k + p]]);
        }
        w1 = w0;
    }
}

}  // namespace

// ---------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------
struct radx_hip_beam {
    int device = 0;
    uint32_t max_batch = 0, max_beams = 0, max_vocab = 0, max_k = 0;
    char* scratch = nullptr;
    uint32_t calls = 0;  // made so far: the next one's counters
};

namespace {

// Slices that the rows of a call are cut into: the workgroups that 256 CUs hold at once.  With more, every slice's first
// threshold and last ranking weigh more, and so does the join; with fewer, CUs have too little in flight (64 x 8 x
// 131072, a call: 35 us at 1024 slices, 37 at 512, 42 at 768, 41 at 1536 and 2048).
constexpr uint64_t kSlicesWanted = 1024;

// Calls within these limits are one launch: the last slice of an item joins its item.  Measured, a call as one launch
// against two (bfloat16): 1 x 8 x 65536, k = 4: 9.9 against 10.2 us; 16 x 8 x 65536, k = 16: 14.2, 14.8; 500 x 2 x 32000,
// k = 8: 23.5, 27.1; 64 x 8 x 131072, k = 16: 35, 35.5.  Not more slices an item, which all count in one word (1 x 12 x
// 131072, k = 8, 192 of them: 12.5, 11.2; 1 x 64 x 131072, 1024 of them: 31, 17), nor more entries or places than the join's 256
// threads (the other join has 1024) are quick with (1 x 2 x 131072, k = 128: 22, 17.4), nor more slices in all than the CUs
// hold at once (2000 x 8 x 32000, k = 8: 260, 227).
constexpr uint32_t kJoinedLists = 128, kJoinedEntries = 4096, kJoinedK = 64;

struct Cut {
    uint32_t tiles_per_slice, slices;
};
Cut cut_of(uint64_t rows, uint64_t vocab, uint64_t tile) {
    const uint64_t tiles = (vocab + tile - 1) / tile;
    uint64_t per = rows * tiles <= kSlicesWanted ? 1 : (rows * tiles + kSlicesWanted - 1) / kSlicesWanted;
    if (per > tiles) per = tiles;
    return Cut{static_cast<uint32_t>(per), static_cast<uint32_t>((tiles + per - 1) / per)};
}

// Bytes for the slices of any call within the limits: rows * ceil(tiles / per) <= kSlicesWanted + rows.
uint64_t most_slices(uint64_t rows, uint64_t vocab) {
    const uint64_t tiles = (vocab + tile_of<float>() - 1) / tile_of<float>();
    const uint64_t all = rows * tiles;
    return all < kSlicesWanted + rows ? all : kSlicesWanted + rows;
}
// Counters for the items of calls that are one launch: such a call has kSlicesWanted slices at most.  A handle's calls take
// its sets of counters in turn, so that two which overlap by mistake, and spoil each other's lists, leave none behind that
// has counted slices of both: every later call would join too early, or never.
constexpr uint32_t kCounterSets = 16;
uint64_t arrived_bytes(uint64_t batch) { return (batch < kSlicesWanted ? batch : kSlicesWanted) * kCounterWords * 4; }
uint64_t scratch_of(uint64_t batch, uint64_t beams, uint64_t vocab, uint64_t k) {
    return kCounterSets * arrived_bytes(batch) + most_slices(batch * beams, vocab) * (sizeof(SliceInfo) + k * 8);
}

uint32_t inverse(uint32_t d) { return static_cast<uint32_t>((0xffffffffull + d) / d); }  // ceil(2^32 / d)

const char* limits_error(uint32_t max_batch, uint32_t max_beams, uint32_t max_vocab, uint32_t max_k) {
    if (max_batch < 1 || max_batch > (1u << 20)) return "batch must be 1..2^20";
    if (max_beams < 1 || max_beams > kMaxBeams) return "beams must be 1..64";
    if (static_cast<uint64_t>(max_batch) * max_beams > (1u << 22)) return "batch x beams must be at most 2^22";
    if (max_vocab < 1 || max_vocab > kMaxVocab) return "vocab must be 1..2^24";
    if (max_k < 1 || max_k > kMaxK) return "k must be 1..128";
    return nullptr;
}

constexpr uint64_t kMaxStride = 1ull << 36;  // of elements or bytes: extents stay below 2^63

bool overlap(const void* p, uint64_t p_bytes, const void* q, uint64_t q_bytes) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(p), b = reinterpret_cast<uintptr_t>(q);
    return p && q && a < b + q_bytes && b < a + p_bytes;
}

// Whether each stride of the rows that are written spans all that the smaller ones do, so that no byte is written twice.
bool nested(const radx_hip_beam_state& t, uint64_t rows) {
    struct { uint64_t count, stride; } dims[3] = {{rows, t.dst_row}, {t.outer[0], t.dst_outer[0]}, {t.outer[1], t.dst_outer[1]}};
    std::sort(dims, dims + 3, [](const auto& p, const auto& q) { return p.stride < q.stride; });
    uint64_t extent = t.units * t.unit_bytes;
    for (const auto& d : dims) {
        if (d.count <= 1) continue;
        if (d.stride < extent) return false;
        extent += (d.count - 1) * d.stride;
    }
    return true;
}

// How a state's rows go to workgroups: threads a piece gets (a power of two, 16 bytes a thread), the parts of a
// longer piece, and workgroups a batch item.
struct RowCut {
    uint32_t threads_log2;
    uint64_t chunks, blocks;
};
RowCut row_cut_of(const radx_hip_beam_state& t) {
    RowCut c{0, 0, 0};
    const uint64_t vecs = (t.units * t.unit_bytes + 15) / 16;
    while (c.threads_log2 < 8 && (1ull << c.threads_log2) < vecs) ++c.threads_log2;
    c.chunks = (vecs + (1ull << c.threads_log2) - 1) >> c.threads_log2;
    const uint64_t per_block = kThreads >> c.threads_log2;
    c.blocks = c.chunks * ((static_cast<uint64_t>(t.outer[0]) * t.outer[1] + per_block - 1) / per_block);
    return c;
}

template <typename T>
void launch_slices(const SelectArgs& a, uint32_t rows, bool joined, hipStream_t stream) {
    const dim3 grid(rows * a.slices), block(kThreads);
    if (a.allowed && joined) hipLaunchKernelGGL((beam_slice_kernel<T, true, true>), grid, block, 0, stream, a);
    else if (a.allowed) hipLaunchKernelGGL((beam_slice_kernel<T, true, false>), grid, block, 0, stream, a);
    else if (joined) hipLaunchKernelGGL((beam_slice_kernel<T, false, true>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((beam_slice_kernel<T, false, false>), grid, block, 0, stream, a);
}

}  // namespace

extern "C" {

size_t radx_hip_beam_scratch_bytes(uint32_t max_batch, uint32_t max_beams, uint32_t max_vocab, uint32_t max_k) {
    if (limits_error(max_batch, max_beams, max_vocab, max_k)) return 0;
    return scratch_of(max_batch, max_beams, max_vocab, max_k);
}

int radx_hip_beam_create(int device, uint32_t max_batch, uint32_t max_beams, uint32_t max_vocab, uint32_t max_k,
                         radx_hip_beam** out) {
    if (!out) return bad_arg("out is NULL");
    *out = nullptr;
    if (const char* what = limits_error(max_batch, max_beams, max_vocab, max_k)) return bad_arg(what);
    int count = 0;
    RADX_TRY(hipGetDeviceCount(&count));
    if (device < 0 || device >= count) return bad_arg("no such HIP device");
    DeviceGuard guard(device);
    RADX_TRY(guard.status());
    radx_hip_beam* h = new (std::nothrow) radx_hip_beam;
    if (!h) return fail(hipErrorOutOfMemory, "new radx_hip_beam");
    h->device = device;
    h->max_batch = max_batch;
    h->max_beams = max_beams;
    h->max_vocab = max_vocab;
    h->max_k = max_k;
    const hipError_t e = hipMalloc(reinterpret_cast<void**>(&h->scratch), radx_hip_beam_scratch_bytes(max_batch, max_beams, max_vocab, max_k));
    if (e != hipSuccess) { delete h; return fail(e, "hipMalloc(scratch)"); }
    hipError_t z = hipMemset(h->scratch, 0, kCounterSets * arrived_bytes(max_batch));
    if (z == hipSuccess) z = hipStreamSynchronize(nullptr);  // other streams do not wait for the null stream
    if (z != hipSuccess) { (void)hipFree(h->scratch); delete h; return fail(z, "hipMemset(scratch)"); }
    *out = h;
    return 0;
}

int radx_hip_beam_destroy(radx_hip_beam* h) {
    if (!h) return 0;
    DeviceGuard guard(h->device);
    const hipError_t e = hipFree(h->scratch);
    delete h;
    if (e != hipSuccess) return fail(e, "hipFree(scratch)");
    return 0;
}

int radx_hip_beam_select(radx_hip_beam* h, const radx_hip_beam_select_args* s, void* stream) {
    if (!s) return bad_arg("args is NULL");
    if (const char* what = limits_error(s->batch ? s->batch : 1, s->beams, s->vocab, s->k)) return bad_arg(what);
    if (s->dtype != RADX_HIP_F32 && s->dtype != RADX_HIP_BF16 && s->dtype != RADX_HIP_F16)
        return bad_arg("dtype must be RADX_HIP_F32, RADX_HIP_BF16 or RADX_HIP_F16");
    if (s->batch == 0) return 0;
    const uint64_t rows = static_cast<uint64_t>(s->batch) * s->beams, places = static_cast<uint64_t>(s->batch) * s->k;
    const uint64_t size = s->dtype == RADX_HIP_F32 ? 4 : 2;
    if (!s->logits || !s->cum || !s->scores || !s->parents || !s->tokens) return bad_arg("NULL buffer");
    if ((s->finished == nullptr) != (s->out_finished == nullptr)) return bad_arg("finished and out_finished go together");
    if (s->finished && (s->end_token < 0 || static_cast<uint32_t>(s->end_token) >= s->vocab)) return bad_arg("end_token outside the vocabulary");
    if (s->row_stride != 0 && s->row_stride < s->vocab) return bad_arg("row_stride must be 0 or at least vocab");
    const uint64_t words = (static_cast<uint64_t>(s->vocab) + 31) / 32;
    if (s->allowed && s->allowed_stride != 0 && s->allowed_stride < words) return bad_arg("allowed_stride must be 0 or at least ceil(vocab / 32)");
    if (s->row_stride > kMaxStride || s->allowed_stride > kMaxStride) return bad_arg("stride out of range");
    if (reinterpret_cast<uintptr_t>(s->logits) % size || reinterpret_cast<uintptr_t>(s->cum) % 4 || reinterpret_cast<uintptr_t>(s->allowed) % 4 ||
        reinterpret_cast<uintptr_t>(s->scores) % 4 || reinterpret_cast<uintptr_t>(s->parents) % 4 || reinterpret_cast<uintptr_t>(s->tokens) % 4)
        return bad_arg("buffer is not aligned to its elements");
    const struct { const void* p; uint64_t bytes; } in[4] = {
        {s->logits, ((rows - 1) * s->row_stride + s->vocab) * size}, {s->cum, rows * 4},
        {s->allowed, (s->allowed_stride ? (rows - 1) * s->allowed_stride + words : words) * 4}, {s->finished, rows}};
    const struct { const void* p; uint64_t bytes; } to[4] = {{s->scores, places * 4}, {s->parents, places * 4}, {s->tokens, places * 4},
                                                             {s->out_finished, places}};
    for (int o = 0; o < 4; ++o) {
        for (const auto& i : in)
            if (overlap(to[o].p, to[o].bytes, i.p, i.bytes)) return bad_arg("an output overlaps an input");
        for (int q = 0; q < o; ++q)
            if (overlap(to[o].p, to[o].bytes, to[q].p, to[q].bytes)) return bad_arg("two outputs overlap");
    }
    if (!h) return bad_arg("handle is NULL");
    if (s->batch > h->max_batch || s->beams > h->max_beams || s->vocab > h->max_vocab || s->k > h->max_k)
        return bad_arg("batch, beams, vocab or k exceeds the handle's limits");
    DeviceGuard guard(h->device);
    RADX_TRY(guard.status());
    SelectArgs a{};
    a.logits = s->logits;
    a.row_stride = static_cast<int64_t>(s->row_stride);
    a.cum = s->cum;
    a.allowed = s->allowed;
    a.allowed_stride = static_cast<int64_t>(s->allowed_stride);
    a.finished = s->finished;
    a.end_token = s->finished ? s->end_token : -1;
    a.normalize = s->normalize;
    a.beams = s->beams;
    a.vocab = s->vocab;
    a.k = s->k;
    const Cut cut = cut_of(rows, s->vocab, size == 4 ? tile_of<float>() : tile_of<BF16>());
    a.slices = cut.slices;
    a.tiles_per_slice = cut.tiles_per_slice;
    a.k_inverse = inverse(a.k);
    a.slices_inverse = inverse(a.slices);
    a.arrived = reinterpret_cast<uint32_t*>(h->scratch + h->calls++ % kCounterSets * arrived_bytes(h->max_batch));
    char* const slices = h->scratch + kCounterSets * arrived_bytes(h->max_batch);
    a.info = reinterpret_cast<SliceInfo*>(slices);
    a.best = reinterpret_cast<uint64_t*>(slices + most_slices(static_cast<uint64_t>(h->max_batch) * h->max_beams, h->max_vocab) * sizeof(SliceInfo));
    a.scores = s->scores;
    a.parents = s->parents;
    a.tokens = s->tokens;
    a.out_finished = s->out_finished;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const uint32_t n_rows = static_cast<uint32_t>(rows);
    // the join's threads go to the lists evenly, and no list gets more than it has entries
    const uint32_t lists = a.beams * a.slices;
    auto parts_log2 = [&](uint32_t threads) {
        uint32_t log2 = 0;
        while ((lists << (log2 + 1)) <= threads && (1u << log2) < a.k && log2 < 6) ++log2;
        return log2;
    };
    auto held = [&](uint32_t log2) { return (a.k + (1u << log2) - 1) >> log2; };
    a.merge_parts_log2 = parts_log2(kThreads);
    const bool joined = n_rows * a.slices <= kSlicesWanted && lists <= kJoinedLists && lists * a.k <= kJoinedEntries && a.k <= kJoinedK;
    if (!joined) a.merge_parts_log2 = parts_log2(kMergeThreads);
    if (s->dtype == RADX_HIP_F32) launch_slices<float>(a, n_rows, joined, st);
    else if (s->dtype == RADX_HIP_BF16) launch_slices<BF16>(a, n_rows, joined, st);
    else launch_slices<_Float16>(a, n_rows, joined, st);
    RADX_TRY(hipGetLastError());
    if (joined) return 0;
    const dim3 items(s->batch), block(kMergeThreads);
    if (lists <= kMergeThreads && held(a.merge_parts_log2) <= kHeld) hipLaunchKernelGGL(beam_merge_kernel<true>, items, block, 0, st, a);
    else hipLaunchKernelGGL(beam_merge_kernel<false>, items, block, 0, st, a);
    RADX_TRY(hipGetLastError());
    return 0;
}

int radx_hip_beam_reorder(const radx_hip_beam_state* states, uint32_t n_states, const int32_t* parents, const int32_t* lengths,
                          uint32_t batch, uint32_t src_beams, uint32_t dst_beams, uint32_t k, void* stream) {
    if (src_beams < 1 || dst_beams < 1 || k < 1 || k > RADX_HIP_BEAM_MAX_ROWS) return bad_arg("k must be 1..64, beams at least 1");
    if (k > dst_beams) return bad_arg("k exceeds the rows of a batch item");
    if (batch > 65535) return bad_arg("batch must be < 2^16");
    if (static_cast<uint64_t>(batch) * src_beams > (1u << 24) || static_cast<uint64_t>(batch) * dst_beams > (1u << 24))
        return bad_arg("a state has more than 2^24 rows");
    if (batch == 0 || n_states == 0) return 0;
    if (!states || !parents) return bad_arg("NULL argument");
    if (reinterpret_cast<uintptr_t>(parents) % 4 || reinterpret_cast<uintptr_t>(lengths) % 4) return bad_arg("buffer is not aligned to its elements");
    for (uint32_t i = 0; i < n_states; ++i) {
        const radx_hip_beam_state& t = states[i];
        if (t.units == 0 || t.unit_bytes == 0 || t.outer[0] == 0 || t.outer[1] == 0) continue;
        if (!t.src || !t.dst) return bad_arg("a state is NULL");
        const uint64_t piece = t.units * t.unit_bytes;
        if (t.units > kMaxStride || t.unit_bytes > kMaxStride || t.units > kMaxStride / t.unit_bytes) return bad_arg("a state's rows are too long");
        if (static_cast<uint64_t>(t.outer[0]) * t.outer[1] > (1u << 24)) return bad_arg("a state has more than 2^24 pieces a row");
        if (row_cut_of(t).blocks >= 1u << 24) return bad_arg("a state's rows are too long for one call");  // a grid has 2^32 threads
        uint64_t reach[2] = {piece, piece};
        for (int o = 0; o < 2; ++o) {
            reach[0] += (t.outer[o] - 1) * t.src_outer[o];
            reach[1] += (t.outer[o] - 1) * t.dst_outer[o];
            if (t.outer[o] > 1 && (t.src_outer[o] > kMaxStride || t.dst_outer[o] > kMaxStride)) return bad_arg("a state's stride is out of range");
            if (t.outer[o] > 1 && t.dst_outer[o] < piece) return bad_arg("a state's pieces overlap");
        }
        if (t.dst_row < piece && static_cast<uint64_t>(batch) * dst_beams > 1) return bad_arg("a state's rows overlap");
        if (t.src_row > kMaxStride || t.dst_row > kMaxStride) return bad_arg("a state's stride is out of range");
        const bool same = t.src == t.dst;
        if (same && (t.src_row != t.dst_row || src_beams != dst_beams || t.src_outer[0] != t.dst_outer[0] || t.src_outer[1] != t.dst_outer[1]))
            return bad_arg("a state in place has two layouts");
        if (!nested(t, static_cast<uint64_t>(batch) * dst_beams)) return bad_arg("a state's rows and pieces overlap");
        if (!same && overlap(t.src, (static_cast<uint64_t>(batch) * src_beams - 1) * t.src_row + reach[0], t.dst,
                             (static_cast<uint64_t>(batch) * dst_beams - 1) * t.dst_row + reach[1]))
            return bad_arg("a state's source and destination overlap");
        for (uint32_t j = 0; j < i; ++j)
            if (t.dst == states[j].dst || t.dst == states[j].src || t.src == states[j].dst)
                return bad_arg("a state is written twice, or read and written as two states");
    }
    RADX_ON_DEVICE_OF(parents);
    hipStream_t st = static_cast<hipStream_t>(stream);
    ReorderArgs a{};
    a.parents = parents;
    a.lengths = lengths;
    a.src_beams = src_beams;
    a.dst_beams = dst_beams;
    a.k = k;
    uint32_t held = 0;
    uint64_t blocks = 0;
    for (uint32_t i = 0; i <= n_states; ++i) {
        if (held == kStatesPerLaunch || (i == n_states && held)) {
            const dim3 grid(static_cast<uint32_t>(blocks), held, batch), block(kThreads);
            if (k <= 4) hipLaunchKernelGGL(beam_reorder_kernel<4>, grid, block, 0, st, a);
            else if (k <= 8) hipLaunchKernelGGL(beam_reorder_kernel<8>, grid, block, 0, st, a);
            else if (k <= 16) hipLaunchKernelGGL(beam_reorder_kernel<16>, grid, block, 0, st, a);
            else if (k <= 32) hipLaunchKernelGGL(beam_reorder_kernel<32>, grid, block, 0, st, a);
            else hipLaunchKernelGGL(beam_reorder_kernel<64>, grid, block, 0, st, a);
            RADX_TRY(hipGetLastError());
            held = 0;
            blocks = 0;
        }
        if (i == n_states) break;
        const radx_hip_beam_state& t = states[i];
        if (t.units == 0 || t.unit_bytes == 0 || t.outer[0] == 0 || t.outer[1] == 0) continue;
        StateDesc& d = a.state[held];
        d.src = static_cast<const char*>(t.src);
        d.dst = static_cast<char*>(t.dst);
        d.src_row = static_cast<int64_t>(t.src_row);
        d.dst_row = static_cast<int64_t>(t.dst_row);
        for (int o = 0; o < 2; ++o) {
            d.outer[o] = t.outer[o];
            d.src_outer[o] = static_cast<int64_t>(t.src_outer[o]);
            d.dst_outer[o] = static_cast<int64_t>(t.dst_outer[o]);
        }
        d.unit_bytes = t.unit_bytes;
        d.units = t.units;
        const RowCut cut = row_cut_of(t);
        d.threads_log2 = cut.threads_log2;
        d.chunks = static_cast<uint32_t>(cut.chunks);
        if (cut.blocks > blocks) blocks = cut.blocks;
        ++held;
    }
    return 0;
}

int radx_hip_beam_backtrace(const int32_t* tokens, const int32_t* parents, const int32_t* steps, uint32_t total_steps, uint32_t batch,
                            uint32_t k, int32_t* out, uint64_t out_stride, void* stream) {
    if (k < 1 || k > kMaxK) return bad_arg("k must be 1..128");
    if (batch > 65535) return bad_arg("batch must be < 2^16");
    if (total_steps >= (1u << 24)) return bad_arg("total_steps must be < 2^24");
    if (batch == 0 || total_steps == 0) return 0;
    if (!tokens || !parents || !out) return bad_arg("NULL buffer");
    if (out_stride < total_steps || out_stride > kMaxStride) return bad_arg("out_stride must be at least total_steps");
    for (const void* p : {static_cast<const void*>(tokens), static_cast<const void*>(parents), static_cast<const void*>(steps), static_cast<const void*>(out)})
        if (reinterpret_cast<uintptr_t>(p) % 4) return bad_arg("buffer is not aligned to its elements");
    const uint64_t places = static_cast<uint64_t>(batch) * k, in_bytes = places * total_steps * 4;
    const uint64_t out_bytes = ((places - 1) * out_stride + total_steps) * 4;
    if (overlap(out, out_bytes, tokens, in_bytes) || overlap(out, out_bytes, parents, in_bytes) || overlap(out, out_bytes, steps, batch * 4ull))
        return bad_arg("out overlaps an input");
    RADX_ON_DEVICE_OF(out);
    // a workgroup a CU where the sequences are long enough to be cut
    const uint64_t most = (static_cast<uint64_t>(total_steps) * k + kOwn / 2 - 1) / (kOwn / 2);
    uint64_t segments = batch >= 256 ? 1 : 256 / batch;
    if (segments > most) segments = most;
    const uint32_t segment = static_cast<uint32_t>((total_steps + segments - 1) / segments);
    const uint32_t cuts = (total_steps + segment - 1) / segment;
    const BacktraceArgs a{tokens, parents, steps, out, static_cast<int64_t>(out_stride), total_steps, batch, k,
                          inverse(k), inverse(k >= 4 ? k / 4 : 1), cuts, segment};
    hipLaunchKernelGGL(beam_backtrace_kernel, dim3(cuts * batch), dim3(kTraceThreads), 0, static_cast<hipStream_t>(stream), a);
    RADX_TRY(hipGetLastError());
    return 0;
}

}  // extern "C"
