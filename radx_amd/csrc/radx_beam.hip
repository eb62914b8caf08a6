// radx_beam.hip — beam search beside the sort: selection over beams and vocabulary, reordering of
// the survivors' states, and the sequences out of the recorded choices (include/radx_hip.h).
//
// Selection is the sort's relative — the first k of a descending float order, ties by index — and
// reordering is radx_hip_permutation's: rows moved by an index.
#include <hip/hip_runtime.h>

#include <math.h>
#include <stdint.h>
#include <string.h>

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
constexpr uint32_t kLowestFinite = 0x00800000u;  // ordered(-FLT_MAX): everything below is -inf

__device__ __forceinline__ float wave_max(float v) {
    for (int o = 32; o; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
    return v;
}
__device__ __forceinline__ double wave_sum(double v) {
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

// Elements of one 16-byte vector as floats.
template <typename T> struct Vec;
template <> struct Vec<float> {
    static constexpr int n = 4;
    static constexpr int kOrderedBits = 32;  // leading bits of the ordered image that differ between values
    static __device__ __forceinline__ void unpack(const uint32_t* w, float* f) {
        for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(w[i]);
    }
    static __device__ __forceinline__ float one(const float* p) { return *p; }
};
template <> struct Vec<BF16> {
    static constexpr int n = 8;
    static constexpr int kOrderedBits = 16;
    static __device__ __forceinline__ void unpack(const uint32_t* w, float* f) {
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = __uint_as_float(w[i] << 16);
            f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
    static __device__ __forceinline__ float one(const BF16* p) { return __uint_as_float(static_cast<uint32_t>(p->bits) << 16); }
};
template <> struct Vec<_Float16> {
    static constexpr int n = 8;
    static constexpr int kOrderedBits = 19;  // sign, 8 exponent bits of the float, 10 of the fraction
    static __device__ __forceinline__ void unpack(const uint32_t* w, float* f) {
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(w[i])));
            f[2 * i + 1] = static_cast<float>(__builtin_bit_cast(_Float16, static_cast<uint16_t>(w[i] >> 16)));
        }
    }
    static __device__ __forceinline__ float one(const _Float16* p) { return static_cast<float>(*p); }
};

// A threshold that at least k (k <= 256) of 256 ordered values reach, as high as it gets: the k-th
// largest of them, or a value that exactly k reach.  Every wave computes the same from LDS.
template <int BITS>
__device__ __forceinline__ uint32_t reached_by(const uint32_t* v256, uint32_t k) {
    const uint32_t lane = threadIdx.x & 63u;
    const uint32_t a0 = v256[lane], a1 = v256[lane + 64], a2 = v256[lane + 128], a3 = v256[lane + 192];
    uint32_t t = 0;
    for (int bit = 31; bit >= 32 - BITS; --bit) {
        const uint32_t c = t | (1u << bit);
        const uint32_t n = __popcll(__ballot(a0 >= c)) + __popcll(__ballot(a1 >= c)) + __popcll(__ballot(a2 >= c)) +
                           __popcll(__ballot(a3 >= c));
        if (n >= k) t = c;
        if (n == k) break;
    }
    // the bits that are alike in all values of one sign
    if (BITS < 32 && !(t >> 31)) t |= (1u << (32 - BITS)) - 1u;
    return t;
}

// ---------------------------------------------------------------------------------------------
// selection, first kernel: one workgroup takes a slice of one row
// ---------------------------------------------------------------------------------------------
// score(row, token) = cum[row] + ((x - M) - log sum exp(x - M)): within a row the order of the scores
// is the order of the logits, so a slice can be searched for its own k best before M and the sum
// are known.  A slice leaves its maximum, its sum of exponentials relative to that maximum, and its
// k best logits, sorted.
struct SliceInfo {
    double sum;      // of exp(x - max)
    uint64_t head;   // the slice's best entry (0: none)
    float max;
    uint32_t count;  // entries left in best[]
};

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
    SliceInfo* info;            // [row][slice]
    uint64_t* best;             // [row][slice][k]: ordered logit, then ~token
    float* scores;
    int32_t* parents;
    int32_t* tokens;
    uint8_t* out_finished;
};

__device__ __forceinline__ bool finite(float x) { return fabsf(x) < INFINITY; }

constexpr int kVecs = 4;  // 16-byte vectors a thread holds: a tile is 16 KiB of logits
template <typename T> constexpr uint32_t tile_of() { return kThreads * kVecs * Vec<T>::n; }

// Entries a workgroup can stage between two prunings.  A tile holds at most 32 elements a thread; of those above the
// threshold at most k - 1 threads have any, and of those equal to it at most k are taken.
constexpr uint32_t stage_entries(uint32_t k) { return 33 * k < 1024 ? 1024 : 33 * k; }

// The k largest of from[0..n_from) and stage[0..n) into to[], sorted.  Keys are unique: an entry's place is
// the number of larger ones.
__device__ __forceinline__ uint32_t prune(const uint64_t* from, uint32_t n_from, const uint64_t* stage, uint32_t n, uint64_t* to, uint32_t k) {
    const uint32_t all = n_from + n;
    for (uint32_t i = threadIdx.x; i < all; i += kThreads) {
        const uint64_t key = i < n_from ? from[i] : stage[i - n_from];
        uint32_t above = 0;
        for (uint32_t j = 0; j < n_from; ++j) above += from[j] > key;
        for (uint32_t j = 0; j < n; ++j) above += stage[j] > key;
        if (above < k) to[above] = key;
    }
    __syncthreads();
    return all < k ? all : k;
}

template <typename T, bool MASKED>
__global__ __launch_bounds__(kThreads) void beam_slice_kernel(SelectArgs a) {
    extern __shared__ uint64_t stage[];
    __shared__ uint64_t kept_in_turn[2][kMaxK];
    __shared__ uint32_t lane_max[kThreads];
    __shared__ uint32_t staged, equals[kWaves];
    __shared__ float wave_ref[kWaves];
    __shared__ double wave_total[kWaves];
    constexpr int V = Vec<T>::n;
    constexpr uint32_t kTile = tile_of<T>();

    const uint32_t row = blockIdx.x / a.slices, slice = blockIdx.x - row * a.slices;
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    SliceInfo* info = a.info + static_cast<size_t>(row) * a.slices + slice;
    if (!finite(a.cum[row]) || (a.finished && a.finished[row])) {
        if (threadIdx.x == 0) *info = SliceInfo{0.0, 0, -INFINITY, 0};
        return;
    }
    const T* x = static_cast<const T*>(a.logits) + static_cast<int64_t>(row) * a.row_stride;
    const uint8_t* mask = MASKED ? reinterpret_cast<const uint8_t*>(a.allowed + static_cast<int64_t>(row) * a.allowed_stride) : nullptr;
    const uint32_t first = slice * a.tiles_per_slice * kTile;
    const uint32_t last = min(a.vocab, first + a.tiles_per_slice * kTile);

    double sum = 0.0;            // this lane's share, relative to ref
    float ref = -INFINITY;       // the wave's maximum so far
    uint64_t* kept = kept_in_turn[0];
    uint64_t* spare = kept_in_turn[1];
    uint32_t n_kept = 0;
    float floor_x = -INFINITY;   // an element has to be above it: the k-th best so far
    if (threadIdx.x == 0) staged = 0;

    for (uint32_t tile = first; tile < last; tile += kTile) {
        float f[kVecs * V];
#pragma unroll
        for (int j = 0; j < kVecs; ++j) {
            const uint32_t at = tile + (j * kThreads + threadIdx.x) * V;
            uint32_t bits = ~0u;
            if (at + V <= a.vocab) {
                const Bytes16 b = *reinterpret_cast<const Bytes16*>(x + at);
                Vec<T>::unpack(b.w, f + j * V);
                if (MASKED) bits = mask[at >> 3] >> (at & 7u);
            } else {
                for (int e = 0; e < V; ++e) f[j * V + e] = at + e < a.vocab ? Vec<T>::one(x + at + e) : -INFINITY;
                if (MASKED && at < a.vocab) bits = mask[at >> 3] >> (at & 7u);
            }
            if (MASKED)
                for (int e = 0; e < V; ++e) f[j * V + e] = (bits >> e) & 1u ? f[j * V + e] : -INFINITY;
        }
        float top = f[0];
#pragma unroll
        for (int e = 1; e < kVecs * V; ++e) top = fmaxf(top, f[e]);

        // sum of exponentials relative to the wave's maximum; 2^(d * log2 e) with log2 e in two parts
        const float new_ref = fmaxf(ref, wave_max(top));
        if (new_ref != ref) {
            if (ref > -INFINITY) sum *= exp(static_cast<double>(ref) - static_cast<double>(new_ref));
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

        // candidates: everything above the k-th best so far; a threshold from the threads' maxima where that is too much
        __syncthreads();  // staged is 0
        float above = floor_x;
        bool or_equal = false;
        if (n_kept < a.k) {
            lane_max[threadIdx.x] = ordered(top);
            __syncthreads();
            const uint32_t t = reached_by<Vec<T>::kOrderedBits>(lane_max, a.k);
            above = t < kLowestFinite ? -INFINITY : from_ordered(t);
            or_equal = t >= kLowestFinite;
        }
        const uint32_t room = stage_entries(a.k);
        if (top > above || (or_equal && top == above))
#pragma unroll
            for (int j = 0; j < kVecs; ++j)
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const float v = f[j * V + e];
                    if (v > above || (or_equal && v == above)) {
                        const uint32_t at = atomicAdd(&staged, 1u);
                        const uint32_t token = tile + (j * kThreads + threadIdx.x) * V + e;
                        if (at < room) stage[at] = static_cast<uint64_t>(ordered(v)) << 32 | (0xffffffffu - token);
                    }
                }
        __syncthreads();
        uint32_t n = staged;
        if (n > room) {
            // too many are equal to the threshold (or pass it): take those above a threshold first,
            // then the first k of those equal to it, in order of their tokens
            __syncthreads();
            if (threadIdx.x == 0) staged = 0;
            float cut = above;
            if (!or_equal) {
                float fresh = -INFINITY;
                for (int e = 0; e < kVecs * V; ++e) fresh = fmaxf(fresh, f[e]);
                lane_max[threadIdx.x] = ordered(fresh);
                __syncthreads();
                const uint32_t t = reached_by<Vec<T>::kOrderedBits>(lane_max, a.k);
                cut = t < kLowestFinite ? -INFINITY : fmaxf(above, from_ordered(t));
            }
            __syncthreads();
#pragma unroll
            for (int j = 0; j < kVecs; ++j)
#pragma unroll
                for (int e = 0; e < V; ++e)
                    if (f[j * V + e] > cut) {
                        const uint32_t at = atomicAdd(&staged, 1u);
                        const uint32_t token = tile + (j * kThreads + threadIdx.x) * V + e;
                        if (at < room) stage[at] = static_cast<uint64_t>(ordered(f[j * V + e])) << 32 | (0xffffffffu - token);
                    }
            uint32_t taken = 0;
            if (cut > above || or_equal)
#pragma unroll
                for (int j = 0; j < kVecs; ++j) {
                    uint32_t mine = 0;
#pragma unroll
                    for (int e = 0; e < V; ++e) mine += f[j * V + e] == cut;
                    uint32_t before = mine;
                    for (int o = 1; o < 64; o <<= 1) {
                        const uint32_t u = __shfl_up(before, o);
                        if (lane >= static_cast<uint32_t>(o)) before += u;
                    }
                    if (lane == 63u) equals[wave] = before;
                    before -= mine;
                    __syncthreads();
                    uint32_t all = 0;
                    for (uint32_t w = 0; w < kWaves; ++w) {
                        if (w < wave) before += equals[w];
                        all += equals[w];
                    }
                    before += taken;
#pragma unroll
                    for (int e = 0; e < V; ++e)
                        if (f[j * V + e] == cut) {
                            if (before < a.k) {
                                const uint32_t at = atomicAdd(&staged, 1u);
                                const uint32_t token = tile + (j * kThreads + threadIdx.x) * V + e;
                                if (at < room) stage[at] = static_cast<uint64_t>(ordered(cut)) << 32 | (0xffffffffu - token);
                            }
                            ++before;
                        }
                    taken += all;
                    __syncthreads();
                }
            __syncthreads();
            n = min(staged, room);
        }
        if (n) {
            n_kept = prune(kept, n_kept, stage, n, spare, a.k);
            uint64_t* const was = kept;
            kept = spare;
            spare = was;
            if (n_kept == a.k) floor_x = from_ordered(static_cast<uint32_t>(kept[a.k - 1] >> 32));
            if (threadIdx.x == 0) staged = 0;
        }
    }

    const double total = wave_sum(sum);
    if (lane == 0) {
        wave_ref[wave] = ref;
        wave_total[wave] = total;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        float m = wave_ref[0];
        for (int w = 1; w < kWaves; ++w) m = fmaxf(m, wave_ref[w]);
        double s = 0.0;
        for (int w = 0; w < kWaves; ++w)
            s += wave_ref[w] > -INFINITY ? wave_total[w] * exp(static_cast<double>(wave_ref[w]) - static_cast<double>(m)) : wave_total[w];
        *info = SliceInfo{s, n_kept ? kept[0] : 0, m, n_kept};
    }
    uint64_t* best = a.best + (static_cast<size_t>(row) * a.slices + slice) * a.k;
    for (uint32_t i = threadIdx.x; i < n_kept; i += kThreads) best[i] = kept[i];
}

// ---------------------------------------------------------------------------------------------
// selection, second kernel: one workgroup takes one batch item
// ---------------------------------------------------------------------------------------------
// The rows' maxima and sums are joined from their slices, every slice's entries get their scores in
// 64 bits, and the k best come out in the order (score down, beam up, logit down, token up).
// Within a beam that is the slices' own order.
constexpr uint32_t kMergeStage = 1024;

struct Entry {
    uint64_t score;  // ordered64
    uint64_t rest;   // beam, ~ordered logit, token: smaller is better
};
__device__ __forceinline__ bool better(const Entry& p, const Entry& q) {
    return p.score > q.score || (p.score == q.score && p.rest < q.rest);
}

struct RowBase {
    double top, log_sum, cum;
    int live;
};

__device__ __forceinline__ Entry entry_of(const RowBase& r, uint32_t beam, uint64_t key) {
    const uint32_t o = static_cast<uint32_t>(key >> 32), token = 0xffffffffu - static_cast<uint32_t>(key);
    const double s = r.cum + ((static_cast<double>(from_ordered(o)) - r.top) - r.log_sum);
    return Entry{ordered64(s), static_cast<uint64_t>(beam) << 56 | static_cast<uint64_t>(~o) << 24 | token};
}

__device__ __forceinline__ uint32_t prune(const Entry* from, uint32_t n_from, const Entry* stage, uint32_t n, Entry* to, uint32_t k) {
    const uint32_t all = n_from + n;
    for (uint32_t i = threadIdx.x; i < all; i += kThreads) {
        const Entry e = i < n_from ? from[i] : stage[i - n_from];
        uint32_t above = 0;
        for (uint32_t j = 0; j < n_from; ++j) above += better(from[j], e);
        for (uint32_t j = 0; j < n; ++j) above += better(stage[j], e);
        if (above < k) to[above] = e;
    }
    __syncthreads();
    return all < k ? all : k;
}

__global__ __launch_bounds__(kThreads) void beam_merge_kernel(SelectArgs a) {
    __shared__ RowBase base[kMaxBeams];
    __shared__ Entry kept_in_turn[2][kMaxK];
    __shared__ Entry stage[kMergeStage];
    __shared__ uint32_t lane_max[kThreads];
    __shared__ uint32_t staged;
    const uint32_t item = blockIdx.x;
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const uint32_t lists = a.beams * a.slices;
    const SliceInfo* info = a.info + static_cast<size_t>(item) * lists;
    const uint64_t* best = a.best + static_cast<size_t>(item) * lists * a.k;

    if (threadIdx.x == 0) staged = 0;
    for (uint32_t i = wave; i < a.beams; i += kWaves) {
        const uint32_t row = item * a.beams + i;
        const float cum = a.cum[row];
        const bool ended = a.finished && a.finished[row];
        float m = -INFINITY;
        for (uint32_t s = lane; s < a.slices; s += 64) m = fmaxf(m, info[i * a.slices + s].max);
        m = wave_max(m);
        double sum = 0.0;
        for (uint32_t s = lane; s < a.slices; s += 64) {
            const SliceInfo p = info[i * a.slices + s];
            if (p.max > -INFINITY || !(p.sum == 0.0)) sum += p.sum * exp(static_cast<double>(p.max) - static_cast<double>(m));
        }
        sum = wave_sum(sum);
        if (lane == 0) {
            // a NaN or +inf among the allowed logits has made the sum a NaN
            const bool live = !ended && finite(cum) && finite(m) && sum > 0.0 && sum < INFINITY;
            base[i] = RowBase{a.normalize ? static_cast<double>(m) : 0.0, a.normalize ? log(sum) : 0.0, static_cast<double>(cum), live};
        }
        if (ended && finite(cum) && lane == 0) {
            const uint32_t at = atomicAdd(&staged, 1u);
            stage[at] = Entry{ordered64(cum), static_cast<uint64_t>(i) << 56 | static_cast<uint32_t>(a.end_token)};
        }
    }
    __syncthreads();

    // a threshold that k heads of lists (or finished beams) reach
    uint32_t top = threadIdx.x < staged ? static_cast<uint32_t>(stage[threadIdx.x].score >> 32) : 0;
    for (uint32_t l = threadIdx.x; l < lists; l += kThreads) {
        const uint32_t beam = l / a.slices;
        if (base[beam].live && info[l].count) top = max(top, static_cast<uint32_t>(entry_of(base[beam], beam, info[l].head).score >> 32));
    }
    lane_max[threadIdx.x] = top;
    __syncthreads();
    const uint32_t cut = reached_by<32>(lane_max, a.k);
    const uint32_t ended_beams = staged;
    __syncthreads();

    for (uint32_t l = wave; l < lists; l += kWaves) {
        const uint32_t beam = l / a.slices;
        if (!base[beam].live) continue;
        const uint32_t count = info[l].count;
        if (!count || static_cast<uint32_t>(entry_of(base[beam], beam, info[l].head).score >> 32) < cut) continue;
        for (uint32_t j = lane; j < count; j += 64) {
            const Entry e = entry_of(base[beam], beam, best[static_cast<size_t>(l) * a.k + j]);
            if (static_cast<uint32_t>(e.score >> 32) < cut) continue;
            const uint32_t at = atomicAdd(&staged, 1u);
            if (at < kMergeStage) stage[at] = e;
        }
    }
    __syncthreads();
    const Entry* kept = kept_in_turn[0];
    uint32_t n_kept = 0;
    if (staged <= kMergeStage) {
        n_kept = prune(kept, 0, stage, staged, kept_in_turn[0], a.k);
    } else {
        // very many ties: the lists a few at a time
        n_kept = prune(kept, 0, stage, ended_beams, kept_in_turn[0], a.k);
        uint32_t turn = 1;
        const uint32_t step = kMergeStage / a.k;
        for (uint32_t l0 = 0; l0 < lists; l0 += step) {
            if (threadIdx.x == 0) staged = 0;
            __syncthreads();
            const uint32_t some = min(step, lists - l0);
            for (uint32_t i = threadIdx.x; i < some * a.k; i += kThreads) {
                const uint32_t l = l0 + i / a.k, j = i % a.k, beam = l / a.slices;
                if (!base[beam].live || j >= info[l].count) continue;
                const Entry e = entry_of(base[beam], beam, best[static_cast<size_t>(l) * a.k + j]);
                if (n_kept == a.k && !better(e, kept[a.k - 1])) continue;
                stage[atomicAdd(&staged, 1u)] = e;
            }
            __syncthreads();
            n_kept = prune(kept, n_kept, stage, staged, kept_in_turn[turn], a.k);
            kept = kept_in_turn[turn];
            turn ^= 1;
        }
    }

    for (uint32_t i = threadIdx.x; i < a.k; i += kThreads) {
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
        if (a.out_finished)
            a.out_finished[at] = parent >= 0 && (token == a.end_token || a.finished[item * a.beams + parent]);
    }
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
__device__ __forceinline__ void store_bytes(char* p, uint4 v, uint32_t n) {
    if (n >= 16) {
        *reinterpret_cast<Bytes16*>(p) = Bytes16{{v.x, v.y, v.z, v.w}};
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
    uint32_t b = blockIdx.x;
    const uint32_t chunk = b % s.chunks;
    b /= s.chunks;
    const uint32_t group = b % groups;
    const uint32_t item = b / groups;
    // blockIdx.z counts the batch
    if (item) return;
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
};

__global__ __launch_bounds__(kThreads) void beam_backtrace_kernel(BacktraceArgs a) {
    const uint32_t at = blockIdx.x * kThreads + threadIdx.x;
    if (at >= a.batch * a.k) return;
    const uint32_t item = at / a.k;
    uint32_t place = at - item * a.k;
    uint32_t ends = a.total;
    if (a.steps) ends = min(a.total, static_cast<uint32_t>(max(0, a.steps[item])));
    int32_t* out = a.out + static_cast<int64_t>(at) * a.out_stride;
    for (uint32_t t = ends; t-- > 0;) {
        const size_t from = (static_cast<size_t>(t) * a.batch + item) * a.k + place;
        out[t] = a.tokens[from];
        const uint32_t p = static_cast<uint32_t>(a.parents[from]);
        if (p < a.k) place = p;
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
};

namespace {

// Slices of all rows of a call that long vocabularies are cut into: enough workgroups to fill 256
// CUs several times over, and few enough that their k best stay a small part of what is read.
constexpr uint64_t kSlicesWanted = 4096;

struct Cut {
    uint32_t tiles_per_slice, slices;
};
Cut cut_of(uint64_t rows, uint64_t vocab, uint64_t tile) {
    const uint64_t tiles = (vocab + tile - 1) / tile;
    const uint64_t per = rows * tiles <= kSlicesWanted ? 1 : (rows * tiles + kSlicesWanted - 1) / kSlicesWanted;
    return Cut{static_cast<uint32_t>(per), static_cast<uint32_t>((tiles + per - 1) / per)};
}

// Bytes for the slices of any call within the limits: rows * ceil(tiles / per) <= kSlicesWanted + rows.
uint64_t most_slices(uint64_t rows, uint64_t vocab) {
    const uint64_t tiles = (vocab + tile_of<float>() - 1) / tile_of<float>();
    const uint64_t all = rows * tiles;
    return all < kSlicesWanted + rows ? all : kSlicesWanted + rows;
}
uint64_t scratch_of(uint64_t rows, uint64_t vocab, uint64_t k) { return most_slices(rows, vocab) * (sizeof(SliceInfo) + k * 8); }

const char* limits_error(uint32_t max_batch, uint32_t max_beams, uint32_t max_vocab, uint32_t max_k) {
    if (max_batch < 1 || max_batch > (1u << 20)) return "batch must be 1..2^20";
    if (max_beams < 1 || max_beams > kMaxBeams) return "beams must be 1..64";
    if (max_vocab < 1 || max_vocab > kMaxVocab) return "vocab must be 1..2^24";
    if (max_k < 1 || max_k > kMaxK) return "k must be 1..128";
    return nullptr;
}

bool overlap(const void* p, uint64_t p_bytes, const void* q, uint64_t q_bytes) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(p), b = reinterpret_cast<uintptr_t>(q);
    return p && q && a < b + q_bytes && b < a + p_bytes;
}

template <typename T>
void launch_slices(const SelectArgs& a, uint32_t rows, hipStream_t stream) {
    const size_t lds = stage_entries(a.k) * sizeof(uint64_t);
    const dim3 grid(rows * a.slices);
    if (a.allowed) hipLaunchKernelGGL((beam_slice_kernel<T, true>), grid, dim3(kThreads), lds, stream, a);
    else hipLaunchKernelGGL((beam_slice_kernel<T, false>), grid, dim3(kThreads), lds, stream, a);
}

}  // namespace

extern "C" {

size_t radx_hip_beam_scratch_bytes(uint32_t max_batch, uint32_t max_beams, uint32_t max_vocab, uint32_t max_k) {
    if (limits_error(max_batch, max_beams, max_vocab, max_k)) return 0;
    return scratch_of(static_cast<uint64_t>(max_batch) * max_beams, max_vocab, max_k);
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
    if (s->row_stride > (1ull << 40) || s->allowed_stride > (1ull << 40)) return bad_arg("stride out of range");
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
    a.info = reinterpret_cast<SliceInfo*>(h->scratch);
    a.best = reinterpret_cast<uint64_t*>(h->scratch + most_slices(static_cast<uint64_t>(h->max_batch) * h->max_beams, h->max_vocab) * sizeof(SliceInfo));
    a.scores = s->scores;
    a.parents = s->parents;
    a.tokens = s->tokens;
    a.out_finished = s->out_finished;
    hipStream_t st = static_cast<hipStream_t>(stream);
    const uint32_t n_rows = static_cast<uint32_t>(rows);
    if (s->dtype == RADX_HIP_F32) launch_slices<float>(a, n_rows, st);
    else if (s->dtype == RADX_HIP_BF16) launch_slices<BF16>(a, n_rows, st);
    else launch_slices<_Float16>(a, n_rows, st);
    RADX_TRY(hipGetLastError());
    hipLaunchKernelGGL(beam_merge_kernel, dim3(s->batch), dim3(kThreads), 0, st, a);
    RADX_TRY(hipGetLastError());
    return 0;
}

int radx_hip_beam_reorder(const radx_hip_beam_state* states, uint32_t n_states, const int32_t* parents, const int32_t* lengths,
                          uint32_t batch, uint32_t src_beams, uint32_t dst_beams, uint32_t k, void* stream) {
    if (src_beams < 1 || dst_beams < 1 || k < 1 || k > RADX_HIP_BEAM_MAX_ROWS) return bad_arg("k must be 1..64, beams at least 1");
    if (k > dst_beams) return bad_arg("k exceeds the rows of a batch item");
    if (batch > 65535) return bad_arg("batch must be < 2^16");
    if (batch == 0 || n_states == 0) return 0;
    if (!states || !parents) return bad_arg("NULL argument");
    if (reinterpret_cast<uintptr_t>(parents) % 4 || reinterpret_cast<uintptr_t>(lengths) % 4) return bad_arg("buffer is not aligned to its elements");
    for (uint32_t i = 0; i < n_states; ++i) {
        const radx_hip_beam_state& t = states[i];
        if (t.units == 0 || t.unit_bytes == 0 || t.outer[0] == 0 || t.outer[1] == 0) continue;
        if (!t.src || !t.dst) return bad_arg("a state is NULL");
        const uint64_t piece = t.units * t.unit_bytes;
        if (t.units > (1ull << 40) || t.unit_bytes > (1ull << 40) || piece > (1ull << 40)) return bad_arg("a state's rows are too long");
        if (static_cast<uint64_t>(t.outer[0]) * t.outer[1] > (1u << 24)) return bad_arg("a state has more than 2^24 pieces a row");
        uint64_t reach[2] = {piece, piece};
        for (int o = 0; o < 2; ++o) {
            reach[0] += (t.outer[o] - 1) * t.src_outer[o];
            reach[1] += (t.outer[o] - 1) * t.dst_outer[o];
            if (t.outer[o] > 1 && (t.src_outer[o] > (1ull << 40) || t.dst_outer[o] > (1ull << 40))) return bad_arg("a state's stride is out of range");
            if (t.outer[o] > 1 && t.dst_outer[o] < piece) return bad_arg("a state's pieces overlap");
        }
        if (t.dst_row < piece && static_cast<uint64_t>(batch) * dst_beams > 1) return bad_arg("a state's rows overlap");
        if (t.src_row > (1ull << 40) || t.dst_row > (1ull << 40)) return bad_arg("a state's stride is out of range");
        const bool same = t.src == t.dst;
        if (same && (t.src_row != t.dst_row || src_beams != dst_beams || t.src_outer[0] != t.dst_outer[0] || t.src_outer[1] != t.dst_outer[1]))
            return bad_arg("a state in place has two layouts");
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
        const uint64_t vecs = (t.units * t.unit_bytes + 15) / 16;
        d.threads_log2 = 0;
        while (d.threads_log2 < 8 && (1ull << d.threads_log2) < vecs) ++d.threads_log2;
        const uint64_t chunks = (vecs + (1ull << d.threads_log2) - 1) >> d.threads_log2;
        const uint64_t per_block = kThreads >> d.threads_log2;
        const uint64_t need = chunks * ((static_cast<uint64_t>(t.outer[0]) * t.outer[1] + per_block - 1) / per_block);
        if (need > 0x7fffffffull) return bad_arg("a state is too large for one call");
        d.chunks = static_cast<uint32_t>(chunks);
        if (need > blocks) blocks = need;
        ++held;
    }
    return 0;
}

int radx_hip_beam_backtrace(const int32_t* tokens, const int32_t* parents, const int32_t* steps, uint32_t total_steps, uint32_t batch,
                            uint32_t k, int32_t* out, uint64_t out_stride, void* stream) {
    if (k < 1 || k > kMaxK) return bad_arg("k must be 1..128");
    if (batch > (1u << 20)) return bad_arg("batch must be at most 2^20");
    if (total_steps >= (1u << 24)) return bad_arg("total_steps must be < 2^24");
    if (batch == 0 || total_steps == 0) return 0;
    if (!tokens || !parents || !out) return bad_arg("NULL buffer");
    if (out_stride < total_steps || out_stride > (1ull << 40)) return bad_arg("out_stride must be at least total_steps");
    for (const void* p : {static_cast<const void*>(tokens), static_cast<const void*>(parents), static_cast<const void*>(steps), static_cast<const void*>(out)})
        if (reinterpret_cast<uintptr_t>(p) % 4) return bad_arg("buffer is not aligned to its elements");
    const uint64_t places = static_cast<uint64_t>(batch) * k, in_bytes = places * total_steps * 4;
    const uint64_t out_bytes = ((places - 1) * out_stride + total_steps) * 4;
    if (overlap(out, out_bytes, tokens, in_bytes) || overlap(out, out_bytes, parents, in_bytes) || overlap(out, out_bytes, steps, batch * 4ull))
        return bad_arg("out overlaps an input");
    RADX_ON_DEVICE_OF(out);
    const BacktraceArgs a{tokens, parents, steps, out, static_cast<int64_t>(out_stride), total_steps, batch, k};
    hipLaunchKernelGGL(beam_backtrace_kernel, dim3(static_cast<uint32_t>((places + kThreads - 1) / kThreads)), dim3(kThreads), 0,
                       static_cast<hipStream_t>(stream), a);
    RADX_TRY(hipGetLastError());
    return 0;
}

}  // extern "C"
