// Drawing a class from scores: temperature, top-k, top-p, min-p, from one given uniform number per row.
//
//   order    the classes by (score descending, index ascending); NaN and -inf scores take no part
//   weight   w_j = exp((x_j - max x) / T) in f64: a draw is next to the border between two classes as often as not, and
//            f32 sums would move the borders of a flat row by as much as a class
//   kept     the first top_k of the order, of these the shortest prefix whose mass reaches top_p of theirs, of these
//            the weights >= min_p
//   token    the first kept class whose cumulative kept weight, in index order, exceeds u * (kept mass)
//   logprob  log softmax(x)[token], untempered and uncut: its sum is f32, off by (n / 512 + 64) 2^-23 of itself at most
//
// k_sample_row, one workgroup of 1 024 or 512 per row: reading and f64 sums want many waves, but an instruction that all 16 of
// 1 024 threads execute takes 16 cycles, so short lists are left to fewer while the others wait.
//   1. one read of the row: its largest score, softmax's sum, the sum at T (f32, online), the largest score of each
//      thread's share
//   2. a score below which nothing can be kept -- from top_k and the shares, from min_p, or a guess that fits most nuclei
//      -- and a second read (from registers, or cache) that collects what is not below it
//   3. at most kCandidates classes in LDS: a histogram of them over the logarithm of the weight shows the bin in which the
//      order is cut, and only that bin is put in order; the draw takes the masses of 2 048 ranges of classes, then 64
//      classes at once.  Everything is exact there but the mass that top_p refers to when neither top_k nor the row's size
//      bounds it; that one is the f32 sum, and where a border falls into its error the row is read again for the exact one
//   4. everything else: no cut at all (the draw alone), or the same cut from the whole row -- for top_p alone with one pass
//      of f64 weights (find_nucleus), otherwise, and where one bin holds too many (ties), with find_cut, which goes on to a
//      radix search of the keys.  The cut is then (key, quota): every key above `key`, and the first `quota` classes, by
//      index, whose key equals it.  The draw adds the kept weights of kPieces pieces of the row, then of a share of the one
//      that holds the answer for each thread.
// Masses that candidates and atomics add up are whole numbers of 2^-bits (bits <= 45): the order in which they arrive
// changes nothing.  The draw of step 4 adds f64 in a fixed order.
//
// What bounds it: one row, the chain of phases of one workgroup (50 001 bf16, top_k 50, top_p 0.95: 15 us, of which reading
// takes 3); many, instructions: 512 rows of 131 072 bf16 with top_p 0.9 and min_p 0.01 take 73 us = 1.8 TB/s (two rows for
// each compute unit, one after the other: 16 384 candidates leave no room for two), 256 rows of 100 003 f32
// untruncated 50 us = 2.0 TB/s (half of it f64 weights, some 150 cycles for 64); 64 rows of 65 536 f16, each with settings of
// its own, 60 us (the flattest row's; most are done after 20).
#pragma once

#include "class_common.hpp"
#include "row_weights.hpp"

namespace serhip {

constexpr int kBook = 256;
constexpr int kDeep = 8;            // vectors that a thread keeps in registers: with 1 024, a row of 65 536 16-bit scores
constexpr int kFlight = 4;          // vectors in flight of a longer row
constexpr int kSampleBins = 2048;
constexpr int kPieces = 64;         // one for each lane of a wave
constexpr float kBinsPerOctave = 64.0f;   // of the weight; the last bin takes all that is below 2^-32
constexpr int kRanked = 2048;       // candidates that can be put in order
constexpr int kCountRank = 256;     // up to here a rank is counted (n reads each), above it is sorted

struct SampleArgs {
    const void* logits;
    long long n_rows, row_stride;
    int n_classes;
    const float* uniform;
    float temperature, top_p, min_p;   // for all rows, unless the pointers below are set
    int top_k;
    const float* temperature_rows;
    const int* top_k_rows;
    const float* top_p_rows;
    const float* min_p_rows;
    int weight_bits;
    long long* token;
    float* logprob;
};

// the next one
__device__ __forceinline__ float score_above(float x) { return x > -INFINITY ? key_score(score_key(x) + 1) : -0x1.fffffep127f; }

// the digits of a key that a radix search looks at: those below `shift[last]` follow from the type
template <typename T>
struct KeyDigits;
template <>
struct KeyDigits<float> {
    static constexpr int kLevels = 3;
    static constexpr int kShift[3] = {21, 10, 0};
};
template <>
struct KeyDigits<bf16_t> {   // 16 bits of an f32
    static constexpr int kLevels = 2;
    static constexpr int kShift[2] = {21, 16};
};
template <>
struct KeyDigits<f16_t> {    // sign, 8 exponent bits and 10 mantissa bits as an f32
    static constexpr int kLevels = 2;
    static constexpr int kShift[2] = {21, 13};
};

// A batch of vectors of a row's scores from..stop for member `me` of `group` threads: base + (d * group + me) * kLen.  One
// that would reach past `stop` is loaded from stop - kLen instead: no load is conditional.  (stop >= kLen.)
template <int kCount, typename T>
__device__ __forceinline__ void load_vectors(Vec16<T> (&raw)[kCount], const T* __restrict__ x, int base, int stop, int me, int group) {
    constexpr int kLen = Vec16<T>::kLen;
#pragma unroll
    for (int d = 0; d < kCount; ++d) raw[d] = load16(x + min(base + (d * group + me) * kLen, stop - kLen));
}
// f(vector of f32, its first class); a class that belongs to another vector, or to none, is -inf.  The calls are the same
// for all lanes of a wave (whose members follow each other) as far as `base` and `stop` are.
template <int kCount, typename T, typename F>
__device__ __forceinline__ void use_vectors(const Vec16<T> (&raw)[kCount], int base, int stop, int me, int group, F f) {
    constexpr int kLen = Vec16<T>::kLen;
#pragma unroll
    for (int d = 0; d < kCount; ++d) {
        if (base + d * group * kLen >= stop) break;
        const int at = base + (d * group + me) * kLen, from = min(at, stop - kLen);
        float v[kLen];
#pragma unroll
        for (int e = 0; e < kLen; ++e) v[e] = static_cast<float>(raw[d].v[e]);
        if (from != at)
#pragma unroll
            for (int e = 0; e < kLen; ++e) v[e] = from + e < at ? -INFINITY : v[e];
        f(v, from);
    }
}
// the scores from..stop, divided among `group` threads
template <int kCount, typename T, typename F>
__device__ __forceinline__ void stream_vectors(const T* __restrict__ x, int from, int stop, int me, int group, F f) {
#pragma unroll 1
    for (int base = from; base < stop; base += kCount * group * Vec16<T>::kLen) {
        Vec16<T> raw[kCount];
        load_vectors(raw, x, base, stop, me, group);
        use_vectors(raw, base, stop, me, group, f);
    }
}

__device__ constexpr PowerTable kPowerTable;

// a row's settings; what is out of range, or NaN, is off
struct RowSettings {
    int top_k;
    float t, ct;             // temperature and log2 e / T; a temperature below 1e-30 does as 1e-30
    float u;
    double share, least;     // top_p; min_p, or a weight that is too small to be drawn
    bool greedy, use_k, use_p, use_m;
    __device__ __forceinline__ RowSettings(const SampleArgs& a, long long row) {
        const float temperature = a.temperature_rows ? a.temperature_rows[row] : a.temperature;
        const float top_p = a.top_p_rows ? a.top_p_rows[row] : a.top_p;
        const float min_p = a.min_p_rows ? a.min_p_rows[row] : a.min_p;
        top_k = a.top_k_rows ? a.top_k_rows[row] : a.top_k;
        u = fminf(fmaxf(a.uniform[row], 0.0f), 1.0f);   // (1: the last class that is kept.  NaN: 0)
        greedy = !(temperature > 0.0f && temperature < INFINITY);
        use_k = top_k >= 1 && top_k < a.n_classes;
        use_p = top_p < 1.0f;
        use_m = min_p > 0.0f;
        t = fmaxf(temperature, 1e-30f);
        ct = 1.44269504f / t;
        share = fmaxf(top_p, 0.0f);
        least = use_m ? fmaxf(fminf(min_p, 1.0f), 1e-37f) : 1e-37f;
    }
    __device__ __forceinline__ RowWeights weights(float top, int bits) const { return row_weights(top, t, bits); }
};

__device__ __forceinline__ float candidate_score(uint64_t one) { return key_score(~static_cast<uint32_t>(one >> 32)); }

// A row's draw by a workgroup of kThreads, 512 or 1 024.
template <int kThreads>
struct RowSampler {
    static constexpr int kWaves = kThreads / 64;
    static constexpr int kShare = 2048 / kThreads;   // scores of a piece that a thread keeps in registers: all, up to 131 072 classes
    // 16 384 are as many as fit the 160 KB of LDS that one workgroup of 1 024 with 128 registers a thread has for itself;
    // of workgroups of 512 a compute unit takes two
    static constexpr int kCandidates = kThreads == 1024 ? 16384 : 5888;
    static constexpr int kNucleusGuess = kThreads * 900 / 1024;   // of the shares (of a thread each): some 2 candidates in each

// of the histogram: the last bin with anything in it that begins below the target (the first one always does)
struct CutBin {
    int bin, number;             // classes in it
    uint64_t above, before;      // mass and classes before it
    uint64_t mass;               // in it
};

// inclusive prefix sum over the workgroup, in thread order; `total` too
template <typename V>
static __device__ __forceinline__ V block_scan(V x, V* s_part, V& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    x = wave_scan_sum(x);
    __syncthreads();
    if (lane == 63) s_part[wave] = x;
    __syncthreads();
    V before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        if (w < wave) before += s_part[w];
        total += s_part[w];
    }
    return x + before;
}
template <typename V>
static __device__ __forceinline__ V block_total(V x, V* s_part) {
    x = wave_sum(x);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s_part[threadIdx.x >> 6] = x;
    __syncthreads();
    V total = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) total += s_part[w];
    return total;
}

// block_scan over the first kBook threads; the others add nothing and get the total only
template <typename V>
static __device__ __forceinline__ V book_scan(V x, V* s_part, V& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (threadIdx.x < kBook) x = wave_scan_sum(x);
    __syncthreads();
    if (threadIdx.x < kBook && lane == 63) s_part[wave] = x;
    __syncthreads();
    V before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < kBook / 64; ++w) {
        if (w < wave) before += s_part[w];
        total += s_part[w];
    }
    return x + before;
}

template <int kCount = 2, typename T, typename F>
static __device__ __forceinline__ void each_vector(const T* __restrict__ x, int n, F f) {
    stream_vectors<kCount>(x, 0, n, threadIdx.x, kThreads, f);
}

struct SampleShared {
    uint64_t order[kCandidates];         // candidates: ~key and class, which sort by rank
    union {
        struct {
            uint64_t hist[kSampleBins];  // masses
            uint32_t number[kSampleBins];
        };
        uint64_t bins[kSampleBins];      // of a radix search
        uint64_t list[kRanked];          // candidates to put in order
        struct {
            uint64_t mass[64];           // of a wave's draw
            uint32_t cls[64];
        };
    };
    double piece[kPieces];               // of a row: the mass of what is kept whatever its index,
    uint32_t tied[kPieces];              // and how many classes are at the key of the cut
    union {
        uint64_t part[kWaves];
        double part_f64[kWaves];
        uint32_t part_u32[kWaves];
    };
    float stat[3][kWaves];
    uint32_t kth[2][kBook];     // cleared before the first barrier
    double power[kPowers];      // filled before it
    RowWeights rw;              // for find_cut
    CutBin cut;
    uint64_t found_above;
    uint32_t found_bin;
    uint32_t count;
    uint32_t choice;
};

// The workgroup's shared memory, by name wherever it is used: through a reference, a function that is not inlined would
// reach it with flat instructions (ranking 51 candidates: 4.4 us instead of 1.4).
static __device__ __forceinline__ SampleShared& shared_memory() {
    __shared__ SampleShared sh;
    return sh;
}

static __device__ __forceinline__ double weight(const RowWeights& rw, float x) {
    return rw.real(x, [](int j) { return shared_memory().power[j]; });
}

// sh.list[0..n) ascending, n <= kRanked
static __device__ __noinline__ void sort_list(int n) {
    uint64_t* s = shared_memory().list;
    int size = 1;
    while (size < n) size <<= 1;
    for (int i = n + threadIdx.x; i < size; i += kThreads) s[i] = ~0ull;
    for (int k = 2; k <= size; k <<= 1)
        for (int j = k >> 1; j; j >>= 1) {
            __syncthreads();
            for (int i = threadIdx.x; i < size / 2; i += kThreads) {
                const int lo = 2 * i - (i & (j - 1)), hi = lo + j;
                const uint64_t a = s[lo], b = s[hi];
                if ((a > b) == ((lo & k) == 0)) {
                    s[lo] = b;
                    s[hi] = a;
                }
            }
        }
    __syncthreads();
}

// s[0..n) ascending, n <= kCountRank, by counting what is below each (n reads of one address by all lanes)
static __device__ __forceinline__ void rank_few(uint64_t* s, int n) {
    static_assert(kCountRank <= kThreads, "a thread for each");
    uint64_t one = 0;
    int rank = -1;
    if (static_cast<int>(threadIdx.x) < n) {
        one = s[threadIdx.x];
        rank = 0;
#pragma unroll 8
        for (int j = 0; j < n; ++j) rank += s[j] < one;
    }
    __syncthreads();
    if (rank >= 0) s[rank] = one;
    __syncthreads();
}
// sh.list[0..n)
static __device__ __forceinline__ void rank_list(int n) {
    if (n <= kCountRank) rank_few(shared_memory().list, n);
    else sort_list(n);
}

// The lower edge of the 16-bit bin that holds the k-th largest of one key per thread: at least k keys are not below it.
// 0 if fewer than k keys are above 0.
static __device__ inline uint32_t kth_of_threads(uint32_t key, uint32_t k) {
    SampleShared& sh = shared_memory();
    static_assert(kBook == 256, "four bins for each lane of a wave");
    uint32_t prefix = 0, above = 0;
#pragma unroll
    for (int level = 0; level < 2; ++level) {
        const int shift = level ? 16 : 24;
        if (key && (level == 0 || key >> 24 == prefix >> 24)) atomicAdd(&sh.kth[level][(key >> shift) & 255], 1u);
        __syncthreads();
        if (threadIdx.x < 64) {   // lane i: bins 255-4i .. 252-4i
            uint32_t h[4], sum = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) sum += h[i] = sh.kth[level][255 - 4 * threadIdx.x - i];
            uint32_t before = above + wave_scan_sum(sum) - sum;
            if (threadIdx.x == 63 && before + sum < k) sh.found_bin = 0xffffffffu;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (before < k && before + h[i] >= k) {
                    sh.found_bin = 255 - 4 * threadIdx.x - i;
                    sh.found_above = before;
                }
                before += h[i];
            }
        }
        __syncthreads();
        if (sh.found_bin == 0xffffffffu) return 0;
        prefix |= sh.found_bin << shift;
        above = static_cast<uint32_t>(sh.found_above);
    }
    return prefix;
}

// Among the classes that `in` accepts: the largest key for which `above` + mass(keys >= it) reaches `target`; `above`
// becomes the mass above it.  A key's mass is its weight, or 1 where `count`.
template <typename T, typename In>
static __device__ __forceinline__ uint32_t find_key(const T* __restrict__ x, int n, const RowWeights& rw, bool count, In in, double target,
                                          uint64_t& above) {
    SampleShared& sh = shared_memory();
    using D = KeyDigits<T>;
    constexpr int kLen = Vec16<T>::kLen, kPer = kSampleBins / kThreads;
    uint32_t prefix = 0;   // the digits found so far, in place
    for (int level = 0; level < D::kLevels; ++level) {
        const int shift = D::kShift[level];
        const int width = (level == 0 ? 32 : D::kShift[level - 1]) - shift;
        const uint32_t high = level == 0 ? 0 : ~0u << D::kShift[level - 1];
        __syncthreads();
        for (int b = threadIdx.x; b < kSampleBins; b += kThreads) sh.bins[b] = 0;
        if (threadIdx.x == 0) sh.found_bin = 0;
        __syncthreads();
        each_vector<1>(x, n, [&](const float (&v)[kLen], int) {
            for (int e = 0; e < kLen; ++e) {
                const uint32_t k = score_key(v[e]);
                if (v[e] > rw.none && (k & high) == prefix && in(v[e]))
                    atomicAdd(reinterpret_cast<unsigned long long*>(&sh.bins[(k >> shift) & ((1u << width) - 1)]),
                              static_cast<unsigned long long>(count ? 1 : rw.whole(weight(rw, v[e]))));
            }
        });
        __syncthreads();
        // bins from the top, kPer for each thread; the last one that begins below the target and holds anything
        const int first = kSampleBins - 1 - kPer * static_cast<int>(threadIdx.x);
        uint64_t sum = 0, all;
        for (int i = 0; i < kPer; ++i) sum += sh.bins[first - i];
        uint64_t before = above + block_scan(sum, sh.part, all) - sum;
        uint64_t mine = 0;
        int bin = -1;
        for (int i = 0; i < kPer; ++i) {
            const uint64_t h = sh.bins[first - i];
            if (h && static_cast<double>(before) < target) {
                bin = first - i;
                mine = before;
            }
            before += h;
        }
        if (bin >= 0) atomicMax(&sh.found_bin, static_cast<uint32_t>(kSampleBins - bin));
        __syncthreads();
        if (bin >= 0 && sh.found_bin == static_cast<uint32_t>(kSampleBins - bin)) sh.found_above = mine;
        __syncthreads();
        above = sh.found_above;
        prefix |= (kSampleBins - sh.found_bin) << shift;
    }
    // the digits that the type leaves: 0 for positive numbers, ones for the inverted bits of negative ones
    const int rest = D::kShift[D::kLevels - 1];
    return prefix & 0x80000000u ? prefix : prefix | ((1u << rest) - 1);
}

// A wave's draw: lane i has a class and a mass (0: not kept), i < n.  The class at which the mass in index order first
// exceeds `goal`, which is below their sum.  `place` = how many of the classes are lower.
static __device__ __forceinline__ uint32_t draw_of_lanes(uint32_t cls, uint64_t mass, int place, int n, uint64_t goal) {
    SampleShared& sh = shared_memory();
    const int lane = threadIdx.x & 63;
    if (lane < n) {   // into index order
        sh.mass[place] = mass;
        sh.cls[place] = cls;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    const uint64_t upto = wave_scan_sum(lane < n ? sh.mass[lane] : 0);
    return sh.cls[__ffsll(static_cast<unsigned long long>(__ballot(upto > goal))) - 1];
}

// The same for a wave with a candidate in each of its first `n` lanes, not in the order of classes.
static __device__ __forceinline__ uint32_t draw_few(uint32_t cls, uint64_t mass, int n, uint64_t goal) {
    const int lane = threadIdx.x & 63;
    int place = 0;
    for (int j = 0; j < n; ++j) place += static_cast<uint32_t>(__builtin_amdgcn_readlane(cls, j)) < cls;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    return draw_of_lanes(cls, lane < n ? mass : 0, place, n, goal);
}

// The class, of the `found` in sh.order, at which the mass in index order first exceeds `goal` (which is below their sum),
// to the first wave; mass(one) is a candidate's.  The masses of 2 048 ranges of classes, the range that holds the answer,
// and again, down to a range of 64 (the first one, up to 131 072 classes), of which each lane of a wave takes a class.
template <typename Mass>
static __device__ __forceinline__ uint32_t draw_candidate(int found, uint64_t goal, int n, Mass mass) {
    SampleShared& sh = shared_memory();
    constexpr int kBits = 11, kPer = (1 << kBits) / kBook, kLast = 6;
    static_assert(1 << kBits <= kSampleBins, "room for the bins");
    uint32_t prefix = 0;
    uint64_t below = 0;
    int shift = kLast, bits = kBits;
    while (static_cast<int64_t>(1) << (shift + kBits) < n) ++shift;
    for (;;) {
        __syncthreads();
        for (int b = threadIdx.x; b < 1 << bits; b += kThreads) sh.bins[b] = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < found; i += kThreads) {
            const uint64_t one = sh.order[i];
            const uint32_t c = static_cast<uint32_t>(one);
            if (static_cast<uint64_t>(c) >> (shift + bits) == static_cast<uint64_t>(prefix) >> (shift + bits))
                atomicAdd(reinterpret_cast<unsigned long long*>(&sh.bins[(c >> shift) & ((1u << bits) - 1)]),
                          static_cast<unsigned long long>(mass(one)));
        }
        __syncthreads();
        if (shift == 0) break;
        uint64_t sum = 0, all;
        const int first = threadIdx.x * kPer, last = min(first + kPer, 1 << bits);
        if (threadIdx.x < kBook)
            for (int i = first; i < last; ++i) sum += sh.bins[i];
        const uint64_t upto = below + book_scan(sum, sh.part, all);
        if (threadIdx.x < kBook && upto > goal && upto - sum <= goal) {   // one thread
            uint64_t at = upto - sum;
            int b = first;
            while (at + sh.bins[b] <= goal) at += sh.bins[b++];
            sh.found_bin = b;
            sh.found_above = at;
        }
        __syncthreads();
        prefix |= sh.found_bin << shift;
        below = sh.found_above;
        bits = shift == kLast ? kLast : min(kBits, shift - kLast);
        shift -= bits;
    }
    // a class for each lane of the first wave
    const uint64_t upto = below + wave_scan_sum(sh.bins[threadIdx.x & 63]);
    return prefix + __ffsll(static_cast<unsigned long long>(__ballot(upto > goal))) - 1;
}

// Step 3 for at most 64 candidates, by one wave, with the candidates in the lanes: other lanes' values come from
// v_readlane (four instructions a candidate), not from LDS, whose latency a wave alone cannot hide (51 candidates:
// 11 500 cycles from LDS).  share > 1: no top_p.
static __device__ __forceinline__ uint32_t draw_in_wave(int found, const RowWeights& rw, double least, int limit, double share, float u) {
    SampleShared& sh = shared_memory();
    const int lane = threadIdx.x & 63;
    const uint64_t one = lane < found ? sh.order[lane] : ~0ull;
    const uint32_t key = static_cast<uint32_t>(one >> 32), cls = static_cast<uint32_t>(one);
    int rank = 0, place = 0;
    for (int j = 0; j < found; ++j) {
        const uint32_t other = __builtin_amdgcn_readlane(cls, j);
        rank += (static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(key, j))) << 32 | other) < one;
        place += other < cls;
    }
    const double w = weight(rw, key_score(~key));
    const uint64_t mass = lane < found ? rw.whole(w) : 0;
    if (lane < found) sh.mass[rank] = mass;   // into rank order
    const int heavy = __popcll(__ballot(lane < found && w >= least));   // a prefix of the ranks
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    const uint64_t ranked = lane < found && lane < limit ? sh.mass[lane] : 0, upto = wave_scan_sum(ranked);
    const uint64_t all = last_lane(upto);   // (not in a branch: there lane 63 may not have worked `upto` out)
    const bool kept = lane < limit && lane < heavy &&
                      (share > 1.0 || lane == 0 || static_cast<double>(upto - ranked) < share * static_cast<double>(all));
    const int n_kept = __popcll(__ballot(kept));
    const uint64_t total = last_lane(wave_scan_sum(kept ? ranked : 0));
    const uint64_t goal = min(static_cast<uint64_t>(static_cast<double>(u) * static_cast<double>(total)), total - 1);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    return draw_of_lanes(cls, rank < n_kept ? mass : 0, place, found, goal);
}

// the bin of a score in the histogram of step 4: by the logarithm of its weight, 0 = the heaviest
static __device__ __forceinline__ int weight_bin(float v, const RowWeights& rw) {
    return v == rw.top ? 0 : static_cast<int>(fminf((rw.top - v) * (rw.ct * kBinsPerOctave), static_cast<float>(kSampleBins - 1)));
}

// make(mass of all) gives begins(mass before, classes before)
template <typename Begins>
static __device__ __forceinline__ CutBin cut_bin(Begins make) {
    SampleShared& sh = shared_memory();
    constexpr int kPer = kSampleBins / kThreads;
    uint64_t sum = 0, classes = 0, all, all_classes;
    const int first = kPer * threadIdx.x;
    for (int i = 0; i < kPer; ++i) {
        sum += sh.hist[first + i];
        classes += sh.number[first + i];
    }
    uint64_t above = block_scan(sum, sh.part, all) - sum;
    uint64_t before = block_scan(classes, sh.part, all_classes) - classes;
    const auto begins = make(all);
    CutBin mine{-1, 0, 0, 0, 0};
    for (int i = 0; i < kPer; ++i) {
        const uint64_t m = sh.hist[first + i], c = sh.number[first + i];
        if (c && begins(above, before)) mine = {first + i, static_cast<int>(c), above, before, m};
        above += m;
        before += c;
    }
    if (mine.bin >= 0) atomicMax(&sh.found_bin, static_cast<uint32_t>(mine.bin));
    __syncthreads();
    if (mine.bin == static_cast<int>(sh.found_bin)) sh.cut = mine;
    __syncthreads();
    return sh.cut;
}

// a class into the histogram
static __device__ __forceinline__ void count_candidate(const RowWeights& rw, float v) {
    SampleShared& sh = shared_memory();
    const int b = weight_bin(v, rw);
    atomicAdd(reinterpret_cast<unsigned long long*>(&sh.hist[b]), static_cast<unsigned long long>(rw.whole(weight(rw, v))));
    atomicAdd(&sh.number[b], 1u);
}

static __device__ __forceinline__ void clear_histogram() {
    SampleShared& sh = shared_memory();
    __syncthreads();
    for (int i = threadIdx.x; i < kSampleBins; i += kThreads) {
        sh.hist[i] = 0;
        sh.number[i] = 0;
    }
    if (threadIdx.x == 0) {
        sh.found_bin = 0;
        sh.count = 0;
    }
    __syncthreads();
}

// Where the order is cut when `target` of the candidates up to `upto` is kept: the last one of them that is.  `target` is
// a number of classes (`count`), or a share of `mass` (0: of all of these); kUnsure if a border is within `slack` of it, or
// if too many candidates tie.  Ranked are at most kCountRank candidates (which leaves sh.order in order; `ranked`: it is already),
// or those of the bin in which the cut falls (2 100 for a nucleus of three: all of them sorted took 35 us).
static constexpr uint64_t kUnsure = 0;   // (no candidate has such a key)
static __device__ __noinline__ uint64_t cut_candidates(int found, bool ranked, uint64_t upto, bool count, double target, double mass,
                                                double slack) {
    SampleShared& sh = shared_memory();
    const RowWeights rw = sh.rw;
    uint64_t above = 0, before = 0, end = 0;   // masses and classes
    const bool small = found <= kCountRank;
    if (!small) {
        clear_histogram();
        for (int i = threadIdx.x; i < found; i += kThreads) {
            const uint64_t one = sh.order[i];
            if (one <= upto) count_candidate(rw, candidate_score(one));
        }
        __syncthreads();
        const CutBin c = cut_bin([&](uint64_t all) {
            if (!count) target = fmax(target * (mass != 0.0 ? mass : static_cast<double>(all)), 0.5);
            return [=](uint64_t m, uint64_t k) { return static_cast<double>(count ? k : m) < target; };
        });
        if (c.number > kRanked) return kUnsure;
        for (int i = threadIdx.x; i < found; i += kThreads) {
            const uint64_t one = sh.order[i];
            if (one <= upto && weight_bin(candidate_score(one), rw) == c.bin) sh.list[atomicAdd(&sh.count, 1u)] = one;
        }
        __syncthreads();
        rank_list(c.number);
        above = c.above;
        before = c.before;
        end = c.above + c.mass;
        found = c.number;
    } else if (!ranked) {
        rank_few(sh.order, found);
    }
    const uint64_t* s = small ? sh.order : sh.list;
    if (count) return s[static_cast<int64_t>(target) - 1 - static_cast<int64_t>(before)];
    const int per = (found + kBook - 1) / kBook, r0 = threadIdx.x < kBook ? per * threadIdx.x : found, r1 = min(found, r0 + per);
    uint64_t sum = 0, all;
    for (int r = r0; r < r1; ++r) sum += rw.whole(weight(rw, candidate_score(s[r])));
    uint64_t at = above + book_scan(sum, sh.part, all) - sum;
    if (small) target = fmax(target * (mass != 0.0 ? mass : static_cast<double>(all)), 0.5);
    const auto near = [&](uint64_t border) {
        return slack > 0.0 && border > 0 && !(fabs(static_cast<double>(border) - target) > slack * target);
    };
    bool unsure = !small && near(end);
    uint32_t kept = 0;   // a prefix of the ranks
    for (int r = r0; r < r1; ++r) {
        unsure |= near(at);
        kept += static_cast<double>(at) < target;
        at += rw.whole(weight(rw, candidate_score(s[r])));
    }
    if (__syncthreads_or(unsure)) return kUnsure;
    kept = block_total(kept, sh.part_u32);
    return s[kept - 1];
}

struct Cut {
    uint32_t key;      // 0: none
    uint64_t quota;    // classes at the key that are kept
    uint64_t mass;     // of all that is kept
};

// Where the order is cut when `target` of it is kept -- classes (`count`) or a share of the mass (of all classes, or of
// the `mass` given) -- and not more than `limit` classes.
// A function of its own, whose arguments fit registers: what it were handed in memory, every phase would wait for.
template <typename T>
static __device__ __noinline__ Cut find_cut(const T* __restrict__ x, int n, bool count, double target, uint64_t mass, uint64_t limit) {
    SampleShared& sh = shared_memory();
    const RowWeights rw = sh.rw;
    constexpr int kLen = Vec16<T>::kLen;
    clear_histogram();
    each_vector(x, n, [&](const float (&v)[kLen], int) {
        uint64_t w[kLen];
#pragma unroll
        for (int e = 0; e < kLen; ++e) w[e] = rw.whole(weight(rw, v[e]));
#pragma unroll
        for (int e = 0; e < kLen; ++e)
            if (v[e] > rw.none) {
                const int b = weight_bin(v[e], rw);
                atomicAdd(reinterpret_cast<unsigned long long*>(&sh.hist[b]), static_cast<unsigned long long>(w[e]));
                atomicAdd(&sh.number[b], 1u);
            }
    });
    __syncthreads();
    // at least half a unit: the first class is kept whatever the share is
    const CutBin c = cut_bin([&](uint64_t all) {
        if (!count) target = fmax(target * static_cast<double>(mass ? mass : all), 0.5);
        return [=](uint64_t m, uint64_t k) { return k < limit && static_cast<double>(count ? k : m) < target; };
    });
    const auto begins = [&](uint64_t m, uint64_t k) { return k < limit && static_cast<double>(count ? k : m) < target; };
    const int bin = c.bin, number = c.number;
    uint64_t above = c.above, before = c.before, sum, all;
    const auto in = [&](float v) { return weight_bin(v, rw) == bin; };
    Cut cut;
    if (number > kRanked) {   // ties: the key first, then as many of its classes as it takes
        uint64_t reached = count ? before : above;
        cut.key = find_key<T>(x, n, rw, count, in, target, reached);
        uint64_t heavier = 0, more = 0, equal = 0;   // in the bin: mass and number above the key, number at it
        each_vector<1>(x, n, [&](const float (&v)[kLen], int) {
            for (int e = 0; e < kLen; ++e) {
                const uint32_t k = score_key(v[e]);
                if (!(v[e] > rw.none) || k < cut.key || !in(v[e])) continue;
                if (k == cut.key) {
                    ++equal;
                } else {
                    ++more;
                    heavier += rw.whole(weight(rw, v[e]));
                }
            }
        });
        above += block_total(heavier, sh.part);
        more = block_total(more, sh.part);
        equal = block_total(equal, sh.part);
        const uint64_t w = rw.whole(weight(rw, key_score(cut.key)));
        double take = count ? target - static_cast<double>(before + more)
                             : (w ? ceil((target - static_cast<double>(above)) / static_cast<double>(w)) : static_cast<double>(equal));
        take = fmin(fmax(take, 1.0), fmin(static_cast<double>(equal), static_cast<double>(limit - before - more)));
        cut.quota = static_cast<uint64_t>(take);
        cut.mass = above + cut.quota * w;
        return cut;
    }
    each_vector<1>(x, n, [&](const float (&v)[kLen], int at) {
        for (int e = 0; e < kLen; ++e)
            if (v[e] > rw.none && in(v[e]))
                sh.list[atomicAdd(&sh.count, 1u)] = static_cast<uint64_t>(~score_key(v[e])) << 32 | static_cast<uint32_t>(at + e);
    });
    __syncthreads();
    rank_list(number);
    const int per = (number + kThreads - 1) / kThreads, r0 = per * threadIdx.x, r1 = min(number, r0 + per);
    sum = 0;
    for (int r = r0; r < r1; ++r) sum += rw.whole(weight(rw, candidate_score(sh.list[r])));
    uint64_t at = above + block_scan(sum, sh.part, all) - sum;
    uint64_t kept = 0, kept_mass = 0;
    for (int r = r0; r < r1; ++r) {
        const uint64_t w = rw.whole(weight(rw, candidate_score(sh.list[r])));
        if (begins(at, before + r)) {
            ++kept;
            kept_mass += w;
        }
        at += w;
    }
    kept = block_total(kept, sh.part);
    cut.mass = above + block_total(kept_mass, sh.part);
    // the key of the last kept rank, and how many of the kept ranks have it
    const int last = kept ? static_cast<int>(kept) - 1 : 0;
    cut.key = ~static_cast<uint32_t>(sh.list[last] >> 32);
    uint64_t same = 0;
    for (int r = threadIdx.x; r <= last; r += kThreads) same += ~static_cast<uint32_t>(sh.list[r] >> 32) == cut.key;
    cut.quota = block_total(same, sh.part);
    return cut;
}

// scores of a piece of a row, a multiple of what a wave loads at once
template <typename T>
static __device__ __forceinline__ int piece_length(int n) {
    constexpr int kWave = 64 * Vec16<T>::kLen;
    return ((n + kPieces - 1) / kPieces + kWave - 1) / kWave * kWave;
}

// find_cut for a share of the mass of all classes and nothing else, and the masses of the pieces with it, in one pass of f64
// weights: the bin comes from a histogram of f32 weights (in units of 2^-31 of `rough`, the f32 sum at T), the pass adds up
// what is above that bin and lists what is in it.  Key 0 -- then it is find_cut's -- if the cut is not in the bin after
// all, or if the bin holds too many.  (65 536 scores: 32 us, where find_cut takes 31 and the pieces after it 14.)
template <typename T>
static __device__ __noinline__ Cut find_nucleus(const T* __restrict__ x, int n, double share, float rough) {
    SampleShared& sh = shared_memory();
    const RowWeights rw = sh.rw;
    constexpr int kLen = Vec16<T>::kLen, kPer = kSampleBins / kThreads;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const Cut none{0, 0, 0};
    clear_histogram();
    const float unit = 0x1p31f / rough;
    const auto octaves = [&](float v) { return v == rw.top ? 0.0f : (rw.top - v) * rw.ct; };
    each_vector(x, n, [&](const float (&v)[kLen], int) {
#pragma unroll
        for (int e = 0; e < kLen; ++e)
            if (v[e] > rw.none) {
                const float y = octaves(v[e]);
                atomicAdd(&sh.number[static_cast<int>(fminf(y * kBinsPerOctave, static_cast<float>(kSampleBins - 1)))],
                          static_cast<uint32_t>(rintf(exp2_fast(-y) * unit)));   // (cut off, n of them would be short by n / 2)
            }
    });
    __syncthreads();
    uint64_t sum = 0, all;
    const int first = kPer * threadIdx.x;
    for (int i = 0; i < kPer; ++i) sum += sh.number[first + i];
    uint64_t before = block_scan(sum, sh.part, all) - sum;
    const double goal = share * static_cast<double>(all);
    int bin = -1;
    for (int i = 0; i < kPer; ++i) {
        const uint32_t m = sh.number[first + i];
        if (m && static_cast<double>(before) < goal) bin = first + i;
        before += m;
    }
    if (bin >= 0) atomicMax(&sh.found_bin, static_cast<uint32_t>(bin));
    __syncthreads();
    bin = sh.found_bin;
    const float from = static_cast<float>(bin), to = bin == kSampleBins - 1 ? INFINITY : static_cast<float>(bin + 1);
    const int piece = piece_length<T>(n);
    double whole_row = 0.0;
    for (int i = wave; i < kPieces; i += kWaves) {
        double above = 0.0;
        stream_vectors<2>(x, i * piece, min(n, (i + 1) * piece), lane, 64, [&](const float (&v)[kLen], int at) {
            double w[kLen];
#pragma unroll
            for (int e = 0; e < kLen; ++e) w[e] = weight(rw, v[e]);
#pragma unroll
            for (int e = 0; e < kLen; ++e) {
                const float y = octaves(v[e]) * kBinsPerOctave;
                const bool some = v[e] > rw.none;
                above += some && y < from ? w[e] : 0.0;
                whole_row += some ? w[e] : 0.0;
                if (some && y >= from && y < to) {
                    const uint32_t place = atomicAdd(&sh.count, 1u);
                    if (place < kRanked)
                        sh.list[place] = static_cast<uint64_t>(~score_key(v[e])) << 32 | static_cast<uint32_t>(at + e);
                }
            }
        });
        above = wave_sum(above);
        if (lane == 0) {
            sh.piece[i] = above;
            sh.tied[i] = 0;
        }
    }
    whole_row = block_total(whole_row, sh.part_f64);
    const double above = wave_sum(sh.piece[lane]), target = share * whole_row;
    const int number = sh.count;
    if (number == 0 || number > kRanked - kPieces || !(above < target || above == 0.0)) return none;
    rank_list(number);
    const int per = (number + kThreads - 1) / kThreads;
    const int r0 = min(number, per * static_cast<int>(threadIdx.x)), r1 = min(number, r0 + per);
    double mine = 0.0, listed;
    for (int r = r0; r < r1; ++r) mine += weight(rw, candidate_score(sh.list[r]));
    double at = above + block_scan(mine, sh.part_f64, listed) - mine;
    if (bin != kSampleBins - 1 && !(above + listed > target)) return none;
    uint32_t kept = 0;
    for (int r = r0; r < r1; ++r) {
        kept += (r == 0 && above == 0.0) || at < target;
        at += weight(rw, candidate_score(sh.list[r]));
    }
    // at least the first, before which `above` is below the target: with a sum put on and taken off again it may not be, and a cut
    // that keeps nothing leaves nothing to draw from
    kept = max(block_total(kept, sh.part_u32), 1u);
    // into the pieces: whole numbers, whose sum does not depend on the order
    Cut cut;
    cut.key = ~static_cast<uint32_t>(sh.list[kept - 1] >> 32);
    cut.quota = 0;
    cut.mass = 0;
    uint32_t same = 0;
    uint64_t* more = sh.bins + kRanked - kPieces;   // behind the list
    __syncthreads();
    if (threadIdx.x < kPieces) more[threadIdx.x] = 0;
    __syncthreads();
    for (int r = threadIdx.x; r < number; r += kThreads) {
        const uint64_t one = sh.list[r];
        const uint32_t i = static_cast<uint32_t>(one) / static_cast<uint32_t>(piece);
        if (~static_cast<uint32_t>(one >> 32) == cut.key) {
            atomicAdd(&sh.tied[i], 1u);
            same += r < static_cast<int>(kept);
        } else if (r < static_cast<int>(kept)) {
            atomicAdd(reinterpret_cast<unsigned long long*>(&more[i]),
                      static_cast<unsigned long long>(rw.whole(weight(rw, candidate_score(one)))));
        }
    }
    cut.quota = block_total(same, sh.part_u32);
    if (threadIdx.x < kPieces) sh.piece[threadIdx.x] += static_cast<double>(more[threadIdx.x]) / rw.scale;
    __syncthreads();
    return cut;
}

// The class for a row, to thread 0; -1: every class is masked.  logprob = (score - top) - log(soft_sum).
template <typename T>
static __device__ __forceinline__ uint32_t sample_class(const SampleArgs& a, long long row, const T* __restrict__ x,
                                                 float& top, double& soft_sum) {
    SampleShared& sh = shared_memory();
    constexpr int kLen = Vec16<T>::kLen;
    const int n = a.n_classes;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;

    const RowSettings set(a, row);
    const bool greedy = set.greedy, use_k = set.use_k, use_p = set.use_p, use_m = set.use_m;
    const int top_k = set.top_k;
    const float ct = set.ct, u = set.u;
    const double share = set.share, least = set.least;

    // 1. the row's statistics: max, sum of 2^(c (x - max)) for c = log2 e and, where top_p refers to a mass that only this
    // step sees whole, c = log2 e / T
    // (f32 distances past the largest number come out infinite.  Only at temperatures of that size do such classes weigh anything:
    // there top_p is left to find_cut, whose weights are f64; in its bins these classes are in the last one, behind all others)
    const bool f32_mass = use_p && !use_k && n > kCandidates, f32_sound = set.t < 1e30f;
    const bool rough_mass = !greedy && f32_mass && f32_sound && set.t != 1.0f;
    float soft = 0.0f, tempered = 0.0f;
    top = -INFINITY;
    const auto add = [&](const float (&raw)[kLen], int) {
        float v[kLen], most = top;
#pragma unroll
        for (int e = 0; e < kLen; ++e) v[e] = fmaxf(raw[e], -INFINITY);   // NaN is -inf
#pragma unroll
        for (int e = 0; e < kLen; ++e) most = fmaxf(most, v[e]);
        if (most == -INFINITY) return;
        if (most > top) {
            soft *= exp2_fast((top - most) * 1.44269504f);
            if (rough_mass) tempered *= exp2_fast((top - most) * ct);
            top = most;
        }
#pragma unroll
        for (int e = 0; e < kLen; ++e) soft += exp2_fast((v[e] - top) * 1.44269504f);
        if (rough_mass)
#pragma unroll
            for (int e = 0; e < kLen; ++e) tempered += exp2_fast((v[e] - top) * ct);
    };
    static_assert(kPowers <= kThreads, "a thread for each");
    const double power = kPowerTable.v[threadIdx.x & (kPowers - 1)];   // on its way with the scores
    const bool holds = n <= kDeep * kThreads * kLen;
    Vec16<T> raw[kDeep];
    if (holds) {
        load_vectors(raw, x, 0, n, threadIdx.x, kThreads);
        use_vectors(raw, 0, n, threadIdx.x, kThreads, add);
    } else {
        each_vector<kFlight>(x, n, add);
    }
    const uint32_t share_key = score_key(top);
    const auto join = [&](float most) {
        soft *= most > top ? exp2_fast((top - most) * 1.44269504f) : 1.0f;
        tempered *= most > top ? exp2_fast((top - most) * ct) : 1.0f;
        top = most;
    };
    join(wave_max(top));
    soft = wave_sum(soft);
    if (rough_mass) tempered = wave_sum(tempered);
    if (lane == 0) {
        sh.stat[0][wave] = top;
        sh.stat[1][wave] = soft;
        sh.stat[2][wave] = tempered;
    }
    if (threadIdx.x < 2 * kBook) sh.kth[threadIdx.x / kBook][threadIdx.x % kBook] = 0;
    for (int i = threadIdx.x; i < kPowers; i += kThreads) sh.power[i] = power;
    if (threadIdx.x == 0) {
        sh.count = 0;
        sh.choice = 0xffffffffu;
    }
    __syncthreads();
    {   // a lane for each wave, in every row of 16
        static_assert(kWaves <= 16, "a row of lanes");
        const int from = lane % 16;
        const auto add = [](float a, float b) { return a + b; };
        top = sh.stat[0][min(from, kWaves - 1)];
        soft = from < kWaves ? sh.stat[1][from] : 0.0f;
        tempered = from < kWaves ? sh.stat[2][from] : 0.0f;
        join(row_total(top, -INFINITY, [](float a, float b) { return fmaxf(a, b); }));
        soft = row_total(soft, 0.0f, add);
        if (rough_mass) tempered = row_total(tempered, 0.0f, add);
    }
    if (top == -INFINITY) return 0xffffffffu;
    soft_sum = soft;
    double rough = rough_mass ? tempered : soft;
    if (top == INFINITY) {   // the classes at +inf share everything: weight 1 each
        uint64_t infs = 0;
        each_vector(x, n, [&](const float (&v)[kLen], int) {
#pragma unroll
            for (int e = 0; e < kLen; ++e) infs += v[e] == top;
        });
        soft_sum = rough = static_cast<double>(block_total(infs, sh.part));
    }
    if (greedy) {
        uint32_t first = 0xffffffffu;
        each_vector(x, n, [&](const float (&v)[kLen], int at) {
#pragma unroll
            for (int e = kLen - 1; e >= 0; --e)
                if (v[e] == top) first = min(first, static_cast<uint32_t>(at + e));
        });
        if (first != 0xffffffffu) atomicMin(&sh.choice, first);
        __syncthreads();
        return sh.choice;
    }
    const RowWeights rw = set.weights(top, a.weight_bits);

    // 2. a key that every kept class reaches
    uint32_t floor_key = 0;
    bool try_candidates = use_k || use_p || use_m;
    if (n > (use_p && !use_k ? kCandidates : kThreads)) {   // (with all of them, the mass that top_p refers to is exact)
        if (use_k) {
            if (top_k <= kThreads) floor_key = kth_of_threads(share_key, top_k);
            try_candidates = top_k <= kThreads || n <= kCandidates;   // also if few shares hold anything at all
        } else if (use_p && !use_m) {
            floor_key = kth_of_threads(share_key, kNucleusGuess);
            try_candidates = floor_key != 0;
        }
        if (use_m && !(use_k && use_p)) {   // top_p of the first top_k needs all of these
            const float far = set.t * 0.69314718f * __builtin_amdgcn_logf(static_cast<float>(least));   // (log2)
            const float bound = top + far - 1e-5f * (fabsf(top) - far);
            floor_key = max(floor_key, score_key(bound));
            try_candidates = true;
        }
    }
    if (try_candidates && (f32_sound || !f32_mass)) {
        // the least score that takes part: what is not above rw.none, and NaN, does not
        const float floor = fmaxf(floor_key ? key_score(floor_key) : -INFINITY, rw.none > 0.0f ? INFINITY : -0x1.fffffep127f);
        const auto collect = [&](const float (&v)[kLen], int at) {
            // per element one compare, whose result for the wave is a scalar: places are counted there, and only an element
            // that some lane keeps costs more (per lane, with a prefix sum of the lanes' counts, 1 000 of 131 072: 20 us)
            uint64_t hits[kLen];
            uint32_t all = 0;
#pragma unroll
            for (int e = 0; e < kLen; ++e) {
                hits[e] = __ballot(v[e] >= floor);
                all += __popcll(hits[e]);
            }
            if (all == 0) return;
            uint32_t to = 0;
            if (lane == 0) to = atomicAdd(&sh.count, all);
            to = __builtin_amdgcn_readfirstlane(to);
            if (to + all > kCandidates) return;   // (all of them are given up)
#pragma unroll
            for (int e = 0; e < kLen; ++e)
                if (hits[e]) {
                    const uint32_t before = __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(hits[e] >> 32),
                                                                      __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(hits[e]), 0));
                    if (v[e] >= floor)
                        sh.order[to + before] = static_cast<uint64_t>(~score_key(v[e])) << 32 | static_cast<uint32_t>(at + e);
                    to += __popcll(hits[e]);
                }
        };
        if (holds) use_vectors(raw, 0, n, threadIdx.x, kThreads, collect);
        else each_vector<kFlight>(x, n, collect);
        __syncthreads();
        const int found = sh.count;
        // 3. the mass that top_p refers to is exact unless the candidates are not all there is
        const bool exact = floor_key == 0 || use_k;
        if (found <= 64 && (exact || !use_p)) {
            if (wave != 0) return 0;
            return draw_in_wave(found, rw, least, use_k ? top_k : found, use_p ? share : 2.0, u);
        }
        if (found <= kCandidates) {
            if (threadIdx.x == 0) sh.rw = rw;
            __syncthreads();
            const auto mass_of = [&](uint64_t one) {   // nothing if it is too light
                const double w = weight(rw, candidate_score(one));
                return w >= least ? rw.whole(w) : 0;
            };
            const double slack = exact ? 0.0 : (n / kThreads + 64) * 0x1p-23;
            bool cuts = (use_k && found > top_k) || use_p, fits = true;
            uint64_t total = 0, upto = ~0ull;   // the mass of all that is kept, the last in order of it
            uint32_t kept = found;
            if (!cuts || (use_p && !exact)) {
                for (int i = threadIdx.x; i < found; i += kThreads) total += mass_of(sh.order[i]);
                total = block_total(total, sh.part);
                if (use_p) {
                    const double goal = share * rough * rw.scale;
                    if (use_m) cuts = !(static_cast<double>(total) < goal * (1.0 - slack));   // below it top_p takes none away
                    else fits = static_cast<double>(total) > goal * (1.0 + slack);            // a guess has to reach it
                }
            }
            if (cuts && fits) {
                int ranks = found;
                bool ranked = false;
                if (use_k && found > top_k) {
                    upto = cut_candidates(found, false, upto, true, top_k, 0.0, 0.0);
                    ranked = found <= kCountRank;
                    if (ranked) ranks = top_k;
                }
                if (use_p && upto != kUnsure) {
                    const uint64_t first = upto;
                    upto = cut_candidates(ranks, ranked, first, false, share, exact ? 0.0 : rough * rw.scale, slack);
                    if (upto == kUnsure && !exact) {   // the mass of the whole row, exactly
                        uint64_t all = 0;
                        each_vector(x, n, [&](const float (&v)[kLen], int) {
                            uint64_t w[kLen];
#pragma unroll
                            for (int e = 0; e < kLen; ++e) w[e] = rw.whole(weight(rw, v[e]));
#pragma unroll
                            for (int e = 0; e < kLen; ++e) all += v[e] > rw.none ? w[e] : 0;
                        });
                        all = block_total(all, sh.part);
                        upto = cut_candidates(ranks, ranked, first, false, share, static_cast<double>(all), 0.0);
                    }
                }
                fits = upto != kUnsure;
            }
            if (fits && cuts) {   // how much that is, and, of few, which
                __syncthreads();
                if (threadIdx.x == 0) sh.count = 0;
                __syncthreads();
                total = 0;
                for (int i = threadIdx.x; i - lane < found; i += kThreads) {
                    const uint64_t one = i < found ? sh.order[i] : ~0ull, mass = one <= upto && i < found ? mass_of(one) : 0;
                    total += mass;
                    const uint64_t has = __ballot(mass > 0);
                    if (!has) continue;
                    uint32_t to = 0;
                    if (lane == 0) to = atomicAdd(&sh.count, static_cast<uint32_t>(__popcll(has)));
                    to = __builtin_amdgcn_readfirstlane(to) + __popcll(has & ((1ull << lane) - 1));
                    if (mass > 0 && to < 64) sh.list[to] = one;
                }
                total = block_total(total, sh.part);
                kept = sh.count;
            }
            if (fits) {
                const uint64_t goal = min(static_cast<uint64_t>(static_cast<double>(u) * static_cast<double>(total)), total - 1);
                const auto kept_mass = [&](uint64_t one) { return one <= upto ? mass_of(one) : 0; };
                if (kept > 64) return draw_candidate(found, goal, n, kept_mass);
                if (wave != 0) return 0;
                const uint64_t one = lane < static_cast<int>(kept) ? cuts ? sh.list[lane] : sh.order[lane] : ~0ull;
                return draw_few(static_cast<uint32_t>(one), mass_of(one), kept, goal);
            }
        }
    }

    // 4.
    Cut cut{0, 0, 0};
    if (threadIdx.x == 0) sh.rw = rw;
    __syncthreads();
    if (use_k) cut = find_cut<T>(x, n, true, top_k, 0, n);
    bool pieces = false;   // known
    if (use_p && !use_k && !use_m && f32_sound) {
        cut = find_nucleus<T>(x, n, share, static_cast<float>(rough));
        pieces = cut.key != 0;
    }
    if (use_p && !pieces) cut = find_cut<T>(x, n, false, share, cut.mass, use_k ? top_k : n);
    const float cut_score = cut.key ? key_score(cut.key) : rw.none;
    const double cut_weight = cut.key ? weight(rw, cut_score) : 0.0;
    // the scores above the cut and not lighter than `least` -- min_p's, or nothing that any sum notices, which a draw with u = 0
    // would take all the same -- as one bound: comparing the weights would be an f64 instruction each
    float from = score_above(cut_score);
    const double far = use_m ? log(least) : -85.19564844077969;   // (log 1e-37: RowSettings' least without min_p)
    const double bound = fmax(rw.top_wide + static_cast<double>(set.t) * far, -0x1.fffffep127);
    float light = static_cast<float>(bound);
    if (static_cast<double>(light) < bound) light = score_above(light);
    if (light > from) from = light;   // (NaN, which nothing reaches, is what is above +inf)
    const bool cut_counts = cut.key != 0 && cut_score >= light;
    const auto over = [&](float v) {   // the weight of a class that is kept whatever its index, 0 of any other
        const double w = weight(rw, v);
        return v >= from ? w : 0.0;
    };
    __syncthreads();
    // the mass of each piece, and how many classes at the key it holds
    const int piece = piece_length<T>(n);
    for (int i = wave; i < kPieces && !pieces; i += kWaves) {
        const int stop = min(n, (i + 1) * piece);
        double m = 0.0;
        uint32_t ties = 0;
        stream_vectors<2>(x, i * piece, stop, lane, 64, [&](const float (&v)[kLen], int) {
            if (cut.key || use_m) {   // most vectors hold nothing above a cut
                const float least_score = cut_counts ? cut_score : from;
                float most = v[0];
#pragma unroll
                for (int e = 1; e < kLen; ++e) most = fmaxf(most, v[e]);
                if (!__any(most >= least_score)) return;
            }
            double w[kLen];
#pragma unroll
            for (int e = 0; e < kLen; ++e) w[e] = over(v[e]);
#pragma unroll
            for (int e = 0; e < kLen; ++e) {
                m += w[e];
                ties += cut_counts && v[e] == cut_score;
            }
        });
        m = wave_sum(m);
        ties = wave_sum(ties);
        if (lane == 0) {
            sh.piece[i] = m;
            sh.tied[i] = ties;
        }
    }
    __syncthreads();
    // the first piece whose cumulative mass exceeds the goal; past all of them (u >= 1, or rounding): the last with any.
    // Lane i of every wave has piece i
    static_assert(kPieces == 64, "a piece for each lane");
    const uint64_t piece_ties = sh.tied[lane], tied = wave_scan_sum(piece_ties) - piece_ties;   // before the piece
    const uint64_t left = tied < cut.quota ? cut.quota - tied : 0;
    const double piece_mass = sh.piece[lane] + static_cast<double>(piece_ties < left ? piece_ties : left) * cut_weight;
    const double upto = wave_scan_sum(piece_mass);
    const double goal = static_cast<double>(u) * last_lane(upto);
    const uint64_t some = __ballot(piece_mass > 0.0), past = __ballot(piece_mass > 0.0 && upto > goal);
    const int chosen = past ? __ffsll(static_cast<unsigned long long>(past)) - 1 : 63 - __clzll(static_cast<long long>(some));
    const double chosen_before = __shfl(upto - piece_mass, chosen);
    const uint64_t chosen_tied = __shfl(static_cast<unsigned long long>(tied), chosen);
    // the same with a share of the piece for each thread
    const int stop = min(n, (chosen + 1) * piece), per = (piece + kThreads - 1) / kThreads;
    const int begin = min(stop, chosen * piece + static_cast<int>(threadIdx.x) * per), end = min(stop, begin + per);
    float v[kShare];   // the first scores of the share: all of it up to 131 072 classes
#pragma unroll
    for (int i = 0; i < kShare; ++i) v[i] = begin + i < end ? static_cast<float>(x[begin + i]) : -INFINITY;
    const auto each = [&](auto f) {   // f(class, score) for the share
#pragma unroll
        for (int i = 0; i < kShare; ++i)
            if (begin + i < end) f(begin + i, v[i]);
        for (int j = begin + kShare; j < end; ++j) f(j, static_cast<float>(x[j]));
    };
    uint64_t rank0 = chosen_tied;
    if (cut_counts) {
        uint64_t ties = 0, all;
        each([&](int, float s) { ties += s == cut_score; });
        rank0 += block_scan(ties, sh.part, all) - ties;
    }
    uint64_t rank = rank0;
    const auto mine = [&](float s) { return cut_counts && s == cut_score ? (rank++ < cut.quota ? cut_weight : 0.0) : over(s); };
    double m = 0.0;
    each([&](int, float s) { m += mine(s); });
    double all_mass, sum = chosen_before + block_scan(m, sh.part_f64, all_mass) - m;
    // sums of a share in two orders may differ in the last bit: then its last class
    if (threadIdx.x == 0) {
        sh.choice = 0xffffffffu;
        sh.count = 0;
    }
    __syncthreads();
    const bool reaches = m > 0.0 && sum + m > goal;
    int first = -1, last = -1;
    if (m > 0.0) {
        rank = rank0;
        each([&](int j, float s) {
            const double w = mine(s);
            sum += w;
            if (w > 0.0) {
                last = j;
                if (first < 0 && sum > goal) first = j;
            }
        });
        if (reaches) atomicMin(&sh.choice, static_cast<uint32_t>(first >= 0 ? first : last));
        else atomicMax(&sh.count, static_cast<uint32_t>(last));
    }
    __syncthreads();
    return sh.choice != 0xffffffffu ? sh.choice : sh.count;   // past all: the last kept class
}
};

// the answer of a row, by one thread
template <typename T>
__device__ __forceinline__ void store_sample(const SampleArgs& a, long long row, const T* __restrict__ x, uint32_t cls, float top,
                                             double soft_sum) {
    if (cls == 0xffffffffu) {
        a.token[row] = -1;
        a.logprob[row] = -INFINITY;
        return;
    }
    const float v = static_cast<float>(x[cls]);
    a.token[row] = cls;
    a.logprob[row] = static_cast<float>((v == top ? 0.0 : static_cast<double>(v) - static_cast<double>(top)) - log(soft_sum));
}

template <typename T, int kThreads>
__global__ __launch_bounds__(kThreads, 4) void k_sample_row(SampleArgs a) {
    const long long row = blockIdx.x;
    const T* x = static_cast<const T*>(a.logits) + row * a.row_stride;
    float top;
    double soft_sum = 1.0;
    const uint32_t cls = RowSampler<kThreads>::sample_class(a, row, x, top, soft_sum);
    if (threadIdx.x == 0) store_sample(a, row, x, cls, top, soft_sum);
}

// Rows of at most 64 classes: a wave for each, a lane for each class, everything from registers.
constexpr int kSmallThreads = 256;
template <typename T>
__global__ __launch_bounds__(kSmallThreads) void k_sample_small(SampleArgs a) {
    const long long row = static_cast<long long>(blockIdx.x) * (kSmallThreads / 64) + (threadIdx.x >> 6);
    if (row >= a.n_rows) return;
    const int lane = threadIdx.x & 63, n = a.n_classes;
    const T* x = static_cast<const T*>(a.logits) + row * a.row_stride;
    const RowSettings set(a, row);
    const float v = lane < n ? fmaxf(static_cast<float>(x[lane]), -INFINITY) : -INFINITY;   // NaN is -inf
    const float top = wave_max(v);
    const double soft_sum = wave_sum(v == top ? 1.0f : exp2_fast((v - top) * 1.44269504f));
    uint32_t cls = 0xffffffffu;
    if (top > -INFINITY) {
        if (set.greedy) {
            cls = __ffsll(static_cast<unsigned long long>(__ballot(v == top))) - 1;
        } else {
            const RowWeights rw = set.weights(top, a.weight_bits);
            const double w = v > rw.none ? rw.real(v, [](int j) { return kPowerTable.v[j]; }) : 0.0;
            const uint64_t mass = rw.whole(w);
            bool kept = v > rw.none && w >= set.least;
            if (set.use_k || set.use_p) {
                const uint64_t mine = static_cast<uint64_t>(~score_key(v)) << 32 | lane;
                const uint32_t key = ~score_key(v), low = static_cast<uint32_t>(mass), high = static_cast<uint32_t>(mass >> 32);
                int rank = 0;
                for (int i = 0; i < n; ++i)
                    rank += (static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(key, i))) << 32 | i) < mine;
                const bool first = !set.use_k || rank < set.top_k;
                kept = kept && first;
                if (set.use_p) {
                    uint64_t before = 0, all = 0;
                    for (int i = 0; i < n; ++i) {
                        const uint64_t other = static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(high, i))) << 32 |
                                               static_cast<uint32_t>(__builtin_amdgcn_readlane(low, i));
                        const int place = __builtin_amdgcn_readlane(rank, i);
                        if (place < rank) before += other;
                        if (!set.use_k || place < set.top_k) all += other;
                    }
                    kept = kept && (rank == 0 || static_cast<double>(before) < set.share * static_cast<double>(all));
                }
            }
            const uint64_t upto = wave_scan_sum(kept ? mass : 0), total = last_lane(upto);
            const uint64_t goal = min(static_cast<uint64_t>(static_cast<double>(set.u) * static_cast<double>(total)), total - 1);
            cls = __ffsll(static_cast<unsigned long long>(__ballot(upto > goal))) - 1;
        }
    }
    if (lane == 0) store_sample(a, row, x, cls, top, soft_sum);
}

}  // namespace serhip
