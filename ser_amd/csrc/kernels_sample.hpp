// Drawing a class from scores: temperature, top-k, top-p, min-p, from one given uniform number per row.
//
//   order    the classes by (score descending, index ascending); NaN and -inf scores take no part
//   weight   w_j = exp((x_j - max x) / T) in f64: a draw is next to the border between two classes as often as not, and
//            f32 sums would move the borders of a flat row by as much as a class
//   kept     the first top_k of the order, of these the shortest prefix whose mass reaches top_p of theirs, of these
//            the weights >= min_p
//   token    the first kept class whose cumulative kept weight, in index order, exceeds u * (kept mass)
//   logprob  log softmax(x)[token], untempered and uncut
//
// k_sample_row, one workgroup of 1 024 per row: reading and f64 sums want 16 waves (256 threads read a row of 50 001 in
// 5.8 us, 1 024 in 2.3), but an instruction that all 16 execute takes 16 cycles, so lists of candidates are left to the
// first kBook threads while the others wait (scans and reductions of one such row: 16 us by all waves, 9 by four).
//   1. one read of the row: its largest score, softmax's sum, the sum at T (f32, online), the largest score of each of
//      1 024 shares
//   2. a score below which nothing can be kept -- from top_k and the shares, from min_p, or a guess that fits most nuclei
//      -- and a second read (from cache) that collects what is not below it
//   3. at most kCandidates classes: ranked if need be, cut and drawn from in LDS.  Everything is exact there but the mass
//      that top_p refers to when neither top_k nor the row's size bounds it; that one is the f32 sum, and a border that
//      falls into its error sends the row to 4
//   4. everything else: no cut at all (the draw alone), or a histogram of the row over the logarithm of the weight, the
//      bin in which the cut falls, and that bin's classes ranked as in 3 -- or, where one bin holds too many (ties), a
//      radix search of their keys.  The cut is then (key, quota): every key above `key`, and the first `quota` classes,
//      by index, whose key equals it.  The draw adds the kept weights of kPieces pieces of the row, then of a share of the
//      one that holds the answer for each thread.
// Masses that candidates and atomics add up are whole numbers of 2^-bits (bits <= 45): the order in which they arrive
// changes nothing.  The draw of step 4 adds f64 in a fixed order.
#pragma once

#include "class_common.hpp"

namespace serhip {

constexpr int kSampleThreads = 1024;
constexpr int kSampleWaves = kSampleThreads / 64;
constexpr int kBook = 256;
constexpr int kDeep = 8;            // vectors that a thread keeps in registers: a row of 65 536 16-bit scores
constexpr int kFlight = 4;          // vectors in flight of a longer row
constexpr int kSampleBins = 2048;
constexpr int kPieces = 64;         // one for each lane of a wave
constexpr int kShare = 2;           // scores of a piece that a thread keeps in registers
constexpr float kBinsPerOctave = 64.0f;   // of the weight; the last bin takes all that is below 2^-32
constexpr int kCandidates = 4096;
constexpr int kCountRank = 512;     // up to here a rank is counted (n reads each), above it is sorted
constexpr int kNucleusGuess = 900;  // of the 1 024 shares (of a thread each): some 2 200 candidates where scores come in no order

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

// An unsigned number that orders like the score: 0 for -inf and NaN, -0 and +0 alike.
__device__ __forceinline__ uint32_t score_key(float x) {
    if (!(x > -INFINITY)) return 0;
    const uint32_t u = __float_as_uint(x + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key_score(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

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

// inclusive prefix sum over the workgroup, in thread order; `total` too
template <typename V>
__device__ __forceinline__ V block_scan(V x, V* s_part, V& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    x = wave_scan_sum(x);
    __syncthreads();
    if (lane == 63) s_part[wave] = x;
    __syncthreads();
    V before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < kSampleWaves; ++w) {
        if (w < wave) before += s_part[w];
        total += s_part[w];
    }
    return x + before;
}
template <typename V>
__device__ __forceinline__ V block_total(V x, V* s_part) {
    x = wave_sum(x);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s_part[threadIdx.x >> 6] = x;
    __syncthreads();
    V total = 0;
#pragma unroll
    for (int w = 0; w < kSampleWaves; ++w) total += s_part[w];
    return total;
}

// block_scan over the first kBook threads; the others add nothing and get the total only
template <typename V>
__device__ __forceinline__ V book_scan(V x, V* s_part, V& total) {
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
template <int kCount = 2, typename T, typename F>
__device__ __forceinline__ void each_vector(const T* __restrict__ x, int n, F f) {
    stream_vectors<kCount>(x, 0, n, threadIdx.x, kSampleThreads, f);
}

struct RowWeights {
    float top;        // the largest score
    float low;        // a score whose weight is 0
    float none;       // scores up to here have no weight: -inf, or every number where the largest score is +inf
    float ct;         // log2 e / T
    double top_wide;  // `top`; the largest number for +inf
    double ct_wide;
    double scale;     // 2^weight_bits
    // exp((x - top) / T) = 2^n 2^f, |f| < 0.501: n from f32, f from f64 -- 14 f64 instructions, which take twice the time
    // of others.  2^f = 1 + f g(f) with g the polynomial of degree 8 through the nine Chebyshev points of (2^f - 1) / f:
    // 2^-44 of the result.  Exactly 1 at x = top.  Without branches, so that a vector's weights are worked out together;
    // for x > none only.
    __device__ __forceinline__ double real(float x) const {
        const float v = fminf(fmaxf(x, low), 0x1.fffffep127f);
        const float n = fmaxf(rintf((v - fminf(top, 0x1.fffffep127f)) * ct), -1100.0f);
        const double f = fma(static_cast<double>(v) - top_wide, ct_wide, -static_cast<double>(n));
        double g = 1.0203221420017349e-07;
        g = fma(g, f, 1.3255384208086413e-06);
        g = fma(g, f, 1.5252686469189063e-05);
        g = fma(g, f, 0.0001540345525379509);
        g = fma(g, f, 0.001333355817943667);
        g = fma(g, f, 0.009618129160027376);
        g = fma(g, f, 0.05550410866475944);
        g = fma(g, f, 0.24022650695811423);
        g = fma(g, f, 0.6931471805599453);
        return ldexp(fma(g, f, 1.0), static_cast<int>(n));
    }
    // round(w 2^bits), read off the mantissa of a sum with 2^52
    __device__ __forceinline__ uint64_t whole(double w) const {
        return static_cast<uint64_t>(__double_as_longlong(fma(w, scale, 0x1p52))) & ((1ull << 52) - 1);
    }
};

// a row's settings; what is out of range, or NaN, is off
struct RowSettings {
    int top_k;
    float t, ct;             // temperature and log2 e / T; a temperature below 1e-30 does as 1e-30
    float u;
    double share, least;     // top_p, min_p
    bool greedy, use_k, use_p, use_m;
    __device__ __forceinline__ RowSettings(const SampleArgs& a, long long row) {
        const float temperature = a.temperature_rows ? a.temperature_rows[row] : a.temperature;
        const float top_p = a.top_p_rows ? a.top_p_rows[row] : a.top_p;
        const float min_p = a.min_p_rows ? a.min_p_rows[row] : a.min_p;
        top_k = a.top_k_rows ? a.top_k_rows[row] : a.top_k;
        u = fmaxf(a.uniform[row], 0.0f);
        greedy = !(temperature > 0.0f && temperature < INFINITY);
        use_k = top_k >= 1 && top_k < a.n_classes;
        use_p = top_p < 1.0f;
        use_m = min_p > 0.0f;
        t = fmaxf(temperature, 1e-30f);
        ct = 1.44269504f / t;
        share = fmaxf(top_p, 0.0f);
        least = use_m ? fminf(min_p, 1.0f) : 0.0f;
    }
    __device__ __forceinline__ RowWeights weights(float top, int bits) const {
        const float most = 0x1.fffffep127f;
        return {top, top - 1100.0f / ct, top == INFINITY ? most : -INFINITY, ct, static_cast<double>(fminf(top, most)),
                1.4426950408889634 / static_cast<double>(t), static_cast<double>(1ull << bits)};
    }
};

struct SampleShared {
    union {
        uint64_t order[kCandidates];     // candidates: ~key and class, which sort by rank
        uint64_t bins[kSampleBins];      // of a radix search
    };
    union {
        struct {
            uint64_t mass[kCandidates];  // candidates' weights, in whole numbers, ...
            uint32_t cls[kCandidates];   // ... and classes
        };
        struct {
            uint64_t hist[kSampleBins];  // masses
            uint32_t number[kSampleBins];
        };
        struct {
            double piece[kPieces];
            uint32_t tied[kPieces];
        };
    };
    union {
        uint64_t part[kSampleWaves];
        double part_f64[kSampleWaves];
        uint32_t part_u32[kSampleWaves];
    };
    float stat[3][kSampleWaves];
    uint32_t kth[2][kBook];     // cleared before the first barrier
    RowWeights rw;              // for find_cut
    uint64_t found_above, found_before, found_number;
    uint32_t found_bin;
    uint32_t count;
    uint32_t choice;
};

// The workgroup's shared memory, by name wherever it is used: through a reference, a function that is not inlined would
// reach it with flat instructions (ranking 51 candidates: 4.4 us instead of 1.4).
__device__ __forceinline__ SampleShared& shared_memory() {
    __shared__ SampleShared sh;
    return sh;
}

// ascending, n <= kCandidates
__device__ __noinline__ void sort_order(int n) {
    uint64_t* s = shared_memory().order;
    int size = 1;
    while (size < n) size <<= 1;
    for (int i = n + threadIdx.x; i < size; i += kSampleThreads) s[i] = ~0ull;
    for (int k = 2; k <= size; k <<= 1)
        for (int j = k >> 1; j; j >>= 1) {
            __syncthreads();
            for (int i = threadIdx.x; i < size / 2; i += kSampleThreads) {
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

// The lower edge of the 16-bit bin that holds the k-th largest of one key per thread: at least k keys are not below it.
// 0 if fewer than k keys are above 0.
__device__ inline uint32_t kth_of_threads(uint32_t key, uint32_t k) {
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
__device__ __forceinline__ uint32_t find_key(const T* __restrict__ x, int n, const RowWeights& rw, bool count, In in, double target,
                                          uint64_t& above) {
    SampleShared& sh = shared_memory();
    using D = KeyDigits<T>;
    constexpr int kLen = Vec16<T>::kLen, kPer = kSampleBins / kSampleThreads;
    uint32_t prefix = 0;   // the digits found so far, in place
    for (int level = 0; level < D::kLevels; ++level) {
        const int shift = D::kShift[level];
        const int width = (level == 0 ? 32 : D::kShift[level - 1]) - shift;
        const uint32_t high = level == 0 ? 0 : ~0u << D::kShift[level - 1];
        __syncthreads();
        for (int b = threadIdx.x; b < kSampleBins; b += kSampleThreads) sh.bins[b] = 0;
        if (threadIdx.x == 0) sh.found_bin = 0;
        __syncthreads();
        each_vector<1>(x, n, [&](const float (&v)[kLen], int) {
            for (int e = 0; e < kLen; ++e) {
                const uint32_t k = score_key(v[e]);
                if (v[e] > rw.none && (k & high) == prefix && in(v[e]))
                    atomicAdd(reinterpret_cast<unsigned long long*>(&sh.bins[(k >> shift) & ((1u << width) - 1)]),
                              static_cast<unsigned long long>(count ? 1 : rw.whole(rw.real(v[e]))));
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

// sh.order[0..found) -> masses and classes in rank order; how many of them weigh at least `least`
__device__ __forceinline__ int rank_candidates(int found, const RowWeights& rw, double least) {
    SampleShared& sh = shared_memory();
    uint32_t heavy = 0;
    const auto put = [&](int rank, uint64_t one) {
        const double w = rw.real(key_score(~static_cast<uint32_t>(one >> 32)));
        heavy += w >= least;
        sh.cls[rank] = static_cast<uint32_t>(one);
        sh.mass[rank] = rw.whole(w);
    };
    if (found <= kCountRank) {
        for (int i = threadIdx.x; i < found && threadIdx.x < kBook; i += kBook) {
            const uint64_t one = sh.order[i];
            int rank = 0;
#pragma unroll 8
            for (int j = 0; j < found; ++j) rank += sh.order[j] < one;
            put(rank, one);
        }
    } else {
        sort_order(found);
        for (int i = threadIdx.x; i < found; i += kSampleThreads) put(i, sh.order[i]);
    }
    return static_cast<int>(block_total(heavy, sh.part_u32));
}

// A wave's draw: lane i has a class and a mass (0: not kept), i < n.  The class at which the mass in index order first
// exceeds `goal`, which is below their sum.  `place` = how many of the classes are lower.
__device__ __forceinline__ uint32_t draw_of_lanes(uint32_t cls, uint64_t mass, int place, int n, uint64_t goal) {
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

// The class, of the `found` in sh.cls / sh.mass, at which the mass in index order first exceeds `goal` (which is below
// their sum): returned to the first wave.
__device__ __forceinline__ uint32_t draw_candidate(int found, uint64_t goal, int n) {
    SampleShared& sh = shared_memory();
    if (found <= 64) {
        const int lane = threadIdx.x & 63;
        if (threadIdx.x >= 64) return 0;
        const uint32_t cls = lane < found ? sh.cls[lane] : 0xffffffffu;
        const uint64_t mass = lane < found ? sh.mass[lane] : 0;
        int place = 0;
        for (int j = 0; j < found; ++j) place += static_cast<uint32_t>(__builtin_amdgcn_readlane(cls, j)) < cls;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        return draw_of_lanes(cls, mass, place, found, goal);
    }
    constexpr int kBits = 11, kPer = (1 << kBits) / kBook;
    static_assert(1 << kBits <= kSampleBins, "room for the bins");
    uint32_t prefix = 0;
    uint64_t below = 0;
    int shift = 0;
    while (static_cast<int64_t>(1) << (shift + kBits) < n) shift += kBits;
    for (; shift >= 0; shift -= kBits) {
        __syncthreads();
        for (int b = threadIdx.x; b < 1 << kBits; b += kSampleThreads) sh.bins[b] = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < found; i += kSampleThreads) {
            const uint32_t c = sh.cls[i];
            if (static_cast<uint64_t>(c) >> (shift + kBits) == static_cast<uint64_t>(prefix) >> (shift + kBits))
                atomicAdd(reinterpret_cast<unsigned long long*>(&sh.bins[(c >> shift) & ((1 << kBits) - 1)]),
                          static_cast<unsigned long long>(sh.mass[i]));
        }
        __syncthreads();
        uint64_t sum = 0, all;
        if (threadIdx.x < kBook)
            for (int i = 0; i < kPer; ++i) sum += sh.bins[threadIdx.x * kPer + i];
        const uint64_t upto = below + book_scan(sum, sh.part, all);
        if (threadIdx.x < kBook && upto > goal && upto - sum <= goal) {   // one thread
            uint64_t at = upto - sum;
            int b = threadIdx.x * kPer;
            while (at + sh.bins[b] <= goal) at += sh.bins[b++];
            sh.found_bin = b;
            sh.found_above = at;
        }
        __syncthreads();
        prefix |= sh.found_bin << shift;
        below = sh.found_above;
    }
    return prefix;
}

// Step 3 for at most 64 candidates, by one wave, with the candidates in the lanes: other lanes' values come from
// v_readlane (four instructions a candidate), not from LDS, whose latency a wave alone cannot hide (51 candidates:
// 11 500 cycles from LDS).  share > 1: no top_p.
__device__ __forceinline__ uint32_t draw_in_wave(int found, const RowWeights& rw, double least, int limit, double share, float u) {
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
    const double w = rw.real(key_score(~key));
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
__device__ __forceinline__ int weight_bin(float v, const RowWeights& rw) {
    return v == rw.top ? 0 : static_cast<int>(fminf((rw.top - v) * (rw.ct * kBinsPerOctave), static_cast<float>(kSampleBins - 1)));
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
__device__ __noinline__ Cut find_cut(const T* __restrict__ x, int n, bool count, double target, uint64_t mass, uint64_t limit) {
    SampleShared& sh = shared_memory();
    const RowWeights rw = sh.rw;
    constexpr int kLen = Vec16<T>::kLen, kPer = kSampleBins / kSampleThreads;
    __syncthreads();
    for (int i = threadIdx.x; i < kSampleBins; i += kSampleThreads) {
        sh.hist[i] = 0;
        sh.number[i] = 0;
    }
    if (threadIdx.x == 0) {
        sh.found_bin = 0;
        sh.count = 0;
    }
    __syncthreads();
    each_vector(x, n, [&](const float (&v)[kLen], int) {
        uint64_t w[kLen];
#pragma unroll
        for (int e = 0; e < kLen; ++e) w[e] = rw.whole(rw.real(v[e]));
#pragma unroll
        for (int e = 0; e < kLen; ++e)
            if (v[e] > rw.none) {
                const int b = weight_bin(v[e], rw);
                atomicAdd(reinterpret_cast<unsigned long long*>(&sh.hist[b]), static_cast<unsigned long long>(w[e]));
                atomicAdd(&sh.number[b], 1u);
            }
    });
    __syncthreads();
    // the last bin with anything in it that begins below the target and the limit (the first one always does)
    uint64_t sum = 0, classes = 0, all, all_classes;
    const int first = kPer * threadIdx.x;
    for (int i = 0; i < kPer; ++i) {
        sum += sh.hist[first + i];
        classes += sh.number[first + i];
    }
    uint64_t above = block_scan(sum, sh.part, all) - sum;
    uint64_t before = block_scan(classes, sh.part, all_classes) - classes;
    // at least half a unit: the first class is kept whatever the share is
    if (!count) target = fmax(target * static_cast<double>(mass ? mass : all), 0.5);
    const auto begins = [&](uint64_t m, uint64_t c) { return c < limit && static_cast<double>(count ? c : m) < target; };
    uint64_t my_above = 0, my_before = 0, my_number = 0;
    int bin = -1;
    for (int i = 0; i < kPer; ++i) {
        const uint64_t c = sh.number[first + i];
        if (c && begins(above, before)) {
            bin = first + i;
            my_above = above;
            my_before = before;
            my_number = c;
        }
        above += sh.hist[first + i];
        before += c;
    }
    if (bin >= 0) atomicMax(&sh.found_bin, static_cast<uint32_t>(bin));
    __syncthreads();
    if (bin == static_cast<int>(sh.found_bin)) {
        sh.found_above = my_above;
        sh.found_before = my_before;
        sh.found_number = my_number;
    }
    __syncthreads();
    bin = sh.found_bin;
    above = sh.found_above;
    before = sh.found_before;
    const int number = static_cast<int>(sh.found_number);
    const auto in = [&](float v) { return weight_bin(v, rw) == bin; };
    Cut cut;
    if (number > kCandidates) {   // ties: the key first, then as many of its classes as it takes
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
                    heavier += rw.whole(rw.real(v[e]));
                }
            }
        });
        above += block_total(heavier, sh.part);
        more = block_total(more, sh.part);
        equal = block_total(equal, sh.part);
        const uint64_t w = rw.whole(rw.real(key_score(cut.key)));
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
                sh.order[atomicAdd(&sh.count, 1u)] = static_cast<uint64_t>(~score_key(v[e])) << 32 | static_cast<uint32_t>(at + e);
    });
    __syncthreads();
    rank_candidates(number, rw, 0.0);
    const int per = (number + kSampleThreads - 1) / kSampleThreads, r0 = per * threadIdx.x, r1 = min(number, r0 + per);
    sum = 0;
    for (int r = r0; r < r1; ++r) sum += sh.mass[r];
    uint64_t at = above + block_scan(sum, sh.part, all) - sum;
    uint64_t kept = 0, kept_mass = 0;
    for (int r = r0; r < r1; ++r) {
        if (begins(at, before + r)) {
            ++kept;
            kept_mass += sh.mass[r];
        }
        at += sh.mass[r];
    }
    kept = block_total(kept, sh.part);
    cut.mass = above + block_total(kept_mass, sh.part);
    // the key of the last kept rank, and how many of the kept ranks have it
    const int last = kept ? static_cast<int>(kept) - 1 : 0;
    const float v = static_cast<float>(x[sh.cls[last]]);
    cut.key = score_key(v);
    uint64_t same = 0;
    for (int r = threadIdx.x; r <= last; r += kSampleThreads) same += static_cast<float>(x[sh.cls[r]]) == v;
    cut.quota = block_total(same, sh.part);
    return cut;
}

// The class for a row, to thread 0; -1: every class is masked.  logprob = (score - top) - log(soft_sum).
template <typename T>
__device__ __forceinline__ uint32_t sample_class(const SampleArgs& a, long long row, const T* __restrict__ x,
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
    const bool rough_mass = !greedy && use_p && !use_k && n > kCandidates && set.t != 1.0f;
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
    const bool holds = n <= kDeep * kSampleThreads * kLen;
    Vec16<T> raw[kDeep];
    if (holds) {
        load_vectors(raw, x, 0, n, threadIdx.x, kSampleThreads);
        use_vectors(raw, 0, n, threadIdx.x, kSampleThreads, add);
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
    if (threadIdx.x == 0) {
        sh.count = 0;
        sh.choice = 0xffffffffu;
    }
    __syncthreads();
    {   // lane l: wave l % 16
        top = sh.stat[0][lane % kSampleWaves];
        soft = sh.stat[1][lane % kSampleWaves];
        tempered = sh.stat[2][lane % kSampleWaves];
        float most = top;
#pragma unroll
        for (int o = kSampleWaves / 2; o; o >>= 1) most = fmaxf(most, __shfl_xor(most, o));
        join(most);
#pragma unroll
        for (int o = kSampleWaves / 2; o; o >>= 1) soft += __shfl_xor(soft, o);
        if (rough_mass)
#pragma unroll
            for (int o = kSampleWaves / 2; o; o >>= 1) tempered += __shfl_xor(tempered, o);
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
    if (n > kCandidates) {
        if (use_k) {
            if (top_k <= kSampleThreads) floor_key = kth_of_threads(share_key, top_k);
            try_candidates = top_k <= kSampleThreads;   // also if few shares hold anything at all
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
    if (try_candidates) {
        const float floor = floor_key ? key_score(floor_key) : -INFINITY;
        const auto collect = [&](const float (&v)[kLen], int at) {
            float most = v[0];
#pragma unroll
            for (int e = 1; e < kLen; ++e) most = fmaxf(most, v[e]);
            if (!__any(most >= floor && most > rw.none)) return;
            uint32_t hits = 0;
#pragma unroll
            for (int e = 0; e < kLen; ++e) hits |= v[e] >= floor && v[e] > rw.none ? 1u << e : 0;
            // places for the hits of the wave: one atomic, and a prefix sum of 4-bit numbers
            const uint32_t mine = __popc(hits);
            uint32_t before = 0, all = 0;
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const uint64_t has = __ballot((mine >> b) & 1);
                before += __popcll(has & ((1ull << lane) - 1)) << b;
                all += __popcll(has) << b;
            }
            uint32_t to = 0;
            if (lane == 0) to = atomicAdd(&sh.count, all);
            to = __builtin_amdgcn_readfirstlane(to) + before;
            while (hits) {   // (few: the scores once more from cache, instead of eight copies of this)
                const int j = at + __ffs(hits) - 1;
                hits &= hits - 1;
                if (to < kCandidates) sh.order[to] = static_cast<uint64_t>(~score_key(static_cast<float>(x[j]))) << 32 | static_cast<uint32_t>(j);
                ++to;
            }
        };
        if (holds) use_vectors(raw, 0, n, threadIdx.x, kSampleThreads, collect);
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
            const double slack = exact ? 0.0 : (n / kSampleThreads + 64) * 0x1p-23;
            bool unsure = false;
            int listed = found;
            uint64_t total = 0;
            bool rank = (use_k && found > top_k) || use_p;
            if (!rank || (use_p && !exact)) {
                // as they come; those too light weigh nothing
                for (int i = threadIdx.x; i < found; i += kSampleThreads) {   // (one turn unless there are many)
                    const uint64_t one = sh.order[i];
                    const double w = rw.real(key_score(~static_cast<uint32_t>(one >> 32)));
                    sh.cls[i] = static_cast<uint32_t>(one);
                    sh.mass[i] = w >= least ? rw.whole(w) : 0;
                    total += sh.mass[i];
                }
                total = block_total(total, sh.part);
                if (use_p) {
                    const double goal = share * rough * rw.scale;
                    if (use_m) rank = !(static_cast<double>(total) < goal * (1.0 - slack));   // below it top_p takes none away
                    else unsure = !(static_cast<double>(total) > goal * (1.0 + slack));       // a guess has to reach it
                    rank = rank && !unsure;
                }
            }
            if (rank) {
                const int heavy = rank_candidates(found, rw, least);
                const int limit = use_k ? min(top_k, found) : found;
                const int per = (limit + kBook - 1) / kBook, r0 = threadIdx.x < kBook ? per * threadIdx.x : limit, r1 = min(limit, r0 + per);
                uint64_t sum = 0, mass;
                for (int r = r0; r < r1; ++r) sum += sh.mass[r];
                uint64_t before = book_scan(sum, sh.part, mass) - sum;
                const double all = exact ? static_cast<double>(mass) : rough * rw.scale, goal = share * all;
                uint32_t kept = 0;
                int near = 0;
                uint64_t kept_mass = 0;
                for (int r = r0; r < r1; ++r) {
                    const uint64_t w = sh.mass[r];
                    const double b = static_cast<double>(before);
                    near |= use_p && r > 0 && !(fabs(b - goal) >= slack * goal);
                    if (r < heavy && (!use_p || r == 0 || b < goal)) {
                        ++kept;
                        kept_mass += w;
                    }
                    before += w;
                }
                unsure = __syncthreads_or(near);
                listed = static_cast<int>(block_total(kept, sh.part_u32));
                total = block_total(kept_mass, sh.part);
            }
            if (!unsure) {
                const uint64_t goal = static_cast<uint64_t>(static_cast<double>(u) * static_cast<double>(total));
                return draw_candidate(listed, min(goal, total - 1), n);
            }
        }
    }

    // 4.
    Cut cut{0, 0, 0};
    if (threadIdx.x == 0) sh.rw = rw;
    __syncthreads();
    if (use_k) cut = find_cut<T>(x, n, true, top_k, 0, n);
    if (use_p) cut = find_cut<T>(x, n, false, share, cut.mass, use_k ? top_k : n);
    const float cut_score = cut.key ? key_score(cut.key) : rw.none;
    const double cut_weight = cut.key ? rw.real(cut_score) : 0.0;
    const bool cut_counts = cut.key && cut_weight >= least;
    const auto over = [&](float v) {   // the weight of a class above the cut, 0 of any other
        const double w = rw.real(v);
        return v > cut_score && w >= least ? w : 0.0;
    };
    __syncthreads();
    // the mass of each piece, and how many classes at the key it holds
    const int piece = ((n + kPieces - 1) / kPieces + 64 * kLen - 1) / (64 * kLen) * (64 * kLen);
    for (int i = wave; i < kPieces; i += kSampleWaves) {
        const int stop = min(n, (i + 1) * piece);
        double m = 0.0;
        uint32_t ties = 0;
        stream_vectors<2>(x, i * piece, stop, lane, 64, [&](const float (&v)[kLen], int) {
            if (cut.key) {   // most vectors hold nothing above a cut
                float most = v[0];
#pragma unroll
                for (int e = 1; e < kLen; ++e) most = fmaxf(most, v[e]);
                if (!__any(most >= cut_score)) return;
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
    const int stop = min(n, (chosen + 1) * piece), per = (piece + kSampleThreads - 1) / kSampleThreads;
    const int from = min(stop, chosen * piece + static_cast<int>(threadIdx.x) * per), to = min(stop, from + per);
    float v[kShare];   // the first scores of the share: all of it up to 131 072 classes
#pragma unroll
    for (int i = 0; i < kShare; ++i) v[i] = from + i < to ? static_cast<float>(x[from + i]) : -INFINITY;
    const auto each = [&](auto f) {   // f(class, score) for the share
#pragma unroll
        for (int i = 0; i < kShare; ++i)
            if (from + i < to) f(from + i, v[i]);
        for (int j = from + kShare; j < to; ++j) f(j, static_cast<float>(x[j]));
    };
    uint64_t rank0 = chosen_tied;
    if (cut_counts) {
        uint64_t ties = 0, all;
        each([&](int, float s) { ties += s == cut_score; });
        rank0 += block_scan(ties, sh.part, all) - ties;
    }
    uint64_t rank = rank0;
    const auto weight = [&](float s) { return cut_counts && s == cut_score ? (rank++ < cut.quota ? cut_weight : 0.0) : over(s); };
    double m = 0.0;
    each([&](int, float s) { m += weight(s); });
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
            const double w = weight(s);
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

template <typename T>
__global__ __launch_bounds__(kSampleThreads) void k_sample_row(SampleArgs a) {
    const long long row = blockIdx.x;
    const T* x = static_cast<const T*>(a.logits) + row * a.row_stride;
    float top;
    double soft_sum = 1.0;
    const uint32_t cls = sample_class(a, row, x, top, soft_sum);
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
            const double w = v > rw.none ? rw.real(v) : 0.0;
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
