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
// k_sample_row, one workgroup of 1 024 per row:
//   1. one read of the row: its largest score, softmax's sum, the sum at T (f32, online)
//   2. a score below which nothing can be kept -- from top_k and the largest score of every thread's share, from min_p, or
//      a guess that fits most nuclei -- and a second read that collects what is not below it
//   3. at most kCandidates classes: ranked, cut and drawn from in LDS.  Everything is exact there but the mass that top_p
//      refers to when neither top_k nor the row's size bounds it; that one is the f32 sum, and a border that falls into
//      its error sends the row to 4
//   4. everything else: no cut at all (the draw alone), or a histogram of the row over the logarithm of the weight, the
//      bin in which the cut falls, and that bin's classes ranked as in 3 -- or, where one bin holds too many (ties), a
//      radix search of their keys.  The cut is then (key, quota): every key above `key`, and the first `quota` classes,
//      by index, whose key equals it.  Masses are added up there as whole numbers of 2^-bits (bits <= 45), so that the
//      order in which atomics arrive changes nothing.  The draw adds the kept weights of 16 pieces of the row, and of
//      1 024 pieces of the one that holds the answer.
#pragma once

#include "class_common.hpp"

namespace serhip {

constexpr int kSampleThreads = 1024;
constexpr int kSampleWaves = kSampleThreads / 64;
constexpr int kSampleBins = 2048;
constexpr float kBinsPerOctave = 64.0f;   // of the weight; the last bin takes all that is below 2^-32
constexpr int kCandidates = 2048;
constexpr int kCountRank = 512;     // up to here a rank is counted (n reads each), above it is sorted
constexpr int kNucleusGuess = 640;  // of 1 024 threads: some 1 000 candidates where scores come in no order

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

__device__ __forceinline__ uint64_t shfl_up_u64(uint64_t x, int o) {
    return __shfl_up(static_cast<unsigned long long>(x), o);
}

// inclusive prefix sum over the workgroup; `total` too
__device__ __forceinline__ uint64_t block_scan(uint64_t x, uint64_t* s_part, uint64_t& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint64_t y = shfl_up_u64(x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 63) s_part[wave] = x;
    __syncthreads();
    uint64_t before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < kSampleWaves; ++w) {
        if (w < wave) before += s_part[w];
        total += s_part[w];
    }
    return x + before;
}

// f(score, class) for this thread's classes
template <typename T, typename F>
__device__ __forceinline__ void each_class(const T* __restrict__ x, int n, F f) {
    constexpr int kLen = Vec16<T>::kLen;
    for (int at = threadIdx.x * kLen; at < n; at += kSampleThreads * kLen) {
        if (at + kLen <= n) {
            const Vec16<T> v = load16(x + at);
#pragma unroll
            for (int e = 0; e < kLen; ++e) f(static_cast<float>(v.v[e]), at + e);
        } else {
            for (int e = 0; at + e < n; ++e) f(static_cast<float>(x[at + e]), at + e);
        }
    }
}

// e^y for y <= 0: 2^n 2^f with f in [-1/2, 1/2] and the series of 2^f to f^11 (its rest is below 2^-47 there)
__device__ __forceinline__ double exp_down(double y) {
    const double t = fmax(y * 1.4426950408889634, -1100.0);
    const double n = rint(t), f = t - n;
    double p = 4.4455382718708115e-10;
    p = fma(p, f, 7.0549116208011234e-09);
    p = fma(p, f, 1.0178086009239699e-07);
    p = fma(p, f, 1.3215486790144309e-06);
    p = fma(p, f, 1.5252733804059840e-05);
    p = fma(p, f, 1.5403530393381609e-04);
    p = fma(p, f, 1.3333558146428443e-03);
    p = fma(p, f, 9.6181291076284772e-03);
    p = fma(p, f, 5.5504108664821580e-02);
    p = fma(p, f, 2.4022650695910071e-01);
    p = fma(p, f, 6.9314718055994531e-01);
    p = fma(p, f, 1.0);
    return ldexp(p, static_cast<int>(n));
}

struct RowWeights {
    float top;        // the largest score
    double inv_t;
    double scale;     // 2^weight_bits
    __device__ __forceinline__ double real(float x) const {
        return x == top ? 1.0 : exp_down((static_cast<double>(x) - static_cast<double>(top)) * inv_t);
    }
    // round(w 2^bits), read off the mantissa of a sum with 2^52
    __device__ __forceinline__ uint64_t whole(double w) const {
        return static_cast<uint64_t>(__double_as_longlong(fma(w, scale, 0x1p52))) & ((1ull << 52) - 1);
    }
};

struct SampleShared {
    uint64_t hist[kSampleBins];      // masses
    uint32_t number[kSampleBins];    // of classes
    uint64_t order[kCandidates];     // candidates: ~key and class, which sort by rank
    double weight[kCandidates];          // by rank
    uint32_t cls[kCandidates];
    union {
        uint64_t part[kSampleWaves];
        double part_f64[kSampleWaves];
    };
    float stat[3][kSampleWaves];
    uint64_t found_above, found_before, found_number;
    uint32_t found_bin;
    uint32_t count;
    uint32_t choice;
};

// the same over doubles
__device__ __forceinline__ double block_scan_f64(double x, double* s_part, double& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const double y = __shfl_up(x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 63) s_part[wave] = x;
    __syncthreads();
    double before = 0.0;
    total = 0.0;
#pragma unroll
    for (int w = 0; w < kSampleWaves; ++w) {
        if (w < wave) before += s_part[w];
        total += s_part[w];
    }
    return x + before;
}

// ascending, n <= kCandidates
__device__ inline void sort_u64(uint64_t* s, int n) {
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

// The lower edge of the 16-bit bin that holds the k-th largest of one key per thread: at least k keys are not below
// it.  0 if fewer than k keys are above 0.
__device__ inline uint32_t kth_of_threads(uint32_t key, uint32_t k, SampleShared& sh) {
    uint32_t* hist = reinterpret_cast<uint32_t*>(sh.hist);
    uint32_t prefix = 0, above = 0;
    for (int level = 0; level < 2; ++level) {
        const int shift = level ? 16 : 24;
        __syncthreads();
        if (threadIdx.x < 256) hist[threadIdx.x] = 0;
        if (threadIdx.x == 0) sh.count = 0xffffffffu;
        __syncthreads();
        if (key && (level == 0 || key >> 24 == prefix >> 24)) atomicAdd(&hist[(key >> shift) & 255], 1u);
        __syncthreads();
        if (threadIdx.x < 64) {   // lane i: bins 255-4i .. 252-4i
            uint32_t h[4], sum = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) sum += h[i] = hist[255 - 4 * threadIdx.x - i];
            uint32_t upto = sum;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const uint32_t y = __shfl_up(upto, o);
                if (static_cast<int>(threadIdx.x) >= o) upto += y;
            }
            uint32_t before = above + upto - sum;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (before < k && before + h[i] >= k) {
                    sh.count = 255 - 4 * threadIdx.x - i;
                    sh.found_bin = before;
                }
                before += h[i];
            }
        }
        __syncthreads();
        if (sh.count == 0xffffffffu) return 0;
        prefix |= sh.count << shift;
        above = sh.found_bin;
    }
    return prefix;
}

// Among the classes that `in` accepts: the largest key for which `above` + mass(keys >= it) reaches `target`; `above`
// becomes the mass above it.  A key's mass is its weight, or 1 where kCount.
template <typename T, bool kCount, typename In>
__device__ uint32_t find_key(const T* __restrict__ x, int n, const RowWeights& rw, In in, double target, SampleShared& sh,
                             uint64_t& above) {
    using D = KeyDigits<T>;
    uint64_t* bins = sh.order;   // the histogram of the weights is still wanted
    static_assert(kCandidates >= kSampleBins, "room for the bins");
    uint32_t prefix = 0;   // the digits found so far, in place
    for (int level = 0; level < D::kLevels; ++level) {
        const int shift = D::kShift[level];
        const int width = (level == 0 ? 32 : D::kShift[level - 1]) - shift;
        const uint32_t high = level == 0 ? 0 : ~0u << D::kShift[level - 1];
        for (int b = threadIdx.x; b < kSampleBins; b += kSampleThreads) bins[b] = 0;
        __syncthreads();
        each_class(x, n, [&](float v, int) {
            const uint32_t k = score_key(v);
            if (k && (k & high) == prefix && in(v))
                atomicAdd(reinterpret_cast<unsigned long long*>(&bins[(k >> shift) & ((1u << width) - 1)]),
                          static_cast<unsigned long long>(kCount ? 1 : rw.whole(rw.real(v))));
        });
        __syncthreads();
        // bins from the top: thread i takes the bins kSampleBins-1-2i and the one below
        const int b1 = kSampleBins - 1 - 2 * threadIdx.x, b0 = b1 - 1;
        const uint64_t h1 = bins[b1], h0 = bins[b0];
        uint64_t total;
        const uint64_t upto = block_scan(h1 + h0, sh.part, total) + above;
        const uint64_t before = upto - h1 - h0;
        // the first bin that reaches the target; by rounding none may: then the lowest one that holds anything
        if (threadIdx.x == 0) sh.found_bin = 0;
        __syncthreads();
        if (h1 && static_cast<double>(before) < target) atomicMax(&sh.found_bin, 0x10000u - b1);
        if (h0 && static_cast<double>(before + h1) < target) atomicMax(&sh.found_bin, 0x10000u - b0);
        __syncthreads();
        const int bin = 0x10000 - static_cast<int>(sh.found_bin);
        if (b1 == bin) sh.found_above = before;
        if (b0 == bin) sh.found_above = before + h1;
        __syncthreads();
        above = sh.found_above;
        prefix |= static_cast<uint32_t>(bin) << shift;
        __syncthreads();
    }
    // the digits that the type leaves: 0 for positive numbers, ones for the inverted bits of negative ones
    const int rest = D::kShift[D::kLevels - 1];
    return prefix & 0x80000000u ? prefix : prefix | ((1u << rest) - 1);
}

// sh.order[0..found) -> class and weight in rank order
__device__ inline void rank_candidates(SampleShared& sh, int found, const RowWeights& rw) {
    if (found <= kCountRank) {
        if (static_cast<int>(threadIdx.x) < found) {
            const uint64_t mine = sh.order[threadIdx.x];
            int rank = 0;
            for (int i = 0; i < found; ++i) rank += sh.order[i] < mine;
            sh.cls[rank] = static_cast<uint32_t>(mine);
            sh.weight[rank] = rw.real(key_score(~static_cast<uint32_t>(mine >> 32)));
        }
    } else {
        sort_u64(sh.order, found);
        for (int i = threadIdx.x; i < found; i += kSampleThreads) {
            sh.cls[i] = static_cast<uint32_t>(sh.order[i]);
            sh.weight[i] = rw.real(key_score(~static_cast<uint32_t>(sh.order[i] >> 32)));
        }
    }
    __syncthreads();
}

// the bin of a score in the histogram of step 4: by the logarithm of its weight, 0 = the heaviest
__device__ __forceinline__ int weight_bin(float v, float top, float ct) {
    return v == top ? 0 : static_cast<int>(fminf((top - v) * (ct * kBinsPerOctave), static_cast<float>(kSampleBins - 1)));
}

struct Cut {
    uint32_t key;      // 0: none
    uint64_t quota;    // classes at the key that are kept
    uint64_t mass;     // of all that is kept
};

// Where the order is cut when `target` of it is kept -- classes (kCount) or mass -- from the filled histogram.  Not
// more than `limit` classes are kept in any case.
template <typename T, bool kCount>
__device__ Cut find_cut(const T* __restrict__ x, int n, const RowWeights& rw, float ct, double target, uint64_t limit, SampleShared& sh) {
    // the first bin that reaches the target, or the limit
    const int b0 = 2 * threadIdx.x, b1 = b0 + 1;
    const uint64_t m0 = sh.hist[b0], m1 = sh.hist[b1], c0 = sh.number[b0], c1 = sh.number[b1];
    uint64_t all;
    const uint64_t mass1 = block_scan(m0 + m1, sh.part, all) - m1, mass0 = mass1 - m0;   // before each bin
    const uint64_t count1 = block_scan(c0 + c1, sh.part, all) - c1, count0 = count1 - c0;
    __syncthreads();
    if (threadIdx.x == 0) sh.found_bin = 0;
    __syncthreads();
    // the last bin with anything in it that begins below both (the first one always does)
    const auto begins = [&](uint64_t mass, uint64_t count) {
        return count < limit && static_cast<double>(kCount ? count : mass) < target;
    };
    if (c0 && begins(mass0, count0)) atomicMax(&sh.found_bin, static_cast<uint32_t>(b0));
    if (c1 && begins(mass1, count1)) atomicMax(&sh.found_bin, static_cast<uint32_t>(b1));
    __syncthreads();
    const int bin = sh.found_bin;
    if (b0 == bin || b1 == bin) {
        sh.found_above = b0 == bin ? mass0 : mass1;
        sh.found_before = b0 == bin ? count0 : count1;
        sh.found_number = b0 == bin ? c0 : c1;
    }
    if (threadIdx.x == 0) sh.count = 0;
    __syncthreads();
    uint64_t above = sh.found_above;
    const uint64_t before = sh.found_before;
    const int number = static_cast<int>(sh.found_number);
    const auto in = [&](float v) { return weight_bin(v, rw.top, ct) == bin; };
    Cut cut;
    if (number > kCandidates) {   // ties: the key first, then as many of its classes as it takes
        uint64_t reached = kCount ? before : above;
        cut.key = find_key<T, kCount>(x, n, rw, in, target, sh, reached);
        uint64_t heavier = 0, more = 0, equal = 0;   // in the bin: mass and number above the key, number at it
        each_class(x, n, [&](float v, int) {
            const uint32_t k = score_key(v);
            if (!k || k < cut.key || !in(v)) return;
            if (k == cut.key) ++equal;
            else {
                ++more;
                heavier += rw.whole(rw.real(v));
            }
        });
        block_scan(heavier, sh.part, all);
        above += all;
        block_scan(more, sh.part, all);
        more = all;
        block_scan(equal, sh.part, all);
        const uint64_t w = rw.whole(rw.real(key_score(cut.key)));
        double take = kCount ? target - static_cast<double>(before + more)
                             : (w ? ceil((target - static_cast<double>(above)) / static_cast<double>(w)) : static_cast<double>(all));
        take = fmin(fmax(take, 1.0), fmin(static_cast<double>(all), static_cast<double>(limit - before - more)));
        cut.quota = static_cast<uint64_t>(take);
        cut.mass = above + cut.quota * w;
        __syncthreads();
        return cut;
    }
    each_class(x, n, [&](float v, int j) {
        if (v > -INFINITY && in(v)) sh.order[atomicAdd(&sh.count, 1u)] = static_cast<uint64_t>(~score_key(v)) << 32 | static_cast<uint32_t>(j);
    });
    __syncthreads();
    rank_candidates(sh, number, rw);
    const int r0 = 2 * threadIdx.x, r1 = r0 + 1;
    const uint64_t w0 = r0 < number ? rw.whole(sh.weight[r0]) : 0, w1 = r1 < number ? rw.whole(sh.weight[r1]) : 0;
    const uint64_t at1 = above + block_scan(w0 + w1, sh.part, all) - w1, at0 = at1 - w0;
    uint64_t kept = 0, mass = 0, n_kept;
    const auto keep = [&](int r, uint64_t at, uint64_t w) {
        if (r < number && begins(at, before + r)) {
            ++kept;
            mass += w;
        }
    };
    keep(r0, at0, w0);
    keep(r1, at1, w1);
    block_scan(kept, sh.part, n_kept);
    block_scan(mass, sh.part, cut.mass);
    cut.mass += above;
    // the key of the last kept rank, and how many of the kept ranks have it
    const uint32_t last = n_kept ? static_cast<uint32_t>(n_kept) - 1 : 0;
    const float v = static_cast<float>(x[sh.cls[last]]);
    cut.key = score_key(v);
    uint64_t same = 0;
    for (int r = threadIdx.x; r <= static_cast<int>(last); r += kSampleThreads) same += static_cast<float>(x[sh.cls[r]]) == v;
    block_scan(same, sh.part, cut.quota);
    __syncthreads();
    return cut;
}

// f32 statistics of a thread's share of a row
struct ShareStats {
    float top = -INFINITY, soft = 0.0f, tempered = 0.0f;   // max; sum of 2^(c (x - top)) for c = log2 e and log2 e / T
};

__device__ __forceinline__ void join_share(ShareStats& a, float top, float soft, float tempered, float ct) {
    const float both = fmaxf(a.top, top);
    if (both == -INFINITY) return;
    const float fa = (a.top - both) * 1.44269504f, fb = (top - both) * 1.44269504f;
    a.soft = a.soft * exp2_fast(fa) + soft * exp2_fast(fb);
    a.tempered = a.tempered * exp2_fast((a.top - both) * ct) + tempered * exp2_fast((top - both) * ct);
    a.top = both;
}

template <bool kTempered, typename T>
__device__ __forceinline__ void add_vector(ShareStats& a, const Vec16<T>& raw, float ct) {
    constexpr int kLen = Vec16<T>::kLen;
    float v[kLen], top = a.top;
#pragma unroll
    for (int e = 0; e < kLen; ++e) v[e] = fmaxf(static_cast<float>(raw.v[e]), -INFINITY);   // NaN is -inf
#pragma unroll
    for (int e = 0; e < kLen; ++e) top = fmaxf(top, v[e]);
    if (top == -INFINITY) return;
    if (top > a.top) {
        a.soft *= exp2_fast((a.top - top) * 1.44269504f);
        if (kTempered) a.tempered *= exp2_fast((a.top - top) * ct);
        a.top = top;
    }
#pragma unroll
    for (int e = 0; e < kLen; ++e) {
        const float d = v[e] - top;
        a.soft += exp2_fast(d * 1.44269504f);
        if (kTempered) a.tempered += exp2_fast(d * ct);
    }
}

template <bool kTempered, typename T>
__device__ __forceinline__ ShareStats share_stats(const T* __restrict__ x, int n, float ct) {
    constexpr int kLen = Vec16<T>::kLen, kStep = kSampleThreads * kLen, kDeep = 4;
    ShareStats a;
    int at = threadIdx.x * kLen;
    for (; at + (kDeep - 1) * kStep + kLen <= n; at += kDeep * kStep) {   // four vectors in flight
        Vec16<T> raw[kDeep];
#pragma unroll
        for (int u = 0; u < kDeep; ++u) raw[u] = load16(x + at + u * kStep);
#pragma unroll
        for (int u = 0; u < kDeep; ++u) add_vector<kTempered>(a, raw[u], ct);
    }
    for (; at < n; at += kStep) {
        Vec16<T> raw;
        if (at + kLen <= n) {
            raw = load16(x + at);
        } else {
#pragma unroll
            for (int e = 0; e < kLen; ++e) raw.v[e] = at + e < n ? x[at + e] : static_cast<T>(-INFINITY);
        }
        add_vector<kTempered>(a, raw, ct);
    }
    return a;
}

template <typename T>
__global__ __launch_bounds__(kSampleThreads) void k_sample_row(SampleArgs a) {
    constexpr int kLen = Vec16<T>::kLen;
    __shared__ SampleShared sh;
    const long long row = blockIdx.x;
    const int n = a.n_classes;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const T* x = static_cast<const T*>(a.logits) + row * a.row_stride;

    // settings; what is out of range, or NaN, is off
    const float temperature = a.temperature_rows ? a.temperature_rows[row] : a.temperature;
    const int top_k = a.top_k_rows ? a.top_k_rows[row] : a.top_k;
    const float top_p = a.top_p_rows ? a.top_p_rows[row] : a.top_p;
    float min_p = a.min_p_rows ? a.min_p_rows[row] : a.min_p;
    if (min_p > 1.0f) min_p = 1.0f;
    const float u = fmaxf(a.uniform[row], 0.0f);
    const bool greedy = !(temperature > 0.0f && temperature < INFINITY);
    const bool use_k = top_k >= 1 && top_k < n, use_p = top_p < 1.0f, use_m = min_p > 0.0f;
    const float ct = greedy ? 0.0f : 1.44269504f / temperature;

    // 1. the row's statistics
    const bool rough_mass = !greedy && use_p && !use_k && n > kCandidates;   // top_p of a mass that only step 1 sees whole
    ShareStats st = rough_mass && temperature != 1.0f ? share_stats<true>(x, n, ct) : share_stats<false>(x, n, ct);
    const uint32_t share_top = score_key(st.top);
#pragma unroll
    for (int o = 32; o; o >>= 1)
        join_share(st, __shfl_xor(st.top, o), __shfl_xor(st.soft, o), __shfl_xor(st.tempered, o), ct);
    if (lane == 0) {
        sh.stat[0][wave] = st.top;
        sh.stat[1][wave] = st.soft;
        sh.stat[2][wave] = st.tempered;
    }
    if (threadIdx.x == 0) {
        sh.count = 0;
        sh.choice = 0xffffffffu;
    }
    __syncthreads();
    st = ShareStats{};
#pragma unroll
    for (int w = 0; w < kSampleWaves; ++w) join_share(st, sh.stat[0][w], sh.stat[1][w], sh.stat[2][w], ct);
    const float top = st.top;
    if (top == -INFINITY) {   // every class is masked
        if (threadIdx.x == 0) {
            a.token[row] = -1;
            a.logprob[row] = -INFINITY;
        }
        return;
    }
    double soft_sum = st.soft, rough = temperature != 1.0f ? st.tempered : st.soft;
    if (top == INFINITY) {   // the classes at +inf share everything: weight 1 each
        uint64_t infs = 0, all;
        each_class(x, n, [&](float v, int) { infs += v == top; });
        block_scan(infs, sh.part, all);
        soft_sum = rough = static_cast<double>(all);
    }
    if (greedy) {
        uint32_t first = 0xffffffffu;
        each_class(x, n, [&](float v, int j) {
            if (v == top) first = min(first, static_cast<uint32_t>(j));
        });
        if (first != 0xffffffffu) atomicMin(&sh.choice, first);
        __syncthreads();
        if (threadIdx.x == 0) {
            a.token[row] = sh.choice;
            a.logprob[row] = static_cast<float>(-log(soft_sum));
        }
        return;
    }
    const RowWeights rw{top, 1.0 / static_cast<double>(temperature), static_cast<double>(1ull << a.weight_bits)};

    // 2. a key that every kept class reaches
    uint32_t floor_key = 0;
    bool try_candidates;
    if (n > kCandidates) {
        if (use_k) {
            if (top_k <= kSampleThreads) floor_key = kth_of_threads(share_top, top_k, sh);
        } else if (use_p && !use_m) {
            floor_key = kth_of_threads(share_top, kNucleusGuess, sh);
        }
        if (use_m && !(use_k && use_p)) {   // top_p of the first top_k needs all of these
            const double far = static_cast<double>(temperature) * log(static_cast<double>(min_p));
            const double bound = top + far - 1e-6 * (fabs(static_cast<double>(top)) - far);
            floor_key = max(floor_key, score_key(static_cast<float>(bound)));
        }
        try_candidates = floor_key != 0 || (use_k && top_k <= kSampleThreads);   // 0: too few shares hold anything at all
    } else {
        try_candidates = use_k || use_p || use_m;
    }
    if (try_candidates) {
        __syncthreads();
        if (threadIdx.x == 0) sh.count = 0;
        __syncthreads();
        const float floor = floor_key ? key_score(floor_key) : -INFINITY;
        const auto offer = [&](float v, int j) {
            if (v >= floor && v > -INFINITY) {
                const uint32_t to = atomicAdd(&sh.count, 1u);
                if (to < kCandidates) sh.order[to] = static_cast<uint64_t>(~score_key(v)) << 32 | static_cast<uint32_t>(j);
            }
        };
        for (int at = threadIdx.x * kLen; at < n; at += kSampleThreads * kLen) {
            if (at + kLen <= n) {
                const Vec16<T> v = load16(x + at);
                float most = static_cast<float>(v.v[0]);
#pragma unroll
                for (int e = 1; e < kLen; ++e) most = fmaxf(most, static_cast<float>(v.v[e]));
                if (most >= floor)
#pragma unroll
                    for (int e = 0; e < kLen; ++e) offer(static_cast<float>(v.v[e]), at + e);
            } else {
                for (int e = 0; at + e < n; ++e) offer(static_cast<float>(x[at + e]), at + e);
            }
        }
        __syncthreads();
        const int found = sh.count;
        if (found <= kCandidates) {
            // 3.
            rank_candidates(sh, found, rw);
            const int limit = use_k ? min(top_k, found) : found;
            const int r0 = 2 * threadIdx.x, r1 = r0 + 1;
            const double w0 = r0 < limit ? sh.weight[r0] : 0.0, w1 = r1 < limit ? sh.weight[r1] : 0.0;
            double mass;
            const double upto = block_scan_f64(w0 + w1, sh.part_f64, mass);
            const double before1 = upto - w1, before0 = before1 - w0;
            // what top_p is a share of; exact unless the candidates are not all there is
            const bool exact = floor_key == 0 || use_k;
            const double all = exact ? mass : rough;
            const double slack = exact ? 0.0 : (n / 1024 + 64) * 0x1p-23;
            int kept = 0, unsure = 0;
            const auto judge = [&](int r, double before, double w) {
                if (r >= limit || (use_m && w < static_cast<double>(min_p))) return;
                if (use_p && r > 0) {
                    const double goal = fmax(static_cast<double>(top_p), 0.0) * all;
                    unsure |= fabs(before - goal) < slack * goal;
                    if (!(before < goal)) return;
                }
                ++kept;
            };
            judge(r0, before0, w0);
            judge(r1, before1, w1);
            if (use_p) unsure |= !(all < INFINITY);
            // the kept ranks are a prefix.  The guess is too short if the last candidate's mass does not reach the goal
            if (use_p && !exact && !use_m) unsure |= !(mass > fmax(static_cast<double>(top_p), 0.0) * all * (1.0 + slack));
            unsure = __syncthreads_or(unsure);
            if (!unsure) {
                uint64_t n_kept_64;
                block_scan(kept, sh.part, n_kept_64);
                const int n_kept = static_cast<int>(n_kept_64);
                if (n_kept <= kCountRank) {
                    double here = 0.0, total = 0.0;
                    const bool live = static_cast<int>(threadIdx.x) < n_kept;
                    const uint32_t cls = live ? sh.cls[threadIdx.x] : 0;
                    for (int i = 0; i < n_kept; ++i) {
                        const double w = sh.weight[i];
                        total += w;
                        if (sh.cls[i] <= cls) here += w;
                    }
                    if (live && here > static_cast<double>(u) * total) atomicMin(&sh.choice, cls);
                    __syncthreads();
                    if (sh.choice == 0xffffffffu) {   // u >= 1
                        __syncthreads();
                        if (threadIdx.x == 0) sh.choice = 0;
                        __syncthreads();
                        if (live && sh.weight[threadIdx.x] > 0.0) atomicMax(&sh.choice, cls);
                        __syncthreads();
                    }
                } else {
                    for (int i = threadIdx.x; i < n_kept; i += kSampleThreads) sh.order[i] = static_cast<uint64_t>(sh.cls[i]) << 32 | i;
                    sort_u64(sh.order, n_kept);
                    const uint64_t o0 = r0 < n_kept ? sh.order[r0] : 0, o1 = r1 < n_kept ? sh.order[r1] : 0;
                    const double v0 = r0 < n_kept ? sh.weight[static_cast<uint32_t>(o0)] : 0.0;
                    const double v1 = r1 < n_kept ? sh.weight[static_cast<uint32_t>(o1)] : 0.0;
                    double total;
                    const double end1 = block_scan_f64(v0 + v1, sh.part_f64, total), end0 = end1 - v1;
                    const double goal = static_cast<double>(u) * total;
                    if (v0 > 0.0 && end0 > goal) atomicMin(&sh.choice, static_cast<uint32_t>(o0 >> 32));
                    if (v1 > 0.0 && end1 > goal) atomicMin(&sh.choice, static_cast<uint32_t>(o1 >> 32));
                    __syncthreads();
                    if (sh.choice == 0xffffffffu) {
                        __syncthreads();
                        if (threadIdx.x == 0) sh.choice = 0;
                        __syncthreads();
                        if (v0 > 0.0) atomicMax(&sh.choice, static_cast<uint32_t>(o0 >> 32));
                        if (v1 > 0.0) atomicMax(&sh.choice, static_cast<uint32_t>(o1 >> 32));
                        __syncthreads();
                    }
                }
                if (threadIdx.x == 0) {
                    const uint32_t cls = sh.choice;
                    const float v = static_cast<float>(x[cls]);
                    a.token[row] = cls;
                    a.logprob[row] = static_cast<float>((v == top ? 0.0 : static_cast<double>(v) - static_cast<double>(top)) - log(soft_sum));
                }
                return;
            }
        }
    }

    // 4.
    Cut cut{0, 0, 0};
    if (use_k || use_p) {
        __syncthreads();
        for (int i = threadIdx.x; i < kSampleBins; i += kSampleThreads) {
            sh.hist[i] = 0;
            sh.number[i] = 0;
        }
        __syncthreads();
        each_class(x, n, [&](float v, int) {
            if (!(v > -INFINITY)) return;
            const int b = weight_bin(v, top, ct);
            atomicAdd(reinterpret_cast<unsigned long long*>(&sh.hist[b]), static_cast<unsigned long long>(rw.whole(rw.real(v))));
            atomicAdd(&sh.number[b], 1u);
        });
        __syncthreads();
        uint64_t mass;
        block_scan(sh.hist[threadIdx.x] + sh.hist[threadIdx.x + kSampleThreads], sh.part, mass);
        uint64_t limit = n;
        if (use_k) {
            cut = find_cut<T, true>(x, n, rw, ct, top_k, n, sh);
            limit = top_k;
            mass = cut.mass;
        }
        // at least half a unit: the first class is kept whatever top_p is
        if (use_p) cut = find_cut<T, false>(x, n, rw, ct, fmax(static_cast<double>(top_p) * static_cast<double>(mass), 0.5), limit, sh);
    }
    const float cut_score = cut.key ? key_score(cut.key) : -INFINITY;
    const double least = use_m ? static_cast<double>(min_p) : 0.0;
    const double cut_weight = cut.key ? rw.real(cut_score) : 0.0;
    const bool cut_counts = cut.key && cut_weight >= least;
    const auto over = [&](float v) {   // the weight of a class above the cut, 0 of any other
        if (!(v > cut_score)) return 0.0;
        const double w = rw.real(v);
        return w >= least ? w : 0.0;
    };

    // the mass of each wave's piece of the row
    const int piece = ((n + kSampleWaves - 1) / kSampleWaves + 64 * kLen - 1) / (64 * kLen) * (64 * kLen);
    double m = 0.0;
    uint32_t ties = 0;
    {
        const int stop = min(n, (wave + 1) * piece);
        for (int at = wave * piece + lane * kLen; at < stop; at += 64 * kLen) {
            if (at + kLen <= stop) {
                const Vec16<T> raw = load16(x + at);
#pragma unroll
                for (int e = 0; e < kLen; ++e) {
                    m += over(static_cast<float>(raw.v[e]));
                    ties += cut_counts && static_cast<float>(raw.v[e]) == cut_score;
                }
            } else {
                for (int e = 0; at + e < stop; ++e) {
                    m += over(static_cast<float>(x[at + e]));
                    ties += cut_counts && static_cast<float>(x[at + e]) == cut_score;
                }
            }
        }
        m = wave_sum(m);
#pragma unroll
        for (int o = 32; o; o >>= 1) ties += __shfl_xor(ties, o);
        __syncthreads();
        if (lane == 0) {
            sh.weight[wave] = m;
            sh.cls[wave] = ties;
        }
        __syncthreads();
    }
    // the first piece whose cumulative mass exceeds the goal; past all of them (u >= 1, or rounding): the last with any
    double total = 0.0;
    uint64_t tied = 0;
    const auto share = [&](int w) {   // of piece w, and counts its ties
        const uint64_t t = sh.cls[w], left = tied < cut.quota ? cut.quota - tied : 0;
        tied += t;
        return sh.weight[w] + static_cast<double>(t < left ? t : left) * cut_weight;
    };
    for (int w = 0; w < kSampleWaves; ++w) total += share(w);
    const double goal = static_cast<double>(u) * total;
    int chosen = -1, final = 0;
    double before = 0.0, chosen_before = 0.0, final_before = 0.0;
    uint64_t chosen_tied = 0, final_tied = 0;
    tied = 0;
    for (int w = 0; w < kSampleWaves; ++w) {
        const uint64_t tied_here = tied;
        const double mine = share(w);
        if (mine > 0.0) {
            final = w;
            final_before = before;
            final_tied = tied_here;
            if (chosen < 0 && before + mine > goal) {
                chosen = w;
                chosen_before = before;
                chosen_tied = tied_here;
            }
        }
        before += mine;
    }
    if (chosen < 0) {
        chosen = final;
        chosen_before = final_before;
        chosen_tied = final_tied;
    }
    // the same with a share of the piece for each thread
    const int stop = min(n, (chosen + 1) * piece), per = (piece + kSampleThreads - 1) / kSampleThreads;
    const int from = min(stop, chosen * piece + static_cast<int>(threadIdx.x) * per), to = min(stop, from + per);
    ties = 0;
    for (int j = from; j < to; ++j) ties += cut_counts && static_cast<float>(x[j]) == cut_score;
    uint64_t all_ties;
    const uint64_t rank0 = chosen_tied + block_scan(ties, sh.part, all_ties) - ties;
    uint64_t rank = rank0;
    m = 0.0;
    for (int j = from; j < to; ++j) {
        const float v = static_cast<float>(x[j]);
        if (cut_counts && v == cut_score) m += rank++ < cut.quota ? cut_weight : 0.0;
        else m += over(v);
    }
    double piece_mass;
    double sum = chosen_before + block_scan_f64(m, sh.part_f64, piece_mass) - m;
    __syncthreads();
    if (threadIdx.x == 0) {
        sh.choice = 0xffffffffu;
        sh.count = 0;
    }
    __syncthreads();
    if (m > 0.0) {
        int first = -1, last = -1;
        rank = rank0;
        for (int j = from; j < to; ++j) {
            const float v = static_cast<float>(x[j]);
            const double w = cut_counts && v == cut_score ? (rank++ < cut.quota ? cut_weight : 0.0) : over(v);
            sum += w;
            if (w > 0.0) {
                last = j;
                if (first < 0 && sum > goal) first = j;
            }
        }
        if (first >= 0) atomicMin(&sh.choice, static_cast<uint32_t>(first));
        if (last >= 0) atomicMax(&sh.count, static_cast<uint32_t>(last));
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        const uint32_t cls = sh.choice != 0xffffffffu ? sh.choice : sh.count;
        const float v = static_cast<float>(x[cls]);
        a.token[row] = cls;
        a.logprob[row] = static_cast<float>((v == top ? 0.0 : static_cast<double>(v) - static_cast<double>(top)) - log(soft_sum));
    }
}

}  // namespace serhip
