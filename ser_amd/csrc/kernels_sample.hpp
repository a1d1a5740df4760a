// Drawing a class from scores: temperature, top-k, top-p, min-p, from one given uniform number per row.
//
//   order    the classes by (score descending, index ascending); NaN and -inf scores take no part
//   weight   w_j = exp((x_j - max x) / T), held as a whole number of 2^-bits (bits <= 45): sums of them are exact and
//            do not depend on the order of adding, so every cut and every draw is the same in each run and each
//            division of the work; the 2^-46 that a weight is off by is far below the 2^-24 steps of the uniform number
//   kept     the first top_k of the order, of these the shortest prefix whose mass reaches top_p of theirs, of these
//            the weights >= min_p; a cut is held as (key, quota): every key above `key`, and the first `quota`
//            classes, by index, whose key equals it
//   token    the first kept class whose cumulative kept weight, in index order, exceeds u * (kept mass)
//   logprob  log softmax(x)[token], untempered and uncut
//
// k_sample_row: one workgroup of 1 024 per row.
#pragma once

#include "class_common.hpp"

namespace serhip {

constexpr int kSampleThreads = 1024;
constexpr int kSampleWaves = kSampleThreads / 64;
constexpr int kSampleBins = 2048;
constexpr int kSampleCells = 1024;

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

struct RowWeights {
    float top;        // the largest score
    double inv_t;
    double scale;     // 2^weight_bits
    __device__ __forceinline__ double real(float x) const {
        return x == top ? 1.0 : exp((static_cast<double>(x) - static_cast<double>(top)) * inv_t);
    }
    __device__ __forceinline__ uint64_t whole(double w) const { return static_cast<uint64_t>(w * scale + 0.5); }
};

struct SampleShared {
    uint64_t hist[kSampleBins];     // also the cells' masses and tie counts
    uint64_t part[kSampleWaves];
    uint64_t found_above;
    uint32_t found_bin;
    uint32_t choice;
    uint32_t last;
};

// The largest key k >= floor_key, k > 0, for which mass(keys >= k) reaches `target`, and the mass above k.  A key's mass
// is its weight, or 1 where kCount.  The caller has checked that the mass of all keys >= floor_key reaches it.
template <typename T, bool kCount>
__device__ uint32_t find_key(const T* __restrict__ x, int n, const RowWeights& rw, uint32_t floor_key, double target,
                             SampleShared& sh, uint64_t& above) {
    using D = KeyDigits<T>;
    uint32_t prefix = 0;   // the digits found so far, in place
    above = 0;
    for (int level = 0; level < D::kLevels; ++level) {
        const int shift = D::kShift[level];
        const int width = (level == 0 ? 32 : D::kShift[level - 1]) - shift;
        const uint32_t high = level == 0 ? 0 : ~0u << D::kShift[level - 1];
        for (int b = threadIdx.x; b < kSampleBins; b += kSampleThreads) sh.hist[b] = 0;
        __syncthreads();
        each_class(x, n, [&](float v, int) {
            const uint32_t k = score_key(v);
            if (k && k >= floor_key && (k & high) == prefix)
                atomicAdd(reinterpret_cast<unsigned long long*>(&sh.hist[(k >> shift) & ((1u << width) - 1)]),
                          static_cast<unsigned long long>(kCount ? 1 : rw.whole(rw.real(v))));
        });
        __syncthreads();
        // bins from the top: thread i takes the bins kSampleBins-1-2i and the one below
        const int b1 = kSampleBins - 1 - 2 * threadIdx.x, b0 = b1 - 1;
        const uint64_t h1 = sh.hist[b1], h0 = sh.hist[b0];
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

template <typename T>
__global__ __launch_bounds__(kSampleThreads) void k_sample_row(SampleArgs a) {
    constexpr int kLen = Vec16<T>::kLen;
    __shared__ SampleShared sh;
    const long long row = blockIdx.x;
    const int n = a.n_classes;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const T* x = static_cast<const T*>(a.logits) + row * a.row_stride;

    // the largest score, the first class that has it
    uint64_t best = 0;
    each_class(x, n, [&](float v, int j) {
        const uint64_t c = static_cast<uint64_t>(score_key(v)) << 32 | static_cast<uint32_t>(~j);
        best = c > best ? c : best;
    });
#pragma unroll
    for (int o = 32; o; o >>= 1) {
        const uint64_t c = __shfl_xor(static_cast<unsigned long long>(best), o);
        best = c > best ? c : best;
    }
    if (lane == 0) sh.part[wave] = best;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kSampleWaves; ++w) best = sh.part[w] > best ? sh.part[w] : best;
    __syncthreads();
    if (best >> 32 == 0) {   // every class is masked
        if (threadIdx.x == 0) {
            a.token[row] = -1;
            a.logprob[row] = -INFINITY;
        }
        return;
    }
    const float top = key_score(static_cast<uint32_t>(best >> 32));

    // settings; what is out of range, or NaN, is off
    const float temperature = a.temperature_rows ? a.temperature_rows[row] : a.temperature;
    const int top_k = a.top_k_rows ? a.top_k_rows[row] : a.top_k;
    const float top_p = a.top_p_rows ? a.top_p_rows[row] : a.top_p;
    const float min_p = a.min_p_rows ? a.min_p_rows[row] : a.min_p;
    const bool greedy = !(temperature > 0.0f && temperature < INFINITY);
    const RowWeights rw{top, greedy ? 1.0 : 1.0 / static_cast<double>(temperature),
                        static_cast<double>(1ull << a.weight_bits)};

    // sums over all classes that take part: softmax's (f32 terms, f64 from the thread on), their number, their mass
    float soft = 0.0f;
    uint64_t alive = 0, mass = 0;
    each_class(x, n, [&](float v, int) {
        if (!(v > -INFINITY)) return;
        soft += v == top ? 1.0f : exp2_fast((v - top) * 1.44269504f);
        alive += 1;
        if (!greedy) mass += rw.whole(rw.real(v));
    });
    double soft_sum = wave_sum(static_cast<double>(soft));
    double* s_soft = reinterpret_cast<double*>(sh.part);
    if (lane == 0) s_soft[wave] = soft_sum;
    __syncthreads();
    soft_sum = 0.0;
#pragma unroll
    for (int w = 0; w < kSampleWaves; ++w) soft_sum += s_soft[w];
    if (greedy) {
        if (threadIdx.x == 0) {
            a.token[row] = ~static_cast<uint32_t>(best);
            a.logprob[row] = static_cast<float>(-log(soft_sum));
        }
        return;
    }
    uint64_t n_alive, all_mass;
    block_scan(alive, sh.part, n_alive);
    block_scan(mass, sh.part, all_mass);

    // the cut: keys above cut_key, and the first `quota` classes at it
    uint32_t cut_key = 0;
    uint64_t quota = 0;
    uint64_t kept_mass = all_mass, above;
    if (top_k >= 1 && static_cast<uint64_t>(top_k) < n_alive) {
        cut_key = find_key<T, true>(x, n, rw, 0, top_k, sh, above);
        quota = top_k - above;
        uint64_t m = 0;
        each_class(x, n, [&](float v, int) {
            if (score_key(v) > cut_key) m += rw.whole(rw.real(v));
        });
        block_scan(m, sh.part, above);   // mass above the cut
        kept_mass = above + quota * rw.whole(rw.real(key_score(cut_key)));
    } else {
        above = all_mass;
    }
    if (top_p < 1.0f) {
        const double target = fmax(static_cast<double>(top_p), 0.0) * static_cast<double>(kept_mass);
        if (!(target > 0.0)) {
            cut_key = static_cast<uint32_t>(best >> 32);
            quota = 1;
        } else {
            if (!(static_cast<double>(above) < target)) {   // reached above the key of the cut
                cut_key = find_key<T, false>(x, n, rw, cut_key + 1, target, sh, above);
                quota = n;
            }
            // as many of the classes at the key as it takes
            const uint64_t w = rw.whole(rw.real(key_score(cut_key)));
            if (cut_key && w) {
                const double need = ceil((target - static_cast<double>(above)) / static_cast<double>(w));
                quota = need < static_cast<double>(quota) ? static_cast<uint64_t>(fmax(need, 1.0)) : quota;
            }
        }
    }

    // masses of contiguous cells of classes, and how many classes at the key each holds
    const int per_cell = ((n + kSampleCells - 1) / kSampleCells + 64 * kLen - 1) / (64 * kLen) * (64 * kLen);
    const int cells = (n + per_cell - 1) / per_cell;
    uint64_t* s_mass = sh.hist;
    uint64_t* s_ties = sh.hist + kSampleCells;
    const auto keeps = [&](uint32_t k, double w) { return k > cut_key && !(min_p > 0.0f && w < fmin(min_p, 1.0f)); };
    const auto at_key = [&](uint32_t k, double w) {
        return k && k == cut_key && !(min_p > 0.0f && w < fmin(min_p, 1.0f));
    };
    __syncthreads();
    for (int cell = wave; cell < cells; cell += kSampleWaves) {
        uint64_t m = 0;
        uint32_t ties = 0;
        const int stop = min(n, (cell + 1) * per_cell);
        for (int at = cell * per_cell + lane * kLen; at < stop; at += 64 * kLen)
            for (int e = 0; e < kLen && at + e < stop; ++e) {
                const float v = static_cast<float>(x[at + e]);
                const uint32_t k = score_key(v);
                if (k < cut_key || k == 0) continue;
                const double w = rw.real(v);
                if (keeps(k, w)) m += rw.whole(w);
                if (at_key(k, w)) ++ties;
            }
#pragma unroll
        for (int o = 32; o; o >>= 1) {
            m += __shfl_xor(static_cast<unsigned long long>(m), o);
            ties += __shfl_xor(ties, o);
        }
        if (lane == 0) {
            s_mass[cell] = m;
            s_ties[cell] = ties;
        }
    }
    __syncthreads();
    const bool mine = static_cast<int>(threadIdx.x) < cells;
    const uint64_t ties = mine ? s_ties[threadIdx.x] : 0;
    uint64_t total;
    const uint64_t ties_upto = block_scan(ties, sh.part, total);
    const uint64_t ties_before = ties_upto - ties;
    const uint64_t take = ties_before >= quota ? 0 : (ties < quota - ties_before ? ties : quota - ties_before);
    const uint64_t key_whole = cut_key ? rw.whole(rw.real(key_score(cut_key))) : 0;
    const uint64_t cell_mass = (mine ? s_mass[threadIdx.x] : 0) + take * key_whole;
    const uint64_t mass_upto = block_scan(cell_mass, sh.part, total);
    const float u = a.uniform[row];
    uint64_t goal = u > 0.0f ? static_cast<uint64_t>(static_cast<double>(u) * static_cast<double>(total)) : 0;
    if (goal >= total) goal = total - 1;
    if (threadIdx.x == 0) sh.choice = 0xffffffffu;
    __syncthreads();
    if (mass_upto > goal) atomicMin(&sh.choice, threadIdx.x);
    __syncthreads();
    const int cell = sh.choice;
    if (static_cast<int>(threadIdx.x) == cell) {
        s_mass[0] = mass_upto - cell_mass;   // mass and classes at the key before the cell
        s_ties[0] = ties_before;
    }
    __syncthreads();
    if (wave != 0) return;
    uint64_t mass_before = s_mass[0], tied_before = s_ties[0];
    const int stop = min(n, (cell + 1) * per_cell);
    for (int base = cell * per_cell; base < stop; base += 64 * kLen) {
        const int at = base + lane * kLen;
        uint32_t tied = 0;
        for (int e = 0; e < kLen && at + e < stop; ++e) {
            const float v = static_cast<float>(x[at + e]);
            tied += at_key(score_key(v), rw.real(v));
        }
        uint32_t tied_upto = tied;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t y = __shfl_up(tied_upto, o);
            if (lane >= o) tied_upto += y;
        }
        uint64_t rank = tied_before + tied_upto - tied;
        uint64_t m = 0;
        for (int e = 0; e < kLen && at + e < stop; ++e) {
            const float v = static_cast<float>(x[at + e]);
            const uint32_t k = score_key(v);
            const double w = k ? rw.real(v) : 0.0;
            if (keeps(k, w) || (at_key(k, w) && rank++ < quota)) m += rw.whole(w);
        }
        uint64_t upto = m;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const uint64_t y = shfl_up_u64(upto, o);
            if (lane >= o) upto += y;
        }
        const uint64_t here = __ballot(mass_before + upto > goal);
        if (here) {
            if (lane == __ffsll(static_cast<unsigned long long>(here)) - 1) {
                uint64_t sum = mass_before + upto - m;
                rank = tied_before + tied_upto - tied;
                for (int e = 0; e < kLen && at + e < stop; ++e) {
                    const float v = static_cast<float>(x[at + e]);
                    const uint32_t k = score_key(v);
                    const double w = k ? rw.real(v) : 0.0;
                    if (keeps(k, w) || (at_key(k, w) && rank++ < quota)) sum += rw.whole(w);
                    if (sum > goal) {
                        a.token[row] = at + e;
                        const double d = v == top ? 0.0 : static_cast<double>(v) - static_cast<double>(top);
                        a.logprob[row] = static_cast<float>(d - log(soft_sum));
                        break;
                    }
                }
            }
            return;
        }
        mass_before += __shfl(static_cast<unsigned long long>(upto), 63);
        tied_before += __shfl(tied_upto, 63);
    }
}

}  // namespace serhip
