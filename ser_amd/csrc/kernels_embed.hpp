// Embedding lookup with scaling, and the table's gradient by sorted tokens.
//
//   y_n  = s * W[t_n]                      (a token outside 0..V-1 is padding: a row of zeros)
//   dW_v = s * sum_{n : t_n = v} dy_n      (f32, in position order; one rounding at the end)
//
//   k_embed            the lookup: one group of lanes per 16-byte-vector segment of a row
//   k_sort_small       stable radix sort of (token, position) in the LDS of one workgroup, up to 4 096 tokens
//   k_sort_count, k_sort_scan, k_sort_scatter   the same over tiles of 1 024 or 2 048: digits counted, and moved pass by pass
//   k_embed_sum        rows of the gradient: sums of short runs, zeros where no token fell; f32 sums of the pieces of long
//                      runs, one piece per tile of kRunTile sorted tokens
//   k_embed_join       the pieces of a long run, in order
//
// The lookup is bound by its writes (65 536 rows of 1 024 bf16: 45 us; 31, 4.3 TB/s of them, with the table's rows in cache).  The
// gradient by reading N rows and writing V, and where N is small by the chain of its three or six launches (3 001 tokens:
// 22 us; 32 768, 50 001 rows of 1 024 bf16: 95 us, k_embed_sum 68 of them, 47 with the rows in cache).  A run is summed by one
// wave per segment with kInFlight rows on their way: what it takes is a load's latency for every kInFlight rows, so runs are
// cut at kRunTile = 32 (at 128, four in flight, the longest uncut run of a batch of 3 001 took 43 us, twice the whole of it now).
//
// Nothing is accumulated with floating-point atomics: the sorted order fixes the order of every sum, so equal calls
// give equal bits.
#pragma once

#include "class_common.hpp"

namespace serhip {

constexpr int kSortThreads = 512;   // of a sort pass, with kPer tokens each: 2, or 4 above kSortShort tokens, where adding
constexpr int kSortShort = 131072;  // up the tiles' counts costs more than more workgroups give (32 768 tokens of 1 024 bf16
                                    // columns: 70 and 73 us; 262 144 of 64: 139 and 130)
constexpr int kSortMaxBits = 10;    // digit width: 1 024 bins x 8 waves of counters take 32 KB of LDS
constexpr int kScanTiles = 512;     // above so many tiles their counts are added up by a kernel of its own
constexpr int kSmallSort = 4096;    // tokens that one workgroup sorts (3 001, whole gradient: 21 us, with the tiles' kernels 26;
                                    // 4 096: 23 and 22)
constexpr int kSmallThreadsSort = 1024;
constexpr int kSmallBits = 8;
constexpr int kRunTile = 32;        // a run longer than this is summed in pieces of at most this many rows
constexpr int kInFlight = 4;        // rows of a run (8: 65 536 tokens of 1 024 bf16 columns 88 us, 4: 83, with 3 waves more on a SIMD)
constexpr int kJoinInFlight = 8;    // pieces of one
constexpr int kMostRows = 32;       // of the table, for a workgroup

// 2^lane_bits lanes take one segment of a row; blockIdx.y is the segment
template <typename T>
__global__ __launch_bounds__(256) void k_embed(const void* __restrict__ tokens, int tok_i64, long long n_tokens,
                                               const T* __restrict__ table, long long table_stride,
                                               long long n_classes, int width, int lane_bits, float scale,
                                               T* __restrict__ out, long long out_stride) {
    constexpr int kLen = Vec16<T>::kLen;
    const long long row = (static_cast<long long>(blockIdx.x) * 256 + threadIdx.x) >> lane_bits;
    if (row >= n_tokens) return;
    const int col = ((blockIdx.y << lane_bits) + (threadIdx.x & ((1 << lane_bits) - 1))) * kLen;
    if (col >= width) return;
    const int64_t tok = load_index(tokens, tok_i64, row);
    const bool inside = tok >= 0 && tok < n_classes;
    if (width >= kLen) {   // a vector that would reach past the row is the row's last one (two lanes write the same then)
        const int from = min(col, width - kLen);
        Vec16<T> y;
#pragma unroll
        for (int e = 0; e < kLen; ++e) y.v[e] = static_cast<T>(0.0f);
        if (inside) {
            const Vec16<T> x = load16(table + tok * table_stride + from);
#pragma unroll
            for (int e = 0; e < kLen; ++e) y.v[e] = static_cast<T>(static_cast<float>(x.v[e]) * scale);
        }
        store16(out + row * out_stride + from, y);
        return;
    }
    for (int e = 0; e < width; ++e)
        out[row * out_stride + e] = static_cast<T>(inside ? static_cast<float>(table[tok * table_stride + e]) * scale : 0.0f);
}

// ------------------------------------------------------------------------------------------------ sort
// The sort key of a token: the token, or n_classes for padding, which so ends up behind every real row.
__device__ __forceinline__ uint32_t sort_key(const void* tokens, int tok_i64, int64_t i, uint32_t n_classes) {
    const int64_t t = load_index(tokens, tok_i64, i);
    return t >= 0 && t < static_cast<int64_t>(n_classes) ? static_cast<uint32_t>(t) : n_classes;
}

// hist[tile][digit] of a pass over the keys (key == NULL: over the tokens).  A kernel for each pass: counting the next
// pass's digits with atomics while scattering costs more than the launch as soon as a token is frequent (32 768 tokens, 6%
// of them one: 14 us).
template <int kPer>
__global__ __launch_bounds__(kSortThreads) void k_sort_count(const void* __restrict__ tokens, int tok_i64, int n,
                                                             uint32_t n_classes, const uint32_t* __restrict__ key, int shift, int bits,
                                                             uint32_t* __restrict__ hist, uint32_t* __restrict__ long_runs) {
    if (blockIdx.x == 0 && threadIdx.x == 0) *long_runs = 0;   // no long run listed yet
    __shared__ uint32_t s_count[1 << kSortMaxBits];
    const int bins = 1 << bits;
    for (int d = threadIdx.x; d < bins; d += kSortThreads) s_count[d] = 0;
    __syncthreads();
    const int64_t first = static_cast<int64_t>(blockIdx.x) * (kSortThreads * kPer);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int64_t at = first + i * kSortThreads + threadIdx.x;
        if (at < n) atomicAdd(&s_count[((key ? key[at] : sort_key(tokens, tok_i64, at, n_classes)) >> shift) & (bins - 1)], 1u);
    }
    __syncthreads();
    for (int d = threadIdx.x; d < bins; d += kSortThreads) hist[static_cast<int64_t>(blockIdx.x) * bins + d] = s_count[d];
}

// hist[tile][digit] -> the sum over earlier tiles; total[digit].  A thread for each digit.
__global__ __launch_bounds__(kSortThreads) void k_sort_scan(uint32_t* __restrict__ hist, int tiles, int bins, uint32_t* __restrict__ total) {
    const int d = blockIdx.x * kSortThreads + threadIdx.x;
    if (d >= bins) return;
    uint32_t sum = 0;
    for (int t = 0; t < tiles; t += 16) {
        uint32_t c[16];
#pragma unroll
        for (int u = 0; u < 16; ++u) c[u] = t + u < tiles ? hist[static_cast<int64_t>(t + u) * bins + d] : 0;
#pragma unroll
        for (int u = 0; u < 16; ++u)
            if (t + u < tiles) {
                hist[static_cast<int64_t>(t + u) * bins + d] = sum;
                sum += c[u];
            }
    }
    total[d] = sum;
}

// Lanes of a wave that hold the same digit (of `bits` bits), among the `live` ones.
__device__ __forceinline__ uint64_t same_digit(uint32_t digit, int bits, bool live) {
    uint64_t peers = __ballot(live);
    for (int b = 0; b < bits; ++b) {
        const bool one = (digit >> b) & 1;
        const uint64_t ones = __ballot(one);
        peers &= one ? ones : ~ones;
    }
    return peers;
}

// The place of a key among the keys of its digit in its wave, which `count` (of the wave) goes on counting.
__device__ __forceinline__ uint32_t rank_in_wave(uint32_t* count, uint32_t digit, int bits, bool live) {
    const int lane = threadIdx.x & 63;
    const uint64_t peers = same_digit(digit, bits, live);
    const int leader = live ? __ffsll(static_cast<unsigned long long>(peers)) - 1 : lane;
    uint32_t before = 0;
    if (live && lane == leader) {
        before = count[digit];
        count[digit] = before + __popcll(peers);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    return __shfl(before, leader) + __popcll(peers & ((1ull << lane) - 1));
}

// n <= kSmallSort: all passes in one workgroup, keys in registers between them
__global__ __launch_bounds__(kSmallThreadsSort) void k_sort_small(const void* __restrict__ tokens, int tok_i64, int n, uint32_t n_classes,
                                                                  int passes, int bits, uint32_t* __restrict__ key_out,
                                                                  uint32_t* __restrict__ pos_out, uint32_t* __restrict__ long_runs) {
    if (threadIdx.x == 0) *long_runs = 0;   // no long run listed yet
    constexpr int kWaves = kSmallThreadsSort / 64, kPer = kSmallSort / kSmallThreadsSort;
    __shared__ uint32_t s_key[kSmallSort], s_pos[kSmallSort];
    __shared__ uint32_t s_wave[kWaves][1 << kSmallBits];
    __shared__ uint32_t s_sum[(1 << kSmallBits) / 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, bins = 1 << bits;
    const int first = wave * (64 * kPer) + lane;
    uint32_t key[kPer], pos[kPer], rank[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        pos[i] = first + i * 64;
        key[i] = first + i * 64 < n ? sort_key(tokens, tok_i64, first + i * 64, n_classes) : 0;
    }
    for (int p = 0; p < passes; ++p) {
        const int shift = p * bits;
        for (int d = lane; d < bins; d += 64) s_wave[wave][d] = 0;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (int i = 0; i < kPer; ++i)
            rank[i] = rank_in_wave(s_wave[wave], (key[i] >> shift) & (bins - 1), bits, first + i * 64 < n);
        __syncthreads();
        const int d = threadIdx.x;   // (bins <= 256: the first four waves)
        uint32_t sum = 0, upto = 0;
        if (d < (1 << kSmallBits)) {
            if (d < bins)
#pragma unroll
                for (int w = 0; w < kWaves; ++w) {
                    const uint32_t c = s_wave[w][d];
                    s_wave[w][d] = sum;
                    sum += c;
                }
            upto = wave_scan_sum(sum);
            if (lane == 63) s_sum[wave] = upto;
        }
        __syncthreads();
        if (d < bins) {
            uint32_t base = upto - sum;
            for (int w = 0; w < wave; ++w) base += s_sum[w];
#pragma unroll
            for (int w = 0; w < kWaves; ++w) s_wave[w][d] += base;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kPer; ++i)
            if (first + i * 64 < n) {
                const uint32_t to = s_wave[wave][(key[i] >> shift) & (bins - 1)] + rank[i];
                s_key[to] = key[i];
                s_pos[to] = pos[i];
            }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kPer; ++i)
            if (first + i * 64 < n) {
                key[i] = s_key[first + i * 64];
                pos[i] = s_pos[first + i * 64];
            }
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i)
        if (first + i * 64 < n) {
            key_out[first + i * 64] = key[i];
            pos_out[first + i * 64] = pos[i];
        }
}

// One pass: keys move to where the pairs (digit, place before the pass) order them.  The place of a key is the number
// of keys with a smaller digit, plus those with its digit in earlier tiles (both from `hist`), in earlier waves of the
// tile, and earlier in its wave (ballots).  Up to kScanTiles tiles every workgroup adds up `hist` for itself: a read of
// 2 MB at most from L2 instead of a kernel between two passes; of more, k_sort_scan has left the earlier tiles' counts in
// `hist` and the sums in `total` (1 048 576 tokens: 392 us, with the scan 406; twice as many: 784 and 776).
// key_in == NULL: the first pass, which reads the tokens.
template <int kPer>
__global__ __launch_bounds__(kSortThreads) void k_sort_scatter(
    const void* __restrict__ tokens, int tok_i64, int n, uint32_t n_classes, const uint32_t* __restrict__ key_in,
    const uint32_t* __restrict__ pos_in, int shift, int bits, const uint32_t* __restrict__ hist,
    const uint32_t* __restrict__ total, uint32_t* __restrict__ key_out,
    uint32_t* __restrict__ pos_out) {
    constexpr int kWaves = kSortThreads / 64;
    __shared__ uint32_t s_wave[kWaves][1 << kSortMaxBits];
    __shared__ uint32_t s_sum[kWaves];
    const int bins = 1 << bits;
    const int tiles = gridDim.x;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int d = threadIdx.x; d < bins; d += kSortThreads)
#pragma unroll
        for (int w = 0; w < kWaves; ++w) s_wave[w][d] = 0;
    __syncthreads();

    // ranks inside the wave
    const int64_t first = static_cast<int64_t>(blockIdx.x) * (kSortThreads * kPer) + wave * (64 * kPer) + lane;
    uint32_t key[kPer], pos[kPer], rank[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int64_t at = first + i * 64;
        key[i] = 0;
        pos[i] = 0;
        if (at < n) {
            key[i] = key_in ? key_in[at] : sort_key(tokens, tok_i64, at, n_classes);
            pos[i] = key_in ? pos_in[at] : static_cast<uint32_t>(at);
        }
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i)
        rank[i] = rank_in_wave(s_wave[wave], (key[i] >> shift) & (bins - 1), bits, first + i * 64 < n);
    __syncthreads();

    // how many keys of a digit there are, and how many of them in earlier tiles
    constexpr int kDigits = (1 << kSortMaxBits) / kSortThreads;
    uint32_t all[kDigits] = {}, earlier[kDigits] = {};
#pragma unroll
    for (int j = 0; j < kDigits; ++j) {
        const int d = j * kSortThreads + threadIdx.x;
        if (d >= bins) break;
        if (total) {   // added up already
            all[j] = total[d];
            earlier[j] = hist[static_cast<int64_t>(blockIdx.x) * bins + d];
            continue;
        }
#pragma unroll 8
        for (int t = 0; t < tiles; ++t) {
            const uint32_t count = hist[static_cast<int64_t>(t) * bins + d];
            all[j] += count;
            earlier[j] += t < static_cast<int>(blockIdx.x) ? count : 0;
        }
    }
    // first places, digit by digit: scans of kSortThreads digits, one after another
    uint32_t below = 0;
#pragma unroll
    for (int j = 0; j < kDigits; ++j) {
        const int d = j * kSortThreads + threadIdx.x;
        if (j * kSortThreads >= bins) break;
        const uint32_t upto = wave_scan_sum(all[j]);
        __syncthreads();
        if (lane == 63) s_sum[wave] = upto;
        __syncthreads();
        uint32_t at = below + upto - all[j] + earlier[j];
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            if (w < wave) at += s_sum[w];
            below += s_sum[w];
        }
        if (d < bins)
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                const uint32_t c = s_wave[w][d];
                s_wave[w][d] = at;
                at += c;
            }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        if (first + i * 64 >= n) continue;
        const uint32_t to = s_wave[wave][(key[i] >> shift) & (bins - 1)] + rank[i];
        key_out[to] = key[i];
        pos_out[to] = pos[i];
    }
}

// -------------------------------------------------------------------------------------------- gradient
// First place in key[lo, hi) that is >= want.  A whole wave searches: 64 probes a step.
__device__ __forceinline__ int wave_lower_bound(const uint32_t* __restrict__ key, int lo, int hi, uint32_t want) {
    const int lane = threadIdx.x & 63;
    while (hi - lo > 64) {
        const int64_t span = hi - lo;
        const int at = lo + static_cast<int>(span * lane / 64);
        const int below = __popcll(__ballot(key[at] < want));   // probes 0..below-1 are below `want`
        const int new_lo = below ? lo + static_cast<int>(span * (below - 1) / 64) + 1 : lo;
        const int new_hi = below < 64 ? lo + static_cast<int>(span * below / 64) : hi;
        lo = new_lo;
        hi = new_hi > new_lo ? new_hi : new_lo;
    }
    const int at = lo + lane;
    return lo + __popcll(__ballot(at < hi && key[at] < want));
}

// First places in key[0, n) that are >= low and >= high (low < high), to every thread of a workgroup of 256, by 256 probes
// a step: each step is a load's latency that nothing hides.
__device__ __forceinline__ void block_range(const uint32_t* __restrict__ key, int n, uint32_t low, uint32_t high, int (&s_below)[2][4],
                                            int& from, int& to) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int lo[2] = {0, 0}, hi[2] = {n, n};
    const auto count = [&](const bool (&below)[2]) {   // over the workgroup
        int c[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            c[i] = __popcll(__ballot(below[i]));
            if (lane == 0) s_below[i][wave] = c[i];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 2; ++i) c[i] = s_below[i][0] + s_below[i][1] + s_below[i][2] + s_below[i][3];
        __syncthreads();
        from = c[0];
        to = c[1];
    };
    const uint32_t want[2] = {low, high};
    while (max(hi[0] - lo[0], hi[1] - lo[1]) > 256) {
        bool below[2];
        const int64_t span[2] = {hi[0] - lo[0], hi[1] - lo[1]};
#pragma unroll
        for (int i = 0; i < 2; ++i) below[i] = span[i] > 0 && key[lo[i] + span[i] * threadIdx.x / 256] < want[i];
        count(below);
        const int c[2] = {from, to};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if (span[i] == 0) continue;   // probes 0 .. c - 1 are below
            const int l = lo[i];
            lo[i] = c[i] ? l + static_cast<int>(span[i] * (c[i] - 1) / 256) + 1 : l;
            hi[i] = c[i] < 256 ? max(lo[i], l + static_cast<int>(span[i] * c[i] / 256)) : hi[i];
        }
    }
    bool below[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int at = lo[i] + static_cast<int>(threadIdx.x);
        below[i] = at < hi[i] && key[at] < want[i];
    }
    count(below);
    from += lo[0];
    to += lo[1];
}

// The elements that a lane sums up: a vector's, from column `from` on, of which it writes those from `skip` on (a vector
// that would reach past the row is the row's last one; what comes before `skip` in it is another lane's).  `len` < kLen
// only where the row is shorter than a vector.
struct Columns {
    int from, skip, len;
};
__device__ __forceinline__ Columns lane_columns(int col, int width, int vector) {
    const int from = max(0, min(col, width - vector));
    return {from, col - from, min(vector, width - from)};
}

// sum[e] += the rows pos[lo..hi) of `grad`, in order, kInFlight on their way
template <typename TG>
__device__ __forceinline__ void add_rows(const TG* __restrict__ grad, long long stride, const uint32_t* __restrict__ pos,
                                         int lo, int hi, const Columns& c, float* sum) {
    constexpr int kLen = Vec16<TG>::kLen;
    for (int i = lo; i < hi; i += kInFlight) {
        Vec16<TG> x[kInFlight];
#pragma unroll
        for (int u = 0; u < kInFlight; ++u)
            if (i + u < hi) {
                const TG* row = grad + static_cast<int64_t>(pos[i + u]) * stride + c.from;
                if (c.len == kLen) {
                    x[u] = load16(row);
                } else {
#pragma unroll
                    for (int e = 0; e < kLen - 1; ++e) x[u].v[e] = e < c.len ? row[e] : static_cast<TG>(0.0f);
                    x[u].v[kLen - 1] = static_cast<TG>(0.0f);
                }
            }
#pragma unroll
        for (int u = 0; u < kInFlight; ++u)
            if (i + u < hi)
#pragma unroll
                for (int e = 0; e < kLen; ++e) sum[e] += static_cast<float>(x[u].v[e]);
    }
}

// row[from + skip ..] = scale * sum (+ what is there)
template <typename TO, int kLen>
__device__ __forceinline__ void store_row(TO* row, const float* sum, float scale, const Columns& c, bool accumulate) {
    struct __attribute__((packed, aligned(sizeof(TO)))) Out {
        TO v[kLen];
    };
    TO* dst = row + c.from;
    if (c.len == kLen && c.skip == 0) {
        Out y;
        if (accumulate) {
            y = *reinterpret_cast<const Out*>(dst);
#pragma unroll
            for (int e = 0; e < kLen; ++e) y.v[e] = static_cast<TO>(fmaf(sum[e], scale, static_cast<float>(y.v[e])));
        } else {
#pragma unroll
            for (int e = 0; e < kLen; ++e) y.v[e] = static_cast<TO>(sum[e] * scale);
        }
        *reinterpret_cast<Out*>(dst) = y;
        return;
    }
#pragma unroll
    for (int e = 0; e < kLen; ++e)
        if (e >= c.skip && e < c.len)
            dst[e] = static_cast<TO>(accumulate ? fmaf(sum[e], scale, static_cast<float>(dst[e])) : sum[e] * scale);
}

// What a tile [begin, end) of the sorted tokens holds of long runs.  Such a run is longer than a tile, so it reaches
// over one of the tile's ends: `head` = the run of the first token, `tail` = the run of the last one where that is
// another.  One key outside the tile decides whether a run is long.
struct RunPieces {
    int head_end;     // [begin, head_end) is a piece of a long run; begin if not
    int tail_begin;   // [tail_begin, end) is a piece of another long run; end if not
    int tail_starts;  // the place where a long run begins in this tile, -1 if none does
};
__device__ __forceinline__ RunPieces run_pieces(const uint32_t* __restrict__ key, int begin, int end, int n,
                                                uint32_t n_classes) {
    const int lane = threadIdx.x & 63;
    const uint32_t a = key[begin], b = key[end - 1];
    int head = 0, tail = 0;   // tokens of the tile equal to its first / last one
    for (int at = begin; at < end; at += 64) {
        const bool live = at + lane < end;
        const uint32_t k = live ? key[at + lane] : 0;
        head += __popcll(__ballot(live && k == a));
        tail += __popcll(__ballot(live && k == b));
    }
    RunPieces p{begin, end, -1};
    if (a == b) {
        const bool from_before = begin > 0 && key[begin - 1] == a;
        const bool goes_on = end < n && key[end] == a;
        // a run that starts here and fills the tile is long if it goes on; a shorter last tile is checked backwards
        const bool is_long = from_before ? (end - begin == kRunTile || goes_on || (end - 1 - kRunTile >= 0 && key[end - 1 - kRunTile] == a))
                                         : goes_on && end - begin == kRunTile;
        if (is_long && a < n_classes) {
            p.head_end = end;
            if (!from_before) p.tail_starts = begin;
        }
        return p;
    }
    const int head_end = begin + head, tail_begin = end - tail;
    if (a < n_classes && head_end - 1 - kRunTile >= 0 && key[head_end - 1 - kRunTile] == a) p.head_end = head_end;
    if (b < n_classes && tail_begin + kRunTile < n && key[tail_begin + kRunTile] == b) {
        p.tail_begin = tail_begin;
        p.tail_starts = tail_begin;
    }
    return p;
}

// Two kinds of workgroups.  The first piece_blocks: their waves take (tile, 64-vector segment) items of the long runs,
// piece[tile][0] = sum of the head piece, piece[tile][1] = sum of the tail piece (width floats each), and list the places
// where long runs begin (in any order: each is joined by itself).  The others: rows_per_block rows of the table; their runs
// in the sorted tokens are found, then every wave takes (row, segment) items.  A row without tokens is written with zeros
// here (left alone when accumulating), so the gradient needs no clearing pass; a row with more than kRunTile tokens is left
// to the pieces and k_embed_join.
template <typename TG, typename TO>
__global__ __launch_bounds__(256) void k_embed_sum(const TG* __restrict__ grad, long long grad_stride, const uint32_t* __restrict__ key,
                                                   const uint32_t* __restrict__ pos, int n, long long n_classes, int width, float scale,
                                                   int accumulate, TO* __restrict__ out, long long out_stride, int rows_per_block,
                                                   int piece_blocks, float* __restrict__ piece, uint32_t* __restrict__ long_runs) {
    constexpr int kLen = Vec16<TG>::kLen;
    __shared__ int s_start[kMostRows + 1];
    __shared__ int s_below[2][4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int segments = (width + 64 * kLen - 1) / (64 * kLen);
    if (static_cast<int>(blockIdx.x) < piece_blocks) {
        const long long item = static_cast<long long>(blockIdx.x) * 4 + wave;
        const int tile = static_cast<int>(item / segments), segment = static_cast<int>(item % segments);
        if (static_cast<long long>(tile) * kRunTile >= n) return;
        const int begin = tile * kRunTile, end = min(n, begin + kRunTile);
        const RunPieces p = run_pieces(key, begin, end, n, static_cast<uint32_t>(n_classes));
        if (p.tail_starts >= 0 && segment == 0 && lane == 0) long_runs[1 + atomicAdd(long_runs, 1u)] = p.tail_starts;
        const int col = (segment * 64 + lane) * kLen;
        if (col >= width) return;
        const Columns c = lane_columns(col, width, kLen);
        for (int side = 0; side < 2; ++side) {
            const int lo = side ? p.tail_begin : begin, hi = side ? end : p.head_end;
            if (lo >= hi) continue;
            float sum[kLen] = {};
            add_rows(grad, grad_stride, pos, lo, hi, c, sum);
            store_row<float, kLen>(piece + (static_cast<int64_t>(tile) * 2 + side) * width, sum, 1.0f, c, false);
        }
        return;
    }
    const long long r0 = static_cast<long long>(blockIdx.x - piece_blocks) * rows_per_block;
    const int rows = static_cast<int>(min(static_cast<long long>(rows_per_block), n_classes - r0));
    int from, to;
    block_range(key, n, static_cast<uint32_t>(r0), static_cast<uint32_t>(r0 + rows), s_below, from, to);
    // a run begins where a key differs from the one before it: that place is the start of every row since
    for (int i = from + static_cast<int>(threadIdx.x); i <= to; i += 256) {
        const int first = i == from ? 0 : static_cast<int>(key[i - 1] - r0) + 1;
        const int last = i == to ? rows : static_cast<int>(key[i] - r0);
        for (int r = first; r <= last; ++r) s_start[r] = i;
    }
    __syncthreads();
    for (int item = wave; item < rows * segments; item += 4) {
        const int r = item / segments;
        const int lo = s_start[r], hi = s_start[r + 1];
        if (hi - lo > kRunTile || (accumulate && lo == hi)) continue;
        const int col = ((item - r * segments) * 64 + lane) * kLen;
        if (col >= width) continue;
        const Columns c = lane_columns(col, width, kLen);
        float sum[kLen] = {};
        add_rows(grad, grad_stride, pos, lo, hi, c, sum);
        store_row<TO, kLen>(out + (r0 + r) * out_stride, sum, scale, c, accumulate);
    }
}

// Every listed long run: a workgroup for each 256 columns of it adds its pieces up and writes its row.  The pieces are cut
// into four stretches, one for each wave, which are added in order: the result depends on the run alone.
template <typename TO>
__global__ __launch_bounds__(256) void k_embed_join(const uint32_t* __restrict__ key, int n, int width, const float* __restrict__ piece,
                                                    const uint32_t* __restrict__ long_runs, float scale, int accumulate,
                                                    TO* __restrict__ out, long long out_stride) {
    __shared__ float s_sum[3][64][4];
    const int segments = (width + 255) / 256, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long long items = static_cast<long long>(long_runs[0]) * segments;
    for (long long item = blockIdx.x; item < items; item += gridDim.x) {
        const int start = static_cast<int>(long_runs[1 + item / segments]), first = start / kRunTile;
        const uint32_t token = key[start];
        const int count = (wave_lower_bound(key, start, n, token + 1) - 1) / kRunTile - first + 1;
        const int stretch = (count + 3) / 4, lo = wave * stretch, hi = min(count, lo + stretch);
        const int col = (static_cast<int>(item % segments) * 64 + lane) * 4;
        const Columns c = lane_columns(min(col, width - 1), width, 4);
        float sum[4] = {};
        for (int t = lo; t < hi; t += kJoinInFlight) {
            float x[kJoinInFlight][4];
#pragma unroll
            for (int u = 0; u < kJoinInFlight; ++u) {
                // a run that begins behind a tile's first token is that tile's tail piece, and the head piece of later ones
                const int64_t at = (static_cast<int64_t>(first + t + u) * 2 + (t + u == 0 && start % kRunTile ? 1 : 0)) * width + c.from;
#pragma unroll
                for (int e = 0; e < 4; ++e) x[u][e] = 0.0f;
                if (t + u < hi) {
                    if (c.len == 4) {
                        const Vec16<float> y = load16(piece + at);
#pragma unroll
                        for (int e = 0; e < 4; ++e) x[u][e] = y.v[e];
                    } else {
#pragma unroll
                        for (int e = 0; e < 3; ++e)
                            if (e < c.len) x[u][e] = piece[at + e];
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < kJoinInFlight; ++u)
                if (t + u < hi)
#pragma unroll
                    for (int e = 0; e < 4; ++e) sum[e] += x[u][e];
        }
        if (wave)
#pragma unroll
            for (int e = 0; e < 4; ++e) s_sum[wave - 1][lane][e] = sum[e];
        __syncthreads();
        if (wave == 0 && col < width) {
#pragma unroll
            for (int w = 0; w < 3; ++w)
#pragma unroll
                for (int e = 0; e < 4; ++e) sum[e] += s_sum[w][lane][e];
            store_row<TO, 4>(out + static_cast<int64_t>(token) * out_stride, sum, scale, c, accumulate);
        }
        __syncthreads();
    }
}

}  // namespace serhip
