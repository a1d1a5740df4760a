// Distillation from a teacher's top logits.
//
//   p_k = softmax over the row's listed entries of t_k / T     (entries outside the classes, or at -inf, do not count)
//   q_j = softmax over all classes of x_j / T
//   L   = T^2 sum_k p_k (log p_k - log q_{i(k)})
//   dL/dx_j = T (q_j - sum of the p_k with i(k) = j)
//
// With m = max x and S = sum_j exp((x_j - m) / T):  log q_j = (x_j - m) / T - log S.  A row whose entries all drop out
// has loss 0 and gradient 0.  The sums run in f32, where a row's terms are at most 1 and log S is off by some 2^-23 (2^-23 (V / 64
// + 64) at worst); what is done once per row or entry in f64, because the loss is a difference of numbers ten times its size.
// T^2 times that error is what the loss is off by, while the loss of a list that covers the classes stays of the size of their
// scores' variance as T grows: 5e-7 of it at T = 8 (the worst of 200 rows 4e-6), 4e-5 (1e-3) at 100, 5e-3 (5e-2) at 1 000, of 8
// classes, all listed; with f64 sums 2e-8 (6e-8, the answer's rounding).  So above kFlatTemperature S, the entries' weights and
// the listed classes' gradients are f64 (of few long rows S itself is f32 between two kernels).
//
// The row is read once: into registers, where both passes of a softmax and the gradient find it again.  What bounds it is
// the memory: 4 bytes moved per 16-bit class against some 17 instructions per 64 classes of the 32 that its time has room
// for (4 096 rows of 50 001 bf16, loss and gradient: 231 us = 3.6 TB/s; a large copy 4.7).  Streaming stores were 3% faster
// by themselves and are not taken: what reads the gradient next would not find it in the cache.
//
//   k_distill_tiny      at most 32 classes: a lane for each, several rows to a wave
//   k_distill_row       a row held by a wave, 256 or 1 024 threads: loss, gradient or both, one read, one write
//                       (kChunks 0: longer rows, (m, S) online and the loss; k_distill_gradient for what follows)
//   k_distill_stats, k_distill_finish   the same for few long rows, which are divided among workgroups
//   k_distill_gradient  one read, one write, (m, S) given
//   k_distill_flat      loss, gradient or both at temperatures above kFlatTemperature: two or three reads, f64 sums
//   k_distill_flat_stats   in the place of k_distill_stats there, for few long rows
#pragma once

#include "class_common.hpp"

namespace serhip {

constexpr int kDistillThreads = 256;
constexpr int kTinyClasses = 32;     // 16 384 rows of 32: 10 us, a wave for each 17; of 40: 18 and 17
constexpr int kMaxTeacher = 2048;   // entries per row: 3 words each in LDS
constexpr float kFlatTemperature = 8.0f;

struct DistillArgs {
    const void* logits;
    long long n_rows, row_stride;
    int n_classes;
    const void* index;          // [n_rows, n_teacher]
    int index_i64;
    const void* teacher;        // [n_rows, n_teacher]
    int teacher_dtype;
    int n_teacher;
    float temperature;
};

// (m, s) <- (m, s) joined with (m2, s2), where s is relative to 2^(c m)
__device__ __forceinline__ void join_stats(float& m, float& s, float m2, float s2, float c) {
    const float top = fmaxf(m, m2);
    if (top == -INFINITY) {   // nothing but masked classes so far (NaNs keep s a NaN)
        s += s2;
        return;
    }
    // m = -inf comes with s = 0: keep the product 0 * 0, not 0 * NaN
    s = (m == top ? s : s * exp2_fast((m - top) * c)) + (m2 == top ? s2 : s2 * exp2_fast((m2 - top) * c));
    m = top;
}

__device__ __forceinline__ void wave_join(float& m, float& s, float c) {
#pragma unroll
    for (int o = 32; o; o >>= 1) join_stats(m, s, __shfl_xor(m, o), __shfl_xor(s, o), c);
}

// a teacher entry: its logit, or -inf where it does not count
__device__ __forceinline__ float teacher_entry(const DistillArgs& a, long long row, int k, int& cls) {
    const int64_t i = load_index(a.index, a.index_i64, row * a.n_teacher + k);
    const bool inside = i >= 0 && i < a.n_classes;
    cls = inside ? static_cast<int>(i) : -1;
    return inside ? load_float(a.teacher, a.teacher_dtype, row * a.n_teacher + k) : -INFINITY;
}

// one vector into (m, s)
template <int kLen>
__device__ __forceinline__ void add_to_stats(const float (&v)[kLen], float c, float& m, float& s) {
    float top = m;
#pragma unroll
    for (int e = 0; e < kLen; ++e) top = fmaxf(top, v[e]);
    if (top == -INFINITY) {
#pragma unroll
        for (int e = 0; e < kLen; ++e) s += v[e] == -INFINITY ? 0.0f : v[e];   // a NaN
        return;
    }
    if (top > m) {
        s *= exp2_fast((m - top) * c);
        m = top;
    }
    float sum = 0.0f;
#pragma unroll
    for (int e = 0; e < kLen; ++e) sum += exp2_fast((v[e] - m) * c);
    s += sum;
}

// the columns [lo, hi), divided among the workgroup; four vectors in flight
template <int kThreads, typename T>
__device__ __forceinline__ void online_stats(const T* __restrict__ x, int lo, int hi, float c, float& m, float& s) {
    constexpr int kLen = Vec16<T>::kLen, kStep = kThreads * kLen, kFlight = 4;
    int at = lo + static_cast<int>(threadIdx.x) * kLen;
    for (; at + (kFlight - 1) * kStep + kLen <= hi; at += kFlight * kStep) {
        Vec16<T> raw[kFlight];
#pragma unroll
        for (int u = 0; u < kFlight; ++u) raw[u] = load16(x + at + u * kStep);
#pragma unroll
        for (int u = 0; u < kFlight; ++u) {
            float v[kLen];
#pragma unroll
            for (int e = 0; e < kLen; ++e) v[e] = static_cast<float>(raw[u].v[e]);
            add_to_stats(v, c, m, s);
        }
    }
    for (; at < hi; at += kStep) {
        float v[kLen];
        if (at + kLen <= hi) {
            const Vec16<T> raw = load16(x + at);
#pragma unroll
            for (int e = 0; e < kLen; ++e) v[e] = static_cast<float>(raw.v[e]);
        } else {
#pragma unroll
            for (int e = 0; e < kLen; ++e) v[e] = at + e < hi ? static_cast<float>(x[at + e]) : -INFINITY;
        }
        add_to_stats(v, c, m, s);
    }
}

// block = row * splits + split; piece of `cols` columns
template <typename T>
__global__ __launch_bounds__(kDistillThreads) void k_distill_stats(DistillArgs a, int splits, int cols,
                                                                   float2* __restrict__ part) {
    __shared__ float s_m[kDistillThreads / 64], s_s[kDistillThreads / 64];
    const long long row = blockIdx.x / splits;
    const int split = blockIdx.x % splits;
    const float c = 1.44269504f / a.temperature;
    float m = -INFINITY, s = 0.0f;
    online_stats<kDistillThreads>(static_cast<const T*>(a.logits) + row * a.row_stride, split * cols, min(a.n_classes, split * cols + cols), c, m, s);
    wave_join(m, s, c);
    if ((threadIdx.x & 63) == 0) {
        s_m[threadIdx.x >> 6] = m;
        s_s[threadIdx.x >> 6] = s;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
#pragma unroll
        for (int w = 1; w < kDistillThreads / 64; ++w) join_stats(m, s, s_m[w], s_s[w], c);
        part[blockIdx.x] = make_float2(m, s);
    }
}

// An entry's part of a row's loss: its logit, the row's largest and the log of their sum; the student's score of its class, the
// largest and the log of its sum (empty: every class is masked).
__device__ __forceinline__ double entry_loss(double logit, double top, double log_sum, double inv_t, float x, float m, double log_s,
                                             bool empty) {
    const double lp = (logit - top) * inv_t - log_sum, p = exp(lp);
    if (p == 0.0) return 0.0;
    const double lq = empty ? -INFINITY : (static_cast<double>(x) - static_cast<double>(m)) * inv_t - log_s;
    return p * (lp - lq);
}

// Rows of at most kTinyClasses classes: 2^lane_bits lanes for each, a lane for a class, and for every 2^lane_bits-th entry
// of the teacher's list (the first of them in registers: from memory, one entry after the other, 46 080 rows of 8 classes
// and 3 entries take 11 us, 64 rows as long).  An entry's weight goes to its class's lane, a class's score to its entry's.
template <typename T, typename Real>
__global__ __launch_bounds__(kDistillThreads) void k_distill_tiny(DistillArgs a, int lane_bits, const float* __restrict__ weight, float* loss,
                                                                  float2* stats, T* grad, long long grad_stride) {
    const int lanes = 1 << lane_bits, j = threadIdx.x & (lanes - 1), first = (threadIdx.x & 63) - j;
    const long long row = (static_cast<long long>(blockIdx.x) * kDistillThreads + threadIdx.x) >> lane_bits;
    const bool here = row < a.n_rows;   // every lane stays for the shuffles
    const long long r = here ? row : a.n_rows - 1;
    const bool mine = j < a.n_classes;
    const float c = 1.44269504f / a.temperature;
    const double inv_t = 1.0 / static_cast<double>(a.temperature);
    const auto power = [&](float v, float from) -> Real {   // exp((v - from) / T)
        if constexpr (sizeof(Real) == 8) return exp((static_cast<double>(v) - static_cast<double>(from)) * inv_t);
        else return exp2_fast((v - from) * c);
    };
    const float x = mine ? static_cast<float>((static_cast<const T*>(a.logits) + r * a.row_stride)[j]) : -INFINITY;
    int first_cls = -1;
    const float first_t = j < a.n_teacher ? teacher_entry(a, r, j, first_cls) : -INFINITY;
    const auto entry = [&](int k0, int& cls) {   // of this lane, from k0 on
        cls = first_cls;
        if (k0 == 0) return first_t;
        cls = -1;
        return k0 + j < a.n_teacher ? teacher_entry(a, r, k0 + j, cls) : -INFINITY;
    };
    float most = x, top = -INFINITY;
    int cls;
    for (int k0 = 0; k0 < a.n_teacher; k0 += lanes) top = fmaxf(top, entry(k0, cls));
    for (int o = lanes >> 1; o; o >>= 1) {
        most = fmaxf(most, __shfl_xor(most, o));
        top = fmaxf(top, __shfl_xor(top, o));
    }
    const float m = most == -INFINITY ? 0.0f : most;
    const Real e = mine ? power(x, m) : Real(0);
    Real s = e, sum = 0, p = 0;   // of the classes; of the entries; of this class's entries
    for (int k0 = 0; k0 < a.n_teacher; k0 += lanes) {
        const float t = entry(k0, cls);
        const Real w = t == -INFINITY ? Real(0) : power(t, top);
        sum += w;
        const int count = min(lanes, a.n_teacher - k0);
        for (int i = 0; i < count; ++i) {
            const Real other = __shfl(w, first + i);
            p += __shfl(cls, first + i) == j ? other : Real(0);
        }
    }
    for (int o = lanes >> 1; o; o >>= 1) {
        s += __shfl_xor(s, o);
        sum += __shfl_xor(sum, o);
    }
    const bool counts = sum != Real(0);
    if (grad && here && mine) {
        const float w = weight ? weight[row] : 1.0f;
        const Real f = static_cast<Real>(w) * a.temperature;
        const Real g = (s == Real(0) ? Real(0) : f / s) * e - f * (p / sum);
        grad[row * grad_stride + j] = static_cast<T>(static_cast<float>(counts && w != 0.0f ? g : Real(0)));
    }
    if (here && j == 0 && stats) stats[row] = make_float2(most, static_cast<float>(s));
    if (!loss) return;
    const double log_s = log(static_cast<double>(s)), log_sum = log(static_cast<double>(sum));
    double l = 0.0;
    for (int k0 = 0; k0 < a.n_teacher; k0 += lanes) {
        const float t = entry(k0, cls), student = __shfl(x, first + max(cls, 0));
        if (t != -INFINITY) l += entry_loss(t, top, log_sum, inv_t, student, m, log_s, s == Real(0));
    }
    for (int o = lanes >> 1; o; o >>= 1) l += __shfl_xor(l, o);
    if (here && j == 0) loss[row] = counts ? static_cast<float>(l * a.temperature * a.temperature) : 0.0f;
}

// A row's group: a wave (several to a workgroup) or a workgroup.
template <int kGroup>
struct RowGroup {
    static constexpr int kWaves = kGroup / 64;
    static constexpr int kRows = kGroup == 64 ? 4 : 1;             // rows of a workgroup
    static constexpr int kThreads = kGroup * kRows;
    float (&slots)[4][16];   // one set for each reduction of a row, so that one barrier serves it
    int me;
    __device__ __forceinline__ void sync() const {
        if constexpr (kGroup == 64) __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
        else __syncthreads();
    }
    template <typename Op>
    __device__ __forceinline__ float join(float x, int slot, Op op) const {
        if constexpr (kGroup > 64) {
            if ((me & 63) == 0) slots[slot][me >> 6] = x;
            __syncthreads();
            x = slots[slot][0];
#pragma unroll
            for (int w = 1; w < kWaves; ++w) x = op(x, slots[slot][w]);
        }
        return x;
    }
    __device__ __forceinline__ float max(float x, int slot) const {
        return join(wave_max(x), slot, [](float a, float b) { return fmaxf(a, b); });
    }
    __device__ __forceinline__ float sum(float x, int slot) const {
        return join(wave_sum(x), slot, [](float a, float b) { return a + b; });
    }
};

template <int kCap>
struct TeacherShared {
    float p[kCap], x[kCap];   // logit, later weight and at last probability; the student's score of the class
    int cls[kCap];
};

// kChunks vectors of the row for each thread; loss, stats and grad where wanted.
template <typename T, int kGroup, int kChunks, int kCap>
__global__ __launch_bounds__(RowGroup<kGroup>::kThreads, kGroup == 1024 && kChunks <= 8 ? 8 : 4) void k_distill_row(
    DistillArgs a, const float* __restrict__ weight, float* loss, float2* stats, T* grad, long long grad_stride) {
    using G = RowGroup<kGroup>;
    constexpr int kLen = Vec16<T>::kLen;
    __shared__ TeacherShared<kCap> s_teacher[G::kRows];
    __shared__ float s_slots[4][16];
    __shared__ double s_loss[16];
    const int sub = kGroup == 64 ? threadIdx.x >> 6 : 0;
    const G group{s_slots, static_cast<int>(kGroup == 64 ? threadIdx.x & 63 : threadIdx.x)};
    TeacherShared<kCap>& t = s_teacher[sub];
    const int me = group.me, n = a.n_classes;
    const long long row = static_cast<long long>(blockIdx.x) * G::kRows + sub;
    if (row >= a.n_rows) return;
    const float c = 1.44269504f / a.temperature;
    const T* x = static_cast<const T*>(a.logits) + row * a.row_stride;

    // the row: whole vectors, -inf where there are none, and one of the n % kLen scores behind them; the teacher's entries
    const int whole = kChunks ? n / kLen : 0;
    Quad raw[kChunks ? kChunks : 1];
#pragma unroll
    for (int d = 0; d < kChunks; ++d) {
        raw[d] = Quad(minus_infinity_bits<T>());
        if (d * kGroup + me < whole) raw[d] = __builtin_bit_cast(Quad, load16_at(x, (d * kGroup + me) * kLen));
    }
    const int behind = whole * kLen + me;
    const float rest = kChunks && behind < n ? static_cast<float>(x[behind]) : -INFINITY;
    float t_top = -INFINITY;
    for (int k = me; k < a.n_teacher; k += kGroup) {
        int cls;
        const float logit = teacher_entry(a, row, k, cls);
        t.p[k] = logit;
        t.cls[k] = cls;
        t.x[k] = cls >= 0 ? static_cast<float>(x[cls]) : 0.0f;
        t_top = fmaxf(t_top, logit);
    }
    if constexpr (kGroup == 64) group.sync();
    float mine = -INFINITY, s = 0.0f;
    if constexpr (kChunks == 0) online_stats<kGroup>(x, 0, n, c, mine, s);
    // (vector by vector: interleaved by the compiler, eight of them need 130 registers, and one workgroup is all a compute
    // unit takes; at 64 it takes two, and one loads while the other computes)
#pragma unroll
    for (int d = 0; d < kChunks; ++d) {
#pragma unroll
        for (int e = 0; e < kLen; ++e) mine = fmaxf(mine, quad_element<T>(raw[d], e));
        __builtin_amdgcn_sched_barrier(0);
    }
    mine = fmaxf(mine, rest);
    const float most = group.max(mine, 0);
    t_top = group.max(t_top, 1);
    const float m = most == -INFINITY ? 0.0f : most;   // no class left: every 2^(c (x - m)) is 0, and a NaN still shows
    if constexpr (kChunks == 0) s *= exp2_fast((mine - m) * c);
    else s = exp2_fast((rest - m) * c);
#pragma unroll
    for (int d = 0; d < kChunks; ++d) {
        forget(raw[d]);
        float sum = 0.0f;
#pragma unroll
        for (int e = 0; e < kLen; ++e) sum += exp2_fast((quad_element<T>(raw[d], e) - m) * c);
        s += sum;
        __builtin_amdgcn_sched_barrier(0);
    }
    float t_sum = 0.0f;
    for (int k = me; k < a.n_teacher; k += kGroup)
        if (t.p[k] != -INFINITY) t_sum += exp2_fast((t.p[k] - t_top) * c);
    s = group.sum(s, 2);
    t_sum = group.sum(t_sum, 3);   // >= 1, or NaN, where there is any entry
    if (stats && me == 0) stats[row] = make_float2(most, s);
    const bool counts = t_sum != 0.0f;
    const float w = weight ? weight[row] : 1.0f;
    const bool live = counts && w != 0.0f;
    if (kChunks && grad) {
        T* g = grad + row * grad_stride;
        const float f = w * a.temperature, fq = s == 0.0f ? 0.0f : f / s;
        const int me_again = fresh(me);
#pragma unroll
        for (int d = 0; d < kChunks; ++d) {
            forget(raw[d]);
            Vec16<T> y;
#pragma unroll
            for (int e = 0; e < kLen; ++e) y.v[e] = static_cast<T>(fq * exp2_fast((quad_element<T>(raw[d], e) - m) * c));
            if (!live)
#pragma unroll
                for (int e = 0; e < kLen; ++e) y.v[e] = static_cast<T>(0.0f);
            if (d * kGroup + me_again < whole) store16_at(g, (d * kGroup + me_again) * kLen, y);
            __builtin_amdgcn_sched_barrier(0);
        }
        if (behind < n) g[behind] = static_cast<T>(live ? fq * exp2_fast((rest - m) * c) : 0.0f);
        // the classes that the teacher lists, once more with their p: these stores come second
        group.sync();
        if (live) {
            const float inv = 1.0f / t_sum;
            for (int k = me; k < a.n_teacher; k += kGroup) {
                const int cls = t.cls[k];
                if (cls < 0) continue;
                float p = 0.0f;
                for (int i = 0; i < a.n_teacher; ++i)   // a class may be listed twice
                    if (t.cls[i] == cls && t.p[i] != -INFINITY) p += exp2_fast((t.p[i] - t_top) * c);
                g[cls] = static_cast<T>(fq * exp2_fast((t.x[k] - m) * c) - f * (p * inv));
            }
        }
    }
    if (!loss) return;
    double l = 0.0;
    if (counts) {
        const double inv_t = 1.0 / static_cast<double>(a.temperature);
        const double log_s = log(static_cast<double>(s)), log_sum = log(static_cast<double>(t_sum));
        for (int k = me; k < a.n_teacher; k += kGroup)
            if (t.p[k] != -INFINITY) l += entry_loss(t.p[k], t_top, log_sum, inv_t, t.x[k], m, log_s, s == 0.0f);
    }
    l = wave_sum(l);
    if constexpr (kGroup > 64) {
        if (a.n_teacher > 64) {   // more than the first wave had entries
            if ((me & 63) == 0) s_loss[me >> 6] = l;
            __syncthreads();
            l = 0.0;
#pragma unroll
            for (int i = 0; i < G::kWaves; ++i) l += s_loss[i];
        }
    }
    if (me == 0) loss[row] = counts ? static_cast<float>(l * a.temperature * a.temperature) : 0.0f;
}

// one wave per row; Part: float2, or double2 from k_distill_flat_stats
template <typename T, typename Part>
__global__ __launch_bounds__(kDistillThreads) void k_distill_finish(DistillArgs a, int splits, const Part* __restrict__ part,
                                                                    float2* __restrict__ stats, float* __restrict__ loss) {
    const long long row = static_cast<long long>(blockIdx.x) * (kDistillThreads / 64) + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (row >= a.n_rows) return;
    const double inv_t = 1.0 / static_cast<double>(a.temperature);
    float m = -INFINITY;
    decltype(Part::y) s = 0;
    if constexpr (sizeof(Part) == sizeof(float2)) {
        const float c = 1.44269504f / a.temperature;
        for (int i = lane; i < splits; i += 64) {
            const float2 p = part[row * splits + i];
            join_stats(m, s, p.x, p.y, c);
        }
        wave_join(m, s, c);
    } else {
        for (int i = lane; i < splits; i += 64) m = fmaxf(m, static_cast<float>(part[row * splits + i].x));
        m = wave_max(m);
        const double from = m == -INFINITY ? 0.0 : m;   // (a piece of nothing but masked classes has (-inf, 0), or NaN)
        for (int i = lane; i < splits; i += 64) {
            const Part p = part[row * splits + i];
            s += p.y * exp((p.x - from) * inv_t);
        }
        s = wave_sum(s);
    }
    if (lane == 0) stats[row] = make_float2(m, static_cast<float>(s));

    float top = -INFINITY;
    int cls, any = 0;
    for (int k = lane; k < a.n_teacher; k += 64) {
        const float t = teacher_entry(a, row, k, cls);
        top = fmaxf(top, t);
        any |= t > -INFINITY || t != t;
    }
    top = wave_max(top);
    double sum = 0.0;
    for (int k = lane; k < a.n_teacher; k += 64) {
        const float t = teacher_entry(a, row, k, cls);
        if (t != -INFINITY) sum += exp((static_cast<double>(t) - top) * inv_t);
    }
    sum = wave_sum(sum);
    const double log_sum = log(sum), log_s = log(static_cast<double>(s));
    const T* x = static_cast<const T*>(a.logits) + row * a.row_stride;
    double l = 0.0;
    for (int k = lane; k < a.n_teacher; k += 64) {
        const float t = teacher_entry(a, row, k, cls);
        if (t == -INFINITY) continue;
        const double lp = (static_cast<double>(t) - top) * inv_t - log_sum;
        const double p = exp(lp);
        if (p == 0.0) continue;
        const double lq = m == -INFINITY && s == 0 ? -INFINITY : (static_cast<double>(static_cast<float>(x[cls])) - m) * inv_t - log_s;
        l += p * (lp - lq);
    }
    l = wave_sum(l);
    const bool counts = __any(any);
    if (lane == 0) loss[row] = counts ? static_cast<float>(l * a.temperature * a.temperature) : 0.0f;
}

// block = row * splits + split.  weight: what arrives from above for the row's loss (NULL: 1); a row of weight 0, and
// a row without teacher entries, gets zeros whatever its logits hold.  `grad` may be the logits themselves.  Real: what the
// listed classes are held in.
template <typename T, typename Real>
__global__ __launch_bounds__(kDistillThreads) void k_distill_gradient(DistillArgs a, int splits, int cols,
                                                                      const float2* __restrict__ stats,
                                                                      const float* __restrict__ weight, T* grad,
                                                                      long long grad_stride) {
    constexpr int kLen = Vec16<T>::kLen;
    __shared__ Real s_p[kMaxTeacher], s_red[kDistillThreads / 64];
    __shared__ float s_x[kMaxTeacher];
    __shared__ int s_cls[kMaxTeacher];
    const long long row = blockIdx.x / splits;
    const int split = blockIdx.x % splits;
    const int lo = split * cols, hi = min(a.n_classes, lo + cols);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const float c = 1.44269504f / a.temperature;
    const T* x = static_cast<const T*>(a.logits) + row * a.row_stride;
    T* g = grad + row * grad_stride;
    const float w = weight ? weight[row] : 1.0f;

    float top = -INFINITY;
    int any = 0;
    for (int k = threadIdx.x; k < a.n_teacher; k += kDistillThreads) {
        int cls;
        const float t = teacher_entry(a, row, k, cls);
        s_p[k] = t;
        s_cls[k] = cls;
        s_x[k] = cls >= lo && cls < hi ? static_cast<float>(x[cls]) : 0.0f;
        top = fmaxf(top, t);
        any |= t > -INFINITY || t != t;
    }
    top = wave_max(top);
    if (lane == 0) s_red[wave] = top;
    const bool counts = __syncthreads_or(any);
    if (!counts || w == 0.0f) {
        for (int at = lo + threadIdx.x * kLen; at < hi; at += kDistillThreads * kLen) {
            Vec16<T> y = {};
            if (at + kLen <= hi) store16(g + at, y);
            else
                for (int e = 0; at + e < hi; ++e) g[at + e] = y.v[0];
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < kDistillThreads / 64; ++i) top = fmaxf(top, static_cast<float>(s_red[i]));
    const auto power = [&](Real v, float from) -> Real {   // exp((v - from) / T)
        if constexpr (sizeof(Real) == 8) return exp((v - from) / a.temperature);
        else return exp2_fast((v - from) * c);
    };
    Real sum = 0;
    for (int k = threadIdx.x; k < a.n_teacher; k += kDistillThreads) {
        const Real p = s_p[k] == -INFINITY ? Real(0) : power(s_p[k], top);
        s_p[k] = p;
        sum += p;
    }
    sum = wave_sum(sum);
    __syncthreads();
    if (lane == 0) s_red[wave] = sum;
    __syncthreads();
    sum = 0;
#pragma unroll
    for (int i = 0; i < kDistillThreads / 64; ++i) sum += s_red[i];

    const float2 st = stats[row];
    const float m = st.x == -INFINITY ? 0.0f : st.x;   // no class left: q = 0 (or NaN, through fq)
    const float f = w * a.temperature, fq = st.y == 0.0f ? 0.0f : f / st.y;
    for (int at = lo + threadIdx.x * kLen; at < hi; at += kDistillThreads * kLen) {
        if (at + kLen <= hi) {
            Vec16<T> y = load16(x + at);
#pragma unroll
            for (int e = 0; e < kLen; ++e)
                y.v[e] = static_cast<T>(fq * exp2_fast((static_cast<float>(y.v[e]) - m) * c));
            store16(g + at, y);
        } else {
            for (int e = 0; at + e < hi; ++e)
                g[at + e] = static_cast<T>(fq * exp2_fast((static_cast<float>(x[at + e]) - m) * c));
        }
    }
    // the classes that the teacher lists, once more with their p: after the barrier these stores come second
    __syncthreads();
    const Real inv = Real(1) / sum, real_f = static_cast<Real>(w) * a.temperature, real_fq = st.y == 0.0f ? Real(0) : real_f / st.y;
    for (int k = threadIdx.x; k < a.n_teacher; k += kDistillThreads) {
        const int cls = s_cls[k];
        if (cls < lo || cls >= hi) continue;
        Real p = 0;
        for (int i = 0; i < a.n_teacher; ++i) p += s_cls[i] == cls ? s_p[i] : Real(0);   // a class may be listed twice
        const Real q = real_fq * power(s_x[k], m);
        g[cls] = static_cast<T>(static_cast<float>(q - real_f * (p * inv)));
    }
}

// Temperatures above kFlatTemperature: a workgroup for each row, which is read for its largest score, for S in f64 and, where
// the gradient is wanted, once more.  q of the classes that the teacher does not list is nothing's difference and stays f32.
// An f64 exponential for each class is what bounds it (4 096 rows of 50 001 bf16, loss and gradient: 352 us, by k_distill_row
// 233).  Up to kFlatShort classes by 256 threads (2 048 rows of 2 048 bf16: 20 us, by 1 024: 32; of 8 192: 39 and 44, but 64 of
// 8 192: 10.1 and 9.0, of 16 384: 15.4 and 11.9), up to kFlatWave by a wave (4 096 rows of 40: 28.3, by 256 29.2; of 512:
// 32.2 and 33.3 -- and a launch has room for four times as many rows).
constexpr int kFlatWave = 512, kFlatShort = 4096;
// Fewer than 64 rows of more than kFlatWhole classes are divided among workgroups, as f32 sums are (8 rows of 131 072 bf16: 15
// us, by a workgroup each 48; of 50 001: 15 and 27; 63 of 20 001: 17.3 and 16.4).  Their gradient is k_distill_gradient's, which
// gets S rounded to f32: off by 2^-24 T q where the teacher lists a class, which is why it is not done where time allows.
constexpr int kFlatWhole = 65536;
template <typename T, int kThreads>
__global__ __launch_bounds__(kThreads) void k_distill_flat(DistillArgs a, const float* __restrict__ weight, float* loss, float2* stats,
                                                           T* grad, long long grad_stride) {
    constexpr int kLen = Vec16<T>::kLen, kWaves = kThreads / 64;
    __shared__ double s_p[kMaxTeacher], s_sum[kWaves];   // an entry's weight, 0 where it does not count
    __shared__ float s_t[kMaxTeacher], s_x[kMaxTeacher], s_max[2][kWaves];
    __shared__ int s_cls[kMaxTeacher];
    const long long row = blockIdx.x;
    const int n = a.n_classes, me = threadIdx.x, lane = me & 63, wave = me >> 6;
    const double inv_t = 1.0 / static_cast<double>(a.temperature);
    const T* x = static_cast<const T*>(a.logits) + row * a.row_stride;
    const auto each = [&](auto f) {   // f(first class, its vector, how many of it there are)
#pragma unroll 1
        for (int at = me * kLen; at < n; at += kThreads * kLen) {
            Vec16<T> v;
            const int len = min(kLen, n - at);
            if (len == kLen) {
                v = load16(x + at);
            } else {
#pragma unroll
                for (int e = 0; e < kLen; ++e) v.v[e] = e < len ? x[at + e] : static_cast<T>(-INFINITY);
            }
            f(at, v, len);
        }
    };
    const auto total = [&](double v) {   // over the workgroup
        v = wave_sum(v);
        __syncthreads();
        if (lane == 0) s_sum[wave] = v;
        __syncthreads();
        double sum = 0.0;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) sum += s_sum[w];
        return sum;
    };

    float most = -INFINITY, top = -INFINITY;
    each([&](int, const Vec16<T>& v, int) {
#pragma unroll
        for (int e = 0; e < kLen; ++e) most = fmaxf(most, static_cast<float>(v.v[e]));
    });
    for (int k = me; k < a.n_teacher; k += kThreads) {
        int cls;
        const float t = teacher_entry(a, row, k, cls);
        s_t[k] = t;
        s_cls[k] = cls;
        s_x[k] = cls >= 0 ? static_cast<float>(x[cls]) : 0.0f;
        top = fmaxf(top, t);
    }
    most = wave_max(most);
    top = wave_max(top);
    if (lane == 0) {
        s_max[0][wave] = most;
        s_max[1][wave] = top;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        most = fmaxf(most, s_max[0][w]);
        top = fmaxf(top, s_max[1][w]);
    }
    const float m = most == -INFINITY ? 0.0f : most;   // no class left: every weight is 0, and a NaN still shows
    double s = 0.0, t_sum = 0.0;
    each([&](int, const Vec16<T>& v, int) {
#pragma unroll
        for (int e = 0; e < kLen; ++e) s += exp((static_cast<double>(static_cast<float>(v.v[e])) - m) * inv_t);
    });
    for (int k = me; k < a.n_teacher; k += kThreads) {
        s_p[k] = s_t[k] == -INFINITY ? 0.0 : exp((static_cast<double>(s_t[k]) - top) * inv_t);
        t_sum += s_p[k];
    }
    s = total(s);
    t_sum = total(t_sum);   // >= 1, or NaN, where there is any entry
    if (stats && me == 0) stats[row] = make_float2(most, static_cast<float>(s));
    const bool counts = t_sum != 0.0;
    if (grad) {
        const float w = weight ? weight[row] : 1.0f;
        const bool live = counts && w != 0.0f;
        const double f = static_cast<double>(w) * a.temperature, fq = s == 0.0 ? 0.0 : f / s;
        const float c = 1.44269504f / a.temperature, fq_short = static_cast<float>(fq);
        T* g = grad + row * grad_stride;
        each([&](int at, const Vec16<T>& v, int len) {
            Vec16<T> y;
#pragma unroll
            for (int e = 0; e < kLen; ++e)
                y.v[e] = static_cast<T>(live ? fq_short * exp2_fast((static_cast<float>(v.v[e]) - m) * c) : 0.0f);
            if (len == kLen) {
                store16(g + at, y);
            } else {
#pragma unroll
                for (int e = 0; e < kLen; ++e)
                    if (e < len) g[at + e] = y.v[e];
            }
        });
        // the classes that the teacher lists, once more with their p: after the barrier these stores come second
        __syncthreads();
        if (live) {
            for (int k = me; k < a.n_teacher; k += kThreads) {
                const int cls = s_cls[k];
                if (cls < 0) continue;
                double p = 0.0;
                for (int i = 0; i < a.n_teacher; ++i) p += s_cls[i] == cls ? s_p[i] : 0.0;   // a class may be listed twice
                g[cls] = static_cast<T>(static_cast<float>(fq * exp((static_cast<double>(s_x[k]) - m) * inv_t) - f * (p / t_sum)));
            }
        }
    }
    if (!loss) return;
    double l = 0.0;
    const double log_s = log(s), log_sum = log(t_sum);
    for (int k = me; k < a.n_teacher; k += kThreads)
        if (s_t[k] != -INFINITY) l += entry_loss(s_t[k], top, log_sum, inv_t, s_x[k], m, log_s, s == 0.0);
    l = total(l);
    if (me == 0) loss[row] = counts ? static_cast<float>(l * a.temperature * a.temperature) : 0.0f;
}

// (m, S) of a piece of `cols` columns: block = row * splits + split.  The piece is read twice, the second time from cache.
template <typename T>
__global__ __launch_bounds__(kDistillThreads) void k_distill_flat_stats(DistillArgs a, int splits, int cols, double2* __restrict__ part) {
    constexpr int kLen = Vec16<T>::kLen, kWaves = kDistillThreads / 64;
    __shared__ float s_max[kWaves];
    __shared__ double s_sum[kWaves];
    const long long row = blockIdx.x / splits;
    const int split = blockIdx.x % splits, lo = split * cols, hi = min(a.n_classes, lo + cols);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const double inv_t = 1.0 / static_cast<double>(a.temperature);
    const T* x = static_cast<const T*>(a.logits) + row * a.row_stride;
    const auto each = [&](auto f) {   // f(score)
#pragma unroll 1
        for (int at = lo + static_cast<int>(threadIdx.x) * kLen; at < hi; at += kDistillThreads * kLen) {
            if (at + kLen <= hi) {
                const Vec16<T> v = load16(x + at);
#pragma unroll
                for (int e = 0; e < kLen; ++e) f(static_cast<float>(v.v[e]));
            } else {
                for (int e = 0; at + e < hi; ++e) f(static_cast<float>(x[at + e]));
            }
        }
    };
    float m = -INFINITY;
    each([&](float v) { m = fmaxf(m, v); });
    m = wave_max(m);
    if (lane == 0) s_max[wave] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) m = fmaxf(m, s_max[w]);
    const double from = m == -INFINITY ? 0.0 : m;
    double s = 0.0;
    each([&](float v) { s += exp((v - from) * inv_t); });
    s = wave_sum(s);
    if (lane == 0) s_sum[wave] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
#pragma unroll
        for (int w = 1; w < kWaves; ++w) s += s_sum[w];
        part[blockIdx.x] = make_double2(m, s);
    }
}

}  // namespace serhip
