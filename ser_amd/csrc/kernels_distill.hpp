// Distillation from a teacher's top logits.
//
//   p_k = softmax over the row's listed entries of t_k / T     (entries outside the classes, or at -inf, do not count)
//   q_j = softmax over all classes of x_j / T
//   L   = T^2 sum_k p_k (log p_k - log q_{i(k)})
//   dL/dx_j = T (q_j - sum of the p_k with i(k) = j)
//
// With m = max x and S = sum_j exp((x_j - m) / T):  log q_j = (x_j - m) / T - log S.  A row whose entries all drop out
// has loss 0 and gradient 0.  The sums run in f32 (a row's terms are <= 1 and there is no cancellation), what is done
// once per row or entry in f64, because the loss is a difference of numbers ten times its size.
//
// The row is read once: into registers, where both passes of a softmax and the gradient find it again.  What bounds it is
// the memory: 4 bytes moved per 16-bit class against some 17 instructions per 64 classes of the 32 that its time has room
// for (4 096 rows of 50 001 bf16, loss and gradient: 229 us = 3.6 TB/s; a large copy 4.7).  Streaming stores were 3% faster
// by themselves and are not taken: what reads the gradient next would not find it in the cache.
//
//   k_distill_tiny      at most 32 classes: a lane for each, several rows to a wave
//   k_distill_row       a row held by a wave, 256 or 1 024 threads: loss, gradient or both, one read, one write
//                       (kChunks 0: longer rows, (m, S) online and the loss; k_distill_gradient for what follows)
//   k_distill_stats, k_distill_finish   the same for few long rows, which are divided among workgroups
//   k_distill_gradient  one read, one write, (m, S) given
#pragma once

#include "class_common.hpp"

namespace serhip {

constexpr int kDistillThreads = 256;
constexpr int kTinyClasses = 32;     // 16 384 rows of 32: 10 us, a wave for each 17; of 40: 18 and 17
constexpr int kMaxTeacher = 2048;   // entries per row: 3 words each in LDS

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
template <typename T>
__global__ __launch_bounds__(kDistillThreads) void k_distill_tiny(DistillArgs a, int lane_bits, const float* __restrict__ weight, float* loss,
                                                                  float2* stats, T* grad, long long grad_stride) {
    const int lanes = 1 << lane_bits, j = threadIdx.x & (lanes - 1), first = (threadIdx.x & 63) - j;
    const long long row = (static_cast<long long>(blockIdx.x) * kDistillThreads + threadIdx.x) >> lane_bits;
    const bool here = row < a.n_rows;   // every lane stays for the shuffles
    const long long r = here ? row : a.n_rows - 1;
    const bool mine = j < a.n_classes;
    const float c = 1.44269504f / a.temperature;
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
    const float m = most == -INFINITY ? 0.0f : most, e = mine ? exp2_fast((x - m) * c) : 0.0f;
    float s = e, sum = 0.0f, p = 0.0f;   // of the classes; of the entries; of this class's entries
    for (int k0 = 0; k0 < a.n_teacher; k0 += lanes) {
        const float t = entry(k0, cls), w = t == -INFINITY ? 0.0f : exp2_fast((t - top) * c);
        sum += w;
        const int count = min(lanes, a.n_teacher - k0);
        for (int i = 0; i < count; ++i) {
            const float other = __shfl(w, first + i);
            p += __shfl(cls, first + i) == j ? other : 0.0f;
        }
    }
    for (int o = lanes >> 1; o; o >>= 1) {
        s += __shfl_xor(s, o);
        sum += __shfl_xor(sum, o);
    }
    const bool counts = sum != 0.0f;
    if (grad && here && mine) {
        const float w = weight ? weight[row] : 1.0f, f = w * a.temperature;
        const float g = (s == 0.0f ? 0.0f : f / s) * e - f * (p / sum);
        grad[row * grad_stride + j] = static_cast<T>(counts && w != 0.0f ? g : 0.0f);
    }
    if (here && j == 0 && stats) stats[row] = make_float2(most, s);
    if (!loss) return;
    const double inv_t = 1.0 / static_cast<double>(a.temperature);
    const double log_s = log(static_cast<double>(s)), log_sum = log(static_cast<double>(sum));
    double l = 0.0;
    for (int k0 = 0; k0 < a.n_teacher; k0 += lanes) {
        const float t = entry(k0, cls), student = __shfl(x, first + max(cls, 0));
        if (t != -INFINITY) l += entry_loss(t, top, log_sum, inv_t, student, m, log_s, s == 0.0f);
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

// one wave per row
template <typename T>
__global__ __launch_bounds__(kDistillThreads) void k_distill_finish(DistillArgs a, int splits, const float2* __restrict__ part,
                                                                    float2* __restrict__ stats, float* __restrict__ loss) {
    const long long row = static_cast<long long>(blockIdx.x) * (kDistillThreads / 64) + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (row >= a.n_rows) return;
    const float c = 1.44269504f / a.temperature;
    float m = -INFINITY, s = 0.0f;
    for (int i = lane; i < splits; i += 64) {
        const float2 p = part[row * splits + i];
        join_stats(m, s, p.x, p.y, c);
    }
    wave_join(m, s, c);
    if (lane == 0) stats[row] = make_float2(m, s);

    const double inv_t = 1.0 / static_cast<double>(a.temperature);
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
        const double lq = m == -INFINITY && s == 0.0f ? -INFINITY : (static_cast<double>(static_cast<float>(x[cls])) - m) * inv_t - log_s;
        l += p * (lp - lq);
    }
    l = wave_sum(l);
    const bool counts = __any(any);
    if (lane == 0) loss[row] = counts ? static_cast<float>(l * a.temperature * a.temperature) : 0.0f;
}

// block = row * splits + split.  weight: what arrives from above for the row's loss (NULL: 1); a row of weight 0, and
// a row without teacher entries, gets zeros whatever its logits hold.  `grad` may be the logits themselves.
template <typename T>
__global__ __launch_bounds__(kDistillThreads) void k_distill_gradient(DistillArgs a, int splits, int cols,
                                                                      const float2* __restrict__ stats,
                                                                      const float* __restrict__ weight, T* grad,
                                                                      long long grad_stride) {
    constexpr int kLen = Vec16<T>::kLen;
    __shared__ float s_p[kMaxTeacher], s_x[kMaxTeacher];
    __shared__ int s_cls[kMaxTeacher];
    __shared__ float s_red[kDistillThreads / 64];
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
    for (int i = 0; i < kDistillThreads / 64; ++i) top = fmaxf(top, s_red[i]);
    float sum = 0.0f;
    for (int k = threadIdx.x; k < a.n_teacher; k += kDistillThreads) {
        const float p = s_p[k] == -INFINITY ? 0.0f : exp2_fast((s_p[k] - top) * c);
        s_p[k] = p;
        sum += p;
    }
    sum = wave_sum(sum);
    __syncthreads();
    if (lane == 0) s_red[wave] = sum;
    __syncthreads();
    sum = 0.0f;
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
    const float inv = 1.0f / sum;
    for (int k = threadIdx.x; k < a.n_teacher; k += kDistillThreads) {
        const int cls = s_cls[k];
        if (cls < lo || cls >= hi) continue;
        float p = 0.0f;
        for (int i = 0; i < a.n_teacher; ++i) p += s_cls[i] == cls ? s_p[i] : 0.0f;   // a class may be listed twice
        const float q = fq * exp2_fast((s_x[k] - m) * c);
        g[cls] = static_cast<T>(q - f * (p * inv));
    }
}

}  // namespace serhip
