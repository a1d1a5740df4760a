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
//   k_distill_stats     (m, S) of a piece of a row, one read, online
//   k_distill_finish    pieces joined; the loss
//   k_distill_gradient  one read, one write
#pragma once

#include "class_common.hpp"

namespace serhip {

constexpr int kDistillThreads = 256;
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

// this thread's columns [lo, hi) step 256 vectors
template <typename T>
__device__ __forceinline__ void online_stats(const T* __restrict__ x, int lo, int hi, float c, float& m, float& s) {
    constexpr int kLen = Vec16<T>::kLen;
    for (int at = lo + threadIdx.x * kLen; at < hi; at += kDistillThreads * kLen) {
        float v[kLen];
        if (at + kLen <= hi) {
            const Vec16<T> raw = load16(x + at);
#pragma unroll
            for (int e = 0; e < kLen; ++e) v[e] = static_cast<float>(raw.v[e]);
        } else {
#pragma unroll
            for (int e = 0; e < kLen; ++e) v[e] = at + e < hi ? static_cast<float>(x[at + e]) : -INFINITY;
        }
        float top = m;
#pragma unroll
        for (int e = 0; e < kLen; ++e) top = fmaxf(top, v[e]);
        if (top == -INFINITY) {
#pragma unroll
            for (int e = 0; e < kLen; ++e) s += v[e] == -INFINITY ? 0.0f : v[e];   // a NaN
            continue;
        }
        if (top > m) {
            s *= exp2_fast((m - top) * c);
            m = top;
        }
#pragma unroll
        for (int e = 0; e < kLen; ++e) s += exp2_fast((v[e] - m) * c);
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
    online_stats(static_cast<const T*>(a.logits) + row * a.row_stride, split * cols, min(a.n_classes, split * cols + cols), c, m, s);
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
    const float m = st.x;
    const float f = w * a.temperature, fq = st.y == 0.0f ? 0.0f : f / st.y;
    const bool masked = m == -INFINITY;   // no class left: q = 0 (or NaN, through fq)
    for (int at = lo + threadIdx.x * kLen; at < hi; at += kDistillThreads * kLen) {
        if (at + kLen <= hi) {
            Vec16<T> y = load16(x + at);
#pragma unroll
            for (int e = 0; e < kLen; ++e)
                y.v[e] = static_cast<T>(masked ? 0.0f * fq : fq * exp2_fast((static_cast<float>(y.v[e]) - m) * c));
            store16(g + at, y);
        } else {
            for (int e = 0; at + e < hi; ++e)
                g[at + e] = static_cast<T>(masked ? 0.0f * fq : fq * exp2_fast((static_cast<float>(x[at + e]) - m) * c));
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
        const float q = masked ? 0.0f * fq : fq * exp2_fast((s_x[k] - m) * c);
        g[cls] = static_cast<T>(q - f * (p * inv));
    }
}

}  // namespace serhip
