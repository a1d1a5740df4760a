// C entry points of the class / vocabulary operators (include/serhip.h): argument checks, division of the work,
// launches.  A unit of its own: it is compiled without packed f32 instructions, which the FFT unit (serhip.hip) is
// built on.  The calls keep nothing in the context but its device: scratch comes from the caller, so calls on
// different streams and captured graphs share no memory.
#include "../../include/serhip.h"

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <exception>
#include <string>
#include <type_traits>

#include "kernels_distill.hpp"
#include "kernels_embed.hpp"
#include "kernels_sample.hpp"
#include "status.hpp"

using namespace serhip;

namespace {

#define CLASS_TRY(expr)                                                                          \
    do {                                                                                         \
        hipError_t e_ = (expr);                                                                  \
        if (e_ != hipSuccess) return set_error(SERHIP_E_HIP, std::string(#expr) + ": " + hipGetErrorString(e_)); \
    } while (0)

int invalid(const char* entry, const char* what) { return set_error(SERHIP_E_INVALID, std::string(entry) + ": " + what); }
int unsupported(const char* entry, const char* what) {
    return set_error(SERHIP_E_UNSUPPORTED, std::string(entry) + ": " + what);
}

// no exception leaves the library (std::string may throw while a message is put together)
template <typename F>
int guarded(F f) noexcept {
    try {
        return f();
    } catch (const std::exception&) {
        return SERHIP_E_NOMEM;
    } catch (...) {
        return SERHIP_E_HIP;
    }
}

constexpr int64_t kMaxThreads = (static_cast<int64_t>(1) << 32) - 1;   // of a launch

size_t round_up(size_t v, size_t a) { return (v + a - 1) / a * a; }
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
int round_up_log2(int64_t v) {
    int b = 0;
    while ((int64_t{1} << b) < v) ++b;
    return b;
}
int element_size(int dtype) { return dtype == SERHIP_DTYPE_F32 ? 4 : 2; }
bool known_dtype(int dtype) { return dtype >= SERHIP_DTYPE_F32 && dtype <= SERHIP_DTYPE_F16; }
bool aligned_to(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

// calls f with a value of the element type
template <typename F>
void with_type(int dtype, F f) {
    if (dtype == SERHIP_DTYPE_F32) f(float{});
    else if (dtype == SERHIP_DTYPE_BF16) f(bf16_t{});
    else f(f16_t{});
}

// ------------------------------------------------------------------------------------------ distillation
// A row is cut into pieces until there are four workgroups per compute unit of an MI355X (256), but a piece is at
// least one vector per thread.
// Rows too long for registers: one workgroup's, if there are 64 rows or they have at most 16 384 vectors (loss and gradient,
// f32: 8 rows of 50 001 11 us, in pieces 13; 64 of 131 072 26 and 27, 200 of them 53 and 60; but 8 of them 16 and 15).
constexpr int64_t kWholeRows = 64, kWholeVectors = 16384;
// A wave takes a row if there are this many of them (4 096 rows of 512 bf16 classes: 9 us, with 256 threads each 21; 512
// rows of 2 048: 7.1 and 6.7; 64 of them: 7.3 and 6.0).
constexpr int64_t kWaveRows = 512;
constexpr int kWaveTeacher = 256;   // entries whose list fits a wave's part of the LDS
struct DistillSplit {
    int splits, cols;
};
DistillSplit distill_split(int64_t n_rows, int64_t n_classes, int dtype) {
    const int64_t unit = kDistillThreads * (16 / element_size(dtype));
    const int64_t units = ceil_div(n_classes, unit);
    const int64_t want = std::min<int64_t>(units, std::max<int64_t>(1, 1024 / std::max<int64_t>(n_rows, 1)));
    const int64_t cols = ceil_div(units, want) * unit;
    return {static_cast<int>(ceil_div(n_classes, cols)), static_cast<int>(cols)};
}

int check_distill(const char* entry, const serhip_ctx* ctx, const DistillArgs& a, int64_t n_classes, int dtype) {
    if (!ctx) return invalid(entry, "ctx is NULL");
    if (!known_dtype(dtype) || !known_dtype(a.teacher_dtype)) return invalid(entry, "unknown element type");
    if (a.n_rows < 0) return invalid(entry, "n_rows < 0");
    if (n_classes < 1 || n_classes > SERHIP_MAX_CLASSES) return invalid(entry, "n_classes must be 1..SERHIP_MAX_CLASSES");
    if (a.row_stride < 0) return invalid(entry, "a row stride is negative");
    if (a.n_teacher < 1) return invalid(entry, "n_teacher must be at least 1");
    if (a.n_teacher > kMaxTeacher) return unsupported(entry, "more than 2048 teacher entries per row");
    if (!(a.temperature >= 1e-3f && a.temperature <= 1e3f)) return invalid(entry, "temperature must be 1e-3..1e3");
    if (a.n_rows > 0) {
        if (!a.logits || !a.index || !a.teacher) return invalid(entry, "NULL argument");
        if (!aligned_to(a.logits, element_size(dtype)) || !aligned_to(a.teacher, element_size(a.teacher_dtype)) ||
            !aligned_to(a.index, a.index_i64 ? 8 : 4))
            return invalid(entry, "a pointer is not aligned to its element type");
        // threads for a row: a lane for each of few classes, a wave (of so many rows it takes up to 64 classes whatever their
        // type, if the list of entries fits with it); a workgroup, or those of its pieces
        const bool wave = n_classes <= kTinyClasses || (n_classes <= 64 && a.n_teacher <= kWaveTeacher);
        const int64_t threads = wave ? 64 : n_classes <= 64 ? kDistillThreads : std::max(1024, distill_split(a.n_rows, n_classes, dtype).splits * kDistillThreads);
        if (a.n_rows > kMaxThreads / threads - kDistillThreads) return unsupported(entry, "too many rows per call");
    }
    return SERHIP_OK;
}

int check_gradient_out(const char* entry, const DistillArgs& a, const void* grad, int64_t grad_stride, int dtype) {
    if (a.n_rows > 0 && !grad) return invalid(entry, "NULL argument");
    if (!aligned_to(grad, element_size(dtype))) return invalid(entry, "a pointer is not aligned to its element type");
    if (a.n_rows > 1 && grad_stride < a.n_classes) return invalid(entry, "rows of the gradient overlap");
    if (grad == a.logits && grad_stride != a.row_stride && a.n_rows > 1)
        return invalid(entry, "a gradient in place of the logits has their row stride");
    return SERHIP_OK;
}

struct DistillScratch {
    size_t stats, part, total;
};
DistillScratch distill_scratch(int64_t n_rows, int64_t n_classes, int dtype) {
    const size_t stats = round_up(static_cast<size_t>(n_rows) * sizeof(float2), 256);
    const size_t part = round_up(static_cast<size_t>(n_rows) * distill_split(n_rows, n_classes, dtype).splits * sizeof(double2), 256);
    return {0, stats, stats + part};
}

// a wave for a row up to 256 vectors (four rows to a workgroup, no barriers), where its list of entries fits with it
template <typename T>
bool is_wave_row(const DistillArgs& a) {
    return a.n_rows >= kWaveRows && a.n_teacher <= kWaveTeacher && ceil_div(a.n_classes, Vec16<T>::kLen) <= 256;
}

// Rows of more than 8 192 vectors are held, one workgroup to a compute unit, for loss and gradient of this many rows (1 024
// rows of 131 072 bf16: 133 us, in two kernels 160; 200: 29 and 32; 64: 23 and 21; the loss alone of 1 024: 69 and 46).
constexpr int64_t kLongHeldRows = 128;
// What holds a row in registers: threads for it and 16-byte vectors for each; false: nothing does.  (2 048 rows of 4 096 bf16
// classes with 256 threads: 15 us, with 1 024: 44; of 16 384: 31 and 46; 64 of these: 7.7 and 9.0.)
template <typename T, typename F>
bool with_row_form(const DistillArgs& a, bool gradient, F f) {
    const int64_t vectors = ceil_div(a.n_classes, Vec16<T>::kLen);
    const auto form = [&](auto group, auto chunks, auto cap) {
        f(group, chunks, cap);
        return true;
    };
    using std::integral_constant;
    if (is_wave_row<T>(a)) {
        constexpr integral_constant<int, 64> wave;
        constexpr integral_constant<int, kWaveTeacher> cap;
        if (vectors <= 64) return form(wave, integral_constant<int, 1>{}, cap);
        if (vectors <= 128) return form(wave, integral_constant<int, 2>{}, cap);
        return form(wave, integral_constant<int, 4>{}, cap);
    }
    constexpr integral_constant<int, kMaxTeacher> cap;
    if (vectors <= 256 * 2) return form(integral_constant<int, 256>{}, integral_constant<int, 2>{}, cap);
    if (vectors <= 256 * 4) return form(integral_constant<int, 256>{}, integral_constant<int, 4>{}, cap);
    if (vectors <= 256 * 8) return form(integral_constant<int, 256>{}, integral_constant<int, 8>{}, cap);
    if (vectors <= 1024 * 4) return form(integral_constant<int, 1024>{}, integral_constant<int, 4>{}, cap);
    if (vectors <= 1024 * 8) return form(integral_constant<int, 1024>{}, integral_constant<int, 8>{}, cap);
    if (a.n_rows < kLongHeldRows || !gradient) return false;
    if (vectors <= 1024 * 12) return form(integral_constant<int, 1024>{}, integral_constant<int, 12>{}, cap);
    if (vectors <= 1024 * 16) return form(integral_constant<int, 1024>{}, integral_constant<int, 16>{}, cap);
    return false;
}

bool is_flat_split(const DistillArgs& a) {
    return a.temperature > kFlatTemperature && a.n_rows < kWholeRows && a.n_classes > kFlatWhole;
}

// loss and stats, and the gradient too where one kernel has both; true if it has
template <typename T>
bool launch_rows(const DistillArgs& a, const float* weight, void* part, float2* stats, float* loss, T* grad, int64_t grad_stride,
                 hipStream_t stream) {
    const long long gs = grad_stride;
    float2* const kept = grad ? nullptr : stats;   // of a kernel that writes the gradient too nothing reads them
    if (a.n_classes <= kTinyClasses) {
        const int bits = round_up_log2(a.n_classes);
        const dim3 grid(static_cast<unsigned>(ceil_div(a.n_rows << bits, kDistillThreads)));
        hipLaunchKernelGGL((a.temperature > kFlatTemperature ? k_distill_tiny<T, double> : k_distill_tiny<T, float>), grid, dim3(kDistillThreads), 0,
                           stream, a, bits, weight, loss, kept, grad, gs);
        return true;
    }
    const DistillSplit sp = distill_split(a.n_rows, a.n_classes, sizeof(T) == 4 ? SERHIP_DTYPE_F32 : SERHIP_DTYPE_BF16);
    const dim3 pieces(static_cast<unsigned>(a.n_rows * sp.splits)), joins(static_cast<unsigned>(ceil_div(a.n_rows, kDistillThreads / 64)));
    if (is_flat_split(a)) {
        double2* flat_part = static_cast<double2*>(part);
        hipLaunchKernelGGL(k_distill_flat_stats<T>, pieces, dim3(kDistillThreads), 0, stream, a, sp.splits, sp.cols, flat_part);
        hipLaunchKernelGGL((k_distill_finish<T, double2>), joins, dim3(kDistillThreads), 0, stream, a, sp.splits, flat_part, stats, loss);
        return false;
    }
    if (a.temperature > kFlatTemperature) {
        const auto launch = [&](auto kernel, unsigned threads) {
            hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(a.n_rows)), dim3(threads), 0, stream, a, weight, loss, kept, grad, gs);
        };
        if (a.n_classes <= kFlatWave) launch(k_distill_flat<T, 64>, 64);
        else if (a.n_classes <= kFlatShort) launch(k_distill_flat<T, 256>, 256);
        else launch(k_distill_flat<T, 1024>, 1024);
        return true;
    }
    const bool held = with_row_form<T>(a, grad != nullptr, [&](auto group, auto chunks, auto cap) {
        using G = RowGroup<group()>;
        hipLaunchKernelGGL((k_distill_row<T, group(), chunks(), cap()>), dim3(static_cast<unsigned>(ceil_div(a.n_rows, G::kRows))),
                           dim3(G::kThreads), 0, stream, a, weight, loss, kept, grad, gs);
    });
    if (held) return true;
    if (a.n_rows >= kWholeRows || ceil_div(a.n_classes, Vec16<T>::kLen) <= kWholeVectors) {
        hipLaunchKernelGGL((k_distill_row<T, 1024, 0, kMaxTeacher>), dim3(static_cast<unsigned>(a.n_rows)), dim3(1024), 0, stream, a, weight,
                           loss, stats, static_cast<T*>(nullptr), gs);
        return false;
    }
    float2* row_part = static_cast<float2*>(part);
    hipLaunchKernelGGL(k_distill_stats<T>, pieces, dim3(kDistillThreads), 0, stream, a, sp.splits, sp.cols, row_part);
    hipLaunchKernelGGL((k_distill_finish<T, float2>), joins, dim3(kDistillThreads), 0, stream, a, sp.splits, row_part, stats, loss);
    return false;
}

template <typename T>
void launch_gradient(const DistillArgs& a, const float2* stats, const float* weight, T* grad, int64_t grad_stride, hipStream_t stream) {
    const DistillSplit sp = distill_split(a.n_rows, a.n_classes, sizeof(T) == 4 ? SERHIP_DTYPE_F32 : SERHIP_DTYPE_BF16);
    hipLaunchKernelGGL((a.temperature > kFlatTemperature ? k_distill_gradient<T, double> : k_distill_gradient<T, float>), dim3(static_cast<unsigned>(a.n_rows * sp.splits)), dim3(kDistillThreads), 0, stream, a,
                       sp.splits, sp.cols, stats, weight, grad, static_cast<long long>(grad_stride));
}

// --------------------------------------------------------------------------------------------- embedding
int key_bits(int64_t n_classes) {   // of the keys 0..n_classes (padding)
    int b = 1;
    while ((static_cast<int64_t>(1) << b) <= n_classes) ++b;
    return b;
}

int64_t sort_tile(int64_t n_tokens) { return kSortThreads * (n_tokens <= kSortShort ? 2 : 4); }

struct GradientScratch {
    size_t key[2], pos[2], hist, counts, runs, piece, total;
    int passes, bits;
};
GradientScratch gradient_scratch(int64_t n_tokens, int64_t n_classes, int64_t width) {
    GradientScratch s{};
    const int bits = key_bits(n_classes), most = n_tokens <= kSmallSort ? kSmallBits : kSortMaxBits;
    s.passes = (bits + most - 1) / most;
    s.bits = (bits + s.passes - 1) / s.passes;
    size_t at = 0;
    const auto take = [&](size_t bytes) {
        const size_t here = at;
        at += round_up(bytes, 256);
        return here;
    };
    const size_t words = static_cast<size_t>(n_tokens) * 4;
    for (int i = 0; i < 2; ++i) s.key[i] = take(words);
    for (int i = 0; i < 2; ++i) s.pos[i] = take(words);
    s.hist = take(n_tokens <= kSmallSort ? 0 : static_cast<size_t>(ceil_div(n_tokens, sort_tile(n_tokens))) * (4u << s.bits));
    s.counts = take(4u << s.bits);
    s.runs = take(4 * (1 + static_cast<size_t>(n_tokens) / kRunTile));   // a long run has more than kRunTile tokens
    s.piece = take(n_tokens > kRunTile ? static_cast<size_t>(ceil_div(n_tokens, kRunTile)) * 2 * width * sizeof(float) : 0);
    s.total = at;
    return s;
}

// Rows of the table for a workgroup: finding their runs takes as long for 4 as for 32, but the fewer, the more workgroups
// share a small table's work (512 bf16 columns; 30 000 tokens of 10 classes, by 1 and 8 rows: 40 and 54 us; of 8 192, by
// 4, 8 and 1: 53, 62 and 65; 32 768 of 16 384, by 8 and 32: 60 and 82; of 131 072: 101 and 80).
int embed_rows_per_block(int64_t n_classes) {
    return n_classes <= 512 ? 1 : n_classes <= 8192 ? 4 : n_classes <= 32768 ? 8 : kMostRows;
}

int check_embedding(const char* entry, const serhip_ctx* ctx, int dtype, int64_t n_tokens, int64_t n_classes, int64_t width) {
    if (!ctx) return invalid(entry, "ctx is NULL");
    if (!known_dtype(dtype)) return invalid(entry, "unknown element type");
    if (n_tokens < 0) return invalid(entry, "n_tokens < 0");
    if (n_classes < 1 || n_classes > (int64_t{1} << 31) - 2) return invalid(entry, "n_classes must be 1..2^31 - 2");
    if (width < 1 || width > (1 << 20)) return invalid(entry, "width must be 1..2^20");
    return SERHIP_OK;
}

}  // namespace

extern "C" {

int serhip_sample(serhip_ctx* ctx, const void* logits_dev, int dtype, int64_t n_rows, int64_t n_classes, int64_t row_stride,
                  const float* uniform_dev, float temperature, int32_t top_k, float top_p, float min_p,
                  const float* temperature_rows_dev, const int32_t* top_k_rows_dev, const float* top_p_rows_dev,
                  const float* min_p_rows_dev, int64_t* token_dev, float* logprob_dev, void* stream_v) {
    return guarded([&]() -> int {
        const char* entry = "serhip_sample";
        if (!ctx) return invalid(entry, "ctx is NULL");
        if (!known_dtype(dtype)) return invalid(entry, "unknown element type");
        if (n_rows < 0) return invalid(entry, "n_rows < 0");
        if (n_classes < 1 || n_classes > SERHIP_MAX_CLASSES) return invalid(entry, "n_classes must be 1..SERHIP_MAX_CLASSES");
        if (row_stride < 0) return invalid(entry, "row_stride < 0");
        if (n_rows == 0) return SERHIP_OK;
        if (!logits_dev || !uniform_dev || !token_dev || !logprob_dev) return invalid(entry, "NULL argument");
        if (!aligned_to(logits_dev, element_size(dtype))) return invalid(entry, "a pointer is not aligned to its element type");
        if (n_rows > kMaxThreads / (n_classes <= 64 ? 64 : 1024) - 4) return unsupported(entry, "too many rows per call");
        CLASS_TRY(hipSetDevice(context_device(ctx)));
        SampleArgs a{};
        a.logits = logits_dev;
        a.n_rows = n_rows;
        a.row_stride = row_stride;
        a.n_classes = static_cast<int>(n_classes);
        a.uniform = uniform_dev;
        a.temperature = temperature;
        a.top_k = top_k;
        a.top_p = top_p;
        a.min_p = min_p;
        a.temperature_rows = temperature_rows_dev;
        a.top_k_rows = top_k_rows_dev;
        a.top_p_rows = top_p_rows_dev;
        a.min_p_rows = min_p_rows_dev;
        a.weight_bits = std::min(45, 62 - round_up_log2(n_classes));
        a.token = reinterpret_cast<long long*>(token_dev);
        a.logprob = logprob_dev;
        const hipStream_t stream = static_cast<hipStream_t>(stream_v);
        // Workgroups of 512, of which a compute unit takes two, for short rows (1 x 1 000, top_k 50: 7.7 us, of 1 024: 13.5), and
        // where there are more rows than compute units (2 048 x 32 768 bf16, top_k 50: 62 and 95; 1 024 x 50 001 f32,
        // untruncated: 87 and 114; 1 024 x 100 003 bf16, top_p 0.9: 271 and 344) -- except for long ones whose min_p may leave
        // more candidates than fit half a compute unit's LDS (512 x 131 072, min_p 0.01: 145 and 74).  Few long rows are
        // read faster by 1 024 (256 x 100 003 f32: 50, by 512: 56; 128 x 50 001 bf16, top_k 50: 16.8 and 18.7).
        const bool may_be_many = (min_p > 0.0f || min_p_rows_dev) && (top_k <= 0 || top_k_rows_dev);
        const bool narrow = n_classes <= RowSampler<512>::kCandidates || (n_rows > 256 && (n_classes <= 65536 || !may_be_many));
        with_type(dtype, [&](auto z) {
            if (n_classes <= 64)
                hipLaunchKernelGGL(k_sample_small<decltype(z)>, dim3(static_cast<unsigned>(ceil_div(n_rows, kSmallThreads / 64))),
                                   dim3(kSmallThreads), 0, stream, a);
            else if (narrow)
                hipLaunchKernelGGL((k_sample_row<decltype(z), 512>), dim3(static_cast<unsigned>(n_rows)), dim3(512), 0, stream, a);
            else
                hipLaunchKernelGGL((k_sample_row<decltype(z), 1024>), dim3(static_cast<unsigned>(n_rows)), dim3(1024), 0, stream, a);
        });
        CLASS_TRY(hipGetLastError());
        return SERHIP_OK;
    });
}

int64_t serhip_distill_workspace(int64_t n_rows, int64_t n_classes, int dtype) {
    return static_cast<int64_t>(guarded([&]() -> int {
        const char* entry = "serhip_distill_workspace";
        if (!known_dtype(dtype)) return invalid(entry, "unknown element type");
        if (n_rows < 0 || n_rows > kMaxThreads) return invalid(entry, "n_rows out of range");
        if (n_classes < 1 || n_classes > SERHIP_MAX_CLASSES) return invalid(entry, "n_classes must be 1..SERHIP_MAX_CLASSES");
        return SERHIP_OK;
    })) < 0 ? SERHIP_E_INVALID : static_cast<int64_t>(distill_scratch(n_rows, n_classes, dtype).total);
}

int serhip_distill_loss(serhip_ctx* ctx, const void* logits_dev, int dtype, int64_t n_rows, int64_t n_classes,
                        int64_t row_stride, const void* index_dev, int index_is_i64, const void* teacher_dev,
                        int teacher_dtype, int32_t n_teacher, float temperature, float* loss_dev, float* stats_dev,
                        void* workspace_dev, int64_t workspace_bytes, void* stream_v) {
    return guarded([&]() -> int {
        const char* entry = "serhip_distill_loss";
        const DistillArgs a{logits_dev, n_rows, row_stride, static_cast<int>(n_classes), index_dev, index_is_i64,
                            teacher_dev, teacher_dtype, n_teacher, temperature};
        if (int rc = check_distill(entry, ctx, a, n_classes, dtype); rc != SERHIP_OK) return rc;
        if (n_rows == 0) return SERHIP_OK;
        if (!loss_dev || !stats_dev || !workspace_dev) return invalid(entry, "NULL argument");
        if (!aligned_to(stats_dev, 8) || !aligned_to(workspace_dev, 256)) return invalid(entry, "stats or workspace is not aligned");
        const DistillScratch s = distill_scratch(n_rows, n_classes, dtype);
        if (workspace_bytes < static_cast<int64_t>(s.total)) return invalid(entry, "the workspace is too small");
        CLASS_TRY(hipSetDevice(context_device(ctx)));
        with_type(dtype, [&](auto z) {
            using T = decltype(z);
            launch_rows<T>(a, nullptr, static_cast<char*>(workspace_dev) + s.part, reinterpret_cast<float2*>(stats_dev), loss_dev, nullptr, 0, static_cast<hipStream_t>(stream_v));
        });
        CLASS_TRY(hipGetLastError());
        return SERHIP_OK;
    });
}

int serhip_distill_gradient(serhip_ctx* ctx, const void* logits_dev, int dtype, int64_t n_rows, int64_t n_classes,
                            int64_t row_stride, const void* index_dev, int index_is_i64, const void* teacher_dev,
                            int teacher_dtype, int32_t n_teacher, float temperature, const float* stats_dev,
                            const float* row_weight_dev, void* grad_dev, int64_t grad_stride, void* stream_v) {
    return guarded([&]() -> int {
        const char* entry = "serhip_distill_gradient";
        const DistillArgs a{logits_dev, n_rows, row_stride, static_cast<int>(n_classes), index_dev, index_is_i64,
                            teacher_dev, teacher_dtype, n_teacher, temperature};
        if (int rc = check_distill(entry, ctx, a, n_classes, dtype); rc != SERHIP_OK) return rc;
        if (n_rows == 0) return SERHIP_OK;
        if (!stats_dev) return invalid(entry, "NULL argument");
        if (!aligned_to(stats_dev, 8)) return invalid(entry, "stats is not aligned");
        if (int rc = check_gradient_out(entry, a, grad_dev, grad_stride, dtype); rc != SERHIP_OK) return rc;
        CLASS_TRY(hipSetDevice(context_device(ctx)));
        const hipStream_t stream = static_cast<hipStream_t>(stream_v);
        with_type(dtype, [&](auto z) {
            using T = decltype(z);
            // rows that a wave holds are read once either way, and one form of the gradient is enough for them (4 096 rows of 512
            // bf16 classes: 6.5 us, with the row's statistics and a workgroup for each 11); at high temperatures f32 statistics
            // are not enough
            if (n_classes <= kTinyClasses || is_wave_row<T>(a) || (temperature > kFlatTemperature && !is_flat_split(a)))
                launch_rows<T>(a, row_weight_dev, nullptr, nullptr, nullptr, static_cast<T*>(grad_dev), grad_stride, stream);
            else
                launch_gradient<T>(a, reinterpret_cast<const float2*>(stats_dev), row_weight_dev, static_cast<T*>(grad_dev), grad_stride, stream);
        });
        CLASS_TRY(hipGetLastError());
        return SERHIP_OK;
    });
}

int serhip_distill_step(serhip_ctx* ctx, const void* logits_dev, int dtype, int64_t n_rows, int64_t n_classes,
                        int64_t row_stride, const void* index_dev, int index_is_i64, const void* teacher_dev,
                        int teacher_dtype, int32_t n_teacher, float temperature, const float* row_weight_dev,
                        float* loss_dev, void* grad_dev, int64_t grad_stride, void* workspace_dev,
                        int64_t workspace_bytes, void* stream_v) {
    return guarded([&]() -> int {
        const char* entry = "serhip_distill_step";
        const DistillArgs a{logits_dev, n_rows, row_stride, static_cast<int>(n_classes), index_dev, index_is_i64,
                            teacher_dev, teacher_dtype, n_teacher, temperature};
        if (int rc = check_distill(entry, ctx, a, n_classes, dtype); rc != SERHIP_OK) return rc;
        if (n_rows == 0) return SERHIP_OK;
        if (!loss_dev || !workspace_dev) return invalid(entry, "NULL argument");
        if (!aligned_to(workspace_dev, 256)) return invalid(entry, "the workspace is not 256-byte aligned");
        if (int rc = check_gradient_out(entry, a, grad_dev, grad_stride, dtype); rc != SERHIP_OK) return rc;
        const DistillScratch s = distill_scratch(n_rows, n_classes, dtype);
        if (workspace_bytes < static_cast<int64_t>(s.total)) return invalid(entry, "the workspace is too small");
        CLASS_TRY(hipSetDevice(context_device(ctx)));
        const hipStream_t stream = static_cast<hipStream_t>(stream_v);
        char* ws = static_cast<char*>(workspace_dev);
        float2* stats = reinterpret_cast<float2*>(ws + s.stats);
        with_type(dtype, [&](auto z) {
            using T = decltype(z);
            T* grad = static_cast<T*>(grad_dev);
            if (!launch_rows<T>(a, row_weight_dev, ws + s.part, stats, loss_dev, grad, grad_stride, stream))
                launch_gradient<T>(a, stats, row_weight_dev, grad, grad_stride, stream);
        });
        CLASS_TRY(hipGetLastError());
        return SERHIP_OK;
    });
}

int serhip_embed(serhip_ctx* ctx, const void* tokens_dev, int tokens_are_i64, int64_t n_tokens, const void* table_dev,
                 int dtype, int64_t table_stride, int64_t n_classes, int64_t width, float scale, void* out_dev,
                 int64_t out_stride, void* stream_v) {
    return guarded([&]() -> int {
        const char* entry = "serhip_embed";
        if (int rc = check_embedding(entry, ctx, dtype, n_tokens, n_classes, width); rc != SERHIP_OK) return rc;
        if (n_tokens == 0) return SERHIP_OK;
        if (!tokens_dev || !table_dev || !out_dev) return invalid(entry, "NULL argument");
        if (table_stride < 0 || (n_tokens > 1 && out_stride < width)) return invalid(entry, "a row stride is out of range");
        const int size = element_size(dtype);
        if (!aligned_to(table_dev, size) || !aligned_to(out_dev, size) || !aligned_to(tokens_dev, tokens_are_i64 ? 8 : 4))
            return invalid(entry, "a pointer is not aligned to its element type");
        const int64_t vectors = ceil_div(width, 16 / size);
        const int lane_bits = std::min(6, round_up_log2(vectors));
        const int64_t blocks = ceil_div(n_tokens << lane_bits, 256);
        if (n_tokens > (int64_t{1} << 40) || blocks > kMaxThreads / 256) return unsupported(entry, "too many tokens per call");
        CLASS_TRY(hipSetDevice(context_device(ctx)));
        with_type(dtype, [&](auto z) {
            using T = decltype(z);
            hipLaunchKernelGGL(k_embed<T>, dim3(static_cast<unsigned>(blocks), static_cast<unsigned>(ceil_div(vectors, 1 << lane_bits))),
                               dim3(256), 0, static_cast<hipStream_t>(stream_v), tokens_dev, tokens_are_i64,
                               static_cast<long long>(n_tokens), static_cast<const T*>(table_dev),
                               static_cast<long long>(table_stride), static_cast<long long>(n_classes), static_cast<int>(width),
                               lane_bits, scale, static_cast<T*>(out_dev), static_cast<long long>(out_stride));
        });
        CLASS_TRY(hipGetLastError());
        return SERHIP_OK;
    });
}

int64_t serhip_embed_gradient_workspace(int64_t n_tokens, int64_t n_classes, int64_t width) {
    if (n_tokens < 0 || n_tokens > SERHIP_MAX_TOKENS || n_classes < 1 || n_classes > (int64_t{1} << 31) - 2 || width < 1 ||
        width > (1 << 20))
        return guarded([&]() -> int { return invalid("serhip_embed_gradient_workspace", "a size is out of range"); });
    return static_cast<int64_t>(gradient_scratch(n_tokens, n_classes, width).total);
}

int serhip_embed_gradient(serhip_ctx* ctx, const void* grad_dev, int dtype, int64_t grad_stride, const void* tokens_dev,
                          int tokens_are_i64, int64_t n_tokens, int64_t n_classes, int64_t width, float scale,
                          int accumulate, void* out_dev, int out_dtype, int64_t out_stride, void* workspace_dev,
                          int64_t workspace_bytes, void* stream_v) {
    return guarded([&]() -> int {
        const char* entry = "serhip_embed_gradient";
        if (int rc = check_embedding(entry, ctx, dtype, n_tokens, n_classes, width); rc != SERHIP_OK) return rc;
        if (out_dtype != dtype && out_dtype != SERHIP_DTYPE_F32)
            return unsupported(entry, "the table's gradient has the type of the rows or is f32");
        if (n_tokens > SERHIP_MAX_TOKENS) return unsupported(entry, "more than SERHIP_MAX_TOKENS tokens per call");
        const int64_t tiles = n_tokens > kRunTile ? ceil_div(n_tokens, kRunTile) : 0;
        const int64_t piece_blocks = ceil_div(tiles * ceil_div(width, 64 * (16 / element_size(dtype))), 4);
        const int64_t row_blocks = ceil_div(n_classes, embed_rows_per_block(n_classes));
        if (piece_blocks + row_blocks > kMaxThreads / 256)
            return unsupported(entry, "too many classes, or tokens of this width, per call");
        if (!out_dev || (n_tokens > 0 && (!grad_dev || !tokens_dev || !workspace_dev))) return invalid(entry, "NULL argument");
        if (grad_stride < 0 || out_stride < width) return invalid(entry, "a row stride is out of range");
        if (!aligned_to(grad_dev, element_size(dtype)) || !aligned_to(out_dev, element_size(out_dtype)) ||
            !aligned_to(tokens_dev, tokens_are_i64 ? 8 : 4) || !aligned_to(workspace_dev, 256))
            return invalid(entry, "a pointer is not aligned");
        const GradientScratch s = gradient_scratch(n_tokens, n_classes, width);
        if (workspace_bytes < static_cast<int64_t>(s.total)) return invalid(entry, "the workspace is too small");
        CLASS_TRY(hipSetDevice(context_device(ctx)));
        const hipStream_t stream = static_cast<hipStream_t>(stream_v);
        char* ws = static_cast<char*>(workspace_dev);
        const auto words = [&](size_t at) { return reinterpret_cast<uint32_t*>(ws + at); };
        const int n = static_cast<int>(n_tokens);
        const uint32_t v = static_cast<uint32_t>(n_classes);
        const uint32_t *key = nullptr, *pos = nullptr;
        if (n > 0 && n <= kSmallSort) {
            hipLaunchKernelGGL(k_sort_small, dim3(1), dim3(kSmallThreadsSort), 0, stream, tokens_dev, tokens_are_i64, n, v, s.passes, s.bits,
                               words(s.key[0]), words(s.pos[0]), words(s.runs));
            key = words(s.key[0]);
            pos = words(s.pos[0]);
        } else if (n > 0) {
            const int tile_count = static_cast<int>(ceil_div(n, sort_tile(n)));
            const dim3 grid(static_cast<unsigned>(tile_count));
            for (int p = 0; p < s.passes; ++p) {
                uint32_t* key_out = words(s.key[p % 2]);
                uint32_t* pos_out = words(s.pos[p % 2]);
                uint32_t* counts = tile_count > kScanTiles ? words(s.counts) : nullptr;
                hipLaunchKernelGGL(n <= kSortShort ? k_sort_count<2> : k_sort_count<4>, grid, dim3(kSortThreads), 0, stream, tokens_dev,
                                   tokens_are_i64, n, v, key, p * s.bits, s.bits, words(s.hist), words(s.runs));
                if (counts)
                    hipLaunchKernelGGL(k_sort_scan, dim3(static_cast<unsigned>(ceil_div(1 << s.bits, kSortThreads))), dim3(kSortThreads), 0,
                                       stream, words(s.hist), tile_count, 1 << s.bits, counts);
                hipLaunchKernelGGL(n <= kSortShort ? k_sort_scatter<2> : k_sort_scatter<4>, grid, dim3(kSortThreads), 0, stream, tokens_dev,
                                   tokens_are_i64, n, v, key, pos, p * s.bits, s.bits, words(s.hist), counts, key_out, pos_out);
                key = key_out;
                pos = pos_out;
            }
        }
        const auto launch = [&](auto zg, auto zo) {
            using TG = decltype(zg);
            using TO = decltype(zo);
            const TG* g = static_cast<const TG*>(grad_dev);
            TO* o = static_cast<TO*>(out_dev);
            const long long gs = grad_stride, os = out_stride;
            const int w = static_cast<int>(width);
            float* piece = reinterpret_cast<float*>(ws + s.piece);
            hipLaunchKernelGGL((k_embed_sum<TG, TO>), dim3(static_cast<unsigned>(piece_blocks + row_blocks)), dim3(256),
                               0, stream, g, gs, key, pos, n, static_cast<long long>(n_classes), w, scale, accumulate, o, os,
                               embed_rows_per_block(n_classes),
                               static_cast<int>(piece_blocks), piece, words(s.runs));
            if (tiles)
                hipLaunchKernelGGL(k_embed_join<TO>, dim3(static_cast<unsigned>(std::min<int64_t>(tiles * ceil_div(w, 256), 1024))), dim3(256), 0,
                                   stream, key, n, w, piece, words(s.runs), scale, accumulate, o, os);
        };
        with_type(dtype, [&](auto zg) {
            if (out_dtype == dtype) launch(zg, zg);
            else launch(zg, float{});
        });
        CLASS_TRY(hipGetLastError());
        return SERHIP_OK;
    });
}

}  // extern "C"
