// Log probabilities of given classes, the entropy and the largest classes of rows of values.
//
// With M = max x, S = sum exp(x - M) and T = sum exp(x - M) (x - M): log p = x - M - log S, and the entropy is log S - T / S.
#include "common.h"

namespace {

constexpr int kThreads = 256;
typedef unsigned long long u64;

__device__ __forceinline__ float value_of(const float* x, size_t i) { return x[i]; }
__device__ __forceinline__ float value_of(const uint16_t* x, size_t i) { return exhip_h2f(x[i]); }

// Larger for what stands further in front: by value (the zeros alike, NaN above all), then by index.
__device__ __forceinline__ unsigned order_of(float v) {
    if (v != v) return 0xffffffffu;
    const unsigned b = __builtin_bit_cast(unsigned, v + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ u64 place_of(float v, int i) { return (u64)order_of(v) << 32 | (unsigned)~i; }

struct LogpParams {
    const int32_t* ids;
    float *log_p, *entropy, *top_log_p;
    int32_t* top_ids;
    int m, c, x_stride, n_ids, top;
};

// What is written for value v of a row with maximum `most` and logarithm `log_s`.
__device__ __forceinline__ float log_p_of(float v, float most, float log_s) {
    if (most == -INFINITY) return v != v ? v : -INFINITY;
    return v - most - log_s;
}

template <typename T, typename F>
__device__ T over_group(T v, T* shared, F f) {
    __syncthreads();
    shared[threadIdx.x] = v;
    __syncthreads();
    for (int d = kThreads / 2; d > 0; d >>= 1) {
        if ((int)threadIdx.x < d) shared[threadIdx.x] = f(shared[threadIdx.x], shared[threadIdx.x + d]);
        __syncthreads();
    }
    return shared[0];
}

// A group a row.
template <typename T>
__global__ __launch_bounds__(kThreads) void log_probabilities_kernel(const T* __restrict__ x, const LogpParams p) {
    __shared__ float fs[kThreads];
    __shared__ u64 us[kThreads];
    const size_t row = blockIdx.x;
    const T* const src = x + row * p.x_stride;
    float most = -INFINITY;
    for (int i = threadIdx.x; i < p.c; i += kThreads) most = fmaxf(most, value_of(src, i));
    most = over_group(most, fs, [](float a, float b) { return fmaxf(a, b); });
    const float base = most == -INFINITY ? 0.f : most;
    float s = 0.f, t = 0.f;
    for (int i = threadIdx.x; i < p.c; i += kThreads) {
        const float d = value_of(src, i) - base, e = expf(d);
        s += e;
        if (e != 0.f) t += e * d;
    }
    s = over_group(s, fs, [](float a, float b) { return a + b; });
    t = over_group(t, fs, [](float a, float b) { return a + b; });
    const bool empty = most == -INFINITY && s == 0.f;
    const float log_s = logf(s);
    if (threadIdx.x == 0 && p.entropy) p.entropy[row] = empty ? 0.f : log_s - t / s;
    for (int i = threadIdx.x; i < p.n_ids; i += kThreads) {
        const int id = p.ids[row * p.n_ids + i];
        p.log_p[row * p.n_ids + i] = id < 0 ? 0.f : id >= p.c ? NAN : s != s ? s : log_p_of(value_of(src, id), most, log_s);
    }
    u64 last = ~0ull;
    for (int n = 0; n < p.top; ++n) {
        u64 best = 0;
        for (int i = threadIdx.x; i < p.c; i += kThreads) {
            const u64 at = place_of(value_of(src, i), i);
            if (at < last && at > best) best = at;
        }
        last = over_group(best, us, [](u64 a, u64 b) { return a > b ? a : b; });
        if (threadIdx.x == 0) {
            const int id = (int)~(unsigned)last;
            p.top_ids[row * p.top + n] = id;
            p.top_log_p[row * p.top + n] = s != s ? s : log_p_of(value_of(src, id), most, log_s);
        }
    }
}

template <typename T>
int log_probabilities(exhip_ctx* ctx, const char* name, const T* x, int x_stride, int m, int c, const int32_t* ids, int n_ids, float* log_p, float* entropy, int top,
                      int32_t* top_ids, float* top_log_p, void* workspace) {
    EXHIP_REQUIRE(ctx && x && workspace, "%s: NULL argument", name);
    EXHIP_REQUIRE(m > 0 && c > 0 && x_stride >= c, "%s: %d rows of %d values, %d apart", name, m, c, x_stride);
    EXHIP_REQUIRE(n_ids >= 0 && (n_ids == 0 ? !log_p : ids && log_p), "%s: %d classes asked of a row need ids and log_p, none need neither", name, n_ids);
    EXHIP_REQUIRE(top >= 0 && top <= EXHIP_LOG_PROBABILITIES_TOP && top <= c && (top == 0 ? !top_ids && !top_log_p : top_ids && top_log_p),
                  "%s: the %d largest of %d classes: at most %d, with both results", name, top, c, EXHIP_LOG_PROBABILITIES_TOP);
    EXHIP_REQUIRE(log_p || entropy || top, "%s: nothing is asked", name);
    EXHIP_REQUIRE((uintptr_t)x % sizeof(T) == 0 && ((uintptr_t)ids | (uintptr_t)log_p | (uintptr_t)entropy | (uintptr_t)top_ids | (uintptr_t)top_log_p) % 4 == 0 && (uintptr_t)workspace % 16 == 0,
                  "%s: an operand's address is not that of its type", name);
    const LogpParams p = {ids, log_p, entropy, top_log_p, top_ids, m, c, x_stride, n_ids, top};
    const exhip_on_device on(ctx->device);
    EXHIP_CHECK(on.error);
    hipLaunchKernelGGL(log_probabilities_kernel<T>, dim3(m), dim3(kThreads), 0, ctx->stream, x, p);
    EXHIP_LAUNCH_CHECK();
    return 0;
}

}  // namespace

extern "C" size_t exhip_log_probabilities_workspace(int m, int c, int top) {
    if (m <= 0 || c <= 0 || top < 0 || top > EXHIP_LOG_PROBABILITIES_TOP || top > c) {
        exhip_set_error("exhip_log_probabilities_workspace: %d rows of %d values, the %d largest", m, c, top);
        return 0;
    }
    return 16;
}

extern "C" int exhip_log_probabilities_f32(exhip_ctx* ctx, const float* x, int x_stride, int m, int c, const int32_t* ids, int n_ids, float* log_p, float* entropy,
                                           int top, int32_t* top_ids, float* top_log_p, void* workspace) {
    return log_probabilities(ctx, "exhip_log_probabilities_f32", x, x_stride, m, c, ids, n_ids, log_p, entropy, top, top_ids, top_log_p, workspace);
}
extern "C" int exhip_log_probabilities_f16(exhip_ctx* ctx, const uint16_t* x, int x_stride, int m, int c, const int32_t* ids, int n_ids, float* log_p, float* entropy,
                                           int top, int32_t* top_ids, float* top_log_p, void* workspace) {
    return log_probabilities(ctx, "exhip_log_probabilities_f16", x, x_stride, m, c, ids, n_ids, log_p, entropy, top, top_ids, top_log_p, workspace);
}
