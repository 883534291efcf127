// Rows to their experts and back: the choices for each row put in order by expert, and the weighted sum of what a row's experts answered.
#include "inner.h"

namespace {

constexpr int kMostExperts = 1024;
constexpr int kMostEach = 64;
constexpr int kMostChoices = 1 << 28;

__device__ __forceinline__ int ones(unsigned long long v) { return __popcll(v); }

// An expert a group: its waves count, each in its own stretch of the choices, those of earlier experts and those of this one, and go over the stretch again to
// write where they stand. No count depends on another group, so one launch does it and the order is that of the choices.
__global__ __launch_bounds__(1024) void group_rows_kernel(const int* __restrict__ ids, int choices, int each, int experts, int* __restrict__ offsets, int* __restrict__ rows,
                                                          int* __restrict__ places) {
    constexpr int kWaves = 16;
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, expert = blockIdx.x;
    const int stretch = ((choices + kWaves - 1) / kWaves + 63) / 64 * 64;
    const long long from = (long long)wave * stretch;
    const int begin = from < choices ? (int)from : choices, end = min(choices - begin, stretch) + begin;
    __shared__ int before[kWaves], own[kWaves];
    int less = 0, equal = 0;
    for (int at = begin; at < end; at += 64) {
        const int id = at + lane < end ? ids[at + lane] : -1;
        less += ones(__ballot(id >= 0 && id < expert));
        equal += ones(__ballot(id == expert));
    }
    if (lane == 0) {
        before[wave] = less;
        own[wave] = equal;
    }
    __syncthreads();
    int first = 0, all = 0, at_wave = 0;
    for (int w = 0; w < kWaves; ++w) {
        first += before[w];
        if (w < wave) at_wave += own[w];
        all += own[w];
    }
    if (threadIdx.x == 0) {
        offsets[expert] = first;
        if (expert == experts - 1) offsets[experts] = first + all;
    }
    int place = first + at_wave;
    for (int at = begin; at < end; at += 64) {
        const int i = at + lane, id = i < end ? ids[i] : -1;
        const unsigned long long here = __ballot(i < end && id == expert);
        if (i < end && id == expert) {
            const int to = place + ones(here & ((1ull << lane) - 1));
            rows[to] = i / each;
            places[i] = to;
        }
        if (expert == 0 && i < end && (id < 0 || id >= experts)) places[i] = -1;
        place += ones(here);
    }
    if (expert == experts - 1)
        for (int i = first + all + threadIdx.x; i < choices; i += 1024) rows[i] = -1;
}

// A row and a run of 1024 outputs a group.
template <typename O>
__global__ __launch_bounds__(256) void combine_rows_kernel(const uint16_t* __restrict__ z, int z_stride, int z_rows, const int* __restrict__ places, const float* __restrict__ weights,
                                                           int kind, int each, int n, O* __restrict__ y, int y_stride) {
    const int row = blockIdx.x;
    const int* const place = places + (size_t)row * each;
    const float* const weight = weights + (size_t)row * each;
    float top = 0.f, total = 1.f;
    if (kind == EXHIP_WEIGHTS_LOG_NORMALIZED) {
        top = -__builtin_inff();
        for (int j = 0; j < each; ++j) top = fmaxf(top, weight[j]);
        if (top == -__builtin_inff()) top = 0.f;
        total = 0.f;
        for (int j = 0; j < each; ++j) total += expf(weight[j] - top);
    }
    for (int at = blockIdx.y * 1024 + threadIdx.x; at < min(n, (int)(blockIdx.y + 1) * 1024); at += 256) {
        float sum = 0.f;
        for (int j = 0; j < each; ++j) {
            const int from = place[j];
            if (from < 0) continue;
            const float w = kind == EXHIP_WEIGHTS_PLAIN ? weight[j] : total == 0.f ? 0.f : expf(weight[j] - top) / total;
            const float v = from < z_rows ? exhip_h2f(z[(size_t)from * z_stride + at]) : __builtin_nanf("");
            sum = __builtin_fmaf(w, v, sum);
        }
        if constexpr (sizeof(O) == 4) y[(size_t)row * y_stride + at] = sum;
        else y[(size_t)row * y_stride + at] = exhip_f2h(sum);
    }
}

template <typename O>
int combine_rows(exhip_ctx* ctx, const char* name, const uint16_t* z, int z_stride, int z_rows, const int32_t* places, const float* weights, int kind, int m, int each, int n, O* y,
                 int y_stride) {
    EXHIP_REQUIRE(ctx && z && places && weights && y, "%s: NULL argument", name);
    EXHIP_REQUIRE(m > 0 && each > 0 && each <= kMostEach && n > 0 && z_rows > 0, "%s: %d rows of %d choices, %d outputs, %d answers: sizes are positive, at most %d choices", name, m, each, n,
                  z_rows, kMostEach);
    EXHIP_REQUIRE(n <= 1 << 24 && (long long)m * each <= kMostChoices, "%s: %d rows of %d choices, %d outputs are more than one launch takes", name, m, each, n);
    EXHIP_REQUIRE(z_stride >= n && y_stride >= n, "%s: rows of %d values are %d and %d apart", name, n, z_stride, y_stride);
    EXHIP_REQUIRE(kind >= EXHIP_WEIGHTS_PLAIN && kind <= EXHIP_WEIGHTS_LOG_NORMALIZED, "%s: unknown kind of weights %d", name, kind);
    EXHIP_REQUIRE(aligned(z, 2) && aligned(places, 4) && aligned(weights, 4) && aligned(y, sizeof(O)), "%s: an operand's address is not that of its type", name);
    EXHIP_REQUIRE(m <= 0x7fffffff / 256, "%s: %d rows are more than one launch takes", name, m);
    const exhip_on_device on(ctx->device);
    EXHIP_CHECK(on.error);
    hipLaunchKernelGGL(combine_rows_kernel<O>, dim3(m, (n + 1023) / 1024), dim3(256), 0, ctx->stream, z, z_stride, z_rows, places, weights, kind, each, n, y, y_stride);
    EXHIP_LAUNCH_CHECK();
    return 0;
}

}  // namespace

extern "C" int exhip_group_rows(exhip_ctx* ctx, const int32_t* ids, int m, int each, int experts, int32_t* offsets, int32_t* rows, int32_t* places) {
    EXHIP_REQUIRE(ctx && ids && offsets && rows && places, "exhip_group_rows: NULL argument");
    EXHIP_REQUIRE(m > 0 && each > 0 && each <= kMostEach && experts > 0 && experts <= kMostExperts, "exhip_group_rows: %d rows of %d choices, %d experts: sizes are positive, at most %d and %d",
                  m, each, experts, kMostEach, kMostExperts);
    EXHIP_REQUIRE((long long)m * each <= kMostChoices, "exhip_group_rows: %d rows of %d choices are more than one launch takes", m, each);
    EXHIP_REQUIRE(aligned(ids, 4) && aligned(offsets, 4) && aligned(rows, 4) && aligned(places, 4), "exhip_group_rows: an operand's address is not that of its type");
    const exhip_on_device on(ctx->device);
    EXHIP_CHECK(on.error);
    hipLaunchKernelGGL(group_rows_kernel, dim3(experts), dim3(1024), 0, ctx->stream, ids, m * each, each, experts, offsets, rows, places);
    EXHIP_LAUNCH_CHECK();
    return 0;
}

extern "C" int exhip_combine_rows_f32(exhip_ctx* ctx, const uint16_t* z, int z_stride, int z_rows, const int32_t* places, const float* weights, int kind, int m, int each, int n, float* y,
                                      int y_stride) {
    return combine_rows(ctx, "exhip_combine_rows_f32", z, z_stride, z_rows, places, weights, kind, m, each, n, y, y_stride);
}
extern "C" int exhip_combine_rows_f16(exhip_ctx* ctx, const uint16_t* z, int z_stride, int z_rows, const int32_t* places, const float* weights, int kind, int m, int each, int n, uint16_t* y,
                                      int y_stride) {
    return combine_rows(ctx, "exhip_combine_rows_f16", z, z_stride, z_rows, places, weights, kind, m, each, n, y, y_stride);
}
