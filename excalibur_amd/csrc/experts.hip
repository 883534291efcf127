// Rows to their experts and back: the choices for each row put in order by expert, and the weighted sum of what a row's experts answered.
#include "inner.h"

namespace {

constexpr int kMostExperts = 1024;
constexpr int kMostEach = 64;
constexpr int kMostChoices = 1 << 28;

// An expert a group: its waves count, each in its own stretch of the choices, those of earlier experts and those of this one, and go over the stretch again to
// write where they stand. No count depends on another group, so one launch does it and the order is that of the choices. Four choices a lane and 256 a wave at a
// time, of which HELD stay in registers between the counting and the writing; where a stretch has more they are read again. Lanes count for themselves, two instructions a
// choice and count, and are added up once. (65528 choices of 256 experts: every CU reads all of them from L2.)
template <int HELD>
__global__ __launch_bounds__(1024) void group_rows_kernel(const int* __restrict__ ids, int choices, exhip_divisor row_of, int experts, int* __restrict__ offsets,
                                                          int* __restrict__ rows, int* __restrict__ places) {
    constexpr int kWaves = 16;
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), expert = blockIdx.x;
    const int stretch = ((choices + kWaves - 1) / kWaves + 255) / 256 * 256;
    const long long from = (long long)wave * stretch;
    const int begin = from < choices ? (int)from : choices, end = min(choices - begin, stretch) + begin, pieces = (end - begin + 255) / 256;
    const __amdgpu_buffer_rsrc_t view = uniform_view(ids + begin, (unsigned)(end - begin) * 4u);
    __shared__ int before[kWaves], own[kWaves];
    auto four = [&](int piece) { return __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(view, piece * 1024 + lane * 16, 0, 0)); };
    auto ended = [&](v4i v, int piece) {  // -1 behind the end
        if (begin + (piece + 1) * 256 > end)
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = begin + piece * 256 + lane * 4 + e < end ? v[e] : -1;
        return v;
    };
    int less = 0, equal = 0;
    auto count = [&](const v4i& v) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            less += (unsigned)v[e] < (unsigned)expert ? 1 : 0;
            equal += v[e] == expert ? 1 : 0;
        }
    };
    v4i held[HELD];
#pragma unroll
    for (int i = 0; i < HELD; ++i) held[i] = four(i);
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
        held[i] = ended(held[i], i);
        count(held[i]);
    }
#pragma unroll 4
    for (int i = HELD; i < pieces; ++i) count(ended(four(i), i));
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        less += __shfl_xor(less, d);
        equal += __shfl_xor(equal, d);
    }
    if (lane == 0) {
        before[wave] = less;
        own[wave] = equal;
    }
    __syncthreads();
    int first = 0, all = 0, place = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        first += before[w];
        if (w < wave) place += own[w];
        all += own[w];
    }
    place += first;
    if (threadIdx.x == 0) {
        offsets[expert] = first;
        if (expert == experts - 1) offsets[experts] = first + all;
    }
    int its = expert;
    asm volatile("" : "+s"(its));  // or the counting's comparisons are kept, two scalar registers each, and there are not so many
    auto write = [&](int piece, const v4i& v) {
        const int at = begin + piece * 256 + lane * 4;
        unsigned long long mask[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) mask[e] = __ballot(v[e] == its);
        if (mask[0] | mask[1] | mask[2] | mask[3]) {
            int to = place;  // behind those of earlier lanes
#pragma unroll
            for (int e = 0; e < 4; ++e) to = __builtin_amdgcn_mbcnt_hi((unsigned)(mask[e] >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)mask[e], to));
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (mask[e] == 0) continue;
                if (v[e] == its) {
                    rows[to] = (int)row_of(at + e);
                    places[at + e] = to++;
                }
                place += __popcll(mask[e]);
            }
        }
        if (expert == 0) {  // those that chose nothing
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if ((unsigned)v[e] >= (unsigned)experts && at + e < end) places[at + e] = -1;
        }
        __builtin_amdgcn_sched_barrier(0);
    };
#pragma unroll
    for (int i = 0; i < HELD; ++i) write(i, held[i]);
    for (int i = HELD; i < pieces; ++i) write(i, ended(four(i), i));
    if (expert == experts - 1)
        for (int i = first + all + threadIdx.x; i < choices; i += 1024) rows[i] = -1;
}

// ---- the sum of the answers ----
// A row's weights: a choice's own, in a lane each.
__device__ __forceinline__ float weight_of(const float* weights, int kind, int each, int j) {
    const float given = j < each ? weights[j] : -__builtin_inff();
    if (kind == EXHIP_WEIGHTS_PLAIN) return given;
    if (kind == EXHIP_WEIGHTS_LOG) return expf(given);
    float top = given;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
    const float own = j < each ? expf(given - (top == -__builtin_inff() ? 0.f : top)) : 0.f;
    float total = own;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) total += __shfl_xor(total, d);
    return total == 0.f ? 0.f : own / total;
}

// A wave takes a row and eight outputs a lane; its lanes hold the row's places and weights, which the sum takes from them one choice at a time, always in the
// choices' order. AHEAD answers are on their way at a time. Every answer is read once, and past L2, as the
// result is written: what bounds it is the memory (8191 x 6 answers of 4099 to float32 134 us through L2, 115 with answers past it, 102 with both, 5.3 TB/s; with four or eight on their
// way no less).
template <typename O, int AHEAD>
__global__ __launch_bounds__(256) void combine_rows_kernel(const uint16_t* __restrict__ z, int z_stride, int z_rows, const int* __restrict__ places, const float* __restrict__ weights,
                                                           int kind, int each, int n, O* __restrict__ y, int y_stride, int waves_a_row, size_t waves) {
    const size_t wave = (size_t)blockIdx.x * 4 + threadIdx.x / 64;
    if (wave >= waves) return;
    const int lane = threadIdx.x % 64;
    const size_t row = wave / waves_a_row;
    const int at = (int)(wave % waves_a_row) * 512 + lane * 8;
    const int place = lane < each ? places[row * each + lane] : -1;
    const float weight = weight_of(weights + row * each, kind, each, lane);
    const bool whole = at + 8 <= n;
    float sum[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) sum[e] = 0.f;
    for (int first = 0; first < each; first += AHEAD) {
        Eight<uint16_t> got[AHEAD];
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) {
            const int from = first + a < each ? __builtin_amdgcn_readlane(place, first + a) : -1;
            const uint16_t* const src = z + (size_t)max(from, 0) * z_stride + at;
            if (from >= 0 && from < z_rows) {
                if (whole) got[a] = __builtin_bit_cast(Eight<uint16_t>, __builtin_nontemporal_load(reinterpret_cast<const v4i_any*>(src)));
                else
#pragma unroll
                    for (int e = 0; e < 8; ++e) got[a].v[e] = at + e < n ? src[e] : 0;
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) got[a].v[e] = 0x7E00;  // not a number: there is no such row
            }
        }
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) {
            if (first + a >= each || __builtin_amdgcn_readlane(place, first + a) < 0) continue;
            const float w = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, weight), first + a));
#pragma unroll
            for (int e = 0; e < 8; ++e) sum[e] = __builtin_fmaf(w, exhip_h2f(got[a].v[e]), sum[e]);
        }
    }
    O* const to = y + row * y_stride + at;
    Eight<O> out;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        if constexpr (sizeof(O) == 4) out.v[e] = sum[e];
        else out.v[e] = exhip_f2h(sum[e]);
    }
    if (whole) {
        struct Pieces {
            v4i v[sizeof(O) / 2];
        };
        const Pieces pieces = __builtin_bit_cast(Pieces, out);
#pragma unroll
        for (int i = 0; i < (int)sizeof(O) / 2; ++i) __builtin_nontemporal_store(pieces.v[i], reinterpret_cast<v4i_any*>(to) + i);
    }
    else
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (at + e < n) to[e] = out.v[e];
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
    const int waves_a_row = (n + 511) / 512;
    const size_t waves = (size_t)m * waves_a_row, groups = (waves + 3) / 4;
    EXHIP_REQUIRE(groups <= 0x7fffffff / 256, "%s: %d rows of %d outputs are more than one launch takes", name, m, n);
    const exhip_on_device on(ctx->device);
    EXHIP_CHECK(on.error);
    hipLaunchKernelGGL((combine_rows_kernel<O, 2>), dim3((unsigned)groups), dim3(256), 0, ctx->stream, z, z_stride, z_rows, places, weights, kind, each, n, y, y_stride, waves_a_row, waves);
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
    const int choices = m * each;
    exhip_divisor row_of;
    row_of.set(each);
    const auto kernel = choices <= 16 * 256 ? group_rows_kernel<1> : choices <= 16 * 1024 ? group_rows_kernel<4> : group_rows_kernel<16>;
    hipLaunchKernelGGL(kernel, dim3(experts), dim3(1024), 0, ctx->stream, ids, choices, row_of, experts, offsets, rows, places);
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
