// Rows to their experts and back: the choices for each row put in order by expert, and the weighted sum of what a row's experts answered.
#include "inner.h"

namespace {

constexpr int kMostExperts = 1024;
constexpr int kMostEach = 64;
constexpr int kMostChoices = 1 << 28;

// Few choices: an expert a group, whose waves count, each in its own stretch of the choices, those of earlier experts and those of this one, four choices a lane and 256 a wave at
// a time, and write where theirs stand from the registers that they were counted in. Lanes count for themselves, two instructions a choice and count.
constexpr int kWaves = 16, kByExpert = 16384;  // of a group; the most choices

template <int HELD>
__global__ __launch_bounds__(1024) void group_rows_by_expert(const int* __restrict__ ids, int choices, exhip_divisor row_of, int experts, int* __restrict__ offsets,
                                                          int* __restrict__ rows, int* __restrict__ places) {
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), expert = blockIdx.x;
    const int stretch = ((choices + kWaves - 1) / kWaves + 255) / 256 * 256;
    const long long from = (long long)wave * stretch;
    const int begin = from < choices ? (int)from : choices, end = min(choices - begin, stretch) + begin;
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
        if ((wave * HELD + piece) % experts == expert) {  // those that chose nothing: every group has its share of the pieces
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if ((unsigned)v[e] >= (unsigned)experts && at + e < end) places[at + e] = -1;
        }
        __builtin_amdgcn_sched_barrier(0);
    };
#pragma unroll
    for (int i = 0; i < HELD; ++i) write(i, held[i]);
    if (expert == experts - 1)
        for (int i = first + all + threadIdx.x; i < choices; i += 1024) rows[i] = -1;
}

// Many choices: a group has a run of them, 1024 or more, and counts all of them by expert: those ahead of its run and the others, in LDS, where the counts of an expert stand in as
// many copies as there is room for, so that the lanes of an addition meet seldom. From the counts every group has where each expert's rows begin and how many of them stand
// ahead of its run, and it places its own choices, 1024 at a time: behind those of earlier waves, and within a wave behind the earlier lanes with the same expert. Nothing waits for
// another group, so one launch does it; whole numbers are added, so no order of additions shows. What bounds it is a CU's reading of all choices and their additions: 65528 choices of
// 256 experts take 8.3 us and of 1024 9.7, where a group an expert takes 12 and 28; 16384 of 64 take 7, where that takes 5.4. From 262144 choices on, 256 groups, the time grows with the choices:
// 524288 of 64 take 30 us, 8388608 387.
constexpr int kRun = 64 * kWaves, kCounts = 4096;  // choices at a time; counts of either kind in LDS, all copies

__global__ __launch_bounds__(kRun) void group_rows_by_run(const int* __restrict__ ids, int choices, exhip_divisor row_of, int experts, int copies, int bits, int run,
                                                          int* __restrict__ offsets, int* __restrict__ rows, int* __restrict__ places) {
    constexpr int kTogether = 8;  // loads on their way
    __shared__ int counts[2][kCounts + 64];  // [ahead of the run, from there on][expert][copy], and behind them 64 that nothing reads
    __shared__ int base[kMostExperts];       // where the next choice of each expert goes
    __shared__ unsigned short in_wave[kWaves][kMostExperts];
    __shared__ int sums[kWaves];
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), begin = blockIdx.x * run, end = min(choices - begin, run) + begin;
    const __amdgpu_buffer_rsrc_t view = uniform_view(ids, (unsigned)choices * 4u);
    int id = begin + (int)threadIdx.x < end ? ids[begin + threadIdx.x] : -1;  // this thread's choice of the first 1024
    for (int i = threadIdx.x; i < experts * copies; i += kRun) counts[0][i] = counts[1][i] = 0;
    __syncthreads();
    const int copy = lane & (copies - 1);
    for (int first = wave * 256; first < choices; first += kWaves * 256 * kTogether) {
        v4i got[kTogether];
#pragma unroll
        for (int i = 0; i < kTogether; ++i) got[i] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(view, (first + i * (kWaves * 256)) * 4 + lane * 16, 0, 0));
#pragma unroll
        for (int i = 0; i < kTogether; ++i) {
            const int at = first + i * (kWaves * 256);
            if (at >= choices) continue;
            if (at + 256 > choices)
#pragma unroll
                for (int e = 0; e < 4; ++e) got[i][e] = at + lane * 4 + e < choices ? got[i][e] : -1;
            int* const of = counts[at >= begin] + copy;  // (runs begin on multiples of 1024)
#pragma unroll
            for (int e = 0; e < 4; ++e) atomicAdd(of + (int)min((unsigned)got[i][e], (unsigned)experts) * copies, 1);
        }
    }
    __syncthreads();
    // every expert's, a thread each: where its rows begin
    int ahead = 0, all = 0;
    if ((int)threadIdx.x < experts)
        for (int c = 0; c < copies; ++c) {  // each thread from a copy of its own, for the banks
            const int at = threadIdx.x * copies + ((threadIdx.x + c) & (copies - 1));
            ahead += counts[0][at];
            all += counts[1][at];
        }
    all += ahead;
    int upto = all;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int before = __shfl_up(upto, d);
        if (lane >= d) upto += before;
    }
    if (lane == 63) sums[wave] = upto;
    __syncthreads();
    int total = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        if (w < wave) upto += sums[w];
        total += sums[w];
    }
    if ((int)threadIdx.x < experts) {
        base[threadIdx.x] = upto - all + ahead;
        if (blockIdx.x == 0) {
            offsets[threadIdx.x] = upto - all;
            if ((int)threadIdx.x == experts - 1) offsets[experts] = total;
        }
    }
    for (int first = begin; first < end; first += kRun) {
        for (int i = lane; i < experts; i += 64) in_wave[wave][i] = 0;
        const int i = first + threadIdx.x;
        const bool chooses = (unsigned)id < (unsigned)experts;
        unsigned long long same = __ballot(chooses);
        for (int bit = 0; bit < bits; ++bit) {
            const unsigned long long set = __ballot(id >> bit & 1);
            same &= id >> bit & 1 ? set : ~set;
        }
        const int earlier = __builtin_amdgcn_mbcnt_hi((unsigned)(same >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)same, 0));
        if (chooses && earlier == 0) in_wave[wave][id] = (unsigned short)__popcll(same);
        __syncthreads();
        int place = -1;
        if (chooses) {
            place = base[id] + earlier;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) place += w < wave ? in_wave[w][id] : 0;
            rows[place] = (int)row_of(i);
        }
        if (i < end) {
            places[i] = place;
            if (i >= total) rows[i] = -1;
        }
        if (first + kRun < end) {
            id = i + kRun < end ? ids[i + kRun] : -1;
            __syncthreads();
            if ((int)threadIdx.x < experts)
                for (int w = 0; w < kWaves; ++w) base[threadIdx.x] += in_wave[w][threadIdx.x];
            __syncthreads();
        }
    }
}

// ---- the sum of the answers ----
// A row's weights: a choice's own, in a lane each. `none`: all of them are logarithms of 0 and nothing divides them; the row is 0 then, whatever its answers are (0 times
// an infinity, or times what a row that nothing computed holds, would be no number).
__device__ __forceinline__ float weight_of(const float* weights, int kind, int each, int j, bool* none) {
    *none = false;
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
    *none = total == 0.f;
    return own / total;
}

// A wave takes a row and eight outputs a lane; its lanes hold the row's places and weights, which the sum takes from them one choice at a time, always in the
// choices' order. AHEAD answers are on their way at a time. Every answer is read once, and past L2, as the
// result is written: what bounds it is the memory (8191 x 6 answers of 4099 to float32 134 us through L2, 115 with answers past it, 100 with both, 5.3 TB/s; with four or eight on their
// way no less).
template <typename O, int AHEAD>
__global__ __launch_bounds__(256) void combine_rows_kernel(const uint16_t* __restrict__ z, int z_stride, int z_rows, const int* __restrict__ places, const float* __restrict__ weights,
                                                           int kind, int each, int n, O* __restrict__ y, int y_stride, int waves_a_row, size_t waves) {
    const size_t wave = (size_t)blockIdx.x * 4 + threadIdx.x / 64;
    if (wave >= waves) return;
    const int lane = threadIdx.x % 64;
    const size_t row = wave / waves_a_row;
    const int at = (int)(wave % waves_a_row) * 512 + lane * 8;
    const int chosen = lane < each ? places[row * each + lane] : -1;
    bool none;
    const float weight = weight_of(weights + row * each, kind, each, lane, &none);
    const int place = none ? -1 : chosen;
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
    if (choices <= kByExpert && experts <= 256) {
        const auto kernel = choices <= kByExpert / 4 ? group_rows_by_expert<1> : group_rows_by_expert<4>;
        hipLaunchKernelGGL(kernel, dim3(experts), dim3(64 * kWaves), 0, ctx->stream, ids, choices, row_of, experts, offsets, rows, places);
    } else {
        int copies = 64, bits = 0;
        while (copies * experts > kCounts) copies /= 2;
        while ((1 << bits) < experts) ++bits;
        const int run = (choices / 256 + kRun) / kRun * kRun, groups = (choices - 1) / run + 1;  // no more groups than CUs: each reads all choices
        hipLaunchKernelGGL(group_rows_by_run, dim3(groups), dim3(kRun), 0, ctx->stream, ids, choices, row_of, experts, copies, bits, run, offsets, rows, places);
    }
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
