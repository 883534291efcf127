// Log probabilities of given classes, the entropy and the largest classes of rows of values.
//
// With M = max x, S = sum exp(x - M) and T = sum exp(x - M) (x - M): log p = x - M - log S, and the entropy is log S - T / S. The values are read once: a
// group holds its slice of a row in registers, so the maximum comes first and every exponential is taken once. Slices of a row are joined in the order of
// their lanes, whatever order the groups end in.
#include <float.h>

#include "common.h"
#include "largest.h"
#include "on_device.h"

namespace {

constexpr int kMostSlice = 32768, kLongSlice = 16384, kSlice = 8192;  // values of a row that a group of 16, of 8, of 4 waves holds in its registers
static_assert(kMostSlice <= kMostCounted, "a count of a slice's values is half a word");
constexpr int kCandidates = 512;  // places that are held at once
constexpr int kRanked = 128;      // and that are ranked, each against all; of more, those behind the top-th are left out first
typedef unsigned long long u64;

template <typename T, int N>
struct __attribute__((packed, aligned(sizeof(T)))) Run {  // neighbouring values at any alignment of their type
    T v[N];
};
__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(uint16_t v) { return exhip_h2f(v); }
// The largest of a run, NaN left out.
__device__ __forceinline__ float run_max(const Run<float, 4>& r) { return fmaxf(fmaxf(r.v[0], r.v[1]), fmaxf(r.v[2], r.v[3])); }
__device__ __forceinline__ float run_max(const Run<uint16_t, 8>& r) {
    typedef _Float16 v2h __attribute__((ext_vector_type(2)));
    struct Pairs { v2h p[4]; };
    const Pairs h = __builtin_bit_cast(Pairs, r);
    const v2h m = __builtin_elementwise_max(__builtin_elementwise_max(h.p[0], h.p[1]), __builtin_elementwise_max(h.p[2], h.p[3]));
    return fmaxf((float)m[0], (float)m[1]);
}

__device__ __forceinline__ float masked(float) { return -INFINITY; }
__device__ __forceinline__ uint16_t masked(uint16_t) { return 0xfc00; }

// f over the values of a wave's 64 lanes, or of each of its rows of 16, in all of them: lanes one and two apart trade within their quads, quads and
// halves of a row by its mirror images, rows by swaps. Both partners of a trade compute the same, so f has to be symmetric.
template <int CONTROL>
__device__ __forceinline__ float traded(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CONTROL, 0xF, 0xF, true));
}
template <typename F>
__device__ __forceinline__ float over_row(float v, F f) {
    v = f(v, traded<0xB1>(v));   // quad_perm [1, 0, 3, 2]
    v = f(v, traded<0x4E>(v));   // quad_perm [2, 3, 0, 1]
    v = f(v, traded<0x141>(v));  // row_half_mirror
    return f(v, traded<0x140>(v));  // row_mirror
}
template <typename F>
__device__ __forceinline__ float over_wave(float v, F f) {
    v = over_row(v, f);
    const auto bits = [](float x) { return __builtin_bit_cast(unsigned, x); };
    const auto r = __builtin_amdgcn_permlane16_swap(bits(v), bits(v), false, false);
    const unsigned r0 = r[0], r1 = r[1];
    v = f(__builtin_bit_cast(float, r0), __builtin_bit_cast(float, r1));
    const auto h = __builtin_amdgcn_permlane32_swap(bits(v), bits(v), false, false);
    const unsigned h0 = h[0], h1 = h[1];
    return f(__builtin_bit_cast(float, h0), __builtin_bit_cast(float, h1));
}
// A bound that `top` of a wave's values, N of each lane, reach: the top-th largest, by halving, to BITS bits of order_of(), downwards.
template <int BITS, int N>
__device__ __forceinline__ unsigned reached_by(const unsigned (&order)[N], int top) {
    unsigned bound = 0;
#pragma unroll
    for (int bit = 31; bit >= 32 - BITS; --bit) {
        const unsigned up = bound | 1u << bit;
        int reach = 0;
#pragma unroll
        for (int e = 0; e < N; ++e) reach += __popcll(__ballot(order[e] >= up));
        bound = reach >= top ? up : bound;
    }
    return bound;
}
__device__ __forceinline__ float larger(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ float sum(float a, float b) { return a + b; }
// A lane's place among those of a mask.
__device__ __forceinline__ int place_in(u64 mask) { return __builtin_amdgcn_mbcnt_hi((unsigned)(mask >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)mask, 0)); }

// Larger for what stands further in front: by value (the zeros alike, NaN above all), then by index. Never 0.
__device__ __forceinline__ unsigned order_of(float v) {
    if (v != v) return 0xffffffffu;
    const unsigned b = __builtin_bit_cast(unsigned, v + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ u64 place_of(float v, int i) { return (u64)order_of(v) << 32 | (unsigned)~i; }
__device__ __forceinline__ int index_of(u64 place) { return (int)~(unsigned)place; }

// Exponentials are taken as powers of two, logarithms as those to base two.
constexpr float kLog2e = 1.44269504088896341f, kLn2 = 0.69314718055994531f;
constexpr float kNoPart = -300.f;  // two to this has no part in a sum; -infinity must not meet a zero in a product

// Maximum, s = sum exp(x - maximum) and t = sum exp(x - maximum) (x - maximum) log2 e of some values; nothing: -infinity, 0, 0.
struct __attribute__((aligned(16))) Sums {
    float most, s, t, unused;
};
__device__ __forceinline__ float power(float z) { return __builtin_amdgcn_exp2f(z); }
__device__ __forceinline__ Sums joined(const Sums& a, const Sums& b) {
    Sums r;
    r.most = fmaxf(a.most, b.most);
    const float base = r.most == -INFINITY ? 0.f : r.most;
    const float da = fmaxf((a.most - base) * kLog2e, kNoPart), db = fmaxf((b.most - base) * kLog2e, kNoPart), ea = power(da), eb = power(db);
    r.s = a.s * ea + b.s * eb;
    r.t = (a.t + a.s * da) * ea + (b.t + b.s * db) * eb;
    r.unused = 0.f;
    return r;
}
template <int CONTROL>
__device__ __forceinline__ Sums traded(const Sums& a) { return Sums{traded<CONTROL>(a.most), traded<CONTROL>(a.s), traded<CONTROL>(a.t), 0.f}; }
__device__ __forceinline__ Sums from_lane(const Sums& a, int d) {
    return Sums{__shfl_xor(a.most, d), __shfl_xor(a.s, d), __shfl_xor(a.t, d), 0.f};
}

// What lanes of a wave have written into LDS is there for the others.
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// How many of n places (eight zeros behind them) stand in front of `own`: eight reads under way at a time.
__device__ __forceinline__ int rank_of(u64 own, const u64* places, int n) {
    int rank = 0;
    for (int j = 0; j < n; j += 8) {
        u64 o[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = places[j + e];
#pragma unroll
        for (int e = 0; e < 8; ++e) rank += o[e] > own;
    }
    return rank;
}
// The `top` first of n places, in falling order, into sorted, by one wave.
__device__ __forceinline__ void rank_places(u64* places, int n, int top, u64* sorted) {
    const int lane = threadIdx.x % 64;
    if (lane < 8) places[n + lane] = 0;
    wave_sync();
    for (int i = lane; i < n; i += 64) {
        const u64 own = places[i];
        const int rank = rank_of(own, places, n);
        if (rank < top) sorted[rank] = own;
    }
    wave_sync();
}
// Of kHeld places of each lane (0: none) those that reach a bound, into places; how many.
constexpr int kHeld = kCandidates / 64;
__device__ __forceinline__ int keep_reaching(const u64 (&held)[kHeld], unsigned bound, u64* places) {
    int n = 0;
#pragma unroll
    for (int e = 0; e < kHeld; ++e) {
        const bool takes = held[e] != 0 && (unsigned)(held[e] >> 32) >= bound;
        const u64 all_takes = __ballot(takes);
        if (takes) places[n + place_in(all_takes)] = held[e];
        n += __popcll(all_takes);
    }
    return n;
}
__device__ __forceinline__ unsigned reached_by_all(const u64 (&held)[kHeld], int top) {
    unsigned order[kHeld];
#pragma unroll
    for (int e = 0; e < kHeld; ++e) order[e] = (unsigned)(held[e] >> 32);
    return reached_by<16>(order, top);
}

struct LogpParams {
    const int32_t* ids;
    float *log_p, *entropy, *top_log_p;
    int32_t* top_ids;
    Sums* part;   // [row][slice], of rows in several slices
    u64* part_top;  // [row][slice][top]: places in falling order, 0 where there are no more
    int m, c, x_stride, n_ids, top;
    int slices, slice_len;
};

// What is written for value v of a row with these sums.
__device__ __forceinline__ float log_p_of(float v, const Sums& r, float log_s) {
    if (r.s != r.s) return r.s;
    if (r.most == -INFINITY) return -INFINITY;
    return v - r.most - log_s;
}

// The answers of a row, by one wave, from its sums and the places of its largest.
template <typename T>
__device__ __forceinline__ void write_row(const T* __restrict__ src, const LogpParams& p, size_t row, const Sums& r, const u64* places) {
    const int lane = threadIdx.x % 64;
    // The largest has a part of one in s, and none in t has another sign: what rounding leaves below one, or below an entropy of zero, is not there.
    const float log_s = r.s < 1.f ? 0.f : __builtin_amdgcn_logf(r.s) * kLn2;
    if (lane == 0 && p.entropy) p.entropy[row] = r.s != r.s ? r.s : r.most == -INFINITY ? 0.f : fmaxf(log_s - r.t / r.s * kLn2, 0.f);
    for (int i = lane; i < p.n_ids; i += 64) {
        const int id = p.ids[row * p.n_ids + i];
        p.log_p[row * p.n_ids + i] = id < 0 ? 0.f : id >= p.c ? NAN : log_p_of(as_float(src[id]), r, log_s);
    }
    if (lane < p.top) {
        const u64 at = places[lane];
        const unsigned o = (unsigned)(at >> 32);
        p.top_ids[row * p.top + lane] = index_of(at);
        // the value back from its order
        p.top_log_p[row * p.top + lane] = log_p_of(__builtin_bit_cast(float, o & 0x80000000u ? o & 0x7fffffffu : ~o), r, log_s);
    }
}

// A group of W waves a slice of a row, V values a thread, all requested before the first is used. What one wave can do for the group is wave 0's: the others
// would only take its turns.
template <typename T, int W, int V, bool TOP>
__global__ __launch_bounds__(64 * W, 8) void log_probabilities_kernel(const T* __restrict__ x, const LogpParams p) {
    exhip_touch_args(p);
    constexpr int kThreads = 64 * W, N = 16 / sizeof(T), kRuns = V / N;
    static_assert(W == 1 || W == 4 || W == 8 || W == 16, "128 sets of a slice's values; joins of a power of two");
    __shared__ Sums sums[W];
    __shared__ float sets[TOP ? 128 : 1], bound;
    __shared__ u64 places[TOP ? kCandidates + 8 : 1], sorted[TOP ? EXHIP_LOG_PROBABILITIES_TOP : 1];
    __shared__ int count;
    __shared__ unsigned counts[2][W];
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const size_t row = blockIdx.x / p.slices;
    const int slice = blockIdx.x % p.slices, first = slice * p.slice_len, len = min(p.slice_len, p.c - first);
    const T* const src = x + row * p.x_stride + first;
    Run<T, N> r[kRuns];
    auto value = [&](int e) { return as_float(r[e / N].v[e % N]); };
    auto at = [&](int e) { return (e / N * kThreads + (int)threadIdx.x) * N + e % N; };  // of value e in the slice
    auto has = [&](int i) { return (i * kThreads + wave * 64) * N < len; };  // whether run i of the wave has a value at all
    auto read = [&](int i) {
        Run<T, N> run;
        const int k = at(i * N);
        if (k + N <= len) run = *reinterpret_cast<const Run<T, N>*>(src + k);
        else
#pragma unroll
            for (int e = 0; e < N; ++e) run.v[e] = k + e < len ? src[k + e] : masked(T());
        return run;
    };
#pragma unroll
    for (int i = 0; i < kRuns; ++i) {
        const int k = at(i * N);
        if (k + N <= len) r[i] = *reinterpret_cast<const Run<T, N>*>(src + k);
        else if (!has(i))
#pragma unroll
            for (int e = 0; e < N; ++e) r[i].v[e] = masked(T());
        else
#pragma unroll
            for (int e = 0; e < N; ++e) r[i].v[e] = k + e < len ? src[k + e] : masked(T());
    }
    float largest[kRuns], mine = -INFINITY;
#pragma unroll
    for (int i = 0; i < kRuns; ++i) {
        largest[i] = run_max(r[i]);
        mine = fmaxf(mine, largest[i]);
    }
    const float most = over_wave(mine, larger), base = most == -INFINITY ? 0.f : most;
    // (x - base) log2 e. Halves, of which a byte costs twice the exponentials, take one multiply-add: base log2 e is scaled + beside exactly, and `beside`
    // comes in at the end. (Of the largest floats that product is infinite.)
    constexpr bool kOneStep = sizeof(T) == 2;
    const float scaled = base * kLog2e, beside = __builtin_fmaf(base, kLog2e, -scaled);
    float s = 0.f, t = 0.f;
#pragma unroll
    for (int e = 0; e < V; ++e) {
        if (e % N == 0 && !has(e / N)) break;
        const float z = kOneStep ? __builtin_fmaf(value(e), kLog2e, -scaled) : (value(e) - base) * kLog2e, w = power(z);  // a NaN goes on into s
        s += w;
        t = __builtin_fmaf(w, fmaxf(z, kNoPart), t);
    }
    if constexpr (kOneStep) {
        t = (t - beside * s) * power(-beside);
        s *= power(-beside);
    }
    Sums all = {most, over_wave(s, sum), over_wave(t, sum), 0.f};
    if constexpr (W > 1) {
        if (lane == 0) sums[wave] = all;
    }
    if constexpr (TOP) {
        // the largest of each of 128 sets: the values of W / 2 neighbouring lanes, or a lane's even and odd runs
        if constexpr (W > 1) {
            float m = fmaxf(mine, traded<0xB1>(mine));
            if constexpr (W > 4) m = fmaxf(m, traded<0x4E>(m));
            if constexpr (W > 8) m = fmaxf(m, traded<0x141>(m));
            if (lane % (W / 2) == 0) sets[wave * (128 / W) + lane / (W / 2)] = m;
        } else {
            float m[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int i = 0; i < kRuns; ++i) m[i % 2] = fmaxf(m[i % 2], largest[i]);
            sets[lane] = m[0];
            sets[64 + lane] = m[1];
        }
        if (threadIdx.x == 0) count = 0;
    }
    __syncthreads();
    if (wave == 0) {
        __builtin_amdgcn_s_setprio(3);  // the group's other waves wait for this one
        if constexpr (W > 1) {
            all = sums[lane % W];
            all = joined(all, traded<0xB1>(all));
            all = joined(all, traded<0x4E>(all));
            if constexpr (W > 4) all = joined(all, traded<0x141>(all));
            if constexpr (W > 8) all = joined(all, traded<0x140>(all));
        }
        if constexpr (TOP) {
            // `top` sets hold a value that reaches the top-th largest of the sets' largest, so the slice's `top` largest all do. A class of no probability is
            // no candidate whatever the bound; with a NaN nothing is.
            const unsigned of_sets[2] = {order_of(sets[lane]), order_of(sets[64 + lane])};
            const unsigned o = reached_by<16>(of_sets, p.top);
            const float least = o <= 0x007fffffu ? -FLT_MAX : __builtin_bit_cast(float, o & 0x80000000u ? o & 0x7fffffffu : ~o);
            if (lane == 0) bound = all.s != all.s ? INFINITY : least;
        }
    }
    if constexpr (TOP) {
        __syncthreads();
        const float least = bound;
        if (__ballot(mine >= least) != 0)
#pragma unroll
            for (int i = 0; i < kRuns; ++i)
                if (__ballot(largest[i] >= least) != 0) {
                    u64 takes[N];
                    int here = 0, slot = 0;
#pragma unroll
                    for (int e = 0; e < N; ++e) {
                        takes[e] = __ballot(value(i * N + e) >= least);
                        here += __popcll(takes[e]);
                    }
                    if (lane == 0) slot = atomicAdd(&count, here);
                    slot = __builtin_amdgcn_readfirstlane(slot);
#pragma unroll
                    for (int e = 0; e < N; ++e) {
                        const int to = slot + place_in(takes[e]);
                        if (value(i * N + e) >= least && to < kCandidates) places[to] = place_of(value(i * N + e), first + at(i * N + e));
                        slot += __popcll(takes[e]);
                    }
                }
        __syncthreads();
        int n = count;
        const bool many = least == INFINITY || n > kCandidates;  // a NaN (or a +infinity, whose exponential is one), or values close to each other
        if (many) {
            // The bound is raised by halves until between `want` and kRanked values reach it; where more are alike (all of a slice, if its classes are masked
            // with the type's lowest value), as many of these as come first. (300 rows of 100003 equal halves: 75 us with the 8 largest, 117 with 64, of NaN, which the bound
            // reaches last, 404 and 447; a reading of the slice for each of the largest took 187 and 1375.)
            const int want = min(p.top, len);
            int turn = 0;
            const unsigned of_sets[2] = {order_of(sets[lane]), order_of(sets[64 + lane])};
            const Cut cut = find_cut(reached_by<32>(of_sets, want), want, kRanked, len, [&](unsigned o, auto takes) {
                int here = 0, more = 0;
#pragma unroll 1
                for (int i = 0; i < kRuns; ++i) {  // read again: what stays of them for this path costs the other one its waves
                    const Run<T, N> run = read(i);
#pragma unroll
                    for (int e = 0; e < N; ++e) {
                        const unsigned order = order_of(as_float(run.v[e]));
                        here += __popcll(__ballot(takes(order, at(i * N + e))));
                        more += __popcll(__ballot(order > o));
                    }
                }
                unsigned two = two_counts(here, more);
                if constexpr (W > 1) {
                    if (lane == 0) counts[turn][wave] = two;
                    __syncthreads();
                    two = 0;
#pragma unroll
                    for (int w = 0; w < W; ++w) two += counts[turn][w];
                    turn ^= 1;
                }
                return two;
            });
            if (threadIdx.x == 0) count = 0;
            __syncthreads();
#pragma unroll 1
            for (int i = 0; i < kRuns; ++i) {
                const Run<T, N> run = read(i);
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    const float v = as_float(run.v[e]);
                    const unsigned order = order_of(v);
                    const int k = at(i * N + e);
                    if (order > cut.order || (order == cut.order && k < cut.end)) {
                        const int to = atomicAdd(&count, 1);
                        if (to < kCandidates) places[to] = place_of(v, first + k);
                    }
                }
            }
            __syncthreads();
            n = min(count, kCandidates);  // without what stands behind the slice's end
        }
        if (wave != 0) return;
        if (!many && n < p.top) {  // masked classes too, by their index: they are among the first n + top of the slice
            const int reach = min(n + p.top, len);
            for (int i = lane; i - lane < reach; i += 64) {
                const bool takes = i < reach && as_float(src[i]) == -INFINITY;
                const u64 all_takes = __ballot(takes);
                if (takes) places[n + place_in(all_takes)] = place_of(-INFINITY, first + i);
                n += __popcll(all_takes);
            }
        }
        if (lane >= n && lane < p.top) sorted[lane] = 0;
        wave_sync();
        if (n > kRanked) {
            u64 held[kHeld];
#pragma unroll
            for (int e = 0; e < kHeld; ++e) held[e] = e * 64 + lane < n ? places[e * 64 + lane] : 0;
            n = keep_reaching(held, reached_by_all(held, p.top), places);
        }
        rank_places(places, n, p.top, sorted);
    } else if (wave != 0) {
        return;
    }
    if (p.slices == 1) {
        write_row(src, p, row, all, sorted);
    } else {
        if (lane == 0) p.part[blockIdx.x] = all;
        if constexpr (TOP)
            if (lane < p.top) p.part_top[(size_t)blockIdx.x * p.top + lane] = sorted[lane];
    }
}

// The largest of the slices' lists, `top` of them into sorted, by one wave: a batch of entries is held in registers with those found so far in front, and what
// reaches the top-th largest of the lanes' largest is ranked.
__device__ __forceinline__ void join_lists(const u64* __restrict__ from, size_t total, int top, u64* places, u64* sorted) {
    const int lane = threadIdx.x;
    int kept = 0;
    for (size_t done = 0; done < total;) {
        u64 held[kHeld], most = 0;
#pragma unroll
        for (int e = 0; e < kHeld; ++e) {
            const int i = e * 64 + lane;  // the first `kept` of a batch are those found so far
            held[e] = i < kept ? sorted[i] : done + (i - kept) < total ? from[done + (i - kept)] : 0;
        }
#pragma unroll
        for (int e = 0; e < kHeld; ++e) most = held[e] > most ? held[e] : most;
        done += kHeld * 64 - kept;
        unsigned bound;
        if (top > 32) {  // of so many the lanes' largest leave hundreds to rank
            bound = reached_by_all(held, top);
        } else {
            const unsigned of_lane[1] = {(unsigned)(most >> 32)};
            bound = reached_by<16>(of_lane, top);
        }
        const int n = keep_reaching(held, bound, places);
        rank_places(places, n, top, sorted);
        kept = min(n, top);
    }
}

// The slices of a row, joined by one wave.
template <typename T>
__global__ __launch_bounds__(64) void join_slices_kernel(const T* __restrict__ x, const LogpParams p) {
    exhip_touch_args(p);
    __shared__ u64 places[kCandidates + 8], sorted[EXHIP_LOG_PROBABILITIES_TOP];
    const int lane = threadIdx.x;
    const size_t row = blockIdx.x;
    Sums all = {-INFINITY, 0.f, 0.f, 0.f};
    for (int i = lane; i < p.slices; i += 64) all = joined(all, p.part[row * p.slices + i]);
    if (p.top > 0) join_lists(p.part_top + row * p.slices * p.top, (size_t)p.slices * p.top, p.top, places, sorted);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) all = joined(all, from_lane(all, d));
    write_row(x + row * p.x_stride, p, row, all, sorted);
}

// How a row is split. What one group holds is not: 64 rows of 32000 halves with the 20 largest take 8.6 us in one launch, 11.2 in slices that a second joins,
// 4096 of them 70 and 71. Longer rows are in slices of four waves (300 x 100003 halves 17 us, 20 with groups of sixteen). The largest of many slices cost the
// second launch more than groups of eight waves cost the first one, which all but one wait twice: 300 x 100003 with the 64 largest 36 us (42 with four waves, 40
// with sixteen), one row of 262144 with 20 of them 10.6 (12.3 with four); of a few rows in 16 slices not yet, 8 x 131072 with 20 of them 11.4 (10.7).
void split(int m, int c, int top, int* slices, int* slice_len) {
    const bool few = top == 0 || (m <= 32 && c <= 16 * kSlice);
    const int most = c <= kMostSlice ? c : few ? kSlice : kLongSlice;
    *slices = (c - 1) / most + 1;
    const int len = (c - 1) / *slices + 1;
    *slice_len = (len + 7) / 8 * 8;
    *slices = (c - 1) / *slice_len + 1;
}

template <typename T, bool TOP>
void launch_slices(exhip_ctx* ctx, const T* x, const LogpParams& p) {
    const dim3 grid((unsigned)((size_t)p.m * p.slices));
    if (p.slice_len <= 512) hipLaunchKernelGGL((log_probabilities_kernel<T, 1, 8, TOP>), grid, dim3(64), 0, ctx->stream, x, p);
    else if (p.slice_len <= 2048) hipLaunchKernelGGL((log_probabilities_kernel<T, 1, 32, TOP>), grid, dim3(64), 0, ctx->stream, x, p);
    else if (p.slice_len <= kSlice) hipLaunchKernelGGL((log_probabilities_kernel<T, 4, 32, TOP>), grid, dim3(256), 0, ctx->stream, x, p);
    else if (p.slice_len <= kLongSlice) hipLaunchKernelGGL((log_probabilities_kernel<T, 8, 32, TOP>), grid, dim3(512), 0, ctx->stream, x, p);
    else hipLaunchKernelGGL((log_probabilities_kernel<T, 16, 32, TOP>), grid, dim3(1024), 0, ctx->stream, x, p);
}

bool sizes_ok(int m, int c, int top) { return m > 0 && c > 0 && top >= 0 && top <= EXHIP_LOG_PROBABILITIES_TOP && top <= c; }
bool one_launch(int m, int slices) { return (size_t)m * slices <= 0xffffffffu / 1024; }

template <typename T>
int log_probabilities(exhip_ctx* ctx, const char* name, const T* x, int x_stride, int m, int c, const int32_t* ids, int n_ids, float* log_p, float* entropy, int top,
                      int32_t* top_ids, float* top_log_p, void* workspace) {
    EXHIP_REQUIRE(ctx && x && workspace, "%s: NULL argument", name);
    EXHIP_REQUIRE(m > 0 && c > 0 && x_stride >= c, "%s: %d rows of %d values, %d apart", name, m, c, x_stride);
    EXHIP_REQUIRE(n_ids >= 0 && (n_ids == 0 ? !log_p : ids && log_p), "%s: %d classes asked of a row need ids and log_p, none need neither", name, n_ids);
    EXHIP_REQUIRE(sizes_ok(m, c, top) && (top == 0 ? !top_ids && !top_log_p : top_ids && top_log_p), "%s: the %d largest of %d classes: at most %d, with both results", name,
                  top, c, EXHIP_LOG_PROBABILITIES_TOP);
    EXHIP_REQUIRE(log_p || entropy || top, "%s: nothing is asked", name);
    EXHIP_REQUIRE((uintptr_t)x % sizeof(T) == 0 && ((uintptr_t)ids | (uintptr_t)log_p | (uintptr_t)entropy | (uintptr_t)top_ids | (uintptr_t)top_log_p) % 4 == 0 && (uintptr_t)workspace % 16 == 0,
                  "%s: an operand's address is not that of its type", name);
    LogpParams p = {ids, log_p, entropy, top_log_p, top_ids, nullptr, nullptr, m, c, x_stride, n_ids, top, 0, 0};
    split(m, c, top, &p.slices, &p.slice_len);
    EXHIP_REQUIRE(one_launch(m, p.slices), "%s: %d rows of %d values are more than one launch takes", name, m, c);
    if (p.slices > 1) {
        p.part = static_cast<Sums*>(workspace);
        p.part_top = reinterpret_cast<u64*>(p.part + (size_t)m * p.slices);
    }
    const exhip_on_device on(ctx->device);
    EXHIP_CHECK(on.error);
    if (top) launch_slices<T, true>(ctx, x, p);
    else launch_slices<T, false>(ctx, x, p);
    EXHIP_LAUNCH_CHECK();
    if (p.slices > 1) {
        hipLaunchKernelGGL(join_slices_kernel<T>, dim3(m), dim3(64), 0, ctx->stream, x, p);
        EXHIP_LAUNCH_CHECK();
    }
    return 0;
}

}  // namespace

extern "C" size_t exhip_log_probabilities_workspace(int m, int c, int top) {
    if (!sizes_ok(m, c, top)) {
        exhip_set_error("exhip_log_probabilities_workspace: %d rows of %d values, the %d largest", m, c, top);
        return 0;
    }
    int slices, slice_len;
    split(m, c, top, &slices, &slice_len);
    if (!one_launch(m, slices)) {
        exhip_set_error("exhip_log_probabilities_workspace: %d rows of %d values are more than one launch takes", m, c);
        return 0;
    }
    // Of the shortest slices that a row is ever split into, so that it is enough for fewer rows, classes or largest, whatever their own slices are.
    return c > kMostSlice ? (size_t)m * ((c - 1) / kSlice + 1) * (sizeof(Sums) + 8 * top) : 16;
}

extern "C" int exhip_log_probabilities_f32(exhip_ctx* ctx, const float* x, int x_stride, int m, int c, const int32_t* ids, int n_ids, float* log_p, float* entropy,
                                           int top, int32_t* top_ids, float* top_log_p, void* workspace) {
    return log_probabilities(ctx, "exhip_log_probabilities_f32", x, x_stride, m, c, ids, n_ids, log_p, entropy, top, top_ids, top_log_p, workspace);
}
extern "C" int exhip_log_probabilities_f16(exhip_ctx* ctx, const uint16_t* x, int x_stride, int m, int c, const int32_t* ids, int n_ids, float* log_p, float* entropy,
                                           int top, int32_t* top_ids, float* top_log_p, void* workspace) {
    return log_probabilities(ctx, "exhip_log_probabilities_f16", x, x_stride, m, c, ids, n_ids, log_p, entropy, top, top_ids, top_log_p, workspace);
}
