// Inner products in 8-bit integers: the row quantizer, the weights' layout, the product and the gated product, alone and by experts.
//
// A row's codes share a float32 scale, and so do those of an output's weights: neither takes part in the sums, which are those of v_mfma_i32_32x32x32_i8 and
// v_mfma_i32_16x16x64_i8 in 32 bits and exact for as many as 131071 values a row. A result is sum * row's scale * output's scale + bias, rounded in that order; which kernel
// takes a call, and how it cuts the sums, changes no bit of it. Weights are the first operand, rows of the input the second: a lane's results are then
// runs of four neighbouring outputs of one row.
#include <math.h>

#include <type_traits>

#include "i8_rows.h"
#include "inner.h"

namespace {

constexpr int kBlk = 128;                // values of a row that a step takes
constexpr int kTileBlock = 32 * kBlk;    // bytes of a tile's weights for them
constexpr int kMostInputs = 131071;      // 2^14 each, 2^31 - 1 at most together
constexpr int kMostStride = 1 << 22;     // of a row of codes
constexpr int kMostExperts = 1024;
constexpr size_t kRowsPastL2 = 128 << 20;  // half of the cache behind L2
constexpr float kLargest = 127.f;
constexpr float kLeastScale = 0x1p-100f;  // keeps 1 / scale finite and rows of zeros at zero
constexpr int kNonTemporal = 2;           // of a buffer load: past L2
constexpr unsigned kNoRow = 0x80000000u;  // beyond every view of rows: loads there give zeros

// ---- the quantizer ----
// x / scale to the nearest whole number, ties to the even one, exactly: the product with 1 / scale is less than one off, and what it leaves, x - r scale, is
// a multiple of the last place of scale / 2 and has no more bits than a float. A sum with 1.5 * 2^23 rounds to a whole number and has it in its low bits.
constexpr float kWhole = 0x1.8p23f;
__device__ __forceinline__ float nearly(float x, float inverse) { return __builtin_fmaf(x, inverse, kWhole); }
__device__ __forceinline__ float left_of(float x, float near, float scale) { return __builtin_fmaf(kWhole - near, scale, x); }
__device__ __forceinline__ float nearest(float x, float scale, float inverse) {
    const float near = nearly(x, inverse), left = left_of(x, near, scale), off = fabsf(left), half = 0.5f * scale;
    return off > half || (off == half && (__builtin_bit_cast(int, near) & 1)) ? near + (left > 0.f ? 1.f : -1.f) : near;
}
__device__ __forceinline__ int low_bytes(float a, float b, float c, float d) {
    const unsigned ab = __builtin_amdgcn_perm(__builtin_bit_cast(unsigned, b), __builtin_bit_cast(unsigned, a), 0x0c0c0400);
    const unsigned cd = __builtin_amdgcn_perm(__builtin_bit_cast(unsigned, d), __builtin_bit_cast(unsigned, c), 0x0c0c0400);
    return (int)__builtin_amdgcn_perm(cd, ab, 0x05040100);
}

// 16 bytes of a row a lane at a time, at any alignment of their type.
template <typename T>
struct Piece {
    static constexpr int kValues = 16 / sizeof(T);
    struct __attribute__((packed, aligned(sizeof(T)))) Packed {
        T v[kValues];
    };
    T v[kValues];
    template <bool PAST>
    __device__ __forceinline__ void load(const T* row, int at, int k) {  // zeros behind the row's end
        if (at + kValues <= k) {
            Packed p;
            if constexpr (PAST) p = __builtin_bit_cast(Packed, __builtin_nontemporal_load(reinterpret_cast<const v4i_any*>(row + at)));
            else p = *reinterpret_cast<const Packed*>(row + at);
#pragma unroll
            for (int e = 0; e < kValues; ++e) v[e] = p.v[e];
        } else {
#pragma unroll
            for (int e = 0; e < kValues; ++e) v[e] = at + e < k ? row[at + e] : T(0);
        }
    }
    __device__ __forceinline__ float most(float so_far) const {  // NaN stays, as the largest of all
#pragma unroll
        for (int e = 0; e < kValues; ++e) {
            const float a = fabsf(as_float(v[e]));
            so_far = so_far >= a || so_far != so_far ? so_far : a;
        }
        return so_far;
    }
    __device__ __forceinline__ void store(int8_t* row, int at, int k, float scale, float inverse) const {
        float near[kValues], off = 0.f;
#pragma unroll
        for (int e = 0; e < kValues; ++e) {
            near[e] = nearly(as_float(v[e]), inverse);
            off = fmaxf(off, fabsf(left_of(as_float(v[e]), near[e], scale)));
        }
        if (off >= 0.5f * scale)  // a tie, or a neighbour of one: 2 % of a wave's pieces
#pragma unroll
            for (int e = 0; e < kValues; ++e) near[e] = nearest(as_float(v[e]), scale, inverse);
        int codes[kValues / 4];
#pragma unroll
        for (int e = 0; e < kValues / 4; ++e) codes[e] = low_bytes(near[4 * e], near[4 * e + 1], near[4 * e + 2], near[4 * e + 3]);
        if (at + kValues <= k) {
            if constexpr (kValues == 8) *reinterpret_cast<v2i*>(row + at) = v2i{codes[0], codes[1]};
            else *reinterpret_cast<int*>(row + at) = codes[0];
        } else {
#pragma unroll
            for (int e = 0; e < kValues; ++e)
                if (at + e < k) row[at + e] = (int8_t)(codes[e / 4] >> (8 * (e % 4)));
        }
    }
};

// WAVES waves a row (a wave takes its own row where that is one), HELD pieces a lane that stay in registers between the largest value and the codes; what a longer
// row has behind them is read again. PAST: rows go past L2 (a kernel of its own: where both loads stand in one, the compiler makes one of them, without it).
template <typename T, int WAVES, int HELD, bool PAST>
__global__ __launch_bounds__(256) void quantize_rows_i8_kernel(const T* __restrict__ x, int x_stride, int m, int k, int8_t* __restrict__ y, int y_stride, float* __restrict__ scale) {
    constexpr int kStep = 64 * WAVES * Piece<T>::kValues;
    const int wave = threadIdx.x / 64, row = blockIdx.x * (4 / WAVES) + wave / WAVES;
    if (row >= m) return;  // a whole wave, and a whole group where several have a row
    const T* const from = x + (size_t)row * x_stride;
    const int first = threadIdx.x % (64 * WAVES) * Piece<T>::kValues;
    Piece<T> held[HELD];
#pragma unroll
    for (int i = 0; i < HELD; ++i) held[i].template load<PAST>(from, first + i * kStep, k);
    float most = 0.f;
#pragma unroll
    for (int i = 0; i < HELD; ++i) most = held[i].most(most);
    for (int at = first + HELD * kStep; at < k; at += kStep) {
        Piece<T> p;
        p.template load<PAST>(from, at, k);
        most = p.most(most);
    }
    // as whole numbers the bits of values that are not negative are in their order, and those of NaN above all
    int bits = __builtin_bit_cast(int, most);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) bits = max(bits, __shfl_xor(bits, d));
    if constexpr (WAVES > 1) {
        __shared__ int part[WAVES];
        if (threadIdx.x % 64 == 0) part[wave] = bits;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < WAVES; ++w) bits = max(bits, part[w]);
    }
    const bool fine = bits < 0x7f800000;
    const float s = fine ? fmaxf(__builtin_bit_cast(float, bits) / kLargest, kLeastScale) : __builtin_inff(), inverse = 1.f / s;
    if (threadIdx.x % (64 * WAVES) == 0) scale[row] = fine ? s : __builtin_nanf("");
    int8_t* const to = y + (size_t)row * y_stride;
    if (!fine) {
        for (int at = threadIdx.x % (64 * WAVES); at < k; at += 64 * WAVES) to[at] = 0;
        return;
    }
#pragma unroll
    for (int i = 0; i < HELD; ++i)
        if (first + i * kStep < k) held[i].store(to, first + i * kStep, k, s, inverse);
    for (int at = first + HELD * kStep; at < k; at += kStep) {
        Piece<T> p;
        p.template load<PAST>(from, at, k);
        p.store(to, at, k, s, inverse);
    }
}

// ---- the weights' layout ----
// Tiles of 32 outputs x 128 values, a tile row's blocks one after the other, an expert's tiles one after the other: [expert][tile][block][run of 16 values]
// [output][16 bytes]. A wave reads what a product of 32 outputs takes as one run of 1 KB. A gated tile has 16 outputs of the gate and the same 16 of the other
// projection, so that a lane has both sides of its outputs. Outputs and values that do not exist are zeros: what a row's codes are behind its end does not count.
__global__ __launch_bounds__(256) void pack_i8_kernel(const int8_t* __restrict__ w, const int8_t* __restrict__ w_up, int n, int k, int blocks, int tiles, size_t pieces,
                                                      v4i* __restrict__ packed) {
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= pieces) return;
    const int output = i % 32, run = i / 32 % 8;
    const size_t tile_block = i / 256, all = tile_block / blocks;
    const int block = tile_block % blocks, tile = all % tiles;
    const size_t expert = all / tiles;
    const int8_t* const from = w_up && output >= 16 ? w_up : w;
    const int row = w_up ? tile * 16 + output % 16 : tile * 32 + output, col = block * kBlk + run * 16;
    const int8_t* const src = from + (expert * n + row) * k + col;
    if (row < n && col + 16 <= k) {
        packed[i] = *reinterpret_cast<const v4i_any*>(src);
        return;
    }
    union { int8_t b[16]; v4i v; } u;
    for (int e = 0; e < 16; ++e) u.b[e] = row < n && col + e < k ? src[e] : 0;
    packed[i] = u.v;
}

// ---- the products ----
struct I8Params {
    const int8_t* x;
    const float* x_scale;
    const int8_t* w;
    const float *w_scale, *w_scale_up;  // of a gated product: the gate's, the other projection's
    const float *bias, *bias_up;
    float* y_f32;
    uint16_t* y_f16;
    const int *offsets, *rows;  // by experts: where each one's rows begin, and which of the input's each is (NULL: the same)
    int m, n, k, x_stride, y_stride, x_rows;
    int blocks, tiles;  // along k, and of 32 outputs (both projections') of one expert
    int gate, experts;
    int groups_n, groups_m;  // groups side by side along the outputs, and along the rows (the most there may be, by experts)
};

// Which rows a group takes, and whose weights.
struct Part {
    int expert, row0, rows, group_n;
};

// The tiles of ROWS rows. By experts each one's rows are cut by themselves, and every lane of a wave holds an expert, or a run of them where there are more than 64: the
// tiles of its own and of all up to them. (Offsets that do not rise count rows twice; the bound, beyond every launch, keeps the sums of such ones in range.)
template <bool GROUPED, int ROWS>
struct Tiles {
    int total;  // along the rows
    int own, upto, from, count;
    static __device__ __forceinline__ int offset(const I8Params& p, int expert) { return min(max(p.offsets[expert], 0), p.m); }
    static __device__ __forceinline__ int tiles_of(int rows) { return (int)(((unsigned)rows + ROWS - 1) / ROWS); }
    __device__ __forceinline__ explicit Tiles(const I8Params& p) {
        if constexpr (!GROUPED) {
            total = p.groups_m;
        } else {
            const int lane = threadIdx.x % 64, each = (p.experts + 63) / 64;
            own = from = count = 0;
            for (int e = lane * each; e < min((lane + 1) * each, p.experts); ++e) {
                from = offset(p, e);
                count = max(offset(p, e + 1) - from, 0);
                own = min(own + tiles_of(count), 1 << 24);
            }
            upto = own;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const int before = __shfl_up(upto, d);
                if (lane >= d) upto += before;
            }
            total = min(__builtin_amdgcn_readlane(upto, 63), p.groups_m);
        }
    }
    // the group's part; where there are groups_n * total of them. The tiles of an expert follow each other, so that its weights are read from memory once.
    __device__ __forceinline__ Part part(const I8Params& p) const {
        Part part;
        int at = place_of(blockIdx.x, p.groups_n * total), group_m;
        if constexpr (!GROUPED) {
            tile_at(at, p.groups_n, total, &part.group_n, &group_m);
            part.expert = 0;
            part.row0 = group_m * ROWS;
            part.rows = min(ROWS, p.m - part.row0);
        } else {
            const int of = __builtin_ctzll(__ballot(upto > at / p.groups_n));
            int begin = __builtin_amdgcn_readlane(from, of), rows = __builtin_amdgcn_readlane(count, of);
            at -= (__builtin_amdgcn_readlane(upto, of) - __builtin_amdgcn_readlane(own, of)) * p.groups_n;
            part.expert = of;
            if (p.experts > 64) {  // which one of the lane's
                const int each = (p.experts + 63) / 64;
                for (int e = of * each; e < min((of + 1) * each, p.experts); ++e) {
                    begin = offset(p, e);
                    rows = max(offset(p, e + 1) - begin, 0);
                    part.expert = e;
                    if (at < tiles_of(rows) * p.groups_n) break;
                    at -= tiles_of(rows) * p.groups_n;
                }
                begin = __builtin_amdgcn_readfirstlane(begin);
                rows = __builtin_amdgcn_readfirstlane(rows);
                at = __builtin_amdgcn_readfirstlane(at);
                part.expert = __builtin_amdgcn_readfirstlane(part.expert);
            }
            tile_at(at, p.groups_n, tiles_of(rows), &part.group_n, &group_m);
            part.row0 = begin + group_m * ROWS;
            part.rows = min(ROWS, rows - group_m * ROWS);
        }
        return part;
    }
};

// The input's rows that a group reads: a view, where each row begins in it, and each row's scale.
template <bool GROUPED>
struct Rows {
    __amdgpu_buffer_rsrc_t view;
    const float* scales;
    const int* index;
    int rows, x_rows, stride;
    __device__ __forceinline__ Rows(const I8Params& p, const Part& part) : index(nullptr), rows(part.rows), x_rows(p.x_rows), stride(p.x_stride) {
        const int end = (p.k + 15) / 16 * 16;
        if (GROUPED && p.rows) {
            index = p.rows + part.row0;
            scales = p.x_scale;
            view = uniform_view(p.x, (unsigned)(p.x_rows - 1) * p.x_stride + end);
        } else {
            scales = p.x_scale + part.row0;
            view = uniform_view(p.x + (size_t)part.row0 * p.x_stride, (unsigned)(rows - 1) * p.x_stride + end);
        }
    }
    // the row that the group's r-th is, -1 for none
    __device__ __forceinline__ int source(int r) const {
        if (r >= rows) return -1;
        if (!GROUPED || !index) return r;
        const int from = index[r];
        return (unsigned)from < (unsigned)x_rows ? from : -1;
    }
    __device__ __forceinline__ unsigned begin(int source_row) const { return source_row < 0 ? kNoRow : (unsigned)source_row * (unsigned)stride; }
    __device__ __forceinline__ float scale(int source_row) const { return source_row < 0 ? __builtin_nanf("") : scales[source_row]; }
};

__device__ __forceinline__ float result_of(int sum, float row, float output, float bias) { return __builtin_fmaf((float)sum * row, output, bias); }

// The activation of one side times the other, as exact as gated()'s functions in float32, without their branches and range checks.
// silu, sigmoid: 1 / (1 + e^-g) from the hardware's 2^x and 1 / x (one unit of the last place each). What the argument's rounding changes, up to |g| / 2 units, goes back in with the remainder
// of p ln 2 + g; one step of division, q + (n - d q) / d, leaves half a unit, and its fixup infinities. Below -87.3, where e^-g leaves float32, the value there stands: 2^-126, in silu 87 of it.
// gelu: g Phi(g), Phi(-a) = 2^(a P(a)) / 2 and Phi(a) = 1 - Phi(-a), P of degree 9 fitted to log2(2 Phi(-a)) / a over 0 to 6.5 for the least largest error of Phi. Nothing cancels for g < 0, where
// 1 + erf does: over gates of a normal distribution 0.9 of that form's error in norm, between -3 and -1 0.45, at -6 0.01. a P(a) goes on falling behind 6.5; Phi is 4e-11 there.
// (32768 rows of 1536 x 2048: silu 180 us, with expf and a division 188; gelu 182, with erff 320. What rounds each step to the hardware's unit alone takes 176 for silu and is five units off at -10.)
__device__ __forceinline__ float divided(float n, float d) {  // d of normal size
    const float r = __builtin_amdgcn_rcpf(d), q = n * r;
    return __builtin_amdgcn_div_fixupf(__builtin_fmaf(__builtin_fmaf(-d, q, n), r, q), d, n);
}
template <int GATE>
__device__ __forceinline__ float gated_value(float g, float u) {
    if constexpr (GATE == EXHIP_GATE_RELU) return (g > 0.f ? g : g != g ? g : 0.f) * u;
    if constexpr (GATE == EXHIP_GATE_GELU) {
        const float a = fabsf(g);
        float v = __builtin_fmaf(a, -0x1.d748fp-26f, 0x1.b91fb4p-21f);
        v = __builtin_fmaf(v, a, -0x1.61ec36p-17f);
        v = __builtin_fmaf(v, a, 0x1.35d58p-14f);
        v = __builtin_fmaf(v, a, -0x1.1b6deap-12f);
        v = __builtin_fmaf(v, a, -0x1.509986p-16f);
        v = __builtin_fmaf(v, a, 0x1.c8e2cep-8f);
        v = __builtin_fmaf(v, a, -0x1.adbb2ap-5f);
        v = __builtin_fmaf(v, a, -0x1.d63cb4p-2f);
        v = __builtin_fmaf(v, a, -0x1.26aeccp+0f);
        const float tail = 0.5f * __builtin_amdgcn_exp2f(v * a);
        return g * (g < 0.f ? tail : 1.f - tail) * u;
    }
    const float from = __builtin_elementwise_maximum(g, -87.3f), x = __builtin_elementwise_minimum(from, 104.f);  // NaN stays
    const float p = x * -1.44269504088896341f, left = __builtin_fmaf(p, -0.69314718055994531f, -x), e = __builtin_amdgcn_exp2f(p), d = 1.f + __builtin_fmaf(e, left, e);
    return GATE == EXHIP_GATE_SILU ? divided(from, d) * u : divided(u, d);
}
// `values` for an activation that is known when they are compiled: one choice in front of them all, which are then computed side by side (with a choice in each of them
// 4096 rows x 8 of 64 experts of 1536 x 2048 took 6 % longer, one group's 512 x 512 half as long again).
template <typename F>
__device__ __forceinline__ void by_gate(int gate, F values) {
    if (gate == EXHIP_GATE_SILU) values(std::integral_constant<int, EXHIP_GATE_SILU>{});
    else if (gate == EXHIP_GATE_GELU) values(std::integral_constant<int, EXHIP_GATE_GELU>{});
    else if (gate == EXHIP_GATE_RELU) values(std::integral_constant<int, EXHIP_GATE_RELU>{});
    else values(std::integral_constant<int, EXHIP_GATE_SIGMOID>{});
}

// ---- few rows, or few products ----
// A group takes TN x 16 outputs (of both projections), whole tiles or half of one, and 16 TM rows; its WK waves every WK-th block, with nothing between memory and their registers:
// the codes of D of a wave's blocks are on their way at a time. The sums meet in LDS, and every thread finishes four neighbouring outputs of a row. What bounds it is the memory:
// one row of the gated 11264 x 4096 takes 16.6 us, 5.6 TB/s of weights. Four waves a group, so that a CU has several groups, where there are many outputs (that row with eight waves 18.4 us);
// eight where one group a CU has all of them (4096 x 4096 5.2 us, with four 5.7), and then half a tile a group without an activation, so that more CUs have one (16 rows of 4096 x 11264
// 11.5 us, with whole tiles 14.3). More blocks on their way, or sixteen waves, measured no faster.
template <int TN, int TM, int WK, int D, bool PAST, bool GATED, bool GROUPED>
__global__ __launch_bounds__(64 * WK, 2) void i8_rows_kernel(const I8Params p) {
    exhip_touch_args(p);
    constexpr int kRows = 16 * TM, kSide = GATED ? 2 : 1;
    static_assert(TN % 2 == 0 || (TN == 1 && !GATED), "whole tiles, or half of one");
    constexpr int kTiles = (TN + 1) / 2;
    const Tiles<GROUPED, kRows> tiles(p);
    if ((int)blockIdx.x >= p.groups_n * tiles.total) return;
    const Part part = tiles.part(p);
    if (part.rows <= 0) return;  // offsets that do not rise
    const int lane = threadIdx.x % 64, wk = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), q = lane / 16, col = lane % 16;
    const int blocks = p.blocks, row_bytes = blocks * kTileBlock, tile0 = TN == 1 ? part.group_n / 2 : part.group_n * kTiles, last = p.tiles - 1;
    const __amdgpu_buffer_rsrc_t weights = uniform_view(p.w + ((size_t)part.expert * p.tiles + tile0) * row_bytes, (unsigned)(min(kTiles, p.tiles - tile0) * row_bytes));
    const Rows<GROUPED> rows(p, part);
    unsigned off[TM];
#pragma unroll
    for (int t = 0; t < TM; ++t) off[t] = rows.begin(rows.source(16 * t + col)) + q * 16;
    const int at = q * 512 + col * 16 + (TN == 1 ? part.group_n % 2 * 256 : 0);
    struct Codes {
        v4i w[TN][2], x[TM][2];
    } codes[D];
    auto request = [&](Codes& c, int b) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int i = 0; i < TN; ++i)
                c.w[i][h] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(weights, at + i % 2 * 256, min(i / 2, last - tile0) * row_bytes + b * kTileBlock + h * 2048, PAST ? kNonTemporal : 0));
#pragma unroll
            for (int t = 0; t < TM; ++t) c.x[t][h] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(rows.view, off[t] + b * kBlk + h * 64, 0, 0));
        }
    };
    v4i acc[TN][TM];
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int t = 0; t < TM; ++t) acc[i][t] = v4i{0, 0, 0, 0};
#pragma unroll
    for (int d = 0; d < D; ++d)
        if (wk + d * WK < blocks) request(codes[d], wk + d * WK);
    for (int first = wk; first < blocks; first += WK * D) {
#pragma unroll
        for (int d = 0; d < D; ++d) {
            const int b = first + d * WK;
            if (b >= blocks) break;
            const Codes c = codes[d];
            if (b + WK * D < blocks) request(codes[d], b + WK * D);
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < TN; ++i)
#pragma unroll
                    for (int t = 0; t < TM; ++t) acc[i][t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(c.w[i][h], c.x[t][h], acc[i][t], 0, 0, 0);
        }
    }
    constexpr int kWidth = TN * 16, kPitch = kWidth + 4, kThreads = 64 * WK, kQuads = kWidth / 4 / kSide;
    __shared__ __attribute__((aligned(16))) int joined[WK][kRows][kPitch];
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int t = 0; t < TM; ++t) *reinterpret_cast<v4i*>(&joined[wk][16 * t + col][i * 16 + q * 4]) = acc[i][t];
    __syncthreads();
    const size_t own = (size_t)part.expert * p.n;
    for (int i = threadIdx.x; i < kRows * kQuads; i += kThreads) {
        const int quad = i % kQuads, row = i / kQuads, j = part.group_n * (kWidth / kSide) + quad * 4;
        if (row >= part.rows || j >= p.n) continue;
        const float x_scale = rows.scale(rows.source(row));
        const v4f w_scale = four_of(p.w_scale + own, j, p.n), bias = four_of(p.bias ? p.bias + own : nullptr, j, p.n);
        const int from = GATED ? quad / 4 * 32 + quad % 4 * 4 : quad * 4;
        v4i sum = {0, 0, 0, 0}, sum_up = {0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < WK; ++k) {
            sum += *reinterpret_cast<const v4i*>(&joined[k][row][from]);
            if constexpr (GATED) sum_up += *reinterpret_cast<const v4i*>(&joined[k][row][from + 16]);
        }
        v4f v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = result_of(sum[e], x_scale, w_scale[e], bias[e]);
        if constexpr (GATED) {
            const v4f w_scale_up = four_of(p.w_scale_up + own, j, p.n), bias_up = four_of(p.bias_up ? p.bias_up + own : nullptr, j, p.n);
            by_gate(p.gate, [&](auto gate) {
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = gated_value<gate()>(v[e], result_of(sum_up[e], x_scale, w_scale_up[e], bias_up[e]));
            });
        }
        const size_t to = (size_t)(part.row0 + row) * p.y_stride + j;
        const bool whole = j + 4 <= p.n;
        if (p.y_f32) {
            if (whole) *reinterpret_cast<v4f_any*>(p.y_f32 + to) = v;
            else store_cut(p.y_f32 + to, v, p.n - j);
        }
        if (p.y_f16) {
            if (whole) *reinterpret_cast<v4h_any*>(p.y_f16 + to) = __builtin_convertvector(v, v4h);
            else store_cut(p.y_f16 + to, v, p.n - j);
        }
    }
}

// ---- many rows ----
// Results of a group of WN x WM waves, 32 TN outputs (of both projections) and 32 TM rows a wave, from products of 32 x 32: a lane's sums are runs of four neighbouring
// outputs, output 8 run + 4 (lane / 32) and on of each 32, of row lane % 32. They go through LDS, so that whole lines are stored: all rows at once, or those of half of
// the waves after the other's where float32 results of all of them do not fit.
typedef int v16i __attribute__((ext_vector_type(16)));

template <int WIDTH, int ROWS>
struct __attribute__((aligned(16))) Scales {  // of a group's outputs and rows, in LDS
    float output[WIDTH], output_up[WIDTH], bias[WIDTH], bias_up[WIDTH], row[ROWS];
};

template <typename O, int WN, int WM, int TM, int FOURS, int ROOM>
__device__ __forceinline__ void store_group(O* y, size_t stride, const v4f (&v)[FOURS][TM], const Part& part, int j0, int n, int wn, int wm, int lane, char* lds) {
    constexpr int kOwn = FOURS * 8, kWidth = kOwn * WN, kAll = 32 * TM * WM, kPasses = kAll * kWidth * (int)sizeof(O) > ROOM ? 2 : 1, kRows = kAll / kPasses;
    static_assert(kRows * kWidth * sizeof(O) <= ROOM);
#pragma unroll
    for (int pass = 0; pass < kPasses; ++pass) {
        __syncthreads();
#pragma unroll
        for (int t = 0; t < TM; ++t) {
            const int row = (wm * TM + t) * 32 - pass * kRows;  // 32 rows lie in one pass
            if (row < 0 || row >= kRows) continue;
#pragma unroll
            for (int i = 0; i < FOURS; ++i) {
                char* const to = place_in_rows<O, kWidth>(lds, row + lane % 32, wn * kOwn + i * 8 + lane / 32 * 4);
                if constexpr (sizeof(O) == 4) *reinterpret_cast<v4f*>(to) = v[i][t];
                else *reinterpret_cast<v4h*>(to) = __builtin_convertvector(v[i][t], v4h);
            }
        }
        __syncthreads();
        store_rows<O, kWidth, kRows, 64 * WN * WM>(lds, y, stride, part.row0 + pass * kRows, part.rows - pass * kRows, j0, n, ((uintptr_t)y | stride * sizeof(O)) % 128 == 0);
    }
}

template <int WN, int WM, int TN, int TM, bool GATED, int ROOM, int WIDTH, int ROWS>
__device__ __forceinline__ void write_group(const I8Params& p, const Part& part, const v16i (&acc)[TN][TM], int wn, int wm, int lane, char* lds, const Scales<WIDTH, ROWS>& scales) {
    constexpr int kFours = TN * (GATED ? 2 : 4), kOwn = kFours * 8;
    static_assert(kOwn * WN == WIDTH);
    const int at = wn * kOwn + lane / 32 * 4, row = wm * TM * 32 + lane % 32;
    v4f v[kFours][TM];
    auto finish = [&](auto gate) {
#pragma unroll
        for (int i = 0; i < kFours; ++i) {
            const v4f output = *reinterpret_cast<const v4f*>(scales.output + at + i * 8), bias = *reinterpret_cast<const v4f*>(scales.bias + at + i * 8);
            v4f output_up = output, bias_up = bias;
            if constexpr (GATED) {
                output_up = *reinterpret_cast<const v4f*>(scales.output_up + at + i * 8);
                bias_up = *reinterpret_cast<const v4f*>(scales.bias_up + at + i * 8);
            }
#pragma unroll
            for (int t = 0; t < TM; ++t) {
                const float x_scale = scales.row[row + t * 32];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if constexpr (GATED) {
                        const float g = result_of(acc[i / 2][t][i % 2 * 4 + e], x_scale, output[e], bias[e]);
                        v[i][t][e] = gated_value<gate()>(g, result_of(acc[i / 2][t][i % 2 * 4 + 8 + e], x_scale, output_up[e], bias_up[e]));
                    } else {
                        v[i][t][e] = result_of(acc[i / 4][t][i % 4 * 4 + e], x_scale, output[e], bias[e]);
                    }
                }
            }
        }
    };
    if constexpr (GATED) by_gate(p.gate, finish);
    else finish(std::integral_constant<int, 0>{});
    const int j0 = part.group_n * WIDTH;
    if (p.y_f32) store_group<float, WN, WM, TM, kFours, ROOM>(p.y_f32, p.y_stride, v, part, j0, p.n, wn, wm, lane, lds);
    if (p.y_f16) store_group<uint16_t, WN, WM, TM, kFours, ROOM>(p.y_f16, p.y_stride, v, part, j0, p.n, wn, wm, lane, lds);
}

// A group of WN x WM waves takes 32 TN WN outputs and 32 TM WM rows. Rows' codes come straight into LDS, BUFFERS - 1 blocks ahead; a wave's weights from L2 straight into
// registers, D blocks ahead, those of a step of 32 values as soon as that step is done with the ones in their place. Rows are read from LDS a step before their products, or a
// block where a step's products are few, and loads stand between the products one by one. A block's one barrier, at its start, says that the next block's rows are there and that
// the last block's buffer may be filled.
// Two groups of 128 rows x 256 outputs a CU are what measured fastest for many rows: 8192 x 8192 x 4096 in 213 to 227 us, by the box, 2.4 to 2.6 POP/s, where the library's int8 product takes
// 290 to 296. The card's power bounds it: with codes of 0 the same launch takes 149 us beside 221, and the matrix cores are as many cycles busy in both. Eight waves a group with 256 rows took 8 % longer (nothing runs beside
// a group's results), four with 64 x 256 outputs each 5 %, and groups that go on to their next tile, its first blocks on their way while results are stored, 2 to 5 %. Few rows are
// bound by what a CU draws, 85 bytes a ns: 64 rows x 256 outputs, 64 x 128, and 32 rows with weights eight blocks ahead.
constexpr int most_on_their_way(int loads) { return loads < 63 ? loads : 63; }  // as many as a wait can name

template <int TN, int TM, int WN, int WM, int BUFFERS, int D, bool GATED, bool GROUPED>
__global__ __launch_bounds__(64 * WN * WM, 2) void i8_wide_kernel(const I8Params p) {
    exhip_touch_args(p);
    constexpr int kWaves = WN * WM, kRows = 32 * TM * WM, kBuffers = BUFFERS, kBuffer = kRows * kBlk, kLoads = kRows / 8 / kWaves, kWidth = TN * WN * (GATED ? 16 : 32), kProducts = TN * TM;
    constexpr int kAhead = kProducts < 4 ? 4 * TM : TM;  // pieces of rows on their way from LDS: a step's, or a block's where a step's products are too few to wait behind
    static_assert(D * 4 * TM % (2 * kAhead) == 0 && D >= kBuffers - 3);
    constexpr int kResults = kRows * kWidth * 2, kRoom = kBuffers * kBuffer > kResults ? kBuffers * kBuffer : kResults;
    __shared__ __attribute__((aligned(16))) char staged[kRoom];
    __shared__ Scales<kWidth, kRows> scales;
    const Tiles<GROUPED, kRows> tiles(p);
    if ((int)blockIdx.x >= p.groups_n * tiles.total) return;
    const Part part = tiles.part(p);
    if (part.rows <= 0) return;  // offsets that do not rise
    const unsigned lds0 = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char*)staged;
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), wn = wave % WN, wm = wave / WN;
    const int blocks = p.blocks, row_bytes = blocks * kTileBlock, tile0 = (part.group_n * WN + wn) * TN, first = min(tile0, p.tiles - 1);
    const __amdgpu_buffer_rsrc_t weights = uniform_view(p.w + ((size_t)part.expert * p.tiles + first) * row_bytes, (unsigned)(min(TN, p.tiles - first) * row_bytes));
    const Rows<GROUPED> rows(p, part);
    // A wave stages 8 kLoads rows, eight with a load: lane l holds piece (l % 8) ^ (l / 8) of row l / 8, so that a piece of eight neighbouring rows lies in all banks.
    // Pieces behind a row's end, in its last block, are not loaded (the view's bounds do not see the block's offset).
    const int staged_piece = ((lane % 8) ^ (lane / 8)) * 16, staged_blocks = i8_blocks_of_piece(p.k, staged_piece);
    unsigned off[kLoads];
#pragma unroll
    for (int j = 0; j < kLoads; ++j) off[j] = rows.begin(rows.source((wave * kLoads + j) * 8 + lane / 8)) + staged_piece;
    auto stage = [&](int buffer, int j) {  // behind the last block zeros, which nothing reads
        load16_to_lds(rows.view, buffer < staged_blocks ? off[j] : kNoRow, buffer * kBlk, lds0 + buffer % kBuffers * kBuffer + (wave * kLoads + j) * 1024);
    };
    v4i w[D][4][TN];
    auto request = [&](v4i (&w)[4][TN], int b, int s, int i) {
        w[s][i] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(weights, b < blocks ? lane * 16 : kNoRow, min(i, p.tiles - 1 - first) * row_bytes + b * kTileBlock + s * 1024, 0));
    };
    // scales and biases, for the end
    for (int r = threadIdx.x; r < kRows; r += 64 * kWaves) scales.row[r] = rows.scale(rows.source(r));
    for (int r = threadIdx.x; r < kWidth; r += 64 * kWaves) {
        const size_t j = (size_t)part.expert * p.n + min(part.group_n * kWidth + r, p.n - 1);
        scales.output[r] = p.w_scale[j];
        scales.bias[r] = p.bias ? p.bias[j] : 0.f;
        if constexpr (GATED) {
            scales.output_up[r] = p.w_scale_up[j];
            scales.bias_up[r] = p.bias_up ? p.bias_up[j] : 0.f;
        }
    }
    v16i acc[TN][TM];
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int t = 0; t < TM; ++t)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][t][e] = 0;
#pragma unroll
    for (int j = 0; j < (kBuffers - 1) * kLoads; ++j) stage(j / kLoads, j % kLoads);
#pragma unroll
    for (int s = 0; s < 4 * D; ++s)
#pragma unroll
        for (int i = 0; i < TN; ++i) request(w[s / 4], s / 4, s % 4, i);
    auto arrive = [&] {
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(most_on_their_way((kBuffers - 2) * kLoads + 4 * TN * D)) : "memory");
    arrive();
    const int at = (wm * TM * 32 + lane % 32) * kBlk + ((lane / 32) ^ (lane % 8)) * 16;
    auto rows_from = [&](int b, int s, int t) { return *reinterpret_cast<const v4i*>(staged + b % kBuffers * kBuffer + (at ^ (s * 32)) + t * 32 * kBlk); };
    v4i x[2 * kAhead];
#pragma unroll
    for (int f = 0; f < kAhead; ++f) x[f] = rows_from(0, f / TM, f % TM);
    auto block = [&](v4i (&w)[4][TN], int b, int ring) {  // `ring`: where in x its rows begin
        // all but the loads of the block before (and the first ones' weights)
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(most_on_their_way((kBuffers - 3) * (kLoads + 4 * TN))) : "memory");
        arrive();
#pragma unroll
        for (int s = 0; s < 4; ++s) {
#pragma unroll
            for (int u = 0; u < kProducts; ++u) {
                const int t = u / TN, i = u % TN, f = s * TM + t, ahead = f + kAhead;
                if (i == 0) x[(ring + ahead) % (2 * kAhead)] = ahead < 4 * TM ? rows_from(b, ahead / TM, ahead % TM) : rows_from(b + 1, ahead / TM - 4, ahead % TM);
                if (u == kProducts / 4)
#pragma unroll
                    for (int j = s * kLoads / 4; j < (s + 1) * kLoads / 4; ++j) stage(b + kBuffers - 1, j);
                acc[i][t] = __builtin_amdgcn_mfma_i32_32x32x32_i8(w[s][i], x[(ring + f) % (2 * kAhead)], acc[i][t], 0, 0, 0);
                if (u >= kProducts - TN) request(w, b + D, s, u - (kProducts - TN));
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    };
    for (int first_block = 0; first_block < blocks; first_block += D)
#pragma unroll
        for (int d = 0; d < D; ++d)
            if (first_block + d < blocks) block(w[d], first_block + d, d * 4 * TM % (2 * kAhead));
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // what was staged behind the end, in front of the results' barrier
    write_group<WN, WM, TN, TM, GATED, kRoom>(p, part, acc, wn, wm, lane, staged, scales);
}

int blocks_of(int v) { return v / kBlk + (v % kBlk != 0); }
int tiles_of(int n, bool gated_product) { return gated_product ? (n + 15) / 16 : (n + 31) / 32; }
bool sizes_ok(int n, int k) { return n > 0 && k > 0 && n <= (1 << 24) && k <= kMostInputs; }
constexpr char kSizes[] = "sizes are positive, at most 2^24 outputs of 131071 inputs";

template <typename T>
int quantize_rows(exhip_ctx* ctx, const char* name, const T* x, int x_stride, int m, int k, int8_t* y, int y_stride, float* scale) {
    EXHIP_REQUIRE(ctx && x && y && scale, "%s: NULL argument", name);
    EXHIP_REQUIRE(m > 0 && k > 0 && k <= kMostStride && x_stride >= k, "%s: %d rows of %d values, %d apart: sizes are positive, a row at most 2^22 values", name, m, k, x_stride);
    EXHIP_REQUIRE(m <= 1 << 23, "%s: %d rows are more than one launch takes", name, m);
    EXHIP_REQUIRE(y_stride >= k && y_stride % 16 == 0 && y_stride <= kMostStride && aligned(y, 16), "%s: rows of codes begin on 16 bytes and hold the row (stride %d)", name, y_stride);
    EXHIP_REQUIRE(aligned(x, sizeof(T)) && aligned(scale, 4), "%s: an operand's address is not that of its type", name);
    const exhip_on_device on(ctx->device);
    EXHIP_CHECK(on.error);
    constexpr int kWave = 64 * Piece<T>::kValues;
    auto run = [&](auto kernel, int rows) { hipLaunchKernelGGL(kernel, dim3((m - 1) / rows + 1), dim3(256), 0, ctx->stream, x, x_stride, m, k, y, y_stride, scale); };
    // Rows that are read once, and that neither L2 nor the cache behind it, 256 MB, holds together with what else a program has under way, go past L2: 8000 x 5001 floats 38.4 -> 33.8 us,
    // 60000 x 700 40.7 -> 34.5, 65536 x 8192 halves 286 -> 271. Where they are still in that cache it is the longer way: the 8000 x 5001 once more 30.2 -> 33.6, 8192 x 2048 13.9 -> 16.5; and for
    // half rows with a wave each (60000 x 1500 56 -> 54 to 63) and rows that are read again (3000 x 16000 floats 59 -> 61).
    constexpr bool kFloats = sizeof(T) == 4;
    const bool past = (size_t)m * k * sizeof(T) > kRowsPastL2 && (kFloats || k > 3 * kWave) && k <= 32 * kWave;
    // A kernel holds the whole row where there is one that does: with a piece to read again 4096 rows of 5120 floats take 18.7 to 22.9 us, held in six 17.6, one row of 6144 halves 4.0 and 3.6;
    // every piece that a row does not fill costs 0.1 us for a float row alone and 0.3 for a half one, 8 % for each of 16384 rows of one. Up to three waves' values the row has one wave where
    // there are so many rows that a group's barrier costs more than its four times as many waves give: 768 floats 3.2 us with four waves and 3.3 with one at 520 rows, 4.1 and 3.6 at 2048;
    // 1024 halves 3.5 and 4.1 at 768 rows, 5.1 and 4.6 at 2560; 1536 halves 6.6 and 7.2 at 3500, 6.8 and 6.4 at 4096 that stay in cache, 18.0 and 16.4 at 16384.
    if (k <= kWave) run(quantize_rows_i8_kernel<T, 1, 1, false>, 4);
    else if (k <= 2 * kWave && m > (kFloats ? 512 : 2048)) run(past ? quantize_rows_i8_kernel<T, 1, 2, kFloats> : quantize_rows_i8_kernel<T, 1, 2, false>, 4);
    else if (k <= 3 * kWave && m > (kFloats ? 512 : 3500)) run(past ? quantize_rows_i8_kernel<T, 1, 3, kFloats> : quantize_rows_i8_kernel<T, 1, 3, false>, 4);
    else if (k <= 4 * kWave) run(past ? quantize_rows_i8_kernel<T, 4, 1, true> : quantize_rows_i8_kernel<T, 4, 1, false>, 1);
    else if (k <= 8 * kWave) run(past ? quantize_rows_i8_kernel<T, 4, 2, true> : quantize_rows_i8_kernel<T, 4, 2, false>, 1);
    else if (k <= 12 * kWave) run(past ? quantize_rows_i8_kernel<T, 4, 3, true> : quantize_rows_i8_kernel<T, 4, 3, false>, 1);
    else if (k <= 16 * kWave) run(past ? quantize_rows_i8_kernel<T, 4, 4, true> : quantize_rows_i8_kernel<T, 4, 4, false>, 1);
    else if (k <= 24 * kWave) run(past ? quantize_rows_i8_kernel<T, 4, 6, true> : quantize_rows_i8_kernel<T, 4, 6, false>, 1);
    else run(past ? quantize_rows_i8_kernel<T, 4, 8, true> : quantize_rows_i8_kernel<T, 4, 8, false>, 1);
    EXHIP_LAUNCH_CHECK();
    return 0;
}

template <typename K>
int launch(exhip_ctx* ctx, K kernel, I8Params p, int halves, int rows, int threads) {
    p.groups_n = (2 * p.tiles + halves - 1) / halves;
    // By experts each one's rows are cut by themselves: at most rows - 1 missing in each, and no more tiles than rows.
    const long long most = p.offsets ? ((long long)p.m + (long long)p.experts * (rows - 1)) / rows : (p.m - 1) / rows + 1;
    const long long groups_m = most < p.m ? most : p.m, groups = p.groups_n * groups_m;
    EXHIP_REQUIRE(groups <= 0x7fffffff / threads, "inner product: %d rows of %d outputs are more than one launch takes", p.m, p.n);
    p.groups_m = (int)groups_m;
    const exhip_on_device on(ctx->device);
    EXHIP_CHECK(on.error);
    hipLaunchKernelGGL(kernel, dim3((unsigned)groups), dim3(threads), 0, ctx->stream, p);
    EXHIP_LAUNCH_CHECK();
    return 0;
}

// One way to run a product: how many 16 outputs (of both projections) and rows a group takes, how many groups a CU runs at once, how many waves share a group's blocks, and seven figures of
// what a launch takes, in us: `start`; each time that all CUs are given groups, `round`, and for each block of one wave `alone`, or `share` for each group on a CU where that is more;
// `gate` for an activation, each time; but no less than reading the weights from memory and what groups read from L2, weights again and the rows there are, at so many bytes a us.
// The figures are fitted, all of a list's together, to which form is the fastest: what never bounds a form among the shapes (memory at 12.75 TB/s, L2 at 200) has a figure that says so and no more,
// and the times that they give are not those of launches.
struct Form {
    int (*run)(exhip_ctx*, const I8Params&);
    int halves, rows, at_once, split;
    float start, round, alone, share, memory, gate, l2;
};
constexpr long long kManyWeights = 40 << 20;
template <int TN, int TM, int WK, int D, bool GATED, bool GROUPED>
int run_rows(exhip_ctx* ctx, const I8Params& p) {
    // Weights that are read once, by the one tile of rows that there is, and are many: past L2 (one row of the gated 11264 x 4096 18.3 -> 16.5 us, its 8 of 64 experts of 1536 x 2048 11.5 -> 8.8;
    // 4096 x 4096 would take 5.35 instead of 5.25). How many rows an expert has, and which have any, is not known here: a tile each on average, and as many experts as there are rows, is what is
    // expected. Where rows are spread so (1024 rows over 256 experts of 1024 x 2048, gated) it saves 5 to 10 %; where one or two experts have all of them and the same weights are read for many
    // tiles it costs 0 to 6 % for those 1024 and 512 rows, 1 to 2 us for 16 rows x 2 of 16 experts of 4096 x 4096 (10.2 -> 11.7).
    const bool once = GROUPED ? p.m <= p.experts * 4 * TM : p.m <= 16 * TM;
    if (once && (long long)(p.m < p.experts ? p.m : GROUPED ? p.experts : 1) * p.tiles * p.blocks * kTileBlock >= kManyWeights)
        return launch(ctx, i8_rows_kernel<TN, TM, WK, D, true, GATED, GROUPED>, p, TN, 16 * TM, 64 * WK);
    return launch(ctx, i8_rows_kernel<TN, TM, WK, D, false, GATED, GROUPED>, p, TN, 16 * TM, 64 * WK);
}
template <int TN, int TM, int WN, int WM, int BUFFERS, int D, bool GATED, bool GROUPED>
int run_wide(exhip_ctx* ctx, const I8Params& p) {
    return launch(ctx, i8_wide_kernel<TN, TM, WN, WM, BUFFERS, D, GATED, GROUPED>, p, 2 * TN * WN, 32 * TM * WM, 64 * WN * WM);
}
// Chosen so that the form with the least of these times is as near to the fastest as it can be over 952 products and 700 products by experts of 1 to 8192 rows, 64 to 16384
// outputs and inputs and 2 to 256 experts, those of at most 64 rows counted twice (perf/inner_i8_forms.py times the forms and fits the figures): it takes 1.1 % and 1.4 % longer on average, 26 % at
// most, and over 109 and 125 others of these sizes 1.2 % and 1.8 %, 22 % at most. Beyond them, up to the most inputs, 250000 outputs and 1024 experts, 4.5 % over 25 products, 38 % at most (64 rows
// of 130000 gated outputs), and 6.7 % over 16 by experts, 76 % at most (16 rows x 8 of 1024 experts: small tiles, whose groups each search the offsets). Without any one form of the first list
// some product would take 6 to 47 % longer, without one of the second 12 to 32 %.
template <bool GATED>
constexpr Form kPlain[] = {
    {run_rows<GATED ? 2 : 1, 1, 8, 2, GATED, false>, GATED ? 2 : 1, 16, 2, 8, 1.91f, 0.98f, 0.44f, 0.55f, 6.81e6f, 0.2f, 16.53e6f},
    {run_rows<2, 1, 4, 2, GATED, false>, 2, 16, 5, 4, 2.14f, 0.58f, 0.49f, 0.31f, 12.75e6f, 0.17f, 13.59e6f},
    {run_rows<2, 2, 4, 2, GATED, false>, 2, 32, 4, 4, 2.44f, 0.36f, 0.02f, 0.53f, 6.92e6f, 0.06f, 24.24e6f},
    {run_rows<4, 1, 4, 2, GATED, false>, 4, 16, 3, 4, 2.33f, 1.07f, 0.5f, 0.45f, 5.3e6f, 0.f, 24.76e6f},
    {run_rows<4, 2, 4, 1, GATED, false>, 4, 32, 3, 4, 2.63f, 0.17f, 0.65f, 0.87f, 6.47e6f, 0.f, 23.95e6f},
    {run_rows<4, 4, 4, 1, GATED, false>, 4, 64, 2, 4, 4.8f, 0.1f, 0.85f, 0.98f, 7.08e6f, 0.16f, 42.56e6f},
    {run_wide<1, 1, 2, 1, 8, 8, GATED, false>, 4, 32, 4, 1, 1.45f, 2.09f, 0.05f, 0.16f, 2.64e6f, 5.33f, 19.75e6f},
    {run_wide<1, 1, 4, 1, 4, 4, GATED, false>, 8, 32, 4, 1, 1.09f, 1.98f, 0.03f, 0.28f, 4.3e6f, 0.12f, 28e6f},
    {run_wide<1, 2, 4, 1, 4, 4, GATED, false>, 8, 64, 2, 1, 1.26f, 1.82f, 0.41f, 0.33f, 5.45e6f, 0.f, 30.7e6f},
    {run_wide<2, 2, 4, 1, 5, 2, GATED, false>, 16, 64, 3, 1, 0.57f, 4.26f, 0.07f, 0.43f, 2.65e6f, 0.14f, 21.42e6f},
    {run_wide<2, 4, 4, 1, 4, 1, GATED, false>, 16, 128, 2, 1, 0.87f, 4.51f, 0.67f, 0.62f, 4.83e6f, 0.85f, 200e6f},
};
template <bool GATED>
constexpr Form kGrouped[] = {
    {run_rows<2, 1, 4, 2, GATED, true>, 2, 16, 5, 4, 2.88f, 1.05f, 0.16f, 0.44f, 6.27e6f, 0.43f, 18.35e6f},
    {run_rows<4, 1, 4, 2, GATED, true>, 4, 16, 3, 4, 2.83f, 0.68f, 0.42f, 0.93f, 5.38e6f, 0.04f, 29.14e6f},
    {run_rows<4, 2, 4, 1, GATED, true>, 4, 32, 3, 4, 3.4f, 0.87f, 0.02f, 1.12f, 6.34e6f, 0.08f, 19.34e6f},
    {run_wide<1, 1, 4, 1, 4, 4, GATED, true>, 8, 32, 4, 1, 3.36f, 1.96f, 0.41f, 0.25f, 6.04e6f, 0.38f, 33.05e6f},
    {run_wide<1, 2, 4, 1, 4, 4, GATED, true>, 8, 64, 2, 1, 2.33f, 2.75f, 0.1f, 0.49f, 5.5e6f, 0.77f, 17.46e6f},
    {run_wide<2, 2, 4, 1, 5, 2, GATED, true>, 16, 64, 3, 1, 2.8f, 1.93f, 0.47f, 0.78f, 5.97e6f, 1.34f, 27.32e6f},
    {run_wide<2, 4, 4, 1, 4, 1, GATED, true>, 16, 128, 2, 1, 3.1f, 4.97f, 1.14f, 0.89f, 5.96e6f, 2.17f, 39.69e6f},
};

constexpr int kCus = 256;

// How many `of` (a power of two) hold v > 0: the choice is made for every row of a serving program, and divisions are most of it.
int in_all(int v, int of) { return ((v - 1) >> __builtin_ctz(of)) + 1; }
float larger(float a, float b) { return a > b ? a : b; }  // (fmaxf is a call)

// What a launch of a form takes, in us; `experts` that have rows, 1 for a product without.
float time_of(const Form& f, const I8Params& p, float experts, bool gated_product) {
    const float m = (float)p.m;
    // By experts the rows of each are not known here: as many have rows as would have by chance, and the last tile of each is half full.
    const float tiles_m = !p.offsets ? (float)in_all(p.m, f.rows) : larger(experts, m > 0.25f * (float)f.rows * experts ? m / (float)f.rows + 0.5f * experts : 0.f);
    const float groups_n = (float)in_all(2 * p.tiles, f.halves), groups = groups_n * tiles_m, all = (float)p.blocks, blocks = (float)in_all(p.blocks, f.split), gate = gated_product ? f.gate : 0.f;
    const int down = (int)((groups < 1e9f ? groups : 1e9f) * (1.f / kCus)), times = down + ((float)down * kCus < groups ? 1 : 0), full = times / f.at_once, rest = times - full * f.at_once;
    float us = f.start + (float)full * (f.round + blocks * larger(f.alone, (float)f.at_once * f.share)) + gate * (float)times;
    if (rest > 0) us += f.round + blocks * larger(f.alone, (float)rest * f.share);
    const float weights = experts * (float)p.tiles * all * (float)kTileBlock;
    const float again = larger(0.f, all * (groups * (float)(f.halves * (kTileBlock / 2)) + groups_n * m * (float)kBlk) - weights);
    return larger(us, f.start + 1.f + gate + weights / f.memory + again / f.l2);
}

template <int N>
int run_best(exhip_ctx* ctx, const I8Params& p, const Form (&forms)[N], bool gated_product) {
    const int pinned = g_exhip_options.i8_form;
    int best = pinned < N ? pinned - 1 : N - 1;
    if (pinned <= 0) {
        const float experts = p.offsets ? (float)p.experts * (1.f - expf(-(float)p.m / (float)p.experts)) : 1.f;
        float least = 0.f;
        for (int i = 0; i < N; ++i) {
            const float us = time_of(forms[i], p, experts, gated_product);
            if (i == 0 || us < least) {
                least = us;
                best = i;
            }
        }
    }
    return forms[best].run(ctx, p);
}

struct Experts {  // of a product by experts
    int count;
    const int32_t *offsets, *rows;
    int x_rows;
};

int product(exhip_ctx* ctx, const char* name, const exhip_i8_desc* d, const Experts* by, const int8_t* x, const float* x_scale, const void* w, const float* w_scale, const float* w_scale_up,
            const float* bias, const float* bias_up, int gate, bool gated_product, float* y_f32, uint16_t* y_f16) {
    EXHIP_REQUIRE(ctx && d && x && x_scale && w && w_scale && (!gated_product || w_scale_up) && (!by || by->offsets), "%s: NULL argument", name);
    EXHIP_REQUIRE(d->m > 0 && sizes_ok(d->n_out, d->k_in), "%s: %d rows, %d outputs, %d inputs: %s", name, d->m, d->n_out, d->k_in, kSizes);
    EXHIP_REQUIRE(d->x_stride >= d->k_in && d->x_stride % 16 == 0 && d->x_stride <= kMostStride && aligned(x, 16),
                  "%s: rows of codes begin on 16 bytes and hold the row (stride %d)", name, d->x_stride);
    EXHIP_REQUIRE(d->y_stride >= d->n_out, "%s: result rows of %d values are %d apart", name, d->n_out, d->y_stride);
    EXHIP_REQUIRE(aligned(w, 16) && aligned(x_scale, 4) && aligned(w_scale, 4) && aligned(w_scale_up, 4) && aligned(bias, 4) && aligned(bias_up, 4),
                  "%s: an operand's address is not that of its type", name);
    EXHIP_REQUIRE((y_f32 || y_f16) && aligned(y_f32, 4) && aligned(y_f16, 2), "%s: no result, or one whose address is not that of its type", name);
    if (gated_product) {
        EXHIP_REQUIRE(!bias == !bias_up, "%s: both projections have a bias or neither", name);
        EXHIP_REQUIRE(gate >= EXHIP_GATE_SILU && gate <= EXHIP_GATE_RELU, "%s: unknown activation %d", name, gate);
    }
    I8Params p = {};
    p.x = x;
    p.x_scale = x_scale;
    p.w = static_cast<const int8_t*>(w);
    p.w_scale = w_scale;
    p.w_scale_up = w_scale_up;
    p.bias = bias;
    p.bias_up = bias_up;
    p.y_f32 = y_f32;
    p.y_f16 = y_f16;
    p.m = p.x_rows = d->m;
    p.n = d->n_out;
    p.k = d->k_in;
    p.x_stride = d->x_stride;
    p.y_stride = d->y_stride;
    p.blocks = blocks_of(d->k_in);
    p.tiles = tiles_of(d->n_out, gated_product);
    p.gate = gate;
    if (!by) return gated_product ? run_best(ctx, p, kPlain<true>, true) : run_best(ctx, p, kPlain<false>, false);
    EXHIP_REQUIRE(by->count > 0 && by->count <= kMostExperts, "%s: %d experts: 1 to %d", name, by->count, kMostExperts);
    EXHIP_REQUIRE(aligned(by->offsets, 4) && aligned(by->rows, 4), "%s: an operand's address is not that of its type", name);
    p.experts = by->count;
    p.offsets = by->offsets;
    p.rows = by->rows;
    if (by->rows) {
        EXHIP_REQUIRE(by->x_rows > 0 && (long long)by->x_rows * d->x_stride <= 0x7fffffff, "%s: %d rows of the input, %d bytes apart: one at least, 2^31 - 1 bytes at most together", name,
                      by->x_rows, d->x_stride);
        p.x_rows = by->x_rows;
    }
    return gated_product ? run_best(ctx, p, kGrouped<true>, true) : run_best(ctx, p, kGrouped<false>, false);
}

}  // namespace

extern "C" int exhip_quantize_rows_f32_to_i8(exhip_ctx* ctx, const float* x, int x_stride, int m, int k, int8_t* y, int y_stride, float* scale) {
    return quantize_rows(ctx, "exhip_quantize_rows_f32_to_i8", x, x_stride, m, k, y, y_stride, scale);
}
extern "C" int exhip_quantize_rows_f16_to_i8(exhip_ctx* ctx, const uint16_t* x, int x_stride, int m, int k, int8_t* y, int y_stride, float* scale) {
    return quantize_rows(ctx, "exhip_quantize_rows_f16_to_i8", x, x_stride, m, k, y, y_stride, scale);
}

extern "C" size_t exhip_i8_packed_bytes(int experts, int n_out, int k_in, int gated_weights) {
    if (!sizes_ok(n_out, k_in) || experts <= 0 || experts > kMostExperts) {
        exhip_set_error("exhip_i8_packed_bytes: %d experts, %d outputs, %d inputs: %s, 1 to %d experts", experts, n_out, k_in, kSizes, kMostExperts);
        return 0;
    }
    return (size_t)experts * tiles_of(n_out, gated_weights != 0) * blocks_of(k_in) * kTileBlock;
}

extern "C" int exhip_i8_pack_weights(exhip_ctx* ctx, int experts, int n_out, int k_in, const int8_t* w, const int8_t* w_up, void* packed) {
    EXHIP_REQUIRE(ctx && w && packed, "exhip_i8_pack_weights: NULL argument");
    const size_t bytes = exhip_i8_packed_bytes(experts, n_out, k_in, w_up != nullptr);
    if (bytes == 0) return EXHIP_ERR_ARG;
    EXHIP_REQUIRE(aligned(packed, 16), "exhip_i8_pack_weights: packed weights begin on 16 bytes");
    const size_t pieces = bytes / 16, groups = (pieces + 255) / 256;
    EXHIP_REQUIRE(groups <= 0x7fffffff / 256, "exhip_i8_pack_weights: %zu bytes are more than one launch takes", bytes);
    const exhip_on_device on(ctx->device);
    EXHIP_CHECK(on.error);
    hipLaunchKernelGGL(pack_i8_kernel, dim3((unsigned)groups), dim3(256), 0, ctx->stream, w, w_up, n_out, k_in, blocks_of(k_in), tiles_of(n_out, w_up != nullptr), pieces,
                       static_cast<v4i*>(packed));
    EXHIP_LAUNCH_CHECK();
    return 0;
}

extern "C" int exhip_innerproduct_i8(exhip_ctx* ctx, const exhip_i8_desc* d, const int8_t* x, const float* x_scale, const void* w_packed, const float* w_scale, const float* bias, float* y_f32,
                                     uint16_t* y_f16) {
    return product(ctx, "exhip_innerproduct_i8", d, nullptr, x, x_scale, w_packed, w_scale, nullptr, bias, nullptr, 0, false, y_f32, y_f16);
}
extern "C" int exhip_innerproduct_gated_i8(exhip_ctx* ctx, const exhip_i8_desc* d, int gate, const int8_t* x, const float* x_scale, const void* w_packed, const float* w_scale_gate,
                                           const float* w_scale_up, const float* bias_gate, const float* bias_up, float* y_f32, uint16_t* y_f16) {
    return product(ctx, "exhip_innerproduct_gated_i8", d, nullptr, x, x_scale, w_packed, w_scale_gate, w_scale_up, bias_gate, bias_up, gate, true, y_f32, y_f16);
}
extern "C" int exhip_innerproduct_grouped_i8(exhip_ctx* ctx, const exhip_i8_desc* d, int experts, const int32_t* offsets, const int32_t* rows, int x_rows, const int8_t* x, const float* x_scale,
                                             const void* w_packed, const float* w_scale, const float* bias, float* y_f32, uint16_t* y_f16) {
    const Experts by = {experts, offsets, rows, x_rows};
    return product(ctx, "exhip_innerproduct_grouped_i8", d, &by, x, x_scale, w_packed, w_scale, nullptr, bias, nullptr, 0, false, y_f32, y_f16);
}
extern "C" int exhip_innerproduct_grouped_gated_i8(exhip_ctx* ctx, const exhip_i8_desc* d, int gate, int experts, const int32_t* offsets, const int32_t* rows, int x_rows, const int8_t* x,
                                                   const float* x_scale, const void* w_packed, const float* w_scale_gate, const float* w_scale_up, const float* bias_gate,
                                                   const float* bias_up, float* y_f32, uint16_t* y_f16) {
    const Experts by = {experts, offsets, rows, x_rows};
    return product(ctx, "exhip_innerproduct_grouped_gated_i8", d, &by, x, x_scale, w_packed, w_scale_gate, w_scale_up, bias_gate, bias_up, gate, true, y_f32, y_f16);
}
