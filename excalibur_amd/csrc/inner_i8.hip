// Inner products in 8-bit integers: the row quantizer, the weights' layout, the product and the gated product, alone and by experts.
//
// A row's codes share a float32 scale, and so do those of an output's weights: neither takes part in the sums, which are those of v_mfma_i32_32x32x32_i8 and
// v_mfma_i32_16x16x64_i8 in 32 bits and exact for as many as 131071 values a row. A result is sum * row's scale * output's scale + bias, rounded in that order; which kernel
// takes a call, and how it cuts the sums, changes no bit of it. Weights are the first operand, rows of the input the second: a lane's results are then
// runs of four neighbouring outputs of one row.
#include "inner.h"

namespace {

constexpr int kBlk = 128;                // values of a row that a step takes
constexpr int kTileBlock = 32 * kBlk;    // bytes of a tile's weights for them
constexpr int kMostInputs = 131071;      // 2^14 each, 2^31 - 1 at most together
constexpr int kMostStride = 1 << 22;     // of a row of codes
constexpr int kMostExperts = 1024;
constexpr float kLargest = 127.f;
constexpr float kLeastScale = 0x1p-100f;  // keeps 1 / scale finite and rows of zeros at zero
constexpr unsigned kNoRow = 0x80000000u;  // beyond every view of rows: loads there give zeros

// ---- the quantizer ----
// x / scale to the nearest whole number, ties to the even one, exactly: the product with 1 / scale is less than one off, and what it leaves, x - r scale, is
// a multiple of the last place of scale / 2 and has no more bits than a float.
__device__ __forceinline__ int code_of(float x, float scale, float inverse, float half) {
    float r = __builtin_rintf(x * inverse);
    const float left = __builtin_fmaf(-r, scale, x), off = fabsf(left);
    if (off > half || (off == half && ((int)r & 1))) r += left > 0.f ? 1.f : -1.f;
    return (int)r;
}
__device__ __forceinline__ int four_codes(int a, int b, int c, int d) { return (a & 255) | (b & 255) << 8 | (c & 255) << 16 | d << 24; }

// A row a group. Rows are read twice, the second time from L2.
template <typename T>
__global__ __launch_bounds__(256) void quantize_rows_i8_kernel(const T* __restrict__ x, int x_stride, int k, int8_t* __restrict__ y, int y_stride, float* __restrict__ scale) {
    const T* const row = x + (size_t)blockIdx.x * x_stride;
    int8_t* const codes = y + (size_t)blockIdx.x * y_stride;
    __shared__ float part[4];
    __shared__ int odd[4];
    float most = 0.f;
    bool special = false;
    for (int at = threadIdx.x; at < k; at += 256) {
        const float a = fabsf(as_float(row[at]));
        special |= !(a < __builtin_inff());
        most = fmaxf(most, a);
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) most = fmaxf(most, __shfl_xor(most, d));
    if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = most;
    odd[threadIdx.x / 64] = 0;
    if (__any(special)) odd[threadIdx.x / 64] = 1;
    __syncthreads();
    const bool none = odd[0] | odd[1] | odd[2] | odd[3];
    const float s = fmaxf(fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3])) / kLargest, kLeastScale), inverse = 1.f / s;
    if (threadIdx.x == 0) scale[blockIdx.x] = none ? __builtin_nanf("") : s;
    for (int at = threadIdx.x; at < k; at += 256) codes[at] = none ? 0 : (int8_t)code_of(as_float(row[at]), s, inverse, 0.5f * s);
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
__device__ __forceinline__ int rows_before(const I8Params& p, int expert) { return min(max(p.offsets[expert], 0), p.m); }

// The group's part; false where there is none for it. By experts every wave counts the tiles of rows of all of them.
template <bool GROUPED, int ROWS>
__device__ __forceinline__ bool part_of(const I8Params& p, Part* part) {
    int group_m;
    if constexpr (!GROUPED) {
        tile_of(p.groups_n, p.groups_m, &part->group_n, &group_m);
        part->expert = 0;
        part->row0 = group_m * ROWS;
        part->rows = min(ROWS, p.m - part->row0);
        return true;
    } else {
        const int lane = threadIdx.x % 64, each = (p.experts + 63) / 64;
        int own = 0;
        // (Offsets that do not rise count rows twice; the bound, beyond every launch, keeps the sums of such ones in range.)
        for (int e = lane * each; e < min((lane + 1) * each, p.experts); ++e)
            own = min(own + (max(rows_before(p, e + 1) - rows_before(p, e), 0) + ROWS - 1) / ROWS, 1 << 24);
        int upto = own;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int before = __shfl_up(upto, d);
            if (lane >= d) upto += before;
        }
        const int total = min(__builtin_amdgcn_readlane(upto, 63), p.groups_m);
        if ((int)blockIdx.x >= p.groups_n * total) return false;
        tile_of(p.groups_n, total, &part->group_n, &group_m);
        const int of = __builtin_ctzll(__ballot(upto > group_m));
        int left = group_m - (__builtin_amdgcn_readlane(upto, of) - __builtin_amdgcn_readlane(own, of));
        for (int e = of * each; e < min((of + 1) * each, p.experts); ++e) {
            const int from = rows_before(p, e), count = max(rows_before(p, e + 1) - from, 0), tiles = (count + ROWS - 1) / ROWS;
            if (left < tiles) {
                part->expert = __builtin_amdgcn_readfirstlane(e);
                part->row0 = __builtin_amdgcn_readfirstlane(from + left * ROWS);
                part->rows = __builtin_amdgcn_readfirstlane(min(ROWS, count - left * ROWS));
                return true;
            }
            left -= tiles;
        }
        return false;
    }
}

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

// ---- few rows, or few products ----
// A group takes TN x 16 outputs (of both projections) and 16 TM rows; its WK waves every WK-th block, with nothing between memory and their registers: the codes of
// D of a wave's blocks are on their way at a time. The sums meet in LDS, and every thread finishes four neighbouring outputs of a row.
template <int TN, int TM, int WK, int D, bool GATED, bool GROUPED>
__global__ __launch_bounds__(64 * WK, 2) void i8_rows_kernel(const I8Params p) {
    exhip_touch_args(p);
    constexpr int kRows = 16 * TM, kSide = GATED ? 2 : 1;
    static_assert(TN % 2 == 0, "whole tiles");
    Part part;
    if (!part_of<GROUPED, kRows>(p, &part)) return;
    const int lane = threadIdx.x % 64, wk = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), q = lane / 16, col = lane % 16;
    const int blocks = p.blocks, row_bytes = blocks * kTileBlock, tile0 = part.group_n * (TN / 2), last = p.tiles - 1;
    const __amdgpu_buffer_rsrc_t weights = uniform_view(p.w + ((size_t)part.expert * p.tiles + tile0) * row_bytes, (unsigned)(min(TN / 2, p.tiles - tile0) * row_bytes));
    const Rows<GROUPED> rows(p, part);
    unsigned off[TM];
#pragma unroll
    for (int t = 0; t < TM; ++t) off[t] = rows.begin(rows.source(16 * t + col)) + q * 16;
    const int at = q * 512 + col * 16;
    struct Codes {
        v4i w[TN][2], x[TM][2];
    } codes[D];
    auto request = [&](Codes& c, int b) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int i = 0; i < TN; ++i)
                c.w[i][h] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(weights, at + i % 2 * 256, min(i / 2, last - tile0) * row_bytes + b * kTileBlock + h * 2048, 0));
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
    static_assert(kRows * kQuads <= kThreads, "a thread has four outputs of one row");
    __shared__ __attribute__((aligned(16))) int joined[WK][kRows][kPitch];
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int t = 0; t < TM; ++t) *reinterpret_cast<v4i*>(&joined[wk][16 * t + col][i * 16 + q * 4]) = acc[i][t];
    __syncthreads();
    const int quad = threadIdx.x % kQuads, row = threadIdx.x / kQuads, j = part.group_n * (kWidth / kSide) + quad * 4;
    if (row >= part.rows || j >= p.n) return;
    const float x_scale = rows.scale(rows.source(row));
    const size_t own = (size_t)part.expert * p.n;
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
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = gated(p.gate, v[e], result_of(sum_up[e], x_scale, w_scale_up[e], bias_up[e]));
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
    hipLaunchKernelGGL(quantize_rows_i8_kernel<T>, dim3(m), dim3(256), 0, ctx->stream, x, x_stride, k, y, y_stride, scale);
    EXHIP_LAUNCH_CHECK();
    return 0;
}

template <typename K>
int launch(exhip_ctx* ctx, K kernel, I8Params p, int tiles, int rows, int threads) {
    p.groups_n = (p.tiles + tiles - 1) / tiles;
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

template <bool GATED, bool GROUPED>
int run_best(exhip_ctx* ctx, const I8Params& p) {
    return launch(ctx, i8_rows_kernel<2, 1, 8, 2, GATED, GROUPED>, p, 1, 16, 512);
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
    if (!by) return gated_product ? run_best<true, false>(ctx, p) : run_best<false, false>(ctx, p);
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
    return gated_product ? run_best<true, true>(ctx, p) : run_best<false, true>(ctx, p);
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
