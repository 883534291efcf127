// Inner products in 8-bit floating point: the row quantizer, the weights' layout, the product and the gated product.
//
// A block of 128 values shares a float32 scale. Its codes become halves, which hold every e4m3 value exactly, and four v_mfma_f32_16x16x32_f16 (or
// eight v_mfma_f32_32x32x16_f16) sum the block's products of 16 outputs (32) and as many rows, still without scales; the sum goes to the running one with one multiply-add per value, by the product of
// the two blocks' scales. Weights are the first operand, rows of the input the second: a lane's four results are then four neighbouring outputs of
// one row, so the row's scale is one register of the lane and the weights' scale one value of the wave.
//
// The matrix core's own 8-bit products (v_mfma_f32_16x16x128_f8f6f4, v_mfma_f32_16x16x32_fp8_fp8) add groups of eight with 13 bits beneath the largest
// of them; what is smaller is cut off. A product of normal rows is 3e-5 off then (measured), where float32 sums of the exact products are 3e-8 off. Only
// the entry points that say so use them: they take half the time of large products.
#include "common.h"
#include "on_device.h"

typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v4i_any __attribute__((ext_vector_type(4), aligned(1)));  // at any address, and at any of their type's
typedef int int_any __attribute__((aligned(1)));
typedef float v4f_any __attribute__((ext_vector_type(4), aligned(4)));
typedef int v2i __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef _Float16 v4h __attribute__((ext_vector_type(4)));

namespace {

constexpr int kBlk = EXHIP_F8_BLOCK;
constexpr int kRsrcWord3 = 0x00020000;
constexpr float kLargest = 448.f;                   // of e4m3
constexpr float kLeastScale = 0x1p-100f;            // keeps 1 / scale finite and blocks of zeros at zero
constexpr int kMostStride = 1 << 22;                // of a row of codes: offsets inside the 256 rows at most of a group stay below kNoRow
constexpr int kNoRow = 0x7f000000;                  // beyond every group's rows: loads there give zeros

// What the last block's codes of a row are ANDed with: `left` values of 16 are the row's own.
__device__ __forceinline__ v4i keep_first(int left) {
    v4i m;
#pragma unroll
    for (int d = 0; d < 4; ++d) {
        const int v = left - 4 * d;
        m[d] = v >= 4 ? -1 : v <= 0 ? 0 : (1 << (8 * v)) - 1;
    }
    return m;
}

// ---- the quantizer ----
template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Eight {  // eight values at any alignment of their type
    T v[8];
};
__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(uint16_t v) { return exhip_h2f(v); }

// The largest of a block, from 16 lanes of eight values each. (fmaxf leaves NaN out.)
__device__ __forceinline__ float block_max(float a) {
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) a = fmaxf(a, __shfl_xor(a, d));
    return a;
}
__device__ __forceinline__ float scale_of(float most) { return fmaxf(most / kLargest, kLeastScale); }
__device__ __forceinline__ int four_codes(float a, float b, float c, float d) {
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return __builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
}

// 16 rows x one block a group of 256.
template <typename T>
__global__ __launch_bounds__(256) void quantize_rows_kernel(const T* __restrict__ x, int x_stride, int m, int k, uint8_t* __restrict__ y, int y_stride,
                                                            float* __restrict__ scale) {
    const int row = blockIdx.x * 16 + threadIdx.x / 16, b = blockIdx.y, at = b * kBlk + (threadIdx.x % 16) * 8;
    float v[8];
    const T* const src = x + (size_t)(row < m ? row : 0) * x_stride + at;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 0.f;
    if (row < m) {
        if (at + 8 <= k) {
            const Eight<T> t = *reinterpret_cast<const Eight<T>*>(src);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = as_float(t.v[e]);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (at + e < k) v[e] = as_float(src[e]);
        }
    }
    float a = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) a = fmaxf(a, fabsf(v[e]));
    const float s = scale_of(block_max(a)), r = 1.f / s;
    if (row >= m) return;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] *= r;
    const v2i q = {four_codes(v[0], v[1], v[2], v[3]), four_codes(v[4], v[5], v[6], v[7])};
    uint8_t* const dst = y + (size_t)row * y_stride + at;
    if (at + 8 <= k) {
        *reinterpret_cast<v2i*>(dst) = q;
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (at + e < k) dst[e] = (uint8_t)(q[e / 4] >> (8 * (e % 4)));
    }
    if (threadIdx.x % 16 == 0) scale[(size_t)b * m + row] = s;
}

// One 128 x 128 block of a weight matrix a group: 16 rows of four values a thread, held between the maximum and the codes. (8192 x 4096 in 26 us;
// with a second reading of single values 53.)
__global__ __launch_bounds__(256) void quantize_blocks_kernel(const float* __restrict__ w, int n, int k, int blocks_k, uint8_t* __restrict__ y,
                                                              float* __restrict__ scale) {
    const int bn = blockIdx.x / blocks_k, bk = blockIdx.x % blocks_k;
    const int col = bk * kBlk + threadIdx.x % 32 * 4, row0 = bn * kBlk + threadIdx.x / 32;
    __shared__ float part[4];
    v4f v[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int row = row0 + 8 * i;
        const float* const src = w + (size_t)row * k + col;
        v[i] = v4f{0.f, 0.f, 0.f, 0.f};
        if (row < n && col + 4 <= k) v[i] = *reinterpret_cast<const v4f_any*>(src);
        else if (row < n)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (col + e < k) v[i][e] = src[e];
    }
    float a = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) a = fmaxf(fmaxf(a, fmaxf(fabsf(v[i][0]), fabsf(v[i][1]))), fmaxf(fabsf(v[i][2]), fabsf(v[i][3])));
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) a = fmaxf(a, __shfl_xor(a, d));
    if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = a;
    __syncthreads();
    const float s = scale_of(fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]))), inv = 1.f / s;
    if (threadIdx.x == 0) scale[blockIdx.x] = s;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int row = row0 + 8 * i, code = four_codes(v[i][0] * inv, v[i][1] * inv, v[i][2] * inv, v[i][3] * inv);
        uint8_t* const dst = y + (size_t)row * k + col;
        if (row < n && col + 4 <= k) *reinterpret_cast<int_any*>(dst) = code;
        else if (row < n)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (col + e < k) dst[e] = (uint8_t)(code >> (8 * e));
    }
}

// ---- the weights' layout ----
// Tiles of 16 outputs x 128 values, a tile row's blocks one after the other: [tile][block][half of 64 values][lane][16 bytes], where lane l holds output l % 16
// and values 64 half + 16 (l / 16) and on. A wave reads a tile as two runs of 1 KB. Gated weights alternate, 16 outputs of the gate, the same 16 of the other
// projection, so that a wave has both sides of its outputs. Outputs and values that do not exist are zeros.
__global__ __launch_bounds__(256) void pack_f8_kernel(const uint8_t* __restrict__ w, const uint8_t* __restrict__ w_up, int n, int k, int blocks_k, size_t pieces,
                                                      v4i* __restrict__ packed) {
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= pieces) return;
    const int lane = i % 64, half = i / 64 % 2;
    const size_t tile_block = i / 128;
    const int block = tile_block % blocks_k, tile = tile_block / blocks_k;
    const uint8_t* const from = w_up && tile % 2 ? w_up : w;
    const int row = (w_up ? tile / 2 : tile) * 16 + lane % 16, col = block * kBlk + half * 64 + lane / 16 * 16;
    const uint8_t* const src = from + (size_t)row * k + col;
    if (row < n && col + 16 <= k) {
        packed[i] = *reinterpret_cast<const v4i_any*>(src);
        return;
    }
    union { uint8_t b[16]; v4i v; } u;
    for (int e = 0; e < 16; ++e) u.b[e] = row < n && col + e < k ? src[e] : 0;
    packed[i] = u.v;
}

// ---- the products ----
struct F8Params {
    const uint8_t* x;
    const float* x_scale;
    const uint8_t* w;
    const float *w_scale, *w_scale_up;  // of a gated product: the gate's, the other projection's
    const float *bias, *bias_up;
    float* y_f32;
    uint16_t* y_f16;
    uint8_t* y_f8;
    float* y_scale;
    int m, n, k, x_stride, y_stride;
    int blocks_k, tiles;  // blocks along k, tiles of 16 outputs (of both projections)
    int gate;
    int first, last;         // the rows of this launch
    int groups_n, groups_m;  // its groups side by side along the outputs, and along the rows
};

__device__ __forceinline__ float gated(int gate, float g, float u) {
    switch (gate) {
    case EXHIP_GATE_SILU: return g / (1.f + expf(-g)) * u;
    case EXHIP_GATE_GELU: return 0.5f * g * (1.f + erff(g * 0.70710678118654752f)) * u;
    case EXHIP_GATE_SIGMOID: return u / (1.f + expf(-g));
    default: return (g > 0.f ? g : g != g ? g : 0.f) * u;
    }
}

// Sixteen codes as halves, which hold every e4m3 value: piece s of four has the values 4 s .. 4 s + 3 of each of the lane's two runs.
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
__device__ __forceinline__ v8h halves_of(int a, int b) {
    const v2h p = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.f, false), q = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.f, true);
    const v2h r = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.f, false), s = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.f, true);
    return v8h{p[0], p[1], q[0], q[1], r[0], r[1], s[0], s[1]};
}
struct Halves {
    v8h v[4];
};
__device__ __forceinline__ Halves halves_of(v4i lo, v4i hi) {
    Halves h;
#pragma unroll
    for (int s = 0; s < 4; ++s) h.v[s] = halves_of(lo[s], hi[s]);
    return h;
}
typedef int v8i __attribute__((ext_vector_type(8)));
__device__ __forceinline__ Halves halves_of(const v8i& c) {
    return halves_of(__builtin_shufflevector(c, c, 0, 1, 2, 3), __builtin_shufflevector(c, c, 4, 5, 6, 7));
}
// One block's products of 16 outputs and 16 rows.
__device__ __forceinline__ v4f block_product(const Halves& w, const Halves& x) {
    v4f c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < 4; ++s) c = __builtin_amdgcn_mfma_f32_16x16x32_f16(w.v[s], x.v[s], c, 0, 0, 0);
    return c;
}

// Four neighbouring outputs of a row at any alignment of their type, and the first of them where the row ends.
typedef _Float16 v4h_any __attribute__((ext_vector_type(4), aligned(2)));
__device__ __forceinline__ void store_cut(float* y, v4f v, int left) {
    y[0] = v[0];
    if (left > 1) y[1] = v[1];
    if (left > 2) y[2] = v[2];
}
__device__ __forceinline__ void store_cut(uint16_t* y, v4f v, int left) {
    y[0] = exhip_f2h(v[0]);
    if (left > 1) y[1] = exhip_f2h(v[1]);
    if (left > 2) y[2] = exhip_f2h(v[2]);
}

// ---- loads ----
__device__ __forceinline__ v8i both(v4i a, v4i b) { return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7); }
// One 16-byte (4-byte) element per lane from a bounds-checked view straight into LDS, lane l's at lds + 16 l (4 l); lds is the wave's, and so is `more`, an
// offset beside the lane's. vmcnt counts them like any other load. (The bounds need not see `more`: lanes with nothing to load have kNoRow.)
__device__ __forceinline__ void load16_to_lds(__amdgpu_buffer_rsrc_t view, int off, int more, unsigned lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(lds), "v"(off), "s"(view), "s"(more) : "m0", "memory");
}
__device__ __forceinline__ void load4_to_lds(__amdgpu_buffer_rsrc_t view, int off, unsigned lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds" ::"s"(lds), "v"(off), "s"(view) : "m0", "memory");
}
__device__ __forceinline__ __amdgpu_buffer_rsrc_t uniform_view(const void* base, unsigned range) {  // base and range are the wave's
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, range, kRsrcWord3);
}

// Of a wave's own, by scalar loads: a vector load's wait would be one for what else is on its way too.
typedef const __attribute__((address_space(4))) float* Constants;

// A wave's TN tile rows of the packed weights: a view from the first on, and where in it the i-th begins (the last that exists, for those beyond).
struct WeightRows {
    __amdgpu_buffer_rsrc_t view;
    int first, last, row_bytes, at;
    __device__ __forceinline__ WeightRows(const F8Params& p, int tile0, int tiles, int lane)
        : first(min(tile0, p.tiles - 1)), last(p.tiles - 1), row_bytes(p.blocks_k * 2048), at(lane * 16) {
        view = uniform_view(p.w + (size_t)first * row_bytes, (unsigned)(min(tiles, p.tiles - first) * row_bytes));
    }
    // half h of block b of tile i
    __device__ __forceinline__ v4i load(int i, int b, int h) const {
        return __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(view, at + h * 1024, min(i, last - first) * row_bytes + b * 2048, 0));
    }
};

// Which tiles a group takes: each of the 8 XCDs a run of neighbouring ones, in bands of eight row tiles, so that the groups that run on an XCD at a time share
// rows and weights in its L2.
__device__ __forceinline__ void tile_of(int groups_n, int groups_m, int* n, int* m) {
    const int total = groups_n * groups_m, xcd = blockIdx.x % 8, per = total / 8, more = total % 8;
    const int i = xcd * per + min(xcd, more) + blockIdx.x / 8;
    const int band = i / (8 * groups_n), within = i % (8 * groups_n), high = min(8, groups_m - band * 8);
    *m = band * 8 + within % high;
    *n = within / high;
}

// ---- results of the kernels for many rows: through LDS, so that whole lines are stored ----
// (A lane's four neighbouring outputs of one row, stored as they are, are 32 bytes of each of 16 rows at a time: 1.2 TB/s.)
// Row-major results of a group: rows of WIDTH outputs, 16-byte pieces at place piece ^ (row % 8), % 4 where there are four.
template <typename O, int WIDTH>
__device__ __forceinline__ int byte_in_row(int row, int byte) {
    constexpr int kPieces = WIDTH * (int)sizeof(O) / 16, kTurn = kPieces < 8 ? kPieces - 1 : 7;
    return ((byte / 16) ^ (row & kTurn)) * 16 + byte % 16;
}
template <typename O, int WIDTH>
__device__ __forceinline__ char* place_in_rows(char* lds, int row, int j) {
    return lds + row * (WIDTH * (int)sizeof(O)) + byte_in_row<O, WIDTH>(row, j * (int)sizeof(O));
}
// (Nothing but whole pieces in the loop: code that a group runs once comes from memory line by line, 1 us each where a branch leaves the straight line. With
// the cut pieces inside it the same loop took 2 to 14 us a group, by the XCD. The stores go past L2: 8192 x 8192 x 4096 263 -> 237 us.)
template <typename O, int WIDTH, int ROWS, int THREADS>
__device__ __forceinline__ void store_rows(const char* lds, O* y, size_t stride, int row0, int rows, int j0, int n) {
    constexpr int kPer = 16 / sizeof(O), kPieces = WIDTH / kPer, kPitch = WIDTH * (int)sizeof(O), kTogether = THREADS / kPieces;
    static_assert(THREADS % kPieces == 0 && ROWS % kTogether == 0, "every thread stores one piece of every kTogether-th row");
    const int piece = threadIdx.x % kPieces, first = threadIdx.x / kPieces, j = j0 + piece * kPer;
    O* const dst = y + (size_t)(row0 + first) * stride + j;
    const size_t step = (size_t)kTogether * stride;
    const bool whole = j + kPer <= n;
#pragma unroll 4
    for (int i = 0; i < ROWS / kTogether; ++i) {
        const int row = i * kTogether + first;
        const v4i v = *reinterpret_cast<const v4i*>(lds + row * kPitch + byte_in_row<O, WIDTH>(row, piece * 16));
        if (whole && row < rows) __builtin_nontemporal_store(v, reinterpret_cast<v4i_any*>(dst + i * step));
    }
    if (j0 + WIDTH > n && n % kPer != 0) {
        const int at = n / kPer * kPer, left = n - at;
        for (int i = threadIdx.x; i < rows * left; i += THREADS) {
            const int row = i / left, e = i % left, byte = (at - j0) * (int)sizeof(O);
            y[(size_t)(row0 + row) * stride + at + e] = reinterpret_cast<const O*>(lds + row * kPitch + byte_in_row<O, WIDTH>(row, byte))[e];
        }
    }
}
__device__ __forceinline__ v4f four_of(const float* v, int j, int n) {
    v4f r = {0.f, 0.f, 0.f, 0.f};
    if (v)
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = v[min(j + e, n - 1)];
    return r;
}

// Where a lane's sums lie: value i of four neighbouring outputs each, of TN, and rows t. After 16 x 16 products a lane has the outputs of a quarter of each tile and
// one row, after 32 x 32 products those of a half of each eight.
template <int SIDE>
struct Lanes {
    static constexpr int kOfAFour = SIDE == 16 ? 16 : 8;  // the wave's outputs for each four of a lane
    static __device__ __forceinline__ int output(int i, int lane) { return SIDE == 16 ? i * 16 + lane / 16 * 4 : i * 8 + lane / 32 * 4; }
    static __device__ __forceinline__ int row(int t, int lane) { return t * SIDE + lane % SIDE; }
    // of a gated product: the four of the gate, those of the other projection, and where the result of both stands among the wave's 32
    static __device__ __forceinline__ constexpr int gate(int i) { return SIDE == 16 ? 2 * i : i / 2 * 4 + i % 2; }
    static __device__ __forceinline__ constexpr int up(int i) { return SIDE == 16 ? 2 * i + 1 : i / 2 * 4 + i % 2 + 2; }
    static __device__ __forceinline__ int result(int i, int lane) { return SIDE == 16 ? i * 16 + lane / 16 * 4 : i * 8 + lane / 32 * 4; }
};

// The sums of a group of WN x WM waves, FOURS x 4 outputs a lane and SIDE * TM rows each. `lds` is free for at least the group's results as floats (halves where there are no
// others).
template <int SIDE, int WN, int WM, bool FLOATS, int FOURS, int TM>
__device__ __forceinline__ void write_group(const F8Params& p, v4f (&acc)[FOURS][TM], int group_n, int wn, int wm, int row0, int rows, int lane, char* lds) {
    typedef Lanes<SIDE> At;
    constexpr int kOwn = FOURS * At::kOfAFour, kWidth = kOwn * WN, kRows = SIDE * TM * WM, kThreads = 64 * WN * WM;
    const int j0 = group_n * kWidth;
#pragma unroll
    for (int i = 0; i < FOURS; ++i) {
        const v4f bias = four_of(p.bias, j0 + wn * kOwn + At::output(i, lane), p.n);
#pragma unroll
        for (int t = 0; t < TM; ++t) acc[i][t] += bias;
    }
    if (FLOATS && p.y_f32) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < FOURS; ++i)
#pragma unroll
            for (int t = 0; t < TM; ++t) *reinterpret_cast<v4f*>(place_in_rows<float, kWidth>(lds, wm * TM * SIDE + At::row(t, lane), wn * kOwn + At::output(i, lane))) = acc[i][t];
        __syncthreads();
        store_rows<float, kWidth, kRows, kThreads>(lds, p.y_f32, p.y_stride, row0, rows, j0, p.n);
    }
    if (p.y_f16) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < FOURS; ++i)
#pragma unroll
            for (int t = 0; t < TM; ++t)
                *reinterpret_cast<v4h*>(place_in_rows<uint16_t, kWidth>(lds, wm * TM * SIDE + At::row(t, lane), wn * kOwn + At::output(i, lane))) = __builtin_convertvector(acc[i][t], v4h);
        __syncthreads();
        store_rows<uint16_t, kWidth, kRows, kThreads>(lds, p.y_f16, p.y_stride, row0, rows, j0, p.n);
    }
}

// The same of a gated product, whose tiles alternate: half as many outputs. Quantized results (CODES) need a whole block of them in a group, and exact sums.
template <int SIDE, int WN, int WM, bool CODES, int FOURS, int TM>
__device__ __forceinline__ void write_gated_group(const F8Params& p, v4f (&acc)[FOURS][TM], int group_n, int wn, int wm, int row0, int rows, int lane, char* lds) {
    typedef Lanes<SIDE> At;
    constexpr int kResults = FOURS / 2, kOwn = kResults * At::kOfAFour, kWidth = kOwn * WN, kRows = SIDE * TM * WM, kThreads = 64 * WN * WM;
    const int j0 = group_n * kWidth, row_at = wm * TM * SIDE, out_at = wn * kOwn;
#pragma unroll
    for (int i = 0; i < kResults; ++i) {
        const int j = j0 + out_at + At::result(i, lane);
        const v4f bias = four_of(p.bias, j, p.n), bias_up = four_of(p.bias_up, j, p.n);
#pragma unroll
        for (int t = 0; t < TM; ++t) {
            const v4f g = acc[At::gate(i)][t] + bias, u = acc[At::up(i)][t] + bias_up;
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[At::gate(i)][t][e] = j + e < p.n ? gated(p.gate, g[e], u[e]) : 0.f;
        }
    }
    __syncthreads();
    if (p.y_f16) {
#pragma unroll
        for (int i = 0; i < kResults; ++i)
#pragma unroll
            for (int t = 0; t < TM; ++t)
                *reinterpret_cast<v4h*>(place_in_rows<uint16_t, kWidth>(lds, row_at + At::row(t, lane), out_at + At::result(i, lane))) = __builtin_convertvector(acc[At::gate(i)][t], v4h);
        __syncthreads();
        store_rows<uint16_t, kWidth, kRows, kThreads>(lds, p.y_f16, p.y_stride, row0, rows, j0, p.n);
    }
    if constexpr (CODES) {
        static_assert(kWidth == kBlk, "a row's maximum is that of a block");
        if (!p.y_f8) return;
        float* const most = reinterpret_cast<float*>(lds);  // [wave along the outputs][row]
#pragma unroll
        for (int t = 0; t < TM; ++t) {
            float a = 0.f;
#pragma unroll
            for (int i = 0; i < kResults; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) a = fmaxf(a, fabsf(acc[At::gate(i)][t][e]));
#pragma unroll
            for (int d = SIDE; d < 64; d <<= 1) a = fmaxf(a, __shfl_xor(a, d));
            if (lane < SIDE) most[wn * kRows + row_at + At::row(t, lane)] = a;
        }
        __syncthreads();
        float s[TM];
#pragma unroll
        for (int t = 0; t < TM; ++t) {
            const int row = row_at + At::row(t, lane);
            float top = most[row];
#pragma unroll
            for (int o = 1; o < WN; ++o) top = fmaxf(top, most[o * kRows + row]);
            s[t] = scale_of(top);
            if (wn == 0 && lane < SIDE && row < rows) p.y_scale[(size_t)group_n * p.m + row0 + row] = s[t];
        }
        __syncthreads();
#pragma unroll
        for (int t = 0; t < TM; ++t) {
            const float r = 1.f / s[t];
#pragma unroll
            for (int i = 0; i < kResults; ++i) {
                const v4f v = acc[At::gate(i)][t] * r;
                *reinterpret_cast<int*>(place_in_rows<uint8_t, kWidth>(lds, row_at + At::row(t, lane), out_at + At::result(i, lane))) = four_codes(v[0], v[1], v[2], v[3]);
            }
        }
        __syncthreads();
        store_rows<uint8_t, kWidth, kRows, kThreads>(lds, p.y_f8, p.y_stride, row0, rows, j0, p.n);
    }
}

// ---- many rows, cut sums: the matrix core's own 8-bit products ----
// A group of 4 x 2 waves takes 256 outputs and 256 rows, a wave 64 x 128: 128 of its 256 registers are sums. Rows' codes and their scales come straight into
// LDS, two blocks ahead in four buffers; weights from L2 straight into registers, a block ahead. Products are issued one by one, and the multiply-adds of the
// product three places before run while the matrix core works on a new one. A block's one barrier stands in its middle: it says that the next block's rows are
// there, so that a block's end waits for nothing.
template <bool GATED>
__global__ __launch_bounds__(512, 2) void f8_wide_kernel(const F8Params p) {
    exhip_touch_args(p);
    constexpr int WN = 4, TN = 4, TM = 8, kRows = 256, kBuffers = 4, kCodes = kRows * kBlk, kBuffer = kCodes + kRows * 4, kLag = 3;
    __shared__ __attribute__((aligned(16))) char staged[kBuffers * kBuffer];
    const unsigned lds0 = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char*)staged;
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), wn = wave % WN, wm = wave / WN;
    const int q = lane / 16, col = lane % 16;
    int group_n, group_m;
    tile_of(p.groups_n, p.groups_m, &group_n, &group_m);
    const int tile0 = (group_n * WN + wn) * TN, row0 = p.first + group_m * kRows;
    const int rows = min(kRows, p.last - row0), tail = p.k % kBlk, blocks = p.blocks_k;
    const __amdgpu_buffer_rsrc_t xr = uniform_view(p.x + (size_t)row0 * p.x_stride, (rows - 1) * p.x_stride + (p.k + 15) / 16 * 16);
    // A wave stages 32 rows, eight with a load: lane l holds piece (l % 8) ^ (l / 8) of row l / 8, so that a piece of eight neighbouring rows lies in all banks.
    // Pieces behind a row's end are zeros.
    const int piece = (lane % 8) ^ (lane / 8);
    const bool behind = tail && piece * 16 >= tail;
    int off[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int row = wave * 32 + j * 8 + lane / 8;
        off[j] = row < rows ? row * p.x_stride + piece * 16 : kNoRow;
    }
    const int scale_off = min(wave % 4 * 64 + lane, rows - 1) * 4;
    // (Behind the last block that one is staged and requested again, where nothing reads it: every block waits for the same number of loads.)
    auto stage = [&](int buffer, int j) {  // in five loads
        const int b = min(buffer, blocks - 1);
        const unsigned to = lds0 + buffer % kBuffers * kBuffer;
        if (j < 4) load16_to_lds(xr, behind && b == blocks - 1 ? kNoRow : off[j], b * kBlk, to + (wave * 32 + j * 8) * kBlk);
        else load4_to_lds(uniform_view(p.x_scale + (size_t)b * p.m + row0, rows * 4), scale_off, to + kCodes + wave % 4 * 256);
    };
    const WeightRows weights(p, tile0, TN, lane);
    const int block_n = min(GATED ? tile0 / 2 : tile0, (p.n - 1) / 16) / (kBlk / 16);
    const Constants ws = (Constants)(uintptr_t)(p.w_scale + (size_t)block_n * blocks);
    const Constants ws_up = (Constants)(uintptr_t)(GATED ? p.w_scale_up + (size_t)block_n * blocks : nullptr);
    struct Weights {
        v8i v[TN];
    };
    auto request = [&](Weights& w, int b, int j) {  // in eight
        const v4i got = weights.load(j / 2, min(b, blocks - 1), j % 2);
#pragma unroll
        for (int e = 0; e < 4; ++e) w.v[j / 2][j % 2 * 4 + e] = got[e];
    };
    v4f acc[TN][TM];
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int t = 0; t < TM; ++t) acc[i][t] = v4f{0.f, 0.f, 0.f, 0.f};
    const int at = (wm * TM * 16 + col) * kBlk + (q ^ (col & 7)) * 16, at_hi = (wm * TM * 16 + col) * kBlk + (q ^ (col & 7) ^ 4) * 16;
    const int at_scale = kCodes + (wm * TM * 16 + col) * 4;
    struct Rows {
        v8i v;
        float s;
    };
    auto rows_from = [&](int b, int t) {
        const char* const from = staged + b % kBuffers * kBuffer;
        return Rows{both(*reinterpret_cast<const v4i*>(from + at + t * 16 * kBlk), *reinterpret_cast<const v4i*>(from + at_hi + t * 16 * kBlk)),
                    *reinterpret_cast<const float*>(from + at_scale + t * 64)};
    };
    Rows x[2];
    float s_w = ws[0], s_up = GATED ? ws_up[0] : 0.f, s_next = 0.f, s_up_next = 0.f;
    auto block = [&](Weights& w, Weights& next, int b) {
        if (p.k % 16 && b == blocks - 1) {  // the piece that a row's end cuts
            if (threadIdx.x < kRows) {
                v4i* const cut = reinterpret_cast<v4i*>(staged + b % kBuffers * kBuffer + threadIdx.x * kBlk + ((tail / 16) ^ (threadIdx.x & 7)) * 16);
                *cut &= keep_first(tail % 16);
            }
            __syncthreads();
            x[0] = rows_from(b, 0);
        }
        // The weights, requested a block ago, are waited for here: behind the next loads the compiler, which does not see those into LDS, would wait for them too.
#pragma unroll
        for (int i = 0; i < TN; ++i) asm volatile("" : "+v"(w.v[i]));
        v4f part[kLag + 1];
        float s[2], su[2];
#pragma unroll
        for (int u = 0; u < TN * TM + kLag; ++u) {
            const int t = u / TN, i = u % TN;
            // A load beside every second product: thirteen in a row would hold the wave up, 16 cycles of the CU's address unit each, eight waves at a time.
            if (u % 2 == 0 && u / 2 < 5) stage(b + 2, u / 2);
            else if (u % 2 == 0 && u / 2 < 13) request(next, b + 1, u / 2 - 5);
            if (u < TN * TM) {
                if (i == 0) {
                    if (t == TM / 2) {
                        // The next block's rows are older than all nine loads of this block so far; the eight youngest may be on their way.
                        asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
                        __builtin_amdgcn_s_barrier();
                        asm volatile("" ::: "memory");
                        const int after = min(b + 1, blocks - 1);
                        s_next = ws[after];
                        if constexpr (GATED) s_up_next = ws_up[after];
                    }
                    s[t % 2] = s_w * x[t % 2].s;
                    su[t % 2] = s_up * x[t % 2].s;
                    x[(t + 1) % 2] = t + 1 < TM ? rows_from(b, t + 1) : rows_from(b + 1, 0);
                }
                part[u % (kLag + 1)] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w.v[i], x[t % 2].v, v4f{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
            }
            if (u >= kLag) {
                const int v = u - kLag, vt = v / TN, vi = v % TN;
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[vi][vt][e] = __builtin_fmaf(part[v % (kLag + 1)][e], GATED && vi % 2 ? su[vt % 2] : s[vt % 2], acc[vi][vt][e]);
                asm volatile("" : "+v"(acc[vi][vt]));  // here, not where the compiler would like them: together at the end, out of registers
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        s_w = s_next;
        s_up = s_up_next;
    };
    Weights w0, w1;
#pragma unroll
    for (int j = 0; j < 10; ++j) stage(j / 5, j % 5);
#pragma unroll
    for (int j = 0; j < 8; ++j) request(w0, 0, j);
    asm volatile("s_waitcnt vmcnt(13)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    x[0] = rows_from(0, 0);
    for (int b = 0; b < blocks; b += 2) {
        block(w0, w1, b);
        if (b + 1 < blocks) block(w1, w0, b + 1);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // what was staged behind the end, in front of the results' barrier
    if constexpr (!GATED) write_group<16, WN, 2, false>(p, acc, group_n, wn, wm, row0, rows, lane, staged);
    else write_gated_group<16, WN, 2, false>(p, acc, group_n, wn, wm, row0, rows, lane, staged);
}

// ---- few rows, or few products ----
// A group of WN x WK waves takes WN * TN tiles of outputs and 16 TM rows; wave (wn, wk) its own TN tiles and every WK-th block, with nothing between memory and
// its registers: the codes of D of its blocks are on their way at a time, and no wave waits for another before the sums are joined. Those go through LDS;
// a wave joins a share of the tiles, always in the order of wk, and writes them.
// What bounds it is the memory: one row of the gated 11264 x 4096 takes 16.7 us, 5.5 TB/s of weights. A quantized result has a whole block's outputs in one
// group, 88 groups there, and a CU draws no more than 17 bytes a cycle: 26 us, with 16 waves a group (28 with eight).
template <int TN, int TM, int WN, int WK, int D, bool GATED>
__global__ __launch_bounds__(64 * WN * WK, 2) void f8_rows_kernel(const F8Params p) {
    exhip_touch_args(p);
    constexpr int kRows = 16 * TM, kSide = GATED ? 2 : 1;
    static_assert(TN % kSide == 0, "both sides of an output are one wave's");
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), wn = wave % WN, wk = wave / WN;
    const int q = lane / 16, col = lane % 16;
    const int group_n = blockIdx.x % p.groups_n, tile0 = (group_n * WN + wn) * TN, row0 = p.first + blockIdx.x / p.groups_n * kRows;
    const int rows = min(kRows, p.last - row0), tail = p.k % kBlk, blocks = p.blocks_k;
    const __amdgpu_buffer_rsrc_t xr = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(p.x) + (size_t)row0 * p.x_stride, 0,
                                                                      (rows - 1) * p.x_stride + (p.k + 15) / 16 * 16, kRsrcWord3);
    int off[TM];
    unsigned scale_at[TM];
#pragma unroll
    for (int t = 0; t < TM; ++t) {
        const int row = 16 * t + col;
        off[t] = row < rows ? row * p.x_stride + q * 16 : kNoRow;
        scale_at[t] = min(row, rows - 1);
    }
    const WeightRows weights(p, tile0, TN, lane);
    const int block_n = min(tile0 / kSide, (p.n - 1) / 16) / (kBlk / 16);
    const Constants ws = (Constants)(uintptr_t)(p.w_scale + (size_t)block_n * blocks);
    const Constants ws_up = (Constants)(uintptr_t)(GATED ? p.w_scale_up + (size_t)block_n * blocks : nullptr);
    struct Codes {
        v4i w[TN][2], x[TM][2];
        float s[TM];
    } codes[D];
    auto request_x = [&](Codes& c, int b) {
        const float* const scales = p.x_scale + (size_t)b * p.m + row0;
#pragma unroll
        for (int t = 0; t < TM; ++t) {
            c.x[t][0] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(xr, off[t] + b * kBlk, 0, 0));
            c.x[t][1] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(xr, off[t] + b * kBlk + 64, 0, 0));
            c.s[t] = scales[scale_at[t]];
        }
    };
    auto request_w = [&](Codes& c, int b, int i) {
        c.w[i][0] = weights.load(i, b, 0);
        c.w[i][1] = weights.load(i, b, 1);
    };
    v4f acc[TN][TM];
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int t = 0; t < TM; ++t) acc[i][t] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int d = 0; d < D; ++d)
        if (wk + d * WK < blocks) {
#pragma unroll
            for (int i = 0; i < TN; ++i) request_w(codes[d], wk + d * WK, i);
            request_x(codes[d], wk + d * WK);
        }
    for (int first = wk; first < blocks; first += WK * D) {
#pragma unroll
        for (int d = 0; d < D; ++d) {
            const int b = first + d * WK, next = b + WK * D;
            if (b >= blocks) break;
            Codes& c = codes[d];
            const float s_w = ws[b], s_up = GATED ? ws_up[b] : 0.f;
            if (tail && b == blocks - 1)
#pragma unroll
                for (int t = 0; t < TM; ++t) {
                    c.x[t][0] &= keep_first(tail - q * 16);
                    c.x[t][1] &= keep_first(tail - 64 - q * 16);
                }
            Halves x[TM];
            float s[TM];
#pragma unroll
            for (int t = 0; t < TM; ++t) {
                x[t] = halves_of(c.x[t][0], c.x[t][1]);
                s[t] = c.s[t];
            }
            if (next < blocks) request_x(c, next);
            if constexpr (TN * TM > 8) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < TN; ++i) {
                const Halves w = halves_of(c.w[i][0], c.w[i][1]);
                if (next < blocks) request_w(c, next, i);
#pragma unroll
                for (int t = 0; t < TM; ++t) {
                    const v4f part = block_product(w, x[t]);
                    const float f = (GATED && i % 2 ? s_up : s_w) * s[t];
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[i][t][e] = __builtin_fmaf(part[e], f, acc[i][t][e]);
                }
                if constexpr (TN * TM > 8) __builtin_amdgcn_sched_barrier(0);  // a tile's conversions at a time: all of them together do not fit the registers
            }
        }
    }
    // The waves' sums meet in LDS, row by row (four floats more a row, for the banks), and every thread joins four neighbouring outputs in the order of wk.
    constexpr int kWidth = WN * TN * 16, kPitch = kWidth + 4, kThreads = 64 * WN * WK, kQuads = kWidth / 4 / kSide;
    __shared__ __attribute__((aligned(16))) float joined[WK][kRows][kPitch];
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int t = 0; t < TM; ++t) *reinterpret_cast<v4f*>(&joined[wk][16 * t + col][(wn * TN + i) * 16 + q * 4]) = acc[i][t];
    __syncthreads();
    const int j0 = group_n * (kWidth / kSide);
    static_assert(kThreads % kQuads == 0, "a thread has the same outputs of all its rows");
    const int quad = threadIdx.x % kQuads, j = j0 + quad * 4;
    const v4f bias = four_of(p.bias, j, p.n), bias_up = GATED ? four_of(p.bias_up, j, p.n) : bias;
    for (int row = threadIdx.x / kQuads; row < kRows; row += kThreads / kQuads) {
        v4f v = {0.f, 0.f, 0.f, 0.f}, up = v;
        const int at = GATED ? quad / 4 * 32 + quad % 4 * 4 : quad * 4;
#pragma unroll
        for (int k = 0; k < WK; ++k) {
            v += *reinterpret_cast<const v4f*>(&joined[k][row][at]);
            if constexpr (GATED) up += *reinterpret_cast<const v4f*>(&joined[k][row][at + 16]);
        }
        v += bias;
        if constexpr (GATED) {
            up += bias_up;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = j + e < p.n ? gated(p.gate, v[e], up[e]) : 0.f;
        }
        const size_t to = (size_t)(row0 + row) * p.y_stride + j;
        const bool here = row < rows && j < p.n, whole = here && j + 4 <= p.n;
        if constexpr (GATED && kWidth == 256) {  // 32 lanes have a row's whole block of a quantized result
            if (p.y_f8) {
                float most = fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3])));
#pragma unroll
                for (int d = 1; d < 32; d <<= 1) most = fmaxf(most, __shfl_xor(most, d));
                const float scale = scale_of(most), r = 1.f / scale;
                const int code = four_codes(v[0] * r, v[1] * r, v[2] * r, v[3] * r);
                if (row < rows && quad == 0) p.y_scale[(size_t)group_n * p.m + row0 + row] = scale;
                if (whole) *reinterpret_cast<int*>(p.y_f8 + to) = code;
                else if (here)
                    for (int e = 0; j + e < p.n; ++e) p.y_f8[to + e] = (uint8_t)(code >> (8 * e));
            }
        }
        if (!GATED && p.y_f32) {
            if (whole) *reinterpret_cast<v4f_any*>(p.y_f32 + to) = v;
            else if (here) store_cut(p.y_f32 + to, v, p.n - j);
        }
        if (p.y_f16) {
            if (whole) *reinterpret_cast<v4h_any*>(p.y_f16 + to) = __builtin_convertvector(v, v4h);
            else if (here) store_cut(p.y_f16 + to, v, p.n - j);
        }
    }
}

// ---- many rows, exact products ----
// A group of four waves takes 256 outputs and 64 rows, a wave 64 x 64, in products of 32 x 32: of the cycles in which a SIMD can issue they leave
// more to the conversions and multiply-adds than those of 16 x 16 (48 of these beside 32 x 32 x 128 values take 277 cycles, 342 with the smaller ones). A
// block's rows become halves once for the group, on their way into LDS (four buffers); a wave's weights come from L2 as codes, a block ahead, and become halves
// in its registers. A block is four chains of eight products, one chain for 32 outputs and 32 rows, and what else there is to do has its products: the
// multiply-adds of the chain before, the conversions, the loads one by one, the next chain's rows. Each load's place is the
// latest that still covers L2's answer, since all of it together takes every register there is; the barrier says that the next block's rows are there.
// Measured: 8192 x 8192 x 4096 in 465 us, 1.18 PFLOP/s, where the library's product of halves reaches 1.13; the smaller products took 467, the clock gives way
// under either. 1024 x 4096 x 4096 in 39 us, 200 rows of the gated 4096 x 4096 in 38 (42 with the smaller products).
template <bool GATED>
__global__ __launch_bounds__(256, 2) void f8_tile_kernel(const F8Params p) {
    exhip_touch_args(p);
    constexpr int WN = 4, TN = 4, TM = 2, kRows = 32 * TM, kSteps = 16 * TM, kBuffers = 4, kPitch = 272, kBuffer = kRows * (kPitch + 4);
    // [buffer][row][128 halves], a row's pitch 16 bytes more, so that a piece of eight neighbouring rows lies in all banks; the rows' scales behind them
    constexpr int kStaged = kBuffers * kBuffer, kResults = kRows * (GATED ? 32 * WN * 2 : 64 * WN * 4);
    __shared__ __attribute__((aligned(16))) char memory[kStaged > kResults ? kStaged : kResults];
    const int lane = threadIdx.x % 64, wn = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int side = lane / 32, col = lane % 32;
    int group_n, group_m;
    tile_of(p.groups_n, p.groups_m, &group_n, &group_m);
    const int tile0 = (group_n * WN + wn) * TN, row0 = p.first + group_m * kRows;
    const int rows = min(kRows, p.last - row0), tail = p.k % kBlk, blocks = p.blocks_k;
    const __amdgpu_buffer_rsrc_t xr = uniform_view(p.x + (size_t)row0 * p.x_stride, (rows - 1) * p.x_stride + (p.k + 15) / 16 * 16);
    // what this thread stages
    const int own_row = threadIdx.x / 4, own_q = threadIdx.x % 4;
    const int off = own_row < rows ? own_row * p.x_stride + own_q * 16 : kNoRow;
    const int scale_at = own_row * 4;
    v4i codes[2];
    float code_scale = 0.f;
    auto request = [&](int b, int j) {  // in three loads; behind the last block that one again, which nothing reads
        b = min(b, blocks - 1);
        if (j < 2) codes[j] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(xr, off + b * kBlk + j * 64, 0, 0));  // (all in what the bounds see: the last row may end here)
        else code_scale = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(uniform_view(p.x_scale + (size_t)b * p.m + row0, rows * 4), scale_at, 0, 0));
    };
    auto stage = [&](int b, int j) {  // in four pieces of eight values
        char* const to = memory + b % kBuffers * kBuffer;
        *reinterpret_cast<v8h*>(to + own_row * kPitch + j / 2 * 128 + own_q * 32 + j % 2 * 16) = halves_of(codes[j / 2][j % 2 * 2], codes[j / 2][j % 2 * 2 + 1]);
        if (j == 0) *reinterpret_cast<float*>(to + kRows * kPitch + own_row * 4) = code_scale;
    };
    auto cut = [&] {  // the last block's codes where the row ends
        int left = tail - own_q * 16;
        asm volatile("" : "+v"(left));  // or the masks are made before the loop and take eight registers of it
        codes[0] &= keep_first(left);
        codes[1] &= keep_first(left - 64);
    };
    // A lane's weights are those of output lane % 32 of two tiles: of a tile's [half][quarter][output] the quarters 2 side and 2 side + 1. Product s of a chain takes
    // values 8 (s % 2) and on of quarter s / 2 % 2 of half s / 4, and the rows' values in the same order.
    const WeightRows weights(p, tile0, TN, lane);
    int weights_at[2];
#pragma unroll
    for (int f = 0; f < 2; ++f) weights_at[f] = min(2 * f + col / 16, weights.last - weights.first) * weights.row_bytes + side * 512 + col % 16 * 16;
    const int block_n = min(GATED ? tile0 / 2 : tile0, (p.n - 1) / 16) / (kBlk / 16);
    const Constants ws = (Constants)(uintptr_t)(p.w_scale + (size_t)block_n * blocks);
    const Constants ws_up = (Constants)(uintptr_t)(GATED ? p.w_scale_up + (size_t)block_n * blocks : nullptr);
    v4i raw[2][4];
    auto request_w = [&](int b, int f, int j) {  // in four loads of each of the two
        raw[f][j] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(weights.view, weights_at[f], min(b, blocks - 1) * 2048 + j / 2 * 1024 + j % 2 * 256, 0));
    };
    v8h w[2][8], x[8];
    auto convert_w = [&](int f, int s) {
        w[f][s] = halves_of(raw[f][s / 2][s % 2 * 2], raw[f][s / 2][s % 2 * 2 + 1]);
        asm volatile("" : "+v"(w[f][s]));  // here, not together ahead of the chain that takes them
    };
    auto piece_of = [&](int b, int t, int s) {
        return *reinterpret_cast<const v8h*>(memory + b % kBuffers * kBuffer + (t * 32 + col) * kPitch + side * 64 + s / 4 * 128 + s % 4 * 16);
    };
    auto scale_of_row = [&](int b, int t) { return *reinterpret_cast<const float*>(memory + b % kBuffers * kBuffer + kRows * kPitch + (t * 32 + col) * 4); };
    v4f acc[8][TM];
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int t = 0; t < TM; ++t) acc[i][t] = v4f{0.f, 0.f, 0.f, 0.f};
    v16f part[2], none;
#pragma unroll
    for (int e = 0; e < 16; ++e) none[e] = 0.f;
    part[1] = none;
    float sc[TM], sc_up[TM], last = 0.f, last_up = 0.f;  // of the block's rows, and of the chain that the block before ended with
    auto add = [&](int f, int t, int g, float s, float s_up) {  // four of a chain's outputs to their sums
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[f * 4 + g][t][e] = __builtin_fmaf(part[f][g * 4 + e], GATED && g >= 2 ? s_up : s, acc[f * 4 + g][t][e]);
        asm volatile("" : "+v"(acc[f * 4 + g][t]));  // here, not where the compiler would like them: together at the end, out of registers
    };
#pragma unroll
    for (int j = 0; j < 3; ++j) request(0, j);
#pragma unroll
    for (int j = 0; j < 8; ++j) request_w(0, j / 4, j % 4);
    if (tail && blocks == 1) cut();
#pragma unroll
    for (int j = 0; j < 4; ++j) stage(0, j);
#pragma unroll
    for (int s = 0; s < 8; ++s) convert_w(0, s);
    __syncthreads();
#pragma unroll
    for (int s = 0; s < 8; ++s) x[s] = piece_of(0, 0, s);
    float row_scale = scale_of_row(0, 0), s_w = ws[0], s_up = GATED ? ws_up[0] : 0.f, s_next = 0.f, s_up_next = 0.f;
    for (int b = 0; b < blocks; ++b) {
#pragma unroll
        for (int u = 0; u < kSteps; ++u) {
            const int t = u / 16, f = u / 8 % 2, s = u % 8;
            if (u == 12) {
                const int after = min(b + 1, blocks - 1);
                s_next = ws[after];
                if constexpr (GATED) s_up_next = ws_up[after];
            }
            if (u == 20) __syncthreads();
            if (u == 12 && tail && b == blocks - 2) cut();
            if (u % 16 == 0) {
                sc[t] = s_w * row_scale;
                sc_up[t] = s_up * row_scale;
            }
            if (u < 8) convert_w(1, s);
            if (u >= 8 && u < 12) request_w(b + 1, 0, u - 8);
            if (u >= 24 && u < 28) request_w(b + 1, 1, u - 24);
            if (u >= 12 && u < 16) stage(b + 1, u - 12);
            if (u < 3) request(b + 1, u);
            part[f] = __builtin_amdgcn_mfma_f32_32x32x16_f16(w[f][s], x[s], s == 0 ? none : part[f], 0, 0, 0);
            if (f == 1) x[s] = t + 1 < TM ? piece_of(b, t + 1, s) : piece_of(b + 1, 0, s);
            if (f == 1 && s == 7) row_scale = t + 1 < TM ? scale_of_row(b, t + 1) : scale_of_row(b + 1, 0);
            if (u >= 24) convert_w(0, s);
            if (s >= 2 && s < 6) {
                if (u < 8) add(1, TM - 1, s - 2, last, last_up);
                else add(1 - f, f == 1 ? t : t - 1, s - 2, sc[f == 1 ? t : t - 1 < 0 ? 0 : t - 1], sc_up[f == 1 ? t : t - 1 < 0 ? 0 : t - 1]);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        last = sc[TM - 1];
        last_up = sc_up[TM - 1];
        s_w = s_next;
        s_up = s_up_next;
    }
#pragma unroll
    for (int g = 0; g < 4; ++g) add(1, TM - 1, g, last, last_up);
    if constexpr (!GATED) write_group<32, WN, 1, true>(p, acc, group_n, wn, 0, row0, rows, lane, memory);
    else write_gated_group<32, WN, 1, true>(p, acc, group_n, wn, 0, row0, rows, lane, memory);
}

// ---- a tile or two for every CU ----
// Between the two: a group of 2 x WM waves takes 32 WM outputs and 32 WM rows, a wave 16 WM x 32, and both operands' codes come straight into LDS, three blocks
// ahead in four buffers, so that a CU with one group does not wait for memory block by block. WM = 4 takes all the LDS that a CU has. What bounds it is what a CU
// draws from L2, some 27 bytes a cycle: where 128 x 128 leaves CUs without a group, 64 x 64 (WM = 2, two groups a CU) has the others draw too: 128 x 8192 x 8192 with
// cut sums in 20 us (32), 256 x 4096 x 4096 in 12 (18), 64 rows of the gated 8192 x 4096 in 15 (21); 1024 x 4096 x 4096 in 23 us with WM = 4.
// (2 x 2 waves of 64 x 64, one for each SIMD, take longer than 2 x 4: 330 instructions a block, of which a wave alone issues one in 4.5 cycles.)
// EXACT converts each wave's codes to halves, 64 conversions beside 16 products a block: 512 x 4096 x 4096 in float32 takes 25 us, 33 on the larger tiles of
// f8_tile_kernel and 35 on f8_rows_kernel's, 64 x 32000 x 4096 27 (35, 45), 1024 x 4096 x 4096 47 (39); 128 rows of the gated
// 8192 x 4096 in halves 27 (37, 48).
template <int WM, bool GATED, bool EXACT>
__global__ __launch_bounds__(128 * WM, 2) void f8_deep_kernel(const F8Params p) {
    exhip_touch_args(p);
    constexpr int WN = 2, TN = WM, TM = WN, kRows = 16 * TM * WM, kLoads = 5, kBuffers = 4, kWeights = 2048 * TN * WN, kCodes = kRows * kBlk, kBuffer = kWeights + kCodes + kRows * 4;
    __shared__ __attribute__((aligned(16))) char staged[kBuffers * kBuffer];
    const unsigned lds0 = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char*)staged;
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), wn = wave % WN, wm = wave / WN;
    const int q = lane / 16, col = lane % 16;
    int group_n, group_m;
    tile_of(p.groups_n, p.groups_m, &group_n, &group_m);
    const int tile0 = (group_n * WN + wn) * TN, row0 = p.first + group_m * kRows;
    const int rows = min(kRows, p.last - row0), tail = p.k % kBlk, blocks = p.blocks_k;
    const __amdgpu_buffer_rsrc_t xr = uniform_view(p.x + (size_t)row0 * p.x_stride, (rows - 1) * p.x_stride + (p.k + 15) / 16 * 16);
    // A wave stages 16 rows, eight with a load (as in f8_wide_kernel), and one of the group's tiles of weights.
    const int piece = (lane % 8) ^ (lane / 8);
    const bool behind = tail && piece * 16 >= tail;
    int off[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int row = wave * 16 + j * 8 + lane / 8;
        off[j] = row < rows ? row * p.x_stride + piece * 16 : kNoRow;
    }
    const int scale_part = wave % (kRows / 64) * 64, scale_off = min(scale_part + lane, rows - 1) * 4;
    const WeightRows weights(p, group_n * WN * TN + wave, 1, lane);
    auto stage = [&](int buffer, int j) {  // in five loads; behind the last block that one again, which nothing reads
        const int b = min(buffer, blocks - 1);
        const unsigned to = lds0 + buffer % kBuffers * kBuffer;
        if (j < 2) load16_to_lds(weights.view, weights.at, b * 2048 + j * 1024, to + (wave * 2 + j) * 1024);
        else if (j < 4) load16_to_lds(xr, behind && b == blocks - 1 ? kNoRow : off[j - 2], b * kBlk, to + kWeights + (wave * 16 + (j - 2) * 8) * kBlk);
        else load4_to_lds(uniform_view(p.x_scale + (size_t)b * p.m + row0, rows * 4), scale_off, to + kWeights + kCodes + scale_part * 4);
    };
    const int block_n = min(GATED ? tile0 / 2 : tile0, (p.n - 1) / 16) / (kBlk / 16);
    const Constants ws = (Constants)(uintptr_t)(p.w_scale + (size_t)block_n * blocks);
    const Constants ws_up = (Constants)(uintptr_t)(GATED ? p.w_scale_up + (size_t)block_n * blocks : nullptr);
    const int at_w = wn * TN * 2048 + lane * 16;
    auto weights_from = [&](int b, int i) {
        const char* const from = staged + b % kBuffers * kBuffer + at_w + i * 2048;
        return both(*reinterpret_cast<const v4i*>(from), *reinterpret_cast<const v4i*>(from + 1024));
    };
    const int at = kWeights + (wm * TM * 16 + col) * kBlk + (q ^ (col & 7)) * 16, at_hi = kWeights + (wm * TM * 16 + col) * kBlk + (q ^ (col & 7) ^ 4) * 16;
    const int at_scale = kWeights + kCodes + (wm * TM * 16 + col) * 4;
    struct Rows {
        v8i v;
        float s;
    };
    auto rows_from = [&](int b, int t) {
        const char* const from = staged + b % kBuffers * kBuffer;
        return Rows{both(*reinterpret_cast<const v4i*>(from + at + t * 16 * kBlk), *reinterpret_cast<const v4i*>(from + at_hi + t * 16 * kBlk)),
                    *reinterpret_cast<const float*>(from + at_scale + t * 64)};
    };
    v4f acc[TN][TM];
#pragma unroll
    for (int i = 0; i < TN; ++i)
#pragma unroll
        for (int t = 0; t < TM; ++t) acc[i][t] = v4f{0.f, 0.f, 0.f, 0.f};
    auto arrive = [&]() {
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    auto cut_row_end = [&](int b) {  // the piece that a row's end cuts; whether there is one
        if (p.k % 16 && b == blocks - 1) {
            if (threadIdx.x < kRows) {
                v4i* const cut = reinterpret_cast<v4i*>(staged + b % kBuffers * kBuffer + kWeights + threadIdx.x * kBlk + ((tail / 16) ^ (threadIdx.x & 7)) * 16);
                *cut &= keep_first(tail % 16);
            }
            __syncthreads();
            return true;
        }
        return false;
    };
#pragma unroll
    for (int j = 0; j < 3 * kLoads; ++j) stage(j / kLoads, j % kLoads);
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * kLoads) : "memory");
    arrive();
    float s_w = ws[0], s_up = GATED ? ws_up[0] : 0.f, s_next = 0.f, s_up_next = 0.f;
    struct Weights {
        v8i v[TN];
    } w0, w1;
#pragma unroll
    for (int i = 0; i < TN; ++i) w0.v[i] = weights_from(0, i);
    Rows x[2];
    x[0] = rows_from(0, 0);
    constexpr int kLag = 3, kSteps = TN * TM;
    auto block = [&](Weights& w, Weights& next, int b) {
        if (cut_row_end(b)) x[0] = rows_from(b, 0);
        v4f part[kLag + 1];
        float s[2], su[2];
        Halves weights_h[EXACT ? TN : 1], rows_h;
#pragma unroll
        for (int u = 0; u < kSteps + kLag; ++u) {
            const int t = u / TN, i = u % TN;
            if constexpr (EXACT) {
                if (u < kSteps && i == 0) rows_h = halves_of(x[t % 2].v);
                if (u < TN) weights_h[u] = halves_of(w.v[u]);
            }
            if (u == kSteps / 2) {
                asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kLoads) : "memory");  // the next block's are there, the one's behind it are on their way
                arrive();
                const int after = min(b + 1, blocks - 1);
                s_next = ws[after];
                if constexpr (GATED) s_up_next = ws_up[after];
            }
            if (u >= kSteps / 2 && u < kSteps / 2 + kLoads) stage(b + 3, u - kSteps / 2);
            if (u >= kSteps / 2 && u < kSteps / 2 + TN) next.v[u - kSteps / 2] = weights_from(b + 1, u - kSteps / 2);
            if (u < kSteps) {
                if (i == 0) {
                    s[t % 2] = s_w * x[t % 2].s;
                    su[t % 2] = s_up * x[t % 2].s;
                    x[(t + 1) % 2] = t + 1 < TM ? rows_from(b, t + 1) : rows_from(b + 1, 0);
                }
                if constexpr (EXACT) part[u % (kLag + 1)] = block_product(weights_h[i], rows_h);
                else part[u % (kLag + 1)] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w.v[i], x[t % 2].v, v4f{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
            }
            if (u >= kLag) {
                const int v = u - kLag, vt = v / TN, vi = v % TN;
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[vi][vt][e] = __builtin_fmaf(part[v % (kLag + 1)][e], GATED && vi % 2 ? su[vt % 2] : s[vt % 2], acc[vi][vt][e]);
                asm volatile("" : "+v"(acc[vi][vt]));
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        s_w = s_next;
        s_up = s_up_next;
    };
    for (int b = 0; b < blocks; b += 2) {
        block(w0, w1, b);
        if (b + 1 < blocks) block(w1, w0, b + 1);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // what was staged behind the end, in front of the results' barrier
    if constexpr (!GATED) write_group<16, WN, WM, EXACT>(p, acc, group_n, wn, wm, row0, rows, lane, staged);
    else write_gated_group<16, WN, WM, false>(p, acc, group_n, wn, wm, row0, rows, lane, staged);
}

int blocks_of(int v) { return v / kBlk + (v % kBlk != 0); }
bool aligned(const void* p, uintptr_t to) { return (uintptr_t)p % to == 0; }
bool sizes_ok(int n, int k) { return n > 0 && k > 0 && n <= (1 << 24) && k <= kMostStride; }

template <typename T>
int quantize_rows(exhip_ctx* ctx, const char* name, const T* x, int x_stride, int m, int k, uint8_t* y, int y_stride, float* scale) {
    EXHIP_REQUIRE(ctx && x && y && scale, "%s: NULL argument", name);
    EXHIP_REQUIRE(m > 0 && k > 0 && k <= kMostStride && x_stride >= k, "%s: %d rows of %d values, %d apart: sizes are positive, a row at most 2^22 values", name, m, k, x_stride);
    EXHIP_REQUIRE(m <= 1 << 26, "%s: %d rows are more than one launch takes", name, m);
    EXHIP_REQUIRE(y_stride >= k && y_stride % 16 == 0 && y_stride <= kMostStride && aligned(y, 16), "%s: rows of codes begin on 16 bytes and hold the row (stride %d)", name, y_stride);
    EXHIP_REQUIRE(aligned(x, sizeof(T)) && aligned(scale, 4), "%s: an operand's address is not that of its type", name);
    const exhip_on_device on(ctx->device);
    EXHIP_CHECK(on.error);
    hipLaunchKernelGGL(quantize_rows_kernel<T>, dim3(m / 16 + (m % 16 != 0), blocks_of(k)), dim3(256), 0, ctx->stream, x, x_stride, m, k, y, y_stride, scale);
    EXHIP_LAUNCH_CHECK();
    return 0;
}

int check_product(exhip_ctx* ctx, const char* name, const exhip_f8_desc* d, const uint8_t* x, const float* x_scale, const void* w, const float* w_scale, const float* bias) {
    EXHIP_REQUIRE(ctx && d && x && x_scale && w && w_scale, "%s: NULL argument", name);
    EXHIP_REQUIRE(d->m > 0 && sizes_ok(d->n_out, d->k_in), "%s: %d rows, %d outputs, %d inputs: sizes are positive, at most 2^24 outputs of 2^22 inputs", name, d->m, d->n_out, d->k_in);
    EXHIP_REQUIRE(d->x_stride >= d->k_in && d->x_stride % 16 == 0 && d->x_stride <= kMostStride && aligned(x, 16),
                  "%s: rows of codes begin on 16 bytes and hold the row (stride %d)", name, d->x_stride);
    EXHIP_REQUIRE(d->y_stride >= d->n_out, "%s: result rows of %d values are %d apart", name, d->n_out, d->y_stride);
    EXHIP_REQUIRE(aligned(w, 16) && aligned(x_scale, 4) && aligned(w_scale, 4) && aligned(bias, 4), "%s: an operand's address is not that of its type", name);
    return 0;
}

F8Params params_of(const exhip_f8_desc* d, const uint8_t* x, const float* x_scale, const void* w, bool gated_product) {
    F8Params p = {};
    p.x = x;
    p.x_scale = x_scale;
    p.w = static_cast<const uint8_t*>(w);
    p.m = p.last = d->m;
    p.n = d->n_out;
    p.k = d->k_in;
    p.x_stride = d->x_stride;
    p.y_stride = d->y_stride;
    p.blocks_k = blocks_of(d->k_in);
    p.tiles = (d->n_out + 15) / 16 * (gated_product ? 2 : 1);
    return p;
}

template <typename K>
int launch(exhip_ctx* ctx, K kernel, F8Params p, int tiles, int rows, int threads) {
    p.groups_n = (p.tiles + tiles - 1) / tiles;
    p.groups_m = (p.last - p.first - 1) / rows + 1;
    const long long groups = (long long)p.groups_n * p.groups_m;
    EXHIP_REQUIRE(groups <= 0x7fffffff / threads, "inner product: %d rows of %d outputs are more than one launch takes", p.last - p.first, p.n);
    const exhip_on_device on(ctx->device);
    EXHIP_CHECK(on.error);
    hipLaunchKernelGGL(kernel, dim3((unsigned)groups), dim3(threads), 0, ctx->stream, p);
    EXHIP_LAUNCH_CHECK();
    return 0;
}

// One way to run a product: the tiles of 16 outputs (of both projections) and the rows a group takes, how many groups a CU runs at once, how many waves share a
// group's blocks, and what a launch takes: `start` us, and for each time that all CUs are given groups `round` and, for each block that one wave goes through,
// `block`; `alone` where a CU that could run two groups has one.
struct Form {
    int (*run)(exhip_ctx*, const F8Params&);
    int tiles, rows, at_once, split;
    float start, round, block, alone;
    bool drawn;  // whether its loads may be what bounds it
};
template <int TN, int TM, int WN, int WK, int D, bool GATED>
int run_rows(exhip_ctx* ctx, const F8Params& p) {
    return launch(ctx, f8_rows_kernel<TN, TM, WN, WK, D, GATED>, p, TN * WN, 16 * TM, 64 * WN * WK);
}
template <bool GATED>
int run_tile(exhip_ctx* ctx, const F8Params& p) {
    return launch(ctx, f8_tile_kernel<GATED>, p, 16, 64, 256);
}
template <int WM, bool GATED, bool EXACT>
int run_deep(exhip_ctx* ctx, const F8Params& p) {
    return launch(ctx, f8_deep_kernel<WM, GATED, EXACT>, p, 2 * WM, 32 * WM, 128 * WM);
}
template <bool GATED>
int run_wide(exhip_ctx* ctx, const F8Params& p) {
    return launch(ctx, f8_wide_kernel<GATED>, p, 16, 256, 512);
}
// The times are fits to launches of 1 to 2048 rows and matrices from 256 x 512 to 8192 x 8192 and 32000 x 4096, on the GPU's clock. Over 94 to 96 shapes a list the
// launch that they choose takes up to 0.7 % longer than the best form on average, 12 % at most (profiles/inner_f8_forms.txt).
constexpr Form kExact[] = {  // results in float32 or halves
    {run_rows<1, 1, 1, 8, 4, false>, 1, 16, 2, 8, 1.5f, 1.9f, 0.97f, 0.58f, true}, {run_rows<2, 1, 1, 8, 2, false>, 2, 16, 2, 8, 0.3f, 3.1f, 1.74f, 0.64f, true},
    {run_rows<2, 2, 1, 8, 2, false>, 2, 32, 1, 8, 1.7f, 1.5f, 1.37f, 0.f, true},   {run_rows<4, 2, 1, 8, 1, false>, 4, 32, 1, 8, 1.0f, 2.5f, 1.80f, 0.f, true},
    {run_deep<2, false, true>, 4, 64, 2, 1, 2.2f, 1.8f, 0.64f, 0.46f, true},       {run_tile<false>, 16, 64, 2, 1, 0.f, 5.0f, 1.69f, 0.89f, false},
};
constexpr Form kCut[] = {  // results in halves whose sums may be cut
    kExact[0], kExact[1], kExact[2], kExact[3],
    {run_deep<2, false, false>, 4, 64, 2, 1, 0.3f, 3.3f, 0.30f, 0.26f, true}, {run_deep<4, false, false>, 8, 128, 1, 1, 0.5f, 3.7f, 0.50f, 0.f, true},
    {run_wide<false>, 16, 256, 1, 1, 0.f, 7.4f, 1.17f, 0.f, false},
};
constexpr Form kGated[] = {  // results in halves
    {run_rows<2, 1, 1, 8, 2, true>, 2, 16, 2, 8, 2.5f, 1.5f, 1.95f, 0.85f, true}, {run_rows<2, 2, 1, 8, 2, true>, 2, 32, 1, 8, 1.4f, 2.4f, 1.34f, 0.f, true},
    {run_rows<4, 2, 1, 8, 1, true>, 4, 32, 1, 8, 1.3f, 2.6f, 1.90f, 0.f, true},   {run_deep<2, true, true>, 4, 64, 2, 1, 3.4f, 2.2f, 0.665f, 0.465f, true},
    {run_tile<true>, 16, 64, 2, 1, 5.5f, 3.0f, 1.85f, 0.89f, false},
};
constexpr Form kGatedCut[] = {
    kGated[0], kGated[1], kGated[2], {run_deep<2, true, false>, 4, 64, 2, 1, 2.0f, 2.9f, 0.39f, 0.27f, true},
    {run_deep<4, true, false>, 8, 128, 1, 1, 1.6f, 4.3f, 0.55f, 0.f, true}, {run_wide<true>, 16, 256, 1, 1, 0.1f, 15.2f, 1.33f, 0.f, false},
};
constexpr Form kGatedCodes[] = {  // a group has whole blocks of the result: 16 tiles
    {run_rows<4, 1, 4, 4, 1, true>, 16, 16, 1, 4, 0.9f, 3.0f, 2.12f, 0.f, true}, {run_rows<4, 2, 4, 2, 1, true>, 16, 32, 1, 2, 0.f, 5.2f, 1.40f, 0.f, true},
    {run_tile<true>, 16, 64, 2, 1, 0.f, 8.7f, 1.68f, 0.92f, false},
};

constexpr int kCus = 256;

// What a launch of a form takes for some rows, in us.
float time_of(const Form& f, const F8Params& p, int rows) {
    const int groups_n = (p.tiles + f.tiles - 1) / f.tiles, groups_m = (rows - 1) / f.rows + 1;
    const long long times = ((long long)groups_n * groups_m - 1) / kCus + 1, full = times / f.at_once, rest = times % f.at_once;
    const float us = f.start + (float)(full + rest) * f.round + ((float)full * f.block + (float)rest * f.alone) * (float)((p.blocks_k - 1) / f.split + 1);
    if (!f.drawn) return us;
    // all loads together, in bytes a us: the weights once from memory, what groups read again, weights and rows, from L2
    const float weights = (float)p.tiles * (float)p.blocks_k * 2048.f, again = (float)(groups_m - 1) * weights + (float)groups_n * (float)rows * (float)p.blocks_k * 128.f;
    return fmaxf(us, f.start + weights / 7.9e6f + again / 19e6f);
}
template <int N>
int best_of(const Form (&forms)[N], const F8Params& p, int rows, float* us) {
    int best = 0;
    for (int i = 0; i < N; ++i) {
        const float t = time_of(forms[i], p, rows);
        if (i == 0 || t < *us) {
            best = i;
            *us = t;
        }
    }
    return best;
}

// One launch, or two where the last rows would have a few CUs work while the others are done, and a kernel of smaller tiles takes them: 3 us, less than nothing
// for short launches, then 20 % and more for some shapes (1657 x 2920 x 5785 with cut sums 60 -> 48 us, 2711 x 3052 x 2961 in float32 68 -> 56). Over 60 shapes of a list
// for which two are chosen, one launch takes 10 to 18 % longer on average; where the choice is wrong it costs 9 % at most.
// (Quantized results stay in one: their kernels for few rows take what two launches win.)
template <int N>
int run_best(exhip_ctx* ctx, const F8Params& p, const Form (&forms)[N], bool in_two = true) {
    const int pinned = g_exhip_options.f8_form, pinned_front = g_exhip_options.f8_front;
    float us = 0.f;
    int best = best_of(forms, p, p.m, &us), behind = best, rows = p.m;
    if (pinned > 0) best = behind = (pinned < N ? pinned : N) - 1;
    if (pinned_front > 0) rows = pinned_front < p.m ? pinned_front : p.m;
    if (in_two && us > 12.f && pinned <= 0 && pinned_front <= 0) {
        us = us * 0.97f - 3.f;
        for (int i = 0; i < N; ++i) {
            const Form& f = forms[i];
            const int groups_n = (p.tiles + f.tiles - 1) / f.tiles, at_once = kCus * f.at_once;
            const int whole = p.m / f.rows, filled = (int)((long long)groups_n * whole / at_once * at_once / groups_n);  // in tiles of rows
            for (const int some : {whole, filled}) {
                const int front = some * f.rows;
                if (some == 0 || front == p.m) continue;
                float rest = 0.f;
                const int next = best_of(forms, p, p.m - front, &rest);
                const float both = time_of(f, p, front) + rest;
                if (both < us) {
                    us = both;
                    best = i;
                    behind = next;
                    rows = front;
                }
            }
        }
    }
    F8Params part = p;
    part.last = rows;
    const int rc = forms[best].run(ctx, part);
    if (rc != 0 || rows == p.m) return rc;
    part.first = rows;
    part.last = p.m;
    return forms[behind].run(ctx, part);
}

}  // namespace

extern "C" int exhip_quantize_rows_f32_to_f8(exhip_ctx* ctx, const float* x, int x_stride, int m, int k, uint8_t* y, int y_stride, float* scale) {
    return quantize_rows(ctx, "exhip_quantize_rows_f32_to_f8", x, x_stride, m, k, y, y_stride, scale);
}
extern "C" int exhip_quantize_rows_f16_to_f8(exhip_ctx* ctx, const uint16_t* x, int x_stride, int m, int k, uint8_t* y, int y_stride, float* scale) {
    return quantize_rows(ctx, "exhip_quantize_rows_f16_to_f8", x, x_stride, m, k, y, y_stride, scale);
}

extern "C" int exhip_quantize_blocks_f32_to_f8(exhip_ctx* ctx, const float* w, int n, int k, uint8_t* y, float* scale) {
    EXHIP_REQUIRE(ctx && w && y && scale, "exhip_quantize_blocks_f32_to_f8: NULL argument");
    EXHIP_REQUIRE(sizes_ok(n, k), "exhip_quantize_blocks_f32_to_f8: %d x %d: sizes are positive, at most 2^24 outputs of 2^22 inputs", n, k);
    EXHIP_REQUIRE(aligned(w, 4) && aligned(scale, 4), "exhip_quantize_blocks_f32_to_f8: an operand's address is not that of its type");
    const long long blocks = (long long)blocks_of(n) * blocks_of(k);
    EXHIP_REQUIRE(blocks <= 0x7fffffff / 256, "exhip_quantize_blocks_f32_to_f8: %lld blocks are more than one launch takes", blocks);
    const exhip_on_device on(ctx->device);
    EXHIP_CHECK(on.error);
    hipLaunchKernelGGL(quantize_blocks_kernel, dim3((unsigned)blocks), dim3(256), 0, ctx->stream, w, n, k, blocks_of(k), y, scale);
    EXHIP_LAUNCH_CHECK();
    return 0;
}

extern "C" size_t exhip_f8_packed_bytes(int n_out, int k_in, int gated_weights) {
    if (!sizes_ok(n_out, k_in)) {
        exhip_set_error("exhip_f8_packed_bytes: %d outputs, %d inputs: sizes are positive, at most 2^24 outputs of 2^22 inputs", n_out, k_in);
        return 0;
    }
    return (size_t)((n_out + 15) / 16) * (gated_weights ? 2 : 1) * blocks_of(k_in) * 2048;
}

extern "C" int exhip_f8_pack_weights(exhip_ctx* ctx, int n_out, int k_in, const uint8_t* w, const uint8_t* w_up, void* packed) {
    EXHIP_REQUIRE(ctx && w && packed, "exhip_f8_pack_weights: NULL argument");
    const size_t bytes = exhip_f8_packed_bytes(n_out, k_in, w_up != nullptr);
    if (bytes == 0) return EXHIP_ERR_ARG;
    EXHIP_REQUIRE(aligned(packed, 16), "exhip_f8_pack_weights: packed weights begin on 16 bytes");
    const size_t pieces = bytes / 16, groups = (pieces + 255) / 256;
    EXHIP_REQUIRE(groups <= 0x7fffffff / 256, "exhip_f8_pack_weights: %zu bytes are more than one launch takes", bytes);
    const exhip_on_device on(ctx->device);
    EXHIP_CHECK(on.error);
    hipLaunchKernelGGL(pack_f8_kernel, dim3((unsigned)groups), dim3(256), 0, ctx->stream, w, w_up, n_out, k_in, blocks_of(k_in), pieces, static_cast<v4i*>(packed));
    EXHIP_LAUNCH_CHECK();
    return 0;
}

namespace {

int product(exhip_ctx* ctx, const char* name, const exhip_f8_desc* d, const uint8_t* x, const float* x_scale, const void* w_packed, const float* w_scale, const float* bias,
            float* y_f32, uint16_t* y_f16, bool cut) {
    const int rc = check_product(ctx, name, d, x, x_scale, w_packed, w_scale, bias);
    if (rc != 0) return rc;
    EXHIP_REQUIRE((y_f32 || y_f16) && aligned(y_f32, 4) && aligned(y_f16, 2), "%s: no result, or one whose address is not that of its type", name);
    F8Params p = params_of(d, x, x_scale, w_packed, false);
    p.w_scale = w_scale;
    p.bias = bias;
    p.y_f32 = y_f32;
    p.y_f16 = y_f16;
    return cut ? run_best(ctx, p, kCut) : run_best(ctx, p, kExact);
}

int gated_product(exhip_ctx* ctx, const char* name, const exhip_f8_desc* d, int gate, const uint8_t* x, const float* x_scale, const void* w_packed, const float* w_scale_gate,
                  const float* w_scale_up, const float* bias_gate, const float* bias_up, uint16_t* y_f16, uint8_t* y_f8, float* y_scale, bool cut) {
    const int rc = check_product(ctx, name, d, x, x_scale, w_packed, w_scale_gate, bias_gate);
    if (rc != 0) return rc;
    EXHIP_REQUIRE(w_scale_up && aligned(w_scale_up, 4) && aligned(bias_up, 4) && !bias_gate == !bias_up, "%s: both projections have scales, and both a bias or neither", name);
    EXHIP_REQUIRE(gate >= EXHIP_GATE_SILU && gate <= EXHIP_GATE_RELU, "%s: unknown activation %d", name, gate);
    EXHIP_REQUIRE(!y_f16 != !y_f8 && !y_f8 == !y_scale, "%s: one result: halves, or codes and their scales", name);
    EXHIP_REQUIRE(aligned(y_f16, 2) && aligned(y_scale, 4), "%s: a result's address is not that of its type", name);
    EXHIP_REQUIRE(!y_f8 || (aligned(y_f8, 16) && d->y_stride % 16 == 0 && d->y_stride <= kMostStride), "%s: rows of codes begin on 16 bytes (stride %d)", name, d->y_stride);
    F8Params p = params_of(d, x, x_scale, w_packed, true);
    p.w_scale = w_scale_gate;
    p.w_scale_up = w_scale_up;
    p.bias = bias_gate;
    p.bias_up = bias_up;
    p.y_f16 = y_f16;
    p.y_f8 = y_f8;
    p.y_scale = y_scale;
    p.gate = gate;
    if (y_f8) return run_best(ctx, p, kGatedCodes, false);
    return cut ? run_best(ctx, p, kGatedCut) : run_best(ctx, p, kGated);
}

}  // namespace

extern "C" int exhip_innerproduct_f8(exhip_ctx* ctx, const exhip_f8_desc* d, const uint8_t* x, const float* x_scale, const void* w_packed, const float* w_scale,
                                     const float* bias, float* y_f32, uint16_t* y_f16) {
    return product(ctx, "exhip_innerproduct_f8", d, x, x_scale, w_packed, w_scale, bias, y_f32, y_f16, false);
}
extern "C" int exhip_innerproduct_cut_f8(exhip_ctx* ctx, const exhip_f8_desc* d, const uint8_t* x, const float* x_scale, const void* w_packed, const float* w_scale,
                                         const float* bias, uint16_t* y_f16) {
    return product(ctx, "exhip_innerproduct_cut_f8", d, x, x_scale, w_packed, w_scale, bias, nullptr, y_f16, true);
}

extern "C" int exhip_innerproduct_gated_f8(exhip_ctx* ctx, const exhip_f8_desc* d, int gate, const uint8_t* x, const float* x_scale, const void* w_packed,
                                           const float* w_scale_gate, const float* w_scale_up, const float* bias_gate, const float* bias_up, uint16_t* y_f16,
                                           uint8_t* y_f8, float* y_scale) {
    return gated_product(ctx, "exhip_innerproduct_gated_f8", d, gate, x, x_scale, w_packed, w_scale_gate, w_scale_up, bias_gate, bias_up, y_f16, y_f8, y_scale, false);
}
extern "C" int exhip_innerproduct_gated_cut_f8(exhip_ctx* ctx, const exhip_f8_desc* d, int gate, const uint8_t* x, const float* x_scale, const void* w_packed,
                                               const float* w_scale_gate, const float* w_scale_up, const float* bias_gate, const float* bias_up, uint16_t* y_f16) {
    return gated_product(ctx, "exhip_innerproduct_gated_cut_f8", d, gate, x, x_scale, w_packed, w_scale_gate, w_scale_up, bias_gate, bias_up, y_f16, nullptr, nullptr, true);
}
