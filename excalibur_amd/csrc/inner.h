// What the inner products in 8-bit floating point and in 8-bit integers share: loads, which tiles a group takes, results through LDS.
#pragma once
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

constexpr int kRsrcWord3 = 0x00020000;

template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Eight {  // eight values at any alignment of their type
    T v[8];
};
__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(uint16_t v) { return exhip_h2f(v); }

__device__ __forceinline__ float gated(int gate, float g, float u) {
    switch (gate) {
    case EXHIP_GATE_SILU: return g / (1.f + expf(-g)) * u;
    case EXHIP_GATE_GELU: return 0.5f * g * (1.f + erff(g * 0.70710678118654752f)) * u;
    case EXHIP_GATE_SIGMOID: return u / (1.f + expf(-g));
    default: return (g > 0.f ? g : g != g ? g : 0.f) * u;
    }
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

// Which tiles a group takes: each of the 8 XCDs a run of neighbouring ones, in bands of eight row tiles, so that the groups that run on an XCD at a time share
// rows and weights in its L2.
__device__ __forceinline__ int place_of(int group, int total) {
    const int xcd = group % 8, per = total / 8, more = total % 8;
    return xcd * per + min(xcd, more) + group / 8;
}
__device__ __forceinline__ void tile_at(int i, int groups_n, int groups_m, int* n, int* m) {
    const int band = i / (8 * groups_n), within = i % (8 * groups_n), high = min(8, groups_m - band * 8);
    *m = band * 8 + within % high;
    *n = within / high;
}
__device__ __forceinline__ void tile_of(int groups_n, int groups_m, int* n, int* m) { tile_at(place_of(blockIdx.x, groups_n * groups_m), groups_n, groups_m, n, m); }

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
// `past_l2` is for rows that begin on lines: lines that two groups write parts of are put together in L2 (8192 x 5003 in halves 68 us past it, 61 through it).
template <typename O, int WIDTH, int ROWS, int THREADS>
__device__ __forceinline__ void store_rows(const char* lds, O* y, size_t stride, int row0, int rows, int j0, int n, bool past_l2 = true) {
    constexpr int kPer = 16 / sizeof(O), kPieces = WIDTH / kPer, kPitch = WIDTH * (int)sizeof(O), kTogether = THREADS / kPieces;
    static_assert(THREADS % kPieces == 0 && ROWS % kTogether == 0, "every thread stores one piece of every kTogether-th row");
    const int piece = threadIdx.x % kPieces, first = threadIdx.x / kPieces, j = j0 + piece * kPer;
    O* const dst = y + (size_t)(row0 + first) * stride + j;
    const size_t step = (size_t)kTogether * stride;
    const bool whole = j + kPer <= n;
    auto held = [&](int row) { return *reinterpret_cast<const v4i*>(lds + row * kPitch + byte_in_row<O, WIDTH>(row, piece * 16)); };
    if (past_l2) {
#pragma unroll 4
        for (int i = 0; i < ROWS / kTogether; ++i) {
            const int row = i * kTogether + first;
            const v4i v = held(row);
            if (whole && row < rows) __builtin_nontemporal_store(v, reinterpret_cast<v4i_any*>(dst + i * step));
        }
    } else {
#pragma unroll 4
        for (int i = 0; i < ROWS / kTogether; ++i) {
            const int row = i * kTogether + first;
            const v4i v = held(row);
            if (whole && row < rows) *reinterpret_cast<v4i_any*>(dst + i * step) = v;
        }
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

inline bool aligned(const void* p, uintptr_t to) { return (uintptr_t)p % to == 0; }

}  // namespace
