// td_fp8.cuh -- 8-bit floating point (e4m3) in blocks of 128: the scales, and the kernels that go from wider types to
// 8 bits and back.
//
//   a block's m = its largest finite magnitude; e = the smallest integer >= -126 with m 2^-e <= 448; scale = 2^e
//   q = e4m3(v 2^-e), to nearest, ties to even; an infinity or NaN becomes NaN (e4m3 has no infinity)
//
// Scales are powers of two: a product with one is exact, so a value is rounded once, a quantised value is exact in
// bfloat16, and values kept in 8 bits are quantised again along the other axis without a second rounding (but for those
// below the other block's smallest step). Floating-point codes lose nothing by it: their relative step is the same
// anywhere in the range. Blocks are 1 x 128 (activations: along the contraction), 128 x 1 (the same tensors when rows
// are contracted, as in the weight's gradient) or 128 x 128 (weights, whose blocks stay blocks when transposed).
//
// fp8_rows_kernel (1 x 128 alone) reads a row in 16-byte vectors, 128 / VEC lanes to a block. fp8_tile_kernel takes
// 128 x 128 values into registers, once, for any of: the 1 x 128 form, the 128 x 1 form transposed, the 128 x 128 form
// or its transpose, and column sums. Both are bound by memory.
#pragma once

#include <cuda_fp8.h>

#include "td_common.cuh"
#include "td_ptx.cuh"

namespace td {

constexpr int kBlock8 = 128;  // values that share a scale, along an axis

struct E4m3 {  // a stored e4m3 number
    uint8_t bits;
};

// Exponent of a block's scale from its largest finite magnitude: 448 = 1.75 * 2^8, so the mantissa decides by 1.75.
__device__ __forceinline__ int scale_exponent(float amax) {
    const int e = int((__float_as_uint(amax) + 0x1FFFFFu) >> 23) - 135;
    return e < -126 ? -126 : e;
}
__device__ __forceinline__ float exp2_int(int e) { return __uint_as_float(uint32_t(e + 127) << 23); }  // -126 .. 127

// Largest |v|: infinite where there is an infinity; a NaN counts for nothing.
template <int N>
__device__ __forceinline__ float largest(const float* v) {
    float top = fabsf(v[0]) > 0.f ? fabsf(v[0]) : 0.f;
#pragma unroll
    for (int i = 1; i < N; ++i) top = fmaxf(top, fabsf(v[i]));
    return top;
}
// Infinities to NaN, which they become in e4m3 and which counts for nothing above. The kernels look for the largest
// magnitude first, and come here only where that is infinite.
__device__ __forceinline__ bool infinite(float top) { return top == __int_as_float(0x7F800000); }
template <int N>
__device__ __forceinline__ void drop_infinities(float* v) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = fmaf(v[i], 0.f, v[i]);
}

// Two values without infinities times 2^-e as e4m3 (the first in the low byte).
__device__ __forceinline__ uint32_t to_e4m3x2(float a, float b, float inv) {
    return __nv_cvt_float2_to_fp8x2(make_float2(a * inv, b * inv), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ uint32_t to_e4m3x4(const float* v, float inv) {
    return to_e4m3x2(v[0], v[1], inv) | to_e4m3x2(v[2], v[3], inv) << 16;
}

__device__ __forceinline__ float2 from_e4m3x2(uint32_t two) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(__nv_fp8x2_storage_t(two & 0xFFFFu), __NV_E4M3);
    return __half22float2(__half2(h));
}
__device__ __forceinline__ float from_e4m3(uint8_t one) { return from_e4m3x2(one).x; }

// ---- 1 x 128 blocks ---------------------------------------------------------------------------------------------

struct RowsArgs {
    const void* x;        // [M, K] dense
    uint8_t* q;           // [M, pitch]; what lies behind K in a row is written as zeros
    float* scale;         // [M, KB]
    long long M;
    int K, KB, pitch;
};

constexpr int kRowsThreads = 256;

// WIDE: K is a multiple of a 16-byte vector's elements and x is 16-byte aligned; a warp takes 32 vectors of a row.
// Otherwise a warp takes one block, four neighbouring elements a lane.
template <typename T, bool WIDE>
__global__ void __launch_bounds__(kRowsThreads) fp8_rows_kernel(const RowsArgs a) {
    constexpr int VEC = WIDE ? Elem<T>::kVec : 4;
    constexpr int kLanes = kBlock8 / VEC;  // of a block
    const int lane = threadIdx.x & 31;
    const int chunks = (a.K + 32 * VEC - 1) / (32 * VEC);
    const long long tasks = a.M * chunks, step = (long long)gridDim.x * (kRowsThreads / 32);
    grid_dependency_wait();
    launch_dependents();
    for (long long t = (long long)blockIdx.x * (kRowsThreads / 32) + (threadIdx.x >> 5); t < tasks; t += step) {
        const long long row = tasks <= 0x7FFFFFFFLL ? uint32_t(t) / uint32_t(chunks) : t / chunks;
        const int c = (int(t - row * chunks) * 32 + lane) * VEC;
        const T* src = static_cast<const T*>(a.x) + row * a.K + c;
        float v[VEC];
        if constexpr (WIDE) {
            if (c < a.K) load16<T>(src, v);
            else {
#pragma unroll
                for (int i = 0; i < VEC; ++i) v[i] = 0.f;
            }
        } else {
#pragma unroll
            for (int i = 0; i < VEC; ++i) v[i] = c + i < a.K ? to_acc(src[i]) : 0.f;
        }
        float top = largest<VEC>(v);
        if (infinite(top)) {
            drop_infinities<VEC>(v);
            top = largest<VEC>(v);
        }
#pragma unroll
        for (int o = kLanes / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const int e = scale_exponent(top);
        if (c < a.K && lane % kLanes == 0) a.scale[row * a.KB + c / kBlock8] = exp2_int(e);
        const float inv = exp2_int(-e);
        if (c < a.pitch) {  // (the pitch is a multiple of 16)
            uint8_t* dst = a.q + row * a.pitch + c;
            if constexpr (VEC == 8) *reinterpret_cast<uint2*>(dst) = make_uint2(to_e4m3x4(v, inv), to_e4m3x4(v + 4, inv));
            else *reinterpret_cast<uint32_t*>(dst) = to_e4m3x4(v, inv);
        }
    }
}

// K a multiple of 128 (and x 32-byte aligned): blocks follow one another whatever the rows, so nothing is divided. A
// thread takes 16 neighbouring values, eight a block, and has the next 16's loads under way.
__device__ __forceinline__ void load_32b(const void* p, uint4& lo, uint4& hi) {
    asm volatile("ld.global.nc.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(lo.x), "=r"(lo.y), "=r"(lo.z), "=r"(lo.w), "=r"(hi.x), "=r"(hi.y), "=r"(hi.z), "=r"(hi.w)
                 : "l"(p));
}
template <typename T>
__global__ void __launch_bounds__(kRowsThreads) fp8_flat_kernel(const RowsArgs a) {
    constexpr int kRaw = 16 * int(sizeof(T)) / 16;  // 16-byte vectors of 16 values
    const long long total = a.M * (a.K / 16), step = (long long)gridDim.x * kRowsThreads;
    grid_dependency_wait();
    launch_dependents();
    uint4 raw[kRaw];
    auto fetch = [&](long long i) {
        if (i < total) {
            const char* src = static_cast<const char*>(a.x) + i * (16 * int(sizeof(T)));
#pragma unroll
            for (int k = 0; k < kRaw; k += 2) load_32b(src + k * 16, raw[k], raw[k + 1]);
        }
    };
    long long i = (long long)blockIdx.x * kRowsThreads + threadIdx.x;
    fetch(i);
    for (; i < total; i += step) {  // (a block's 8 threads are all in or all out)
        float v[16];
#pragma unroll
        for (int k = 0; k < kRaw; ++k) unpack16<T>(raw[k], v + k * Elem<T>::kVec);
        fetch(i + step);
        float top = largest<16>(v);
        if (infinite(top)) {
            drop_infinities<16>(v);
            top = largest<16>(v);
        }
        const uint32_t eight = 0xFFu << (threadIdx.x & 24);
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(eight, top, o));
        const int e = scale_exponent(top);
        const float inv = exp2_int(-e);
        if ((threadIdx.x & 7) == 0) a.scale[i >> 3] = exp2_int(e);
        *reinterpret_cast<uint4*>(a.q + i * 16) = make_uint4(to_e4m3x4(v, inv), to_e4m3x4(v + 4, inv),
                                                             to_e4m3x4(v + 8, inv), to_e4m3x4(v + 12, inv));
    }
}

// ---- 128 x 128 tiles --------------------------------------------------------------------------------------------

struct TileArgs {
    const void* x;           // [M, C], rows `ld` apart: floating, or e4m3 with
    const float* x_scale;    //   its scales [M, CB] (1 x 128)
    long long ld;
    uint8_t* q;              // or null: [M, q_pitch], in 1 x 128 blocks, or 128 x 128 (TILE)
    float* scale;            //   [M, CB], or [MB, CB]
    uint8_t* qt;             // or null: the transpose [C, qt_pitch], in blocks of 128 rows of x, or 128 x 128
    float* scale_t;          //   [MB, scale_t_pitch] (one for each column), or [CB, MB]
    float* sums;             // or null: [MB, C] sums over a tile's rows
    long long M, q_pitch, qt_pitch, scale_t_pitch;
    int C, CB, MB;
};

constexpr int kTileThreads = 256;

// A thread holds 8 rows x 8 columns of the tile: rows 8 ty .. 8 ty + 7, columns 8 tx .. 8 tx + 7 (tx < 16).
// WIDE: rows of x start on 16-byte boundaries (8-byte ones for e4m3) and C is a multiple of 8.
template <typename T, bool WIDE, bool TILE>
__global__ void __launch_bounds__(kTileThreads) fp8_tile_kernel(const TileArgs a) {
    constexpr bool kFrom8 = sizeof(T) == 1;
    __shared__ float red[16][kBlock8];
    __shared__ __align__(16) uint8_t turned[kBlock8 * kBlock8];
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const int cb = blockIdx.x;
    const long long mb = blockIdx.y + (long long)blockIdx.z * gridDim.y;
    if (mb >= a.MB) return;
    const long long r0 = mb * kBlock8 + ty * 8;
    const int c0 = cb * kBlock8 + tx * 8;
    grid_dependency_wait();
    launch_dependents();
    float v[8][8];
#pragma unroll
    for (int p = 0; p < 8; ++p) {
        const long long row = r0 + p;
        const T* src = static_cast<const T*>(a.x) + row * a.ld + c0;
        if (row >= a.M || c0 >= a.C) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[p][i] = 0.f;
        } else if constexpr (kFrom8) {
            const float s = a.x_scale[row * a.CB + cb];
            if constexpr (WIDE) {
                const uint2 w = __ldg(reinterpret_cast<const uint2*>(src));
                const uint32_t h[4] = {w.x, w.x >> 16, w.y, w.y >> 16};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 f = from_e4m3x2(h[i]);
                    v[p][2 * i] = f.x * s;
                    v[p][2 * i + 1] = f.y * s;
                }
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[p][i] = c0 + i < a.C ? from_e4m3(src[i].bits) * s : 0.f;
            }
        } else if constexpr (WIDE) {
#pragma unroll
            for (int i = 0; i < 8; i += Elem<T>::kVec) load16<T>(src + i, v[p] + i);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[p][i] = c0 + i < a.C ? to_acc(src[i]) : 0.f;
        }
    }
    if (a.sums != nullptr) {  // a thread's rows in order, then the 16 groups of rows in order
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float sum = v[0][i];
#pragma unroll
            for (int p = 1; p < 8; ++p) sum += v[p][i];
            red[ty][tx * 8 + i] = sum;
        }
        __syncthreads();
        const int c = cb * kBlock8 + threadIdx.x;
        if (threadIdx.x < kBlock8 && c < a.C) {
            float sum = red[0][threadIdx.x];
#pragma unroll
            for (int g = 1; g < 16; ++g) sum += red[g][threadIdx.x];
            a.sums[mb * a.C + c] = sum;
        }
        __syncthreads();
    }
    if (infinite(largest<64>(v[0]))) drop_infinities<64>(v[0]);
    auto pack_row = [&](int p, float inv) {
        if (r0 + p >= a.M || c0 >= a.q_pitch) return;
        *reinterpret_cast<uint2*>(a.q + (r0 + p) * a.q_pitch + c0) =
            make_uint2(to_e4m3x4(v[p], inv), to_e4m3x4(v[p] + 4, inv));
    };
    float tile_inv = 0.f;
    if constexpr (TILE) {
        float top = largest<64>(v[0]);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        if ((threadIdx.x & 31) == 0) red[0][threadIdx.x >> 5] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kTileThreads / 32; ++w) top = fmaxf(top, red[0][w]);
        const int e = scale_exponent(top);
        tile_inv = exp2_int(-e);
        if (threadIdx.x == 0) {
            if (a.q != nullptr) a.scale[mb * a.CB + cb] = exp2_int(e);
            if (a.qt != nullptr) a.scale_t[(long long)cb * a.MB + mb] = exp2_int(e);
        }
        if (a.q != nullptr) {
#pragma unroll
            for (int p = 0; p < 8; ++p) pack_row(p, tile_inv);
        }
    } else if (a.q != nullptr) {
#pragma unroll
        for (int p = 0; p < 8; ++p) {
            float top = largest<8>(v[p]);
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            const int e = scale_exponent(top);
            if (tx == 0 && r0 + p < a.M) a.scale[(r0 + p) * a.CB + cb] = exp2_int(e);
            pack_row(p, exp2_int(-e));
        }
    }
    if (a.qt == nullptr) return;
    float inv[8];
    if constexpr (TILE) {
#pragma unroll
        for (int i = 0; i < 8; ++i) inv[i] = tile_inv;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float top = 0.f;
#pragma unroll
            for (int p = 0; p < 8; ++p) top = fmaxf(top, fabsf(v[p][i]));
            red[ty][tx * 8 + i] = top;
        }
        __syncthreads();
        if (threadIdx.x < kBlock8) {
            float top = red[0][threadIdx.x];
#pragma unroll
            for (int g = 1; g < 16; ++g) top = fmaxf(top, red[g][threadIdx.x]);
            const int e = scale_exponent(top), c = cb * kBlock8 + threadIdx.x;
            if (c < a.C) a.scale_t[mb * a.scale_t_pitch + c] = exp2_int(e);
            red[0][threadIdx.x] = exp2_int(-e);
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; ++i) inv[i] = red[0][tx * 8 + i];
    }
    // the transpose through shared memory: row c of `turned` is column c of the tile, its 8-byte pieces exchanged by
    // xor with (c / 8), so that the 16 threads of a group of rows write to all banks
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        float col[8];
#pragma unroll
        for (int p = 0; p < 8; ++p) col[p] = v[p][i];
        *reinterpret_cast<uint2*>(turned + (tx * 8 + i) * kBlock8 + ((ty ^ tx) << 3)) =
            make_uint2(to_e4m3x4(col, inv[i]), to_e4m3x4(col + 4, inv[i]));
    }
    __syncthreads();
    for (int i = threadIdx.x; i < kBlock8 * 8; i += kTileThreads) {
        const int c = i >> 3, piece = i & 7, turn = c >> 3;
        const long long at = mb * kBlock8 + piece * 16;
        if (cb * kBlock8 + c >= a.C || at >= a.qt_pitch) continue;  // (the pitch is a multiple of 16)
        uint4 w = *reinterpret_cast<const uint4*>(turned + c * kBlock8 + ((piece ^ (turn >> 1)) << 4));
        if (turn & 1) w = make_uint4(w.z, w.w, w.x, w.y);
        *reinterpret_cast<uint4*>(a.qt + (long long)(cb * kBlock8 + c) * a.qt_pitch + at) = w;
    }
}

// out[c] = the partial rows [parts][C] added in order: each thread adds every kColumnRows-th part of one column, then
// the threads of a column are added in order.
constexpr int kColumnCols = 32, kColumnRows = 16;
template <typename T, typename A>
__global__ void __launch_bounds__(kColumnCols* kColumnRows)
    column_sum_kernel(const A* __restrict__ partial, T* out, long long parts, int C) {
    __shared__ A sums[kColumnRows][kColumnCols];
    const int tx = threadIdx.x % kColumnCols, ty = threadIdx.x / kColumnCols;
    const int col = blockIdx.x * kColumnCols + tx;
    grid_dependency_wait();
    launch_dependents();
    A sum = 0;
    if (col < C) {
#pragma unroll 4
        for (long long p = ty; p < parts; p += kColumnRows) sum += partial[p * C + col];
    }
    sums[ty][tx] = sum;
    __syncthreads();
    if (ty == 0 && col < C) {
#pragma unroll
        for (int i = 1; i < kColumnRows; ++i) sum += sums[i][tx];
        out[col] = from_acc<T>(sum);
    }
}

// ---- back -------------------------------------------------------------------------------------------------------

struct BackArgs {
    const uint8_t* q;    // [M, pitch]
    const float* scale;  // [M, KB], or [MB, KB] (tiles)
    void* out;           // [M, K]
    long long M, pitch;
    int K, KB, tiles;
};

// A thread takes 8 neighbouring values of a row. WIDE: pitch and K multiples of 8, q 8-byte aligned, out 16-byte.
template <typename T, bool WIDE>
__global__ void __launch_bounds__(256) fp8_back_kernel(const BackArgs a) {
    const int per_row = (a.K + 7) / 8;
    const long long total = a.M * per_row, step = (long long)gridDim.x * 256;
    grid_dependency_wait();
    launch_dependents();
    for (long long t = (long long)blockIdx.x * 256 + threadIdx.x; t < total; t += step) {
        const long long row = total <= 0xFFFFFFFFLL ? uint32_t(t) / uint32_t(per_row) : t / per_row;
        const int c = int(t - row * per_row) * 8;
        const float s = a.scale[(a.tiles ? row / kBlock8 : row) * a.KB + c / kBlock8];
        const uint8_t* src = a.q + row * a.pitch + c;
        T* dst = static_cast<T*>(a.out) + row * a.K + c;
        float v[8];
        if constexpr (WIDE) {
            const uint2 w = __ldg(reinterpret_cast<const uint2*>(src));
            const uint32_t h[4] = {w.x, w.x >> 16, w.y, w.y >> 16};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 f = from_e4m3x2(h[i]);
                v[2 * i] = f.x * s;
                v[2 * i + 1] = f.y * s;
            }
#pragma unroll
            for (int i = 0; i < 8; i += Elem<T>::kVec) store16<T>(dst + i, v + i);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (c + i < a.K) dst[i] = from_acc<T>(from_e4m3(src[i]) * s);
        }
    }
}

// The same where rows follow one another without gaps, K is a multiple of 128, q 16-byte and out 32-byte aligned: a
// thread takes 16 neighbouring values of the blocks that follow one another (1 x 128).
template <typename T>
__global__ void __launch_bounds__(256) fp8_flat_back_kernel(const BackArgs a) {
    const long long total = a.M * (a.K / 16), step = (long long)gridDim.x * 256;
    grid_dependency_wait();
    launch_dependents();
    uint4 raw = make_uint4(0, 0, 0, 0);
    float s = 0.f;
    auto fetch = [&](long long i) {
        if (i < total) {
            raw = __ldg(reinterpret_cast<const uint4*>(a.q + i * 16));
            s = __ldg(a.scale + (i >> 3));
        }
    };
    long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    fetch(i);
    for (; i < total; i += step) {
        const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
        float v[16];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const float2 f = from_e4m3x2(w[k / 2] >> 16 * (k % 2));
            v[2 * k] = f.x * s;
            v[2 * k + 1] = f.y * s;
        }
        fetch(i + step);
        T* dst = static_cast<T*>(a.out) + i * 16;
        uint4 o[16 * sizeof(T) / 16];
#pragma unroll
        for (int k = 0; k < int(sizeof(T)); ++k) store16<T>(reinterpret_cast<T*>(&o[k]), v + k * Elem<T>::kVec);
#pragma unroll
        for (int k = 0; k < int(sizeof(T)); k += 2)
            asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                         ::"l"(reinterpret_cast<char*>(dst) + k * 16), "r"(o[k].x), "r"(o[k].y), "r"(o[k].z),
                           "r"(o[k].w), "r"(o[k + 1].x), "r"(o[k + 1].y), "r"(o[k + 1].z), "r"(o[k + 1].w)
                         : "memory");
    }
}

}  // namespace td
