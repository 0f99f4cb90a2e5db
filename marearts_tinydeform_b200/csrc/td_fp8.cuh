// td_fp8.cuh -- 8-bit floating point (e4m3) in blocks of 128: the scales, and the kernels that go from wider types to
// 8 bits and back.
//
//   a block's m = its largest finite magnitude; e = the smallest integer >= -126 with m 2^-e <= 448; scale = 2^e
//   q = e4m3(v 2^-e), to nearest, ties to even; an infinity or NaN becomes NaN (e4m3 has no infinity)
//
// Scales are powers of two: a product with one is exact, so a value is rounded once, a quantised value is exact in
// float32 (and from 2^-126 on in bfloat16), and values kept in 8 bits are quantised again along the other axis without
// a second rounding (but for those below the other block's smallest step). Floating-point codes lose nothing by it:
// their relative step is the same anywhere in the range. Blocks are 1 x 128 (activations: along the contraction),
// 128 x 1 (the same tensors when rows are contracted, as in the weight's gradient) or 128 x 128 (weights, whose blocks
// stay blocks when transposed).
//
// Rows alone (1 x 128) are bound by memory: fp8_flat_kernel, where blocks follow one another (K a multiple of 128),
// takes 32 bytes a thread and runs at the copy rate (177784 x 1024 bfloat16 88 us, 6.2 TB/s; 177784 x 256 22.8; with
// one 16-byte vector a thread and a division a task 143), fp8_rows_kernel any other rows (8800 x 515 float32 8 us).
// fp8_tile_kernel takes 128 x 128 values into registers, once, for any of: the 1 x 128 form, the 128 x 1 form
// transposed, the 128 x 128 form or its transpose, and column sums. It is bound by instructions (76 % of the issue
// slots): what a training backward lays out at 67200 x 1024 and 67200 x 256, 309 MB, takes 76 us (4.1 TB/s).
// Widening each value once for all three forms gave 1 % of the whole backward and cost its other calls 6 to 10 %.
#pragma once

#include <cuda_fp8.h>

#include <type_traits>

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

enum TileKind : int { kTileBlocks = 0, kTileWhole = 1, kTileFrom8 = 2 };

struct TileArgs {
    const void* x;           // [M, C], rows `ld` elements apart: floating, or (kTileFrom8) e4m3 with
    const float* x_scale;    //   its scales [M, CB] (1 x 128)
    long long ld;
    uint8_t* q;              // or null: [M, q_pitch], in 1 x 128 blocks, or 128 x 128 (kTileWhole)
    float* scale;            //   [M, CB], or [MB, CB]
    uint8_t* qt;             // or null: the transpose, [C, qt_pitch] in blocks of 128 x 128 (kTileWhole), or
                             //   [MB, C, 128], a block of 128 rows of x a column: a tile is 16 KB that follow one another
    float* scale_t;          //   [MB, scale_t_pitch] (one for each column), or [CB, MB]
    float* sums;             // or null: [MB, C] sums over a tile's rows
    long long M, q_pitch, qt_pitch, scale_t_pitch;
    int C, CB, MB;
    int wide;                // rows of x start on 16-byte boundaries (8-byte ones for e4m3), C a multiple of 8
    long long end;           // of the launch's tiles, this job's and those before it
};

constexpr int kTileThreads = 256, kTileJobs = 3;
struct TileJobs {  // independent jobs of one launch, each kind's in its place (their arguments are then constants)
    TileArgs job[kTileJobs];
};

// A thread's 8 rows x 8 columns of a tile, as they came from memory: fewer registers than as float32, and so more
// tiles at once on an SM. pair(p, c): columns 2c and 2c + 1 of row p.
template <typename T>
struct Patch {  // 16-bit types
    uint4 w[8];
    static __device__ __forceinline__ uint32_t word(const uint4& v, int c) {
        return c == 0 ? v.x : c == 1 ? v.y : c == 2 ? v.z : v.w;
    }
    __device__ __forceinline__ void clear(int p) { w[p] = make_uint4(0, 0, 0, 0); }
    __device__ __forceinline__ void load(int p, const T* src, int left, bool wide) {
        if (wide) {
            w[p] = __ldg(reinterpret_cast<const uint4*>(src));
        } else {
            struct __align__(16) Eight {
                T v[8];
            } one;
            static_assert(alignof(Eight) >= alignof(uint4), "one word of eight values");
#pragma unroll
            for (int i = 0; i < 8; ++i) one.v[i] = i < left ? src[i] : from_acc<T>(0.f);
            w[p] = *reinterpret_cast<const uint4*>(one.v);
        }
    }
    __device__ __forceinline__ float2 pair(int p, int c) const {
        return both(word(w[p], c));
    }
    // Columns 2c and 2c + 1 of row p times a pair of scales, as e4m3. bfloat16 has the exponents for the product, which
    // is exact but for what e4m3 rounds to zero anyway; float16 goes through float32.
    static constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
    using Scales = typename std::conditional<kBf16, __nv_bfloat162, float2>::type;
    static __device__ __forceinline__ Scales scales(float x, float y) {
        if constexpr (kBf16) return __floats2bfloat162_rn(x, y);
        else return make_float2(x, y);
    }
    __device__ __forceinline__ uint32_t e4m3x2(int p, int c, const Scales& f) const {
        const uint32_t two = word(w[p], c);
        float2 v;
        if constexpr (kBf16) {
            v = __bfloat1622float2(__hmul2(*reinterpret_cast<const __nv_bfloat162*>(&two), f));
        } else {
            v = both(two);
            v.x *= f.x;
            v.y *= f.y;
        }
        return __nv_cvt_float2_to_fp8x2(v, __NV_SATFINITE, __NV_E4M3);
    }
    // Maxima of packed magnitudes, of which a NaN counts for nothing.
    static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
        using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
        const T2 m = __hmax2(*reinterpret_cast<const T2*>(&a), *reinterpret_cast<const T2*>(&b));
        return *reinterpret_cast<const uint32_t*>(&m);
    }
    static __device__ __forceinline__ float2 both(uint32_t two) {
        if constexpr (std::is_same<T, __half>::value) return __half22float2(*reinterpret_cast<const __half2*>(&two));
        else return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&two));
    }
    __device__ __forceinline__ uint32_t row_max2(int p) const {
        uint32_t m = 0;
#pragma unroll
        for (int c = 0; c < 4; ++c) m = max2(m, word(w[p], c) & 0x7FFF7FFFu);
        return m;
    }
    // Largest magnitudes of rows 2h and 2h + 1 over the tile's columns (two rows to a shuffle).
    __device__ __forceinline__ float2 row_tops(int h) const {
        const uint32_t a = row_max2(2 * h), b = row_max2(2 * h + 1);
        uint32_t m = max2(__byte_perm(a, b, 0x5410), __byte_perm(a, b, 0x7632));
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) m = max2(m, __shfl_xor_sync(0xffffffffu, m, o));
        return both(m);
    }
    // .. of columns 2c and 2c + 1 over the thread's rows
    __device__ __forceinline__ float2 column_tops(int c) const {
        uint32_t m = 0;
#pragma unroll
        for (int p = 0; p < 8; ++p) m = max2(m, word(w[p], c) & 0x7FFF7FFFu);
        return both(m);
    }
    // infinities to NaN (0x7FFF is one in both types)
    __device__ __forceinline__ void drop_infinite() {
        constexpr uint32_t kInf = std::is_same<T, __half>::value ? 0x7C00u : 0x7F80u;
        uint32_t most = 0;
#pragma unroll
        for (int p = 0; p < 8; ++p) most = max2(most, row_max2(p));
        if ((most & 0xFFFFu) < kInf && most >> 16 < kInf) return;
#pragma unroll
        for (int p = 0; p < 8; ++p) {
            uint32_t* v = reinterpret_cast<uint32_t*>(&w[p]);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                if ((v[c] & 0x7FFFu) == kInf) v[c] |= 0x7FFFu;
                if ((v[c] >> 16 & 0x7FFFu) == kInf) v[c] |= 0x7FFF0000u;
            }
        }
    }
};
// The same conversion and maxima through pair().
struct PatchScales {
    using Scales = float2;
    static __device__ __forceinline__ float2 scales(float x, float y) { return make_float2(x, y); }
};
template <typename P>
__device__ __forceinline__ uint32_t patch_e4m3x2(const P& v, int p, int c, float2 f) {
    const float2 two = v.pair(p, c);
    return __nv_cvt_float2_to_fp8x2(make_float2(two.x * f.x, two.y * f.y), __NV_SATFINITE, __NV_E4M3);
}
template <typename P>
__device__ __forceinline__ float2 patch_row_tops(const P& v, int h) {
    float top[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        top[r] = 0.f;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const float2 f = v.pair(2 * h + r, c);
            top[r] = fmaxf(top[r], fmaxf(fabsf(f.x), fabsf(f.y)));
        }
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], o));
    }
    return make_float2(top[0], top[1]);
}
template <typename P>
__device__ __forceinline__ float2 patch_column_tops(const P& v, int c) {
    float2 top = make_float2(0.f, 0.f);
#pragma unroll
    for (int p = 0; p < 8; ++p) {
        const float2 f = v.pair(p, c);
        top.x = fmaxf(top.x, fabsf(f.x));
        top.y = fmaxf(top.y, fabsf(f.y));
    }
    return top;
}
template <>
struct Patch<float> : PatchScales {
    float v[8][8];
    __device__ __forceinline__ void clear(int p) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[p][i] = 0.f;
    }
    __device__ __forceinline__ void load(int p, const float* src, int left, bool wide) {
        if (wide) {
            load16<float>(src, v[p]);
            load16<float>(src + 4, v[p] + 4);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[p][i] = i < left ? src[i] : 0.f;
        }
    }
    __device__ __forceinline__ float2 pair(int p, int c) const { return make_float2(v[p][2 * c], v[p][2 * c + 1]); }
    __device__ __forceinline__ uint32_t e4m3x2(int p, int c, float2 f) const { return patch_e4m3x2(*this, p, c, f); }
    __device__ __forceinline__ float2 row_tops(int h) const { return patch_row_tops(*this, h); }
    __device__ __forceinline__ float2 column_tops(int c) const { return patch_column_tops(*this, c); }
    __device__ __forceinline__ void drop_infinite() {
        float top = 0.f;
#pragma unroll
        for (int p = 0; p < 8; ++p) top = fmaxf(top, largest<8>(v[p]));
        if (!infinite(top)) return;
#pragma unroll
        for (int p = 0; p < 8; ++p) drop_infinities<8>(v[p]);
    }
};
template <>
struct Patch<E4m3> : PatchScales {
    uint2 w[8];
    float s[8];
    __device__ __forceinline__ void clear(int p) {
        w[p] = make_uint2(0, 0);
        s[p] = 0.f;
    }
    __device__ __forceinline__ void load(int p, const E4m3* src, int left, bool wide) {
        if (wide) {
            w[p] = __ldg(reinterpret_cast<const uint2*>(src));
        } else {
            uint32_t two[2] = {0, 0};
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < left) two[i / 4] |= uint32_t(src[i].bits) << 8 * (i % 4);
            w[p] = make_uint2(two[0], two[1]);
        }
    }
    __device__ __forceinline__ float2 pair(int p, int c) const {
        const uint32_t two = c < 2 ? w[p].x : w[p].y;
        const float2 f = from_e4m3x2(two >> 16 * (c % 2));
        return make_float2(f.x * s[p], f.y * s[p]);
    }
    __device__ __forceinline__ uint32_t e4m3x2(int p, int c, float2 f) const { return patch_e4m3x2(*this, p, c, f); }
    __device__ __forceinline__ float2 row_tops(int h) const { return patch_row_tops(*this, h); }
    __device__ __forceinline__ float2 column_tops(int c) const { return patch_column_tops(*this, c); }
    __device__ __forceinline__ void drop_infinite() {}
};

// A thread holds rows 8 ty .. 8 ty + 7 of the tile and columns 8 tx .. 8 tx + 7 (tx < 16).
template <typename T, bool WHOLE>
__device__ __forceinline__ void tile_job(const TileArgs& a, long long tile, float (&red)[16][kBlock8],
                                         uint8_t* turned) {
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const long long mb = tile / a.CB;
    const int cb = int(tile - mb * a.CB);
    const long long r0 = mb * kBlock8 + ty * 8;
    const int c0 = cb * kBlock8 + tx * 8;
    Patch<T> v;
#pragma unroll
    for (int p = 0; p < 8; ++p) {
        v.clear(p);
        if (r0 + p < a.M && c0 < a.C) {
            v.load(p, static_cast<const T*>(a.x) + (r0 + p) * a.ld + c0, a.C - c0, a.wide);
            if constexpr (sizeof(T) == 1) v.s[p] = __ldg(a.x_scale + (r0 + p) * a.CB + cb);
        }
    }
    if (a.sums != nullptr) {  // a thread's rows in order, then the 16 groups of rows in order
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            float2 sum = v.pair(0, c);
#pragma unroll
            for (int p = 1; p < 8; ++p) {
                const float2 f = v.pair(p, c);
                sum.x += f.x;
                sum.y += f.y;
            }
            *reinterpret_cast<float2*>(&red[ty][tx * 8 + 2 * c]) = sum;
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
    v.drop_infinite();
    auto pack_row = [&](int p, float inv) {
        if (r0 + p >= a.M || c0 >= a.q_pitch) return;
        uint32_t w[4];
        const auto f = v.scales(inv, inv);
#pragma unroll
        for (int c = 0; c < 4; ++c) w[c] = v.e4m3x2(p, c, f);
        *reinterpret_cast<uint2*>(a.q + (r0 + p) * a.q_pitch + c0) = make_uint2(w[0] | w[1] << 16, w[2] | w[3] << 16);
    };
    float tile_inv = 0.f;
    if constexpr (WHOLE) {
        float top = 0.f;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const float2 f = v.column_tops(c);
            top = fmaxf(top, fmaxf(f.x, f.y));
        }
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
        for (int h = 0; h < 4; ++h) {
            const float2 top = v.row_tops(h);
            const int e0 = scale_exponent(top.x), e1 = scale_exponent(top.y);
            if (tx < 2 && r0 + 2 * h + tx < a.M) a.scale[(r0 + 2 * h + tx) * a.CB + cb] = exp2_int(tx == 0 ? e0 : e1);
            pack_row(2 * h, exp2_int(-e0));
            pack_row(2 * h + 1, exp2_int(-e1));
        }
    }
    if (a.qt == nullptr) return;
    if constexpr (!WHOLE) {
#pragma unroll
        for (int c = 0; c < 4; ++c) *reinterpret_cast<float2*>(&red[ty][tx * 8 + 2 * c]) = v.column_tops(c);
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
    }
    // the transpose through shared memory: row c of `turned` is column c of the tile, its 8-byte pieces exchanged by
    // xor with (c / 8), so that the 16 threads of a group of rows write to all banks
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        float2 inv = make_float2(tile_inv, tile_inv);
        if constexpr (!WHOLE) inv = *reinterpret_cast<const float2*>(&red[0][tx * 8 + 2 * c]);
        uint32_t two[8];  // of each row: column 2c in the low byte, 2c + 1 above it
        const auto f = v.scales(inv.x, inv.y);
#pragma unroll
        for (int p = 0; p < 8; ++p) two[p] = v.e4m3x2(p, c, f);
        uint32_t lo[2], hi[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t a01 = __byte_perm(two[4 * h], two[4 * h + 1], 0x5140);  // bytes: c of 0, 1; c + 1 of 0, 1
            const uint32_t a23 = __byte_perm(two[4 * h + 2], two[4 * h + 3], 0x5140);
            lo[h] = __byte_perm(a01, a23, 0x5410);
            hi[h] = __byte_perm(a01, a23, 0x7632);
        }
        uint8_t* dst = turned + (tx * 8 + 2 * c) * kBlock8 + ((ty ^ tx) << 3);
        *reinterpret_cast<uint2*>(dst) = make_uint2(lo[0], lo[1]);
        *reinterpret_cast<uint2*>(dst + kBlock8) = make_uint2(hi[0], hi[1]);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < kBlock8 * 8; i += kTileThreads) {
        const int c = i >> 3, piece = i & 7, turn = c >> 3;
        const long long col = cb * kBlock8 + c, at = mb * kBlock8 + piece * 16;
        if (col >= a.C || (WHOLE && at >= a.qt_pitch)) continue;  // (the pitch is a multiple of 16)
        uint4 w = *reinterpret_cast<const uint4*>(turned + c * kBlock8 + ((piece ^ (turn >> 1)) << 4));
        if (turn & 1) w = make_uint4(w.z, w.w, w.x, w.y);
        uint8_t* to = WHOLE ? a.qt + col * a.qt_pitch + at : a.qt + (mb * a.C + col) * kBlock8 + piece * 16;
        *reinterpret_cast<uint4*>(to) = w;
    }
}

// Tile blockIdx.x of the jobs' tiles, one job's behind the other's: what a training pass lays out is one launch.
template <typename T>
__global__ void __launch_bounds__(kTileThreads, sizeof(T) == 4 ? 2 : 4)
    fp8_tile_kernel(const __grid_constant__ TileJobs jobs) {
    __shared__ __align__(16) float red[16][kBlock8];
    __shared__ __align__(16) uint8_t turned[kBlock8 * kBlock8];
    grid_dependency_wait();
    launch_dependents();
    const long long tile = blockIdx.x;
    if (tile < jobs.job[kTileBlocks].end)
        tile_job<T, false>(jobs.job[kTileBlocks], tile, red, turned);
    else if (tile < jobs.job[kTileWhole].end)
        tile_job<T, true>(jobs.job[kTileWhole], tile - jobs.job[kTileBlocks].end, red, turned);
    else
        tile_job<E4m3, false>(jobs.job[kTileFrom8], tile - jobs.job[kTileWhole].end, red, turned);
}

// out[c] = the partial rows [parts][C] added in order, in float64 (parts may cancel): each thread adds every
// kColumnRows-th part of one column, then the threads of a column are added in order. (The bias's gradient over 67200
// rows, with the pass over the gradient: 29.6 us at 1024 columns and 9.4 at 256; 0.2 us more than with float32 sums,
// about 2 less than with 16 rows of threads.)
constexpr int kColumnCols = 32, kColumnRows = 32;
template <typename T, typename A>
__global__ void __launch_bounds__(kColumnCols* kColumnRows)
    column_sum_kernel(const A* __restrict__ partial, T* out, long long parts, int C) {
    __shared__ double sums[kColumnRows][kColumnCols];
    const int tx = threadIdx.x % kColumnCols, ty = threadIdx.x / kColumnCols;
    const int col = blockIdx.x * kColumnCols + tx;
    grid_dependency_wait();
    launch_dependents();
    double sum = 0;
    if (col < C) {
#pragma unroll 8
        for (long long p = ty; p < parts; p += kColumnRows) sum += double(partial[p * C + col]);
    }
    sums[ty][tx] = sum;
    __syncthreads();
    if (ty == 0 && col < C) {
#pragma unroll
        for (int i = 1; i < kColumnRows; ++i) sum += sums[i][tx];
        out[col] = from_acc<T>(A(sum));
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
