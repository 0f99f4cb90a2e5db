// td_fp8_simt.cuh -- the product of two e4m3 operands on CUDA cores, and the end of a product.
//
//   out[m, n] = act(sum_kb sa[m, kb] sb[n, kb] sum_{k in block kb} a[m, k] b[n, k] + bias[n])
//
// fp8_product_simt_kernel takes any sizes and alignments; the tensor-core kernels (td_fp8_tc.cuh, td_fp8_few.cuh) are
// the ones that calls run by default, this one is what the CUDA-core policy runs. A block's 128 products are summed in
// float32 first and scaled once. fp8_finish_kernel adds a split product's float32 parts in order and ends it.
#pragma once

#include "td_fp8.cuh"

namespace td {

enum Activation8 : int { kActNone = 0, kActRelu = 1, kActGelu = 2, kActSilu = 3 };

// 1 / x for 1 <= x, to a step of float32.
__device__ __forceinline__ float reciprocal(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// GELU, v Phi(v), by the upper tail h = 1 - Phi(|v|) = exp(-v^2 / 2) R, which keeps the digits of a lower tail that
// 1 + erf loses (a tenth of the value at -5, all of it below -5.6). R = erfcx(|v| / sqrt 2) / 2 is smooth, in
// t = 1 / (1 + 0.35 |v|) a polynomial times t, fitted to |v| < 15 (beyond, the tail is less than float32 holds) for the
// least relative error, 3e-8. 177784 x 256 x 1024 with 8-bit results: 306 us, by erfcf 768, by 1 + erff 336.
__device__ __forceinline__ float gelu(float v) {
    const float a = fabsf(v), t = reciprocal(fmaf(0.35f, a, 1.f));
    float p = -0.029163928f;
    p = fmaf(p, t, 0.14406084f);
    p = fmaf(p, t, -0.25590193f);
    p = fmaf(p, t, 0.15939298f);
    p = fmaf(p, t, -0.023263887f);
    p = fmaf(p, t, 0.10557482f);
    p = fmaf(p, t, 0.11981549f);
    p = fmaf(p, t, 0.13986434f);
    p = fmaf(p, t, 0.13962126f);
    const float h = exp2f(v * v * -0.72134752f) * (p * t);  // -log2(e) / 2
    return v * (v < 0.f ? h : 1.f - h);
}

// SiLU, v / (1 + exp(-v)), with the exponential at most 1, so that neither it nor the denominator leaves the range. The
// same call 226 us; 206 with __expf(-v) and __fdividef, which is zero below -87.
__device__ __forceinline__ float silu(float v) {
    const float e = expf(-fabsf(v));
    return (v < 0.f ? v * e : v) * reciprocal(1.f + e);
}

__device__ __forceinline__ float activate(float v, int act) {
    if (act == kActRelu) {  // a NaN stays one
        float d;
        asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(d) : "f"(v));
        return d;
    }
    if (act == kActGelu) return gelu(v);
    if (act == kActSilu) return silu(v);
    return v;
}

// One operand [rows, K] of a product: rows along K, `pitch` bytes apart, or (blocks) [K / 128, rows, 128], laid out a
// block of K at a time. Value k of row r is at q[r * pitch + k / 128 * block + k % 128] in both.
struct Operand8 {
    const uint8_t* q;
    const float* scale;  // of row r and block kb: scale[r / rows_per_scale * scale_row + kb * scale_k]
    long long pitch, scale_row, scale_k;
    int rows_per_scale;  // 1 or 128
    bool blocks;
    long long block;
};

// How a product ends: bias, activation, and the type it is written in.
struct End8 {
    const void* bias;  // [N] of `bias_dtype`, or null
    void* out;         // [M, N] dense; e4m3: [M, pitch] in 1 x 128 blocks, zeros behind N
    float* scale;      // e4m3: [M, ceil(N / 128)]
    int bias_dtype, act, pitch;
};

__device__ __forceinline__ float bias_at(const End8& e, int n) {
    if (e.bias == nullptr) return 0.f;
    switch (e.bias_dtype) {
        case 0: return __ldg(static_cast<const float*>(e.bias) + n);
        case 1: return to_acc(static_cast<const __half*>(e.bias)[n]);
        default: return to_acc(static_cast<const __nv_bfloat16*>(e.bias)[n]);
    }
}

constexpr int kSimtRows8 = 64, kSimtStep8 = 32, kSimtThreads8 = 256;

// Tile blockIdx.x of 64 x 128 (columns fastest), 4 rows x 8 columns a thread (columns tx, tx + 16, ..); 32 values of K
// at a time.
template <typename T>
__global__ void __launch_bounds__(kSimtThreads8)
    fp8_product_simt_kernel(const Operand8 a, const Operand8 b, const End8 end, long long M, int N, int K) {
    __shared__ float sa[kSimtStep8][kSimtRows8 + 1], sb[kSimtStep8][kBlock8 + 1];
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    const int n_tiles = (N + kBlock8 - 1) / kBlock8, nb = int(blockIdx.x % unsigned(n_tiles)), n0 = nb * kBlock8;
    const long long m0 = (long long)(blockIdx.x / unsigned(n_tiles)) * kSimtRows8;
    grid_dependency_wait();
    launch_dependents();
    float acc[4][8] = {};
    for (int k0 = 0; k0 < K; k0 += kBlock8) {
        float part[4][8] = {};
        for (int k1 = k0; k1 < k0 + kBlock8 && k1 < K; k1 += kSimtStep8) {
            for (int i = threadIdx.x; i < (kSimtRows8 + kBlock8) * kSimtStep8; i += kSimtThreads8) {
                const int r = i / kSimtStep8, c = i % kSimtStep8, k = k1 + c, n = n0 + r - kSimtRows8;
                const int kb = k / kBlock8, at = k % kBlock8;
                if (r < kSimtRows8)
                    sa[c][r] = m0 + r < M && k < K ? from_e4m3(a.q[(m0 + r) * a.pitch + kb * a.block + at]) : 0.f;
                else
                    sb[c][r - kSimtRows8] = n < N && k < K ? from_e4m3(b.q[n * b.pitch + kb * b.block + at]) : 0.f;
            }
            __syncthreads();
#pragma unroll 4
            for (int c = 0; c < kSimtStep8; ++c) {
                float x[4], y[8];
#pragma unroll
                for (int i = 0; i < 4; ++i) x[i] = sa[c][ty * 4 + i];
#pragma unroll
                for (int j = 0; j < 8; ++j) y[j] = sb[c][tx + 16 * j];
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 8; ++j) part[i][j] = fmaf(x[i], y[j], part[i][j]);
            }
            __syncthreads();
        }
        const long long kb = k0 / kBlock8;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const long long m = m0 + ty * 4 + i;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int n = n0 + tx + 16 * j;
                if (m < M && n < N)
                    acc[i][j] = fmaf(part[i][j], a.scale[m / a.rows_per_scale * a.scale_row + kb * a.scale_k] *
                                                     b.scale[n / b.rows_per_scale * b.scale_row + kb * b.scale_k],
                                     acc[i][j]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const long long m = m0 + ty * 4 + i;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int n = n0 + tx + 16 * j;
            acc[i][j] = n < N ? activate(acc[i][j] + bias_at(end, n), end.act) : 0.f;
        }
        if constexpr (sizeof(T) == 1) {
            drop_infinities<8>(acc[i]);
            float top = largest<8>(acc[i]);
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            const int e = scale_exponent(top);
            if (m >= M) continue;
            if (tx == 0) end.scale[m * n_tiles + nb] = exp2_int(e);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int n = n0 + tx + 16 * j;
                if (n < end.pitch)
                    static_cast<uint8_t*>(end.out)[m * end.pitch + n] =
                        uint8_t(to_e4m3x2(acc[i][j], 0.f, exp2_int(-e)));
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int n = n0 + tx + 16 * j;
                if (m < M && n < N) static_cast<T*>(end.out)[m * N + n] = from_acc<T>(acc[i][j]);
            }
        }
    }
}

// out = end(sum of the parts [parts][M][N], in order); T = E4m3: in 8 bits. A warp takes 128 columns of a row, four
// neighbouring ones a lane.
template <typename T>
__global__ void __launch_bounds__(256)
    fp8_finish_kernel(const float* __restrict__ partial, int parts, const End8 end, long long M, int N) {
    const int lane = threadIdx.x & 31, blocks = (N + kBlock8 - 1) / kBlock8;
    const long long tasks = M * blocks, step = (long long)gridDim.x * 8, size = M * N;
    const bool wide = N % 4 == 0;  // (the parts are 16-byte aligned)
    grid_dependency_wait();
    launch_dependents();
    for (long long t = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); t < tasks; t += step) {
        const long long m = tasks <= 0xFFFFFFFFLL ? uint32_t(t) / uint32_t(blocks) : t / blocks;
        const int nb = int(t - m * blocks), n = nb * kBlock8 + lane * 4;
        float v[4] = {0.f, 0.f, 0.f, 0.f};
        const float* src = partial + m * N + n;
        for (int p = 0; p < parts; ++p, src += size) {
            if (wide) {
                if (n < N) {
                    const float4 f = *reinterpret_cast<const float4*>(src);
                    v[0] += f.x; v[1] += f.y; v[2] += f.z; v[3] += f.w;
                }
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (n + i < N) v[i] += src[i];
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = n + i < N ? activate(v[i] + bias_at(end, n + i), end.act) : 0.f;
        if constexpr (sizeof(T) == 1) {
            drop_infinities<4>(v);
            float top = largest<4>(v);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            const int e = scale_exponent(top);
            if (lane == 0) end.scale[m * blocks + nb] = exp2_int(e);
            if (n < end.pitch)
                *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(end.out) + m * end.pitch + n) =
                    to_e4m3x4(v, exp2_int(-e));
        } else {
            T* dst = static_cast<T*>(end.out) + m * N + n;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (n + i < N) dst[i] = from_acc<T>(v[i]);
        }
    }
}

// ---- rows to 16-byte boundaries -----------------------------------------------------------------------------------

struct PitchArgs {
    const uint8_t* from;  // [M, from_pitch], anywhere
    uint8_t* to;          // [M, to_pitch], 16-byte aligned, the pitch a multiple of 16; zeros behind K
    long long M, from_pitch, to_pitch;
    int K;
};
// A thread takes 16 bytes of a row.
__global__ void __launch_bounds__(256) fp8_pitch_kernel(const PitchArgs a) {
    const int per_row = int(a.to_pitch / 16);
    const long long total = a.M * per_row, step = (long long)gridDim.x * 256;
    grid_dependency_wait();
    launch_dependents();
    for (long long t = (long long)blockIdx.x * 256 + threadIdx.x; t < total; t += step) {
        const long long row = t / per_row;
        const int c = int(t - row * per_row) * 16;
        const uint8_t* src = a.from + row * a.from_pitch + c;
        uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (c + i < a.K) w[i / 4] |= uint32_t(__ldg(src + i)) << 8 * (i % 4);
        *reinterpret_cast<uint4*>(a.to + row * a.to_pitch + c) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

}  // namespace td
