// td_fp8_few.cuh -- the product of a few rows (up to 16, a serving batch's single tokens) with an e4m3 weight.
//
//   out[m, n] = act(sum_kb sa[m, kb] sb[n / 128, kb] sum_{k in block kb} a[m, k] b[n, k] + bias[n])
//
// Bound by reading the weight, so its rows are spread over the whole GPU: a CTA takes 16 of them, and its 8 warps every
// eighth block of K each, with three blocks' bytes under way while one is multiplied. The tensor cores take e4m3
// fragments of m16n8k32 (16 weight rows by 8 of x): a thread's 16 bytes of a row are two K steps' worth, in an order of
// K that both operands share, so fragments are what memory holds. (As float16 they would be converted, 48 numbers a
// thread and block: 20.8 us for the 16.2 below.) A block's sums start from zero and enter float32 registers times its
// scales; the warps' sums are added in order.
//
// Up to four short rows of x may be wider than 8 bits (X): each warp then rounds its own blocks instead of another
// launch before this one. An 8-bit result's blocks of 128 columns are the work of a cluster of 8 CTAs, which exchange
// their rows' largest magnitudes. One row, the weight from memory: 4096 x 4096 5.6 us (3.0 TB/s), 8192 x 8192 16.2
// (4.1 TB/s); a weight in the L2, 1024 x 256, 1.7 us. 16 rows, 4096 x 4096: 9.1.
#pragma once

#include "td_fp8_simt.cuh"

namespace td {

constexpr int kFewThreads = 256, kFewWarps = 8, kFewRows = 16;  // rows of the weight
constexpr int kFewMost = 16, kFewWide = 4;  // rows of x: in 8 bits, and wider

struct FewArgs {
    const void* x;         // e4m3, rows x_pitch apart (16-byte aligned), or wider and dense
    const float* x_scale;  // [M, KB] (e4m3)
    const uint8_t* w;      // rows w_pitch apart (16-byte aligned)
    const float* w_scale;  // [NB, KB]
    End8 end;
    long long x_pitch, w_pitch;
    int M, N, K, KB, x_wide;  // x_wide: four values of a wider x are one aligned word
};

__device__ __forceinline__ void mma_16832(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                          uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The 16 bytes at p to shared memory, or those of them before `left` with zeros behind.
__device__ __forceinline__ void copy_bytes(uint32_t dst, const void* p, int left) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(p), "r"(min(max(left, 0), 16))
                 : "memory");
}

// Pieces of 16 bytes a thread has of a block: 4 of the weight, 2 of each 8 rows of an 8-bit x.
template <typename X, int TILES>
constexpr int few_pieces() {
    return 4 + (sizeof(X) == 1 ? 2 * TILES : 0);
}
constexpr int kFewStages = 4;
template <typename X, int TILES>
constexpr size_t few_smem() {
    return size_t(kFewStages) * few_pieces<X, TILES>() * kFewThreads * 16;
}

template <typename X, typename T, int TILES>  // TILES of 8 rows of x
__device__ __forceinline__ void few_rows(const FewArgs& a) {
    constexpr bool kFrom8 = sizeof(X) == 1, kTo8 = sizeof(T) == 1;
    constexpr int kWideRows = kFrom8 ? 1 : kFewWide;
    __shared__ float sums[kFewWarps][kFewRows][8 * TILES + 1];
    __shared__ __align__(16) float tops[8 * TILES];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int n0 = blockIdx.x * kFewRows;
    const int blocks = n0 < a.N && warp < a.KB ? (a.KB - 1 - warp) / kFewWarps + 1 : 0;  // this warp's
    const uint8_t* w_row[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) w_row[i] = a.w + (long long)min(n0 + g + 8 * i, a.N - 1) * a.w_pitch;
    const float* w_scale = a.w_scale + (long long)(min(n0, a.N - 1) / kBlock8) * a.KB;
    // Bytes go through shared memory, three blocks ahead: each thread copies its own pieces there (weight rows g and
    // g + 8, pieces t and t + 4 of the block's 8; row g of an 8-bit x likewise) and reads them back, so no barrier is
    // needed.
    extern __shared__ __align__(16) unsigned char smem[];
    constexpr int P = few_pieces<X, TILES>();
    auto place = [&](int stage, int piece) {
        return smem + ((stage * P + piece) * kFewThreads + threadIdx.x) * 16;
    };
    auto issue = [&](int i) {
        if (i < blocks) {
            const int stage = i % kFewStages, kb = warp + i * kFewWarps;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int k = kb * kBlock8 + (t + 4 * h) * 16, left = a.K - k;
#pragma unroll
                for (int r = 0; r < 2; ++r)
                    copy_bytes(smem_addr(place(stage, 2 * r + h)), left > 0 ? w_row[r] + k : w_row[r], left);
                if constexpr (kFrom8) {
#pragma unroll
                    for (int n = 0; n < TILES; ++n) {
                        const int m = n * 8 + g;
                        const bool there = m < a.M && left > 0;
                        const uint8_t* x = static_cast<const uint8_t*>(a.x);
                        copy_bytes(smem_addr(place(stage, 4 + 2 * n + h)), there ? x + m * a.x_pitch + k : x,
                                   there ? left : 0);
                    }
                }
            }
        }
        copy_commit();
    };
    // scales and a wider x (four neighbouring values of each row a lane) one block ahead, in registers
    struct Ahead {
        __align__(4 * sizeof(X)) X x[kWideRows][4];  // (a row's four are read as one word)
        float sx[TILES], sw;
    };
    static_assert(alignof(Ahead) >= 4 * sizeof(X), "words of four values");
    auto load = [&](int i, Ahead& b) {
        if (i >= blocks) return;
        const int kb = warp + i * kFewWarps;
        b.sw = __ldg(w_scale + kb);
        if constexpr (kFrom8) {
#pragma unroll
            for (int n = 0; n < TILES; ++n) {
                const int m = n * 8 + g;
                b.sx[n] = m < a.M ? __ldg(a.x_scale + (long long)m * a.KB + kb) : 0.f;
            }
        } else {
            const int k = kb * kBlock8 + lane * 4;
#pragma unroll
            for (int m = 0; m < kWideRows; ++m) {
                if (m >= a.M) break;
                const X* src = static_cast<const X*>(a.x) + (long long)m * a.K + k;
                using Four = typename std::conditional<sizeof(X) == 4, uint4, uint2>::type;
                if (a.x_wide && k < a.K) {
                    *reinterpret_cast<Four*>(b.x[m]) = __ldg(reinterpret_cast<const Four*>(src));
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j) b.x[m][j] = !a.x_wide && k + j < a.K ? src[j] : from_acc<X>(0.f);
                }
            }
        }
    };
    float acc[TILES][4] = {};
    auto multiply = [&](int stage, Ahead& b) {
        uint4 x[TILES][2];
        if constexpr (kFrom8) {
#pragma unroll
            for (int n = 0; n < TILES; ++n)
#pragma unroll
                for (int h = 0; h < 2; ++h) x[n][h] = *reinterpret_cast<const uint4*>(place(stage, 4 + 2 * n + h));
        } else {  // a row at a time to 8 bits by the whole warp, and its pieces to the lanes that multiply them
            x[0][0] = x[0][1] = make_uint4(0, 0, 0, 0);
            b.sx[0] = 0.f;
#pragma unroll
            for (int m = 0; m < kWideRows; ++m) {
                if (m >= a.M) break;
                float v[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = to_acc(b.x[m][j]);
                drop_infinities<4>(v);
                float top = largest<4>(v);
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                const int e = scale_exponent(top);
                const uint32_t four = to_e4m3x4(v, exp2_int(-e));
                uint32_t w[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) w[j] = __shfl_sync(0xffffffffu, four, (j / 4) * 16 + 4 * t + j % 4);
                if (g == m) {
                    x[0][0] = make_uint4(w[0], w[1], w[2], w[3]);
                    x[0][1] = make_uint4(w[4], w[5], w[6], w[7]);
                    b.sx[0] = exp2_int(e);
                }
            }
        }
        float part[TILES][4] = {};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint4 a0 = *reinterpret_cast<const uint4*>(place(stage, h));
            const uint4 a1 = *reinterpret_cast<const uint4*>(place(stage, 2 + h));
#pragma unroll
            for (int n = 0; n < TILES; ++n) {
                const uint4& q = x[n][h];
                mma_16832(part[n], a0.x, a1.x, a0.y, a1.y, q.x, q.y);
                mma_16832(part[n], a0.z, a1.z, a0.w, a1.w, q.z, q.w);
            }
        }
#pragma unroll
        for (int n = 0; n < TILES; ++n) {
            // results are of rows 2t and 2t + 1 of x
            const float s0 = __shfl_sync(0xffffffffu, b.sx[n], t * 8) * b.sw;
            const float s1 = __shfl_sync(0xffffffffu, b.sx[n], t * 8 + 4) * b.sw;
            acc[n][0] = fmaf(part[n][0], s0, acc[n][0]);
            acc[n][1] = fmaf(part[n][1], s1, acc[n][1]);
            acc[n][2] = fmaf(part[n][2], s0, acc[n][2]);
            acc[n][3] = fmaf(part[n][3], s1, acc[n][3]);
        }
    };
    grid_dependency_wait();
    launch_dependents();
    {
#pragma unroll
        for (int i = 0; i < kFewStages - 1; ++i) issue(i);
        Ahead b0, b1;
        load(0, b0);
        for (int i = 0; i < blocks; i += 2) {
            copy_wait<kFewStages - 2>();
            issue(i + kFewStages - 1);
            load(i + 1, b1);
            multiply(i % kFewStages, b0);
            if (i + 1 >= blocks) break;
            copy_wait<kFewStages - 2>();
            issue(i + kFewStages);
            load(i + 2, b0);
            multiply((i + 1) % kFewStages, b1);
        }
        copy_wait<0>();
    }
#pragma unroll
    for (int n = 0; n < TILES; ++n) {
        sums[warp][g][n * 8 + 2 * t] = acc[n][0];
        sums[warp][g][n * 8 + 2 * t + 1] = acc[n][1];
        sums[warp][g + 8][n * 8 + 2 * t] = acc[n][2];
        sums[warp][g + 8][n * 8 + 2 * t + 1] = acc[n][3];
    }
    if (kTo8 && threadIdx.x < 8 * TILES) tops[threadIdx.x] = 0.f;
    __syncthreads();
    // 16 neighbouring threads end a row's 16 columns
    const int r = threadIdx.x & 15, m = threadIdx.x >> 4, n = n0 + r;
    const bool mine = m < 8 * TILES && m < a.M;
    float v = 0.f;
    if (mine && n < a.N) {
#pragma unroll
        for (int w = 0; w < kFewWarps; ++w) v += sums[w][r][m];
        v = activate(v + bias_at(a.end, n), a.end.act);
    }
    if constexpr (kTo8) {
        drop_infinities<1>(&v);
        float top = largest<1>(&v);
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        if (m < 8 * TILES && r == 0) tops[m] = top;
        cluster_arrive();
        cluster_wait();
        float peer = 0.f;  // lane r < 8 reads CTA r's
        if (m < 8 * TILES && r < 8) {
            const uint32_t at = cluster_map(smem_addr(&tops[m & ~3]), uint32_t(r));
            const uint4 four = ld_cluster_v4(at);
            peer = __uint_as_float((m & 3) == 0 ? four.x : (m & 3) == 1 ? four.y : (m & 3) == 2 ? four.z : four.w);
        }
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) peer = fmaxf(peer, __shfl_xor_sync(0xffffffffu, peer, o));
        top = __shfl_sync(0xffffffffu, peer, threadIdx.x & 16);
        cluster_arrive();
        if (mine) {
            const int e = scale_exponent(top);
            if (n < a.end.pitch)
                static_cast<uint8_t*>(a.end.out)[(long long)m * a.end.pitch + n] =
                    uint8_t(to_e4m3x2(v, 0.f, exp2_int(-e)));
            if (n < a.N && n % kBlock8 == 0)
                a.end.scale[(long long)m * ((a.N + kBlock8 - 1) / kBlock8) + n / kBlock8] = exp2_int(e);
        }
        cluster_wait();  // (no CTA leaves while another may read its maxima)
    } else {
        if (mine && n < a.N) static_cast<T*>(a.end.out)[(long long)m * a.N + n] = from_acc<T>(v);
    }
}

template <typename X, typename T, int TILES>
__global__ void __launch_bounds__(kFewThreads) fp8_few_kernel(const FewArgs a) {
    few_rows<X, T, TILES>(a);
}
template <typename X, int TILES>
__global__ void __cluster_dims__(8, 1, 1) __launch_bounds__(kFewThreads) fp8_few_to8_kernel(const FewArgs a) {
    few_rows<X, E4m3, TILES>(a);
}

}  // namespace td
