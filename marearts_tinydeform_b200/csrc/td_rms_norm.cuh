// td_rms_norm.cuh -- root-mean-square norm with the residual added inside, forward (its result in 8 bits if asked) and
// backward.
//
//   s = x + residual;  rstd = 1 / sqrt(sum(s^2) / C + eps);  y = s * rstd * weight
//   8 bits: y, not rounded before, in blocks of 128 channels (td_fp8.cuh)
//   backward, with z = s * rstd and g = dy * weight:
//     ds = rstd * (g - z * sum(g * z) / C) + dtotal      (the gradient of x and of residual alike; dtotal: of s itself,
//     dweight = sum over rows of dy * z                   where the caller takes the sum as well)
//
// Bound by memory. The layout is the layer norm's (td_norm.cuh): G threads hold a row in registers, EPT elements each,
// walk over rows with the next row's loads under way, and the backward's column sums stay in registers until the end.
// s is formed from x and residual in float32 (float64) in both passes, never from its rounded copy.
//
// A block of 128 channels is 128 / VEC neighbouring lanes of one vector, so its largest magnitude is a few shuffles;
// without vectors (rows that start anywhere) it is 128 / G vectors of a warp's lanes, or four warps of one, which meet
// in shared memory. 177784 x 256 bfloat16 with the residual: in 8 bits 42 us (5.4 TB/s), with the sum 57.5 (6.3 TB/s),
// backward with the sum's gradient 78 (5.8 TB/s, with its column sums); 8800 x 515 float32, whose rows start anywhere,
// forward and backward together 44.
#pragma once

#include "td_fp8.cuh"
#include "td_norm.cuh"

namespace td {

template <typename T>
struct RmsArgs {
    using acc = typename Elem<T>::acc;
    const T* x;
    const T* residual;    // or null
    const T* weight;
    const T* grad_y;      // backward
    const T* grad_total;  // backward; or null
    T* out;               // forward: y, or null where it goes to q; backward: the gradient of x
    T* total;             // forward: s, or null
    uint8_t* q;           // forward, 8 bits: [rows, pitch]; what lies behind C in a row is written as zeros
    float* scale;         // [rows, ceil(C / 128)]
    acc* rstd;            // [rows], forward: written unless null; backward: read
    acc* partial;         // backward: [gridDim][C] partial column sums
    long long rows;
    int C, pitch;
    acc eps;
};

template <typename T, int VEC, int G, int EPT, bool Q8>
__global__ void __launch_bounds__(kNormThreads, norm_ctas<T, VEC, EPT, false>())
    rms_forward_kernel(const RmsArgs<T> a) {
    using acc = typename Elem<T>::acc;
    constexpr int NV = EPT / VEC, kGroups = kNormThreads / G;
    __shared__ acc red[2][1][kNormThreads / 32];
    constexpr bool kMeet = Q8 && VEC == 1 && G > 32;  // a block's warps meet in shared memory
    __shared__ float tops[2][kMeet ? NV : 1][kNormThreads / 32];
    int half = 0, turn = 0;
    const int group = threadIdx.x / G, lane = threadIdx.x % G;
    grid_dependency_wait();
    launch_dependents();
    RowRegs<T, VEC, NV> w, x, r;
    w.template load<G>(a.weight, lane, a.C);
    const acc inv = acc(1) / acc(a.C);
    const long long step = (long long)gridDim.x * kGroups;
    auto fetch = [&](long long row) {
        if (row < a.rows) {
            x.template load<G>(a.x + row * a.C, lane, a.C);
            if (a.residual != nullptr) r.template load<G>(a.residual + row * a.C, lane, a.C);
        } else {
            x.zero();
        }
    };
    r.zero();
    long long row = (long long)blockIdx.x * kGroups + group;
    fetch(row);
    for (; row < a.rows; row += step) {
        acc s[EPT], t[EPT];
        x.widen(s);
        if (a.residual != nullptr) {
            r.widen(t);
#pragma unroll
            for (int i = 0; i < EPT; ++i) s[i] += t[i];
        }
        fetch(row + step);
        if (a.total != nullptr) store_row<T, VEC, NV, G>(a.total + row * a.C, s, lane, a.C);
        acc sq[1] = {0};
#pragma unroll
        for (int i = 0; i < EPT; ++i) sq[0] += s[i] * s[i];  // elements outside the row are zero
        group_sum<G>(sq, red, half);
        const acc rstd = acc(1) / sqrt(sq[0] * inv + a.eps);
        if (a.rstd != nullptr && lane == 0) a.rstd[row] = rstd;
        w.widen(t);
#pragma unroll
        for (int i = 0; i < EPT; ++i) s[i] = s[i] * rstd * t[i];
        if constexpr (!Q8) {
            store_row<T, VEC, NV, G>(a.out + row * a.C, s, lane, a.C);
        } else {
            float top[NV], v[EPT];
#pragma unroll
            for (int i = 0; i < EPT; ++i) v[i] = float(s[i]);
            if (infinite(largest<EPT>(v))) drop_infinities<EPT>(v);
#pragma unroll
            for (int i = 0; i < NV; ++i) top[i] = largest<VEC>(v + i * VEC);
            if constexpr (VEC == 1 && G == 32) {
#pragma unroll
                for (int i = 0; i < NV; i += 4)
                    top[i] = top[i + 1] = top[i + 2] = top[i + 3] =
                        fmaxf(fmaxf(top[i], top[i + 1]), fmaxf(top[i + 2], top[i + 3]));
            }
            constexpr int kLanes = VEC == 1 ? 32 : kBlock8 / VEC;
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int o = kLanes / 2; o > 0; o >>= 1) top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], o));
            if constexpr (kMeet) {
                // whoever writes a half again has passed the barrier behind its last reading (as in group_sum)
                const int warp = threadIdx.x >> 5, first = warp & ~3;
                if ((threadIdx.x & 31) == 0) {
#pragma unroll
                    for (int i = 0; i < NV; ++i) tops[turn][i][warp] = top[i];
                }
                named_barrier(1 + int(threadIdx.x) / G, G);
#pragma unroll
                for (int i = 0; i < NV; ++i)
                    top[i] = fmaxf(fmaxf(tops[turn][i][first], tops[turn][i][first + 1]),
                                   fmaxf(tops[turn][i][first + 2], tops[turn][i][first + 3]));
                turn ^= 1;
            }
            const int blocks = (a.C + kBlock8 - 1) / kBlock8;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = (lane + i * G) * VEC, e = scale_exponent(top[i]);
                if (c < a.C && c % kBlock8 == 0) a.scale[row * blocks + c / kBlock8] = exp2_int(e);
                if (c >= a.pitch) continue;  // (the pitch is a multiple of 16)
                uint8_t* dst = a.q + row * a.pitch + c;
                const float f = exp2_int(-e);
                float* w8 = v + i * VEC;
                if (c >= a.C) {  // zeros, where a NaN as the row's norm has made the products of zeros NaN
#pragma unroll
                    for (int k = 0; k < VEC; ++k) w8[k] = 0.f;
                }
                if constexpr (VEC == 8)
                    *reinterpret_cast<uint2*>(dst) = make_uint2(to_e4m3x4(w8, f), to_e4m3x4(w8 + 4, f));
                else if constexpr (VEC == 4) *reinterpret_cast<uint32_t*>(dst) = to_e4m3x4(w8, f);
                else *dst = uint8_t(to_e4m3x2(w8[0], 0.f, f));
            }
        }
    }
}

// The backward's rows ahead in shared memory, as in td_norm.cuh: stages, and tensors staged (x, dy, residual, dtotal;
// the last one through registers where a row's four would not fit).
template <typename T, int VEC, int EPT>
constexpr int rms_stages() {
    if (VEC == 1 || sizeof(T) == 8) return 0;
    return EPT / VEC == 1 ? 4 : EPT / VEC <= 4 ? 3 : 2;
}
template <typename T, int VEC, int EPT>
constexpr int rms_staged() {
    return EPT / VEC <= 4 ? 4 : 3;
}
template <typename T, int VEC, int EPT>
constexpr size_t rms_smem() {
    return size_t(rms_stages<T, VEC, EPT>()) * rms_staged<T, VEC, EPT>() * (EPT / VEC) * kNormThreads * 16;
}

template <typename T, int VEC, int G, int EPT>
__global__ void __launch_bounds__(kNormThreads, norm_ctas<T, VEC, EPT, true>())
    rms_backward_kernel(const RmsArgs<T> a) {
    using acc = typename Elem<T>::acc;
    constexpr int NV = EPT / VEC, kGroups = kNormThreads / G;
    constexpr int kCols = G * EPT;  // widest row of this form
    __shared__ acc red[2][1][kNormThreads / 32];
    int half = 0;
    __shared__ acc cols[kGroups > 1 ? kCols : 1];
    const int group = threadIdx.x / G, lane = threadIdx.x % G;
    grid_dependency_wait();
    launch_dependents();
    RowRegs<T, VEC, NV> w, x, r, d, u;
    w.template load<G>(a.weight, lane, a.C);
    r.zero();
    u.zero();
    const acc inv = acc(1) / acc(a.C);
    const long long step = (long long)gridDim.x * kGroups;
    constexpr int S = rms_stages<T, VEC, EPT>(), W = rms_staged<T, VEC, EPT>();
    extern __shared__ __align__(16) unsigned char smem[];
    auto place = [&](int stage, int which, int i) {
        return smem + (((stage * W + which) * NV + i) * kNormThreads + threadIdx.x) * 16;
    };
    auto issue = [&](long long row, int stage) {
        if (row < a.rows) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = (lane + i * G) * VEC;
                const long long at = c < a.C ? row * a.C + c : 0;
                copy16(smem_addr(place(stage, 0, i)), a.x + at, c < a.C);
                copy16(smem_addr(place(stage, 1, i)), a.grad_y + at, c < a.C);
                if (a.residual != nullptr) copy16(smem_addr(place(stage, 2, i)), a.residual + at, c < a.C);
                if (W == 4 && a.grad_total != nullptr)
                    copy16(smem_addr(place(stage, W - 1, i)), a.grad_total + at, c < a.C);
            }
        }
        copy_commit();
    };
    // the reciprocal norms of the group's next 32 rows, a lane's each, so that their latency shows once in 32 rows
    acc rstd_l = 0, rstd_n = 0;
    auto fetch = [&](long long row) {
        if (row < a.rows) {
            x.template load<G>(a.x + row * a.C, lane, a.C);
            d.template load<G>(a.grad_y + row * a.C, lane, a.C);
            if (a.residual != nullptr) r.template load<G>(a.residual + row * a.C, lane, a.C);
            rstd_n = a.rstd[row];
        } else {
            x.zero();
            d.zero();
            r.zero();
            rstd_n = 0;
        }
    };
    acc dw[EPT];
#pragma unroll
    for (int i = 0; i < EPT; ++i) dw[i] = 0;
    long long row = (long long)blockIdx.x * kGroups + group;
    if constexpr (S > 0) {
#pragma unroll
        for (int s = 0; s < S - 1; ++s) issue(row + s * step, s);
    } else {
        fetch(row);
    }
    int stage = 0;
    for (int n = 0; row < a.rows; row += step, ++n) {
        acc z[EPT], g[EPT], t[EPT];
        if constexpr (S > 0) {
            if (n % 32 == 0) {
                const long long mine = row + (threadIdx.x % 32) * step;
                rstd_l = mine < a.rows ? a.rstd[mine] : acc(0);
            }
            rstd_n = __shfl_sync(0xffffffffu, rstd_l, n % 32);
            copy_wait<S - 2>();
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                if constexpr (VEC > 1) {
                    x.wide[i] = *reinterpret_cast<const uint4*>(place(stage, 0, i));
                    d.wide[i] = *reinterpret_cast<const uint4*>(place(stage, 1, i));
                    if (a.residual != nullptr) r.wide[i] = *reinterpret_cast<const uint4*>(place(stage, 2, i));
                    if (W == 4 && a.grad_total != nullptr)
                        u.wide[i] = *reinterpret_cast<const uint4*>(place(stage, W - 1, i));
                }
            }
        }
        if ((S == 0 || W < 4) && a.grad_total != nullptr) u.template load<G>(a.grad_total + row * a.C, lane, a.C);
        x.widen(z);
        if (a.residual != nullptr) {
            r.widen(t);
#pragma unroll
            for (int i = 0; i < EPT; ++i) z[i] += t[i];
        }
        d.widen(g);
        const acc rstd = rstd_n;
        if constexpr (S > 0) {
            issue(row + (S - 1) * step, stage == 0 ? S - 1 : stage - 1);
            stage = stage == S - 1 ? 0 : stage + 1;
        } else {
            fetch(row + step);
        }
        w.widen(t);
        acc sum[1] = {0};  // of g z
#pragma unroll
        for (int i = 0; i < EPT; ++i) {
            z[i] *= rstd;  // zero outside the row, as g
            dw[i] += g[i] * z[i];
            g[i] *= t[i];
            sum[0] += g[i] * z[i];
        }
        group_sum<G>(sum, red, half);
        const acc sgz = sum[0] * inv;
        u.widen(t);
#pragma unroll
        for (int i = 0; i < EPT; ++i) g[i] = (g[i] - z[i] * sgz) * rstd + t[i];
        store_row<T, VEC, NV, G>(a.out + row * a.C, g, lane, a.C);
    }
    if constexpr (S > 0) copy_wait<0>();
    // the CTA's column sums: group 0's, + group 1's, .. in order
    acc* part = a.partial + (long long)blockIdx.x * a.C;
    for (int turn = 0; turn < kGroups; ++turn) {
        if (group == turn) {
#pragma unroll
            for (int i = 0; i < EPT; ++i) {
                const int c = (lane + i / VEC * G) * VEC + i % VEC;
                acc sum = dw[i];
                if constexpr (kGroups > 1) {
                    if (turn > 0) sum += cols[c];
                    cols[c] = sum;
                }
                if (turn == kGroups - 1 && c < a.C) part[c] = sum;
            }
        }
        __syncthreads();
    }
}

}  // namespace td
