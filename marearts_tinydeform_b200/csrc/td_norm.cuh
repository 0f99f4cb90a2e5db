// td_norm.cuh -- layer norm with the residual added inside, forward and backward.
//
//   s = x + residual;  mean = sum(s) / C;  rstd = 1 / sqrt(sum((s - mean)^2) / C + eps)
//   y = (s - mean) * rstd * weight + bias
//   backward, with z = (s - mean) * rstd and g = dy * weight:
//     ds = rstd * (g - sum(g) / C - z * sum(g * z) / C)      (the gradient of x and of residual alike)
//     dweight = sum over rows of dy * z,  dbias = sum over rows of dy
//
// Bound by memory: a row is read once, into registers, and every sum over it is taken there -- the variance from the
// centred values. Where a row's mean is more than its deviation, the centred values are summed once more, so that what
// the first sum lost of large values does not move the row: one far from zero is normed as well as one at zero, but for
// its mean's rounding where the backward reads it. (Every row summed so: 54.6 us for the 49.4 below.) s is not rounded
// to the input type: both passes form it from x and residual in float32 (float64 for float64), as they do all sums.
//
// A group of G threads holds a row, EPT elements a thread (VEC = elements of a 16-byte vector, or 1 where C or an
// address is not a multiple of it), and walks over rows blockIdx, blockIdx + gridDim, .., the next row's loads issued
// before the present row's sums are taken (the backward, whose sums leave fewer warps an SM, has three rows ahead in
// shared memory). The backward's column sums stay in the group's registers over all of its rows; the groups of a CTA
// add theirs in order through shared memory, each CTA stores one float32 partial row, and norm_reduce_kernel adds those
// in a fixed order: no atomics, the same bits every time. 177784 rows x 256 in bfloat16: forward 49.4 us (5.5 TB/s),
// backward with its reduction 65.7 us (5.5 TB/s; 85 with one row ahead in registers, 75 with 4 CTAs an SM instead of
// 3); 8800 x 515 in float32, whose rows start anywhere, 14.3 and 19.6 us (3.8 and 3.7 TB/s).
#pragma once

#include "td_common.cuh"
#include "td_ptx.cuh"

namespace td {

constexpr int kNormThreads = 256;

template <typename T>
struct NormArgs {
    using acc = typename Elem<T>::acc;
    const T* x;
    const T* residual;  // or null
    const T* weight;
    const T* bias;      // forward; or null
    const T* grad_y;    // backward
    T* out;             // forward: y; backward: the gradient of x
    acc* mean;          // [rows], forward: written unless null; backward: read
    acc* rstd;
    acc* partial;       // backward: [gridDim][2][C] partial column sums
    long long rows;
    int C;
    acc eps;
};

// A thread's EPT elements of a row as raw vectors: VEC-element vectors at group stride G.
template <typename T, int VEC, int NV>
struct RowRegs {
    static constexpr bool kWide = VEC > 1;
    uint4 wide[kWide ? NV : 1];
    T one[kWide ? 1 : NV];

    template <int G>
    __device__ __forceinline__ void load(const T* __restrict__ p, int lane, int C) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (lane + i * G) * VEC;
            if constexpr (kWide) {
                wide[i] = c < C ? __ldg(reinterpret_cast<const uint4*>(p + c)) : make_uint4(0, 0, 0, 0);
            } else {
                one[i] = c < C ? p[c] : from_acc<T>(typename Elem<T>::acc(0));
            }
        }
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if constexpr (kWide) wide[i] = make_uint4(0, 0, 0, 0);
            else one[i] = from_acc<T>(typename Elem<T>::acc(0));
        }
    }
    __device__ __forceinline__ void widen(typename Elem<T>::acc* o) const {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if constexpr (kWide) unpack16<T>(wide[i], o + i * VEC);
            else o[i] = to_acc(one[i]);
        }
    }
};

template <typename T, int VEC, int NV, int G>
__device__ __forceinline__ void store_row(T* __restrict__ p, const typename Elem<T>::acc* v, int lane, int C) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (lane + i * G) * VEC;
        if (c >= C) continue;
        if constexpr (VEC > 1) store16<T>(p + c, v + i * VEC);
        else p[c] = from_acc<T>(v[i]);
    }
}

// Sums of N values over the G threads of the calling group, the same bits in each (an xor butterfly, then the warps in
// order). For G > 32 the warps meet at the group's own barrier, once a call: calls alternate between the two halves of
// `red`, and whoever writes a half again has passed the barrier behind its last reading.
template <int G, int N, typename A>
__device__ __forceinline__ void group_sum(A (&v)[N], A (&red)[2][N][kNormThreads / 32], int& half) {
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v[n] += __shfl_xor_sync(0xffffffffu, v[n], o);
    if constexpr (G > 32) {
        const int warp = threadIdx.x >> 5, first = warp / (G / 32) * (G / 32);
        if ((threadIdx.x & 31) == 0) {
#pragma unroll
            for (int n = 0; n < N; ++n) red[half][n][warp] = v[n];
        }
        named_barrier(1 + int(threadIdx.x) / G, G);
#pragma unroll
        for (int n = 0; n < N; ++n) {
            v[n] = red[half][n][first];
#pragma unroll
            for (int i = 1; i < G / 32; ++i) v[n] += red[half][n][first + i];
        }
        half ^= 1;
    }
}

// CTAs an SM holds of a form, by the registers it needs; a launch has one wave of them, so that all end together.
template <typename T, int VEC, int EPT, bool BWD>
constexpr int norm_ctas() {
    if (sizeof(T) == 8) return 1;
    if (EPT == 8) return BWD ? (sizeof(T) == 2 && VEC > 1 ? 3 : 2) : VEC > 1 ? 4 : 3;
    return EPT == 16 && !BWD ? 2 : 1;
}

template <typename T, int VEC, int G, int EPT>
__global__ void __launch_bounds__(kNormThreads, norm_ctas<T, VEC, EPT, false>())
    norm_forward_kernel(const NormArgs<T> a) {
    using acc = typename Elem<T>::acc;
    constexpr int NV = EPT / VEC, kGroups = kNormThreads / G;
    __shared__ acc red[2][1][kNormThreads / 32];
    int half = 0;
    const int group = threadIdx.x / G, lane = threadIdx.x % G;
    grid_dependency_wait();
    launch_dependents();
    RowRegs<T, VEC, NV> w, b, x, r;
    w.template load<G>(a.weight, lane, a.C);
    if (a.bias != nullptr) b.template load<G>(a.bias, lane, a.C);
    else b.zero();
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
        acc sum[1] = {0}, sq[1] = {0};
#pragma unroll
        for (int i = 0; i < EPT; ++i) sum[0] += s[i];  // elements outside the row are zero
        group_sum<G>(sum, red, half);
        const acc mean = sum[0] * inv;
#pragma unroll
        for (int i = 0; i < EPT; ++i) {
            const int c = (lane + i / VEC * G) * VEC + i % VEC;
            s[i] = c < a.C ? s[i] - mean : acc(0);
            sq[0] += s[i] * s[i];
        }
        group_sum<G>(sq, red, half);
        acc var = sq[0] * inv, more = 0;  // what the mean is short of
        if (mean * mean > var) {  // (the same in the whole group)
            sum[0] = 0;
#pragma unroll
            for (int i = 0; i < EPT; ++i) sum[0] += s[i];
            group_sum<G>(sum, red, half);
            more = sum[0] * inv;
            var = cmax(var - more * more, acc(0));
        }
        const acc rstd = acc(1) / sqrt(var + a.eps), shift = -more * rstd;
        if (a.mean != nullptr && lane == 0) {
            a.mean[row] = mean + more;
            a.rstd[row] = rstd;
        }
        acc u[EPT];
        w.widen(t);
        b.widen(u);
#pragma unroll
        for (int i = 0; i < EPT; ++i) s[i] = (s[i] * rstd + shift) * t[i] + u[i];
        store_row<T, VEC, NV, G>(a.out + row * a.C, s, lane, a.C);
    }
}

// Rows a backward group has in flight or at hand in shared memory: each thread copies its own vectors of them there
// and reads them back, so no barrier is needed. 0 where rows go through registers, one ahead.
template <typename T, int VEC, int EPT>
constexpr int norm_stages() {
    if (VEC == 1 || sizeof(T) == 8) return 0;
    return EPT / VEC <= 4 ? 4 : 2;
}
template <typename T, int VEC, int EPT>
constexpr size_t norm_smem() {
    return size_t(norm_stages<T, VEC, EPT>()) * 3 * (EPT / VEC) * kNormThreads * 16;
}

template <typename T, int VEC, int G, int EPT>
__global__ void __launch_bounds__(kNormThreads, norm_ctas<T, VEC, EPT, true>())
    norm_backward_kernel(const NormArgs<T> a) {
    using acc = typename Elem<T>::acc;
    constexpr int NV = EPT / VEC, kGroups = kNormThreads / G;
    constexpr int kCols = G * EPT;  // widest row of this form
    __shared__ acc red[2][2][kNormThreads / 32];
    int half = 0;
    __shared__ acc cols[kGroups > 1 ? kCols : 1];
    const int group = threadIdx.x / G, lane = threadIdx.x % G;
    grid_dependency_wait();
    launch_dependents();
    RowRegs<T, VEC, NV> w, x, r, d;
    w.template load<G>(a.weight, lane, a.C);
    r.zero();
    const acc inv = acc(1) / acc(a.C);
    const long long step = (long long)gridDim.x * kGroups;
    constexpr int S = norm_stages<T, VEC, EPT>();
    extern __shared__ __align__(16) unsigned char smem[];
    auto place = [&](int stage, int which, int i) {
        return smem + (((stage * 3 + which) * NV + i) * kNormThreads + threadIdx.x) * 16;
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
            }
        }
        copy_commit();
    };
    // the statistics of the group's next 32 rows, a lane's each, so that their latency shows once in 32 rows
    acc mean_l = 0, rstd_l = 0;
    acc mean_n = 0, rstd_n = 0;
    auto fetch = [&](long long row) {
        if (row < a.rows) {
            x.template load<G>(a.x + row * a.C, lane, a.C);
            d.template load<G>(a.grad_y + row * a.C, lane, a.C);
            if (a.residual != nullptr) r.template load<G>(a.residual + row * a.C, lane, a.C);
            mean_n = a.mean[row];
            rstd_n = a.rstd[row];
        } else {  // adds nothing to the column sums
            x.zero();
            d.zero();
            r.zero();
            mean_n = rstd_n = 0;
        }
    };
    acc dw[EPT], db[EPT];
#pragma unroll
    for (int i = 0; i < EPT; ++i) dw[i] = db[i] = 0;
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
                mean_l = mine < a.rows ? a.mean[mine] : acc(0);
                rstd_l = mine < a.rows ? a.rstd[mine] : acc(0);
            }
            mean_n = __shfl_sync(0xffffffffu, mean_l, n % 32);
            rstd_n = __shfl_sync(0xffffffffu, rstd_l, n % 32);
            copy_wait<S - 2>();
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                if constexpr (VEC > 1) {
                    x.wide[i] = *reinterpret_cast<const uint4*>(place(stage, 0, i));
                    d.wide[i] = *reinterpret_cast<const uint4*>(place(stage, 1, i));
                    if (a.residual != nullptr) r.wide[i] = *reinterpret_cast<const uint4*>(place(stage, 2, i));
                }
            }
        }
        x.widen(z);
        if (a.residual != nullptr) {
            r.widen(t);
#pragma unroll
            for (int i = 0; i < EPT; ++i) z[i] += t[i];
        }
        d.widen(g);
        const acc mean = mean_n, rstd = rstd_n;
        if constexpr (S > 0) {
            issue(row + (S - 1) * step, stage == 0 ? S - 1 : stage - 1);
            stage = stage == S - 1 ? 0 : stage + 1;
        } else {
            fetch(row + step);
        }
        w.widen(t);
        acc sums[2] = {0, 0};  // of g and of g z
#pragma unroll
        for (int i = 0; i < EPT; ++i) {
            // outside the row g is zero (dy was loaded as zero), so z's value there counts for nothing
            z[i] = (z[i] - mean) * rstd;
            db[i] += g[i];
            dw[i] += g[i] * z[i];
            g[i] *= t[i];
            sums[0] += g[i];
            sums[1] += g[i] * z[i];
        }
        group_sum<G>(sums, red, half);
        const acc sg = sums[0] * inv, sgz = sums[1] * inv;
#pragma unroll
        for (int i = 0; i < EPT; ++i) g[i] = (g[i] - sg - z[i] * sgz) * rstd;
        store_row<T, VEC, NV, G>(a.out + row * a.C, g, lane, a.C);
    }
    if constexpr (S > 0) copy_wait<0>();
    // the CTA's column sums: group 0's, + group 1's, .. in order
    acc* part = a.partial + (long long)blockIdx.x * 2 * a.C;
    auto add_up = [&](const acc(&v)[EPT], acc* out) {
        for (int turn = 0; turn < kGroups; ++turn) {
            if (group == turn) {
#pragma unroll
                for (int i = 0; i < EPT; ++i) {
                    const int c = (lane + i / VEC * G) * VEC + i % VEC;
                    acc sum = v[i];
                    if constexpr (kGroups > 1) {
                        if (turn > 0) sum += cols[c];
                        cols[c] = sum;
                    }
                    if (turn == kGroups - 1 && c < a.C) out[c] = sum;
                }
            }
            __syncthreads();
        }
    };
    add_up(dw, part);
    add_up(db, part + a.C);
}

// grad_weight and grad_bias from the CTAs' partial rows [parts][2][C]: each thread adds every kReduceRows-th row of
// one column, then the threads of a column are added in order.
constexpr int kReduceCols = 32, kReduceRows = 16;
template <typename T>
__global__ void __launch_bounds__(kReduceCols* kReduceRows)
    norm_reduce_kernel(const typename Elem<T>::acc* __restrict__ partial, T* grad_weight, T* grad_bias, int parts,
                       int C) {
    using acc = typename Elem<T>::acc;
    __shared__ acc sums[kReduceRows][kReduceCols];
    const int tx = threadIdx.x % kReduceCols, ty = threadIdx.x / kReduceCols;
    const int col = blockIdx.x * kReduceCols + tx;  // of 2 * C
    grid_dependency_wait();
    launch_dependents();
    acc sum = 0;
    if (col < 2 * C) {
#pragma unroll 4
        for (int p = ty; p < parts; p += kReduceRows) sum += partial[(long long)p * 2 * C + col];
    }
    sums[ty][tx] = sum;
    __syncthreads();
    if (ty == 0 && col < 2 * C) {
#pragma unroll
        for (int i = 1; i < kReduceRows; ++i) sum += sums[i][tx];
        T* out = col < C ? grad_weight : grad_bias;
        if (out != nullptr) out[col < C ? col : col - C] = from_acc<T>(sum);
    }
}

}  // namespace td
