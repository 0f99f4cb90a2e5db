// td_attention.cuh -- softmax attention with its backward pass: arguments shared by its kernels, and the CUDA-core
// kernels, which take every type and head width up to 128.
//
//   S_ij = scale * q_i . k_j, over the keys j that query i may use;  L_i = log sum_j exp(S_ij)
//   P_ij = exp(S_ij - L_i);  o_i = sum_j P_ij v_j
//   backward, from do_i:  delta_i = do_i . o_i;  dP_ij = do_i . v_j;  dS_ij = P_ij (dP_ij - delta_i)
//     dq_i = scale * sum_j dS_ij k_j;  dk_j = scale * sum_i dS_ij q_i;  dv_j = sum_i P_ij do_i
//
// The backward keeps no probabilities: it forms P again from S and L. A query that may use no key has o = 0, and its
// L is stored as +infinity, which makes every P of its row exp(-infinity) = 0 in the backward, and so its gradients
// zero. With fewer key heads than query heads, query head h reads key head h / (H / Hk), and dk, dv are summed over
// the query heads of their group inside the kernel.
//
// delta is the one sum of the backward whose terms cancel: dP_ij - delta_i is small against either where a row has few
// keys of weight, and a delta from the rounded result is off by as much as a rounding of dS itself would be. A forward
// that a backward follows therefore keeps, for 16-bit types, what the rounding took from each result as a second 16-bit
// tensor, and delta is formed from both.
//
// Logarithms are base 2 in the kernels: c = scale * log2(e), lse = L * log2(e).
//
// CUDA-core kernels: 256 threads, a 16 x 16 grid of R x R register tiles (the forward takes 1 x R for few queries, and
// is in td_attention_split.cuh). The tile of S (16 R x 16 R) is formed from
// rows in shared memory, the online softmax's maximum and sum run in registers (16 lanes hold a row), and P goes
// through shared memory for the product with the second operand, whose accumulator (16 R rows x DP columns) stays in
// registers. Bound by the FMA units: an R x R tile needs 2 R vector loads for 4 R^2 FMAs (R = 4).
#pragma once

#include <type_traits>

#include "td_common.cuh"
#include "td_ptx.cuh"

namespace td {

constexpr int kAttnMaxHeadDim = 128;
constexpr int kAttnRowPad = 128;  // lse and delta rows hold Q rounded up to this

// Strides are in elements; the innermost stride of every tensor is 1.
struct AttnArgs {
    const void *q, *k, *v;
    const void *out_in, *grad_out;  // backward: the forward's result and its gradient, [B, Q, H * D]
    const void* rest_in;            // backward, 16-bit types: what rounding took from the result, or null
    void* out;                      // forward: [B, Q, H * D]
    void* rest;                     // forward, 16-bit types: written unless null
    void *grad_q, *grad_k, *grad_v; // backward: [B, Q, H, D], [B, N, Hk, D] twice
    void* lse;                      // [B, H, Qp] in the accumulator type; forward: written unless null
    void* delta;                    // backward workspace, [B, H, Qp]
    long long q_b, q_t, q_h, k_b, k_t, k_h, v_b, v_t, v_h;
    const uint8_t* mask;            // nonzero = blocked, at b * m_b + h * m_h + i * m_q + j; or null
    long long m_b, m_h, m_q;
    const uint8_t* padding;         // [B, N], nonzero = no key there; or null
    int B, Q, N, H, Hk, D, Qp;
    // CUDA-core and TF32 backward: the query tiles of a tile of keys are shared by k_splits CTAs, the key tiles of a
    // tile of queries by q_splits. With more than one, split s leaves its sums, in the accumulator type, at s times the
    // size of the gradient in these, and attn_join_kernel adds them.
    int k_splits, q_splits;
    void *part_k, *part_v, *part_q;
    int vec_q, vec_k, vec_v, vec_g; // CUDA-core kernels: rows of q, k, v, grad_out are whole aligned 16-byte vectors
    int causal;                     // key j is open to query i while j <= i + (N - Q)
    double scale;
};

// Whether query i of head h may use key j (both inside their ranges).
__device__ __forceinline__ bool attn_open(const AttnArgs& a, const uint8_t* mask_row, const uint8_t* pad, int i,
                                          int j) {
    if (a.causal && j > i + (a.N - a.Q)) return false;
    if (pad != nullptr && pad[j] != 0) return false;
    return mask_row == nullptr || mask_row[j] == 0;
}

template <typename A> __device__ __forceinline__ A attn_exp2(A x);
template <> __device__ __forceinline__ float attn_exp2<float>(float x) { return exp2f(x); }
template <> __device__ __forceinline__ double attn_exp2<double>(double x) { return exp2(x); }
template <typename A> __device__ __forceinline__ A attn_log2(A x);
template <> __device__ __forceinline__ float attn_log2<float>(float x) { return log2f(x); }
template <> __device__ __forceinline__ double attn_log2<double>(double x) { return log2(x); }

// ---- CUDA-core kernels --------------------------------------------------------------------------------------------

template <typename A, int DP, int RM, int RN>
struct SimtTile {
    static constexpr int kVN = 16 / int(sizeof(A));  // accumulators of a 16-byte load
    static constexpr int kRows = 16 * RM, kCols = 16 * RN;  // of S
    static constexpr int kLd = DP + kVN;              // row pitch of an operand tile
    static constexpr int kLdP = kCols + kVN;          // row pitch of the P tile
    static constexpr int kWidth = DP / 16;            // accumulator columns a thread
    static constexpr size_t kRowBytes = size_t(kRows) * kLd * sizeof(A);  // an operand of S's rows
    static constexpr size_t kColBytes = size_t(kCols) * kLd * sizeof(A);  // of its columns
    static constexpr size_t kP = size_t(kRows) * kLdP * sizeof(A);
};

// ROWS rows from t0 on of a [tokens, D] slice into shared memory, widened; rows at or past n, padded rows and columns
// past D are zero. vec: rows are whole 16-byte vectors on 16-byte boundaries; all of a thread's loads are then in
// flight together (one 64 x 64 tile in float32: 12.0 us with single elements).
template <typename T, typename A, int DP, int ROWS>
__device__ __forceinline__ void simt_load(A* dst, const T* src, long long stride, int t0, int n, int D,
                                          const uint8_t* pad, bool vec) {
    constexpr int kLd = SimtTile<A, DP, 1, 1>::kLd;
    if (vec) {
        constexpr int V = Elem<T>::kVec, kPieces = DP / V, kTurns = (ROWS * kPieces + 255) / 256;
        uint4 x[kTurns];
#pragma unroll
        for (int u = 0; u < kTurns; ++u) {
            const int i = int(threadIdx.x) + 256 * u, r = i / kPieces, c = i % kPieces * V;
            x[u] = make_uint4(0u, 0u, 0u, 0u);
            if (i < ROWS * kPieces && t0 + r < n && c < D && (pad == nullptr || pad[t0 + r] == 0))
                x[u] = __ldg(reinterpret_cast<const uint4*>(src + (t0 + r) * stride + c));
        }
#pragma unroll
        for (int u = 0; u < kTurns; ++u) {
            const int i = int(threadIdx.x) + 256 * u, r = i / kPieces, c = i % kPieces * V;
            if (i >= ROWS * kPieces) continue;
            struct alignas(16) Wide { A e[V]; } w;
            unpack16<T>(x[u], w.e);
            *reinterpret_cast<Wide*>(dst + r * kLd + c) = w;
        }
        return;
    }
#pragma unroll 4
    for (int i = threadIdx.x; i < ROWS * DP; i += 256) {
        const int r = i / DP, c = i % DP;
        A x = 0;
        if (t0 + r < n && c < D && (pad == nullptr || pad[t0 + r] == 0)) x = to_acc(src[(t0 + r) * stride + c]);
        dst[r * kLd + c] = x;
    }
}

// s[r][c] = row (ty + 16 r) of x . row (tx + 16 c) of y
template <typename A, int DP, int RM, int RN>
__device__ __forceinline__ void simt_dot(const A* x, const A* y, int ty, int tx, A (&s)[RM][RN]) {
    using Tile = SimtTile<A, DP, RM, RN>;
    constexpr int V = Tile::kVN;
    struct alignas(16) Vec { A e[V]; };
#pragma unroll
    for (int r = 0; r < RM; ++r)
#pragma unroll
        for (int c = 0; c < RN; ++c) s[r][c] = 0;
#pragma unroll 2
    for (int k = 0; k < DP; k += V) {
        Vec xv[RM], yv[RN];
#pragma unroll
        for (int r = 0; r < RM; ++r) xv[r] = *reinterpret_cast<const Vec*>(x + (ty + 16 * r) * Tile::kLd + k);
#pragma unroll
        for (int c = 0; c < RN; ++c) yv[c] = *reinterpret_cast<const Vec*>(y + (tx + 16 * c) * Tile::kLd + k);
#pragma unroll
        for (int r = 0; r < RM; ++r)
#pragma unroll
            for (int c = 0; c < RN; ++c)
#pragma unroll
                for (int e = 0; e < V; ++e) s[r][c] += xv[r].e[e] * yv[c].e[e];
    }
}

// o[r][c] += sum_j p[ty + 16 r][j] * y[j][tx + 16 c]
template <typename A, int DP, int RM, int RN>
__device__ __forceinline__ void simt_accumulate(const A* p, const A* y, int ty, int tx,
                                                A (&o)[RM][SimtTile<A, DP, RM, RN>::kWidth]) {
    using Tile = SimtTile<A, DP, RM, RN>;
    constexpr int V = Tile::kVN;
    struct alignas(16) Vec { A e[V]; };
#pragma unroll 2
    for (int j = 0; j < Tile::kCols; j += V) {
        Vec pv[RM];
#pragma unroll
        for (int r = 0; r < RM; ++r) pv[r] = *reinterpret_cast<const Vec*>(p + (ty + 16 * r) * Tile::kLdP + j);
#pragma unroll
        for (int e = 0; e < V; ++e)
#pragma unroll
            for (int c = 0; c < Tile::kWidth; ++c) {
                const A b = y[(j + e) * Tile::kLd + tx + 16 * c];
#pragma unroll
                for (int r = 0; r < RM; ++r) o[r][c] += pv[r].e[e] * b;
            }
    }
}

// Sum or maximum over the 16 lanes that hold a row.
template <typename A> __device__ __forceinline__ A row_sum(A v) {
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
template <typename A> __device__ __forceinline__ A row_max(A v) {
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) v = cmax(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// The end of the keys that rows i < row_end may use: everything, or the causal edge of the last row.
__device__ __forceinline__ int attn_key_end(const AttnArgs& a, int row_end) {
    if (!a.causal) return a.N;
    const int last = min(row_end, a.Q) + (a.N - a.Q);
    return max(0, min(a.N, last));
}

// delta[b, h, i] = grad_out . out over a query's head; zero in the rows behind the last query. A thread per row, adding
// in simt_dot's order: where a query has one key only, its result is that key's value and dP - delta is exactly zero.
template <typename T>
__global__ void __launch_bounds__(256) attn_delta_kernel(const AttnArgs a) {
    using A = typename Elem<T>::acc;
    const long long row = (long long)blockIdx.x * 256 + threadIdx.x;  // (b * H + h) * Qp + i
    grid_dependency_wait();
    launch_dependents();
    if (row >= (long long)a.B * a.H * a.Qp) return;
    const int i = int(row % a.Qp);
    const long long bh = row / a.Qp;
    A sum = 0;
    if (i < a.Q) {
        const long long at = ((bh / a.H * a.Q + i) * a.H + bh % a.H) * a.D;
        const T* o = static_cast<const T*>(a.out_in) + at;
        const T* g = static_cast<const T*>(a.grad_out) + at;
        const T* rest = static_cast<const T*>(a.rest_in);
        for (int d = 0; d < a.D; ++d)
            sum += (rest == nullptr ? to_acc(o[d]) : to_acc(o[d]) + to_acc(rest[at + d])) * to_acc(g[d]);
    }
    static_cast<A*>(a.delta)[row] = sum;
}

// What a backward CTA found for element `at` of a gradient of `size` elements.
template <typename T, typename A>
__device__ __forceinline__ void attn_put_grad(void* grad, void* part, int splits, int split, long long size,
                                              long long at, A x) {
    if (splits == 1) static_cast<T*>(grad)[at] = from_acc<T>(x);
    else static_cast<A*>(part)[split * size + at] = x;
}

// Adds the splits of a gradient in their order, a thread per element: those of the keys, the values, then the queries
// (without those that were not split).
template <typename T>
__global__ void __launch_bounds__(256) attn_join_kernel(const AttnArgs a) {
    using A = typename Elem<T>::acc;
    const long long size_k = (long long)a.B * a.N * a.Hk * a.D, size_q = (long long)a.B * a.Q * a.H * a.D;
    long long at = (long long)blockIdx.x * 256 + threadIdx.x;
    grid_dependency_wait();
    launch_dependents();
    const bool keys = a.k_splits > 1 && at < 2 * size_k, values = keys && at >= size_k;
    if (!keys && a.k_splits > 1) at -= 2 * size_k;
    if (values) at -= size_k;
    const long long size = keys ? size_k : size_q;
    const int splits = keys ? a.k_splits : a.q_splits;
    if (splits == 1 || at >= size) return;
    const A* part = static_cast<const A*>(values ? a.part_v : keys ? a.part_k : a.part_q) + at;
    A sum = 0;
#pragma unroll 8
    for (int s = 0; s < splits; ++s) sum += part[s * size];
    static_cast<T*>(values ? a.grad_v : keys ? a.grad_k : a.grad_q)[at] = from_acc<T>(sum);
}

// The gradient of the keys and values (blocks below kv_blocks: one tile of keys of one key head, over the query heads
// of its group and their query tiles) and of the queries (the other blocks: one tile of queries of one head), the
// splits of a tile beside each other.
template <typename T, int DP, int R>
__global__ void __launch_bounds__(256) attn_simt_backward_kernel(const AttnArgs a, int kv_blocks) {
    using A = typename Elem<T>::acc;
    using Tile = SimtTile<A, DP, R, R>;
    constexpr int M = Tile::kRows;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    A* qs = reinterpret_cast<A*>(smem_raw);
    A* gs = qs + M * Tile::kLd;
    A* ks = gs + M * Tile::kLd;
    A* vs = ks + M * Tile::kLd;
    A* ps = vs + M * Tile::kLd;
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    const int group = a.H / a.Hk;
    const A c = A(a.scale * 1.4426950408889634), scale = A(a.scale);
    const T* q = static_cast<const T*>(a.q);
    const T* k = static_cast<const T*>(a.k);
    const T* v = static_cast<const T*>(a.v);
    const T* g = static_cast<const T*>(a.grad_out);
    const A* lse = static_cast<const A*>(a.lse);
    const A* delta = static_cast<const A*>(a.delta);
    grid_dependency_wait();
    launch_dependents();
    if (int(blockIdx.x) < kv_blocks) {
        const int tiles = (a.N + M - 1) / M, split = blockIdx.x % a.k_splits, blk = blockIdx.x / a.k_splits;
        const int j0 = blk % tiles * M, hk = blk / tiles % a.Hk, b = blk / tiles / a.Hk;
        const uint8_t* pad = a.padding == nullptr ? nullptr : a.padding + (long long)b * a.N;
        simt_load<T, A, DP, M>(ks, k + b * a.k_b + hk * a.k_h, a.k_t, j0, a.N, a.D, pad, a.vec_k != 0);
        simt_load<T, A, DP, M>(vs, v + b * a.v_b + hk * a.v_h, a.v_t, j0, a.N, a.D, pad, a.vec_v != 0);
        A dk[R][Tile::kWidth], dv[R][Tile::kWidth];
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int x = 0; x < Tile::kWidth; ++x) dk[r][x] = dv[r][x] = 0;
        // the first query that may use key j0
        const int first = a.causal ? max(0, min(a.Q, j0 - (a.N - a.Q))) / M * M : 0;
        const int cols = (a.Q - first + M - 1) / M;
        int n = int((long long)cols * group * split / a.k_splits);
        const int end = int((long long)cols * group * (split + 1) / a.k_splits);
        while (n < end) {
            const int h = hk * group + n / cols;
            const uint8_t* mask = a.mask == nullptr ? nullptr : a.mask + b * a.m_b + h * a.m_h;
            const A* lse_h = lse + ((long long)b * a.H + h) * a.Qp;
            const A* delta_h = delta + ((long long)b * a.H + h) * a.Qp;
            const int head_end = min(end, (n / cols + 1) * cols);
            for (; n < head_end; ++n) {
                const int i0 = first + n % cols * M;
                __syncthreads();
                simt_load<T, A, DP, M>(qs, q + b * a.q_b + h * a.q_h, a.q_t, i0, a.Q, a.D, nullptr, a.vec_q != 0);
                simt_load<T, A, DP, M>(gs, g + ((long long)b * a.Q * a.H + h) * a.D, (long long)a.H * a.D, i0, a.Q,
                                       a.D, nullptr, a.vec_g != 0);
                __syncthreads();
                A s[R][R], p[R][R];
                simt_dot<A, DP, R, R>(ks, qs, ty, tx, s);
#pragma unroll
                for (int x = 0; x < R; ++x) {
                    const int i = i0 + tx + 16 * x;
                    const A li = i < a.Q ? lse_h[i] : A(INFINITY);
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        const int j = j0 + ty + 16 * r;
                        const bool open = i < a.Q && j < a.N &&
                                          attn_open(a, mask == nullptr ? nullptr : mask + i * a.m_q, pad, i, j);
                        p[r][x] = open ? attn_exp2<A>(s[r][x] * c - li) : A(0);
                        ps[(ty + 16 * r) * Tile::kLdP + tx + 16 * x] = p[r][x];
                    }
                }
                __syncwarp();
                simt_accumulate<A, DP, R, R>(ps, gs, ty, tx, dv);
                simt_dot<A, DP, R, R>(vs, gs, ty, tx, s);
                __syncwarp();
#pragma unroll
                for (int x = 0; x < R; ++x) {
                    const int i = i0 + tx + 16 * x;
                    const A di = i < a.Q ? delta_h[i] : A(0);
#pragma unroll
                    for (int r = 0; r < R; ++r)
                        ps[(ty + 16 * r) * Tile::kLdP + tx + 16 * x] =
                            p[r][x] == A(0) ? A(0) : p[r][x] * (s[r][x] - di);
                }
                __syncwarp();
                simt_accumulate<A, DP, R, R>(ps, qs, ty, tx, dk);
            }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int j = j0 + ty + 16 * r;
            if (j >= a.N) continue;
#pragma unroll
            for (int x = 0; x < Tile::kWidth; ++x) {
                const int d = tx + 16 * x;
                if (d >= a.D) continue;
                const long long at = (((long long)b * a.N + j) * a.Hk + hk) * a.D + d;
                const long long size = (long long)a.B * a.N * a.Hk * a.D;
                attn_put_grad<T, A>(a.grad_k, a.part_k, a.k_splits, split, size, at, dk[r][x] * scale);
                attn_put_grad<T, A>(a.grad_v, a.part_v, a.k_splits, split, size, at, dv[r][x]);
            }
        }
        return;
    }
    const int split = (int(blockIdx.x) - kv_blocks) % a.q_splits, blk = (int(blockIdx.x) - kv_blocks) / a.q_splits;
    const int tiles = (a.Q + M - 1) / M;
    const int i0 = blk % tiles * M, h = blk / tiles % a.H, b = blk / tiles / a.H, hk = h / group;
    const uint8_t* pad = a.padding == nullptr ? nullptr : a.padding + (long long)b * a.N;
    const uint8_t* mask = a.mask == nullptr ? nullptr : a.mask + b * a.m_b + h * a.m_h;
    simt_load<T, A, DP, M>(qs, q + b * a.q_b + h * a.q_h, a.q_t, i0, a.Q, a.D, nullptr, a.vec_q != 0);
    simt_load<T, A, DP, M>(gs, g + ((long long)b * a.Q * a.H + h) * a.D, (long long)a.H * a.D, i0, a.Q, a.D, nullptr,
                           a.vec_g != 0);
    A dq[R][Tile::kWidth], li[R], di[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int i = i0 + ty + 16 * r;
        const long long at = ((long long)b * a.H + h) * a.Qp + i;
        li[r] = i < a.Q ? lse[at] : A(INFINITY);
        di[r] = i < a.Q ? delta[at] : A(0);
#pragma unroll
        for (int x = 0; x < Tile::kWidth; ++x) dq[r][x] = 0;
    }
    const int cols = (attn_key_end(a, i0 + M) + M - 1) / M;
    const int end = int((long long)cols * (split + 1) / a.q_splits);
    for (int n = int((long long)cols * split / a.q_splits); n < end; ++n) {
        const int j0 = n * M;
        __syncthreads();
        simt_load<T, A, DP, M>(ks, k + b * a.k_b + hk * a.k_h, a.k_t, j0, a.N, a.D, pad, a.vec_k != 0);
        simt_load<T, A, DP, M>(vs, v + b * a.v_b + hk * a.v_h, a.v_t, j0, a.N, a.D, pad, a.vec_v != 0);
        __syncthreads();
        A s[R][R], dp[R][R];
        simt_dot<A, DP, R, R>(qs, ks, ty, tx, s);
        simt_dot<A, DP, R, R>(gs, vs, ty, tx, dp);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int i = i0 + ty + 16 * r;
#pragma unroll
            for (int x = 0; x < R; ++x) {
                const int j = j0 + tx + 16 * x;
                const bool open = i < a.Q && j < a.N &&
                                  attn_open(a, mask == nullptr ? nullptr : mask + i * a.m_q, pad, i, j);
                ps[(ty + 16 * r) * Tile::kLdP + tx + 16 * x] =
                    open ? attn_exp2<A>(s[r][x] * c - li[r]) * (dp[r][x] - di[r]) : A(0);
            }
        }
        __syncwarp();
        simt_accumulate<A, DP, R, R>(ps, ks, ty, tx, dq);
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int i = i0 + ty + 16 * r;
        if (i >= a.Q) continue;
#pragma unroll
        for (int x = 0; x < Tile::kWidth; ++x) {
            const int d = tx + 16 * x;
            if (d < a.D)
                attn_put_grad<T, A>(a.grad_q, a.part_q, a.q_splits, split, (long long)a.B * a.Q * a.H * a.D,
                                    (((long long)b * a.Q + i) * a.H + h) * a.D + d, dq[r][x] * scale);
        }
    }
}

}  // namespace td
