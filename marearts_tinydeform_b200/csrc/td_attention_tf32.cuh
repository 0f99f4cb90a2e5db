// td_attention_tf32.cuh -- float32 attention on tensor cores: every product in three TF32 ones.
//
// x = hi + lo with hi = x rounded to TF32's 11 bits and lo = x - hi (exact; the tensor core cuts it to 11 bits), so a b
// ~ hi hi + hi lo + lo hi to about 22 bits. Tiles of 64 rows, four warps of 16, as mma.sync m16n8k8 fragments; the
// other side streams through two buffers of shared memory by asynchronous copies. What bounds it: the rate of these
// products (about 38 TFLOP/s are left of three) and, with few tiles a CTA, one warp's chain of some 1500 instructions a
// tile. 8 heads x 32, 4 x 1100 tokens: forward 216 us (a quarter less in one wave of four CTAs an SM with spills, but
// 18 instead of 15 for 2 x 300), backward 527 us (three CTAs an SM; a tenth more with two, a quarter with four); 8
// heads x 64, 4096 tokens: 980 and 2500 to 2650 us; the CUDA-core kernels take 234, 708, 1293 and 3517. The mma.sync
// pipe is 38 % (forward) and 44 % (backward) busy, the issue slots 43 and 40 %; waits on fixed latencies come first.
//
// Accuracy, relative to float64 over 2 x 1100 tokens x 8 heads x 32: 3.4e-7 forward, 5e-7 backward (float32 matrix
// products of a library: 6.4e-7). With hi cut instead of rounded and one sum over all keys it was 8.6e-6, in
// three quarters of the time.
//
// Fragments need no shuffles: the order of a summed index is free. For row . row products (S, dP) a thread's 4
// consecutive elements of a row are its slots t, t + 4 of two K steps, in both operands. For P . rows products the
// accumulator's columns 2 t, 2 t + 1 are slots t, t + 4 of the A operand, and rows 2 t, 2 t + 1 of the B operand.
#pragma once

#include "td_attention_split.cuh"

namespace td {

constexpr int kTf32Threads = 128, kTf32Rows = 64;
// CTAs an SM holds, by registers and, for wide heads, shared memory.
template <int DP, bool BWD> constexpr int kTf32Ctas = DP == 32 ? 3 : DP == 64 ? (BWD ? 3 : 2) : 1;

template <int DP, int NT>
struct Tf32Layout {
    static constexpr int kPitch = DP + 4;  // floats: rows 2 t of a fragment fall on different banks
    static constexpr int kFixed = kTf32Rows * kPitch, kTile = NT * kPitch;
};

__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo) {
    hi = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
    lo = __float_as_uint(x - __uint_as_float(hi));
}

__device__ __forceinline__ void mma_1688(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// big[i] + small[i] += a b[i] for M independent tiles in three products each: one product of every tile before the next
// of any, as each waits for the last into its tile. The tensor core cuts its sums where float32 would round them, which
// adds up in one direction: the two small products have sums of their own, where that does not show, and neither sum
// lasts longer than a tile.
template <int M>
__device__ __forceinline__ void mma_split(float (*big)[4], float (*small)[4], const uint32_t (&ah)[4],
                                          const uint32_t (&al)[4], const uint32_t (&bh)[M][2],
                                          const uint32_t (&bl)[M][2]) {
#pragma unroll
    for (int i = 0; i < M; ++i) mma_1688(small[i], al, bh[i][0], bh[i][1]);
#pragma unroll
    for (int i = 0; i < M; ++i) mma_1688(big[i], ah, bh[i][0], bh[i][1]);
#pragma unroll
    for (int i = 0; i < M; ++i) mma_1688(small[i], ah, bl[i][0], bl[i][1]);
}

// ROWS rows from t0 on of a [tokens, D] slice into shared memory (16-byte copies; rows past n, padded rows and columns
// past D are zero), as one asynchronous group of the caller's.
template <int DP, int ROWS>
__device__ __forceinline__ void tf32_load(float* dst, const float* src, long long stride, int t0, int n, int D,
                                          const uint8_t* pad) {
    constexpr int kPieces = DP / 4, kPitch = DP + 4;
#pragma unroll
    for (int u = 0; u < ROWS * kPieces / kTf32Threads; ++u) {
        const int i = int(threadIdx.x) + kTf32Threads * u, r = i / kPieces, c = i % kPieces * 4;
        const bool real = t0 + r < n && c < D && (pad == nullptr || pad[t0 + r] == 0);
        copy16(smem_addr(dst + r * kPitch + c), real ? src + (t0 + r) * stride + c : src, real);
    }
}

// s[j] = rows g, g + 8 of a . rows 8 j .. of b. CHECK: infinities come out as float32 has them.
template <int DP, int NT, bool CHECK>
__device__ __forceinline__ void tf32_scores(const float* a, const float* b, int g, int t, float (&s)[NT / 8][4]) {
    constexpr int kPitch = DP + 4;
    float small[NT / 8][4];
#pragma unroll
    for (int j = 0; j < NT / 8; ++j)
#pragma unroll
        for (int y = 0; y < 4; ++y) s[j][y] = small[j][y] = 0.f;
#pragma unroll 1
    for (int k = 0; k < DP; k += 16) {
        const float4 a0 = *reinterpret_cast<const float4*>(a + g * kPitch + k + 4 * t);
        const float4 a1 = *reinterpret_cast<const float4*>(a + (g + 8) * kPitch + k + 4 * t);
        uint32_t ah[2][4], al[2][4];
        split_tf32(a0.x, ah[0][0], al[0][0]);
        split_tf32(a1.x, ah[0][1], al[0][1]);
        split_tf32(a0.y, ah[0][2], al[0][2]);
        split_tf32(a1.y, ah[0][3], al[0][3]);
        split_tf32(a0.z, ah[1][0], al[1][0]);
        split_tf32(a1.z, ah[1][1], al[1][1]);
        split_tf32(a0.w, ah[1][2], al[1][2]);
        split_tf32(a1.w, ah[1][3], al[1][3]);
#pragma unroll
        for (int j0 = 0; j0 < NT / 8; j0 += 4) {
            uint32_t bh[2][4][2], bl[2][4][2];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float4 x = *reinterpret_cast<const float4*>(b + (8 * (j0 + j) + g) * kPitch + k + 4 * t);
                split_tf32(x.x, bh[0][j][0], bl[0][j][0]);
                split_tf32(x.y, bh[0][j][1], bl[0][j][1]);
                split_tf32(x.z, bh[1][j][0], bl[1][j][0]);
                split_tf32(x.w, bh[1][j][1], bl[1][j][1]);
            }
            mma_split<4>(s + j0, small + j0, ah[0], al[0], bh[0], bl[0]);
            mma_split<4>(s + j0, small + j0, ah[1], al[1], bh[1], bl[1]);
        }
    }
    bool bad = false;
#pragma unroll
    for (int j = 0; j < NT / 8; ++j)
#pragma unroll
        for (int y = 0; y < 4; ++y) {
            s[j][y] += small[j][y];
            if (CHECK) bad = bad || s[j][y] != s[j][y];
        }
    // An infinity (or a number that TF32 rounds to one) has no low part, inf - inf, and its products with a low part of
    // zero are none either. A warp that found one forms its scores in plain float32.
    if (!CHECK || !__any_sync(0xffffffffu, bad)) return;
    float plain[NT / 2];  // in local memory, so that this seldom taken way is short
#pragma unroll 1
    for (int i = 0; i < NT / 2; ++i) {
        const float *x = a + (g + 8 * (i >> 1 & 1)) * kPitch, *z = b + (8 * (i >> 2) + 2 * t + (i & 1)) * kPitch;
        float sum = 0.f;
#pragma unroll 1
        for (int k = 0; k < DP; ++k) sum = fmaf(x[k], z[k], sum);
        plain[i] = sum;
    }
#pragma unroll
    for (int i = 0; i < NT / 2; ++i) s[i / 4][i % 4] = plain[i];
}

// o[i] += p . rows of b, columns 8 i ..
template <int DP, int NT>
__device__ __forceinline__ void tf32_product(const float (&p)[NT / 8][4], const float* b, int g, int t,
                                             float (&o)[DP / 8][4]) {
    constexpr int kPitch = DP + 4;
#pragma unroll
    for (int i0 = 0; i0 < DP / 8; i0 += 4) {
        float big[4][4], small[4][4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int y = 0; y < 4; ++y) big[i][y] = small[i][y] = 0.f;
#pragma unroll
        for (int j = 0; j < NT / 8; ++j) {
            uint32_t ah[4], al[4], bh[4][2], bl[4][2];
            split_tf32(p[j][0], ah[0], al[0]);
            split_tf32(p[j][2], ah[1], al[1]);
            split_tf32(p[j][1], ah[2], al[2]);
            split_tf32(p[j][3], ah[3], al[3]);
            const float* rows = b + (8 * j + 2 * t) * kPitch + g;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                split_tf32(rows[8 * (i0 + i)], bh[i][0], bl[i][0]);
                split_tf32(rows[kPitch + 8 * (i0 + i)], bh[i][1], bl[i][1]);
            }
            mma_split<4>(big, small, ah, al, bh, bl);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int y = 0; y < 4; ++y) o[i0 + i][y] += big[i][y] + small[i][y];
    }
}

// A block takes 64 queries of one head and the keys of one split. grid as attn_simt_forward_kernel's.
template <int DP, int NT>
__global__ void __launch_bounds__(kTf32Threads, kTf32Ctas<DP, false>)
    attn_tf32_forward_kernel(const SplitArgs args) {
    using Lay = Tf32Layout<DP, NT>;
    const AttnArgs& a = args.a;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    float* qs = reinterpret_cast<float*>(smem_raw);
    auto tile = [&](int buf, int which) { return qs + Lay::kFixed + (2 * buf + which) * Lay::kTile; };
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
    const int split = blockIdx.x % args.splits, x = blockIdx.x / args.splits;
    const int i0 = x % args.row_tiles * kTf32Rows, bh = x / args.row_tiles, h = bh % a.H, b = bh / a.H;
    const int hk = h / (a.H / a.Hk), off = a.N - a.Q;
    const float c = float(a.scale * 1.4426950408889634);
    const float* k = static_cast<const float*>(a.k) + b * a.k_b + hk * a.k_h;
    const float* v = static_cast<const float*>(a.v) + b * a.v_b + hk * a.v_h;
    const uint8_t* pad = a.padding == nullptr ? nullptr : a.padding + (long long)b * a.N;
    const uint8_t* mask = a.mask == nullptr ? nullptr : a.mask + b * a.m_b + h * a.m_h;
    grid_dependency_wait();
    launch_dependents();
    const int first = split * args.split_keys;
    const int end = min((long long)attn_key_end(a, i0 + kTf32Rows), (long long)first + args.split_keys);
    tf32_load<DP, kTf32Rows>(qs, static_cast<const float*>(a.q) + b * a.q_b + h * a.q_h, a.q_t, i0, a.Q, a.D, nullptr);
    auto fetch = [&](int j0, int buf) {
        if (j0 < end) {
            tf32_load<DP, NT>(tile(buf, 0), k, a.k_t, j0, a.N, a.D, pad);
            tf32_load<DP, NT>(tile(buf, 1), v, a.v_t, j0, a.N, a.D, pad);
        }
        copy_commit();
    };
    fetch(first, 0);
    const int row[2] = {i0 + 16 * warp + g, i0 + 16 * warp + g + 8};
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, o[DP / 8][4];
#pragma unroll
    for (int i = 0; i < DP / 8; ++i)
#pragma unroll
        for (int y = 0; y < 4; ++y) o[i][y] = 0.f;
    int buf = 0;
    for (int j0 = first; j0 < end; j0 += NT, buf ^= 1) {
        fetch(j0 + NT, buf ^ 1);
        copy_wait<1>();
        __syncthreads();
        float s[NT / 8][4];
        tf32_scores<DP, NT, true>(qs + 16 * warp * Lay::kPitch, tile(buf, 0), g, t, s);
        const bool plain = mask == nullptr && pad == nullptr && j0 + NT <= a.N &&
                           (!a.causal || j0 + NT - 1 <= i0 + off);
        float keep[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float top = m[e];
#pragma unroll
            for (int j = 0; j < NT / 8; ++j)
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    float& sv = s[j][2 * e + y];
                    sv *= c;
                    if (!plain) {
                        const int key = j0 + 8 * j + 2 * t + y;
                        if (row[e] >= a.Q || key >= a.N ||
                            !attn_open(a, mask == nullptr ? nullptr : mask + row[e] * a.m_q, pad, row[e], key))
                            sv = -INFINITY;
                    }
                    top = fmaxf(top, sv);
                }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const float ref = top == -INFINITY ? 0.f : top;
            keep[e] = exp2f(m[e] - ref);
            m[e] = top;
            float sum = 0.f;
#pragma unroll
            for (int j = 0; j < NT / 8; ++j)
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    s[j][2 * e + y] = exp2f(s[j][2 * e + y] - ref);
                    sum += s[j][2 * e + y];
                }
            l[e] = l[e] * keep[e] + sum;
        }
#pragma unroll
        for (int i = 0; i < DP / 8; ++i) {
            o[i][0] *= keep[0]; o[i][1] *= keep[0]; o[i][2] *= keep[1]; o[i][3] *= keep[1];
        }
        tf32_product<DP, NT>(s, tile(buf, 1), g, t, o);
        __syncthreads();  // the buffer has been read
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
        l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
        if (row[e] >= a.Q) continue;
        const long long r = (long long)bh * a.Q + row[e], at = r * args.splits + split;
        const float inv = l[e] == 0.f ? 0.f : 1.f / l[e];
#pragma unroll
        for (int i = 0; i < DP / 8; ++i)
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                const int d = 8 * i + 2 * t + y;
                if (d >= a.D) continue;
                if (args.splits == 1) attn_store<float, float>(a, r, d, o[i][2 * e + y], inv);
                else static_cast<float*>(args.part_o)[at * a.D + d] = o[i][2 * e + y];
            }
        if (t != 0) continue;
        if (args.splits == 1) {
            attn_store_lse<float>(a, r, m[e], l[e]);
        } else {
            static_cast<float*>(args.part_ml)[2 * at] = m[e];
            static_cast<float*>(args.part_ml)[2 * at + 1] = l[e];
        }
    }
    copy_wait<0>();
}

// The gradients, blocks as in attn_simt_backward_kernel: below kv_blocks 64 keys of a key head over its query heads and
// their queries, the others 64 queries of a head over the keys.
template <int DP, int NT, bool KEYS>
__device__ __forceinline__ void attn_tf32_backward_block(const AttnArgs& a, int block, float* smem) {
    using Lay = Tf32Layout<DP, NT>;
    float *fix1 = smem, *fix2 = smem + Lay::kFixed, *stats = smem + 2 * Lay::kFixed + 4 * Lay::kTile;
    auto tile = [&](int buf, int which) { return smem + 2 * Lay::kFixed + (2 * buf + which) * Lay::kTile; };
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
    const int group = a.H / a.Hk, off = a.N - a.Q;
    const float c = float(a.scale * 1.4426950408889634), scale = float(a.scale);
    const int heads = KEYS ? a.Hk : a.H, rows = KEYS ? a.N : a.Q;
    const int tiles = (rows + kTf32Rows - 1) / kTf32Rows;
    const int splits = KEYS ? a.k_splits : a.q_splits, split = block % splits;
    block /= splits;
    const int r0 = block % tiles * kTf32Rows, head = block / tiles % heads, b = block / tiles / heads;
    const int hk = KEYS ? head : head / group, h0 = KEYS ? head * group : head, h1 = KEYS ? h0 + group : h0 + 1;
    const float* q = static_cast<const float*>(a.q) + b * a.q_b;
    const float* k = static_cast<const float*>(a.k) + b * a.k_b + hk * a.k_h;
    const float* v = static_cast<const float*>(a.v) + b * a.v_b + hk * a.v_h;
    const float* go = static_cast<const float*>(a.grad_out) + (long long)b * a.Q * a.H * a.D;
    const long long go_t = (long long)a.H * a.D;
    const uint8_t* pad = a.padding == nullptr ? nullptr : a.padding + (long long)b * a.N;
    const int c0 = KEYS && a.causal ? max(0, min(a.Q, r0 - off)) / NT * NT : 0;
    const int c1 = KEYS ? a.Q : attn_key_end(a, r0 + kTf32Rows);
    if (KEYS) {
        tf32_load<DP, kTf32Rows>(fix1, k, a.k_t, r0, a.N, a.D, pad);
        tf32_load<DP, kTf32Rows>(fix2, v, a.v_t, r0, a.N, a.D, pad);
    } else {
        tf32_load<DP, kTf32Rows>(fix1, q + h0 * a.q_h, a.q_t, r0, a.Q, a.D, nullptr);
        tf32_load<DP, kTf32Rows>(fix2, go + (long long)h0 * a.D, go_t, r0, a.Q, a.D, nullptr);
    }
    auto fetch = [&](int h, int col, int buf) {
        if (KEYS) {
            tf32_load<DP, NT>(tile(buf, 0), q + h * a.q_h, a.q_t, col, a.Q, a.D, nullptr);
            tf32_load<DP, NT>(tile(buf, 1), go + (long long)h * a.D, go_t, col, a.Q, a.D, nullptr);
            if (threadIdx.x < NT / 2) {  // lse, then delta, of the tile's queries (rows of Qp, a multiple of the tile)
                const int which = threadIdx.x / (NT / 4), at = threadIdx.x % (NT / 4) * 4;
                const float* src = static_cast<const float*>(which == 0 ? a.lse : a.delta);
                copy16(smem_addr(stats + (2 * buf + which) * NT + at),
                       src + ((long long)b * a.H + h) * a.Qp + col + at, true);
            }
        } else {
            tf32_load<DP, NT>(tile(buf, 0), k, a.k_t, col, a.N, a.D, pad);
            tf32_load<DP, NT>(tile(buf, 1), v, a.v_t, col, a.N, a.D, pad);
        }
    };
    const int row[2] = {r0 + 16 * warp + g, r0 + 16 * warp + g + 8};
    float lse[2], delta[2];
    if (!KEYS)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const long long at = ((long long)b * a.H + h0) * a.Qp + row[e];
            lse[e] = static_cast<const float*>(a.lse)[at];
            delta[e] = static_cast<const float*>(a.delta)[at];
        }
    float acc[DP / 8][4], acc2[KEYS ? DP / 8 : 1][4];
#pragma unroll
    for (int i = 0; i < DP / 8; ++i)
#pragma unroll
        for (int y = 0; y < 4; ++y) {
            acc[i][y] = 0.f;
            if constexpr (KEYS) acc2[i][y] = 0.f;
        }
    const int cols = c1 > c0 ? (c1 - c0 + NT - 1) / NT : 0;
    const long long work = (long long)cols * (h1 - h0);
    const int from = int(work * split / splits), total = int(work * (split + 1) / splits) - from;
    int h = cols > 0 ? h0 + from / cols : h0, col = cols > 0 ? c0 + from % cols * NT : c0;
    if (total > 0) fetch(h, col, 0);
    copy_commit();
    for (int n = 0; n < total; ++n) {
        const int buf = n & 1;
        int next_h = h, next = col + NT;
        if (next >= c1) {
            next = c0;
            ++next_h;
        }
        if (n + 1 < total) fetch(next_h, next, buf ^ 1);
        copy_commit();
        copy_wait<1>();
        __syncthreads();
        float p[NT / 8][4], s[NT / 8][4];
        tf32_scores<DP, NT, true>(fix1 + 16 * warp * Lay::kPitch, tile(buf, 0), g, t, p);
        tf32_scores<DP, NT, false>(fix2 + 16 * warp * Lay::kPitch, tile(buf, 1), g, t, s);
        const uint8_t* mask = a.mask == nullptr ? nullptr : a.mask + b * a.m_b + h * a.m_h;
        // (the queries behind the last, which are zeros, do not count: an infinite key makes NaN of them)
        const bool plain = mask == nullptr && (KEYS || pad == nullptr) && col + NT <= (KEYS ? a.Q : a.N) &&
                           (!a.causal || (KEYS ? r0 + kTf32Rows - 1 <= col + off : col + NT - 1 <= r0 + off));
        const float* st = stats + 2 * buf * NT;
#pragma unroll
        for (int j = 0; j < NT / 8; ++j)
#pragma unroll
            for (int y = 0; y < 4; ++y) {
                const int e = y >> 1, cc = 8 * j + 2 * t + (y & 1);
                const float li = KEYS ? st[cc] : lse[e], di = KEYS ? st[NT + cc] : delta[e];
                bool open = true;
                if (!plain) {
                    const int i = KEYS ? col + cc : row[e], key = KEYS ? row[e] : col + cc;
                    open = i < a.Q && key < a.N &&
                           attn_open(a, mask == nullptr ? nullptr : mask + i * a.m_q, KEYS ? nullptr : pad, i, key);
                }
                // (lse is +infinity in the rows behind the last query)
                p[j][y] = open ? exp2f(p[j][y] * c - li) : 0.f;
                s[j][y] = open ? p[j][y] * (s[j][y] - di) : 0.f;
            }
        if constexpr (KEYS) tf32_product<DP, NT>(p, tile(buf, 1), g, t, acc2);
        tf32_product<DP, NT>(s, tile(buf, 0), g, t, acc);
        __syncthreads();
        h = next_h;
        col = next;
    }
    copy_wait<0>();
    const long long size = (long long)a.B * rows * heads * a.D;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        if (row[e] >= rows) continue;
        const bool gone = KEYS && pad != nullptr && pad[row[e]] != 0;
        const long long at = KEYS ? (((long long)b * a.N + row[e]) * a.Hk + hk) * a.D
                                  : (((long long)b * a.Q + row[e]) * a.H + h0) * a.D;
#pragma unroll
        for (int i = 0; i < DP / 8; ++i)
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                const int d = 8 * i + 2 * t + y;
                if (d >= a.D) continue;
                const float x = gone ? 0.f : acc[i][2 * e + y] * scale;
                if constexpr (KEYS) {
                    const float x2 = gone ? 0.f : acc2[i][2 * e + y];
                    attn_put_grad<float>(a.grad_k, a.part_k, splits, split, size, at + d, x);
                    attn_put_grad<float>(a.grad_v, a.part_v, splits, split, size, at + d, x2);
                } else {
                    attn_put_grad<float>(a.grad_q, a.part_q, splits, split, size, at + d, x);
                }
            }
    }
}

template <int DP, int NT>
__global__ void __launch_bounds__(kTf32Threads, kTf32Ctas<DP, true>)
    attn_tf32_backward_kernel(const AttnArgs a, int kv_blocks) {
    extern __shared__ __align__(16) unsigned char smem_raw[];
    float* smem = reinterpret_cast<float*>(smem_raw);
    grid_dependency_wait();
    launch_dependents();
    if (int(blockIdx.x) < kv_blocks) attn_tf32_backward_block<DP, NT, true>(a, int(blockIdx.x), smem);
    else attn_tf32_backward_block<DP, NT, false>(a, int(blockIdx.x) - kv_blocks, smem);
}

}  // namespace td
