// td_attention_split.cuh -- attention of few queries over many keys (one new token, some tracked objects): the keys of
// a head are split over CTAs, each of which leaves a partial softmax, and attn_combine_kernel joins them.
//
// Partial of a row over a set of keys: m = max S, l = sum exp2(S - m), o = sum exp2(S - m) v. Two sets join to
// M = max(m1, m2), l = l1 exp2(m1 - M) + l2 exp2(m2 - M), o likewise; a set without an open key is (-inf, 0, 0). The
// sets and their order follow from the sizes alone, so the result is the same every time.
//
// Bound by reading K and V once, from HBM. A tile has 16 rows: the queries of a key head's whole group of query heads,
// so shared keys are read once for all of them. Each warp streams its own keys through a ring of its own in shared
// memory (asynchronous 16-byte copies, two steps ahead, nothing shared between warps until the end) into mma.sync
// fragments: the order of the summed index is free, so a thread's 8 consecutive elements of a key row are two K steps'
// fragments (the queries are loaded in the same order), and a thread's consecutive elements of a value row are the
// same column of as many 8-wide result tiles; the pairs of keys that a value fragment packs are made with byte
// permutes. Tensor cores matter little here, but a 16-row product on them costs what a one-row product on CUDA cores
// would. One query over 22223 keys, 8 images of 8 heads x 32 in bfloat16, lengths falling to half: 45 us (3.2 TB/s),
// which the latency of the twelve warps an SM sets, not the memory; loads straight into registers took 62 with P in one
// part, where these took 41.
#pragma once

#include "td_attention.cuh"

namespace td {

struct SplitArgs {
    AttnArgs a;
    int splits, split_keys;  // keys split s takes: [s * split_keys, (s + 1) * split_keys)
    int row_tiles;           // ceil(group * Q / rows of a tile)
    // partials, in the accumulator type: o [B * H * Q][splits][D], ml [B * H * Q][splits][2]; unused with one split
    void *part_o, *part_ml;
};

constexpr int kSplitWarps = 4, kSplitStages = 3;

// A warp's ring slot: keys a step, K rows then V rows, padded so that rows fall on different banks.
template <int DP>
struct SplitLayout {
    static constexpr int kKeys = DP == 128 ? 16 : 32;
    static constexpr int kPitch = DP * 2 + 16;
    static constexpr int kStage = 2 * kKeys * kPitch;
    static constexpr int kJoin = kSplitWarps * 16 * (DP + 4) * 4;  // the warps' results take the ring's place
    static constexpr int kRing = kSplitWarps * kSplitStages * kStage;
    static constexpr size_t kSmem = kRing > kJoin ? kRing : kJoin;
};

// The result's row `row` (of B * H * Q, head-major): o / l rounded, what the rounding took, and lse.
template <typename T, typename A>
__device__ __forceinline__ void attn_store(const AttnArgs& a, long long row, int d, A o, A inv) {
    const long long bh = row / a.Q, i = row % a.Q;
    const long long at = ((bh / a.H * a.Q + i) * a.H + bh % a.H) * a.D + d;
    const T rounded = from_acc<T>(o * inv);
    static_cast<T*>(a.out)[at] = rounded;
    if (a.rest != nullptr) static_cast<T*>(a.rest)[at] = from_acc<T>(o * inv - to_acc(rounded));
}
template <typename A>
__device__ __forceinline__ void attn_store_lse(const AttnArgs& a, long long row, A m, A l) {
    if (a.lse == nullptr) return;
    A* lse = static_cast<A*>(a.lse) + row / a.Q * a.Qp;
    const int i = int(row % a.Q);
    lse[i] = l == A(0) ? A(INFINITY) : m + attn_log2<A>(l);
    if (i == a.Q - 1)  // the rows behind the last query
        for (int x = a.Q; x < a.Qp; ++x) lse[x] = A(INFINITY);
}

// D += A x B, 16 x 8 x 16, float32 accumulators.
template <typename T>
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma_16816<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma_16816<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                                         uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float fast_exp2(float x) {  // 2 ulp
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <typename T> __device__ __forceinline__ uint32_t pack_pair(float lo, float hi) {
    const T v[2] = {from_acc<T>(lo), from_acc<T>(hi)};
    return *reinterpret_cast<const uint32_t*>(v);
}

// DP: 32, 64 or 128, D <= DP a multiple of 8. P goes through its product in two 16-bit parts, as in
// attn_tc_forward_kernel: two more products on data at hand, next to what the keys' way here takes. grid: splits x row
// tiles x key heads x images, splits fastest.
template <typename T, int DP>
__global__ void __launch_bounds__(kSplitWarps * 32) attn_split_kernel(const SplitArgs args) {
    using Lay = SplitLayout<DP>;
    constexpr int kKeys = Lay::kKeys;               // keys a warp takes at a time
    constexpr int kChunks = DP / 32;                // 16-byte pieces a thread has of a key row
    constexpr int kDims = DP / 8;                   // columns a thread has of a value row
    constexpr int kG = kKeys / 16;
    const AttnArgs& a = args.a;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    float (*sm_o)[16][DP + 4] = reinterpret_cast<float (*)[16][DP + 4]>(smem_raw);
    __shared__ float sm_ml[kSplitWarps][16][2];
    __shared__ uint32_t sm_live[kSplitWarps][kSplitStages];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
    const int group = a.H / a.Hk, rows = group * a.Q;
    int x = blockIdx.x;
    const int split = x % args.splits;
    x /= args.splits;
    const int r0 = x % args.row_tiles * 16;
    x /= args.row_tiles;
    const int hk = x % a.Hk, b = x / a.Hk;
    const float c = float(a.scale * 1.4426950408889634);
    grid_dependency_wait();
    launch_dependents();

    // rows r0 + g and r0 + g + 8 of the group: query (row % Q) of head hk * group + row / Q
    uint32_t q[2][kChunks][4];
    int qi[2];
    const uint8_t* mask_row[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const int r = r0 + g + 8 * e;
        const bool in = r < rows;
        const int h = hk * group + (in ? r / a.Q : 0);
        qi[e] = in ? r % a.Q : 0;
        mask_row[e] = a.mask == nullptr ? nullptr : a.mask + b * a.m_b + h * a.m_h + qi[e] * a.m_q;
        const T* src = static_cast<const T*>(a.q) + b * a.q_b + h * a.q_h + qi[e] * a.q_t;
#pragma unroll
        for (int k = 0; k < kChunks; ++k) {
            uint4 v = make_uint4(0u, 0u, 0u, 0u);
            if (in && 32 * k + 8 * t < a.D) v = __ldg(reinterpret_cast<const uint4*>(src + 32 * k + 8 * t));
            q[e][k][0] = v.x; q[e][k][1] = v.y; q[e][k][2] = v.z; q[e][k][3] = v.w;
        }
    }
    const T* kp = static_cast<const T*>(a.k) + b * a.k_b + hk * a.k_h;
    const T* vp = static_cast<const T*>(a.v) + b * a.v_b + hk * a.v_h;
    const uint8_t* pad = a.padding == nullptr ? nullptr : a.padding + (long long)b * a.N;
    const int off = a.N - a.Q;
    const int end = int(min((long long)attn_key_end(a, a.Q), (split + 1LL) * args.split_keys));

    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, o[kDims][4];
#pragma unroll
    for (int i = 0; i < kDims; ++i)
#pragma unroll
        for (int y = 0; y < 4; ++y) o[i][y] = 0.f;

    unsigned char* ring = smem_raw + warp * kSplitStages * Lay::kStage;
    constexpr int kStep = kSplitWarps * kKeys, kPieces = DP / 8;  // 16-byte pieces of a row
    const int first = split * args.split_keys + warp * kKeys;
    const int steps = first < end ? (end - first + kStep - 1) / kStep : 0;
    // a bit per key of a step: not behind the end, not padded; the padding's bytes are read a step before they are used
    auto key_there = [&](int step) {
        const int j = first + step * kStep + lane;
        return step < steps && lane < kKeys && j < end && (pad == nullptr || __ldg(pad + j) == 0);
    };
    bool there = key_there(0);
    // this lane's pieces: column c of rows r, r + kRowsPer, ..
    constexpr int kRowsPer = 32 / kPieces;
    const int pr = lane / kPieces, pc = lane % kPieces;
    const bool col = 8 * pc < a.D;
    const T* kl = kp + (long long)(first + pr) * a.k_t + (col ? 8 * pc : 0);
    const T* vl = vp + (long long)(first + pr) * a.v_t + (col ? 8 * pc : 0);
    const uint32_t dst = smem_addr(ring) + pr * Lay::kPitch + 16 * pc;
    int fill = 0;  // the ring slot the next fetch goes to
    auto fetch = [&](int step) {
        if (step < steps) {
            const uint32_t all = __ballot_sync(0xffffffffu, there), live = all >> pr;
            there = key_there(step + 1);
            if (lane == 0) sm_live[warp][fill] = all;
            const uint32_t to = dst + fill * Lay::kStage;
            fill = fill == kSplitStages - 1 ? 0 : fill + 1;
#pragma unroll
            for (int i = 0; i < kKeys / kRowsPer; ++i) {
                const bool real = col && ((live >> (i * kRowsPer)) & 1u) != 0;
                copy16(to + i * kRowsPer * Lay::kPitch, real ? kl + i * kRowsPer * a.k_t : kp, real);
                copy16(to + (kKeys + i * kRowsPer) * Lay::kPitch, real ? vl + i * kRowsPer * a.v_t : vp, real);
            }
            kl += kStep * a.k_t;
            vl += kStep * a.v_t;
        }
        copy_commit();
    };
    const bool both = rows - r0 > 8;  // whether the tile has rows 8 .. 15
    int slot = 0;
#pragma unroll
    for (int step = 0; step < kSplitStages - 1; ++step) fetch(step);
    for (int step = 0; step < steps; ++step) {
        __syncwarp();  // the slot's last readers are done
        fetch(step + kSplitStages - 1);
        copy_wait<kSplitStages - 1>();
        __syncwarp();
        const int j0 = first + step * kStep;
        const uint32_t live = sm_live[warp][slot];
        const unsigned char* ks = ring + slot * Lay::kStage;
        slot = slot == kSplitStages - 1 ? 0 : slot + 1;
        if (live == 0) continue;
        const unsigned char* vs = ks + kKeys * Lay::kPitch;
        uint4 kv[2 * kG][kChunks];
        uint32_t vv[4 * kG][kDims / 2];
#pragma unroll
        for (int u = 0; u < 2 * kG; ++u)  // keys g, g + 8, ..
#pragma unroll
            for (int k = 0; k < kChunks; ++k)
                kv[u][k] = *reinterpret_cast<const uint4*>(ks + (8 * u + g) * Lay::kPitch + 64 * k + 16 * t);
#pragma unroll
        for (int u = 0; u < 4 * kG; ++u) {  // keys 2 t, 2 t + 1, 2 t + 8, 2 t + 9 of each 16
            const int key = 16 * (u / 4) + 8 * ((u >> 1) & 1) + 2 * t + (u & 1);
            if constexpr (DP == 32) {
                const uint2 w = *reinterpret_cast<const uint2*>(vs + key * Lay::kPitch + 8 * g);
                vv[u][0] = w.x; vv[u][1] = w.y;
            } else {
#pragma unroll
                for (int k = 0; k < DP / 64; ++k) {
                    const uint4 w = *reinterpret_cast<const uint4*>(vs + key * Lay::kPitch + 128 * k + 16 * g);
                    vv[u][4 * k] = w.x; vv[u][4 * k + 1] = w.y; vv[u][4 * k + 2] = w.z; vv[u][4 * k + 3] = w.w;
                }
            }
        }
        float s[2 * kG][4];
#pragma unroll
        for (int u = 0; u < 2 * kG; ++u) {
#pragma unroll
            for (int y = 0; y < 4; ++y) s[u][y] = 0.f;
#pragma unroll
            for (int k = 0; k < kChunks; ++k) {
                const uint32_t a0[4] = {q[0][k][0], q[1][k][0], q[0][k][1], q[1][k][1]};
                const uint32_t a1[4] = {q[0][k][2], q[1][k][2], q[0][k][3], q[1][k][3]};
                mma_16816<T>(s[u], a0, kv[u][k].x, kv[u][k].y);
                mma_16816<T>(s[u], a1, kv[u][k].z, kv[u][k].w);
            }
        }
        const bool plain = live == (kKeys == 32 ? 0xffffffffu : (1u << kKeys) - 1u) && !a.causal && a.mask == nullptr;
        float keep[2] = {1.f, 1.f}, ref[2] = {0.f, 0.f}, sum[2] = {0.f, 0.f};
#pragma unroll
        for (int e = 0; e < 2; ++e) {  // rows g, g + 8; element y of score tile u: key 8 u + 2 t + y
            if (e == 1 && !both) continue;
            float top = m[e];
#pragma unroll
            for (int u = 0; u < 2 * kG; ++u)
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    float& sv = s[u][2 * e + y];
                    sv *= c;
                    if (!plain) {
                        const int key = 8 * u + 2 * t + y, j = j0 + key;
                        bool open = ((live >> key) & 1u) != 0;
                        if (a.causal) open = open && j <= qi[e] + off;
                        if (open && mask_row[e] != nullptr) open = mask_row[e][j] == 0;
                        if (!open) sv = -INFINITY;
                    }
                    top = fmaxf(top, sv);
                }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            ref[e] = top == -INFINITY ? 0.f : top;
            keep[e] = fast_exp2(m[e] - ref[e]);
            m[e] = top;
        }
#pragma unroll
        for (int i = 0; i < kDims; ++i) {
            o[i][0] *= keep[0]; o[i][1] *= keep[0]; o[i][2] *= keep[1]; o[i][3] *= keep[1];
        }
#pragma unroll
        for (int w = 0; w < kG; ++w) {
            uint32_t p[4], rest[4];
#pragma unroll
            for (int y = 0; y < 4; ++y) {  // fragment registers: rows g, g + 8 of keys 0 .. 7, then of 8 .. 15
                const int u = 2 * w + (y >> 1), e = y & 1;
                p[y] = 0u;
                rest[y] = 0u;
                if (e == 1 && !both) continue;
                const float p0 = fast_exp2(s[u][2 * e] - ref[e]), p1 = fast_exp2(s[u][2 * e + 1] - ref[e]);
                sum[e] += p0 + p1;
                p[y] = pack_pair<T>(p0, p1);
                const T* r = reinterpret_cast<const T*>(&p[y]);
                rest[y] = pack_pair<T>(p0 - to_acc(r[0]), p1 - to_acc(r[1]));
            }
#pragma unroll
            for (int i = 0; i < kDims; i += 2) {
                const uint32_t v0 = vv[4 * w][i / 2], v1 = vv[4 * w + 1][i / 2];
                const uint32_t v2 = vv[4 * w + 2][i / 2], v3 = vv[4 * w + 3][i / 2];
                const uint32_t b0 = __byte_perm(v0, v1, 0x5410), b1 = __byte_perm(v2, v3, 0x5410);
                const uint32_t b2 = __byte_perm(v0, v1, 0x7632), b3 = __byte_perm(v2, v3, 0x7632);
                mma_16816<T>(o[i], p, b0, b1);
                mma_16816<T>(o[i + 1], p, b2, b3);
                mma_16816<T>(o[i], rest, b0, b1);
                mma_16816<T>(o[i + 1], rest, b2, b3);
            }
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) l[e] = l[e] * keep[e] + sum[e];
    }
    // the quads' sums, then the warps' partials through shared memory, joined in warp order
    copy_wait<0>();
    __syncthreads();  // the rings have been read
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
        l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
        if (t == 0) {
            sm_ml[warp][g + 8 * e][0] = m[e];
            sm_ml[warp][g + 8 * e][1] = l[e];
        }
    }
#pragma unroll
    for (int i = 0; i < kDims; ++i)
#pragma unroll
        for (int y = 0; y < 4; ++y) {  // result column n = 2 t + y % 2 of tile i: that thread group's i-th column
            const int n = 2 * t + (y & 1);
            const int d = DP == 32 ? 4 * n + i : 64 * (i / 8) + 8 * n + i % 8;
            sm_o[warp][g + 8 * (y >> 1)][d] = o[i][y];
        }
    __syncthreads();
    for (int e = threadIdx.x; e < 16 * DP; e += kSplitWarps * 32) {
        const int r = e / DP, d = e % DP;
        if (r0 + r >= rows || d >= a.D) continue;
        float top = -INFINITY, sum = 0.f, acc = 0.f;
#pragma unroll
        for (int w = 0; w < kSplitWarps; ++w) top = fmaxf(top, sm_ml[w][r][0]);
        const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int w = 0; w < kSplitWarps; ++w) {
            const float f = exp2f(sm_ml[w][r][0] - ref);
            sum += sm_ml[w][r][1] * f;
            acc += sm_o[w][r][d] * f;
        }
        const int h = hk * group + (r0 + r) / a.Q;
        const long long row = ((long long)b * a.H + h) * a.Q + (r0 + r) % a.Q;
        if (args.splits == 1) {
            attn_store<T, float>(a, row, d, acc, sum == 0.f ? 0.f : 1.f / sum);
            if (d == 0) attn_store_lse<float>(a, row, top, sum);
        } else {
            const long long at = row * args.splits + split;
            static_cast<float*>(args.part_o)[at * a.D + d] = acc;
            if (d == 0) {
                static_cast<float*>(args.part_ml)[2 * at] = top;
                static_cast<float*>(args.part_ml)[2 * at + 1] = sum;
            }
        }
    }
}

// Joins the partials of a row by W of a block's 8 warps: warp w of a row adds splits w, w + W, .. (their loads in
// flight together), then the warps' sums are added in order. Eight for few rows of many splits, one for many rows.
constexpr int kCombineWarps = 8;
template <typename T, int W>
__global__ void __launch_bounds__(kCombineWarps * 32) attn_combine_kernel(const SplitArgs args) {
    using A = typename Elem<T>::acc;
    const AttnArgs& a = args.a;
    const int warp = threadIdx.x / 32 % W, lane = threadIdx.x % 32;
    const long long row = (long long)blockIdx.x * (kCombineWarps / W) + threadIdx.x / (32 * W);
    grid_dependency_wait();
    launch_dependents();
    if (row >= (long long)a.B * a.H * a.Q) return;  // whole warps, and whole blocks where they meet below
    const A* ml = static_cast<const A*>(args.part_ml) + row * args.splits * 2;
    const A* po = static_cast<const A*>(args.part_o) + row * args.splits * a.D;
    A top = -A(INFINITY), sum = 0;
    for (int s = lane; s < args.splits; s += 32) top = cmax(top, ml[2 * s]);
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) top = cmax(top, __shfl_xor_sync(0xffffffffu, top, x));
    const A ref = top == -A(INFINITY) ? A(0) : top;
    for (int s = lane; s < args.splits; s += 32) sum += ml[2 * s + 1] * attn_exp2<A>(ml[2 * s] - ref);
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
    const A inv = sum == A(0) ? A(0) : A(1) / sum;
    __shared__ A part[W > 1 ? W : 1][W > 1 ? kAttnMaxHeadDim : 1];
    for (int d = lane; d < a.D; d += 32) {
        A o = 0;
#pragma unroll 4
        for (int s = warp; s < args.splits; s += W) o += po[(long long)s * a.D + d] * attn_exp2<A>(ml[2 * s] - ref);
        if constexpr (W > 1) part[warp][d] = o;
        else attn_store<T, A>(a, row, d, o, inv);
    }
    if constexpr (W > 1) {
        static_assert(W == kCombineWarps, "a row is a block");
        __syncthreads();
        for (int d = threadIdx.x; d < a.D; d += W * 32) {
            A o = 0;
#pragma unroll
            for (int w = 0; w < W; ++w) o += part[w][d];
            attn_store<T, A>(a, row, d, o, inv);
        }
    }
    if (warp == 0 && lane == 0) attn_store_lse<A>(a, row, top, sum);
}

// ---- CUDA-core forward: every type and head width (see td_attention.cuh) ------------------------------------------
// A block takes 16 RM queries of one head and the keys of one split. grid: splits x query tiles x heads x images,
// splits fastest.
template <typename T, int DP, int RM, int RN>
__global__ void __launch_bounds__(256) attn_simt_forward_kernel(const SplitArgs args) {
    using A = typename Elem<T>::acc;
    using Tile = SimtTile<A, DP, RM, RN>;
    constexpr int M = Tile::kRows, KN = Tile::kCols;
    const AttnArgs& a = args.a;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    A* qs = reinterpret_cast<A*>(smem_raw);
    A* ks = qs + M * Tile::kLd;
    A* vs = ks + KN * Tile::kLd;
    A* ps = vs + KN * Tile::kLd;
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    const int split = blockIdx.x % args.splits, tile = blockIdx.x / args.splits;
    const int i0 = tile % args.row_tiles * M, bh = tile / args.row_tiles, h = bh % a.H, b = bh / a.H;
    const int hk = h / (a.H / a.Hk);
    const A ninf = -A(INFINITY), c = A(a.scale * 1.4426950408889634);
    const uint8_t* pad = a.padding == nullptr ? nullptr : a.padding + (long long)b * a.N;
    const uint8_t* mask = a.mask == nullptr ? nullptr : a.mask + b * a.m_b + h * a.m_h;
    grid_dependency_wait();
    launch_dependents();
    simt_load<T, A, DP, M>(qs, static_cast<const T*>(a.q) + b * a.q_b + h * a.q_h, a.q_t, i0, a.Q, a.D, nullptr,
                            a.vec_q != 0);
    A m[RM], l[RM], o[RM][Tile::kWidth];
#pragma unroll
    for (int r = 0; r < RM; ++r) {
        m[r] = ninf;
        l[r] = 0;
#pragma unroll
        for (int x = 0; x < Tile::kWidth; ++x) o[r][x] = 0;
    }
    const int key_end = min((long long)attn_key_end(a, i0 + M), (long long)(split + 1) * args.split_keys);
    for (int j0 = split * args.split_keys; j0 < key_end; j0 += KN) {
        __syncthreads();  // the tiles of the turn before have been read
        simt_load<T, A, DP, KN>(ks, static_cast<const T*>(a.k) + b * a.k_b + hk * a.k_h, a.k_t, j0, a.N, a.D, pad,
                                 a.vec_k != 0);
        simt_load<T, A, DP, KN>(vs, static_cast<const T*>(a.v) + b * a.v_b + hk * a.v_h, a.v_t, j0, a.N, a.D, pad,
                                 a.vec_v != 0);
        __syncthreads();
        A s[RM][RN];
        simt_dot<A, DP, RM, RN>(qs, ks, ty, tx, s);
#pragma unroll
        for (int r = 0; r < RM; ++r) {
            const int i = i0 + ty + 16 * r;
            A top = m[r];
#pragma unroll
            for (int x = 0; x < RN; ++x) {
                const int j = j0 + tx + 16 * x;
                const bool open = i < a.Q && j < a.N &&
                                  attn_open(a, mask == nullptr ? nullptr : mask + i * a.m_q, pad, i, j);
                s[r][x] = open ? s[r][x] * c : ninf;
                top = cmax(top, s[r][x]);
            }
            top = row_max(top);
            const A ref = top == ninf ? A(0) : top;  // no key so far: exp2(-inf - 0) = 0
            const A keep = attn_exp2<A>(m[r] - ref);
            A sum = 0;
#pragma unroll
            for (int x = 0; x < RN; ++x) {
                s[r][x] = attn_exp2<A>(s[r][x] - ref);
                sum += s[r][x];
                ps[(ty + 16 * r) * Tile::kLdP + tx + 16 * x] = s[r][x];
            }
            l[r] = l[r] * keep + row_sum(sum);
            m[r] = top;
#pragma unroll
            for (int x = 0; x < Tile::kWidth; ++x) o[r][x] *= keep;
        }
        __syncwarp();  // a row's P is written and read by the same half warp
        simt_accumulate<A, DP, RM, RN>(ps, vs, ty, tx, o);
    }
#pragma unroll
    for (int r = 0; r < RM; ++r) {
        const int i = i0 + ty + 16 * r;
        if (i >= a.Q) continue;
        const long long row = (long long)bh * a.Q + i, at = row * args.splits + split;
        const A inv = l[r] == A(0) ? A(0) : A(1) / l[r];
#pragma unroll
        for (int x = 0; x < Tile::kWidth; ++x) {
            const int d = tx + 16 * x;
            if (d >= a.D) continue;
            if (args.splits == 1) attn_store<T, A>(a, row, d, o[r][x], inv);
            else static_cast<A*>(args.part_o)[at * a.D + d] = o[r][x];
        }
        if (tx != 0) continue;
        if (args.splits == 1) {
            attn_store_lse<A>(a, row, m[r], l[r]);
        } else {
            static_cast<A*>(args.part_ml)[2 * at] = m[r];
            static_cast<A*>(args.part_ml)[2 * at + 1] = l[r];
        }
    }
}

}  // namespace td
