// td_attention_tc.cuh -- attention on tcgen05 tensor cores, float16 and bfloat16 (the mathematics: td_attention.cuh).
//
// Every product is a tcgen05.mma of 128 rows (TMEM lanes) whose elementwise work one thread does per row:
//   forward          S = Q K^T (lanes = queries), P = exp2 over it, O += P V
//   queries' grad    S = Q K^T, dP = dO V^T (lanes = queries), dS = P (dP - delta), dQ += dS K
//   keys' grad       S^T = K Q^T, dP^T = V dO^T (lanes = keys), dV += P^T dO, dK += dS^T Q
// so a 128-row operand stays in shared memory (K-major), tiles of 64 rows of the other side stream through a ring of
// TMA slots, and each streamed tile serves as a K-major operand of one product and as an MN-major operand of another. P
// and dS are written back to TMEM over the scores they came from, as the A operand of the next product: neither ever
// reaches shared memory. The products take 16 bits, so both are kept in two parts, a rounding and what that took (in
// the room that float32 scores leave), and each part goes through the product: with float32 sums, the results' own
// roundings are the only ones to 16 bits. P and dS rounded once put the gradients 1.4 times as far from float64, in
// three quarters of the time (encoder backward below: 489 us; grouped: 96). The two gradients are separate blocks of
// one launch, each of which forms S and dP itself: 7 products instead of 5 and twice the exponentials, but every sum
// has one owner and one order (no atomics, and no float32 gradient in memory but where a few long rows of work are
// shared by several CTAs, whose partial sums are then joined in order).
//
// Columns past D (D < DP) and rows past the last token are zero through the tensor maps' fill. Scores of closed pairs
// are replaced by -infinity (P, dS by zero); tiles without an open pair are skipped by every role alike, from one
// flag byte per tile (attn_pack_kernel), and tiles whose pairs are all open skip the tests. Rows of padded keys, which
// may hold anything, are cleared in shared memory where they are summed over (V in the forward, K in the queries'
// gradient): zero times infinity is no zero.
//
// What bounds them is the time a tile takes through its stations rather than any unit: barrier, product, commit and
// TMEM latencies and, in the elementwise warps, instructions that wait for one another. So the forward runs two CTAs an
// SM (256 TMEM columns each) with the next scores formed meanwhile, the backward two elementwise warpgroups over two or
// three score buffers; products of scores and of P, dS are issued by a warp each, which overlaps their waits (827 to
// 598 us for the encoder's backward, with P and dS in one part); everything between two tiles is kept short. Measured:
// 2 x 4096 tokens, 16 / 4 heads x 64, causal, bfloat16: 146 us (472 TFLOP/s; issue slots 51 % busy, the tcgen05 pipe 58
// %). 8400 tokens, 8 heads x 32 (the encoder's): forward 300 us, backward 675 (268 TFLOP/s of the products that P and
// dS in one part would take; issue slots 55 %, the pipe 59 %). 2 x 2047, 8 / 2 heads x 128, causal, float16: forward 49
// us, backward 125 (343 TFLOP/s; 33 and 61 %).
#pragma once

#include <type_traits>

#include "td_attention.cuh"
#include "td_ptx.cuh"

namespace td {

struct AttnTcArgs {
    AttnArgs a;
    // forward and queries' gradient: open-pair bits (1 = open, N rounded up to 64 bits a row) and tile flags (bit 0:
    // some pair open, bit 1: all open) per 128 queries x 64 keys, padding included; strides 0 where shared; or null
    const uint32_t* row_bits;
    const uint8_t* row_flags;
    long long rb_b, rb_h, rb_q, rf_b, rf_h, rf_q;
    // keys' gradient: the same per key over the queries (128 keys x 64 queries), padding not included; or null
    const uint32_t* col_bits;
    const uint8_t* col_flags;
    long long cb_b, cb_h, cf_b, cf_h;
    int col_words;              // words a key's row of col_bits has
    int col_tiles;              // flags a row of col_flags has
    // float16 backward: |dO|^2 of every row [B, H, Qp]; of each (image, key head) and block of the delta kernel the
    // largest |dO|^2, then the same of |V|^2 [2][B, Hk, amax_parts]
    const float *row_g, *amax;
    int amax_parts;
    const float* keys_lse;      // backward: lse as the keys' blocks take it (see attn_p_bits)
    int kv_blocks;              // backward: blocks of the keys' gradient, launched first
    // forward: the key tiles of a query tile are shared by `splits` CTAs; with more than one these take their partial
    // results, o [B * H * Q][splits][D] and (maximum, sum) [B * H * Q][splits][2], for attn_combine_kernel
    int splits;
    float *part_o, *part_ml;
};

constexpr int kAttnBM = 128, kAttnBN = 64;

// An operand tile in shared memory: boxes of min(DP, 64) columns, rows of 64 bytes (64-byte swizzle, DP = 32) or 128
// bytes (128-byte swizzle), in atoms of 8 rows.
template <int DP>
struct AttnBox {
    static constexpr int kCols = DP < 64 ? DP : 64;
    static constexpr int kBoxes = DP / kCols;
    static constexpr uint32_t kRow = kCols * 2;
    static constexpr uint32_t kFixed = kAttnBM * kRow;  // a box of the resident operand
    static constexpr uint32_t kTile = kAttnBN * kRow;   // a box of a streamed tile
    static constexpr int kSteps = kCols / 16;           // K steps of a box
    static_assert(DP == 32 || DP == 64 || DP == 128, "head width");
};

// ---- PTX ----------------------------------------------------------------------------------------------------------
// The MMA warps stay converged: every lane forms the (equal) operands, which the compiler so keeps in uniform
// registers, and the lane with `leader` set issues. Inside a branch that one lane takes, each descriptor would be moved
// there anew, which cost more than the products: a tile's 16 took about 1100 cycles to issue.
// D[tmem] (+)= A[smem desc] x B[smem desc]^T
__device__ __forceinline__ void mma_ss(uint32_t leader, uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc,
                                       uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 q, %5, 0;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(leader)
        : "memory");
}
// D[tmem] (+)= A[tmem] x B[smem desc]: A is 128 lanes x K packed 16-bit elements, two a column.
__device__ __forceinline__ void mma_ts(uint32_t leader, uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc,
                                       uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 q, %5, 0;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(leader)
        : "memory");
}
__device__ __forceinline__ void commit(uint32_t leader, uint64_t* bar) {
    asm volatile(
        "{\n\t.reg .pred q;\n\t"
        "setp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}"
        ::"r"(smem_addr(bar)), "r"(leader)
        : "memory");
}

__device__ __forceinline__ void tmem_st_32x32b_x16(uint32_t taddr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};"
        ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
          "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_st_32x32b_x32(uint32_t taddr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};"
        ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
          "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
          "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
          "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 4-D tiled load of box (x, y, z, w), completing its bytes on the mbarrier (x * element size a multiple of 16 bytes).
__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z,
                                            int w, uint64_t pol) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint"
        " [%0], [%1, {%3, %4, %5, %6}], [%2], %7;"
        ::"r"(smem_addr(dst)), "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_addr(bar)), "r"(x), "r"(y), "r"(z),
          "r"(w), "l"(pol)
        : "memory");
}
// Plain copy of `bytes` (a multiple of 16, both addresses 16-byte aligned) into shared memory.
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
        ::"r"(smem_addr(dst)), "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes), "r"(smem_addr(bar))
        : "memory");
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Two float32 operations in one instruction (sm_100): pairs in 64-bit registers.
using F2 = unsigned long long;
__device__ __forceinline__ F2 f2(float lo, float hi) {
    F2 d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(lo), "f"(hi));
    return d;
}
__device__ __forceinline__ F2 f2(uint32_t lo, uint32_t hi) {
    F2 d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(lo), "r"(hi));
    return d;
}
__device__ __forceinline__ void f2_split(F2 a, float& lo, float& hi) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(a));
}
__device__ __forceinline__ F2 f2_fma(F2 a, F2 b, F2 c) {
    F2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ F2 f2_add(F2 a, F2 b) {
    F2 d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ F2 f2_mul(F2 a, F2 b) {
    F2 d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// Two floats rounded to T, lo in the low half.
template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

template <typename T> __device__ __forceinline__ float2 unpack2(uint32_t v);
template <> __device__ __forceinline__ float2 unpack2<__half>(uint32_t v) {
    return __half22float2(*reinterpret_cast<const __half2*>(&v));
}
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t v) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}

// Two floats in two 16-bit parts: their roundings, and the rounding of what those took.
template <typename T>
__device__ __forceinline__ void pack_parts(float x0, float x1, uint32_t& part, uint32_t& rest) {
    part = pack2<T>(x0, x1);
    const float2 r = unpack2<T>(part);
    rest = pack2<T>(x0 - r.x, x1 - r.y);
}

// All lanes of a warp wait; false in every lane if any gave up.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, unsigned int code) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, code));
}

// Calls f(tile, all pairs open by the flags) for the tiles in [t0, t1) with an open pair, in order, in whole warps,
// until f returns false. flags: one byte a tile, or null (every tile, all open).
template <typename F>
__device__ __forceinline__ bool for_tiles(int t0, int t1, const uint8_t* flags, F&& f) {
    if (flags == nullptr) {
        for (int t = t0; t < t1; ++t)
            if (!f(t, true)) return false;
        return true;
    }
    const int lane = threadIdx.x & 31;
    for (int base = t0; base < t1; base += 32) {
        const int t = base + lane;
        const unsigned fl = t >= t1 ? 0u : unsigned(__ldg(flags + t));
        unsigned any = __ballot_sync(0xffffffffu, (fl & 1u) != 0);
        const unsigned all = __ballot_sync(0xffffffffu, (fl & 2u) != 0);
        while (any != 0) {
            const int x = __ffs(int(any)) - 1;
            any &= any - 1;
            if (!f(base + x, ((all >> x) & 1u) != 0)) return false;
        }
    }
    return true;
}

// A place in a ring of N and the parity of its round, stepped instead of divided: on a warp alone on its scheduler
// every instruction between two tiles shows.
template <int N>
struct Ring {
    int at = 0;
    uint32_t parity = 0;
    __device__ __forceinline__ explicit Ring(int start = 0) : at(start) {}
    template <int STEP = 1>
    __device__ __forceinline__ void step() {
        static_assert(STEP <= N, "at most a round");
        at += STEP;
        if (at >= N) {
            at -= N;
            parity ^= 1u;
        }
    }
};

// Bits of [0, 64) below `n` (n may be negative or above 64).
__device__ __forceinline__ unsigned long long bits_below(int n) {
    return n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1ull;
}

// Instruction descriptor: f32 accumulator, A K-major, B K-major or MN-major, 128 x N.
template <typename T, bool B_MN>
__device__ __forceinline__ constexpr uint32_t attn_idesc(int N) {
    return idesc_f16(std::is_same<T, __nv_bfloat16>::value, 128, N) | (uint32_t(B_MN) << 16);
}

// K-major operand: atoms of 8 rows stacked along M / N.
template <int DP>
__device__ __forceinline__ uint64_t sdesc_k(uint32_t saddr) {
    if constexpr (DP >= 64) return sdesc_sw128(saddr);
    uint64_t d = uint64_t((saddr & 0x3FFFFu) >> 4);
    d |= uint64_t(512 >> 4) << 32;
    d |= uint64_t(1) << 46;
    d |= uint64_t(4) << 61;  // SWIZZLE_64B
    return d;
}

// MN-major operand made of boxes of 64 rows (of K): the next 8 K rows an atom on, the next 64 columns a box on.
template <int DP>
__device__ __forceinline__ uint64_t sdesc_mn(uint32_t saddr) {
    return sdesc_k<DP>(saddr) | uint64_t(AttnBox<DP>::kTile >> 4) << 16;
}

// D = A x B^T over DP columns: A 128 rows, B 64 rows, both K-major.
template <typename T, int DP>
__device__ __forceinline__ void issue_scores(uint32_t leader, uint32_t d, uint32_t a_smem, uint32_t b_smem) {
    using Box = AttnBox<DP>;
    constexpr uint32_t idesc = attn_idesc<T, false>(kAttnBN);
#pragma unroll
    for (int k = 0; k < DP / 16; ++k) {
        const int box = k / Box::kSteps, step = k % Box::kSteps;
        const uint64_t da = sdesc_k<DP>(a_smem + box * Box::kFixed) + uint64_t(2 * step);
        const uint64_t db = sdesc_k<DP>(b_smem + box * Box::kTile) + uint64_t(2 * step);
        mma_ss(leader, d, da, db, idesc, k != 0);
    }
}

// acc (+)= A x B: A 128 lanes x 64 packed elements in TMEM, 16 of them every STEP columns, B 64 rows x DP columns in
// shared memory.
template <typename T, int DP, int STEP>
__device__ __forceinline__ void issue_product(uint32_t leader, uint32_t acc, uint32_t a_tmem, uint32_t b_smem,
                                              bool first) {
    constexpr uint32_t idesc = attn_idesc<T, true>(DP);
    const uint64_t db = sdesc_mn<DP>(b_smem);
#pragma unroll
    for (int k = 0; k < 4; ++k)
        mma_ts(leader, acc, a_tmem + STEP * k, db + uint64_t(AttnBox<DP>::kRow * k), idesc, !(first && k == 0));
}

// Clears the rows of padded keys in a slot's tile of 64 rows x DP columns. One warp.
template <int DP>
__device__ __forceinline__ void clear_padded(unsigned char* tile, const uint8_t* pad, int j0, int N) {
    const int lane = threadIdx.x & 31;
    const bool p0 = j0 + lane < N && pad[j0 + lane] != 0, p1 = j0 + 32 + lane < N && pad[j0 + 32 + lane] != 0;
    unsigned long long rows = (unsigned long long)__ballot_sync(0xffffffffu, p0) |
                              (unsigned long long)__ballot_sync(0xffffffffu, p1) << 32;
    while (rows != 0) {
        const int r = __ffsll((long long)rows) - 1;
        rows &= rows - 1;
#pragma unroll
        for (int box = 0; box < AttnBox<DP>::kBoxes; ++box)  // a whole row: the swizzle only permutes inside it
            if (uint32_t(lane) * 4 < AttnBox<DP>::kRow)
                *reinterpret_cast<uint32_t*>(tile + box * AttnBox<DP>::kTile + r * AttnBox<DP>::kRow + lane * 4) = 0u;
    }
    fence_proxy_async_smem();
    __syncwarp();
}

// ---- forward ------------------------------------------------------------------------------------------------------
template <int DP>
struct AttnFwdLayout {
    static constexpr int kBoxes = AttnBox<DP>::kBoxes;
    static constexpr uint32_t kQBytes = AttnBox<DP>::kFixed * kBoxes;
    static constexpr uint32_t kTileBytes = AttnBox<DP>::kTile * kBoxes;  // of K or of V
    static constexpr int kStages = DP == 128 ? 2 : 4;                    // two CTAs an SM
    static constexpr uint32_t kStageBytes = 2 * kTileBytes;
    static constexpr uint32_t kRing = kQBytes;
    static constexpr uint32_t kBars = kRing + kStages * kStageBytes;
    // qfull, kfull[S], vfull[S], empty[S], sfull[2], pfull[2], done[2], finished
    static constexpr int kNumBars = 1 + 3 * kStages + 7;
    static constexpr uint32_t kSlot = kBars + kNumBars * 8;
    static constexpr uint32_t kSmemBytes = kSlot + 16 + 1024;
    static constexpr uint32_t kTmemCols = 256;  // two score tiles of 64, the output's DP
    static_assert(128 + DP <= 256, "TMEM");
    static_assert(2 * kSmemBytes <= 227 * 1024, "two CTAs an SM");
};

constexpr int kAttnFwdThreads = 224;  // loads, scores, products, four softmax warps

// P is kept as two 16-bit parts, its rounding and what that took, which both go through the product (one product more a
// tile), so that the result's own rounding is the only one; a forward that a backward follows keeps what that one took
// as well (see delta in td_attention.cuh). P rounded once would put the result 1.3 to 1.4 times as far from float64.
template <typename T, int DP>
__global__ void __launch_bounds__(kAttnFwdThreads, 2)
    attn_tc_forward_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                           const __grid_constant__ CUtensorMap map_v, const AttnTcArgs args) {
    using Lay = AttnFwdLayout<DP>;
    constexpr int S = Lay::kStages, KB = Lay::kBoxes;
    const AttnArgs& a = args.a;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    unsigned char* smem = smem_raw + ((1024 - (smem_addr(smem_raw) & 1023)) & 1023);
    uint64_t* qfull = reinterpret_cast<uint64_t*>(smem + Lay::kBars);
    uint64_t *kfull = qfull + 1, *vfull = kfull + S, *empty = vfull + S, *sfull = empty + S, *pfull = sfull + 2,
             *done = pfull + 2, *finished = done + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + Lay::kSlot);
    auto k_tile = [&](int s) { return smem + Lay::kRing + s * Lay::kStageBytes; };
    auto v_tile = [&](int s) { return smem + Lay::kRing + s * Lay::kStageBytes + Lay::kTileBytes; };

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // the last query tiles first: under the causal rule they are the longest
    const int q_tiles = (a.Q + kAttnBM - 1) / kAttnBM;
    const int bh = blockIdx.x % (a.B * a.H), split = blockIdx.x / (a.B * a.H) % args.splits;
    const int qt = q_tiles - 1 - int(blockIdx.x / (a.B * a.H)) / args.splits;
    const int h = bh % a.H, b = bh / a.H, hk = h / (a.H / a.Hk), i0 = qt * kAttnBM, off = a.N - a.Q;
    const long long all_tiles = (attn_key_end(a, i0 + kAttnBM) + kAttnBN - 1) / kAttnBN;
    const int t0 = int(all_tiles * split / args.splits), t1 = int(all_tiles * (split + 1) / args.splits);
    const uint8_t* flags = args.row_flags == nullptr
                               ? nullptr
                               : args.row_flags + b * args.rf_b + h * args.rf_h + qt * args.rf_q;

    if (threadIdx.x == 0) {
        mbar_init(qfull, 2 * KB);
        for (int s = 0; s < S; ++s) {
            mbar_init(&kfull[s], KB);
            mbar_init(&vfull[s], KB);
            mbar_init(&empty[s], 1);
        }
        for (int g = 0; g < 2; ++g) {
            mbar_init(&sfull[g], 1);
            mbar_init(&pfull[g], 4);  // a warp of the four, not a thread: arrivals on one word are served in turn
            mbar_init(&done[g], 1);
        }
        mbar_init(finished, 1);
        mbar_fence_init();
        tma_prefetch_desc(&map_q);
        tma_prefetch_desc(&map_k);
        tma_prefetch_desc(&map_v);
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, Lay::kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
    grid_dependency_wait();
    launch_dependents();

    if (warp == 0) {
        // a lane per box of the ring: TMA copies of one thread are served one after another, those of different threads
        // overlap
        const uint64_t pol = l2_evict_last();  // keys and values are read again by the other query tiles
        if (lane < 2 * KB && t1 > t0) {  // the queries in halves of 64
            mbar_arrive_expect_tx(qfull, AttnBox<DP>::kTile);
            tma_load_4d(smem + lane * AttnBox<DP>::kTile, &map_q, qfull, 64 * (lane / 2), i0 + 64 * (lane % 2), h, b,
                        l2_evict_first());
        }
        int n = 0;
        Ring<S> ring;
        for_tiles(t0, t1, flags, [&](int t, bool) {
            const int s = ring.at;
            if (!warp_wait(&empty[s], ring.parity ^ 1u, kErrSlotWait)) return false;
            ring.template step<>();
            const int job = lane - 2 * KB * s, box = job % KB;
            if (job >= 0 && job < 2 * KB) {
                uint64_t* bar = job < KB ? &kfull[s] : &vfull[s];
                mbar_arrive_expect_tx(bar, AttnBox<DP>::kTile);
                tma_load_4d((job < KB ? k_tile(s) : v_tile(s)) + box * AttnBox<DP>::kTile,
                            job < KB ? &map_k : &map_v, bar, 64 * box, t * kAttnBN, hk, b, pol);
            }
            __syncwarp();
            ++n;
            return true;
        });
        // no copy and no product is in flight when the CTA ends
        for (int i = n > S ? n - S : 0; i < n; ++i)
            if (!warp_wait(&empty[i % S], uint32_t((i / S) & 1), kErrSlotWait)) {
                warp_wait(&kfull[i % S], uint32_t((i / S) & 1), kErrTmaWait);
                warp_wait(&vfull[i % S], uint32_t((i / S) & 1), kErrTmaWait);
            }
    } else if (warp == 1) {
        const uint32_t leader = lane == 0;
        Ring<S> ring;
        Ring<2> buf;
        if (t1 <= t0 || warp_wait(qfull, 0u, kErrTmaWait))
            for_tiles(t0, t1, flags, [&](int, bool) {
                if (!warp_wait(&kfull[ring.at], ring.parity, kErrTmaWait)) return false;
                // the buffer's P before these scores (none in the first round) has been read by its product
                if (!warp_wait(&done[buf.at], buf.parity ^ 1u, kErrMmaWait)) return false;
                tc_fence_after();
                issue_scores<T, DP>(leader, tmem + 64 * buf.at, smem_addr(smem), smem_addr(k_tile(ring.at)));
                commit(leader, &sfull[buf.at]);
                ring.template step<>();
                buf.template step<>();
                return true;
            });
    } else if (warp == 2) {
        const uint32_t leader = lane == 0;
        const uint8_t* pad = a.padding == nullptr ? nullptr : a.padding + (long long)b * a.N;
        bool first = true;
        Ring<S> ring;
        Ring<2> buf;
        const bool ok = for_tiles(t0, t1, flags, [&](int t, bool all) {
            unsigned char* v = v_tile(ring.at);
            if (!warp_wait(&vfull[ring.at], ring.parity, kErrTmaWait)) return false;
            if (pad != nullptr && !all) clear_padded<DP>(v, pad, t * kAttnBN, a.N);
            if (!warp_wait(&pfull[buf.at], buf.parity, kErrMmaWait)) return false;
            tc_fence_after();
            const uint32_t p = tmem + 64 * buf.at;
            issue_product<T, DP, 8>(leader, tmem + 128, p, smem_addr(v), first);
            issue_product<T, DP, 8>(leader, tmem + 128, p + 32, smem_addr(v), false);
            commit(leader, &empty[ring.at]);
            commit(leader, &done[buf.at]);
            first = false;
            ring.template step<>();
            buf.template step<>();
            return true;
        });
        if (ok && !first) commit(leader, finished);
    } else {
        const int quarter = warp & 3, i = i0 + quarter * 32 + lane;
        const uint32_t lanes = tmem + (uint32_t(quarter * 32) << 16);
        const float c = float(a.scale * 1.4426950408889634);
        // The reference of a row's exponentials follows its maximum only when that grew by more than 8 (base 2), so
        // P stays below 2^8 and the output, in TMEM, is seldom rescaled.
        const float slack = 8.0f / c;
        const uint32_t* bits = args.row_bits == nullptr
                                   ? nullptr
                                   : args.row_bits + b * args.rb_b + h * args.rb_h + min(i, a.Q - 1) * args.rb_q;
        float ref = -INFINITY, sum = 0.f;
        int n = 0;
        Ring<2> buf;
        const bool ok = for_tiles(t0, t1, flags, [&](int t, bool all) {
            const int j0 = t * kAttnBN;
            const bool open = all && j0 + kAttnBN <= a.N && (!a.causal || j0 + kAttnBN - 1 <= i0 + off);
            unsigned long long w = ~0ull;
            if (!open) {
                w = bits_below(a.N - j0);
                if (a.causal) w &= bits_below(i + off - j0 + 1);
                if (bits != nullptr) {
                    const uint2 x = __ldg(reinterpret_cast<const uint2*>(bits + 2 * t));
                    w &= (unsigned long long)x.y << 32 | x.x;
                }
            }
            if (!warp_wait(&sfull[buf.at], buf.parity, kErrMmaWait)) return false;
            tc_fence_after();
            const uint32_t sc = lanes + 64 * buf.at;
            uint32_t v[2][32];
            tmem_ld_32x32b_x32(sc, v[0]);
            tmem_ld_32x32b_x32(sc + 32, v[1]);
            tmem_ld_wait();
            // four chains each for the maximum and the sum: one of 64 dependent steps would cost more than the work
            float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                if (!open) {
                    const uint32_t wg = uint32_t(w >> (32 * g));
#pragma unroll
                    for (int x = 0; x < 32; ++x)
                        if (((wg >> x) & 1u) == 0) v[g][x] = 0xff800000u;  // -infinity
                }
#pragma unroll
                for (int x = 0; x < 32; x += 2)
                    tops[x / 2 % 4] = max3(tops[x / 2 % 4], __uint_as_float(v[g][x]), __uint_as_float(v[g][x + 1]));
            }
            const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
            if (__any_sync(0xffffffffu, top > ref + slack)) {
                const float next = fmaxf(ref, top);
                const float keep = next == -INFINITY ? 1.f : ex2((ref - next) * c);
                ref = next;
                sum *= keep;
                if (n > 0) {
                    // the output so far is complete once the last product is (a barrier each for even and odd tiles:
                    // a parity wait tells one phase from the next only, and not every phase is waited for)
                    if (!warp_wait(&done[(n - 1) & 1], uint32_t(((n - 1) >> 1) & 1), kErrMmaWait)) return false;
                    tc_fence_after();
#pragma unroll 1
                    for (int d = 0; d < DP; d += 32) {
                        uint32_t o[32];
                        tmem_ld_32x32b_x32(lanes + 128 + d, o);
                        tmem_ld_wait();
#pragma unroll
                        for (int x = 0; x < 32; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * keep);
                        tmem_st_32x32b_x32(lanes + 128 + d, o);
                    }
                }
            }
            const float shift = ref == -INFINITY ? 0.f : -ref * c;
            uint32_t p[32];
            const F2 c2 = f2(c, c), shift2 = f2(shift, shift);
            F2 sums[4] = {f2(sum, 0.f), 0ull, 0ull, 0ull};
#pragma unroll
            for (int x = 0; x < 32; ++x) {
                float x0, x1;
                f2_split(f2_fma(f2(v[x / 16][2 * (x % 16)], v[x / 16][2 * (x % 16) + 1]), c2, shift2), x0, x1);
                const float p0 = ex2(x0), p1 = ex2(x1);
                sums[x % 4] = f2_add(sums[x % 4], f2(p0, p1));
                pack_parts<T>(p0, p1, p[x], v[x / 16][x % 16]);  // (v's two registers of this pair are free)
            }
            {
                float s0, s1;
                f2_split(f2_add(f2_add(sums[0], sums[1]), f2_add(sums[2], sums[3])), s0, s1);
                sum = s0 + s1;
            }
            tmem_st_32x32b_x32(sc, p);
            tmem_st_32x32b_x16(sc + 32, v[0]);
            tmem_st_32x32b_x16(sc + 48, v[1]);
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&pfull[buf.at]);
            buf.template step<>();
            ++n;
            return true;
        });
        const bool got = ok && (n == 0 || warp_wait(finished, 0u, kErrMmaWait));
        tc_fence_after();
        if (got) {
            const float inv = sum == 0.f ? 0.f : 1.f / sum;
            const long long at = (((long long)b * a.Q + i) * a.H + h) * a.D;
            const long long place = ((long long)bh * a.Q + i) * args.splits + split;
#pragma unroll 1
            for (int d = 0; d < DP && d < a.D; d += 32) {
                uint32_t o[32];
                __syncwarp();
                if (n > 0) {
                    tmem_ld_32x32b_x32(lanes + 128 + d, o);
                    tmem_ld_wait();
                } else {
#pragma unroll
                    for (int x = 0; x < 32; ++x) o[x] = 0u;
                }
                if (i >= a.Q) continue;
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    if (d + 8 * g >= a.D) break;  // D is a multiple of 8
                    if (args.splits > 1) {
                        uint4* part = reinterpret_cast<uint4*>(args.part_o + place * a.D + d + 8 * g);
                        part[0] = make_uint4(o[8 * g], o[8 * g + 1], o[8 * g + 2], o[8 * g + 3]);
                        part[1] = make_uint4(o[8 * g + 4], o[8 * g + 5], o[8 * g + 6], o[8 * g + 7]);
                        continue;
                    }
                    uint32_t q[4], rest[4];
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const float o0 = __uint_as_float(o[8 * g + 2 * x]) * inv;
                        const float o1 = __uint_as_float(o[8 * g + 2 * x + 1]) * inv;
                        q[x] = pack2<T>(o0, o1);
                        const float2 r = unpack2<T>(q[x]);
                        rest[x] = pack2<T>(o0 - r.x, o1 - r.y);
                    }
                    *reinterpret_cast<uint4*>(static_cast<T*>(a.out) + at + d + 8 * g) =
                        make_uint4(q[0], q[1], q[2], q[3]);
                    if (a.rest != nullptr)
                        *reinterpret_cast<uint4*>(static_cast<T*>(a.rest) + at + d + 8 * g) =
                            make_uint4(rest[0], rest[1], rest[2], rest[3]);
                }
            }
            if (args.splits > 1) {
                if (i < a.Q) *reinterpret_cast<float2*>(args.part_ml + 2 * place) = make_float2(ref * c, sum);
            } else if (a.lse != nullptr)  // Qp is a multiple of the tile
                static_cast<float*>(a.lse)[(long long)bh * a.Qp + i] =
                    i < a.Q && sum != 0.f ? fmaf(ref, c, log2f(sum)) : INFINITY;
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, Lay::kTmemCols);
    }
}

// ---- backward -----------------------------------------------------------------------------------------------------
template <int DP>
struct AttnBwdLayout {
    static constexpr int kBoxes = AttnBox<DP>::kBoxes;
    static constexpr uint32_t kFixedBytes = AttnBox<DP>::kFixed * kBoxes;  // one resident operand
    static constexpr uint32_t kTileBytes = AttnBox<DP>::kTile * kBoxes;    // one streamed operand
    // score buffers (S and dP, 64 columns each) and ring slots. A buffer goes from the scores' product through the
    // elementwise work to the products that read P and dS, about 2000 cycles in all, so the tiles in flight set the
    // pace: three where TMEM holds them, two beside the accumulators of wide heads
    static constexpr int kBufs = DP == 128 ? 2 : 3;
    static constexpr int kStages = DP == 128 ? 4 : 6;
    static constexpr uint32_t kAcc = kBufs * 128;  // first accumulator's TMEM column
    static constexpr int kGroups = 2;  // warpgroups of the elementwise work (encoder with three: 676 us against 677)
    static constexpr int kThreads = 128 * (1 + kGroups);  // loads, scores, products, -, the warpgroups
    static constexpr uint32_t kStageBytes = 2 * kTileBytes;
    static constexpr uint32_t kRing = 2 * kFixedBytes;
    static constexpr uint32_t kStats = kRing + kStages * kStageBytes;  // per stage: lse[64], delta[64]
    static constexpr uint32_t kBars = kStats + kStages * 2 * kAttnBN * 4;
    // fixed, full[S], empty[S], sfull[bufs], pfull[bufs], done[bufs], finished
    static constexpr int kNumBars = 1 + 2 * kStages + 3 * kBufs + 1;
    static constexpr uint32_t kSlot = kBars + kNumBars * 8;
    static constexpr uint32_t kSmemBytes = kSlot + 16 + 1024;
    static constexpr uint32_t kTmemCols = 512;
    static_assert(kAcc + 2 * DP <= 512, "TMEM");
    static_assert(kSmemBytes <= 227 * 1024, "shared memory");
};


// A key's P may be about 1 / N for every query, from some 16000 keys on below float16's normal numbers. So the keys'
// gradient in float16 keeps it times 2^15 (P is at most one), from an lse that is 15 less, and divides dV by that.
// bfloat16 has float32's exponents.
template <typename T> constexpr int attn_p_bits() { return std::is_same<T, __half>::value ? 15 : 0; }

// float16 keeps dS times a power of two that makes its bound 2^15 or little less, so that dS cannot overflow and is a
// normal number down to 2^-29 of the bound. |dS_ij| <= P_ij |dO_i| (|v_j| + |o_i|) <= 2 |dO_i| max|v|, the maximum over
// the keys of the (image, key head). A row of the queries' gradient is a lane's own and has a scale of its own, row_g
// being its |dO_i|^2. The keys' gradient sums over queries, so there one scale holds for the (image, key head), from
// the largest |dO_i|. bfloat16 has float32's exponents and needs no scale.
template <bool KEYS>
__device__ __forceinline__ float attn_ds_scale(const AttnTcArgs& args, int bhk, float row_g) {  // one warp
    const float* amax = args.amax + (long long)bhk * args.amax_parts;
    const long long values = (long long)args.a.B * args.a.Hk * args.amax_parts;
    float g = KEYS ? 0.f : row_g, v = 0.f;
    for (int i = threadIdx.x & 31; i < args.amax_parts; i += 32) {
        if (KEYS) g = fmaxf(g, amax[i]);
        v = fmaxf(v, amax[values + i]);
    }
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) {
        if (KEYS) g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, x));
        v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, x));
    }
    const float square = g * v;  // of finite float16 numbers: 2^-96 .. 2^78, or zero
    if (!(square > 0.f) || !(square < INFINITY)) return 1.f;
    return exp2f(14.f - ceilf(0.5f * log2f(square)));
}

// P and dS of one row of a tile of 64 columns, from the scores at sc and sc + 64 to packed pairs in the same places: of
// every 16 columns, 8 for the roundings, then 8 for what they took. The statistics are the row's own, or (KEYS) the
// columns', lse[64] and delta[64] at st. MASKED: w has a bit per open pair.
template <typename T, bool KEYS, bool MASKED>
__device__ __forceinline__ void elementwise(uint32_t sc, const float* st, float row_lse, float row_delta, float c,
                                            float ds_scale, unsigned long long w) {
    constexpr bool kHalf = std::is_same<T, __half>::value;
    uint32_t s[2][16], d[2][16];
    tmem_ld_32x32b_x16(sc, s[0]);
    tmem_ld_32x32b_x16(sc + 64, d[0]);
#pragma unroll
    for (int part = 0; part < 4; ++part) {
        tmem_ld_wait();
        if (part < 3) {
            tmem_ld_32x32b_x16(sc + 16 * (part + 1), s[(part + 1) & 1]);
            tmem_ld_32x32b_x16(sc + 64 + 16 * (part + 1), d[(part + 1) & 1]);
        }
        uint32_t p[16], e[16];  // the roundings, then what they took
        const F2 nc = f2(-c, -c), minus = f2(-1.f, -1.f), scale = f2(ds_scale, ds_scale);
        const uint32_t open = MASKED ? uint32_t(w >> (16 * part)) : 0u;
#pragma unroll
        for (int x = 0; x < 16; x += 4) {
            F2 ls[2] = {f2(row_lse, row_lse), f2(row_lse, row_lse)};
            F2 de[2] = {f2(row_delta, row_delta), f2(row_delta, row_delta)};
            if constexpr (KEYS) {
                const ulonglong2 a = *reinterpret_cast<const ulonglong2*>(st + 16 * part + x);
                const ulonglong2 b = *reinterpret_cast<const ulonglong2*>(st + kAttnBN + 16 * part + x);
                ls[0] = a.x; ls[1] = a.y; de[0] = b.x; de[1] = b.y;
            }
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                const int at = x + 2 * y;
                // lse - c S, whose negative the exponential takes; dP - delta
                float l0, l1, e0, e1;
                f2_split(f2_fma(f2(s[part & 1][at], s[part & 1][at + 1]), nc, ls[y]), l0, l1);
                float p0 = ex2(-l0), p1 = ex2(-l1);
                F2 diff = f2_fma(de[y], minus, f2(d[part & 1][at], d[part & 1][at + 1]));
                if constexpr (kHalf) diff = f2_mul(diff, scale);
                f2_split(f2_mul(f2(p0, p1), diff), e0, e1);
                if constexpr (MASKED) {
                    if (((open >> at) & 1u) == 0) p0 = e0 = 0.f;
                    if (((open >> (at + 1)) & 1u) == 0) p1 = e1 = 0.f;
                }
                if constexpr (KEYS) pack_parts<T>(p0, p1, p[at / 2], p[8 + at / 2]);
                pack_parts<T>(e0, e1, e[at / 2], e[8 + at / 2]);
            }
        }
        if constexpr (KEYS) tmem_st_32x32b_x16(sc + 16 * part, p);
        tmem_st_32x32b_x16(sc + 64 + 16 * part, e);
    }
}

// One block of the keys' gradient (KEYS) or of the queries' gradient.
template <typename T, int DP, bool KEYS>
__device__ __forceinline__ void attn_tc_backward_block(const CUtensorMap& map_fixed1, const CUtensorMap& map_fixed2,
                                                       const CUtensorMap& map_b1, const CUtensorMap& map_b2,
                                                       const AttnTcArgs& args, int block, unsigned char* smem,
                                                       uint32_t tmem) {
    using Lay = AttnBwdLayout<DP>;
    constexpr int S = Lay::kStages, KB = Lay::kBoxes, NB = Lay::kBufs;
    constexpr bool kHalf = std::is_same<T, __half>::value;
    const AttnArgs& a = args.a;
    uint64_t* fixed = reinterpret_cast<uint64_t*>(smem + Lay::kBars);
    uint64_t *full = fixed + 1, *empty = full + S, *sfull = empty + S, *pfull = sfull + NB, *done = pfull + NB,
             *finished = done + NB;
    auto tile1 = [&](int s) { return smem + Lay::kRing + s * Lay::kStageBytes; };
    auto tile2 = [&](int s) { return smem + Lay::kRing + s * Lay::kStageBytes + Lay::kTileBytes; };
    auto stats = [&](int s) { return reinterpret_cast<float*>(smem + Lay::kStats) + s * 2 * kAttnBN; };

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, off = a.N - a.Q, group = a.H / a.Hk;
    // the block's rows: keys r0 .. of key head hk, over the query heads h0 .. h1 and their query tiles; or queries
    // r0 .. of head h0, over the key tiles
    const int heads = KEYS ? a.Hk : a.H, rows = KEYS ? a.N : a.Q;
    const int row_tiles = (rows + kAttnBM - 1) / kAttnBM;
    const int bx = block % (a.B * heads), splits = KEYS ? a.k_splits : a.q_splits;
    const int split = block / (a.B * heads) % splits, tile = block / (a.B * heads) / splits;
    // the longest blocks under the causal rule first: the first keys, the last queries
    const int rt = KEYS ? tile : row_tiles - 1 - tile;
    const int head = bx % heads, b = bx / heads, r0 = rt * kAttnBM;
    const int hk = KEYS ? head : head / group, h0 = KEYS ? head * group : head, h1 = KEYS ? h0 + group : h0 + 1;
    const int t0 = KEYS && a.causal ? max(0, min(a.Q, r0 - off)) / kAttnBN : 0;
    const int t1 = KEYS ? (a.Q + kAttnBN - 1) / kAttnBN
                        : (attn_key_end(a, r0 + kAttnBM) + kAttnBN - 1) / kAttnBN;
    // this split's tiles, counted over the heads
    const long long work = (long long)(t1 - t0) * (h1 - h0);
    const int from = int(work * split / splits), to = int(work * (split + 1) / splits);
    auto each_tile = [&](auto&& f) {  // f(head, tile, all open by the flags)
        for (int h = h0; h < h1; ++h) {
            const int first = t0 - (h - h0) * (t1 - t0), lo = max(t0, first + from), hi = min(t1, first + to);
            if (lo >= hi) continue;
            const uint8_t* flags = nullptr;
            if (KEYS && args.col_flags != nullptr)
                flags = args.col_flags + b * args.cf_b + h * args.cf_h + (long long)rt * args.col_tiles;
            if (!KEYS && args.row_flags != nullptr)
                flags = args.row_flags + b * args.rf_b + h * args.rf_h + rt * args.rf_q;
            if (!for_tiles(lo, hi, flags, [&](int t, bool all) { return f(h, t, all); })) return false;
        }
        return true;
    };

    if (warp == 0) {
        const uint64_t pol = l2_evict_last();
        if (lane < 4 * KB) {  // the two resident operands, in halves of 64 rows
            const int job = lane % (2 * KB), op = lane / (2 * KB);
            mbar_arrive_expect_tx(fixed, AttnBox<DP>::kTile);
            tma_load_4d(smem + op * Lay::kFixedBytes + job * AttnBox<DP>::kTile, op == 0 ? &map_fixed1 : &map_fixed2,
                        fixed, 64 * (job / 2), r0 + 64 * (job % 2), head, b, pol);
        }
        int n = 0;
        Ring<S> ring;
        each_tile([&](int h, int t, bool) {
            const int s = ring.at;
            if (!warp_wait(&empty[s], ring.parity ^ 1u, kErrSlotWait)) return false;
            ring.template step<>();
            constexpr int kJobs = 2 * KB + (KEYS ? 2 : 0);
            static_assert(kJobs * S <= 32, "a lane per copy of the ring");
            const int job = lane - kJobs * s, box = job % KB;
            if (job >= 0 && job < 2 * KB) {
                mbar_arrive_expect_tx(&full[s], AttnBox<DP>::kTile);
                tma_load_4d((job < KB ? tile1(s) : tile2(s)) + box * AttnBox<DP>::kTile,
                            job < KB ? &map_b1 : &map_b2, &full[s], 64 * box, t * kAttnBN, KEYS ? h : hk, b, pol);
            } else if (job >= 2 * KB && job < kJobs) {
                const float* src = job == 2 * KB ? args.keys_lse : static_cast<const float*>(a.delta);
                mbar_arrive_expect_tx(&full[s], kAttnBN * 4u);
                bulk_load(stats(s) + (job - 2 * KB) * kAttnBN,
                          src + ((long long)b * a.H + h) * a.Qp + t * kAttnBN, kAttnBN * 4u, &full[s]);
            }
            __syncwarp();
            ++n;
            return true;
        });
        warp_wait(fixed, 0u, kErrTmaWait);
        for (int i = n > S ? n - S : 0; i < n; ++i)
            if (!warp_wait(&empty[i % S], uint32_t((i / S) & 1), kErrSlotWait))
                warp_wait(&full[i % S], uint32_t((i / S) & 1), kErrTmaWait);
    } else if (warp == 1) {
        const uint32_t leader = lane == 0;
        Ring<S> ring;
        Ring<NB> buf;
        if (warp_wait(fixed, 0u, kErrTmaWait))
            each_tile([&](int, int, bool) {
                if (!warp_wait(&full[ring.at], ring.parity, kErrTmaWait)) return false;
                // the buffer's P and dS before these scores (none in the first round) have been read by their products
                if (!warp_wait(&done[buf.at], buf.parity ^ 1u, kErrMmaWait)) return false;
                tc_fence_after();
                const uint32_t sc = tmem + 128 * buf.at;
                issue_scores<T, DP>(leader, sc, smem_addr(smem), smem_addr(tile1(ring.at)));
                issue_scores<T, DP>(leader, sc + 64, smem_addr(smem + Lay::kFixedBytes), smem_addr(tile2(ring.at)));
                commit(leader, &sfull[buf.at]);
                if (lane == 0) mbar_arrive(&sfull[buf.at]);  // for the statistics, which this warp's wait has seen land
                ring.template step<>();
                buf.template step<>();
                return true;
            });
    } else if (warp == 2) {
        const uint32_t leader = lane == 0;
        const uint8_t* pad = KEYS || a.padding == nullptr ? nullptr : a.padding + (long long)b * a.N;
        bool first = true;
        Ring<S> ring;
        Ring<NB> buf;
        const bool ok = each_tile([&](int, int t, bool all) {
            const uint32_t sc = tmem + 128 * buf.at;
            if (!warp_wait(&pfull[buf.at], buf.parity, kErrMmaWait)) return false;
            // (this tile's scores are formed: what they made of padded rows has been replaced)
            if (pad != nullptr && !all) clear_padded<DP>(tile1(ring.at), pad, t * kAttnBN, a.N);
            tc_fence_after();
            if constexpr (KEYS) {  // dV += P^T dO
                issue_product<T, DP, 16>(leader, tmem + Lay::kAcc + DP, sc, smem_addr(tile2(ring.at)), first);
                issue_product<T, DP, 16>(leader, tmem + Lay::kAcc + DP, sc + 8, smem_addr(tile2(ring.at)), false);
            }
            // dK += dS^T Q, dQ += dS K
            issue_product<T, DP, 16>(leader, tmem + Lay::kAcc, sc + 64, smem_addr(tile1(ring.at)), first);
            issue_product<T, DP, 16>(leader, tmem + Lay::kAcc, sc + 72, smem_addr(tile1(ring.at)), false);
            commit(leader, &empty[ring.at]);
            commit(leader, &done[buf.at]);
            first = false;
            ring.template step<>();
            buf.template step<>();
            return true;
        });
        if (ok && !first) commit(leader, finished);
    } else if (warp >= 4) {
        const int quarter = warp & 3, wg = (warp - 4) >> 2, r = r0 + quarter * 32 + lane;
        const uint32_t lanes = tmem + (uint32_t(quarter * 32) << 16);
        const float c = float(a.scale * 1.4426950408889634);
        float row_lse = INFINITY, row_delta = 0.f, row_g = 0.f;
        if (!KEYS) {  // the rows' own statistics (the arrays hold Qp rows, a multiple of the tile)
            const long long at = ((long long)b * a.H + h0) * a.Qp + r;
            row_lse = static_cast<const float*>(a.lse)[at];
            row_delta = static_cast<const float*>(a.delta)[at];
            if constexpr (kHalf) row_g = args.row_g[at];
        }
        const float ds_scale = kHalf ? attn_ds_scale<KEYS>(args, b * a.Hk + hk, row_g) : 1.f;
        constexpr float kP = float(1 << (KEYS ? attn_p_bits<T>() : 0));  // what P is kept times
        // the warpgroups take the tiles in turn
        constexpr int NG = Lay::kGroups;
        int n = 0, turn = wg;
        Ring<S> ring(wg);
        Ring<NB> buf(wg);
        bool ok = each_tile([&](int h, int t, bool all) {
            ++n;
            if (turn-- != 0) return true;
            turn = NG - 1;
            const int c0 = t * kAttnBN;  // the tile's first column: a query (KEYS) or a key
            bool open = all;
            unsigned long long w = ~0ull;
            if constexpr (KEYS) {
                // (the queries behind the last, which are zeros, do not count: an infinite key makes NaN of them)
                open = open && c0 + kAttnBN <= a.Q && (!a.causal || r0 + kAttnBM - 1 <= c0 + off);
                if (!open) {
                    w = bits_below(a.Q - c0);
                    if (a.causal) w &= ~bits_below(r - off - c0);
                    if (args.col_bits != nullptr && r < a.N) {
                        const uint2 x = __ldg(reinterpret_cast<const uint2*>(
                            args.col_bits + b * args.cb_b + h * args.cb_h + (long long)r * args.col_words + 2 * t));
                        w &= (unsigned long long)x.y << 32 | x.x;
                    }
                }
            } else {
                open = open && c0 + kAttnBN <= a.N && (!a.causal || c0 + kAttnBN - 1 <= r0 + off);
                if (!open) {
                    w = bits_below(a.N - c0);
                    if (a.causal) w &= bits_below(r + off - c0 + 1);
                    if (args.row_bits != nullptr) {
                        const uint2 x = __ldg(reinterpret_cast<const uint2*>(
                            args.row_bits + b * args.rb_b + h * args.rb_h + min(r, a.Q - 1) * args.rb_q + 2 * t));
                        w &= (unsigned long long)x.y << 32 | x.x;
                    }
                }
            }
            if (!warp_wait(&sfull[buf.at], buf.parity, kErrMmaWait)) return false;
            tc_fence_after();
            const uint32_t sc = lanes + 128 * buf.at;
            // 16 columns at a time, the next ones' loads in flight meanwhile; P and dS go where the first scores were
            if (open)
                elementwise<T, KEYS, false>(sc, stats(ring.at), row_lse, row_delta, c, ds_scale / kP, w);
            else
                elementwise<T, KEYS, true>(sc, stats(ring.at), row_lse, row_delta, c, ds_scale / kP, w);
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&pfull[buf.at]);
            ring.template step<NG>();
            buf.template step<NG>();
            return true;
        });
        ok = ok && (n == 0 || warp_wait(finished, 0u, kErrMmaWait));
        tc_fence_after();
        // the gradients' rows: a warpgroup an accumulator for the keys' block, else half of the columns each
        if (ok) {
            const bool is_v = KEYS && wg == 1;
            const float f = is_v ? 1.f / kP : float(a.scale) / ds_scale;
            const bool gone = KEYS && a.padding != nullptr && r < a.N && a.padding[(long long)b * a.N + r] != 0;
            const long long at = (((long long)b * rows + r) * heads + head) * a.D;
            T* out = static_cast<T*>(KEYS ? (is_v ? a.grad_v : a.grad_k) : a.grad_q) + at;
            float* part = static_cast<float*>(KEYS ? (is_v ? a.part_v : a.part_k) : a.part_q) +
                          split * ((long long)a.B * rows * heads * a.D) + at;
            const int d_first = KEYS ? 0 : 32 * wg, d_step = KEYS ? 32 : 64;
#pragma unroll 1
            for (int d = d_first; d < DP && d < a.D; d += d_step) {
                uint32_t o[32];
                __syncwarp();
                if (n > 0) {
                    tmem_ld_32x32b_x32(lanes + Lay::kAcc + (is_v ? DP : 0) + d, o);
                    tmem_ld_wait();
                }
                if (r >= rows) continue;
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    if (d + 8 * g >= a.D) break;
                    if (splits > 1) {
#pragma unroll
                        for (int x = 0; x < 8; x += 4) {
                            float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
                            const uint32_t* z = o + 8 * g + x;
                            if (n > 0 && !gone)
                                y = make_float4(__uint_as_float(z[0]) * f, __uint_as_float(z[1]) * f,
                                                __uint_as_float(z[2]) * f, __uint_as_float(z[3]) * f);
                            *reinterpret_cast<float4*>(part + d + 8 * g + x) = y;
                        }
                        continue;
                    }
                    uint4 q = make_uint4(0u, 0u, 0u, 0u);
                    uint32_t* qw = &q.x;
                    if (n > 0 && !gone) {
#pragma unroll
                        for (int x = 0; x < 4; ++x)
                            qw[x] = pack2<T>(__uint_as_float(o[8 * g + 2 * x]) * f,
                                             __uint_as_float(o[8 * g + 2 * x + 1]) * f);
                    }
                    *reinterpret_cast<uint4*>(out + d + 8 * g) = q;
                }
            }
        }
    }
}

template <typename T, int DP>
__global__ void __launch_bounds__(AttnBwdLayout<DP>::kThreads, 1)
    attn_tc_backward_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_g,
                            const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                            const AttnTcArgs args) {
    using Lay = AttnBwdLayout<DP>;
    constexpr int S = Lay::kStages, KB = Lay::kBoxes, NB = Lay::kBufs;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    unsigned char* smem = smem_raw + ((1024 - (smem_addr(smem_raw) & 1023)) & 1023);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + Lay::kSlot);
    const bool keys = int(blockIdx.x) < args.kv_blocks;
    if (threadIdx.x == 0) {
        uint64_t* fixed = reinterpret_cast<uint64_t*>(smem + Lay::kBars);
        uint64_t *full = fixed + 1, *empty = full + S, *sfull = empty + S, *pfull = sfull + NB, *done = pfull + NB;
        mbar_init(fixed, 4 * KB);
        for (int s = 0; s < S; ++s) {
            mbar_init(&full[s], 2 * KB + (keys ? 2 : 0));
            mbar_init(&empty[s], 1);
        }
        for (int g = 0; g < NB; ++g) {
            mbar_init(&sfull[g], 2);
            mbar_init(&pfull[g], 4);  // as in the forward
            mbar_init(&done[g], 1);
        }
        mbar_init(done + NB, 1);  // finished
        mbar_fence_init();
    }
    if ((threadIdx.x >> 5) == 1) {
        tmem_alloc(tmem_slot, Lay::kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
    grid_dependency_wait();
    launch_dependents();
    if (keys)
        attn_tc_backward_block<T, DP, true>(map_k, map_v, map_q, map_g, args, int(blockIdx.x), smem, tmem);
    else
        attn_tc_backward_block<T, DP, false>(map_q, map_g, map_k, map_v, args, int(blockIdx.x) - args.kv_blocks, smem,
                                             tmem);
    tc_fence_before();
    __syncthreads();
    if ((threadIdx.x >> 5) == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, Lay::kTmemCols);
    }
}

// ---- what the kernels above are given ---------------------------------------------------------------------------
// Open-pair bits and tile flags from the byte masks. A block takes 128 queries x 128 keys of one (image, head) of the
// mask: a warp's ballot makes a row's word, and the words of 32 rows, transposed through shared memory, a key's.
struct PackArgs {
    const uint8_t* mask;     // as in AttnArgs; or null: one row per image, from the padding alone
    const uint8_t* padding;
    long long m_b, m_h, m_q;
    uint32_t* row_bits;      // [images, heads, rows, words]
    uint8_t* row_flags;      // [images, heads, row tiles of 128, tiles of 64 keys]
    uint32_t* col_bits;      // [mask images, heads, N, q words], or null
    uint8_t* col_flags;      // [mask images, heads, key tiles of 128, tiles of 64 queries]
    int images, heads, rows, N;      // rows: Q, or 1 without a mask
    int mask_images;                 // images the mask itself has (col_bits exist for these)
    int words, col_words;            // 2 * ceil(N / 64), 2 * ceil(Q / 64)
};

constexpr int kPackThreads = 512;
__global__ void __launch_bounds__(kPackThreads) attn_pack_kernel(const PackArgs a) {
    __shared__ uint32_t pairs[128][4], all_rows[128][4];  // the mask's bits, and with the padding's
    __shared__ uint32_t cols[128][4];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int q_tiles = (a.rows + 127) / 128, k_tiles = (a.N + 127) / 128;
    int x = blockIdx.x;
    const int kt = x % k_tiles;
    x /= k_tiles;
    const int qt = x % q_tiles;
    x /= q_tiles;
    const int h = x % a.heads, b = x / a.heads;
    grid_dependency_wait();
    launch_dependents();
    const uint8_t* mask = a.mask == nullptr ? nullptr : a.mask + b * a.m_b + h * a.m_h;
    const uint8_t* pad = a.padding == nullptr ? nullptr : a.padding + (long long)b * a.N;
    uint32_t padded[4];
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const int j = kt * 128 + 32 * w + lane;
        padded[w] = __ballot_sync(0xffffffffu, j < a.N && (pad == nullptr || pad[j] == 0));
    }
    // four rows a warp at a time, so that 16 loads are in flight
    const int rows = min(128, a.rows - qt * 128);
    for (int r0 = warp * 4; r0 < 128; r0 += kPackThreads / 8) {
        bool open[4][4];
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const int j = kt * 128 + 32 * w + lane;
                open[x][w] = r0 + x < rows && j < a.N &&
                             (mask == nullptr || __ldg(mask + (long long)(qt * 128 + r0 + x) * a.m_q + j) == 0);
            }
#pragma unroll
        for (int x = 0; x < 4; ++x)
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const uint32_t word = __ballot_sync(0xffffffffu, open[x][w]);
                if (lane == w) {
                    pairs[r0 + x][w] = word;
                    all_rows[r0 + x][w] = word & padded[w];
                }
            }
    }
    __syncthreads();
    const long long bh = (long long)b * a.heads + h;
    for (int e = threadIdx.x; e < 128 * 4; e += kPackThreads) {
        const int i = qt * 128 + e / 4, w = kt * 4 + e % 4;
        if (i < a.rows && w < a.words) a.row_bits[(bh * a.rows + i) * a.words + w] = all_rows[e / 4][e % 4];
    }
    if (warp < 2) {  // flags of the block's two 128 x 64 tiles
        const int t = kt * 2 + warp;
        uint32_t any = 0, every = 0xffffffffu;
        for (int r = lane; r < 128; r += 32) {
            const uint32_t w0 = all_rows[r][2 * warp], w1 = all_rows[r][2 * warp + 1];
            any |= w0 | w1;
            if (qt * 128 + r < a.rows) every &= w0 & w1;
        }
        const bool some = __any_sync(0xffffffffu, any != 0), full = __all_sync(0xffffffffu, every == 0xffffffffu);
        const int tiles = a.words / 2;
        if (lane == 0 && t < tiles) a.row_flags[(bh * q_tiles + qt) * tiles + t] = uint8_t(some) | uint8_t(full) << 1;
    }
    if (a.col_bits == nullptr || b >= a.mask_images) return;
    for (int e = threadIdx.x; e < 128 * 4; e += kPackThreads) {
        const int key = e % 128, qw = e / 128;
        uint32_t word = 0;
#pragma unroll 8
        for (int r = 0; r < 32; ++r) word |= ((pairs[32 * qw + r][key / 32] >> (key % 32)) & 1u) << r;
        cols[key][qw] = word;
        const int j = kt * 128 + key, w = qt * 4 + qw;
        if (j < a.N && w < a.col_words) a.col_bits[(bh * a.N + j) * a.col_words + w] = word;
    }
    __syncthreads();
    if (warp < 2) {  // flags of the block's two tiles of 128 keys x 64 queries
        const int t = qt * 2 + warp;
        uint32_t any = 0, every = 0xffffffffu;
        const int left = a.rows - (qt * 128 + 64 * warp);  // queries of this tile
        const unsigned long long range = left >= 64 ? ~0ull : left <= 0 ? 0ull : (1ull << left) - 1ull;
        for (int k = lane; k < 128; k += 32) {
            const uint32_t w0 = cols[k][2 * warp], w1 = cols[k][2 * warp + 1];
            any |= w0 | w1;
            if (kt * 128 + k < a.N) every &= (w0 | ~uint32_t(range)) & (w1 | ~uint32_t(range >> 32));
        }
        const bool some = __any_sync(0xffffffffu, any != 0), full = __all_sync(0xffffffffu, every == 0xffffffffu);
        const int tiles = a.col_words / 2;
        if (lane == 0 && t < tiles) a.col_flags[(bh * k_tiles + kt) * tiles + t] = uint8_t(some) | uint8_t(full) << 1;
    }
}

// delta as in attn_delta_kernel for 16-bit types with D a multiple of 8: 16-byte loads, `lanes` (a power of two, at
// least D / 8) threads a row, `parts` CTAs for the rows of each (image, key head), its whole group of query heads.
// float16: keys_lse takes lse less attn_p_bits, row_g each row's |dO|^2, amax the largest of them in the CTA's rows and
// the largest |V|^2 in its share of the keys that are there (a maximum of maxima has no order).
constexpr int kDeltaThreads = 512;
template <typename T>
__global__ void __launch_bounds__(kDeltaThreads)
    attn_delta_tc_kernel(const AttnArgs a, int lanes, int parts, float* keys_lse, float* row_g, float* amax) {
    constexpr bool kHalf = std::is_same<T, __half>::value;
    const int sub = threadIdx.x % lanes, bhk = blockIdx.x / parts, part = blockIdx.x % parts;
    const long long step = (long long)parts * (kDeltaThreads / lanes);
    const long long first = (long long)part * (kDeltaThreads / lanes) + threadIdx.x / lanes;
    const bool col = sub * 8 < a.D;
    grid_dependency_wait();
    launch_dependents();
    float top_g = 0.f, top_v = 0.f;
    const long long rows = (long long)(a.H / a.Hk) * a.Qp;  // of (image, key head) bhk, which lie together
    // whole warps take the same number of turns (a warp holds whole rows)
    for (long long r = first, warp0 = first - threadIdx.x % 32 / lanes; warp0 < rows; r += step, warp0 += step) {
        const long long row = bhk * rows + r, bh = row / a.Qp;
        const int i = int(row % a.Qp);
        float sum = 0.f, square = 0.f;
        if (r < rows && i < a.Q && col) {
            const long long at = ((bh / a.H * a.Q + i) * a.H + bh % a.H) * a.D + sub * 8;
            float o[8], g[8], e[8];
            load16<T>(static_cast<const T*>(a.out_in) + at, o);
            load16<T>(static_cast<const T*>(a.grad_out) + at, g);
            load16<T>(static_cast<const T*>(a.rest_in) + at, e);
#pragma unroll
            for (int x = 0; x < 8; ++x) {
                sum += (o[x] + e[x]) * g[x];
                if constexpr (kHalf) square += g[x] * g[x];
            }
        }
        for (int x = lanes / 2; x > 0; x >>= 1) {
            sum += __shfl_xor_sync(0xffffffffu, sum, x);
            if constexpr (kHalf) square += __shfl_xor_sync(0xffffffffu, square, x);
        }
        top_g = fmaxf(top_g, square);
        if (r < rows && sub == 0) {
            static_cast<float*>(a.delta)[row] = sum;
            if constexpr (kHalf) {
                row_g[row] = square;
                keys_lse[row] = static_cast<const float*>(a.lse)[row] - float(attn_p_bits<T>());
            }
        }
    }
    if constexpr (kHalf) {
        const long long b = bhk / a.Hk;
        const T* values = static_cast<const T*>(a.v) + b * a.v_b + bhk % a.Hk * a.v_h + sub * 8;
        const uint8_t* pad = a.padding == nullptr ? nullptr : a.padding + b * a.N;
        for (long long j = first, warp0 = first - threadIdx.x % 32 / lanes; warp0 < a.N; j += step, warp0 += step) {
            float v[8], square = 0.f;
            if (j < a.N && col && (pad == nullptr || pad[j] == 0)) {
                load16<T>(values + j * a.v_t, v);
#pragma unroll
                for (int x = 0; x < 8; ++x) square += v[x] * v[x];
            }
            for (int x = lanes / 2; x > 0; x >>= 1) square += __shfl_xor_sync(0xffffffffu, square, x);
            top_v = fmaxf(top_v, square);
        }
        __shared__ float tops[2][kDeltaThreads / 32];
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) {
            top_g = fmaxf(top_g, __shfl_xor_sync(0xffffffffu, top_g, x));
            top_v = fmaxf(top_v, __shfl_xor_sync(0xffffffffu, top_v, x));
        }
        if (threadIdx.x % 32 == 0) {
            tops[0][threadIdx.x / 32] = top_g;
            tops[1][threadIdx.x / 32] = top_v;
        }
        __syncthreads();
        if (threadIdx.x < 2) {
            float top = 0.f;
            for (int x = 0; x < kDeltaThreads / 32; ++x) top = fmaxf(top, tops[threadIdx.x][x]);
            amax[(long long)threadIdx.x * gridDim.x + blockIdx.x] = top;
        }
    }
}

}  // namespace td
