// td_fp8_tc.cuh -- the product of two e4m3 operands on tcgen05 tensor cores, with a scale for each block of 128.
//
//   out[m, n] = act(sum_kb sa[m, kb] sb[n, kb] sum_{k in block kb} a[m, k] b[n, k] + bias[n])
//
// A block of K is one 128-byte row of a swizzled tile: four tcgen05.mma of kind::f8f6f4 (M = 128, N = BN, K = 32) sum
// its 128 products in TMEM, from zero, and the epilogue warps add that times the scales to float32 registers while the
// tensor cores work on the next block in another part of TMEM. The scales are so any float32 numbers, and the tensor
// cores' own sums are never longer than 128 products, however long K is. What bounds it: a 128 x 256 block takes the
// tensor cores 512 cycles, shared memory 768 by count (48 KB in, 48 KB out, 128 bytes a cycle) and the 8 epilogue warps
// about 890 each (128 multiply-adds, 128 columns from TMEM, waits); with two TMEM buffers between them it goes around
// in 1100. Three sets of operands in turn, 16-bit results: 8192 x 4096 x 4096 in 145 us (1.90 PFLOP/s), 177784 x 1024
// x 256 72, 177784 x 256 x 1024 97, 2400 x 256 x 1024 5.6, 300 x 256 x 1024 4.3. Where K is short a tile's end counts
// as much as its blocks: 67200 x 256 x 1024 38.5, with a bias 44; 177784 rows of it with 8-bit results 100, with a bias
// 123, GELU as well 306.
//
// Persistent, one CTA an SM, output tiles of 128 x BN (columns fastest, so that the CTAs which share rows of A run
// together). A tile's K may be split over `splits` units whose float32 parts another kernel adds in order (a long sum
// behind few tiles: the weight's gradient). Roles: warps 0 - 7 the epilogue (TMEM lanes 32 (w % 4) .., columns
// w / 4 * BN / 2 ..), warp 8 the TMA producers, two lanes a slot (as in td_gemm_tc.cuh, whose notes on the waits apply
// here), warp 9 the MMA issuer (10 and 11 fill its warpgroup).
// COLS (the weight's gradient): both operands are laid out a block of K at a time, so that a tile is bytes that follow
// one another in memory, and B has a scale for each row and block, which the producers bring to shared memory.
// In 8-bit results a block of 128 columns of a row is one thread's (BN = 256), or two threads' (BN = 128).
#pragma once

#include "td_fp8_simt.cuh"

namespace td {

constexpr int kTc8Threads = 384, kTc8Epi = 8, kTc8Rows = 128;
constexpr int kTc8Ring = 8;  // blocks whose scales an epilogue thread has at hand or on their way

struct Tc8Args {
    const float *sa, *sb;
    long long sa_row, sa_k, sb_row, sb_k;  // sb: of a block of 128 rows; COLS: of a row (sb_row = 1)
    End8 end;
    float* partial;  // splits > 1: [splits][M][N], instead of end's output
    int M, N, k_blocks, n_tiles, tiles, splits, kb_per_split;
    int boxes;  // the output's rows start on 16-byte boundaries: map_out (boxes of 32 rows x 128 bytes) stores it
};

template <int BN, bool COLS>
struct Tc8Layout {
    static constexpr int kStages = BN == 256 ? 3 : 5;
    static constexpr int kBufs = 512 / BN;  // of BN TMEM columns
    static constexpr uint32_t kABytes = kTc8Rows * 128, kBBytes = BN * 128, kStageBytes = kABytes + kBBytes;
    // bytes of results a warp stages: two boxes of 32 rows x 128 bytes, or one (and 32 x 33 floats)
    static constexpr size_t kStageOut = BN == 256 ? 8192 : 5120;
    static constexpr size_t kOutOffset = size_t(kStages) * kStageBytes;
    static constexpr size_t kScaleOffset = kOutOffset + kTc8Epi * kStageOut;
    static constexpr size_t kBiasOffset = kScaleOffset + (COLS ? size_t(kStages) * BN * 4 : 0);
    // a warp's columns of the bias, as they come and as float32 (COLS: products without one)
    static constexpr size_t kTopOffset = kBiasOffset + (COLS ? 0 : 2 * kTc8Epi * (BN / 2) * 4);
    static constexpr size_t kRingOffset = kTopOffset + 2 * kTc8Rows * 4;
    static constexpr size_t kBarOffset = kRingOffset + kTc8Ring * (kTc8Epi * 32 + kTc8Epi) * 4;
    static constexpr size_t kSlotOffset = kBarOffset + (4 * kStages + 2 * kBufs) * 8;
    static constexpr size_t kBytes = kSlotOffset + 16 + 1024;  // + alignment of the tiles
};

// The issuing thread and the epilogue's warps go around once a block of K, and each instruction on the issuing thread's
// way costs about six cycles: barriers are plain addresses here, descriptors a changing low and a constant high word.
__device__ __forceinline__ bool mbar_try_at(uint32_t bar, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    return done != 0;
}
// Wait for the phase with the given parity; false (and the error word set) after about a second.
__device__ __forceinline__ bool mbar_wait_at(uint32_t bar, uint32_t parity, unsigned int err_code) {
    if (mbar_try_at(bar, parity)) return true;
    const long long t0 = clock64();
    while (!mbar_try_at(bar, parity)) {
        if (clock64() - t0 > kSpinLimitCycles) {
            record_error(err_code);
            return false;
        }
    }
    return true;
}
__device__ __forceinline__ void mbar_arrive_at(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void mma_commit_at(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
// D[tmem] = (the first: , the others: +=) A B^T of the 4 K steps of a block; a_lo, b_lo: the low words of the tiles'
// descriptors, whose K steps are 32 bytes apart.
__device__ __forceinline__ void mma_f8_block(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t hi,
                                             uint32_t idesc) {
    asm volatile(
        "{\n\t.reg .pred no, yes;\n\t.reg .b64 a, b;\n\t.reg .b32 x, y;\n\t"
        "setp.ne.b32 no, %3, %3;\n\tsetp.eq.b32 yes, %3, %3;\n\t"
        "mov.b64 a, {%1, %3};\n\tmov.b64 b, {%2, %3};\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a, b, %4, no;\n\t"
        "add.u32 x, %1, 2;\n\tadd.u32 y, %2, 2;\n\tmov.b64 a, {x, %3};\n\tmov.b64 b, {y, %3};\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a, b, %4, yes;\n\t"
        "add.u32 x, %1, 4;\n\tadd.u32 y, %2, 4;\n\tmov.b64 a, {x, %3};\n\tmov.b64 b, {y, %3};\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a, b, %4, yes;\n\t"
        "add.u32 x, %1, 6;\n\tadd.u32 y, %2, 6;\n\tmov.b64 a, {x, %3};\n\tmov.b64 b, {y, %3};\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], a, b, %4, yes;\n\t}"
        ::"r"(d_tmem), "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc)
        : "memory");
}

// 4 bytes from global to shared memory.
__device__ __forceinline__ void copy4(uint32_t dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}

// `bytes` (a multiple of 16) from global to shared memory, both 16-byte aligned, completing on the mbarrier.
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(smem_addr(dst)), "l"(src), "r"(bytes), "r"(smem_addr(bar))
                 : "memory");
}

// tcgen05.wait::ld, on which the registers of an outstanding load depend.
__device__ __forceinline__ void tmem_ld_wait_for(uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]),
                   "+r"(r[15])
                 :
                 : "memory");
}

// Block k of the rows from `row` on, of rows along K or (BLOCKS) of a tensor laid out a block at a time.
template <bool BLOCKS>
__device__ __forceinline__ void load_box(void* dst, const CUtensorMap* map, uint64_t* bar, int k, int row,
                                         uint64_t pol) {
    if constexpr (BLOCKS) tma_load_3d(dst, map, bar, 0, row, k, pol);
    else tma_load_2d(dst, map, bar, k * kBlock8, row, pol);
}

// 3-D tiled store of the box at (x, y, z) from shared memory; what lies outside the tensor is not written. x * element
// size is a multiple of 16 bytes, no coordinate is negative.
__device__ __forceinline__ void tma_store_box(const CUtensorMap* map, const void* src, int x, int y, int z) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];"
                 ::"l"(reinterpret_cast<uint64_t>(map)), "r"(smem_addr(src)), "r"(x), "r"(y), "r"(z)
                 : "memory");
}

template <int BN, typename T, bool COLS>
__global__ void __launch_bounds__(kTc8Threads, 1)
    fp8_product_tc_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                          const __grid_constant__ CUtensorMap map_out, const Tc8Args a) {
    using Lay = Tc8Layout<BN, COLS>;
    constexpr int S = Lay::kStages, NB = Lay::kBufs, CW = BN / 2;
    constexpr bool kTo8 = sizeof(T) == 1;
    constexpr bool kShare = kTo8 && CW < kBlock8;  // a block's maximum is found by two threads
    extern __shared__ __align__(16) unsigned char smem_raw[];
    unsigned char* smem = smem_raw + ((1024 - (smem_addr(smem_raw) & 1023)) & 1023);
    float* scales = reinterpret_cast<float*>(smem + Lay::kScaleOffset);
    float* tops = reinterpret_cast<float*>(smem + Lay::kTopOffset);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + Lay::kBarOffset);
    uint64_t *empty = full + S, *sfull = empty + S, *sempty = sfull + S, *tfull = sempty + S, *tempty = tfull + NB;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + Lay::kSlotOffset);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) {
            mbar_init(&full[s], 2);
            mbar_init(&empty[s], 1);
            mbar_init(&sfull[s], 1);
            mbar_init(&sempty[s], kTc8Epi);
        }
        for (int i = 0; i < NB; ++i) {
            mbar_init(&tfull[i], 1);
            mbar_init(&tempty[i], kTc8Epi);
        }
        mbar_fence_init();
        tma_prefetch_desc(&map_a);
        tma_prefetch_desc(&map_b);
        if (a.boxes) tma_prefetch_desc(&map_out);
    }
    __syncwarp();
    if (warp == 9) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const int units = a.tiles * a.splits;
    // unit -> its first block of K and how many it has
    auto first_kb = [&](int unit) { return a.splits == 1 ? 0 : unit / a.tiles * a.kb_per_split; };
    auto count_kb = [&](int unit) {
        return a.splits == 1 ? a.k_blocks : min(a.kb_per_split, a.k_blocks - first_kb(unit));
    };
    auto tile_of = [&](int unit, int& m0, int& n0) {
        const int t = a.splits == 1 ? unit : unit % a.tiles, mt = t / a.n_tiles;
        m0 = mt * kTc8Rows;
        n0 = (t - mt * a.n_tiles) * BN;
    };
    // The epilogue's sums want more registers than an even share: 256 threads of 224 and 128 of 56 are the
    // 64512 that the block has at 168 each, exactly.
    if (warp >= kTc8Epi) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        if (warp == 8) {
            // lanes 2s, 2s + 1: the boxes of A and B of slot s; lane 2S + s (COLS): B's scales of their own ring
            const bool scale_lane = lane >= 2 * S;
            const int s = scale_lane ? lane - 2 * S : lane >> 1;
            if (lane < (COLS ? 3 * S : 2 * S)) {
                uint64_t* const free = scale_lane ? &sempty[s] : &empty[s];
                uint64_t* const landed = scale_lane ? &sfull[s] : &full[s];
                // (A's rows are read by the CTAs that run together, B by all)
                const uint64_t pol_a = l2_evict_first(), pol_b = l2_evict_last();
                int unit = blockIdx.x, kb = s, round = 0;
                grid_dependency_wait();
                launch_dependents();
                long long t0 = clock64();  // (the time that the kernel before this one takes does not count)
                // (a last pass only waits, so that nothing is still to arrive on the slot when the CTA exits)
                for (;;) {
                    while (unit < units && kb >= count_kb(unit)) {
                        kb -= count_kb(unit);
                        unit += gridDim.x;
                    }
                    if (mbar_test(free, uint32_t(round & 1) ^ 1u)) {
                        if (unit >= units) break;
                        int m0, n0;
                        tile_of(unit, m0, n0);
                        const int k = first_kb(unit) + kb;
                        if (scale_lane) {
                            mbar_arrive_expect_tx(landed, BN * 4);
                            bulk_load(scales + s * BN, a.sb + n0 + k * a.sb_k, BN * 4, landed);
                        } else if ((lane & 1) == 0) {
                            mbar_arrive_expect_tx(landed, Lay::kABytes);
                            load_box<COLS>(smem + s * Lay::kStageBytes, &map_a, landed, k, m0, pol_a);
                        } else {
                            mbar_arrive_expect_tx(landed, Lay::kBBytes);
                            load_box<COLS>(smem + s * Lay::kStageBytes + Lay::kABytes, &map_b, landed, k, n0, pol_b);
                        }
                        ++round;
                        kb += S;
                        t0 = clock64();
                    } else if (clock64() - t0 > kSpinLimitCycles) {
                        record_error(kErrSlotWait);
                        if (round > 0) mbar_wait(landed, uint32_t(round - 1) & 1u, kErrTmaWait);
                        break;
                    } else {
                        __nanosleep(32);
                    }
                }
            }
        } else if (warp == 9) {
            if (lane == 0) {
                // f32 accumulator, e4m3 (format 0) by e4m3, both K-major
                constexpr uint32_t idesc = (1u << 4) | (uint32_t(BN >> 3) << 17) | (uint32_t(kTc8Rows >> 4) << 24);
                const uint64_t first = sdesc_sw128(smem_addr(smem));
                const uint32_t hi = uint32_t(first >> 32), lo = uint32_t(first);
                const uint32_t full0 = smem_addr(full), empty0 = smem_addr(empty), tfull0 = smem_addr(tfull),
                               tempty0 = smem_addr(tempty);
                uint32_t s = 0, b = 0, s_phase = 0, b_phase = 1;
                bool ok = true;
                // its waits give up after a second of their own, not of the kernel's before this one
                grid_dependency_wait();
                for (int unit = blockIdx.x; ok && unit < units; unit += gridDim.x) {
                    for (int kb = count_kb(unit); kb > 0; --kb) {
                        ok = mbar_wait_at(tempty0 + 8 * b, b_phase, kErrSlotWait) &&
                             mbar_wait_at(full0 + 8 * s, s_phase, kErrTmaWait);
                        if (!ok) break;
                        tc_fence_after();
                        const uint32_t a_lo = lo + s * (Lay::kStageBytes >> 4);
                        mma_f8_block(tmem + b * BN, a_lo, a_lo + (Lay::kABytes >> 4), hi, idesc);
                        mma_commit_at(empty0 + 8 * s);
                        mma_commit_at(tfull0 + 8 * b);
                        if (++s == S) {
                            s = 0;
                            s_phase ^= 1;
                        }
                        if (++b == NB) {
                            b = 0;
                            b_phase ^= 1;
                        }
                    }
                }
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
        const int quarter = warp & 3, c_lo = warp / 4 * CW;
        const uint32_t lanes = tmem + (uint32_t(quarter * 32) << 16) + uint32_t(c_lo);
        unsigned char* const staged = smem + Lay::kOutOffset + warp * Lay::kStageOut;
        const int n_blocks = (a.N + kBlock8 - 1) / kBlock8;
        bool dead = false;  // after a wait that gave up: walk on and meet at the barriers, but wait and store no more
        const uint32_t tfull0 = smem_addr(tfull), tempty0 = smem_addr(tempty), sfull0 = smem_addr(sfull),
                       sempty0 = smem_addr(sempty);
        uint32_t at_b = 0, b_phase = 0, at_s = 0, s_phase = 0, slot = 0;
        // The scales of the blocks ahead, over the tiles' borders: each thread copies its row's, and lane 0 the warp's
        // of B, into rings of their own. (Read where they are used, they cost more than all else: 262 us for the 136
        // of the same products without scales, at 8192 x 4096 x 4096.)
        float* const ring_a = reinterpret_cast<float*>(smem + Lay::kRingOffset) + threadIdx.x;
        float* const ring_b = reinterpret_cast<float*>(smem + Lay::kRingOffset) + kTc8Ring * kTc8Epi * 32 + warp;
        int next_unit = blockIdx.x, next_left = 0, next_slot = 0;
        const float *next_sa = nullptr, *next_sb = nullptr;
        auto fetch = [&] {
            if (next_unit < units) {
                if (next_left == 0) {
                    int m0, n0;
                    tile_of(next_unit, m0, n0);
                    const long long k0 = first_kb(next_unit);
                    next_left = count_kb(next_unit);
                    next_sa = a.sa + (long long)min(m0 + quarter * 32 + lane, a.M - 1) * a.sa_row + k0 * a.sa_k;
                    if (!COLS) next_sb = a.sb + min((n0 + c_lo) / kBlock8, n_blocks - 1) * a.sb_row + k0 * a.sb_k;
                }
                copy4(smem_addr(ring_a + next_slot * kTc8Epi * 32), next_sa);
                if (!COLS && lane == 0) copy4(smem_addr(ring_b + next_slot * kTc8Epi), next_sb);
                next_sa += a.sa_k;
                if (!COLS) next_sb += a.sb_k;
                if (--next_left == 0) next_unit += gridDim.x;
                next_slot = next_slot + 1 == kTc8Ring ? 0 : next_slot + 1;
            }
            copy_commit();
        };
        // the warp's columns of the next unit's bias, as they are in memory, on their way while a unit's products are
        // added; they are added behind the products, so that a large one is rounded once and not with every block
        const bool biased = !COLS && a.end.bias != nullptr;
        unsigned char* const raw_bias = smem + Lay::kBiasOffset + warp * CW * 4;
        float* const wide_bias = reinterpret_cast<float*>(raw_bias + kTc8Epi * CW * 4);
        const int bias_shift = a.end.bias_dtype == 0 ? 2 : 1;  // log2 of its bytes
        const bool bias_words = (reinterpret_cast<uintptr_t>(a.end.bias) & 3) == 0;
        auto fetch_bias = [&](int next) {
            if (next < units) {
                int m0, n0;
                tile_of(next, m0, n0);
                const int n = n0 + c_lo;
                const char* const src = static_cast<const char*>(a.end.bias) + ((long long)n << bias_shift);
                const int bytes = min(CW, a.N - n) << bias_shift;  // (none behind the last column)
                for (int i = lane * 4; i < bytes; i += 128) {
                    if (bias_words && i + 4 <= bytes) {
                        copy4(smem_addr(raw_bias + i), src + i);
                    } else {  // (a float32 bias comes in words)
                        *reinterpret_cast<uint16_t*>(raw_bias + i) = *reinterpret_cast<const uint16_t*>(src + i);
                        if (i + 4 <= bytes)
                            *reinterpret_cast<uint16_t*>(raw_bias + i + 2) =
                                *reinterpret_cast<const uint16_t*>(src + i + 2);
                    }
                }
            }
            copy_commit();
        };
        grid_dependency_wait();
        if (biased) fetch_bias(blockIdx.x);
#pragma unroll
        for (int i = 0; i < kTc8Ring - 1; ++i) fetch();
        int behind = kTc8Ring - 1;  // groups of copies behind the bias's
        for (int unit = blockIdx.x; unit < units; unit += gridDim.x) {
            int m0, n0;
            tile_of(unit, m0, n0);
            const int row = quarter * 32 + lane, m = m0 + row, n = n0 + c_lo;
            const int count = count_kb(unit);
            float v[CW];
#pragma unroll
            for (int i = 0; i < CW; ++i) v[i] = 0.f;
            if (biased) {
                if (behind > 1) copy_wait<2>();
                else copy_wait<1>();
                __syncwarp();
#pragma unroll
                for (int i = lane; i < CW; i += 32) {
                    float f = 0.f;
                    if (n + i < a.N) {
                        if (a.end.bias_dtype == 0) f = reinterpret_cast<const float*>(raw_bias)[i];
                        else if (a.end.bias_dtype == 1) f = to_acc(reinterpret_cast<const __half*>(raw_bias)[i]);
                        else f = to_acc(reinterpret_cast<const __nv_bfloat16*>(raw_bias)[i]);
                    }
                    wide_bias[i] = f;
                }
                __syncwarp();
                fetch_bias(unit + gridDim.x);
                behind = count;
            }
            for (int kb = 0; kb < count; ++kb) {
                copy_wait<kTc8Ring - 2>();
                __syncwarp();
                const float f = ring_a[slot * kTc8Epi * 32] * (COLS ? 1.f : ring_b[slot * kTc8Epi]);
                fetch();
                const uint32_t b = at_b, s = at_s;  // TMEM buffer, slot of B's scales
                bool ready = !dead && mbar_wait_at(tfull0 + 8 * b, b_phase, kErrMmaWait);
                if (COLS) ready = ready && mbar_wait_at(sfull0 + 8 * s, s_phase, kErrTmaWait);
                dead = !__all_sync(0xffffffffu, ready);
                slot = (slot + 1) % kTc8Ring;
                if (++at_b == NB) {
                    at_b = 0;
                    b_phase ^= 1;
                }
                if (COLS && ++at_s == S) {
                    at_s = 0;
                    s_phase ^= 1;
                }
                if (dead) continue;
                tc_fence_after();
                // a chunk of 16 columns is on its way from TMEM while the one before it is added
                uint32_t v0[16], v1[16];
                auto add = [&](int j, const uint32_t(&w)[16]) {
#pragma unroll
                    for (int i = 0; i < 16; i += 4) {
                        float4 c = make_float4(f, f, f, f);
                        if constexpr (COLS) {
                            c = *reinterpret_cast<const float4*>(scales + s * BN + c_lo + j + i);
                            c.x *= f; c.y *= f; c.z *= f; c.w *= f;
                        }
                        float* const to = v + j + i;
                        to[0] = fmaf(__uint_as_float(w[i]), c.x, to[0]);
                        to[1] = fmaf(__uint_as_float(w[i + 1]), c.y, to[1]);
                        to[2] = fmaf(__uint_as_float(w[i + 2]), c.z, to[2]);
                        to[3] = fmaf(__uint_as_float(w[i + 3]), c.w, to[3]);
                    }
                };
                const uint32_t from = lanes + uint32_t(b * BN);
                tmem_ld_32x32b_x16(from, v0);
                tmem_ld_wait_for(v0);
#pragma unroll
                for (int j = 0; j < CW; j += 32) {
                    tmem_ld_32x32b_x16(from + uint32_t(j + 16), v1);
                    add(j, v0);
                    tmem_ld_wait_for(v1);
                    if (j + 32 < CW) {
                        tmem_ld_32x32b_x16(from + uint32_t(j + 32), v0);
                    } else {  // all of it is in registers
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive_at(tempty0 + 8 * b);
                    }
                    add(j + 16, v1);
                    if (j + 32 < CW) tmem_ld_wait_for(v0);
                }
                if constexpr (COLS) {
                    __syncwarp();
                    if (lane == 0) mbar_arrive_at(sempty0 + 8 * s);
                }
            }
            // the end: bias, activation, and the row's CW columns out
            if (biased) {
#pragma unroll
                for (int i = 0; i < CW; i += 4) {
                    const float4 c = *reinterpret_cast<const float4*>(wide_bias + i);
                    v[i] += c.x; v[i + 1] += c.y; v[i + 2] += c.z; v[i + 3] += c.w;
                }
            }
            // the boxes of the unit before have been read (they are written again from here on)
            if (lane < 2) bulk_wait_read();
            __syncwarp();
            if (a.end.act == kActRelu) {
#pragma unroll
                for (int i = 0; i < CW; ++i) v[i] = activate(v[i], kActRelu);
            } else if (a.end.act == kActGelu) {
#pragma unroll
                for (int i = 0; i < CW; ++i) v[i] = activate(v[i], kActGelu);
            } else if (a.end.act == kActSilu) {
#pragma unroll
                for (int i = 0; i < CW; ++i) v[i] = activate(v[i], kActSilu);
            }
            const bool stores = !dead && m < a.M;
            if constexpr (kTo8) {
                if (n + CW > a.N) {  // (products of zeros, but for NaN in A's row or the scales)
#pragma unroll
                    for (int i = 0; i < CW; ++i)
                        if (n + i >= a.N) v[i] = 0.f;
                }
                float top = largest<CW>(v);
                if (infinite(top)) {
                    drop_infinities<CW>(v);
                    top = largest<CW>(v);
                }
                if constexpr (kShare) {
                    named_barrier(1, kTc8Epi * 32);  // (the unit before's are read)
                    tops[(warp / 4) * kTc8Rows + row] = top;
                    named_barrier(1, kTc8Epi * 32);
                    top = fmaxf(top, tops[(1 - warp / 4) * kTc8Rows + row]);
                }
                const int e = scale_exponent(top);
                const float inv = exp2_int(-e);
                if (stores && n < a.N && n % kBlock8 == 0)
                    a.end.scale[(long long)m * n_blocks + n / kBlock8] = exp2_int(e);
                if constexpr (CW == kBlock8) {  // a row of 128 bytes: the warp's one box
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        uint4 w;
                        w.x = to_e4m3x4(v + 16 * i, inv);
                        w.y = to_e4m3x4(v + 16 * i + 4, inv);
                        w.z = to_e4m3x4(v + 16 * i + 8, inv);
                        w.w = to_e4m3x4(v + 16 * i + 12, inv);
                        *reinterpret_cast<uint4*>(staged + lane * 128 + ((i ^ (lane & 7)) << 4)) = w;
                    }
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0 && !dead && m < a.M && n < a.end.pitch) {
                        tma_store_box(&map_out, staged, n, m0 + quarter * 32, 0);
                        bulk_commit();
                    }
                } else if (stores) {
                    uint8_t* dst = static_cast<uint8_t*>(a.end.out) + (long long)m * a.end.pitch + n;
#pragma unroll
                    for (int i = 0; i < CW; i += 16) {
                        const uint4 w = make_uint4(to_e4m3x4(v + i, inv), to_e4m3x4(v + i + 4, inv),
                                                   to_e4m3x4(v + i + 8, inv), to_e4m3x4(v + i + 12, inv));
                        if (n + i < a.end.pitch) *reinterpret_cast<uint4*>(dst + i) = w;
                    }
                }
            } else if (a.boxes) {
                constexpr int kBoxCols = 128 / sizeof(T), kBoxes = CW / kBoxCols, kOnce = BN == 256 ? 2 : 1;
#pragma unroll
                for (int h = 0; h < kBoxes; h += kOnce) {
                    if (h > 0) {
                        if (lane < kOnce) bulk_wait_read();
                        __syncwarp();
                    }
#pragma unroll
                    for (int o = 0; o < kOnce; ++o)
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            store16<T>(reinterpret_cast<T*>(staged + o * 4096 + lane * 128 + ((i ^ (lane & 7)) << 4)),
                                       v + (h + o) * kBoxCols + i * (kBoxCols / 8));
                    fence_proxy_async_smem();
                    __syncwarp();
                    const int col = n + (h + lane) * kBoxCols, first = m0 + quarter * 32;
                    if (lane < kOnce && !dead && first < a.M && col < a.N) {
                        tma_store_box(&map_out, staged + lane * 4096, col, first,
                                      a.splits == 1 ? 0 : unit / a.tiles);
                        bulk_commit();
                    }
                }
            } else {  // rows that start anywhere: 32 x 32 results at a time, turned so that a warp stores a row's 32
                T* out = a.splits == 1 ? static_cast<T*>(a.end.out)
                                       : reinterpret_cast<T*>(a.partial + (long long)(unit / a.tiles) * a.M * a.N);
                float* const turned = reinterpret_cast<float*>(staged);
                const int first = m0 + quarter * 32, rows = dead ? 0 : min(32, a.M - first);
#pragma unroll
                for (int i = 0; i < CW; i += 32) {
                    __syncwarp();
#pragma unroll
                    for (int k = 0; k < 32; ++k) turned[lane * 33 + k] = v[i + k];
                    __syncwarp();
                    const int col = n + i + lane;
                    if (col < a.N) {
                        for (int r = 0; r < rows; ++r)
                            out[(long long)(first + r) * a.N + col] = from_acc<T>(turned[r * 33 + lane]);
                    }
                }
            }
        }
        bulk_wait_read();  // the CTA may exit once its stores have read the staged boxes
    }
    copy_wait<0>();
    tc_fence_before();
    __syncthreads();
    if (warp == 9) {
        __syncwarp();
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

}  // namespace td
