// td_fp8.cu -- the 8-bit entry points of the C ABI (quantising, products, their backward): argument contract, kernel
// choice, workspaces and launches.
#include <algorithm>
#include <type_traits>

#include "td_fp8.cuh"
#include "td_fp8_few.cuh"
#include "td_fp8_simt.cuh"
#include "td_fp8_tc.cuh"
#include "td_host.h"

namespace td {

cudaError_t fp8_device_error(int clear, unsigned int* code) {
    cudaError_t e = cudaMemcpyFromSymbol(code, g_device_error, sizeof(*code));
    if (e == cudaSuccess && clear) {
        const unsigned int zero = 0;
        e = cudaMemcpyToSymbol(g_device_error, &zero, sizeof(zero));
    }
    return e;
}

namespace {

using host::fail;

bool aligned(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
int64_t up(int64_t v, int64_t n) { return (v + n - 1) / n * n; }
int64_t blocks_of(int64_t v) { return (v + kBlock8 - 1) / kBlock8; }
bool wide_type(int dtype) { return dtype >= TD_F32 && dtype <= TD_BF16; }
size_t type_bytes(int dtype) { return dtype == TD_F32 ? 4 : dtype == TD_E4M3 ? 1 : 2; }

// Calls f with a value of the C++ type of a floating dtype.
template <typename F>
int by_type(int dtype, F f) {
    switch (dtype) {
        case TD_F32: return f(float());
        case TD_F16: return f(__half());
        default: return f(__nv_bfloat16());
    }
}

int check_sizes(int64_t M, int64_t K, int64_t N, char* err, size_t err_len) {
    if (M < 0 || M > TD_MAX_FP8_ROWS)
        return fail(err, err_len, TD_ERR_ARG, "rows must be between 0 and %d", TD_MAX_FP8_ROWS);
    if (K < 1 || K > TD_MAX_FP8_WIDTH || N < 1 || N > TD_MAX_FP8_WIDTH)
        return fail(err, err_len, TD_ERR_ARG, "widths must be between 1 and %d", TD_MAX_FP8_WIDTH);
    return TD_OK;
}

// 8-bit rows that this library writes: 16-byte aligned, `width` rounded up to 16 apart.
int check_written(const void* q, int64_t pitch, int64_t width, const float* scale, char* err, size_t err_len) {
    if (q == nullptr || scale == nullptr) return fail(err, err_len, TD_ERR_ARG, "null tensor pointer");
    if (pitch != up(width, 16) || !aligned(q, 16))
        return fail(err, err_len, TD_ERR_ARG, "8-bit rows must be 16-byte aligned, their width rounded up to 16 apart");
    return TD_OK;
}

// A workspace handed out in 256-byte steps from its first 256-byte boundary; with a null base it only counts.
struct Cut {
    uintptr_t at;
    size_t used = 0;
    explicit Cut(void* base) : at((reinterpret_cast<uintptr_t>(base) + 255) & ~uintptr_t(255)) {}
    template <typename T>
    T* take(int64_t count) {
        T* p = reinterpret_cast<T*>(at + used);
        used += size_t(up(count * int64_t(sizeof(T)), 256));
        return p;
    }
    size_t bytes() const { return used + 256; }
};

// ---- quantising -------------------------------------------------------------------------------------------------

int launch_rows(int dtype, const void* x, uint8_t* q, int64_t pitch, float* scale, int64_t M, int64_t K,
                cudaStream_t stream, char* err, size_t err_len) {
    RowsArgs a = {x, q, scale, M, int(K), int(blocks_of(K)), int(pitch)};
    return by_type(dtype, [&](auto zero) {
        using T = decltype(zero);
        constexpr int V = Elem<T>::kVec;
        if (K % kBlock8 == 0 && aligned(x, 32)) {
            const dim3 flat(unsigned(std::min<int64_t>((M * (K / 16) + 255) / 256, int64_t(kSms) * 8)));
            return host::launch(err, err_len, "fp8_flat_kernel", fp8_flat_kernel<T>, flat, dim3(kRowsThreads), 0,
                                stream, true, a);
        }
        const bool wide = K % V == 0 && aligned(x, 16);
        const int64_t tasks = M * ((K + 32 * (wide ? V : 4) - 1) / (32 * (wide ? V : 4)));
        const dim3 grid(unsigned(std::min<int64_t>((tasks + 7) / 8, int64_t(kSms) * 8)));
        return wide ? host::launch(err, err_len, "fp8_rows_kernel", fp8_rows_kernel<T, true>, grid, dim3(kRowsThreads),
                                   0, stream, true, a)
                    : host::launch(err, err_len, "fp8_rows_kernel", fp8_rows_kernel<T, false>, grid,
                                   dim3(kRowsThreads), 0, stream, true, a);
    });
}

// One launch of up to kTileJobs jobs (those with M > 0); dtype: the floating type of those that read one.
int launch_tiles(int dtype, TileJobs jobs, cudaStream_t stream, char* err, size_t err_len) {
    int64_t tiles = 0;
    for (int kind = 0; kind < kTileJobs; ++kind) {
        TileArgs& a = jobs.job[kind];
        const int64_t e = kind == kTileFrom8 ? 1 : int64_t(type_bytes(dtype)), step = kind == kTileFrom8 ? 8 : 16;
        a.CB = int(blocks_of(a.C));
        a.MB = int(blocks_of(a.M));
        a.wide = a.C % 8 == 0 && aligned(a.x, uintptr_t(step)) && a.ld * e % step == 0;
        tiles += int64_t(a.CB) * a.MB;
        a.end = tiles;
    }
    if (tiles > INT32_MAX) return fail(err, err_len, TD_ERR_ARG, "too many tiles");
    return by_type(dtype, [&](auto zero) {
        return host::launch(err, err_len, "fp8_tile_kernel", fp8_tile_kernel<decltype(zero)>, dim3(unsigned(tiles)),
                            dim3(kTileThreads), 0, stream, true, jobs);
    });
}

// Copies rows [M, K] of 8-bit data to 16-byte boundaries; *q and *pitch are the rows' own, then the copy's.
int launch_pitch(const uint8_t** q, long long* pitch, uint8_t* to, int64_t M, int64_t K, cudaStream_t stream,
                 char* err, size_t err_len) {
    const PitchArgs a = {*q, to, M, *pitch, up(K, 16), int(K)};
    *q = to;
    *pitch = up(K, 16);
    const dim3 grid(unsigned(std::min<int64_t>((M * (up(K, 16) / 16) + 255) / 256, int64_t(kSms) * 8)));
    return host::launch(err, err_len, "fp8_pitch_kernel", fp8_pitch_kernel, grid, dim3(256), 0, stream, true, a);
}

// ---- products ---------------------------------------------------------------------------------------------------

int launch_simt(const Operand8& a, const Operand8& b, const End8& end, int out_dtype, int64_t M, int64_t N, int64_t K,
                cudaStream_t stream, char* err, size_t err_len) {
    const int64_t tiles = (M + kSimtRows8 - 1) / kSimtRows8 * blocks_of(N);
    if (tiles > INT32_MAX) return fail(err, err_len, TD_ERR_ARG, "too many output tiles");
    auto go = [&](auto zero) {
        return host::launch(err, err_len, "fp8_product_simt_kernel", fp8_product_simt_kernel<decltype(zero)>,
                            dim3(unsigned(tiles)), dim3(kSimtThreads8), 0, stream, true, a, b, end,
                            static_cast<long long>(M), int(N), int(K));
    };
    return out_dtype == TD_E4M3 ? go(E4m3()) : by_type(out_dtype, go);
}

// How the tensor cores take a product: the tile's width, and how many parts K is split into.
struct TcPlan {
    int bn, splits, kb_per_split;
    bool fits;
};

// A model of the time in microseconds: the longest CTA's blocks and tile ends, and with several parts their way
// through memory and another launch. Its constants are from launches of one tile width each (256 against 128 columns):
// 300 x 4096 x 4096 22.5 and 17.1 us, 300 x 1024 x 256 8.3 and 6.5, 2400 x 256 x 1024 5.2 and 5.5, 8192 x 512 x 8192
// 55 and 63; 64 x 4096 x 4096 in 1, 2 and 4 parts of 128 columns 16.0, 13.4 and 10.9; a weight's gradient, 1024 x 256
// over 67200 rows with what it lays out, in 18 parts of 256 columns 98, in 9 of 128 101, in one 475 and 334.
TcPlan plan_tc(int64_t M, int64_t N, int64_t K) {
    const int64_t KB = blocks_of(K);
    TcPlan best = {0, 1, int(KB), false};
    double least = 0;
    for (const int bn : {256, 128}) {
        const int64_t tiles = (M + kTc8Rows - 1) / kTc8Rows * ((N + bn - 1) / bn);
        if (tiles > INT32_MAX / 2) continue;
        const int64_t most = std::max<int64_t>(1, std::min<int64_t>(KB, kSms / tiles));
        for (int64_t s = 1; s <= most; ++s) {
            const int64_t per = (KB + s - 1) / s;
            if (s > 1 && (KB + per - 1) / per != s) continue;  // the last part would be empty
            const double rounds = double((tiles * s + kSms - 1) / kSms);
            double t = rounds * (double(per) * (bn == 256 ? 0.57 : 0.44) + (bn == 256 ? 1.6 : 1.0));
            if (s > 1) t += 2.5 + double(s) * double(M) * double(N) * 8e-6 / 4.0;
            if (best.bn == 0 || t < least) {
                least = t;
                best = {bn, int(s), int(per), true};
            }
        }
    }
    return best;
}

size_t partial_floats(int64_t M, int64_t N, int64_t K) {
    const TcPlan p = plan_tc(M, N, K);
    return p.splits > 1 ? size_t(p.splits) * size_t(M) * size_t(N) : 0;
}

int make_map8(CUtensorMap* map, const Operand8& o, int64_t rows, int64_t K, int box_rows, char* err, size_t err_len) {
    const CUresult r =
        !o.blocks
            ? host::encode_tiled_u8(map, o.q, uint64_t(K), uint64_t(rows), uint64_t(o.pitch), kBlock8,
                                    uint32_t(box_rows), CU_TENSOR_MAP_SWIZZLE_128B)
            : host::encode_tiled_rows(map, 1, o.q, kBlock8, uint64_t(rows), uint64_t(blocks_of(K)), kBlock8,
                                      uint32_t(box_rows), CU_TENSOR_MAP_SWIZZLE_128B);
    if (r == CUDA_SUCCESS) return TD_OK;
    return fail(err, err_len, TD_ERR_CUDA, "cuTensorMapEncodeTiled (8-bit product) failed (%d)", int(r));
}

template <int BN, typename T, bool COLS>
int launch_tc_of(const CUtensorMap& ma, const CUtensorMap& mb, const CUtensorMap& mo, const Tc8Args& t,
                 cudaStream_t stream, char* err, size_t err_len) {
    constexpr auto kernel = fp8_product_tc_kernel<BN, T, COLS>;
    constexpr size_t smem = Tc8Layout<BN, COLS>::kBytes;
    static_assert(smem <= 227 * 1024, "shared memory of a CTA");
    if (int rc = host::allow_smem<kernel>(smem, err, err_len)) return rc;
    const int grid = std::min(t.tiles * t.splits, kSms);
    return host::launch(err, err_len, "fp8_product_tc_kernel", kernel, dim3(unsigned(grid)), dim3(kTc8Threads), smem,
                        stream, true, ma, mb, mo, t);
}

int launch_tc(const TcPlan& p, const Operand8& a, const Operand8& b, const End8& end, int out_dtype, int64_t M,
              int64_t N, int64_t K, float* partial, cudaStream_t stream, char* err, size_t err_len) {
    CUtensorMap ma, mb;
    if (int rc = make_map8(&ma, a, M, K, kTc8Rows, err, err_len)) return rc;
    if (int rc = make_map8(&mb, b, N, K, p.bn, err, err_len)) return rc;
    Tc8Args t = {};
    t.sa = a.scale;
    t.sb = b.scale;
    t.sa_row = a.scale_row;
    t.sa_k = a.scale_k;
    t.sb_row = b.scale_row;
    t.sb_k = b.scale_k;
    t.end = end;
    t.partial = partial;
    t.M = int(M);
    t.N = int(N);
    t.k_blocks = int(blocks_of(K));
    t.n_tiles = int((N + p.bn - 1) / p.bn);
    t.tiles = int((M + kTc8Rows - 1) / kTc8Rows * t.n_tiles);
    t.splits = p.splits;
    t.kb_per_split = p.kb_per_split;
    if (p.splits > 1) {
        t.end.bias = nullptr;
        t.end.act = kActNone;
    }
    // results whose rows start on 16-byte boundaries leave in boxes of 32 rows x 128 bytes
    const int written = p.splits > 1 ? int(TD_F32) : out_dtype;
    const void* out = p.splits > 1 ? partial : end.out;
    const int64_t width = written == TD_E4M3 ? end.pitch : N, e = int64_t(type_bytes(written));
    CUtensorMap mo = mb;  // (any map, where it is not used)
    t.boxes = aligned(out, 16) && width * e % 16 == 0;
    if (t.boxes) {
        const CUresult r = host::encode_tiled_rows(&mo, int(e), out, uint64_t(width), uint64_t(M), uint64_t(p.splits),
                                                   uint32_t(128 / e), 32, CU_TENSOR_MAP_SWIZZLE_128B);
        if (r != CUDA_SUCCESS)
            return fail(err, err_len, TD_ERR_CUDA, "cuTensorMapEncodeTiled (8-bit product) failed (%d)", int(r));
    }
    auto go = [&](auto zero) {
        using T = decltype(zero);
        if constexpr (sizeof(T) == 1)
            return p.bn == 256 ? launch_tc_of<256, T, false>(ma, mb, mo, t, stream, err, err_len)
                               : launch_tc_of<128, T, false>(ma, mb, mo, t, stream, err, err_len);
        else if (b.blocks)  // (as a is, and with a scale for each row)
            return p.bn == 256 ? launch_tc_of<256, T, true>(ma, mb, mo, t, stream, err, err_len)
                               : launch_tc_of<128, T, true>(ma, mb, mo, t, stream, err, err_len);
        else
            return p.bn == 256 ? launch_tc_of<256, T, false>(ma, mb, mo, t, stream, err, err_len)
                               : launch_tc_of<128, T, false>(ma, mb, mo, t, stream, err, err_len);
    };
    if (p.splits == 1) return out_dtype == TD_E4M3 ? go(E4m3()) : by_type(out_dtype, go);
    if (int rc = go(float())) return rc;
    const dim3 grid(unsigned(std::min<int64_t>((M * blocks_of(N) + 7) / 8, int64_t(kSms) * 8)));
    auto finish = [&](auto zero) {
        return host::launch(err, err_len, "fp8_finish_kernel", fp8_finish_kernel<decltype(zero)>, grid, dim3(256), 0,
                            stream, true, static_cast<const float*>(partial), p.splits, end,
                            static_cast<long long>(M), int(N));
    };
    return out_dtype == TD_E4M3 ? finish(E4m3()) : by_type(out_dtype, finish);
}

// partial: partial_floats(M, N, K) of them. Operands start on 16-byte boundaries, as do their rows. (Products with a
// scale for each row of both operands, whose b.scale_row is 1, have a result in a floating type, and scales a tile's
// width beyond N.)
int launch_product(const Operand8& a, const Operand8& b, const End8& end, int out_dtype, int64_t M, int64_t N,
                   int64_t K, float* partial, cudaStream_t stream, char* err, size_t err_len) {
    const TcPlan p = plan_tc(M, N, K);
    if (host::best_policy() && p.fits)
        return launch_tc(p, a, b, end, out_dtype, M, N, K, partial, stream, err, err_len);
    return launch_simt(a, b, end, out_dtype, M, N, K, stream, err, err_len);
}

// Whether a product of M rows that come in x_dtype is one of few (td_fp8_few.cuh). Rows wider than 8 bits are rounded
// there as long as they are short: every CTA does that again, at 0.5 us a row and 1024 of K, where a launch of its own
// is 1.2 us on the GPU and 2.5 us of the host's time (1 x 1024 x 256: 1.75 us against 3.0; 1 x 4096 x 4096: 7.7 against
// 6.9, 18 against 20 with the host; 4 x 4096 x 1024: 7.1 against 4.9). By these costs the GPU alone would change over
// at about 2500 values and the whole call at about 7600; the limit lies between, so a captured graph pays up to 0.8 us
// for what a call gains.
bool few_takes(int x_dtype, int64_t M, int64_t K) {
    if (!host::best_policy()) return false;
    return x_dtype == TD_E4M3 ? M <= kFewMost : M <= kFewWide && M * K <= 4096;
}

template <typename X, typename T, int TILES>
int launch_few_of(const FewArgs& a, cudaStream_t stream, char* err, size_t err_len) {
    const unsigned ctas = unsigned((a.N + kFewRows - 1) / kFewRows);
    constexpr size_t smem = few_smem<X, TILES>();
    if constexpr (sizeof(T) == 1) {
        constexpr auto kernel = fp8_few_to8_kernel<X, TILES>;
        if (int rc = host::allow_smem<kernel>(smem + 16384, err, err_len)) return rc;
        return host::launch(err, err_len, "fp8_few_to8_kernel", kernel, dim3((ctas + 7) / 8 * 8), dim3(kFewThreads),
                            smem, stream, true, a);
    } else {
        constexpr auto kernel = fp8_few_kernel<X, T, TILES>;
        if (int rc = host::allow_smem<kernel>(smem + 16384, err, err_len)) return rc;
        return host::launch(err, err_len, "fp8_few_kernel", kernel, dim3(ctas), dim3(kFewThreads), smem, stream, true,
                            a);
    }
}

int launch_few(int x_dtype, FewArgs a, int out_dtype, cudaStream_t stream, char* err, size_t err_len) {
    auto from = [&](auto x) {
        using X = decltype(x);
        a.x_wide = a.K % 4 == 0 && aligned(a.x, 4 * sizeof(X));
        auto to = [&](auto zero) {
            using T = decltype(zero);
            if constexpr (sizeof(X) == 1) {
                if (a.M > 8) return launch_few_of<X, T, 2>(a, stream, err, err_len);
            }
            return launch_few_of<X, T, 1>(a, stream, err, err_len);
        };
        return out_dtype == TD_E4M3 ? to(E4m3()) : by_type(out_dtype, to);
    };
    return x_dtype == TD_E4M3 ? from(E4m3()) : by_type(x_dtype, from);
}

// What a forward call keeps in its workspace: the input in 8 bits, where it comes wider, 8-bit operands whose rows do
// not start on 16-byte boundaries on such, and a split product's parts.
struct LinearPlan {
    uint8_t *q, *w;
    float *scale, *partial;
    size_t bytes;
};

LinearPlan plan_linear(int x_dtype, int64_t M, int64_t K, int64_t N, bool copy_x, bool copy_w, void* workspace) {
    LinearPlan p = {};
    Cut cut(workspace);
    if (x_dtype != TD_E4M3 || copy_x) p.q = cut.take<uint8_t>(M * up(K, 16));
    if (x_dtype != TD_E4M3) p.scale = cut.take<float>(M * blocks_of(K));
    if (copy_w) p.w = cut.take<uint8_t>(N * up(K, 16));
    p.partial = cut.take<float>(int64_t(partial_floats(M, N, K)));
    p.bytes = cut.used == 0 ? 0 : cut.bytes();
    return p;
}

// A training forward's workspace: the weight in 8 bits, and a split product's parts.
struct TrainPlan {
    uint8_t* w;
    float *w_scale, *partial;
    size_t bytes;
};

TrainPlan plan_train(int64_t M, int64_t K, int64_t N, void* workspace) {
    TrainPlan p = {};
    Cut cut(workspace);
    p.w = cut.take<uint8_t>(N * up(K, 16));
    p.w_scale = cut.take<float>(blocks_of(N) * blocks_of(K));
    p.partial = cut.take<float>(int64_t(partial_floats(M, N, K)));
    p.bytes = cut.bytes();
    return p;
}

// A backward call's workspace: the gradient in 1 x 128 blocks, and, transposed, in blocks of 128 rows ([MB, N, 128]),
// as is the input ([MB, K, 128]); the transposed weight; the parts of the bias's column sums, and of split products,
// one after the other.
struct BackwardPlan {
    uint8_t *dy, *dyt, *xt, *wt;
    float *dy_scale, *dyt_scale, *xt_scale, *wt_scale, *sums, *partial;
    int64_t n_pad, k_pad;  // columns of the scales [MB, ..] of the transposed operands
    size_t bytes;
};

BackwardPlan plan_backward(int64_t M, int64_t K, int64_t N, bool want_x, bool want_w, bool want_b, void* workspace) {
    BackwardPlan p = {};
    Cut cut(workspace);
    const int64_t MB = blocks_of(M);
    p.n_pad = up(N, 256);
    p.k_pad = up(K, 256);
    if (want_x) {
        p.dy = cut.take<uint8_t>(M * up(N, 16));
        p.dy_scale = cut.take<float>(M * blocks_of(N));
        p.wt = cut.take<uint8_t>(K * up(N, 16));
        p.wt_scale = cut.take<float>(blocks_of(K) * blocks_of(N));
    }
    if (want_w) {
        p.dyt = cut.take<uint8_t>(N * MB * kBlock8);
        p.dyt_scale = cut.take<float>(MB * p.n_pad);
        p.xt = cut.take<uint8_t>(K * MB * kBlock8);
        p.xt_scale = cut.take<float>(MB * p.k_pad);
    }
    if (want_b) p.sums = cut.take<float>(MB * N);
    p.partial = cut.take<float>(int64_t(std::max(want_x ? partial_floats(M, K, N) : 0,
                                                 want_w ? partial_floats(N, K, M) : 0)));
    p.bytes = cut.bytes();
    return p;
}

int check_workspace(const void* workspace, size_t have, size_t need, char* err, size_t err_len) {
    if (need > 0 && (workspace == nullptr || have < need))
        return fail(err, err_len, TD_ERR_WORKSPACE, "workspace must be of %zu bytes (got %zu)", need, have);
    return TD_OK;
}

}  // namespace
}  // namespace td

extern "C" {

int td_fp8_quantize(int dtype, const void* x, void* q, int64_t q_pitch, float* scale, int64_t M, int64_t K, int tiles,
                    void* stream, char* err, size_t err_len) {
    using namespace td;
    if (!wide_type(dtype)) return fail(err, err_len, TD_ERR_ARG, "unsupported dtype %d", dtype);
    if (int rc = check_sizes(M, K, 1, err, err_len)) return rc;
    if (M == 0) return TD_OK;
    if (x == nullptr) return fail(err, err_len, TD_ERR_ARG, "null tensor pointer");
    if (int rc = check_written(q, q_pitch, K, scale, err, err_len)) return rc;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (!tiles) return launch_rows(dtype, x, static_cast<uint8_t*>(q), q_pitch, scale, M, K, s, err, err_len);
    TileJobs jobs = {};
    TileArgs& a = jobs.job[kTileWhole];
    a.x = x;
    a.ld = K;
    a.q = static_cast<uint8_t*>(q);
    a.scale = scale;
    a.M = M;
    a.q_pitch = q_pitch;
    a.C = int(K);
    return launch_tiles(dtype, jobs, s, err, err_len);
}

int td_fp8_dequantize(int dtype, const void* q, int64_t q_pitch, const float* scale, void* out, int64_t M, int64_t K,
                      int tiles, void* stream, char* err, size_t err_len) {
    using namespace td;
    if (!wide_type(dtype)) return fail(err, err_len, TD_ERR_ARG, "unsupported dtype %d", dtype);
    if (int rc = check_sizes(M, K, 1, err, err_len)) return rc;
    if (M == 0) return TD_OK;
    if (q == nullptr || scale == nullptr || out == nullptr)
        return fail(err, err_len, TD_ERR_ARG, "null tensor pointer");
    if (q_pitch < K) return fail(err, err_len, TD_ERR_ARG, "8-bit rows must not overlap");
    const BackArgs a = {static_cast<const uint8_t*>(q), scale, out, M, q_pitch, int(K), int(blocks_of(K)), tiles};
    const bool wide = K % 8 == 0 && q_pitch % 8 == 0 && aligned(q, 8) && aligned(out, 16);
    const dim3 grid(unsigned(std::min<int64_t>((M * ((K + 7) / 8) + 255) / 256, int64_t(kSms) * 8)));
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool flat = !tiles && K % kBlock8 == 0 && q_pitch == K && aligned(q, 16) && aligned(out, 32);
    return by_type(dtype, [&](auto zero) {
        using T = decltype(zero);
        if (flat)
            return host::launch(err, err_len, "fp8_flat_back_kernel", fp8_flat_back_kernel<T>, grid, dim3(256), 0, s,
                                true, a);
        return wide ? host::launch(err, err_len, "fp8_back_kernel", fp8_back_kernel<T, true>, grid, dim3(256), 0, s,
                                   true, a)
                    : host::launch(err, err_len, "fp8_back_kernel", fp8_back_kernel<T, false>, grid, dim3(256), 0, s,
                                   true, a);
    });
}

size_t td_fp8_linear_workspace_bytes(int x_dtype, int64_t M, int64_t K, int64_t N, int copy_x, int copy_weight) {
    using namespace td;
    if ((!wide_type(x_dtype) && x_dtype != TD_E4M3) || M <= 0 || check_sizes(M, K, N, nullptr, 0) != TD_OK) return 0;
    return plan_linear(x_dtype, M, K, N, copy_x != 0, copy_weight != 0, nullptr).bytes;
}

int td_fp8_linear(int x_dtype, const void* x, int64_t x_pitch, const float* x_scale, const void* weight,
                  int64_t w_pitch, const float* w_scale, int bias_dtype, const void* bias, int activation,
                  int out_dtype, void* out, int64_t out_pitch, float* out_scale, int64_t M, int64_t K, int64_t N,
                  void* workspace, size_t workspace_bytes, void* stream, char* err, size_t err_len) {
    using namespace td;
    if ((!wide_type(x_dtype) && x_dtype != TD_E4M3) || (!wide_type(out_dtype) && out_dtype != TD_E4M3))
        return fail(err, err_len, TD_ERR_ARG, "unsupported dtype");
    if (bias != nullptr && !wide_type(bias_dtype)) return fail(err, err_len, TD_ERR_ARG, "unsupported dtype of bias");
    if (activation < kActNone || activation > kActSilu)
        return fail(err, err_len, TD_ERR_ARG, "unknown activation %d", activation);
    if (int rc = check_sizes(M, K, N, err, err_len)) return rc;
    if (M == 0) return TD_OK;
    if (x == nullptr || weight == nullptr || w_scale == nullptr || out == nullptr)
        return fail(err, err_len, TD_ERR_ARG, "null tensor pointer");
    if (out_dtype == TD_E4M3) {
        if (int rc = check_written(out, out_pitch, N, out_scale, err, err_len)) return rc;
    }
    if (x_dtype == TD_E4M3 && (x_scale == nullptr || x_pitch < K))
        return fail(err, err_len, TD_ERR_ARG, "an 8-bit input has scales, and rows that do not overlap");
    if (w_pitch < K) return fail(err, err_len, TD_ERR_ARG, "the weight's rows must not overlap");
    if (std::max(w_pitch, x_dtype == TD_E4M3 ? x_pitch : 0) >= int64_t(1) << 39)
        return fail(err, err_len, TD_ERR_ARG, "rows are too far apart");
    const bool copy_x = x_dtype == TD_E4M3 && (!aligned(x, 16) || x_pitch % 16 != 0);
    const bool copy_w = !aligned(weight, 16) || w_pitch % 16 != 0;
    const LinearPlan p = plan_linear(x_dtype, M, K, N, copy_x, copy_w, workspace);
    if (int rc = check_workspace(workspace, workspace_bytes, p.bytes, err, err_len)) return rc;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int64_t KB = blocks_of(K);
    const End8 end = {bias, out, out_scale, bias_dtype, activation, int(out_pitch)};
    Operand8 a = {static_cast<const uint8_t*>(x), x_scale, x_pitch, KB, 1, 1, false, kBlock8};
    if (copy_x) {
        if (int rc = launch_pitch(&a.q, &a.pitch, p.q, M, K, s, err, err_len)) return rc;
    }
    const uint8_t* w8 = static_cast<const uint8_t*>(weight);
    if (copy_w) {
        long long pitch = w_pitch;
        if (int rc = launch_pitch(&w8, &pitch, p.w, N, K, s, err, err_len)) return rc;
        w_pitch = pitch;
    }
    auto few = [&](int dtype) {
        const FewArgs f = {dtype == TD_E4M3 ? a.q : x, a.scale, w8, w_scale, end,
                           a.pitch, w_pitch, int(M), int(N), int(K), int(KB), 0};
        return launch_few(dtype, f, out_dtype, s, err, err_len);
    };
    if (few_takes(x_dtype, M, K)) return few(x_dtype);
    if (x_dtype != TD_E4M3) {
        a.q = p.q;
        a.scale = p.scale;
        a.pitch = up(K, 16);
        if (int rc = launch_rows(x_dtype, x, p.q, a.pitch, p.scale, M, K, s, err, err_len)) return rc;
    }
    if (few_takes(TD_E4M3, M, K)) return few(TD_E4M3);
    const Operand8 b = {w8, w_scale, w_pitch, KB, 1, kBlock8, false, kBlock8};
    return launch_product(a, b, end, out_dtype, M, N, K, p.partial, s, err, err_len);
}

size_t td_fp8_linear_train_workspace_bytes(int64_t M, int64_t K, int64_t N) {
    using namespace td;
    if (M <= 0 || check_sizes(M, K, N, nullptr, 0) != TD_OK) return 0;
    return plan_train(M, K, N, nullptr).bytes;
}

int td_fp8_linear_train(int dtype, const void* x, const void* weight, const void* bias, void* q, int64_t q_pitch,
                        float* scale, void* out, int64_t M, int64_t K, int64_t N, void* workspace,
                        size_t workspace_bytes, void* stream, char* err, size_t err_len) {
    using namespace td;
    if (!wide_type(dtype)) return fail(err, err_len, TD_ERR_ARG, "unsupported dtype %d", dtype);
    if (int rc = check_sizes(M, K, N, err, err_len)) return rc;
    if (M == 0) return TD_OK;
    if (x == nullptr || weight == nullptr || out == nullptr)
        return fail(err, err_len, TD_ERR_ARG, "null tensor pointer");
    if (int rc = check_written(q, q_pitch, K, scale, err, err_len)) return rc;
    const TrainPlan p = plan_train(M, K, N, workspace);
    if (int rc = check_workspace(workspace, workspace_bytes, p.bytes, err, err_len)) return rc;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    TileJobs jobs = {};
    TileArgs& w = jobs.job[kTileWhole];
    w.x = weight;
    w.ld = K;
    w.q = p.w;
    w.scale = p.w_scale;
    w.M = N;
    w.q_pitch = up(K, 16);
    w.C = int(K);
    // Many rows by the kernel for rows (67200 x 256: 5.6 us for this one's 15), few with the weight in one launch.
    if (M * K >= int64_t(4) << 20) {
        if (int rc = launch_rows(dtype, x, static_cast<uint8_t*>(q), q_pitch, scale, M, K, s, err, err_len)) return rc;
    } else {
        TileArgs& xs = jobs.job[kTileBlocks];
        xs.x = x;
        xs.ld = K;
        xs.q = static_cast<uint8_t*>(q);
        xs.scale = scale;
        xs.M = M;
        xs.q_pitch = q_pitch;
        xs.C = int(K);
    }
    if (int rc = launch_tiles(dtype, jobs, s, err, err_len)) return rc;
    const int64_t KB = blocks_of(K);
    const Operand8 a = {static_cast<const uint8_t*>(q), scale, q_pitch, KB, 1, 1, false, kBlock8};
    const Operand8 b = {p.w, p.w_scale, up(K, 16), KB, 1, kBlock8, false, kBlock8};
    const End8 end = {bias, out, nullptr, dtype, kActNone, 0};
    return launch_product(a, b, end, dtype, M, N, K, p.partial, s, err, err_len);
}

size_t td_fp8_linear_backward_workspace_bytes(int64_t M, int64_t K, int64_t N, int want_input, int want_weight,
                                              int want_bias) {
    using namespace td;
    if (M <= 0 || check_sizes(M, K, N, nullptr, 0) != TD_OK) return 0;
    return plan_backward(M, K, N, want_input != 0, want_weight != 0, want_bias != 0, nullptr).bytes;
}

int td_fp8_linear_backward(int dtype, const void* grad_out, const void* x, int64_t x_pitch, const float* x_scale,
                           const void* weight, void* grad_x, void* grad_weight, void* grad_bias, int64_t M, int64_t K,
                           int64_t N, void* workspace, size_t workspace_bytes, void* stream, char* err,
                           size_t err_len) {
    using namespace td;
    if (!wide_type(dtype)) return fail(err, err_len, TD_ERR_ARG, "unsupported dtype %d", dtype);
    if (int rc = check_sizes(M, K, N, err, err_len)) return rc;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (M == 0) {
        const size_t e = type_bytes(dtype);
        if ((grad_weight != nullptr && cudaMemsetAsync(grad_weight, 0, e * size_t(N) * size_t(K), s) != cudaSuccess) ||
            (grad_bias != nullptr && cudaMemsetAsync(grad_bias, 0, e * size_t(N), s) != cudaSuccess))
            return fail(err, err_len, TD_ERR_CUDA, "memset: %s", cudaGetErrorString(cudaGetLastError()));
        return TD_OK;
    }
    if (grad_out == nullptr || (grad_x != nullptr && weight == nullptr) ||
        (grad_weight != nullptr && (x == nullptr || x_scale == nullptr)))
        return fail(err, err_len, TD_ERR_ARG, "null tensor pointer");
    if (grad_weight != nullptr && x_pitch < K) return fail(err, err_len, TD_ERR_ARG, "8-bit rows must not overlap");
    const BackwardPlan p = plan_backward(M, K, N, grad_x != nullptr, grad_weight != nullptr, grad_bias != nullptr,
                                         workspace);
    if (int rc = check_workspace(workspace, workspace_bytes, p.bytes, err, err_len)) return rc;
    const int64_t NB = blocks_of(N), MB = blocks_of(M);
    // all that is laid out, in one launch: the gradient (read once for all that follows) ..
    TileJobs jobs = {};
    TileArgs& g = jobs.job[kTileBlocks];
    g.x = grad_out;
    g.ld = N;
    if (grad_x != nullptr) g.q = p.dy;
    g.scale = p.dy_scale;
    if (grad_weight != nullptr) g.qt = p.dyt;
    g.scale_t = p.dyt_scale;
    if (grad_bias != nullptr) g.sums = p.sums;
    g.M = M;
    g.q_pitch = up(N, 16);
    g.scale_t_pitch = p.n_pad;
    g.C = int(N);
    if (grad_weight != nullptr) {  // .. the kept input, in blocks of rows
        TileArgs& x8 = jobs.job[kTileFrom8];
        x8.x = x;
        x8.x_scale = x_scale;
        x8.ld = x_pitch;
        x8.qt = p.xt;
        x8.scale_t = p.xt_scale;
        x8.M = M;
        x8.scale_t_pitch = p.k_pad;
        x8.C = int(K);
    }
    if (grad_x != nullptr) {  // .. and the weight's blocks, as the forward's, transposed
        TileArgs& w = jobs.job[kTileWhole];
        w.x = weight;
        w.ld = K;
        w.qt = p.wt;
        w.scale_t = p.wt_scale;
        w.M = N;
        w.qt_pitch = up(N, 16);
        w.C = int(K);
    }
    if (int rc = launch_tiles(dtype, jobs, s, err, err_len)) return rc;
    if (grad_bias != nullptr) {
        const int rc = by_type(dtype, [&](auto zero) {
            using T = decltype(zero);
            return host::launch(err, err_len, "column_sum_kernel", column_sum_kernel<T, float>,
                                dim3(unsigned((N + kColumnCols - 1) / kColumnCols)), dim3(kColumnCols * kColumnRows),
                                0, s, true, static_cast<const float*>(p.sums), static_cast<T*>(grad_bias),
                                static_cast<long long>(MB), int(N));
        });
        if (rc) return rc;
    }
    if (grad_x != nullptr) {
        const Operand8 a = {p.dy, p.dy_scale, up(N, 16), NB, 1, 1, false, kBlock8};
        const Operand8 b = {p.wt, p.wt_scale, up(N, 16), NB, 1, kBlock8, false, kBlock8};
        const End8 end = {nullptr, grad_x, nullptr, dtype, kActNone, 0};
        if (int rc = launch_product(a, b, end, dtype, M, K, N, p.partial, s, err, err_len)) return rc;
    }
    if (grad_weight != nullptr) {
        const Operand8 a = {p.dyt, p.dyt_scale, kBlock8, 1, p.n_pad, 1, true, N * kBlock8};
        const Operand8 b = {p.xt, p.xt_scale, kBlock8, 1, p.k_pad, 1, true, K * kBlock8};
        const End8 end = {nullptr, grad_weight, nullptr, dtype, kActNone, 0};
        if (int rc = launch_product(a, b, end, dtype, N, K, M, p.partial, s, err, err_len)) return rc;
    }
    return TD_OK;
}

}  // extern "C"
