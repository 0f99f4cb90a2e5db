// td_attention.cu -- the attention entry points of the C ABI: argument contract, kernel choice and launches.
#include <algorithm>

#include "td_attention_plan.h"
#include "td_attention_tf32.cuh"

namespace td {

namespace {

using host::fail;

int64_t pad_rows(int64_t Q) { return (Q + kAttnRowPad - 1) / kAttnRowPad * kAttnRowPad; }
size_t elem_bytes(int dtype) { return dtype == TD_F64 ? 8 : dtype == TD_F32 ? 4 : 2; }

// How a forward is split over the keys: about `splits` CTAs of split_keys keys each, a multiple of `step`.
void split_plan(int64_t N, int64_t splits, int64_t step, SplitArgs* p) {
    splits = std::max<int64_t>(1, splits);
    const int64_t keys = std::max((N + splits - 1) / splits, int64_t(1));  // one without any key, too
    p->split_keys = int((keys + step - 1) / step * step);
    p->splits = int(std::max<int64_t>(1, (N + p->split_keys - 1) / p->split_keys));
}

// The mma.sync split kernel's plan: the rows of a key head's group in tiles of 16. One wave of long splits where every
// image has all its keys; shorter ones where some have not, so that the CTAs of the full ones do not end last (8 images
// of 22223 keys, the lengths falling to half: 51 us with 2, 44 with 6; without padding: 47 and 45; one image: 13 and
// 17). No split of fewer than 256 keys, two of the kernel's tiles.
SplitArgs mma_split_plan(int64_t B, int64_t Q, int64_t N, int64_t H, int64_t Hk, bool padding) {
    SplitArgs p = {};
    p.row_tiles = int((H / Hk * Q + 15) / 16);
    const int64_t blocks = std::max(B * Hk * p.row_tiles, int64_t(1));
    split_plan(N, std::min(((padding ? 6 : 2) * kSms + blocks - 1) / blocks, N / 256), 128, &p);
    return p;
}

// The CUDA-core forward's register tile: 4 x 4, 2 x 2 for float64 (whose operand tiles take twice the bytes); one row
// a thread for up to 16 queries, where most of a taller tile would be empty.
template <typename T> constexpr int simt_r() { return std::is_same<T, double>::value ? 2 : 4; }

// The CUDA-core and the TF32 forward's plan: down to one tile of 64 keys a CTA, as long as all the CTAs are resident at
// once, three an SM (float32, 8 heads of 32, 2 x 64 queries on 200 keys: 22 us in one split, 12 in four). 16-bit calls
// of the usual widths come here only misaligned or short: they do without partials.
SplitArgs simt_split_plan(int dtype, int64_t B, int64_t Q, int64_t N, int64_t H, int64_t D) {
    SplitArgs p = {};
    const bool whole = (dtype == TD_F16 || dtype == TD_BF16) && D % 8 == 0;
    const int rows = Q <= 16 ? 16 : 16 * (dtype == TD_F64 ? 2 : 4);
    p.row_tiles = int((Q + rows - 1) / rows);
    const int64_t blocks = std::max(B * H * p.row_tiles, int64_t(1));
    split_plan(N, whole ? 1 : std::min(3 * kSms / blocks, (N + 63) / 64), 64, &p);
    return p;
}

// The backward: how many CTAs share the tiles that one tile of keys, or of queries, goes over, so that a few long ones
// do not hold the others up: a key head's block goes over the queries of its whole group, and few queries make few
// blocks. A CTA gets at most about the work of one of three on every SM, or, on tensor cores (one CTA an SM), of two;
// but at least two tiles there, sixteen here, since partial sums and the launch that joins them cost about as much.
// 16-bit causal 2 x 2047 x 8 heads (2 of keys) x 128: 183 us unsplit, 125; 1 query on 8400 keys x 8 heads x 32: 90 us
// and 36, in float32 798 and 80; 2 x 300 queries on 8400 keys in float32: 1044 and 577.
void grad_splits(int dtype, int64_t B, int64_t Q, int64_t N, int64_t H, int64_t Hk, int64_t D, int64_t* k, int64_t* q) {
    const bool tc = (dtype == TD_F16 || dtype == TD_BF16) && D % 8 == 0 && N > 1;  // (unless misaligned)
    const int64_t rows = tc ? 128 : dtype == TD_F64 ? 32 : 64, cols = std::min<int64_t>(rows, 64);
    auto tiles = [](int64_t n, int64_t of) { return (n + of - 1) / of; };
    const int64_t kc = H / Hk * tiles(Q, cols), qc = tiles(N, cols);
    const int64_t work = B * (Hk * tiles(N, rows) * kc + H * tiles(Q, rows) * qc);
    const int64_t chunk = std::max<int64_t>(tc ? 16 : 2, tiles(work, (tc ? 2 : 3) * kSms));
    *k = std::max<int64_t>(1, (kc + chunk / 2) / chunk);
    *q = std::max<int64_t>(1, (qc + chunk / 2) / chunk);
}

// The parts of a call's workspace. The mask's bits and flags are laid out for 16-bit types only (the tensor-core
// kernels read them); a mask shared by images or heads is packed once. The partials of a split forward are sized for
// whichever kernel takes the call.
AttnWorkspace attn_workspace(int dtype, int64_t B, int64_t Q, int64_t N, int64_t H, int64_t Hk, int64_t D, int64_t mb,
                             int64_t mh, bool padding, bool backward) {
    AttnWorkspace w = {};
    auto take = [&](size_t bytes) {
        const size_t at = w.total;
        w.total += (bytes + 255) / 256 * 256;
        return at;
    };
    const size_t acc = dtype == TD_F64 ? 8 : 4;
    const bool half = dtype == TD_F16 || dtype == TD_BF16;
    if (backward) {
        if (dtype == TD_F16) {
            w.amax = take(2 * size_t(B) * Hk * attn_delta_parts(B * Hk) * sizeof(float));
            w.row_g = take(size_t(B) * H * pad_rows(Q) * sizeof(float));
            w.keys_lse = take(size_t(B) * H * pad_rows(Q) * sizeof(float));
        }
        w.delta = take(size_t(B) * H * pad_rows(Q) * acc);
        int64_t k, q;
        grad_splits(dtype, B, Q, N, H, Hk, D, &k, &q);
        if (k > 1) {
            w.part_k = take(size_t(B) * N * Hk * D * k * acc);
            w.part_v = take(size_t(B) * N * Hk * D * k * acc);
        }
        if (q > 1) w.part_q = take(size_t(B) * Q * H * D * q * acc);
    } else {
        int64_t splits = simt_split_plan(dtype, B, Q, N, H, D).splits;
        if (half)
            splits = std::max({splits, int64_t(mma_split_plan(B, Q, N, H, Hk, padding).splits),
                               attn_tc_splits(B, Q, N, H)});
        if (splits > 1) {
            w.part_o = take(size_t(B) * H * Q * splits * D * acc);
            w.part_ml = take(size_t(B) * H * Q * splits * 2 * acc);
        }
    }
    if (half && (mb > 0 || padding)) {
        w.images = padding ? B : mb;
        w.heads = mb > 0 ? mh : 1;
        w.rows = mb > 0 ? Q : 1;
        w.words = 2 * ((N + 63) / 64);
        const int64_t bh = w.images * w.heads, q_tiles = (w.rows + 127) / 128;
        w.row_bits = take(size_t(bh) * w.rows * w.words * 4);
        w.row_flags = take(size_t(bh) * q_tiles * (w.words / 2));
        if (backward && mb > 0) {
            w.col_words = 2 * ((Q + 63) / 64);
            w.col_bits = take(size_t(mb) * mh * N * w.col_words * 4);
            w.col_flags = take(size_t(mb) * mh * ((N + 127) / 128) * (w.col_words / 2));
        }
    }
    return w;
}

int check_workspace(const void* workspace, size_t bytes, size_t need, char* err, size_t err_len) {
    if (need == 0 || (workspace != nullptr && bytes >= need && (reinterpret_cast<uintptr_t>(workspace) & 15u) == 0))
        return TD_OK;
    return fail(err, err_len, TD_ERR_WORKSPACE, "workspace must be 16-byte aligned, of %zu bytes (got %zu)", need,
                bytes);
}

int check_sizes(int dtype, int64_t B, int64_t Q, int64_t N, int64_t H, int64_t Hk, int64_t D, double scale, char* err,
                size_t err_len) {
    if (dtype < TD_F32 || dtype > TD_F64) return fail(err, err_len, TD_ERR_ARG, "unsupported dtype %d", dtype);
    if (B < 0 || Q < 0 || N < 0) return fail(err, err_len, TD_ERR_ARG, "sizes must be non-negative");
    if (H <= 0 || Hk <= 0) return fail(err, err_len, TD_ERR_ARG, "need at least one head");
    if (H % Hk != 0) return fail(err, err_len, TD_ERR_ARG, "query heads must be a multiple of the key heads");
    if (D < 1 || D > TD_MAX_HEAD_DIM)
        return fail(err, err_len, TD_ERR_ARG, "head width must be between 1 and %d", TD_MAX_HEAD_DIM);
    // tiles and rows are counted in 32 bits, with room for a tile behind the last row
    const double most = double(INT32_MAX) - 4096;
    if (double(Q) > most || double(N) > most || double(B) * double(H) * double(pad_rows(Q)) > most ||
        double(B) * double(Hk) * double(pad_rows(N)) > most)
        return fail(err, err_len, TD_ERR_ARG, "too many (batch, token, head) rows");
    if (!(scale >= 1e-30) || !(scale <= 1e30))  // so that the kernels' float32 multiples of it stay in range
        return fail(err, err_len, TD_ERR_ARG, "scale must be between 1e-30 and 1e30");
    return TD_OK;
}

AttnArgs make_args(int dtype, const void* q, const void* k, const void* v_, const int64_t* strides, const uint8_t* mask,
                   const int64_t* mask_strides, const uint8_t* padding, int64_t B, int64_t Q, int64_t N, int64_t H,
                   int64_t Hk, int64_t D, double scale, int causal) {
    AttnArgs a = {};
    a.q = q; a.k = k; a.v = v_;
    a.q_b = strides[0]; a.q_t = strides[1]; a.q_h = strides[2];
    a.k_b = strides[3]; a.k_t = strides[4]; a.k_h = strides[5];
    a.v_b = strides[6]; a.v_t = strides[7]; a.v_h = strides[8];
    a.mask = mask;
    if (mask != nullptr) {
        a.m_b = mask_strides[0]; a.m_h = mask_strides[1]; a.m_q = mask_strides[2];
    }
    a.padding = padding;
    a.B = int(B); a.Q = int(Q); a.N = int(N); a.H = int(H); a.Hk = int(Hk); a.D = int(D);
    a.Qp = int(pad_rows(Q));
    a.causal = causal != 0;
    a.scale = scale;
    const int64_t v = 16 / int64_t(elem_bytes(dtype));
    auto whole = [&](const void* p, long long s_b, long long s_t, long long s_h) {
        return D % v == 0 && s_b % v == 0 && s_t % v == 0 && s_h % v == 0 &&
               (reinterpret_cast<uintptr_t>(p) & 15u) == 0;
    };
    a.vec_q = whole(q, a.q_b, a.q_t, a.q_h);
    a.vec_k = whole(k, a.k_b, a.k_t, a.k_h);
    a.vec_v = whole(v_, a.v_b, a.v_t, a.v_h);
    return a;
}

int zero(void* p, size_t bytes, cudaStream_t stream, char* err, size_t err_len) {
    if (p == nullptr || bytes == 0) return TD_OK;
    const cudaError_t e = cudaMemsetAsync(p, 0, bytes, stream);
    if (e == cudaSuccess) return TD_OK;
    cudaGetLastError();
    return fail(err, err_len, TD_ERR_CUDA, "memset: %s", cudaGetErrorString(e));
}

template <typename T, int DP, int RM>
int simt_forward_tile(const SplitArgs& p, cudaStream_t stream, char* err, size_t err_len) {
    constexpr int RN = simt_r<T>();
    using Tile = SimtTile<typename Elem<T>::acc, DP, RM, RN>;
    constexpr size_t smem = Tile::kRowBytes + 2 * Tile::kColBytes + Tile::kP;
    constexpr auto kernel = attn_simt_forward_kernel<T, DP, RM, RN>;
    if (int rc = host::allow_smem<kernel>(smem, err, err_len)) return rc;
    const long long grid = (long long)p.splits * p.row_tiles * p.a.B * p.a.H;
    if (int rc = host::launch(err, err_len, "attn_simt_forward_kernel", kernel, dim3(unsigned(grid)), dim3(256), smem,
                              stream, true, p))
        return rc;
    return combine<T>(p, stream, err, err_len);
}

template <typename T, int DP>
int simt_forward(const AttnArgs& a, int dtype, const AttnWorkspace& w, unsigned char* workspace, cudaStream_t stream,
                 char* err, size_t err_len) {
    SplitArgs p = simt_split_plan(dtype, a.B, a.Q, a.N, a.H, a.D);
    p.a = a;
    p.part_o = workspace + w.part_o;
    p.part_ml = workspace + w.part_ml;
    return a.Q <= 16 ? simt_forward_tile<T, DP, 1>(p, stream, err, err_len)
                     : simt_forward_tile<T, DP, simt_r<T>()>(p, stream, err, err_len);
}

template <typename T, int DP>
int mma_split(const SplitArgs& p, cudaStream_t stream, char* err, size_t err_len) {
    const long long grid = (long long)p.splits * p.row_tiles * p.a.B * p.a.Hk;
    constexpr auto kernel = attn_split_kernel<T, DP>;
    constexpr size_t smem = SplitLayout<DP>::kSmem;
    if (int rc = host::allow_smem<kernel>(smem, err, err_len)) return rc;
    if (int rc = host::launch(err, err_len, "attn_split_kernel", kernel, dim3(unsigned(grid)),
                              dim3(kSplitWarps * 32), smem, stream, true, p))
        return rc;
    return combine<T>(p, stream, err, err_len);
}

template <typename T>
int mma_split_forward(const AttnArgs& a, const AttnWorkspace& w, unsigned char* workspace, cudaStream_t stream,
                      char* err, size_t err_len) {
    SplitArgs p = mma_split_plan(a.B, a.Q, a.N, a.H, a.Hk, a.padding != nullptr);
    p.a = a;
    p.part_o = workspace + w.part_o;
    p.part_ml = workspace + w.part_ml;
    if (a.D <= 32) return mma_split<T, 32>(p, stream, err, err_len);
    if (a.D <= 64) return mma_split<T, 64>(p, stream, err, err_len);
    return mma_split<T, 128>(p, stream, err, err_len);
}

// Whether the split kernel takes a 16-bit forward that the tensor-core kernel could take as well. A tensor-core CTA's
// time goes with its keys, and a launch that joins splits adds to it; the split kernel's goes with its 16-row tiles
// times keys, behind two launches. The constants stand for both, fitted to the choice rather than the times: of 432
// calls of 1 to 8 images, 8 and 16 heads, D = 32, 64 and 128, 1024 to 22223 keys and 1 to 300 queries on B200, the
// slower kernel is taken by more than 2 % in 24, at worst 1.37 times as slow (64-wide heads, 2 images, one query on
// 22223 keys: 32 us against 24), and all of them together lose 0.7 % to the faster one each time. Below 1024 keys the
// two differ by little (300 keys, one query: 7.8 on tensor cores against 5.4 at D = 32, 9.8 against 9.4 at D = 128).
bool prefer_split(const AttnArgs& a) {
    if (a.N < 1024) return false;
    const double ctas = double((a.Q + 127) / 128) * a.B * a.H;
    const double tiles = double((a.H / a.Hk * (long long)a.Q + 15) / 16) * a.B * a.Hk;
    const double splits = double(attn_tc_splits(a.B, a.Q, a.N, a.H));
    const double walk = (splits > 1 ? 7.0 : 3.3) +
                        0.0103 * a.N / splits * (a.D > 64 ? 1.25 : 1.0) * std::max(1.0, ctas / (2 * kSms));
    const double split = 6.0 + tiles * a.N * (a.D <= 32 ? 3e-5 : a.D <= 64 ? 6e-5 : 1.2e-4);
    return split < walk;
}

// float32 on tensor cores: rows of whole 16-byte vectors and at least 256 keys. Below, where a CTA has a few tiles, its
// four warps' longer chains show (one head, 64 x 64: 12 us at D = 32 and 44 at D = 128 against 9 and 24 on CUDA cores;
// 256 keys: 14 and 30 against 14 and 31; 4 x 1100 x 8 heads x 32: 216 against 234, the backward 527 against 708).
bool tf32_fits(const AttnArgs& a) {
    return host::best_policy() && a.N >= 256 && a.vec_q && a.vec_k && a.vec_v && (a.grad_q == nullptr || a.vec_g) &&
           (reinterpret_cast<uintptr_t>(a.lse) & 15u) == 0;
}

template <int DP, int NT>
int tf32_forward(const AttnArgs& a, const AttnWorkspace& w, unsigned char* workspace, cudaStream_t stream, char* err,
                 size_t err_len) {
    using Lay = Tf32Layout<DP, NT>;
    SplitArgs p = simt_split_plan(TD_F32, a.B, a.Q, a.N, a.H, a.D);
    p.a = a;
    p.part_o = workspace + w.part_o;
    p.part_ml = workspace + w.part_ml;
    constexpr auto kernel = attn_tf32_forward_kernel<DP, NT>;
    constexpr size_t smem = (Lay::kFixed + 4 * Lay::kTile) * sizeof(float);
    if (int rc = host::allow_smem<kernel>(smem, err, err_len)) return rc;
    const long long grid = (long long)p.splits * p.row_tiles * a.B * a.H;
    if (int rc = host::launch(err, err_len, "attn_tf32_forward_kernel", kernel, dim3(unsigned(grid)),
                              dim3(kTf32Threads), smem, stream, true, p))
        return rc;
    return combine<float>(p, stream, err, err_len);
}

template <int DP, int NT>
int tf32_backward(const AttnArgs& a, cudaStream_t stream, char* err, size_t err_len) {
    using Lay = Tf32Layout<DP, NT>;
    constexpr auto kernel = attn_tf32_backward_kernel<DP, NT>;
    constexpr size_t smem = (2 * Lay::kFixed + 4 * Lay::kTile + 4 * NT) * sizeof(float);
    if (int rc = host::allow_smem<kernel>(smem, err, err_len)) return rc;
    const long long rows = (long long)a.B * a.H * a.Qp;
    if (int rc = host::launch(err, err_len, "attn_delta_kernel", attn_delta_kernel<float>,
                              dim3(unsigned((rows + 255) / 256)), dim3(256), 0, stream, true, a))
        return rc;
    const int kv_blocks = (a.N + kTf32Rows - 1) / kTf32Rows * a.B * a.Hk * a.k_splits;
    const int q_blocks = (a.Q + kTf32Rows - 1) / kTf32Rows * a.B * a.H * a.q_splits;
    if (int rc = host::launch(err, err_len, "attn_tf32_backward_kernel", kernel, dim3(unsigned(kv_blocks) + q_blocks),
                              dim3(kTf32Threads), smem, stream, true, a, kv_blocks))
        return rc;
    return join<float>(a, stream, err, err_len);
}

template <typename T, int DP>
int simt_backward(const AttnArgs& a, cudaStream_t stream, char* err, size_t err_len) {
    constexpr int R = simt_r<T>();
    using Tile = SimtTile<typename Elem<T>::acc, DP, R, R>;
    constexpr size_t smem = 4 * Tile::kRowBytes + Tile::kP;
    constexpr auto kernel = attn_simt_backward_kernel<T, DP, R>;
    if (int rc = host::allow_smem<kernel>(smem, err, err_len)) return rc;
    const long long rows = (long long)a.B * a.H * a.Qp;
    if (int rc = host::launch(err, err_len, "attn_delta_kernel", attn_delta_kernel<T>,
                              dim3(unsigned((rows + 255) / 256)), dim3(256), 0, stream, true, a))
        return rc;
    const int kv_blocks = (a.N + Tile::kRows - 1) / Tile::kRows * a.B * a.Hk * a.k_splits;
    const int q_blocks = (a.Q + Tile::kRows - 1) / Tile::kRows * a.B * a.H * a.q_splits;
    if (int rc = host::launch(err, err_len, "attn_simt_backward_kernel", kernel, dim3(unsigned(kv_blocks) + q_blocks),
                              dim3(256), smem, stream, true, a, kv_blocks))
        return rc;
    return join<T>(a, stream, err, err_len);
}

template <typename T>
int forward(const AttnArgs& a, int dtype, const AttnWorkspace& w, unsigned char* workspace, cudaStream_t stream,
            char* err, size_t err_len) {
    if constexpr (std::is_same<T, float>::value) {
        if (a.Q > 16 && tf32_fits(a)) {
            if (a.D <= 32) return tf32_forward<32, 64>(a, w, workspace, stream, err, err_len);
            if (a.D <= 64) return tf32_forward<64, 64>(a, w, workspace, stream, err, err_len);
            return tf32_forward<128, 32>(a, w, workspace, stream, err, err_len);
        }
    }
    if (a.D <= 32) return simt_forward<T, 32>(a, dtype, w, workspace, stream, err, err_len);
    if (a.D <= 64) return simt_forward<T, 64>(a, dtype, w, workspace, stream, err, err_len);
    return simt_forward<T, 128>(a, dtype, w, workspace, stream, err, err_len);
}

template <typename T>
int backward(const AttnArgs& a, cudaStream_t stream, char* err, size_t err_len) {
    if constexpr (std::is_same<T, float>::value) {
        if (tf32_fits(a)) {
            if (a.D <= 32) return tf32_backward<32, 64>(a, stream, err, err_len);
            if (a.D <= 64) return tf32_backward<64, 32>(a, stream, err, err_len);
            return tf32_backward<128, 32>(a, stream, err, err_len);
        }
    }
    if (a.D <= 32) return simt_backward<T, 32>(a, stream, err, err_len);
    if (a.D <= 64) return simt_backward<T, 64>(a, stream, err, err_len);
    return simt_backward<T, 128>(a, stream, err, err_len);
}

}  // namespace
}  // namespace td

extern "C" {

size_t td_attention_workspace_bytes(int dtype, int64_t B, int64_t Q, int64_t N, int64_t H, int64_t Hk, int64_t D,
                                    int64_t mask_b, int64_t mask_h, int has_padding, int backward) {
    using namespace td;
    if (check_sizes(dtype, B, Q, N, H, Hk, D, 1.0, nullptr, 0) != TD_OK || B == 0 || Q == 0 || N == 0) return 0;
    return attn_workspace(dtype, B, Q, N, H, Hk, D, mask_b, mask_h, has_padding != 0, backward != 0).total;
}

int td_attention_forward(int dtype, const void* query, const void* key, const void* value, const int64_t* strides,
                         const uint8_t* attn_mask, const int64_t* mask_strides, const uint8_t* key_padding_mask,
                         void* out, void* rest, void* lse, int64_t B, int64_t Q, int64_t N, int64_t H, int64_t Hk,
                         int64_t D, double scale, int causal, void* workspace, size_t workspace_bytes, void* stream,
                         char* err, size_t err_len) {
    using namespace td;
    if (int rc = check_sizes(dtype, B, Q, N, H, Hk, D, scale, err, err_len)) return rc;
    if (B == 0 || Q == 0) return TD_OK;
    if (query == nullptr || out == nullptr || strides == nullptr || (N > 0 && (key == nullptr || value == nullptr)) ||
        (attn_mask != nullptr && mask_strides == nullptr))
        return fail(err, err_len, TD_ERR_ARG, "null tensor pointer");
    const int64_t mb = attn_mask == nullptr ? 0 : mask_strides[0] != 0 ? B : 1;
    const int64_t mh = attn_mask == nullptr ? 0 : mask_strides[1] != 0 ? H : 1;
    const AttnWorkspace ws = attn_workspace(dtype, B, Q, N, H, Hk, D, mb, mh, key_padding_mask != nullptr, false);
    if (int rc = check_workspace(workspace, workspace_bytes, N > 0 ? ws.total : 0, err, err_len)) return rc;
    AttnArgs a = make_args(dtype, query, key, value, strides, attn_mask, mask_strides, key_padding_mask, B, Q, N, H,
                           Hk, D, scale, causal);
    a.out = out;
    a.rest = dtype == TD_F16 || dtype == TD_BF16 ? rest : nullptr;
    a.lse = lse;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    unsigned char* wp = static_cast<unsigned char*>(workspace);
    if (N > 0 && attn_tc_fits(dtype, a)) {
        if (!prefer_split(a)) return attn_tc_forward(dtype, a, ws, mb, mh, wp, s, err, err_len);
        return dtype == TD_F16 ? mma_split_forward<__half>(a, ws, wp, s, err, err_len)
                               : mma_split_forward<__nv_bfloat16>(a, ws, wp, s, err, err_len);
    }
    switch (dtype) {
        case TD_F32: return forward<float>(a, dtype, ws, wp, s, err, err_len);
        case TD_F16: return forward<__half>(a, dtype, ws, wp, s, err, err_len);
        case TD_BF16: return forward<__nv_bfloat16>(a, dtype, ws, wp, s, err, err_len);
        default: return forward<double>(a, dtype, ws, wp, s, err, err_len);
    }
}

int td_attention_backward(int dtype, const void* query, const void* key, const void* value, const int64_t* strides,
                          const uint8_t* attn_mask, const int64_t* mask_strides, const uint8_t* key_padding_mask,
                          const void* out, const void* rest, const void* lse, const void* grad_out, void* grad_query,
                          void* grad_key, void* grad_value, int64_t B, int64_t Q, int64_t N, int64_t H, int64_t Hk,
                          int64_t D, double scale, int causal, void* workspace, size_t workspace_bytes, void* stream,
                          char* err, size_t err_len) {
    using namespace td;
    if (int rc = check_sizes(dtype, B, Q, N, H, Hk, D, scale, err, err_len)) return rc;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (B == 0) return TD_OK;
    if (Q == 0 || N == 0) {  // no pair: whatever exists has a gradient of zero
        if ((Q > 0 && grad_query == nullptr) || (N > 0 && (grad_key == nullptr || grad_value == nullptr)))
            return fail(err, err_len, TD_ERR_ARG, "null tensor pointer");
        const size_t row = size_t(B) * D * elem_bytes(dtype);
        if (int rc = zero(grad_query, row * Q * H, s, err, err_len)) return rc;
        if (int rc = zero(grad_key, row * N * Hk, s, err, err_len)) return rc;
        return zero(grad_value, row * N * Hk, s, err, err_len);
    }
    if (query == nullptr || key == nullptr || value == nullptr || strides == nullptr || out == nullptr ||
        lse == nullptr || grad_out == nullptr || grad_query == nullptr || grad_key == nullptr ||
        grad_value == nullptr || (attn_mask != nullptr && mask_strides == nullptr))
        return fail(err, err_len, TD_ERR_ARG, "null tensor pointer");
    const int64_t mb = attn_mask == nullptr ? 0 : mask_strides[0] != 0 ? B : 1;
    const int64_t mh = attn_mask == nullptr ? 0 : mask_strides[1] != 0 ? H : 1;
    const AttnWorkspace ws = attn_workspace(dtype, B, Q, N, H, Hk, D, mb, mh, key_padding_mask != nullptr, true);
    if (int rc = check_workspace(workspace, workspace_bytes, ws.total, err, err_len)) return rc;
    AttnArgs a = make_args(dtype, query, key, value, strides, attn_mask, mask_strides, key_padding_mask, B, Q, N, H,
                           Hk, D, scale, causal);
    a.out_in = out;
    a.rest_in = dtype == TD_F16 || dtype == TD_BF16 ? rest : nullptr;
    a.lse = const_cast<void*>(lse);
    a.grad_out = grad_out;
    a.vec_g = D % (16 / int64_t(elem_bytes(dtype))) == 0 && (reinterpret_cast<uintptr_t>(grad_out) & 15u) == 0;
    a.grad_q = grad_query;
    a.grad_k = grad_key;
    a.grad_v = grad_value;
    a.delta = static_cast<unsigned char*>(workspace) + ws.delta;
    int64_t k_splits, q_splits;
    grad_splits(dtype, B, Q, N, H, Hk, D, &k_splits, &q_splits);
    a.k_splits = int(k_splits);
    a.q_splits = int(q_splits);
    a.part_k = static_cast<unsigned char*>(workspace) + ws.part_k;
    a.part_v = static_cast<unsigned char*>(workspace) + ws.part_v;
    a.part_q = static_cast<unsigned char*>(workspace) + ws.part_q;
    if (attn_tc_fits(dtype, a))
        return attn_tc_backward(dtype, a, ws, mb, mh, static_cast<unsigned char*>(workspace), s, err, err_len);
    switch (dtype) {
        case TD_F32: return backward<float>(a, s, err, err_len);
        case TD_F16: return backward<__half>(a, s, err, err_len);
        case TD_BF16: return backward<__nv_bfloat16>(a, s, err, err_len);
        default: return backward<double>(a, s, err, err_len);
    }
}

}  // extern "C"
