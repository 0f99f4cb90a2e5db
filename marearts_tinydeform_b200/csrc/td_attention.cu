// td_attention.cu -- the attention entry points of the C ABI: argument contract, kernel choice and launches.
#include "td_attention_plan.h"

namespace td {

namespace {

using host::fail;

int64_t pad_rows(int64_t Q) { return (Q + kAttnRowPad - 1) / kAttnRowPad * kAttnRowPad; }
size_t elem_bytes(int dtype) { return dtype == TD_F64 ? 8 : dtype == TD_F32 ? 4 : 2; }

// The parts of a call's workspace. The mask's bits and flags are laid out for 16-bit types only (the tensor-core
// kernels read them); a mask shared by images or heads is packed once.
AttnWorkspace attn_workspace(int dtype, int64_t B, int64_t Q, int64_t N, int64_t H, int64_t mb, int64_t mh,
                             bool padding, bool backward) {
    AttnWorkspace w = {};
    auto take = [&](size_t bytes) {
        const size_t at = w.total;
        w.total += (bytes + 255) / 256 * 256;
        return at;
    };
    if (backward) {
        w.amax = take(2 * sizeof(unsigned int));
        w.delta = take(size_t(B) * H * pad_rows(Q) * (dtype == TD_F64 ? 8 : 4));
    }
    if ((dtype == TD_F16 || dtype == TD_BF16) && (mb > 0 || padding)) {
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

AttnArgs make_args(const void* q, const void* k, const void* v, const int64_t* strides, const uint8_t* mask,
                   const int64_t* mask_strides, const uint8_t* padding, int64_t B, int64_t Q, int64_t N, int64_t H,
                   int64_t Hk, int64_t D, double scale, int causal) {
    AttnArgs a = {};
    a.q = q; a.k = k; a.v = v;
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
    return a;
}

int zero(void* p, size_t bytes, cudaStream_t stream, char* err, size_t err_len) {
    if (p == nullptr || bytes == 0) return TD_OK;
    const cudaError_t e = cudaMemsetAsync(p, 0, bytes, stream);
    if (e == cudaSuccess) return TD_OK;
    cudaGetLastError();
    return fail(err, err_len, TD_ERR_CUDA, "memset: %s", cudaGetErrorString(e));
}

// Register tile of the CUDA-core kernels: 4 x 4, 2 x 2 for float64 (whose operand tiles take twice the bytes).
template <typename T> constexpr int simt_r() { return std::is_same<T, double>::value ? 2 : 4; }

template <typename T, int DP>
int simt_forward(const AttnArgs& a, cudaStream_t stream, char* err, size_t err_len) {
    constexpr int R = simt_r<T>();
    using Tile = SimtTile<typename Elem<T>::acc, DP, R>;
    constexpr size_t smem = 3 * Tile::kOperand + Tile::kP;
    auto kernel = attn_simt_forward_kernel<T, DP, R>;
    if (int rc = host::allow_smem(kernel, smem, err, err_len)) return rc;
    const unsigned grid = unsigned((a.Q + Tile::kRows - 1) / Tile::kRows * a.B * a.H);
    return host::launch(err, err_len, "attn_simt_forward_kernel", kernel, dim3(grid), dim3(256), smem, stream, true,
                        a);
}

template <typename T, int DP>
int simt_backward(const AttnArgs& a, cudaStream_t stream, char* err, size_t err_len) {
    constexpr int R = simt_r<T>();
    using Tile = SimtTile<typename Elem<T>::acc, DP, R>;
    constexpr size_t smem = 4 * Tile::kOperand + Tile::kP;
    auto kernel = attn_simt_backward_kernel<T, DP, R>;
    if (int rc = host::allow_smem(kernel, smem, err, err_len)) return rc;
    const long long rows = (long long)a.B * a.H * a.Qp;
    if (int rc = host::launch(err, err_len, "attn_delta_kernel", attn_delta_kernel<T>,
                              dim3(unsigned((rows + 255) / 256)), dim3(256), 0, stream, true, a))
        return rc;
    const int kv_blocks = (a.N + Tile::kRows - 1) / Tile::kRows * a.B * a.Hk;
    const int q_blocks = (a.Q + Tile::kRows - 1) / Tile::kRows * a.B * a.H;
    return host::launch(err, err_len, "attn_simt_backward_kernel", kernel, dim3(unsigned(kv_blocks) + q_blocks),
                        dim3(256), smem, stream, true, a, kv_blocks);
}

template <typename T>
int forward(const AttnArgs& a, cudaStream_t stream, char* err, size_t err_len) {
    if (a.D <= 32) return simt_forward<T, 32>(a, stream, err, err_len);
    if (a.D <= 64) return simt_forward<T, 64>(a, stream, err, err_len);
    return simt_forward<T, 128>(a, stream, err, err_len);
}

template <typename T>
int backward(const AttnArgs& a, cudaStream_t stream, char* err, size_t err_len) {
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
    return attn_workspace(dtype, B, Q, N, H, mask_b, mask_h, has_padding != 0, backward != 0).total;
}

int td_attention_forward(int dtype, const void* query, const void* key, const void* value, const int64_t* strides,
                         const uint8_t* attn_mask, const int64_t* mask_strides, const uint8_t* key_padding_mask,
                         void* out, void* rest, void* lse, int64_t B, int64_t Q, int64_t N, int64_t H, int64_t Hk, int64_t D,
                         double scale, int causal, void* workspace, size_t workspace_bytes, void* stream, char* err,
                         size_t err_len) {
    using namespace td;
    if (int rc = check_sizes(dtype, B, Q, N, H, Hk, D, scale, err, err_len)) return rc;
    if (B == 0 || Q == 0) return TD_OK;
    if (query == nullptr || out == nullptr || strides == nullptr || (N > 0 && (key == nullptr || value == nullptr)) ||
        (attn_mask != nullptr && mask_strides == nullptr))
        return fail(err, err_len, TD_ERR_ARG, "null tensor pointer");
    const int64_t mb = attn_mask == nullptr ? 0 : mask_strides[0] != 0 ? B : 1;
    const int64_t mh = attn_mask == nullptr ? 0 : mask_strides[1] != 0 ? H : 1;
    const AttnWorkspace ws = attn_workspace(dtype, B, Q, N, H, mb, mh, key_padding_mask != nullptr, false);
    if (int rc = check_workspace(workspace, workspace_bytes, N > 0 ? ws.total : 0, err, err_len)) return rc;
    AttnArgs a = make_args(query, key, value, strides, attn_mask, mask_strides, key_padding_mask, B, Q, N, H, Hk, D,
                           scale, causal);
    a.out = out;
    a.rest = dtype == TD_F16 || dtype == TD_BF16 ? rest : nullptr;
    a.lse = lse;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (N > 0 && attn_tc_fits(dtype, a))
        return attn_tc_forward(dtype, a, ws, mb, mh, static_cast<unsigned char*>(workspace), s, err, err_len);
    switch (dtype) {
        case TD_F32: return forward<float>(a, s, err, err_len);
        case TD_F16: return forward<__half>(a, s, err, err_len);
        case TD_BF16: return forward<__nv_bfloat16>(a, s, err, err_len);
        default: return forward<double>(a, s, err, err_len);
    }
}

int td_attention_backward(int dtype, const void* query, const void* key, const void* value, const int64_t* strides,
                          const uint8_t* attn_mask, const int64_t* mask_strides, const uint8_t* key_padding_mask,
                          const void* out, const void* rest, const void* lse, const void* grad_out, void* grad_query, void* grad_key,
                          void* grad_value, int64_t B, int64_t Q, int64_t N, int64_t H, int64_t Hk, int64_t D,
                          double scale, int causal, void* workspace, size_t workspace_bytes, void* stream, char* err,
                          size_t err_len) {
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
    const AttnWorkspace ws = attn_workspace(dtype, B, Q, N, H, mb, mh, key_padding_mask != nullptr, true);
    if (int rc = check_workspace(workspace, workspace_bytes, ws.total, err, err_len)) return rc;
    AttnArgs a = make_args(query, key, value, strides, attn_mask, mask_strides, key_padding_mask, B, Q, N, H, Hk, D,
                           scale, causal);
    a.out_in = out;
    a.rest_in = dtype == TD_F16 || dtype == TD_BF16 ? rest : nullptr;
    a.lse = const_cast<void*>(lse);
    a.grad_out = grad_out;
    a.grad_q = grad_query;
    a.grad_k = grad_key;
    a.grad_v = grad_value;
    a.delta = static_cast<unsigned char*>(workspace) + ws.delta;
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
