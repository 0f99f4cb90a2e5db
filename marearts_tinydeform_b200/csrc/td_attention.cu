// td_attention.cu -- the attention entry points of the C ABI: argument contract, kernel choice and launches.
#include <cmath>

#include "td_attention.cuh"
#include "td_host.h"

namespace td {

cudaError_t attention_device_error(int clear, unsigned int* code) {
    cudaError_t e = cudaMemcpyFromSymbol(code, g_device_error, sizeof(*code));
    if (e == cudaSuccess && clear) {
        const unsigned int zero = 0;
        e = cudaMemcpyToSymbol(g_device_error, &zero, sizeof(zero));
    }
    return e;
}

namespace {

using host::fail;

int64_t pad_rows(int64_t Q) { return (Q + kAttnRowPad - 1) / kAttnRowPad * kAttnRowPad; }
size_t elem_bytes(int dtype) { return dtype == TD_F64 ? 8 : dtype == TD_F32 ? 4 : 2; }
size_t acc_bytes(int dtype) { return dtype == TD_F64 ? 8 : 4; }

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
    if (!(scale > 0) || !std::isfinite(scale))
        return fail(err, err_len, TD_ERR_ARG, "scale must be positive and finite");
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
                              dim3(unsigned((rows + 7) / 8)), dim3(256), 0, stream, true, a))
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
    (void)mask_b; (void)mask_h; (void)has_padding;
    if (check_sizes(dtype, B, Q, N, H, Hk, D, 1.0, nullptr, 0) != TD_OK) return 0;
    return backward ? size_t(B) * H * pad_rows(Q) * acc_bytes(dtype) : 0;
}

int td_attention_forward(int dtype, const void* query, const void* key, const void* value, const int64_t* strides,
                         const uint8_t* attn_mask, const int64_t* mask_strides, const uint8_t* key_padding_mask,
                         void* out, void* lse, int64_t B, int64_t Q, int64_t N, int64_t H, int64_t Hk, int64_t D,
                         double scale, int causal, void* workspace, size_t workspace_bytes, void* stream, char* err,
                         size_t err_len) {
    using namespace td;
    if (int rc = check_sizes(dtype, B, Q, N, H, Hk, D, scale, err, err_len)) return rc;
    if (B == 0 || Q == 0) return TD_OK;
    if (query == nullptr || out == nullptr || strides == nullptr || (N > 0 && (key == nullptr || value == nullptr)) ||
        (attn_mask != nullptr && mask_strides == nullptr))
        return fail(err, err_len, TD_ERR_ARG, "null tensor pointer");
    (void)workspace; (void)workspace_bytes;
    AttnArgs a = make_args(query, key, value, strides, attn_mask, mask_strides, key_padding_mask, B, Q, N, H, Hk, D,
                           scale, causal);
    a.out = out;
    a.lse = lse;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    switch (dtype) {
        case TD_F32: return forward<float>(a, s, err, err_len);
        case TD_F16: return forward<__half>(a, s, err, err_len);
        case TD_BF16: return forward<__nv_bfloat16>(a, s, err, err_len);
        default: return forward<double>(a, s, err, err_len);
    }
}

int td_attention_backward(int dtype, const void* query, const void* key, const void* value, const int64_t* strides,
                          const uint8_t* attn_mask, const int64_t* mask_strides, const uint8_t* key_padding_mask,
                          const void* out, const void* lse, const void* grad_out, void* grad_query, void* grad_key,
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
    const size_t need = td_attention_workspace_bytes(dtype, B, Q, N, H, Hk, D, 0, 0, 0, 1);
    if (workspace == nullptr || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15u) != 0)
        return fail(err, err_len, TD_ERR_WORKSPACE, "workspace must be 16-byte aligned, of %zu bytes (got %zu)", need,
                    workspace_bytes);
    AttnArgs a = make_args(query, key, value, strides, attn_mask, mask_strides, key_padding_mask, B, Q, N, H, Hk, D,
                           scale, causal);
    a.out_in = out;
    a.lse = const_cast<void*>(lse);
    a.grad_out = grad_out;
    a.grad_q = grad_query;
    a.grad_k = grad_key;
    a.grad_v = grad_value;
    a.delta = workspace;
    switch (dtype) {
        case TD_F32: return backward<float>(a, s, err, err_len);
        case TD_F16: return backward<__half>(a, s, err, err_len);
        case TD_BF16: return backward<__nv_bfloat16>(a, s, err, err_len);
        default: return backward<double>(a, s, err, err_len);
    }
}

}  // extern "C"
