// td_norm.cu -- the layer norm entry points of the C ABI: argument contract, kernel choice and launches.
#include <algorithm>
#include <type_traits>

#include "td_host.h"
#include "td_norm.cuh"

namespace td {
namespace {

using host::fail;

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int check_norm(int dtype, int64_t rows, int64_t C, double eps, char* err, size_t err_len) {
    if (dtype < TD_F32 || dtype > TD_F64) return fail(err, err_len, TD_ERR_ARG, "unsupported dtype %d", dtype);
    if (rows < 0) return fail(err, err_len, TD_ERR_ARG, "sizes must be non-negative");
    if (C < 1 || C > TD_MAX_CHANNELS)
        return fail(err, err_len, TD_ERR_ARG, "channels must be between 1 and %d", TD_MAX_CHANNELS);
    if (!(eps >= 0)) return fail(err, err_len, TD_ERR_ARG, "eps must not be negative");
    return TD_OK;
}

// Rows a CTA holds at once: a warp a row up to 512 channels, 4 warps up to 2048, 8 above.
int groups_of(int64_t C) { return C <= 512 ? 8 : C <= 2048 ? 2 : 1; }

// The CTAs of a launch with `per_sm` on each SM: one wave, or fewer when there are fewer rows.
int norm_grid(int64_t rows, int64_t C, int per_sm) {
    const int64_t need = (rows + groups_of(C) - 1) / groups_of(C);
    return int(std::min<int64_t>(need, int64_t(kSms) * per_sm));
}
constexpr int kMostCtas = 3;  // of any backward form: the workspace's partial rows

template <typename T, int VEC, bool BWD>
int launch_norm(const NormArgs<T>& a, int* grid, cudaStream_t stream, char* err, size_t err_len) {
    auto go = [&](auto g, auto ept) {
        constexpr int G = decltype(g)::value, EPT = decltype(ept)::value, kCtas = norm_ctas<T, VEC, EPT, BWD>();
        static_assert(!BWD || kCtas <= kMostCtas, "workspace");
        *grid = norm_grid(a.rows, a.C, kCtas);
        if constexpr (BWD) {
            constexpr auto kernel = norm_backward_kernel<T, VEC, G, EPT>;
            constexpr size_t smem = norm_smem<T, VEC, EPT>();
            // (the kernel's static arrays count towards the 48 KB that need no raising)
            if (int rc = host::allow_smem<kernel>(smem > 0 ? smem + 8192 : 0, err, err_len)) return rc;
            return host::launch(err, err_len, "norm_backward_kernel", kernel, dim3(unsigned(*grid)),
                                dim3(kNormThreads), smem, stream, true, a);
        } else
            return host::launch(err, err_len, "norm_forward_kernel", norm_forward_kernel<T, VEC, G, EPT>,
                                dim3(unsigned(*grid)), dim3(kNormThreads), 0, stream, true, a);
    };
    using std::integral_constant;
    const integral_constant<int, 32> warp;
    const integral_constant<int, 128> four;
    const integral_constant<int, 256> eight;
    const integral_constant<int, 8> e8;
    const integral_constant<int, 16> e16;
    const integral_constant<int, 32> e32;
    if (a.C <= 256) return go(warp, e8);
    if (a.C <= 512) return go(warp, e16);
    if (a.C <= 1024) return go(four, e8);
    if (a.C <= 2048) return go(four, e16);
    if (a.C <= 4096) return go(eight, e16);
    return go(eight, e32);
}

template <typename T, bool BWD>
int pick_norm(const NormArgs<T>& a, int* grid, cudaStream_t stream, char* err, size_t err_len) {
    constexpr int V = Elem<T>::kVec;
    // 16-byte vectors where every row starts on a 16-byte boundary
    const bool wide = a.C % V == 0 && aligned16(a.x) && aligned16(a.residual) && aligned16(a.weight) &&
                      aligned16(a.bias) && aligned16(a.grad_y) && aligned16(a.out);
    return wide ? launch_norm<T, V, BWD>(a, grid, stream, err, err_len)
                : launch_norm<T, 1, BWD>(a, grid, stream, err, err_len);
}

template <typename T>
int forward(const void* x, const void* residual, const void* weight, const void* bias, void* y, void* mean,
            void* rstd, int64_t rows, int64_t C, double eps, cudaStream_t stream, char* err, size_t err_len) {
    using acc = typename Elem<T>::acc;
    NormArgs<T> a = {};
    a.x = static_cast<const T*>(x);
    a.residual = static_cast<const T*>(residual);
    a.weight = static_cast<const T*>(weight);
    a.bias = static_cast<const T*>(bias);
    a.out = static_cast<T*>(y);
    a.mean = static_cast<acc*>(mean);
    a.rstd = static_cast<acc*>(rstd);
    a.rows = rows;
    a.C = int(C);
    a.eps = acc(eps);
    int grid = 0;
    return pick_norm<T, false>(a, &grid, stream, err, err_len);
}

template <typename T>
int backward(const void* grad_y, const void* x, const void* residual, const void* weight, const void* mean,
             const void* rstd, void* grad_x, void* grad_weight, void* grad_bias, int64_t rows, int64_t C,
             void* workspace, cudaStream_t stream, char* err, size_t err_len) {
    using acc = typename Elem<T>::acc;
    NormArgs<T> a = {};
    a.x = static_cast<const T*>(x);
    a.residual = static_cast<const T*>(residual);
    a.weight = static_cast<const T*>(weight);
    a.grad_y = static_cast<const T*>(grad_y);
    a.out = static_cast<T*>(grad_x);
    a.mean = static_cast<acc*>(const_cast<void*>(mean));
    a.rstd = static_cast<acc*>(const_cast<void*>(rstd));
    a.partial = static_cast<acc*>(workspace);
    a.rows = rows;
    a.C = int(C);
    int grid = 0;
    if (int rc = pick_norm<T, true>(a, &grid, stream, err, err_len)) return rc;
    return host::launch(err, err_len, "norm_reduce_kernel", norm_reduce_kernel<T>,
                        dim3(unsigned((2 * C + kReduceCols - 1) / kReduceCols)), dim3(kReduceCols * kReduceRows), 0,
                        stream, true, static_cast<const acc*>(a.partial), static_cast<T*>(grad_weight),
                        static_cast<T*>(grad_bias), grid, int(C));
}

}  // namespace
}  // namespace td

extern "C" {

int td_layer_norm_forward(int dtype, const void* x, const void* residual, const void* weight, const void* bias,
                          void* y, void* mean, void* rstd, int64_t rows, int64_t C, double eps, void* stream,
                          char* err, size_t err_len) {
    using namespace td;
    if (int rc = check_norm(dtype, rows, C, eps, err, err_len)) return rc;
    if (rows == 0) return TD_OK;
    if (x == nullptr || weight == nullptr || y == nullptr || (mean == nullptr) != (rstd == nullptr))
        return fail(err, err_len, TD_ERR_ARG, "null tensor pointer");
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    switch (dtype) {
        case TD_F32: return forward<float>(x, residual, weight, bias, y, mean, rstd, rows, C, eps, s, err, err_len);
        case TD_F16: return forward<__half>(x, residual, weight, bias, y, mean, rstd, rows, C, eps, s, err, err_len);
        case TD_BF16:
            return forward<__nv_bfloat16>(x, residual, weight, bias, y, mean, rstd, rows, C, eps, s, err, err_len);
        default: return forward<double>(x, residual, weight, bias, y, mean, rstd, rows, C, eps, s, err, err_len);
    }
}

size_t td_layer_norm_workspace_bytes(int dtype, int64_t rows, int64_t C) {
    using namespace td;
    if (dtype < TD_F32 || dtype > TD_F64 || rows <= 0 || C <= 0) return 0;
    return size_t(norm_grid(rows, C, kMostCtas)) * 2 * size_t(C) * (dtype == TD_F64 ? 8 : 4);
}

int td_layer_norm_backward(int dtype, const void* grad_y, const void* x, const void* residual, const void* weight,
                           const void* mean, const void* rstd, void* grad_x, void* grad_weight, void* grad_bias,
                           int64_t rows, int64_t C, void* workspace, size_t workspace_bytes, void* stream, char* err,
                           size_t err_len) {
    using namespace td;
    if (int rc = check_norm(dtype, rows, C, 0, err, err_len)) return rc;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (rows == 0) {
        const size_t bytes = size_t(C) * (dtype == TD_F64 ? 8 : dtype == TD_F32 ? 4 : 2);
        for (void* p : {grad_weight, grad_bias})
            if (p != nullptr && cudaMemsetAsync(p, 0, bytes, s) != cudaSuccess)
                return fail(err, err_len, TD_ERR_CUDA, "memset: %s", cudaGetErrorString(cudaGetLastError()));
        return TD_OK;
    }
    if (grad_y == nullptr || x == nullptr || weight == nullptr || mean == nullptr || rstd == nullptr ||
        grad_x == nullptr)
        return fail(err, err_len, TD_ERR_ARG, "null tensor pointer");
    const size_t need = td_layer_norm_workspace_bytes(dtype, rows, C);
    if (workspace == nullptr || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 7u) != 0)
        return fail(err, err_len, TD_ERR_WORKSPACE, "workspace must be 8-byte aligned, of %zu bytes (got %zu)", need,
                    workspace_bytes);
    switch (dtype) {
        case TD_F32:
            return backward<float>(grad_y, x, residual, weight, mean, rstd, grad_x, grad_weight, grad_bias, rows, C,
                                   workspace, s, err, err_len);
        case TD_F16:
            return backward<__half>(grad_y, x, residual, weight, mean, rstd, grad_x, grad_weight, grad_bias, rows, C,
                                    workspace, s, err, err_len);
        case TD_BF16:
            return backward<__nv_bfloat16>(grad_y, x, residual, weight, mean, rstd, grad_x, grad_weight, grad_bias,
                                           rows, C, workspace, s, err, err_len);
        default:
            return backward<double>(grad_y, x, residual, weight, mean, rstd, grad_x, grad_weight, grad_bias, rows, C,
                                    workspace, s, err, err_len);
    }
}

}  // extern "C"
