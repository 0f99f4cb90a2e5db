// td_rms_norm.cu -- the root-mean-square norm entry points of the C ABI: argument contract, kernel choice and launches.
#include <algorithm>
#include <type_traits>

#include "td_host.h"
#include "td_rms_norm.cuh"

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

enum Pass { kForward, kForward8, kBackward };

template <typename T, int VEC, Pass P>
int launch_rms(const RmsArgs<T>& a, int* grid, cudaStream_t stream, char* err, size_t err_len) {
    auto go = [&](auto g, auto ept) {
        constexpr int G = decltype(g)::value, EPT = decltype(ept)::value;
        constexpr int kCtas = norm_ctas<T, VEC, EPT, P == kBackward>();
        *grid = norm_grid(a.rows, a.C, kCtas);
        if constexpr (P == kBackward) {
            static_assert(kCtas <= kMostCtas, "workspace");
            constexpr auto kernel = rms_backward_kernel<T, VEC, G, EPT>;
            constexpr size_t smem = rms_smem<T, VEC, EPT>();
            static_assert((smem + 9216 + 1024) * kCtas <= 228 * 1024, "shared memory of an SM");
            // (the kernel's static arrays count towards the 48 KB that need no raising)
            if (int rc = host::allow_smem<kernel>(smem > 0 ? smem + 8192 : 0, err, err_len)) return rc;
            return host::launch(err, err_len, "rms_backward_kernel", kernel, dim3(unsigned(*grid)),
                                dim3(kNormThreads), smem, stream, true, a);
        } else
            return host::launch(err, err_len, "rms_forward_kernel", rms_forward_kernel<T, VEC, G, EPT, P == kForward8>,
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

template <typename T, Pass P>
int pick_rms(const RmsArgs<T>& a, int* grid, cudaStream_t stream, char* err, size_t err_len) {
    constexpr int V = Elem<T>::kVec;
    // 16-byte vectors where every row starts on a 16-byte boundary (the 8-bit rows do by their pitch)
    const bool wide = a.C % V == 0 && aligned16(a.x) && aligned16(a.residual) && aligned16(a.weight) &&
                      aligned16(a.grad_y) && aligned16(a.grad_total) && aligned16(a.out) && aligned16(a.total);
    return wide ? launch_rms<T, V, P>(a, grid, stream, err, err_len)
                : launch_rms<T, 1, P>(a, grid, stream, err, err_len);
}

template <typename T>
int forward(RmsArgs<T> a, const void* x, const void* residual, const void* weight, void* y, void* total, void* rstd,
            double eps, cudaStream_t stream, char* err, size_t err_len) {
    using acc = typename Elem<T>::acc;
    a.x = static_cast<const T*>(x);
    a.residual = static_cast<const T*>(residual);
    a.weight = static_cast<const T*>(weight);
    a.out = static_cast<T*>(y);
    a.total = static_cast<T*>(total);
    a.rstd = static_cast<acc*>(rstd);
    a.eps = acc(eps);
    int grid = 0;
    if constexpr (!std::is_same<T, double>::value) {
        if (a.q != nullptr) return pick_rms<T, kForward8>(a, &grid, stream, err, err_len);
    }
    return pick_rms<T, kForward>(a, &grid, stream, err, err_len);
}

template <typename T>
int backward(const void* grad_y, const void* grad_total, const void* x, const void* residual, const void* weight,
             const void* rstd, void* grad_x, void* grad_weight, int64_t rows, int64_t C, void* workspace,
             cudaStream_t stream, char* err, size_t err_len) {
    using acc = typename Elem<T>::acc;
    RmsArgs<T> a = {};
    a.x = static_cast<const T*>(x);
    a.residual = static_cast<const T*>(residual);
    a.weight = static_cast<const T*>(weight);
    a.grad_y = static_cast<const T*>(grad_y);
    a.grad_total = static_cast<const T*>(grad_total);
    a.out = static_cast<T*>(grad_x);
    a.rstd = static_cast<acc*>(const_cast<void*>(rstd));
    a.partial = static_cast<acc*>(workspace);
    a.rows = rows;
    a.C = int(C);
    int grid = 0;
    if (int rc = pick_rms<T, kBackward>(a, &grid, stream, err, err_len)) return rc;
    if (grad_weight == nullptr) return TD_OK;
    return host::launch(err, err_len, "column_sum_kernel", column_sum_kernel<T, acc>,
                        dim3(unsigned((C + kColumnCols - 1) / kColumnCols)), dim3(kColumnCols * kColumnRows), 0,
                        stream, true, static_cast<const acc*>(a.partial), static_cast<T*>(grad_weight),
                        static_cast<long long>(grid), int(C));
}

}  // namespace
}  // namespace td

extern "C" {

int td_rms_norm_forward(int dtype, const void* x, const void* residual, const void* weight, void* y, void* total,
                        void* q, int64_t q_pitch, float* scale, void* rstd, int64_t rows, int64_t C, double eps,
                        void* stream, char* err, size_t err_len) {
    using namespace td;
    if (int rc = check_norm(dtype, rows, C, eps, err, err_len)) return rc;
    if (q != nullptr) {
        if (dtype == TD_F64) return fail(err, err_len, TD_ERR_ARG, "no 8-bit output for float64");
        if (scale == nullptr || y != nullptr)
            return fail(err, err_len, TD_ERR_ARG, "an 8-bit output has scales, and takes the place of y");
        if (q_pitch < C || q_pitch >= C + 16 || q_pitch % 16 != 0 || (reinterpret_cast<uintptr_t>(q) & 15u) != 0)
            return fail(err, err_len, TD_ERR_ARG, "8-bit rows must be 16-byte aligned, C rounded up to 16 apart");
    }
    if (rows == 0) return TD_OK;
    if (x == nullptr || weight == nullptr || (y == nullptr && q == nullptr))
        return fail(err, err_len, TD_ERR_ARG, "null tensor pointer");
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    auto run = [&](auto zero) {
        using T = decltype(zero);
        RmsArgs<T> a = {};
        a.q = static_cast<uint8_t*>(q);
        a.scale = scale;
        a.rows = rows;
        a.C = int(C);
        a.pitch = int(q_pitch);
        return forward<T>(a, x, residual, weight, y, total, rstd, eps, s, err, err_len);
    };
    switch (dtype) {
        case TD_F32: return run(float());
        case TD_F16: return run(__half());
        case TD_BF16: return run(__nv_bfloat16());
        default: return run(double());
    }
}

size_t td_rms_norm_workspace_bytes(int dtype, int64_t rows, int64_t C) {
    using namespace td;
    if (dtype < TD_F32 || dtype > TD_F64 || rows <= 0 || C <= 0) return 0;
    return size_t(norm_grid(rows, C, kMostCtas)) * size_t(C) * (dtype == TD_F64 ? 8 : 4);
}

int td_rms_norm_backward(int dtype, const void* grad_y, const void* grad_total, const void* x, const void* residual,
                         const void* weight, const void* rstd, void* grad_x, void* grad_weight, int64_t rows,
                         int64_t C, void* workspace, size_t workspace_bytes, void* stream, char* err,
                         size_t err_len) {
    using namespace td;
    if (int rc = check_norm(dtype, rows, C, 0, err, err_len)) return rc;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (rows == 0) {
        const size_t bytes = size_t(C) * (dtype == TD_F64 ? 8 : dtype == TD_F32 ? 4 : 2);
        if (grad_weight != nullptr && cudaMemsetAsync(grad_weight, 0, bytes, s) != cudaSuccess)
            return fail(err, err_len, TD_ERR_CUDA, "memset: %s", cudaGetErrorString(cudaGetLastError()));
        return TD_OK;
    }
    if (grad_y == nullptr || x == nullptr || weight == nullptr || rstd == nullptr || grad_x == nullptr)
        return fail(err, err_len, TD_ERR_ARG, "null tensor pointer");
    const size_t need = td_rms_norm_workspace_bytes(dtype, rows, C);
    if (workspace == nullptr || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 7u) != 0)
        return fail(err, err_len, TD_ERR_WORKSPACE, "workspace must be 8-byte aligned, of %zu bytes (got %zu)", need,
                    workspace_bytes);
    auto run = [&](auto zero) {
        return backward<decltype(zero)>(grad_y, grad_total, x, residual, weight, rstd, grad_x, grad_weight, rows, C,
                                        workspace, s, err, err_len);
    };
    switch (dtype) {
        case TD_F32: return run(float());
        case TD_F16: return run(__half());
        case TD_BF16: return run(__nv_bfloat16());
        default: return run(double());
    }
}

}  // extern "C"
