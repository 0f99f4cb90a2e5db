// td_attention_plan.h -- what the attention's two translation units share on the host: the workspace's layout and the
// tensor-core launches (td_attention_tc.cu) behind the entry points (td_attention.cu).
#pragma once

#include "td_attention_split.cuh"
#include "td_host.h"

namespace td {

// Byte offsets into a call's workspace, and the sizes of the packed mask (rows = 1: from the padding alone).
struct AttnWorkspace {
    size_t part_o, part_ml, part_k, part_v, part_q, amax, row_g, keys_lse, delta;
    size_t row_bits, row_flags, col_bits, col_flags, total;
    int64_t images, heads, rows, words, col_words;
};

// Joins the partials of a split forward.
template <typename T>
int combine(const SplitArgs& p, cudaStream_t stream, char* err, size_t err_len) {
    if (p.splits == 1) return TD_OK;
    const long long rows = (long long)p.a.B * p.a.H * p.a.Q;
    const bool wide = rows <= 8 * kSms;  // (2 x 300 x 8 rows of 6 splits: 13 us wide, 4 narrow)
    const long long blocks = wide ? rows : (rows + kCombineWarps - 1) / kCombineWarps;
    return host::launch(err, err_len, "attn_combine_kernel",
                        wide ? attn_combine_kernel<T, kCombineWarps> : attn_combine_kernel<T, 1>,
                        dim3(unsigned(blocks)), dim3(kCombineWarps * 32), 0, stream, true, p);
}

// Adds the partial gradients of a split backward.
template <typename T>
int join(const AttnArgs& a, cudaStream_t stream, char* err, size_t err_len) {
    const long long n = (a.k_splits > 1 ? 2LL * a.B * a.N * a.Hk * a.D : 0) +
                        (a.q_splits > 1 ? (long long)a.B * a.Q * a.H * a.D : 0);
    if (n == 0) return TD_OK;
    return host::launch(err, err_len, "attn_join_kernel", attn_join_kernel<T>, dim3(unsigned((n + 255) / 256)),
                        dim3(256), 0, stream, true, a);
}

// CTAs of the tensor-core backward's delta kernel for each of `pairs` (image, key head) pairs, at most: two an SM in
// all.
inline int64_t attn_delta_parts(int64_t pairs) { return pairs < 2 * kSms ? 2 * kSms / pairs : 1; }
// How many CTAs share the keys of a query tile in the tensor-core forward.
int64_t attn_tc_splits(int64_t B, int64_t Q, int64_t N, int64_t H);
// Whether the tensor-core kernels take this call.
bool attn_tc_fits(int dtype, const AttnArgs& a);
// mb, mh: images and heads the mask has of its own (0: no mask).
int attn_tc_forward(int dtype, const AttnArgs& a, const AttnWorkspace& w, int64_t mb, int64_t mh,
                    unsigned char* workspace, cudaStream_t stream, char* err, size_t err_len);
int attn_tc_backward(int dtype, const AttnArgs& a, const AttnWorkspace& w, int64_t mb, int64_t mh,
                     unsigned char* workspace, cudaStream_t stream, char* err, size_t err_len);

}  // namespace td
