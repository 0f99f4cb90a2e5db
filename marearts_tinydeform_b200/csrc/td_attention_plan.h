// td_attention_plan.h -- what the attention's two translation units share on the host: the workspace's layout and the
// tensor-core launches (td_attention_tc.cu) behind the entry points (td_attention.cu).
#pragma once

#include "td_attention_split.cuh"
#include "td_host.h"

namespace td {

// Byte offsets into a call's workspace, and the sizes of the packed mask (rows = 1: from the padding alone).
struct AttnWorkspace {
    size_t part_o, part_ml, amax, delta, row_bits, row_flags, col_bits, col_flags, total;
    int64_t images, heads, rows, words, col_words;
};

// Whether the tensor-core kernels take this call.
bool attn_tc_fits(int dtype, const AttnArgs& a);
// mb, mh: images and heads the mask has of its own (0: no mask).
int attn_tc_forward(int dtype, const AttnArgs& a, const AttnWorkspace& w, int64_t mb, int64_t mh,
                    unsigned char* workspace, cudaStream_t stream, char* err, size_t err_len);
int attn_tc_backward(int dtype, const AttnArgs& a, const AttnWorkspace& w, int64_t mb, int64_t mh,
                     unsigned char* workspace, cudaStream_t stream, char* err, size_t err_len);

}  // namespace td
