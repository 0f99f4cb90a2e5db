// td_attention_tc.cu -- launches of the attention's tensor-core kernels: conditions, tensor maps, packed masks.
#include <algorithm>

#include "td_attention_plan.h"
#include "td_attention_tc.cuh"

namespace td {

cudaError_t attention_tc_device_error(int clear, unsigned int* code) {
    cudaError_t e = cudaMemcpyFromSymbol(code, g_device_error, sizeof(*code));
    if (e == cudaSuccess && clear) {
        const unsigned int zero = 0;
        e = cudaMemcpyToSymbol(g_device_error, &zero, sizeof(zero));
    }
    return e;
}

namespace {

using host::fail;

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// A [B, T, heads, D] operand with its element strides, as the tensor maps see it.
struct Operand {
    const void* base;
    int tokens, heads;
    long long s_b, s_t, s_h;
};

Operand query_of(const AttnArgs& a) { return {a.q, a.Q, a.H, a.q_b, a.q_t, a.q_h}; }
Operand key_of(const AttnArgs& a) { return {a.k, a.N, a.Hk, a.k_b, a.k_t, a.k_h}; }
Operand value_of(const AttnArgs& a) { return {a.v, a.N, a.Hk, a.v_b, a.v_t, a.v_h}; }
Operand grad_of(const AttnArgs& a) {
    const long long row = (long long)a.H * a.D;
    return {a.grad_out, a.Q, a.H, a.Q * row, row, a.D};
}

// The stride of a dimension of one element says nothing: any legal one will do.
long long map_stride(long long stride, int size, const AttnArgs& a) { return size > 1 ? stride : (a.D + 7) / 8 * 8; }

bool operand_fits(const Operand& o, const AttnArgs& a) {
    const long long s[3] = {map_stride(o.s_t, o.tokens, a), map_stride(o.s_h, o.heads, a), map_stride(o.s_b, a.B, a)};
    for (long long x : s)
        if (x <= 0 || x % 8 != 0 || x >= (1LL << 38)) return false;
    return aligned16(o.base);
}

// Boxes of min(DP, 64) columns x 64 tokens of one head of one image (a resident operand of 128 rows takes two, which
// lie behind one another as one of 128 would); what lies outside reads as zero.
template <int DP>
int make_map(CUtensorMap* map, const Operand& o, const AttnArgs& a, char* err, size_t err_len) {
    const uint64_t dims[4] = {uint64_t(a.D), uint64_t(o.tokens), uint64_t(o.heads), uint64_t(a.B)};
    const uint64_t strides[3] = {uint64_t(map_stride(o.s_t, o.tokens, a)) * 2,
                                 uint64_t(map_stride(o.s_h, o.heads, a)) * 2,
                                 uint64_t(map_stride(o.s_b, a.B, a)) * 2};
    const uint32_t box[4] = {uint32_t(AttnBox<DP>::kCols), uint32_t(kAttnBN), 1, 1};
    const CUresult r = host::encode_tiled_u16(map, 4, o.base, dims, strides, box,
                                              DP == 32 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B);
    if (r == CUDA_SUCCESS) return TD_OK;
    return fail(err, err_len, TD_ERR_CUDA, "cuTensorMapEncodeTiled (attention) failed (%d)", int(r));
}

// Packs the masks of a call (if any) and fills args' pointers and strides.
int pack_masks(AttnTcArgs& t, const AttnWorkspace& w, int64_t mb, int64_t mh, bool backward, unsigned char* workspace,
               cudaStream_t stream, char* err, size_t err_len) {
    const AttnArgs& a = t.a;
    if (w.images == 0) return TD_OK;
    PackArgs p = {};
    p.mask = a.mask;
    p.padding = a.padding;
    p.m_b = a.m_b; p.m_h = a.m_h; p.m_q = a.m_q;
    p.images = int(w.images); p.heads = int(w.heads); p.rows = int(w.rows); p.N = a.N;
    p.words = int(w.words);
    p.row_bits = reinterpret_cast<uint32_t*>(workspace + w.row_bits);
    p.row_flags = workspace + w.row_flags;
    const long long q_tiles = (w.rows + 127) / 128, k_tiles = (a.N + 127) / 128;
    t.row_bits = p.row_bits;
    t.row_flags = p.row_flags;
    t.rb_q = mb > 0 ? w.words : 0;
    t.rb_h = w.heads > 1 ? w.rows * w.words : 0;
    t.rb_b = w.images > 1 ? w.heads * w.rows * w.words : 0;
    t.rf_q = mb > 0 ? w.words / 2 : 0;
    t.rf_h = w.heads > 1 ? q_tiles * (w.words / 2) : 0;
    t.rf_b = w.images > 1 ? w.heads * q_tiles * (w.words / 2) : 0;
    if (backward && mb > 0) {
        p.mask_images = int(mb);
        p.col_words = int(w.col_words);
        p.col_bits = reinterpret_cast<uint32_t*>(workspace + w.col_bits);
        p.col_flags = workspace + w.col_flags;
        t.col_bits = p.col_bits;
        t.col_flags = p.col_flags;
        t.col_words = p.col_words;
        t.col_tiles = p.col_words / 2;
        t.cb_h = mh > 1 ? (long long)a.N * w.col_words : 0;
        t.cb_b = mb > 1 ? mh * (long long)a.N * w.col_words : 0;
        t.cf_h = mh > 1 ? k_tiles * t.col_tiles : 0;
        t.cf_b = mb > 1 ? mh * k_tiles * t.col_tiles : 0;
    }
    const long long blocks = w.images * w.heads * q_tiles * k_tiles;
    if (blocks > INT32_MAX) return fail(err, err_len, TD_ERR_ARG, "attn_mask is too large");
    return host::launch(err, err_len, "attn_pack_kernel", attn_pack_kernel, dim3(unsigned(blocks)),
                        dim3(kPackThreads), 0, stream, true, p);
}

template <typename T, int DP>
int forward(AttnTcArgs& t, const AttnWorkspace& w, int64_t mb, int64_t mh, unsigned char* workspace,
            cudaStream_t stream, char* err, size_t err_len) {
    const AttnArgs& a = t.a;
    CUtensorMap q, k, v;
    if (int rc = make_map<DP>(&q, query_of(a), a, err, err_len)) return rc;
    if (int rc = make_map<DP>(&k, key_of(a), a, err, err_len)) return rc;
    if (int rc = make_map<DP>(&v, value_of(a), a, err, err_len)) return rc;
    if (int rc = pack_masks(t, w, mb, mh, false, workspace, stream, err, err_len)) return rc;
    constexpr auto kernel = attn_tc_forward_kernel<T, DP>;
    constexpr size_t smem = AttnFwdLayout<DP>::kSmemBytes;
    if (int rc = host::allow_smem<kernel>(smem, err, err_len)) return rc;
    t.splits = int(attn_tc_splits(a.B, a.Q, a.N, a.H));
    SplitArgs p = {};
    p.a = a;
    p.splits = t.splits;
    p.part_o = workspace + w.part_o;
    p.part_ml = workspace + w.part_ml;
    t.part_o = static_cast<float*>(p.part_o);
    t.part_ml = static_cast<float*>(p.part_ml);
    const unsigned grid = unsigned((a.Q + kAttnBM - 1) / kAttnBM) * unsigned(a.B * a.H * t.splits);
    if (int rc = host::launch(err, err_len, "attn_tc_forward_kernel", kernel, dim3(grid), dim3(kAttnFwdThreads), smem,
                              stream, true, q, k, v, t))
        return rc;
    return combine<T>(p, stream, err, err_len);
}

template <typename T, int DP>
int backward(AttnTcArgs& t, const AttnWorkspace& w, int64_t mb, int64_t mh, unsigned char* workspace,
             cudaStream_t stream, char* err, size_t err_len) {
    const AttnArgs& a = t.a;
    CUtensorMap q, g, k, v;
    if (int rc = make_map<DP>(&q, query_of(a), a, err, err_len)) return rc;
    if (int rc = make_map<DP>(&g, grad_of(a), a, err, err_len)) return rc;
    if (int rc = make_map<DP>(&k, key_of(a), a, err, err_len)) return rc;
    if (int rc = make_map<DP>(&v, value_of(a), a, err, err_len)) return rc;
    if (int rc = pack_masks(t, w, mb, mh, true, workspace, stream, err, err_len)) return rc;
    int lanes = 1;
    while (lanes * 8 < a.D) lanes *= 2;
    const long long rows = std::max((long long)(a.H / a.Hk) * a.Qp, (long long)a.N);
    const int per_block = kDeltaThreads / lanes, pairs = a.B * a.Hk;
    float* row_g = reinterpret_cast<float*>(workspace + w.row_g);
    float* amax = reinterpret_cast<float*>(workspace + w.amax);
    float* keys_lse = reinterpret_cast<float*>(workspace + w.keys_lse);
    t.keys_lse = attn_p_bits<T>() != 0 ? keys_lse : static_cast<const float*>(a.lse);
    t.row_g = row_g;
    t.amax = amax;
    t.amax_parts = int(std::min<long long>(attn_delta_parts(pairs), (rows + per_block - 1) / per_block));
    if (int rc = host::launch(err, err_len, "attn_delta_tc_kernel", attn_delta_tc_kernel<T>,
                              dim3(unsigned(pairs) * unsigned(t.amax_parts)), dim3(kDeltaThreads), 0, stream, true, a,
                              lanes, t.amax_parts, keys_lse, row_g, amax))
        return rc;
    t.kv_blocks = (a.N + kAttnBM - 1) / kAttnBM * a.B * a.Hk * a.k_splits;
    constexpr auto kernel = attn_tc_backward_kernel<T, DP>;
    constexpr size_t smem = AttnBwdLayout<DP>::kSmemBytes;
    if (int rc = host::allow_smem<kernel>(smem, err, err_len)) return rc;
    const unsigned grid =
        unsigned(t.kv_blocks) + unsigned((a.Q + kAttnBM - 1) / kAttnBM) * unsigned(a.B * a.H * a.q_splits);
    if (int rc = host::launch(err, err_len, "attn_tc_backward_kernel", kernel, dim3(grid),
                              dim3(AttnBwdLayout<DP>::kThreads), smem, stream, true, q, g, k, v, t))
        return rc;
    return join<T>(a, stream, err, err_len);
}

}  // namespace

// One wave of two CTAs an SM (300 queries on 8400 keys, 8 heads of 32: 112 us unsplit, 23 in 12 splits; 2 images 112
// and 35), of at least 512 keys a split and where two splits save more than joining them costs for any number of images
// (1024 keys: 16.6 us unsplit, in two 13.5 for one image and 19.3 for four; 1600 keys: 24 and 15).
int64_t attn_tc_splits(int64_t B, int64_t Q, int64_t N, int64_t H) {
    const int64_t ctas = (Q + kAttnBM - 1) / kAttnBM * B * H;
    if (N < 1536 || ctas == 0) return 1;
    return std::max<int64_t>(1, std::min<int64_t>(2 * kSms / ctas, N / 512));
}

bool attn_tc_fits(int dtype, const AttnArgs& a) {
    if ((dtype != TD_F16 && dtype != TD_BF16) || !host::best_policy()) return false;
    if (a.D % 8 != 0) return false;
    // One key, where the gradients of queries and keys are zero: the CUDA-core kernels form dP and delta in one order
    // and find it so (8 images of 8 heads x 32, 32 queries: 7.7 us forward against 4.6).
    if (a.N < 2) return false;
    if (!operand_fits(query_of(a), a) || !operand_fits(key_of(a), a) || !operand_fits(value_of(a), a)) return false;
    if (!aligned16(a.lse)) return false;
    if (a.grad_q == nullptr) return aligned16(a.out) && aligned16(a.rest);
    return operand_fits(grad_of(a), a) && aligned16(a.out_in) && a.rest_in != nullptr && aligned16(a.rest_in) &&
           aligned16(a.grad_q) && aligned16(a.grad_k) && aligned16(a.grad_v);
}

int attn_tc_forward(int dtype, const AttnArgs& a, const AttnWorkspace& w, int64_t mb, int64_t mh,
                    unsigned char* workspace, cudaStream_t stream, char* err, size_t err_len) {
    AttnTcArgs t = {};
    t.a = a;
    auto go = [&](auto type) {
        using T = decltype(type);
        if (a.D <= 32) return forward<T, 32>(t, w, mb, mh, workspace, stream, err, err_len);
        if (a.D <= 64) return forward<T, 64>(t, w, mb, mh, workspace, stream, err, err_len);
        return forward<T, 128>(t, w, mb, mh, workspace, stream, err, err_len);
    };
    return dtype == TD_F16 ? go(__half{}) : go(__nv_bfloat16{});
}

int attn_tc_backward(int dtype, const AttnArgs& a, const AttnWorkspace& w, int64_t mb, int64_t mh,
                     unsigned char* workspace, cudaStream_t stream, char* err, size_t err_len) {
    AttnTcArgs t = {};
    t.a = a;
    auto go = [&](auto type) {
        using T = decltype(type);
        if (a.D <= 32) return backward<T, 32>(t, w, mb, mh, workspace, stream, err, err_len);
        if (a.D <= 64) return backward<T, 64>(t, w, mb, mh, workspace, stream, err, err_len);
        return backward<T, 128>(t, w, mb, mh, workspace, stream, err, err_len);
    };
    return dtype == TD_F16 ? go(__half{}) : go(__nv_bfloat16{});
}

}  // namespace td
