"""marearts-tinydeform on B200: value projection + multi-scale deformable attention for DETR-style decoders.

The operator of upstream ``marearts_tinydeform`` (``marearts_tinydeform/__init__.py:1-79``), computed by hand-written
sm_100a kernels behind a C ABI (include/tinydeform.h). The drop-in for upstream's callers is the import name
``marearts_tinydeform``, whose ``ma_deform_attn`` keeps upstream's contract exactly (inference only); this package's
own ``ma_deform_attn`` takes the same arguments plus the additions below and also differentiates:

    ma_deform_attn(memory, value_weight, value_bias, spatial_shapes, level_start_index,
                   sampling_locations, attention_weights, mode='auto')  -> [B, Q, H * D]

  mode='fused'    gather memory rows first, then project one vector per (query, head)
  mode='project'  project every memory token (our own GEMM kernel), then sample per head
  mode='auto'     choose_mode() picks one from the shapes, with crossovers measured on B200

Around the operator (additions; upstream has only the operator):

    deform_attn_layer(query, reference_points, memory, spatial_shapes, level_start_index, n_heads, n_points,
                      sampling_weight, sampling_bias, value_weight, value_bias, ...)   -> [B, Q, H * D | C_out]
    sampling_producer(query, reference_points, spatial_shapes, n_heads, n_points, sampling_weight, sampling_bias)
        -> sampling_locations, attention_weights
    pack_sampling_weights(offset_weight, offset_bias, attention_weight, attention_bias) -> the packed pair

the whole MSDeformAttn layer (query -> offsets and softmaxed weights -> attention -> output_proj) in one library call.
The rest of a decoder layer's attention half, forward and backward:

    attention(query, key, value, key_padding_mask, attn_mask, causal, scale)   -> [B, Q, H * D]
    layer_norm(x, weight, bias, residual, eps)                                -> x's shape

the self attention among the queries, and the norm over a sublayer's result plus its residual. Its feed-forward half,
with products in 8-bit floating point (e4m3, a scale for each block of 128), forward and backward:

    rms_norm(x, weight, residual, eps, return_sum, quantize)                   -> x's shape, or 8-bit (data, scale)
    linear_fp8(x, weight, bias, activation, quantize, dtype)                   -> [..., N], or 8-bit (data, scale)
    quantize_fp8(x), quantize_weight_fp8(weight), dequantize_fp8(data, scale, dtype)

CPU tensors run ``ma_deform_attn_reference`` (as upstream does). CUDA tensors run only the native library; if it is
missing, the call raises. Unlike upstream (inference only), this package's ``ma_deform_attn`` differentiates CUDA
inputs that require grad: the forward runs the same kernels and the backward runs this library's backward kernels
(``autograd.py``).
"""

import functools

import torch
from torch.autograd import forward_ad

from . import _native
from .autograd import (AttentionFunction, LayerNormFunction, LinearFp8Function, RmsNormFunction, linear_train,
                       ma_deform_attn_train, producer_train)
from .reference import (attention_reference, deform_attn_layer_reference, dequantize_fp8_reference,
                        layer_norm_reference, linear_fp8_reference, ma_deform_attn_reference,
                        quantize_fp8_reference, quantize_weight_fp8_reference, rms_norm_reference,
                        sampling_producer_reference)

__all__ = ['ma_deform_attn', 'ma_deform_attn_reference', 'choose_mode', 'deform_attn_layer', 'sampling_producer',
           'pack_sampling_weights', 'deform_attn_layer_reference', 'sampling_producer_reference', 'attention',
           'attention_reference', 'layer_norm', 'layer_norm_reference', 'rms_norm', 'rms_norm_reference',
           'linear_fp8', 'linear_fp8_reference', 'quantize_fp8', 'quantize_fp8_reference', 'quantize_weight_fp8',
           'quantize_weight_fp8_reference', 'dequantize_fp8', 'dequantize_fp8_reference']
__version__ = '0.1.1+b200'

MODES = ('auto', 'fused', 'project')

# auto picks 'fused' while   queries * levels * points * 4 / (tokens * head_dim)  <  a + b / batch
# (upstream marearts_tinydeform/__init__.py:22-30, 39-46). 'fused' costs ~ batch * queries * samples * C row reads,
# 'project' ~ batch * tokens * C * H * D plus a fixed part that matters at batch 1.
# FUSED_LIMIT and FUSED_LIMIT_SM75 are upstream's tables (RTX 4090 / RTX 2080 Super); FUSED_LIMIT_SM100 is fitted
# to crossovers measured with this library on B200 (bench.py --sweep over upstream's query/batch grid, c4 and the
# c5 grid, 114 cases; profiles/auto_sweep_b200.md), used for compute capability 10.x. float32: the pick is within
# 10 % of the faster order in all 38 cases -- the fused order (a warp per row) wins up to about 300 queries per image
# at every batch, as the float32 projection runs three TF32 products per K step. float16 / bfloat16: 74 of 76; the
# fused order wins at 50-100 queries at batch 1-8 (RT-DETR shapes) and at batch 64 with 50 queries (c5), the project
# order above; no (a, b) also takes DINO batch 1 with 300 queries (fused 10.7 against 13.5 us), since the c5 shapes
# at batch 4-8 need the limit below its ratio.
FUSED_LIMIT = {torch.float32: (0.073, 0.032), torch.float16: (0.023, 0.031), torch.bfloat16: (0.023, 0.031)}
FUSED_LIMIT_SM75 = {torch.float32: (0.068, 0.0), torch.float16: (0.020, 0.0), torch.bfloat16: (0.132, 0.0)}
FUSED_LIMIT_SM100 = {torch.float32: (0.0775, 0.028), torch.float16: (0.024, -0.006), torch.bfloat16: (0.024, -0.006)}


@functools.lru_cache(maxsize=None)
def _limits(device_index):
    major, _ = torch.cuda.get_device_capability(device_index)
    if major == 10:
        return FUSED_LIMIT_SM100
    return FUSED_LIMIT if major >= 8 else FUSED_LIMIT_SM75


def choose_mode(memory, value_weight, sampling_locations):
    """The mode 'auto' runs: 'fused' for few queries per image, 'project' (project every token first) for many."""
    _, n_qry, n_head, n_lvl, n_pt, _ = sampling_locations.shape
    return _pick(memory, value_weight, n_qry, n_head, n_lvl, n_pt)


def _pick(memory, value_weight, n_qry, n_head, n_lvl, n_pt, limits=None):
    n_img, n_tok, _ = memory.shape
    head_dim = value_weight.shape[0] // n_head
    if limits is None:
        limits = _limits(memory.get_device()) if memory.is_cuda else FUSED_LIMIT
    a, b = limits.get(memory.dtype, limits[torch.float16])
    ratio = n_qry * n_lvl * n_pt * 4 / max(n_tok * head_dim, 1)
    return 'fused' if ratio < a + b / max(n_img, 1) else 'project'


def _outproj_in_epilogue(memory, value_weight, n_qry, n_head, output_weight):
    """Whether the project order would run output_proj in the sampler's cluster epilogue (td_set_output_proj_plan's
    automatic plan; the conditions of sample_outproj_kernel's 16-bit form)."""
    if output_weight is None or not memory.is_cuda or memory.dtype not in (torch.float16, torch.bfloat16):
        return False
    if _native.output_proj_plan() == _native.OUTPROJ_CHAINED:
        return False
    e = memory.element_size()
    hd = value_weight.shape[0]
    row = hd // n_head * e
    if hd * e != 512 or 8 % n_head or output_weight.shape[0] > 256:
        return False
    if row % 16 or row > 512 or (row // 16) & (row // 16 - 1):
        return False
    sms = torch.cuda.get_device_properties(memory.device).multi_processor_count
    return -(-memory.shape[0] * n_qry * n_head // 8) <= 3 * sms


def _pick_with_outproj(memory, value_weight, n_qry, n_head, n_lvl, n_pt, output_weight):
    """auto with output_proj: at batch 1, when the project order would fold output_proj into the sampler's
    epilogue, the project order (measured on B200, float16, C_out = 256: 1 x 20 queries 8.2 against 8.9 us fused
    + chained GEMM, 1 x 50 8.4 / 9.1, 1 x 100 8.7 / 9.5; at batch 2 and more the fused order with the chained GEMM
    is faster, 2 x 100 11.1 / 12.7); otherwise the operator's own pick."""
    if memory.shape[0] == 1 and _outproj_in_epilogue(memory, value_weight, n_qry, n_head, output_weight):
        return 'project'
    return _pick(memory, value_weight, n_qry, n_head, n_lvl, n_pt)


def ma_deform_attn(memory, value_weight, value_bias, spatial_shapes, level_start_index,
                   sampling_locations, attention_weights, mode='auto', value_padding_mask=None,
                   output_weight=None, output_bias=None):
    """value = memory @ value_weight.T + value_bias, then multi-scale deformable attention; [B, Q, H * D].

    Same arguments, shapes and result as ma_deform_attn_reference (grid_sample, bilinear, zero padding,
    align_corners=False). CUDA tensors (float32, float16, bfloat16, float64; float32 accumulation, float64 for
    float64) run the B200 kernels in the order `mode` names; CPU tensors run the reference.

    value_padding_mask (an addition; the upstream operator has none): bool [B, N], True = padded token. As
    Deformable-DETR's input_padding_mask, the projected value of a padded token is zeroed (its bias included)
    before sampling, so it contributes nothing.

    output_weight / output_bias (an addition): the decoder's output_proj (an nn.Linear [C_out, H * D]) applied to the
    result, so the call returns [B, Q, C_out]; on CUDA it runs as a tensor-core GEMM queued right behind the
    attention kernel (in the same library call in the project order), overlapping its start with it.
    """
    if mode not in MODES:
        raise ValueError(f'mode must be one of {MODES}, got {mode!r}')
    if output_bias is not None and output_weight is None:
        raise ValueError('output_bias needs output_weight')
    if not memory.is_cuda:
        out = ma_deform_attn_reference(memory, value_weight, value_bias, spatial_shapes, level_start_index,
                                       sampling_locations, attention_weights, value_padding_mask)
        return out if output_weight is None else torch.nn.functional.linear(out, output_weight, output_bias)
    _native.load()  # raises RuntimeError when the native library is missing: there is no fallback
    if mode == 'auto':
        _, n_qry, n_head, n_lvl, n_pt, _ = sampling_locations.shape
        mode = _pick_with_outproj(memory, value_weight, n_qry, n_head, n_lvl, n_pt, output_weight)
    if _wants_grad(memory, value_weight, value_bias, sampling_locations, attention_weights, output_weight,
                   output_bias):
        # training: the same forward kernels behind autograd Functions whose backward runs this library's
        # backward kernels (autograd.py), output_proj included
        _native.check_geometry(memory, spatial_shapes, level_start_index, sampling_locations, attention_weights)
        _native.check_projection(memory, value_weight, value_bias, sampling_locations.shape[2])
        out = ma_deform_attn_train(memory, value_weight, value_bias, spatial_shapes, level_start_index,
                                   sampling_locations, attention_weights, mode, value_padding_mask)
        if output_weight is None:
            return out
        _native.check_output_proj(output_weight, output_bias, out.shape[-1], out)
        return linear_train(out, output_weight, output_bias)
    if mode == 'project':
        # output_proj, if any, in the same library call
        return _native.project_forward(memory, value_weight, value_bias, spatial_shapes, level_start_index,
                                       sampling_locations, attention_weights, value_padding_mask, output_weight,
                                       output_bias)
    out = _native.fused_forward(memory, value_weight, value_bias, spatial_shapes, level_start_index,
                                sampling_locations, attention_weights, value_padding_mask)
    return out if output_weight is None else _native.linear(out, output_weight, output_bias)


def _in_dual_level():
    """Whether forward-mode differentiation is under way (without torch's own name for it: its tensors are asked)."""
    return getattr(forward_ad, '_current_level', 0) >= 0


def _wants_grad(*ts):
    """Whether a call of these operands is differentiated. Forward-mode tangents, which the kernels would drop without a
    word, are refused (the CPU path carries them)."""
    if _in_dual_level() and any(
            t is not None and t.is_cuda and forward_ad.unpack_dual(t).tangent is not None for t in ts):
        raise RuntimeError('no forward-mode derivative on CUDA: differentiate in reverse mode')
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts)


def pack_sampling_weights(offset_weight, offset_bias, attention_weight, attention_bias):
    """The layer's two query projections as one: sampling_offsets ([2 * H * L * P, Cq], rows (head, level, point,
    x/y)) stacked over attention_weights ([H * L * P, Cq], rows (head, level, point)), as the nn.Linear modules of
    Deformable-DETR's MSDeformAttn hold them. Pack once per model, not per call."""
    weight = torch.cat([offset_weight, attention_weight], 0)
    bias = None
    if offset_bias is not None or attention_bias is not None:
        zeros = offset_weight.new_zeros
        bias = torch.cat([offset_bias if offset_bias is not None else zeros(offset_weight.shape[0]),
                          attention_bias if attention_bias is not None else zeros(attention_weight.shape[0])])
    return weight, bias


def sampling_producer(query, reference_points, spatial_shapes, n_heads, n_points, sampling_weight, sampling_bias):
    """sampling_locations [B, Q, H, L, P, 2] and attention_weights [B, Q, H, L, P] from the query [B, Q, Cq] and
    reference points [B, Q, L, 2] (x, y) or reference boxes [B, Q, L, 4] (cx, cy, w, h), as
    sampling_producer_reference defines them. CUDA: the projection kernel, then the producer kernel."""
    if not query.is_cuda:
        return sampling_producer_reference(query, reference_points, spatial_shapes, n_heads, n_points,
                                           sampling_weight, sampling_bias)
    _native.load()
    L = spatial_shapes.shape[0]
    if sampling_weight.dim() != 2 or sampling_weight.shape[0] != 3 * n_heads * L * n_points:
        raise RuntimeError('sampling_weight must be [3 * H * L * P, Cq]: the offset rows, then the attention rows')
    if _wants_grad(query, reference_points, sampling_weight, sampling_bias):
        # training: the same kernels behind autograd Functions whose backward runs this library's kernels (the
        # producer's backward, then the query projection's gradient GEMMs)
        return producer_train(query, reference_points, spatial_shapes, n_heads, n_points, sampling_weight,
                              sampling_bias)
    proj = _native.linear(query, sampling_weight, sampling_bias)
    return _native.sampling_producer(proj, reference_points, spatial_shapes, n_heads, n_points)


def deform_attn_layer(query, reference_points, memory, spatial_shapes, level_start_index, n_heads, n_points,
                      sampling_weight, sampling_bias, value_weight, value_bias, output_weight=None, output_bias=None,
                      value_padding_mask=None, mode='auto', residual=None, norm_weight=None, norm_bias=None,
                      norm_eps=1e-5):
    """One multi-scale deformable attention layer (the forward of Deformable-DETR's MSDeformAttn, whose core is
    ma_deform_attn): [B, Q, H * D], or [B, Q, C_out] with output_weight.

    query [B, Q, Cq]; reference_points [B, Q, L, 2] or [B, Q, L, 4]; memory [B, N, C] (the value input);
    sampling_weight / sampling_bias: pack_sampling_weights of the offset and attention-weight projections;
    value_weight / value_bias: value_proj; output_weight / output_bias: output_proj (optional);
    value_padding_mask: bool [B, N], True = padded token. Same result as deform_attn_layer_reference.

    norm_weight / norm_bias / norm_eps and residual (the layer's output shape): the decoder layer's norm behind the
    attention, layer_norm(output, norm_weight, norm_bias, residual, norm_eps), as the call's last kernel.

    CUDA, mode 'project' (or 'auto' choosing it): three kernels in one library call (query projection, value
    projection, and the sampler computing the softmax and locations in its prologue), plus the output projection.
    Mode 'fused': query projection, producer kernel, fused gather-then-project kernel.
    """
    if mode not in MODES:
        raise ValueError(f'mode must be one of {MODES}, got {mode!r}')
    if output_bias is not None and output_weight is None:
        raise ValueError('output_bias needs output_weight')
    if norm_weight is None and (norm_bias is not None or residual is not None):
        raise ValueError('norm_bias and residual need norm_weight')
    if norm_weight is not None:
        out = deform_attn_layer(query, reference_points, memory, spatial_shapes, level_start_index, n_heads, n_points,
                                sampling_weight, sampling_bias, value_weight, value_bias, output_weight, output_bias,
                                value_padding_mask, mode)
        return layer_norm(out, norm_weight, norm_bias, residual, norm_eps)
    if not memory.is_cuda:
        return deform_attn_layer_reference(query, reference_points, memory, spatial_shapes, level_start_index,
                                           n_heads, n_points, sampling_weight, sampling_bias, value_weight,
                                           value_bias, output_weight, output_bias, value_padding_mask)
    _native.load()
    if mode == 'auto':
        mode = _pick_with_outproj(memory, value_weight, query.shape[1], n_heads, spatial_shapes.shape[0], n_points,
                                  output_weight)
    if _wants_grad(query, reference_points, memory, sampling_weight, sampling_bias, value_weight, value_bias,
                   output_weight, output_bias):
        # training: the producer and the attention behind autograd Functions on this library's kernels
        loc, attn = sampling_producer(query, reference_points, spatial_shapes, n_heads, n_points, sampling_weight,
                                      sampling_bias)
        return ma_deform_attn(memory, value_weight, value_bias, spatial_shapes, level_start_index, loc, attn,
                              mode=mode, value_padding_mask=value_padding_mask, output_weight=output_weight,
                              output_bias=output_bias)
    return _native.layer_forward(query, reference_points, memory, spatial_shapes, level_start_index, n_heads,
                                 n_points, sampling_weight, sampling_bias, value_weight, value_bias, output_weight,
                                 output_bias, value_padding_mask, order=mode)


def attention(query, key, value, key_padding_mask=None, attn_mask=None, causal=False, scale=None):
    """Softmax attention: the self attention among a decoder's queries, or any attention over N keys; [B, Q, H * D].

    query [B, Q, H, D]; key, value [B, N, Hk, D], H a multiple of Hk (query head h uses key head h // (H // Hk)),
    D <= 128; float32, float16, bfloat16 or float64. Views of a packed projection are read in place.
    key_padding_mask: bool [B, N], True = no key there (its rows may hold anything). attn_mask: bool [Q, N] or
    [B or 1, H or 1, Q, N], True = query i may not use key j (DINO's denoising mask); what a blocked pair's key and
    value hold must still be finite. causal: query i uses the keys up to i + N - Q. A query left without any key gets
    zeros, and passes no gradient. scale: positive, 1 / sqrt(D) unless given. An infinite key that makes a score minus
    infinity has no probability there; an infinite value or any NaN makes what uses it infinite or NaN.

    CUDA tensors run this library's kernels, forward and backward (no probabilities are kept; sums run in float32,
    float64 for float64; gradients are the same bits every time); CPU tensors run attention_reference. The backward
    can be captured in a CUDA graph with the forward; as with every autograd backward under capture, no graph of the
    same leaves that was built outside the capture may be alive then.
    """
    if scale is None:
        scale = query.shape[-1] ** -0.5 if query.dim() == 4 and query.shape[-1] > 0 else 1.0
    _native.check_attention(query, key, value, key_padding_mask, attn_mask, scale)
    if not query.is_cuda:
        return attention_reference(query, key, value, key_padding_mask, attn_mask, causal, scale)
    _native.load()
    if _wants_grad(query, key, value):
        return AttentionFunction.apply(query, key, value, key_padding_mask, attn_mask, bool(causal), float(scale))
    return _native.attention_forward(query, key, value, key_padding_mask, attn_mask, bool(causal), float(scale))


def layer_norm(x, weight, bias=None, residual=None, eps=1e-5):
    """Layer norm of x + residual over the last dimension (up to 8192 wide), in x's shape and dtype.

    weight, bias and residual have x's dtype and device. The sum is not rounded before the norm, and the statistics are
    float32 (float64 for float64). CUDA tensors run this library's kernels, forward and backward (the column sums of the
    weight's and bias's gradients in a fixed order); CPU tensors run layer_norm_reference.
    """
    _native.check_layer_norm(x, weight, bias, residual, eps)
    if not x.is_cuda:
        return layer_norm_reference(x, weight, bias, residual, eps)
    _native.load()
    if _wants_grad(x, weight, bias, residual):
        return LayerNormFunction.apply(x, weight, bias, residual, float(eps))
    return _native.layer_norm_forward(x, weight, bias, residual, float(eps))[0]


def rms_norm(x, weight, residual=None, eps=1e-6, return_sum=False, quantize=False):
    """Root-mean-square norm of s = x + residual over the last dimension (up to 8192 wide): s / sqrt(mean(s^2) + eps)
    * weight, in x's shape and dtype.

    weight and residual have x's dtype and device. s is not rounded before the norm, and the mean is float32 (float64
    for float64), so squares have to stay in its range. return_sum: the pair (result, s), s being what the next layer
    adds to. quantize: the result in 8 bits, as a pair (data, scale) like quantize_fp8's, rounded once; for calls without
    gradients, not for float64. CUDA tensors run this library's kernels, forward and backward (the weight's gradient
    summed in a fixed order); CPU tensors run rms_norm_reference.
    """
    _native.check_rms_norm(x, weight, residual, eps, quantize)
    grad = _wants_grad(x, weight, residual)
    if grad and quantize:
        raise RuntimeError('an 8-bit result has no gradient: leave quantize off, or run under torch.no_grad()')
    if not x.is_cuda:
        return rms_norm_reference(x, weight, residual, eps, return_sum, quantize)
    _native.load()
    if grad:
        return RmsNormFunction.apply(x, weight, residual, float(eps), bool(return_sum))
    y, total, _ = _native.rms_norm_forward(x, weight, residual, float(eps), return_sum, quantize)
    return (y, total) if return_sum else y


def quantize_fp8(x):
    """x [..., K] in 8 bits (e4m3), a scale for each 128 values along the last dimension: the pair (data, scale) of
    float8_e4m3fn [..., K] and float32 [..., ceil(K / 128)]; x is about data * scale.

    x: float32, float16 or bfloat16, up to 65536 wide (and 2^31 - 256 rows). Scales are powers of two, the smallest that
    bring a block's largest finite magnitude to at most 448 (e4m3's largest); values are rounded to nearest, ties to
    even; infinities and NaN become NaN. data's rows start 16 bytes apart or a multiple of that, so it is a view where K
    is not one. What is in 8 bits has no gradient, so an x that requires grad is refused (linear_fp8 takes it as it is).
    """
    _native.check_fp8_source(x)
    if _wants_grad(x):
        raise RuntimeError('what is in 8 bits has no gradient: detach x, or run under torch.no_grad()')
    x = x.detach()
    return _native.fp8_quantize(x) if x.is_cuda else quantize_fp8_reference(x)


def quantize_weight_fp8(weight):
    """A weight [N, K] in 8 bits as linear_fp8 takes it, to be laid out once: (data, scale) as quantize_fp8's, with a
    scale for each block of 128 x 128, float32 [ceil(N / 128), ceil(K / 128)]. The pair is the weight's values alone, a
    parameter's too: no gradient goes back through it (training takes the weight itself)."""
    _native.check_fp8_source(weight, 'weight')
    if weight.dim() != 2 or not 1 <= weight.shape[0] <= _native.MAX_FP8_WIDTH:
        raise RuntimeError(f'weight must be [N, K], both between 1 and {_native.MAX_FP8_WIDTH}')
    weight = weight.detach()
    return _native.fp8_quantize(weight, tiles=True) if weight.is_cuda else quantize_weight_fp8_reference(weight)


def dequantize_fp8(data, scale, dtype):
    """data * scale in `dtype` (float32, float16 or bfloat16): what quantize_fp8's pair, or quantize_weight_fp8's, stands
    for. float32 holds the values of this package's own pairs exactly, bfloat16 those from 2^-126 on (below, its numbers
    are further apart than theirs). Scales that require grad are refused: a pair has no gradient."""
    tiles = isinstance(data, torch.Tensor) and isinstance(scale, torch.Tensor) and data.dim() == 2 and \
        scale.dim() == 2 and scale.shape[0] != data.shape[0]
    _native.check_fp8_pair((data, scale), 'the input', tiles)
    if dtype not in (torch.float32, torch.float16, torch.bfloat16):
        raise RuntimeError('dtype must be float32, float16 or bfloat16')
    if _wants_grad(data, scale):
        raise RuntimeError('what is in 8 bits has no gradient: detach the scales, or run under torch.no_grad()')
    if not data.is_cuda:
        return dequantize_fp8_reference(data, scale, dtype)
    return _native.fp8_dequantize(data, scale, dtype, tiles)


def _tensors(operand):
    """An operand's tensors: itself, or a pair's."""
    if isinstance(operand, torch.Tensor):
        return (operand,)
    return [t for t in operand if isinstance(t, torch.Tensor)] if isinstance(operand, (tuple, list)) else ()


def linear_fp8(x, weight, bias=None, activation=None, quantize=False, dtype=None):
    """activation(x @ weight.T + bias) with both operands in 8 bits (e4m3), over the last dimension of x; [..., N].

    x: float32, float16 or bfloat16 [..., K] (quantised by the call as quantize_fp8 does), or a pair (data, scale).
    weight: a pair from quantize_weight_fp8 (or any other such pair: scales may be any float32 numbers, as long as the
    product of a scale of x and one of weight is one too), or a floating [N, K] of x's dtype, laid out by the call.
    bias: [N], floating. activation: None, 'relu', 'gelu' (with erf) or 'silu'. dtype: the result's, x's unless given
    (needed where x is a pair). quantize: the result in 8 bits instead, a pair that the next product takes. The
    products of a block are summed in float32, then scaled, and the result is rounded once.

    Training: where x (floating), weight (floating) or bias requires grad, the backward runs too, with the input kept
    for it only in 8 bits; no activation, quantize or other dtype then. With Q the roundings to 8 bits, whose own
    derivative counts as 1: grad_x = Q(g) Q(weight), grad_weight = Q(g)^T Q(Q(x)), the last two in blocks of 128 rows,
    grad_bias = the sum of g. Sums are taken in a fixed order. CUDA tensors run this library's kernels; CPU tensors
    linear_fp8_reference. The backward can be captured in a CUDA graph with the forward; as with every autograd backward
    under capture, no graph of the same leaves that was built outside the capture may be alive then.
    """
    grad = (torch.is_grad_enabled() or _in_dual_level()) and \
        _wants_grad(*_tensors(x), *_tensors(weight), bias)
    dtype = _native.check_linear_fp8(x, weight, bias, activation, quantize, dtype, grad)
    cuda = (x if isinstance(x, torch.Tensor) else x[0]).is_cuda
    if cuda:
        _native.load()
    if grad:
        return LinearFp8Function.apply(x, weight, bias)
    if isinstance(weight, torch.Tensor):
        weight = quantize_weight_fp8(weight)
    if cuda:
        return _native.linear_fp8_forward(x, weight, bias, activation, quantize, dtype)
    if isinstance(x, torch.Tensor):
        x = quantize_fp8_reference(x)
    return linear_fp8_reference(x, weight, bias, activation, quantize, dtype)
