"""The plain-PyTorch definition of the operator: project every memory token, then bilinear-sample per level.

This is the public ``ma_deform_attn_reference`` of the drop-in API (upstream
``marearts_tinydeform/reference.py:13-40``). It defines what ``ma_deform_attn`` returns: ``nn.Linear`` on every
memory token, then ``F.grid_sample`` with bilinear interpolation, zero padding and ``align_corners=False`` on each
level, then the attention-weighted sum over levels x points. It runs on CPU and GPU in any float dtype and supports
autograd (the CUDA path has its own backward kernel).

CPU tensors passed to ``ma_deform_attn`` come here, exactly as upstream ``marearts_tinydeform/__init__.py:62-64``
routes them. CUDA tensors never do: the CUDA path raises when its native library is missing.
"""

import torch
import torch.nn.functional as F


def ma_deform_attn_reference(memory, value_weight, value_bias, spatial_shapes, level_start_index,
                             sampling_locations, attention_weights, value_padding_mask=None):
    """value = memory @ value_weight.T + value_bias, then multi-scale deformable attention.

    memory              [B, N, C]
    value_weight        [H * D, C]      (an nn.Linear weight)
    value_bias          [H * D] or None
    spatial_shapes      [L, 2] int64    (height, width) of each level; tokens are laid out level after level
    level_start_index   [L] int64       first token of each level
    sampling_locations  [B, Q, H, L, P, 2]  (x, y) normalised to [0, 1]
    attention_weights   [B, Q, H, L, P]     already normalised (softmax over L * P)
    value_padding_mask  [B, N] bool or None: True zeroes that token's projected value (Deformable-DETR's
                        input_padding_mask; an addition to the upstream signature, which has no mask)
    returns             [B, Q, H * D]
    """
    n_img, n_tok, _ = memory.shape
    _, n_qry, n_head, n_lvl, n_pt, _ = sampling_locations.shape
    value = F.linear(memory, value_weight, value_bias)                 # [B, N, H*D]
    if value_padding_mask is not None:
        value = value.masked_fill(value_padding_mask.to(torch.bool)[..., None], 0)
    head_dim = value.shape[-1] // n_head
    # grid_sample wants (x, y) in [-1, 1]; one image per (batch, head) pair, D channels each
    grid = sampling_locations.mul(2).sub(1).permute(0, 2, 1, 3, 4, 5)  # [B, H, Q, L, P, 2]
    grid = grid.reshape(n_img * n_head, n_qry, n_lvl, n_pt, 2)
    per_head = value.view(n_img, n_tok, n_head, head_dim).permute(0, 2, 3, 1)  # [B, H, D, N]
    per_head = per_head.reshape(n_img * n_head, head_dim, n_tok)
    sampled = []
    for lvl in range(n_lvl):
        # level geometry is read on the host, like any grid_sample caller
        height, width = int(spatial_shapes[lvl, 0]), int(spatial_shapes[lvl, 1])
        first = int(level_start_index[lvl])
        image = per_head[:, :, first:first + height * width].reshape(n_img * n_head, head_dim, height, width)
        sampled.append(F.grid_sample(image, grid[:, :, lvl], mode='bilinear', padding_mode='zeros',
                                     align_corners=False))             # [B*H, D, Q, P]
    stacked = torch.cat(sampled, dim=-1)                               # [B*H, D, Q, L*P]
    weights = attention_weights.permute(0, 2, 1, 3, 4).reshape(n_img * n_head, 1, n_qry, n_lvl * n_pt)
    out = (stacked * weights).sum(-1)                                  # [B*H, D, Q]
    return out.view(n_img, n_head * head_dim, n_qry).transpose(1, 2).contiguous()


def sampling_producer_reference(query, reference_points, spatial_shapes, n_heads, n_points, sampling_weight,
                                sampling_bias):
    """sampling_locations [B, Q, H, L, P, 2] and attention_weights [B, Q, H, L, P] of the multi-scale deformable
    attention layer (Deformable-DETR's MSDeformAttn, RT-DETR's decoder). sampling_weight = [W_offsets; W_attention]
    ([3 * H * L * P, Cq]; the offset rows ordered (head, level, point, x/y), the attention rows (head, level, point)),
    sampling_bias likewise. The logits are normalised by a softmax over the L * P points of each head, and the
    offsets move the reference points: ref + offset / (w_l, h_l) for reference_points [B, Q, L, 2],
    ref.xy + offset / P * ref.wh * 0.5 for reference boxes [B, Q, L, 4]. The upstream operator takes both results as
    inputs and has no producer."""
    B, Q, _ = query.shape
    L = spatial_shapes.shape[0]
    H, P = n_heads, n_points
    proj = F.linear(query, sampling_weight, sampling_bias)
    offsets = proj[..., :2 * H * L * P].reshape(B, Q, H, L, P, 2)
    logits = proj[..., 2 * H * L * P:].reshape(B, Q, H, L * P)
    attention = logits.softmax(-1).view(B, Q, H, L, P)
    if reference_points.shape[-1] == 2:
        norm = torch.stack([spatial_shapes[:, 1], spatial_shapes[:, 0]], -1).to(query.dtype)   # (w, h) per level
        loc = reference_points[:, :, None, :, None, :] + offsets / norm[None, None, None, :, None, :]
    else:
        loc = (reference_points[:, :, None, :, None, :2]
               + offsets / P * reference_points[:, :, None, :, None, 2:] * 0.5)
    return loc, attention


def deform_attn_layer_reference(query, reference_points, memory, spatial_shapes, level_start_index, n_heads,
                                n_points, sampling_weight, sampling_bias, value_weight, value_bias,
                                output_weight=None, output_bias=None, value_padding_mask=None):
    """One deformable attention layer with torch operators: the producer above, ma_deform_attn_reference, and the
    optional output projection."""
    loc, attention = sampling_producer_reference(query, reference_points, spatial_shapes, n_heads, n_points,
                                                 sampling_weight, sampling_bias)
    out = ma_deform_attn_reference(memory, value_weight, value_bias, spatial_shapes, level_start_index, loc,
                                   attention, value_padding_mask)
    return out if output_weight is None else F.linear(out, output_weight, output_bias)


def attention_reference(query, key, value, key_padding_mask=None, attn_mask=None, causal=False, scale=None):
    """Softmax attention with torch operators; the definition ``attention`` follows (see there for the arguments).
    Sums and probabilities are float32 for float16 / bfloat16 inputs, and the result is rounded once."""
    B, Q, H, D = query.shape
    N, Hk = key.shape[1:3]
    acc = torch.float32 if query.dtype in (torch.float16, torch.bfloat16) else query.dtype
    q, k, v = query.to(acc), key.to(acc), value.to(acc)
    if key_padding_mask is not None:  # a padded key is not there at all, whatever its rows hold
        gone = key_padding_mask.to(torch.bool)[:, :, None, None]
        k, v = k.masked_fill(gone, 0), v.masked_fill(gone, 0)
    if Hk != H:
        k, v = k.repeat_interleave(H // Hk, 2), v.repeat_interleave(H // Hk, 2)
    scores = torch.einsum('bihd,bjhd->bhij', q, k) * (D ** -0.5 if scale is None else scale)
    blocked = torch.zeros((1, 1, Q, N), dtype=torch.bool, device=query.device)
    if key_padding_mask is not None:
        blocked = blocked | key_padding_mask.to(torch.bool)[:, None, None, :]
    if attn_mask is not None:
        blocked = blocked | attn_mask.to(torch.bool)
    if causal:
        blocked = blocked | torch.ones((Q, N), dtype=torch.bool, device=query.device).triu(N - Q + 1)
    # rows without an open key: softmax over finite scores, then zeroed, so that their gradients are zeros too
    empty = blocked.all(-1, keepdim=True)
    scores = scores.masked_fill(blocked & ~empty, float('-inf'))
    probs = scores.softmax(-1).masked_fill(empty | blocked, 0)
    return torch.einsum('bhij,bjhd->bihd', probs, v).reshape(B, Q, H * D).to(query.dtype)


def layer_norm_reference(x, weight, bias=None, residual=None, eps=1e-5):
    """Layer norm over the last dimension with the residual added inside, with torch operators; the definition
    ``layer_norm`` follows. float32 arithmetic for float16 / bfloat16 inputs, rounded once."""
    acc = torch.float32 if x.dtype in (torch.float16, torch.bfloat16) else x.dtype
    s = x.to(acc) if residual is None else x.to(acc) + residual.to(acc)
    return F.layer_norm(s, s.shape[-1:], weight.to(acc), None if bias is None else bias.to(acc), eps).to(x.dtype)


def rms_norm_reference(x, weight, residual=None, eps=1e-6, return_sum=False, quantize=False):
    """Root-mean-square norm over the last dimension with the residual added inside, with torch operators; the
    definition ``rms_norm`` follows. float32 arithmetic for float16 / bfloat16 inputs; each result is rounded once."""
    acc = torch.float32 if x.dtype in (torch.float16, torch.bfloat16) else x.dtype
    s = x.to(acc) if residual is None else x.to(acc) + residual.to(acc)
    y = s * torch.rsqrt(s.square().mean(-1, keepdim=True) + eps) * weight.to(acc)
    y = quantize_fp8_reference(y) if quantize else y.to(x.dtype)
    return (y, s.to(x.dtype)) if return_sum else y


def _fp8_blocks(x, rows):
    """x [..., R, C] in float32, zeros behind its edges, as [..., R / rows, rows, C / 128, 128]."""
    R, C = x.shape[-2:]
    p = F.pad(x.float(), (0, -C % 128, 0, -R % rows))
    return p.view(*p.shape[:-2], p.shape[-2] // rows, rows, p.shape[-1] // 128, 128)


def _fp8_quantize(x, rows):
    """x [R, C] in blocks of rows x 128: e4m3 data [R, C], scales [R / rows, C / 128] (rounded up)."""
    R, C = x.shape
    p = _fp8_blocks(x, rows)
    top = p.abs().masked_fill(~p.isfinite(), 0).amax((1, 3))
    mantissa, exponent = torch.frexp(top)  # top = mantissa * 2^exponent, mantissa in [0.5, 1); 448 = 0.875 * 2^9
    e = (exponent - 9 + (mantissa > 0.875).int()).clamp(min=-126).masked_fill(top == 0, -126)
    scale = ((e + 127) << 23).int().view(torch.float32)
    q = p * ((127 - e) << 23).int().view(torch.float32)[:, None, :, None]
    q = q.masked_fill(~q.isfinite(), float('nan')).to(torch.float8_e4m3fn)
    return q.view(p.shape[0] * rows, p.shape[2] * 128)[:R, :C].contiguous(), scale


def quantize_fp8_reference(x):
    """x [..., K] in 8 bits with torch operators; the definition ``quantize_fp8`` follows."""
    rows = x.numel() // x.shape[-1]
    q, scale = _fp8_quantize(x.reshape(rows, x.shape[-1]), 1)
    return q.view(x.shape), scale.view(*x.shape[:-1], scale.shape[1])


def quantize_weight_fp8_reference(weight):
    """weight [N, K] in 8 bits with torch operators; the definition ``quantize_weight_fp8`` follows."""
    return _fp8_quantize(weight, 128)


def dequantize_fp8_reference(data, scale, dtype):
    """What 8-bit data stands for, with torch operators; the definition ``dequantize_fp8`` follows."""
    K = data.shape[-1]
    per_row = scale.repeat_interleave(128, -1)[..., :K]
    if scale.shape[:-1] != data.shape[:-1]:
        per_row = per_row.repeat_interleave(128, 0)[:data.shape[0]]
    return (data.float() * per_row).to(dtype)


def linear_fp8_reference(x, weight, bias=None, activation=None, quantize=False, dtype=None):
    """The product of two 8-bit operands (pairs) with torch operators; the definition ``linear_fp8`` follows."""
    y = torch.matmul(dequantize_fp8_reference(*x, torch.float32), dequantize_fp8_reference(*weight, torch.float32).t())
    if bias is not None:
        y = y + bias.float()
    if activation == 'relu':
        y = F.relu(y)
    elif activation is not None:  # in 64 bits: float32 loses the lower tails' digits
        d = y.double()
        y = (0.5 * d * torch.special.erfc(d * -0.5 ** 0.5) if activation == 'gelu' else F.silu(d)).float()
    return quantize_fp8_reference(y) if quantize else y.to(dtype)


def linear_fp8_backward_reference(grad_out, x8, weight, want_x, want_w, want_b):
    """The gradients of ``linear_fp8`` with torch operators: grad_x from the weight, grad_weight from the input's 8-bit
    copy."""
    g = grad_out.reshape(-1, grad_out.shape[-1])
    grad_x = grad_w = grad_b = None
    if want_x:
        w8 = dequantize_fp8_reference(*_fp8_quantize(weight, 128), torch.float32)
        g8 = dequantize_fp8_reference(*_fp8_quantize(g, 1), torch.float32)
        grad_x = torch.matmul(g8, w8).view(*grad_out.shape[:-1], weight.shape[1]).to(grad_out.dtype)
    if want_w:
        x = dequantize_fp8_reference(*x8, torch.float32).reshape(-1, x8[0].shape[-1])
        cols = [dequantize_fp8_reference(*_fp8_quantize(t.t(), 1), torch.float32) for t in (g, x)]
        grad_w = torch.matmul(cols[0], cols[1].t()).to(grad_out.dtype)
    if want_b:
        grad_b = g.float().sum(0).to(grad_out.dtype)
    return grad_x, grad_w, grad_b
