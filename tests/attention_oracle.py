"""softmax attention and layer norm in float64, with elementwise error bounds for the kernels' results.

The bounds count roundings. u is half a step of the result's type (finfo.eps / 2), e half a step of the type sums are
held in. Attention, forward: the scores are sums of D products and c = scale * log2(e), their error at most
d = (D + 8) e sum|q||k| scale, which is a relative error of P; exp2 and log2 add at most 16 e; P is rounded once to a
16-bit type for the product (u), the product's sums add g(n) = (n + 64) 2 e of the sum of magnitudes, and the result
is rounded once (u). Backward: dS adds the rounding of dS (u), the result's own bound in delta and the
sums of D products behind dP and delta ((D + 8) e). float16 also flushes what falls under its smallest step: 2^-25 of
a P whose row maximum is at least 1, and of a dS scaled so that 2 D max|do| max|v| is at least 2^14."""

import math

import torch

U = {torch.float64: 2.0 ** -53, torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
# what a result below the smallest normal number may lose
TINY = {torch.float64: 0.0, torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -133}


def blocked_pairs(B, Q, N, key_padding_mask, attn_mask, causal, device):
    blocked = torch.zeros((B, 1, Q, N), dtype=torch.bool, device=device)
    if key_padding_mask is not None:
        blocked = blocked | key_padding_mask.bool()[:, None, None, :]
    if attn_mask is not None:
        blocked = blocked | attn_mask.bool()
    if causal:
        i, j = torch.arange(Q, device=device)[:, None], torch.arange(N, device=device)[None, :]
        blocked = blocked | (j > i + (N - Q))
    return blocked


def attention_exact(q, k, v, key_padding_mask=None, attn_mask=None, causal=False, scale=None, grad=None):
    """[(value, bound), ...] of out and, with grad, of the gradients of q, k and v."""
    dtype = q.dtype
    B, Q, H, D = q.shape
    N, Hk = k.shape[1:3]
    G = H // Hk
    scale = D ** -0.5 if scale is None else scale
    u, e, tiny = U[dtype], U[torch.float64 if dtype == torch.float64 else torch.float32], TINY[dtype]
    half = u if dtype in (torch.float16, torch.bfloat16) else 0.0  # the rounding of P and dS
    blocked = blocked_pairs(B, Q, N, key_padding_mask, attn_mask, causal, q.device)
    q, k, v = q.double().transpose(1, 2), k.double().transpose(1, 2), v.double().transpose(1, 2)
    if key_padding_mask is not None:
        gone = key_padding_mask.bool()[:, None, :, None]
        k, v = k.masked_fill(gone, 0), v.masked_fill(gone, 0)
    kh, vh = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
    s = (q @ kh.transpose(2, 3) * scale).masked_fill(blocked, -math.inf)
    top = s.amax(3, keepdim=True) if N else s.new_zeros(B, H, Q, 1)
    p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(3, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    out = p @ vh
    mag = (q.abs() @ kh.abs().transpose(2, 3)) * scale
    d = (D + 8) * e * (mag.amax().item() if mag.numel() else 0.0) * 2 + 16 * e  # in P and in the row's sum
    flush = 2.0 ** -25 if dtype == torch.float16 else 0.0

    def rows(t):
        return t.transpose(1, 2)

    bound = u * out.abs() + (half + 2 * d + (N + 64) * 2 * e) * (p @ vh.abs()) + \
        flush * vh.abs().sum(2, keepdim=True) + tiny
    found = [(rows(out).reshape(B, Q, H * D), rows(bound).reshape(B, Q, H * D) * 1.01)]
    if grad is None:
        return found
    do = grad.double().view(B, Q, H, D).transpose(1, 2)
    dp, delta = do @ vh.transpose(2, 3), (do * out).sum(3, keepdim=True)
    ds = p * (dp - delta)
    mo = (do.abs() * out.abs()).sum(3, keepdim=True)
    ds_err = p * ((half + 3 * d) * (dp - delta).abs() + (do.abs() * bound).sum(3, keepdim=True)
                  + (D + 8) * e * (do.abs() @ vh.abs().transpose(2, 3) + mo))
    if dtype == torch.float16:
        ds_err = ds_err + 2.0 ** -39 * 2 * D * do.abs().amax() * vh.abs().amax()

    def per_key_head(t):
        return t.view(B, Hk, G, N, D).sum(2)

    dq, dk, dv = ds @ kh * scale, per_key_head(ds.transpose(2, 3) @ q) * scale, per_key_head(p.transpose(2, 3) @ do)
    dq_b = u * dq.abs() + (ds_err @ kh.abs() + (N + 64) * 2 * e * (ds.abs() @ kh.abs())) * scale + tiny
    dk_b = u * dk.abs() + tiny + per_key_head(
        ds_err.transpose(2, 3) @ q.abs() + (G * Q + 64) * 2 * e * (ds.abs().transpose(2, 3) @ q.abs())) * scale
    dv_b = u * dv.abs() + tiny + per_key_head(
        (half + 2 * d + (G * Q + 64) * 2 * e) * (p.transpose(2, 3) @ do.abs())
        + flush * do.abs().sum(2, keepdim=True))
    return found + [(rows(x), rows(b) * 1.01) for x, b in ((dq, dq_b), (dk, dk_b), (dv, dv_b))]


def layer_norm_exact(x, weight, bias=None, residual=None, eps=1e-5, grad=None):
    """[(value, bound), ...] of y and, with grad, of the gradients of x, weight and bias. The sums of C terms and the
    statistics are good to g = (C + 32) e of the terms' magnitudes, the column sums of R rows to (R + 32) e."""
    dtype, C = x.dtype, x.shape[-1]
    u, e, tiny = U[dtype], U[torch.float64 if dtype == torch.float64 else torch.float32], TINY[dtype]
    s = x.double() if residual is None else x.double() + residual.double()
    w = weight.double()
    mean = s.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt(((s - mean) ** 2).mean(-1, keepdim=True) + eps)
    z = (s - mean) * rstd
    g = (C + 32) * e
    z_err = g * (s.abs().mean(-1, keepdim=True) * rstd + z.abs()) + 4 * e * s.abs() * rstd
    y = z * w + (0 if bias is None else bias.double())
    found = [(y, (u + 4 * e) * y.abs() + z_err * w.abs() + 4 * e * (z * w).abs() + tiny)]
    if grad is None:
        return found
    dy = grad.double()
    h = dy * w
    m1, m2 = h.mean(-1, keepdim=True), (h * z).mean(-1, keepdim=True)
    dx = rstd * (h - m1 - z * m2)
    a1, a2 = h.abs().mean(-1, keepdim=True), (h * z).abs().mean(-1, keepdim=True)
    rel = g * (1 + (s.abs().mean(-1, keepdim=True) * rstd))  # of rstd and the sums
    dx_b = u * dx.abs() + tiny + rstd * (4 * rel * (h.abs() + a1 + z.abs() * a2)
                                        + z_err * a2 + z.abs() * (h.abs() * z_err).mean(-1, keepdim=True))
    rows = dy.reshape(-1, C)
    zr, ze = z.reshape(-1, C), z_err.reshape(-1, C)
    dw, db = (rows * zr).sum(0), rows.sum(0)
    r = (rows.shape[0] + 32) * e
    dw_b = u * dw.abs() + r * (rows * zr).abs().sum(0) + (rows.abs() * (ze + 4 * e * zr.abs())).sum(0) + tiny
    db_b = u * db.abs() + r * rows.abs().sum(0) + tiny
    return found + [(dx, dx_b), (dw, dw_b), (db, db_b)]


def check(got, exact, what):
    """Every element within its bound; NaN nowhere."""
    value, bound = exact
    assert tuple(got.shape) == tuple(value.shape), f'{what}: shape {tuple(got.shape)}'
    diff = (got.double() - value).abs()
    bad = ~(diff <= bound)
    if bad.any():
        at = int((torch.where(torch.isnan(diff), math.inf, diff) / bound.clamp_min(1e-300)).flatten().argmax())
        raise AssertionError(f'{what}: {int(bad.sum())} of {bad.numel()} outside their bound; at {at} got '
                             f'{got.flatten()[at].item()}, want {value.flatten()[at].item()} '
                             f'+- {bound.flatten()[at].item()}')
