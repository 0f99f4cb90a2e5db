"""8-bit blocks, root-mean-square norm and 8-bit products in float64, with elementwise error bounds.

u is half a step of the result's type (finfo.eps / 2), e half a step of float32 (of float64 for float64). A value
rounded to 8 bits is off by at most 2^-4 of itself, or half the smallest step, 2^-10 times the block's scale. A sum of n
products on the tensor cores is good to (n + 64) 2 e of the products' magnitudes (as the attention's, whose sums they
cut instead of rounding); the products themselves are exact."""

import torch

from attention_oracle import TINY, U

E4M3 = torch.float8_e4m3fn


def two_to(e):
    """2^e in float64 for a tensor of integers."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def quantized(x, rows, cols):
    """x [R, C] in blocks of rows x cols: (the stored numbers, the scales [R / rows, C / cols]), both in float64."""
    R, C = x.shape
    x = x.double()
    q = torch.empty_like(x)
    scale = torch.empty((-(-R // rows), -(-C // cols)), dtype=torch.float64, device=x.device)
    p = torch.nn.functional.pad(x, (0, -C % cols, 0, -R % rows)).view(scale.shape[0], rows, scale.shape[1], cols)
    top = torch.where(p.isfinite(), p.abs(), 0.0).amax((1, 3))
    scale.fill_(2.0 ** -126)
    for e in range(-126, 121):  # the first power of two that fits
        scale = torch.where((top > 448 * scale) & (top > 448 * 2.0 ** (e - 1)), 2.0 ** e, scale)
    v = p / scale[:, None, :, None]
    step = two_to((torch.frexp(v.nan_to_num(0, 0, 0))[1] - 1).clamp_min(-6) - 3)
    q = torch.where(v.isfinite(), torch.round(v / step) * step, float('nan'))
    return q.view(p.shape[0] * rows, -1)[:R, :C], scale


def worth(q, scale, rows, cols):
    """The values that stored numbers stand for, in float64."""
    s = scale.double().repeat_interleave(rows, 0)[:q.shape[0]].repeat_interleave(cols, 1)[:, :q.shape[1]]
    return q.double() * s


def through(x, rows, cols):
    return worth(*quantized(x, rows, cols), rows, cols)


def check_quantized(pair, exact, what):
    """A pair in 1 x 128 blocks against the value and bound of what was rounded to it: each scale a power of two that
    the block's largest value calls for, each number within half a step."""
    data, scale = (t.double().reshape(-1, t.shape[-1]) for t in pair)
    value, bound = (t.reshape(data.shape) for t in exact)
    C = data.shape[1]
    for b in range(scale.shape[1]):
        part = slice(128 * b, min(C, 128 * b + 128))
        s, v, err = scale[:, b:b + 1], value[:, part], bound[:, part]
        top, slack = v.abs().amax(1, keepdim=True), err.amax(1, keepdim=True)
        assert (torch.frexp(s)[0] == 0.5).all(), f'{what}: scales'
        assert (top - slack <= 448 * s).all() and ((top + slack > 224 * s) | (s == 2.0 ** -126)).all(), f'{what}: scales'
        off = (data[:, part] * s - v).abs()
        allowed = err + 2.0 ** -4 * (v.abs() + err) + 2.0 ** -10 * s
        assert (off <= allowed).all(), f'{what}: {(off / allowed).max().item()} of what it may be off'


def rms_norm_exact(x, weight, residual=None, eps=1e-6, grad=None, grad_sum=None):
    """[(value, bound), ...] of y, s and, with grad, of the gradients of x and weight. Sums of C terms are good to
    (C + 32) e of the terms' magnitudes, column sums of R rows to (R + 32) e; the mean's terms are all positive, so the
    reciprocal norm is good to g = (C + 40) e."""
    dtype, C = x.dtype, x.shape[-1]
    u, e, tiny = U[dtype], U[torch.float64 if dtype == torch.float64 else torch.float32], TINY[dtype]
    s = x.double() if residual is None else x.double() + residual.double()
    w = weight.double()
    rstd = 1 / torch.sqrt((s ** 2).mean(-1, keepdim=True) + eps)
    z, g = s * rstd, (C + 40) * e
    y = z * w
    found = [(y, (u + g + 8 * e) * y.abs() + tiny), (s, (u + e) * s.abs() + tiny)]
    if grad is None:
        return found
    dy = grad.double()
    h = dy * w
    m = (h * z).mean(-1, keepdim=True)
    ds = rstd * (h - z * m)
    a = (h * z).abs().mean(-1, keepdim=True)
    b = rstd * ((g + 8 * e) * h.abs() + (4 * g + 16 * e) * z.abs() * a)
    if grad_sum is not None:
        ds = ds + grad_sum.double()
        b = b + 2 * e * grad_sum.double().abs()
    rows, zr = dy.reshape(-1, C), z.reshape(-1, C)
    dw = (rows * zr).sum(0)
    dw_b = u * dw.abs() + ((rows.shape[0] + 32) * e + g + 8 * e) * (rows * zr).abs().sum(0) + tiny
    return found + [(ds, u * ds.abs() + b + tiny), (dw, dw_b)]


def product_exact(x, w, dtype, bias=None, act=None):
    """(value, bound) of act(x w^T + bias) in `dtype`, for the values x [M, K] and w [N, K] of 8-bit operands. The
    activations' slopes are at most 1.13 and their own error 16 e of the value and its argument."""
    e, u, tiny = 2.0 ** -24, U[dtype], TINY[dtype]
    x, w = x.double(), w.double()
    v, mag = x @ w.t(), x.abs() @ w.abs().t()
    if bias is not None:
        v, mag = v + bias.double(), mag + bias.double().abs()
    err = (x.shape[1] + 64) * 2 * e * mag
    y = v
    if act is not None:
        y = {'relu': lambda t: t.clamp_min(0), 'silu': lambda t: t * torch.sigmoid(t),
             'gelu': lambda t: t * 0.5 * torch.erfc(-t / 2 ** 0.5)}[act](v)
        err = 1.13 * err + (0 if act == 'relu' else 16 * e) * v.abs()
    return y, (u * (y.abs() + err) + err) * 1.01 + tiny + 2.0 ** -149


def linear_train_exact(x, weight, bias, grad):
    """[(value, bound), ...] of y and of the gradients of x, weight and bias (None without a bias)."""
    dtype, e = x.dtype, 2.0 ** -24
    x8, w8 = through(x, 1, 128), through(weight, 128, 128)
    found = [product_exact(x8, w8, dtype, bias)]
    found.append(product_exact(through(grad, 1, 128), w8.t(), dtype))
    found.append(product_exact(through(grad, 128, 1).t(), through(x8, 128, 1).t(), dtype))
    g = grad.double()
    db = g.sum(0)
    found.append(None if bias is None else
                 (db, U[dtype] * db.abs() + (g.shape[0] + 32) * e * g.abs().sum(0) * 1.01 + TINY[dtype]))
    return found


def behind_rows(data):
    """The bytes behind each row of 8-bit data that the library made, whose rows are a multiple of 16 bytes apart."""
    C = data.shape[-1]
    pitch = -(-C // 16) * 16
    rows = data.numel() // C
    raw = torch.empty(0, dtype=torch.uint8, device=data.device).set_(data.untyped_storage())
    return raw[:rows * pitch].view(rows, pitch)[:, C:]
