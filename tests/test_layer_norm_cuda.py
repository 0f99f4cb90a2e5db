"""layer_norm on the GPU, forward and backward, against float64 with counted error bounds, and a decoder layer made of
the library's attention, norm and deformable attention."""

import pytest
import torch

from attention_oracle import U, check, layer_norm_exact
from cases import make_layer
from marearts_tinydeform_b200 import (attention, attention_reference, deform_attn_layer, deform_attn_layer_reference,
                                      layer_norm, layer_norm_reference)

pytestmark = pytest.mark.gpu

DTYPES = (torch.float32, torch.float16, torch.bfloat16, torch.float64)
# rows and width: one element; every kernel form, its widest and one past it; odd widths; more rows than a wave
SHAPES = [(1, 1), (3, 7), (1, 256), (300, 256), (17, 257), (5, 512), (9, 513), (33, 515), (4, 1024), (3, 2048),
          (5, 2056), (2, 4096), (3, 4099), (2, 8192), (2, 8191), (20011, 64), (7001, 256), (1500, 640)]
NAMES = ('y', 'grad_x', 'grad_weight', 'grad_bias')


def inputs(rows, C, dtype, seed=0):
    g = torch.Generator(device='cuda').manual_seed(seed)
    x, r, dy = (torch.randn((rows, C), generator=g, device='cuda') for _ in range(3))
    w, b = 1 + 0.2 * torch.randn(C, generator=g, device='cuda'), torch.randn(C, generator=g, device='cuda')
    return [t.to(dtype) for t in (x, w, b, 2 * r + 1, dy * 0.1)]


def run(x, w, b, r, dy):
    leaves = [t.detach().requires_grad_() for t in (x, w, b, r) if t is not None]
    it = iter(leaves)
    args = [None if t is None else next(it) for t in (x, w, b, r)]
    y = layer_norm(*args)
    return [y.detach()] + list(torch.autograd.grad(y, leaves, dy))


@pytest.mark.parametrize('shape', SHAPES, ids=str)
@pytest.mark.parametrize('dtype', DTYPES, ids=str)
def test_layer_norm(cuda, dtype, shape):
    x, w, b, r, dy = inputs(*shape, dtype)
    exact = layer_norm_exact(x, w, b, r, grad=dy)
    with torch.inference_mode():
        check(layer_norm(x, w, b, r), exact[0], 'y (inference)')
    y, dx, dw, db, dr = run(x, w, b, r, dy)
    for name, got, want in zip(NAMES, (y, dx, dw, db), exact):
        check(got, want, name)
    assert torch.equal(dx, dr)
    plain = layer_norm_exact(x, w, grad=dy)
    for name, got, want in zip(NAMES[:3], run(x, w, None, None, dy), plain):
        check(got, want, f'{name} (no residual, no bias)')


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
def test_shapes_strides_and_offsets(cuda, dtype):
    x, w, b, r, dy = inputs(60, 256, dtype, 1)
    want = run(x, w, b, r, dy)
    forms = [lambda t: t.view(3, 4, 5, 256), lambda t: t.t().contiguous().t(),
             lambda t: torch.cat([t.new_zeros(1), t.reshape(-1)])[1:].view(t.shape)]
    for f in forms:
        got = run(f(x), w, b, f(r), f(dy))
        for i, (a, e) in enumerate(zip(got, want)):
            # another load width groups a row's sum differently: compare through the bound instead of bits
            if i not in (2, 3):
                a = a.reshape(e.shape)
        exact = layer_norm_exact(x, w, b, r, grad=dy)
        check(got[0].reshape(60, 256), exact[0], 'y')
        check(got[1].reshape(60, 256), exact[1], 'grad_x')
        check(got[2], exact[2], 'grad_weight')
        check(got[3], exact[3], 'grad_bias')
    assert layer_norm(x[:0], w, b).shape == (0, 256)
    none = run(x[:0], w, b, r[:0], dy[:0])
    assert not none[2].any() and not none[3].any()
    assert layer_norm(x[0], w, b).shape == (256,)


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
def test_rows_far_from_zero_and_constant_rows(cuda, dtype):
    x, w, b, _, dy = inputs(40, 300, dtype, 2)
    far = (x.double() + 100).to(dtype)
    for name, got, want in zip(NAMES, run(far, w, b, None, dy), layer_norm_exact(far, w, b, grad=dy)):
        check(got, want, f'far {name}')
    flat = torch.full_like(x, 2.0)
    y = layer_norm(flat, w, b)
    assert torch.equal(y, b.expand_as(y))
    assert all(torch.isfinite(t).all() for t in run(flat, w, b, None, dy))


@pytest.mark.parametrize('C', (7, 256, 300, 515, 1024, 2048, 4099, 8192))
@pytest.mark.parametrize('dtype, far', [(torch.float32, 1e4), (torch.float32, -3e5), (torch.float64, 1e9),
                                        (torch.float16, 1e3), (torch.bfloat16, 1e3)], ids=str)
def test_rows_very_far_from_zero(cuda, dtype, far, C):
    """Offsets thousands of deviations wide. Each centred value is a difference of near numbers and exact, so their
    sums err by (C + 32) e of the centred values and not of the offset, and z by that; only the saved mean, which the backward
    subtracts, is rounded to e of the offset (e: half a step of the accumulators' type)."""
    x, w, b, _, dy = inputs(40, C, dtype, 6)
    x = (x.double() * max(1.0, abs(far) * U[dtype] * 8) + far).to(dtype)  # a few steps of the type wide at least
    e, u = U[torch.float64 if dtype == torch.float64 else torch.float32], U[dtype]
    s, wd, d = x.double(), w.double(), dy.double()
    mean = s.mean(1, keepdim=True)
    c = s - mean
    c = c - c.mean(1, keepdim=True)  # (float64 itself loses some of such a mean)
    rstd = 1 / torch.sqrt((c ** 2).mean(1, keepdim=True) + 1e-5)
    z, g = c * rstd, (C + 32) * e
    z_err = g * (c.abs().mean(1, keepdim=True) * rstd + z.abs()) + 4 * e * z.abs()
    y = z * wd + b.double()
    got = run(x, w, b, None, dy)
    check(got[0], (y, (u + 4 * e) * y.abs() + z_err * wd.abs() + 4 * e * (z * wd).abs()), 'y')
    z_err = z_err + 1.01 * e * mean.abs() * rstd
    h = d * wd
    a1, a2 = h.abs().mean(1, keepdim=True), (h * z).abs().mean(1, keepdim=True)
    dx = rstd * (h - h.mean(1, keepdim=True) - z * (h * z).mean(1, keepdim=True))
    check(got[1], (dx, u * dx.abs() + rstd * (8 * g * (h.abs() + a1 + z.abs() * a2) + z_err * a2
                                              + z.abs() * (h.abs() * z_err).mean(1, keepdim=True))), 'grad_x')
    dw = (d * z).sum(0)
    check(got[2], (dw, u * dw.abs() + (40 + 32) * e * (d * z).abs().sum(0) + (d.abs() * z_err).sum(0)), 'grad_weight')


def test_same_bits_every_time(cuda):
    x, w, b, r, dy = inputs(9000, 256, torch.float16, 3)
    first = run(x, w, b, r, dy)
    assert all(torch.equal(p, q) for _ in range(3) for p, q in zip(first, run(x, w, b, r, dy)))


def test_gradients_against_differences(cuda):
    torch.manual_seed(0)
    x, r = (torch.randn((3, 5, 7), dtype=torch.float64, device='cuda', requires_grad=True) for _ in range(2))
    w, b = (torch.randn(7, dtype=torch.float64, device='cuda', requires_grad=True) for _ in range(2))
    assert torch.autograd.gradcheck(layer_norm, (x, w, b, r))
    # the same tensor as input and residual: its gradient counts twice
    assert torch.autograd.gradcheck(lambda t: layer_norm(t, w, b, t), (x,))
    y = layer_norm(x, w, b, r)
    y.sum().backward()  # two leaves with one gradient tensor: accumulating into one leaves the other alone
    keep = r.grad.clone()
    x.grad.add_(1)
    assert torch.equal(r.grad, keep)


def test_graph_capture(cuda):
    x, w, b, r, dy = inputs(700, 256, torch.bfloat16, 4)
    leaves = [t.requires_grad_() for t in (x, w, b, r)]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for _ in range(2):
            torch.autograd.grad(layer_norm(*leaves), leaves, dy)
        graph = torch.cuda.CUDAGraph()
        stream.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            y = layer_norm(*leaves)
            grads = torch.autograd.grad(y, leaves, dy)
    fresh = inputs(700, 256, torch.bfloat16, 5)
    with torch.no_grad():
        for t, f in zip((*leaves, dy), fresh):
            t.copy_(f)
    graph.replay()
    torch.cuda.synchronize()
    for got, want in zip((y, *grads), run(*fresh)):
        assert torch.equal(got, want)


# ---- the operators together: one decoder layer --------------------------------------------------------------------

def decoder_layer(p, attend, norm, cross):
    """DETR's decoder layer without its feed-forward half: self attention and its norm, deformable attention and its
    norm, on the parameters p."""
    tgt, qkv_w = p['query'], p['qkv_w']
    B, Q, C = tgt.shape
    q, k, v = torch.nn.functional.linear(tgt, qkv_w).view(B, Q, 3, p['H'], C // p['H']).unbind(2)
    tgt = norm(attend(q, k, v, attn_mask=p['mask']), p['n1_w'], p['n1_b'], tgt)
    return cross(tgt, p)


def library_cross(tgt, p):
    return deform_attn_layer(tgt, p['ref'], p['memory'], p['shapes'], p['starts'], p['H'], p['P'], p['sw'], p['sb'],
                             p['vw'], p['vb'], output_weight=p['ow'], residual=tgt, norm_weight=p['n2_w'],
                             norm_bias=p['n2_b'])


def reference_cross(tgt, p):
    out = deform_attn_layer_reference(tgt, p['ref'], p['memory'], p['shapes'], p['starts'], p['H'], p['P'], p['sw'],
                                      p['sb'], p['vw'], p['vb'], p['ow'])
    return layer_norm_reference(out, p['n2_w'], p['n2_b'], tgt)


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
def test_decoder_layer(cuda, dtype):
    H, P, C = 8, 4, 256
    args = make_layer(2, 90, C, H, C // H, C, [(12, 10), (6, 5)], P, ref_dim=4, dtype=dtype, seed=21)
    q, ref, mem, shapes, starts, sw, sb, vw, vb = [None if t is None else t.cuda() for t in args]
    g = torch.Generator(device='cuda').manual_seed(22)

    def normal(*s, std):
        return (torch.randn(s, generator=g, device='cuda') * std).to(dtype)

    mask = torch.zeros((90, 90), dtype=torch.bool, device='cuda')
    mask[30:, :30] = True
    p = dict(query=q, qkv_w=normal(3 * C, C, std=C ** -0.5), H=H, P=P, mask=mask, ref=ref, memory=mem, shapes=shapes,
             starts=starts, sw=sw, sb=sb, vw=vw, vb=vb, ow=normal(C, C, std=C ** -0.5), n1_w=1 + normal(C, std=0.1),
             n1_b=normal(C, std=0.1), n2_w=1 + normal(C, std=0.1), n2_b=normal(C, std=0.1))
    names = ('query', 'qkv_w', 'memory', 'vw', 'ow', 'n1_w', 'n1_b', 'n2_w', 'n2_b')
    grad = normal(2, 90, C, std=0.1)

    def both(p, *parts):
        p = dict(p, **{n: p[n].detach().requires_grad_() for n in names})
        out = decoder_layer(p, *parts)
        return [out.detach()] + list(torch.autograd.grad(out, [p[n] for n in names], grad.to(out.dtype)))

    wide = {n: t.double() if torch.is_tensor(t) and t.is_floating_point() else t for n, t in p.items()}
    want = both(wide, attention_reference, layer_norm_reference, reference_cross)
    got = both(p, attention, layer_norm, library_cross)
    # ten roundings to the type lie on the longest way through the layer and as many on the way back, each of half a
    # step of its tensor; a sampling location off by half a step of the type moves a sample by up to 12 pixels' half
    # step, which the bilinear slope turns into a relative error of a value: 12 more.
    # The slope itself jumps at the pixels' borders. A location rounded by u (of coordinates up to 1, on maps up to 12
    # pixels wide) moves by up to 12 u pixels and so crosses a border with a probability of up to 24 u in each of two
    # directions; a crossed sample's slope is another one of the same size, off by sqrt(2) of itself in the mean
    # square. Gradients that come through the locations are so off by up to sqrt(2 * 48 u) in norm (0.22 in float16,
    # 0.61 in bfloat16); in float32 the 23040 coordinates cross 0.03 borders, and nothing is allowed for it.
    cross = (2 * 48 * U[dtype]) ** 0.5 if dtype in (torch.float16, torch.bfloat16) else 0.0
    for name, a, b in zip(('out', *names), got, want):
        rel = ((a.double() - b).norm() / b.norm()).item()
        allowed = 32 * U[dtype] + 2e-6 * (dtype == torch.float32) + 1e-13
        if name in ('query', 'qkv_w', 'n1_w', 'n1_b'):
            allowed += cross
        assert rel <= allowed, f'{name}: {rel}'
    with torch.inference_mode():
        assert torch.equal(decoder_layer(p, attention, layer_norm, library_cross).isfinite().all(),
                           torch.tensor(True, device='cuda'))


def library_cross_at(tgt, p):
    """library_cross with sampling locations and weights that pass no gradient."""
    return deform_attn_layer(tgt.detach(), p['ref'], p['memory'], p['shapes'], p['starts'], p['H'], p['P'], p['sw'],
                             p['sb'], p['vw'], p['vb'], output_weight=p['ow'], residual=tgt, norm_weight=p['n2_w'],
                             norm_bias=p['n2_b'])


def reference_cross_at(tgt, p):
    out = deform_attn_layer_reference(tgt.detach(), p['ref'], p['memory'], p['shapes'], p['starts'], p['H'], p['P'],
                                      p['sw'], p['sb'], p['vw'], p['vb'], p['ow'])
    return layer_norm_reference(out, p['n2_w'], p['n2_b'], tgt)


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
def test_decoder_layer_with_fixed_locations(cuda, dtype):
    """The decoder layer's gradients where nothing jumps: the sampling locations pass none, so that no sample's slope
    changes at a pixel's border, and every gradient is held to the count of roundings alone (as above: twenty of half a
    step on the way there and back, and 12 for a sample moved by a rounded location)."""
    H, P, C = 8, 4, 256
    args = make_layer(2, 90, C, H, C // H, C, [(12, 10), (6, 5)], P, ref_dim=4, dtype=dtype, seed=23)
    q, ref, mem, shapes, starts, sw, sb, vw, vb = [None if t is None else t.cuda() for t in args]
    g = torch.Generator(device='cuda').manual_seed(24)

    def normal(*s, std):
        return (torch.randn(s, generator=g, device='cuda') * std).to(dtype)

    mask = torch.zeros((90, 90), dtype=torch.bool, device='cuda')
    mask[30:, :30] = True
    p = dict(query=q, qkv_w=normal(3 * C, C, std=C ** -0.5), H=H, P=P, mask=mask, ref=ref, memory=mem, shapes=shapes,
             starts=starts, sw=sw, sb=sb, vw=vw, vb=vb, ow=normal(C, C, std=C ** -0.5), n1_w=1 + normal(C, std=0.1),
             n1_b=normal(C, std=0.1), n2_w=1 + normal(C, std=0.1), n2_b=normal(C, std=0.1))
    names = ('query', 'qkv_w', 'memory', 'vw', 'ow', 'n1_w', 'n1_b', 'n2_w', 'n2_b')
    grad = normal(2, 90, C, std=0.1)

    def both(p, *parts):
        p = dict(p, **{n: p[n].detach().requires_grad_() for n in names})
        out = decoder_layer(p, *parts)
        return [out.detach()] + list(torch.autograd.grad(out, [p[n] for n in names], grad.to(out.dtype)))

    wide = {n: t.double() if torch.is_tensor(t) and t.is_floating_point() else t for n, t in p.items()}
    want = both(wide, attention_reference, layer_norm_reference, reference_cross_at)
    got = both(p, attention, layer_norm, library_cross_at)
    for name, a, b in zip(('out', *names), got, want):
        rel = ((a.double() - b).norm() / b.norm()).item()
        assert rel <= 32 * U[dtype] + 2e-6 * (dtype == torch.float32) + 1e-13, f'{name}: {rel}'
