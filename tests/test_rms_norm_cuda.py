"""rms_norm on the GPU, forward, in 8 bits and backward, against float64 with counted error bounds."""

import pytest
import torch

from attention_oracle import check
from fp8_oracle import behind_rows, check_quantized, rms_norm_exact
from marearts_tinydeform_b200 import quantize_fp8, rms_norm

pytestmark = pytest.mark.gpu

DTYPES = (torch.float32, torch.float16, torch.bfloat16, torch.float64)
# rows and width: one element; every kernel form, its widest and one past it; odd widths; more rows than a wave
SHAPES = [(1, 1), (3, 7), (1, 256), (300, 256), (17, 257), (5, 264), (5, 512), (9, 513), (33, 515), (4, 1024),
          (4, 1032), (3, 2048), (5, 2056), (2, 4096), (3, 4099), (2, 4104), (2, 8192), (2, 8191), (20011, 64),
          (7001, 256), (1500, 640), (700, 4096), (600, 8192), (513, 1000)]


def inputs(rows, C, dtype, seed=0):
    g = torch.Generator(device='cuda').manual_seed(seed)
    x, r, dy, ds = (torch.randn((rows, C), generator=g, device='cuda') for _ in range(4))
    w = 1 + 0.2 * torch.randn(C, generator=g, device='cuda')
    return [t.to(dtype) for t in (x, w, 2 * r + 0.5, dy * 0.1, ds * 0.1)]


def run(x, w, r, dy, ds=None):
    """[y, sum, gradients of x, weight and residual], the sum and its gradient where ds is given."""
    leaves = [t.detach().requires_grad_() for t in (x, w, r) if t is not None]
    out = rms_norm(leaves[0], leaves[1], leaves[2] if r is not None else None, return_sum=ds is not None)
    outs = [out] if ds is None else list(out)
    return [t.detach() for t in outs] + list(torch.autograd.grad(outs, leaves, [dy] if ds is None else [dy, ds]))


@pytest.mark.parametrize('shape', SHAPES, ids=str)
@pytest.mark.parametrize('dtype', DTYPES, ids=str)
def test_rms_norm(cuda, dtype, shape):
    x, w, r, dy, ds = inputs(*shape, dtype)
    exact = rms_norm_exact(x, w, r, grad=dy, grad_sum=ds)
    with torch.inference_mode():
        y, s = rms_norm(x, w, r, return_sum=True)
        check(y, exact[0], 'y (inference)')
        check(s, exact[1], 'sum (inference)')
        if dtype != torch.float64:
            y8, s8 = rms_norm(x, w, r, return_sum=True, quantize=True)
            check_quantized(y8, exact[0], 'y in 8 bits')
            assert torch.equal(s8, s)
            assert not behind_rows(y8[0]).any()
            check_quantized(rms_norm(x, w, quantize=True), rms_norm_exact(x, w)[0], 'y in 8 bits (no residual)')
    y, s, dx, dw, dr = run(x, w, r, dy, ds)
    for name, got, want in zip(('y', 'sum', 'grad_x', 'grad_weight'), (y, s, dx, dw), exact):
        check(got, want, name)
    assert torch.equal(dx, dr)
    plain = rms_norm_exact(x, w, grad=dy)
    for name, got, want in zip(('y', 'grad_x', 'grad_weight'), run(x, w, None, dy), (plain[0], *plain[2:])):
        check(got, want, f'{name} (no residual)')


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
def test_shapes_strides_and_offsets(cuda, dtype):
    x, w, r, dy, ds = inputs(60, 256, dtype, 1)
    exact = rms_norm_exact(x, w, r, grad=dy, grad_sum=ds)
    forms = [lambda t: t.view(3, 4, 5, 256), lambda t: t.t().contiguous().t(),
             lambda t: torch.cat([t.new_zeros(1), t.reshape(-1)])[1:].view(t.shape)]
    for f in forms:
        for got, want in zip(run(f(x), w, f(r), f(dy), f(ds))[:4], exact):
            check(got.reshape(want[0].shape), want, 'form')
        if dtype != torch.float64:
            data, scale = rms_norm(f(x), w, f(r), quantize=True)
            assert data.shape == f(x).shape and scale.shape == (*f(x).shape[:-1], 2)
            check_quantized((data, scale), exact[0], 'form in 8 bits')
    assert rms_norm(x[:0], w).shape == (0, 256) and rms_norm(x[0], w).shape == (256,)
    assert not run(x[:0], w, r[:0], dy[:0], ds[:0])[3].any()


def test_rows_at_the_types_ends(cuda):
    """Zero rows, tiny rows, and rows whose 8-bit blocks differ by all of a type's range."""
    w = torch.ones(384, device='cuda')
    x = torch.zeros(4, 384, device='cuda')
    x[1] = 1e-18
    x[2, :128], x[2, 128:256], x[2, 256:] = 1e-12, 1.0, 1e12
    x[3, 5] = float('nan')
    y = rms_norm(x, w, eps=1e-30)
    check(y[:3], rms_norm_exact(x[:3], w, eps=1e-30)[0], 'ends')
    assert y[3].isnan().all()
    data, scale = rms_norm(x, w, eps=1e-30, quantize=True)
    check_quantized((data[:3], scale[:3]), rms_norm_exact(x[:3], w, eps=1e-30)[0], 'ends in 8 bits')
    assert data[3].float().isnan().all() and not data[0].float().any()


def test_quantized_result_is_its_rounded_once(cuda):
    """float32 rows: the 8-bit result is the float32 result, quantised."""
    for C in (256, 515, 1030, 4099):
        x, w, r, _, _ = inputs(50, C, torch.float32, 8)
        for a, b in zip(rms_norm(x, w, r, quantize=True), quantize_fp8(rms_norm(x, w, r))):
            assert torch.equal(a.float(), b.float())


def test_either_output_alone(cuda):
    x, w, r, dy, ds = inputs(40, 256, torch.float32, 2)
    leaves = [t.requires_grad_() for t in (x, w, r)]
    both = torch.autograd.grad(rms_norm(*leaves, return_sum=True), leaves, (dy, ds))
    y, s = rms_norm(*leaves, return_sum=True)
    alone = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    for a, b in zip(alone, torch.autograd.grad(rms_norm(*leaves), leaves, dy)):
        assert torch.equal(a, b)
    assert torch.equal(torch.autograd.grad(s, (leaves[0], leaves[2]), ds)[0], ds)
    torch.testing.assert_close(both[0], alone[0] + ds, rtol=1e-6, atol=1e-7)
    x8 = torch.randn(3, 256, device='cuda', requires_grad=True)
    with pytest.raises(RuntimeError, match='no gradient'):
        rms_norm(x8, w, quantize=True)


def test_offsets_past_31_bits(cuda):
    """More than 2^31 values: the last rows are the same rows' alone."""
    rows, C = 2100000, 1024
    x, w = torch.randn(rows, C, dtype=torch.bfloat16, device='cuda'), inputs(1, C, torch.bfloat16)[1]
    part = x[-300:].clone()
    with torch.inference_mode():
        (data, scale), s = rms_norm(x, w, quantize=True, return_sum=True)
        want = rms_norm(part, w, quantize=True)
        assert torch.equal(data[-300:].float(), want[0].float()) and torch.equal(scale[-300:], want[1])
        assert torch.equal(s[-300:], part)
        del data, s
    leaf = x.requires_grad_()
    grad = torch.autograd.grad(rms_norm(leaf, w), leaf, x.detach())[0]
    alone = part.requires_grad_()
    assert torch.equal(grad[-300:], torch.autograd.grad(rms_norm(alone, w), alone, part.detach())[0])


def test_same_bits_every_time(cuda):
    x, w, r, dy, ds = inputs(9000, 256, torch.float16, 3)
    first = run(x, w, r, dy, ds)
    assert all(torch.equal(p, q) for _ in range(3) for p, q in zip(first, run(x, w, r, dy, ds)))


def test_gradients_against_differences(cuda):
    torch.manual_seed(0)
    x, r = (torch.randn((3, 5, 7), dtype=torch.float64, device='cuda', requires_grad=True) for _ in range(2))
    w = torch.randn(7, dtype=torch.float64, device='cuda', requires_grad=True)
    assert torch.autograd.gradcheck(rms_norm, (x, w, r))
    assert torch.autograd.gradcheck(lambda a, b, c: rms_norm(a, b, c, return_sum=True), (x, w, r))
    assert torch.autograd.gradcheck(lambda t: rms_norm(t, w, t), (x,))


def test_graph_capture(cuda):
    x, w, r, dy, ds = inputs(700, 256, torch.bfloat16, 4)
    leaves = [t.requires_grad_() for t in (x, w, r)]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for _ in range(2):
            torch.autograd.grad(rms_norm(*leaves, return_sum=True), leaves, (dy, ds))
        graph = torch.cuda.CUDAGraph()
        stream.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            out = rms_norm(*leaves, return_sum=True)
            grads = torch.autograd.grad(out, leaves, (dy, ds))
    fresh = inputs(700, 256, torch.bfloat16, 5)
    with torch.no_grad():
        for t, f in zip((*leaves, dy, ds), fresh):
            t.copy_(f)
    graph.replay()
    torch.cuda.synchronize()
    for got, want in zip((*out, *grads), run(*fresh)):
        assert torch.equal(got, want)
