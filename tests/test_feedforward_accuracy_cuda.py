"""The feed-forward operators where roundings add up or digits cancel: results that are exact, or held to a count of the
roundings that the kernels make."""

import pytest
import torch
from torch.autograd import forward_ad

from fp8_oracle import behind_rows, quantized, through, worth
from marearts_tinydeform_b200 import (attention, deform_attn_layer, dequantize_fp8, layer_norm, linear_fp8, ma_deform_attn,
                                      quantize_fp8, quantize_weight_fp8, rms_norm, sampling_producer)
from test_feedforward_cpu import check_feed_forward, keeps_what_its_gradients_read
from test_linear_fp8_cuda import ACTS, DTYPES, SHAPES, normal

pytestmark = pytest.mark.gpu

E = 2.0 ** -24  # half a step of float32, relative


@pytest.mark.parametrize('M, K', [(2, 128), (40, 128), (40, 4096), (2400, 128)])
def test_activations_keep_their_digits(policy, M, K):
    """GELU and SiLU relative to their own values, where those are far smaller than the argument too.

    E is half a step of float32. GELU, v (1 - Phi(|v|)) below zero: the tail's smooth factor is good to 7 E (its fit 1,
    nine fused steps and a reciprocal good to a step the rest), its exponential to 2 steps (4 E), whose argument, rounded
    twice behind a rounded constant, adds at most 1.5 v^2 E; a product, and 1 - tail or v times it: (14 + 2 v^2) E. SiLU,
    v exp(-|v|) / (1 + exp(-|v|)) below zero: an exponential good to 2 steps (4 E, and no more again through the sum), a
    product, a sum, a reciprocal good to a step and its product: 14 E. Below float32's normal numbers each of these steps
    may be off by 2^-149, times up to |v| + 1."""
    N = 1024 if M > 1000 else 270
    v = torch.linspace(-14, 14, N, device='cuda')
    v[:9] = torch.tensor([-110., -100, -96, -90, -88.5, -88, -87, -40, -20], device='cuda')
    x = torch.ones(M, K, device='cuda')
    w8 = quantize_weight_fp8(torch.zeros(N, K, device='cuda'))
    d = v.double()
    exact = {'gelu': (0.5 * d * torch.erfc(-d / 2 ** 0.5), (14 + 2 * d * d) * E), 'silu': (d * torch.sigmoid(d), 14 * E)}
    for act, (want, bound) in exact.items():
        got = linear_fp8(x, w8, v, act)
        off = (got.double() - want).abs()
        allowed = bound * want.abs() + (d.abs() + 1) * 2.0 ** -148
        assert (off <= allowed).all(), f'{act}: {(off / allowed).max().item()} of what it may be off'


@pytest.mark.parametrize('M, K, N', [(1, 2048, 260), (16, 2048, 260), (40, 2048, 260), (2400, 2048, 1024),
                                     (300, 2048, 4100)])
def test_a_large_bias_is_rounded_once(policy, M, K, N):
    """Each block of 128 adds 1/4 to a bias of 2^23, whose neighbours are 1 away: with the products first the result is
    the exact sum, 2^23 + 4."""
    x, w = torch.ones(M, K, device='cuda'), torch.full((N, K), 2.0 ** -9, device='cuda')
    got = linear_fp8(x, quantize_weight_fp8(w), torch.full((N,), 2.0 ** 23, device='cuda'))
    assert (got == 2.0 ** 23 + K / 512).all()
    leaves = [t.requires_grad_() for t in (x, w)]
    assert (linear_fp8(*leaves, torch.full((N,), 2.0 ** 23, device='cuda')) == 2.0 ** 23 + K / 512).all()


def test_column_sums_that_cancel(cuda):
    """Gradients summed over rows, where the first and the last rows' 2^26 cancel and ones lie between: what CTAs have
    added is joined in float64, so the ones are all there."""
    g = torch.zeros(100 * 128, 40, device='cuda')  # 100 blocks of 128 rows
    g[::128] = 1
    g[0], g[99 * 128] = 2.0 ** 26, -2.0 ** 26
    leaves = [torch.ones(s, device='cuda', requires_grad=True) for s in ((g.shape[0], 8), (40, 8), (40,))]
    assert (torch.autograd.grad(linear_fp8(*leaves), leaves[2], g)[0] == 98).all()
    rows, C = 148 * 8, 256  # a row for each of a CTA's warps
    g = torch.ones(rows, C, device='cuda')
    g[:8] = g[-8:] = 0
    g[0], g[-1] = 2.0 ** 26, -2.0 ** 26
    x, w = (torch.ones(s, device='cuda', requires_grad=True) for s in ((rows, C), (C,)))
    assert (torch.autograd.grad(rms_norm(x, w, eps=0.0), w, g)[0] == rows - 16).all()


def test_the_graph_keeps_what_its_gradients_read(policy):
    keeps_what_its_gradients_read('cuda')
    x = torch.randn(4096, 1024, device='cuda', dtype=torch.bfloat16, requires_grad=True)
    w = torch.randn(128, 1024, device='cuda', dtype=torch.bfloat16)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    y = linear_fp8(x, w)
    assert torch.cuda.memory_allocated() - before == y.numel() * 2  # a frozen weight: nothing of the input is kept


def test_forward_mode_tangents_are_refused(cuda):
    """An operator that dropped its operand's tangent would give a constant."""
    x, w, q = (torch.randn(s, device='cuda') for s in ((6, 64), (64, 64), (1, 6, 2, 32)))
    shapes, start = torch.tensor([[4, 4]], device='cuda'), torch.tensor([0], device='cuda')
    loc, attn = torch.rand(1, 5, 2, 1, 4, 2, device='cuda'), torch.rand(1, 5, 2, 1, 4, device='cuda')
    memory, query, ref = (torch.randn(s, device='cuda') for s in ((1, 16, 64), (1, 5, 64), (1, 5, 1, 2)))
    sw = torch.randn(2 * 4 * 3, 64, device='cuda')
    calls = [(x, lambda t: rms_norm(t, w[0])), (w, lambda t: linear_fp8(x, t)),
             (x, lambda t: linear_fp8(t, quantize_weight_fp8(w))), (x, quantize_fp8), (x, lambda t: layer_norm(t, w[0])),
             (q, lambda t: attention(t, q, q)),
             (memory, lambda t: ma_deform_attn(t, w, None, shapes, start, loc, attn)),
             (query, lambda t: sampling_producer(t, ref, shapes, 2, 4, sw, None)),
             (memory, lambda t: deform_attn_layer(query, ref, t, shapes, start, 2, 4, sw, None, w, None))]
    for operand, call in calls:
        call(operand)
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(operand, torch.ones_like(operand))
            with pytest.raises(RuntimeError, match='forward-mode'):
                call(dual)
            with pytest.raises(RuntimeError, match='forward-mode'), torch.no_grad():  # (of reverse mode alone)
                call(dual)
            call(operand)


def test_zeros_behind_rows_of_nan(policy):
    """What lies behind an 8-bit row is zero, whatever the row holds: an infinity or a NaN in it, or (without eps) none
    but zeros."""
    for C in (129, 130, 136, 520, 521, 1030, 2057, 4099, 8190):
        x = torch.randn(5, C, device='cuda')
        x[0, 3], x[1, C - 1], x[2] = float('nan'), float('inf'), 0
        w8 = quantize_weight_fp8(torch.randn(C, C if C < 2000 else 300, device='cuda'))
        for x in (x, x.half(), x.repeat(60, 1)):
            y = rms_norm(x, x.new_ones(C), eps=0.0, quantize=True)[0]
            assert y[:3].float().isnan().any(1).all() and not behind_rows(y).any()
            assert not behind_rows(quantize_fp8(x)[0]).any()
            y = linear_fp8(x[:, :w8[0].shape[1]], w8, quantize=True)[0]
            assert y[0].float().isnan().all() and not behind_rows(y).any()


def whole(*shape, seed, wide=None):
    """Whole numbers from -15 to 15 (four bits, which survive any of the roundings to 8 bits), every 61st index along
    the dimension `wide` times 8."""
    gen = torch.Generator(device='cuda').manual_seed(seed)
    v = torch.randint(-15, 16, shape, generator=gen, device='cuda').float()
    if wide is not None:
        v.select(wide, 0).mul_(8) if shape[wide] < 61 else v.movedim(wide, 0)[::61].mul_(8)
    return v


@pytest.mark.parametrize('shape', SHAPES, ids=str)
@pytest.mark.parametrize('dtype', DTYPES, ids=str)
def test_whole_numbers_are_exact(policy, dtype, shape):
    """Products and all three gradients of whole numbers whose sums stay below 2^24 (at most 8200 * 225 + 135 * 64 * 225):
    every partial sum is one, so the results are the exact ones, rounded once."""
    M, K, N = shape
    x, w = whole(M, K, seed=1, wide=1).to(dtype), whole(N, K, seed=2, wide=1).to(dtype)
    b, g = whole(N, seed=3).to(dtype), whole(M, N, seed=4).to(dtype)
    xd, wd, gd = x.double(), w.double(), g.double()
    want = xd @ wd.t() + b.double()
    w8 = quantize_weight_fp8(w)
    assert torch.equal(linear_fp8(x, w8, b), want.to(dtype))
    assert torch.equal(linear_fp8(quantize_fp8(x), w8, b, dtype=torch.float32).double(), want)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    y = linear_fp8(*leaves)
    assert torch.equal(y, want.to(dtype))
    for got, exact in zip(torch.autograd.grad(y, leaves, g), (gd @ wd, gd.t() @ xd, gd.sum(0))):
        assert torch.equal(got, exact.to(dtype))


def test_a_bad_gradient_leaves_the_other_rows(policy):
    """An infinity and a NaN in the incoming gradient take their row of grad_x and of grad_weight; the others keep their
    bits."""
    x, w, g = normal(300, 200), normal(140, 200, seed=1), normal(300, 140, seed=3)

    def grads():
        leaves = [t.detach().requires_grad_() for t in (x, w)]
        return torch.autograd.grad(linear_fp8(*leaves), leaves, g)

    clean = grads()
    g[7, 3], g[250, 139] = float('inf'), float('nan')
    for got, want, bad in zip(grads(), clean, ([7, 250], [3, 139])):
        rest = [i for i in range(got.shape[0]) if i not in bad]
        assert got[bad].isnan().all() and torch.equal(got[rest], want[rest])


@pytest.mark.parametrize('act', ACTS, ids=str)
@pytest.mark.parametrize('M', (1, 9, 200))
def test_bad_columns_leave_an_8_bit_block_its_rounding(policy, M, act):
    """NaN in columns of a block: the others are the float32 results rounded with the scale that these call for, to half a
    step (2^-4 of the value, 2^-10 of the scale; 2^-20 for the sums' own roundings)."""
    x, w, b = normal(M, 300), normal(270, 300, seed=1), normal(270, seed=2)
    bad = [5, 140, 269]
    w[5, 299], w[140, 0], b[269] = float('nan'), float('inf'), float('nan')
    w8 = quantize_weight_fp8(w)
    v = linear_fp8(x, w8, b, act).double()
    data, scale = (t.double() for t in linear_fp8(x, w8, b, act, quantize=True))
    assert data[:, bad].isnan().all()
    for block in range(3):
        cols = [n for n in range(128 * block, min(270, 128 * block + 128)) if n not in bad]
        s, top = scale[:, block], v[:, cols].abs().amax(1)
        assert (top <= 448 * s * (1 + 2.0 ** -20)).all() and (top > 224 * s * (1 - 2.0 ** -20)).all()
        off = (data[:, cols] * s[:, None] - v[:, cols]).abs()
        assert (off <= (2.0 ** -4 + 2.0 ** -20) * v[:, cols].abs() + 2.0 ** -10 * s[:, None]).all()


@pytest.mark.parametrize('dtype', (torch.float32, torch.bfloat16), ids=str)
def test_tiny_values_go_to_8_bits_and_back(cuda, dtype):
    """Below float32's normal numbers, where the scale cannot be smaller: data as by definition, from each kernel that
    rounds, and back exactly."""
    for C in (128, 136, 130):
        x = whole(40, C, seed=9).double() * 2.0 ** -torch.arange(108, 148, device='cuda').double()[:, None]
        x = x.float().to(dtype)
        for make, rows in ((quantize_fp8, 1), (quantize_weight_fp8, 128)):
            for part in (x, x[20:].contiguous()):
                q, s = quantized(part, rows, 128)
                data, scale = make(part)
                assert torch.equal(scale.double(), s) and torch.equal(data.double(), q)
                assert torch.equal(dequantize_fp8(data, scale, torch.float32).double(), worth(q, s, rows, 128))
        leaves = [t.requires_grad_() for t in (x, x[:30].clone())]
        y = linear_fp8(*leaves)
        data, scale, _ = y.grad_fn.saved_tensors  # a training call's copy of its input
        q, s = quantized(x.detach(), 1, 128)
        assert torch.equal(scale.double(), s) and torch.equal(data.double(), q)


def held_to_blocks(got, a, b):
    """got = a b^T in float32: a block's 128 exact products are added in float32 (128 roundings or cuts), the blocks of K
    in turn, and perhaps the parts of a split sum, no more than there are blocks; 16 more for the scales and the rest."""
    a, b = a.double(), b.double()
    mag, blocks = a.abs() @ b.abs().t(), -(-a.shape[1] // 128)
    off, allowed = (got.double() - a @ b.t()).abs(), (128 + 2 * blocks + 16) * 2 * E * mag + 2.0 ** -149
    assert (off <= allowed).all(), f'{(off / allowed).max().item()} of what it may be off'


@pytest.mark.parametrize('shape', [(1, 4096, 700), (16, 4100, 512), (33, 4099, 40), (130, 8200, 130), (5000, 384, 1000),
                                   (40, 300, 20000), (20000, 100, 60)], ids=str)
def test_long_sums_are_held_to_float32(policy, shape):
    """Sums over many blocks, in the product and in both gradients, to roundings that count blocks and not values."""
    M, K, N = shape
    x, w, g = normal(M, K), normal(N, K, seed=1), normal(M, N, seed=2)
    leaves = [t.requires_grad_() for t in (x, w)]
    y = linear_fp8(*leaves)
    gx, gw = torch.autograd.grad(y, leaves, g)
    x, w, y = x.detach(), w.detach(), y.detach()
    x8, w8 = through(x, 1, 128), through(w, 128, 128)
    held_to_blocks(y, x8, w8)
    with torch.no_grad():
        held_to_blocks(linear_fp8(x, quantize_weight_fp8(w)), x8, w8)
    held_to_blocks(gx, through(g, 1, 128), w8.t())
    held_to_blocks(gw, through(g, 128, 1).t(), through(x8, 128, 1).t())


def test_a_models_feed_forward_half_in_serving(policy):
    check_feed_forward('cuda')
