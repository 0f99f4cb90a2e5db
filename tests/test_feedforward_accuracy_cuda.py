"""The feed-forward operators where roundings add up or digits cancel: results that are exact, or held to a count of the
roundings that the kernels make."""

import pytest
import torch
from torch.autograd import forward_ad

from fp8_oracle import behind_rows
from marearts_tinydeform_b200 import (attention, deform_attn_layer, layer_norm, linear_fp8, ma_deform_attn, quantize_fp8,
                                      quantize_weight_fp8, rms_norm, sampling_producer)
from test_feedforward_cpu import keeps_what_its_gradients_read

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
