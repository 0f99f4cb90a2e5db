"""16-bit attention on the GPU, over whole results: what is left besides the result's own rounding.

Element by element a bound has to allow for every term of a sum at its worst, and cannot tell a factor that was rounded
to 16 bits from one that was not. Over a whole result the roundings add up as a random walk does, and can. The measure
is the result's distance from float64, in units of the distance that rounding float64's result to the type leaves (a
step of relative size u = finfo.eps / 2 is off by 0.29 u to 0.58 u in the mean square, as the mantissa has it).

What else is allowed. A factor kept in two 16-bit parts is off by u^2. Scores and sums are float32: D <= 128 products
and scores of a few units make 2^-19 of a probability; a tensor core cuts its running sum by up to 2^-24 for every 8
terms, in one direction: 2^-15 over 4200 terms. Against u = 2^-11 that is u / 16, so at most (u / 16) / (0.29 u) = 0.22
of the measure where it all adds up in line with the rounding. One factor rounded once to 16 bits adds about 0.4 u at
random instead: sqrt(2) of the measure or nearly so."""

import pytest
import torch

from attention_oracle import U, attention_exact, blocked_pairs
from marearts_tinydeform_b200 import _native, attention
from test_attention_cuda import NAMES, inputs, masks, run

pytestmark = pytest.mark.gpu

HALVES = (torch.float16, torch.bfloat16)
LIMIT = 1.22
# B, Q, N, H, Hk, D: a decoder's, a tile or two with every width, shared heads, keys split among CTAs (tensor cores),
# one and few queries (the split kernel), an odd width (CUDA cores)
SHAPES = [(1, 300, 300, 8, 8, 32), (2, 520, 640, 4, 2, 64), (1, 300, 515, 4, 2, 128), (2, 200, 333, 6, 3, 24),
          (1, 300, 4200, 4, 4, 32), (2, 1, 2500, 8, 4, 64), (4, 9, 1500, 6, 2, 32), (2, 3, 4200, 8, 2, 128),
          (1, 90, 150, 4, 4, 20)]


def off(got, exact, dtype):
    """The measure above; a result of zeros that should be zeros is off by nothing."""
    own = (exact.to(dtype).double() - exact).norm()
    return 0.0 if own == 0 and not (got.double() != exact).any() else ((got.double() - exact).norm() / own).item()


@pytest.mark.parametrize('kind', ('none', 'pairs', 'causal', 'padding'))
@pytest.mark.parametrize('shape', SHAPES, ids=str)
@pytest.mark.parametrize('dtype', HALVES, ids=str)
def test_only_the_result_is_rounded(cuda, dtype, shape, kind):
    q, k, v, _ = inputs(shape, dtype, 41)
    kw = masks(kind, shape, 41)
    exact = attention_exact(q, k, v, **kw)[0][0]
    with torch.inference_mode():
        found = off(attention(q, k, v, **kw), exact, dtype)
    assert found < LIMIT, found
    trained = attention(*(t.detach().requires_grad_() for t in (q, k, v)), **kw).detach()
    assert off(trained, exact, dtype) < LIMIT


@pytest.mark.parametrize('kind', ('none', 'pairs', 'causal', 'padding'))
@pytest.mark.parametrize('shape', SHAPES, ids=str)
@pytest.mark.parametrize('dtype', HALVES, ids=str)
def test_rest_is_what_rounding_took(cuda, dtype, shape, kind):
    """The forward that a backward follows leaves its result in two 16-bit parts: together within u / 16 of float64 (by
    the same count as above), where the result alone is at 0.29 u at best."""
    q, k, v, _ = inputs(shape, dtype, 42)
    kw = masks(kind, shape, 42)
    _, tensors, _ = _native.attention_forward(q, k, v, kw['key_padding_mask'], kw['attn_mask'], kw['causal'],
                                              shape[5] ** -0.5, for_backward=True)
    out, rest = tensors[5], tensors[6]
    exact = attention_exact(q, k, v, **kw)[0][0]
    if not exact.any():
        assert not out.any() and not rest.any()
        return
    assert (out.double() + rest.double() - exact).norm() / exact.norm() < U[dtype] / 16
    assert (out.double() - exact).norm() / exact.norm() > U[dtype] / 4


@pytest.mark.parametrize('kind', ('none', 'pairs', 'causal', 'padding'))
@pytest.mark.parametrize('shape', SHAPES, ids=str)
@pytest.mark.parametrize('dtype', HALVES, ids=str)
def test_only_the_gradients_are_rounded(cuda, dtype, shape, kind):
    q, k, v, grad = inputs(shape, dtype, 43)
    kw = masks(kind, shape, 43)
    for name, got, want in zip(NAMES, run(q, k, v, grad, **kw), attention_exact(q, k, v, grad=grad, **kw)):
        found = off(got, want[0], dtype)
        assert found < LIMIT, (name, found)


@pytest.mark.parametrize('shape', [(2, 300, 1100, 4, 4, 32), (3, 260, 300, 4, 2, 64), (2, 140, 400, 2, 1, 128),
                                   (2, 300, 4200, 2, 2, 32)], ids=str)
@pytest.mark.parametrize('dtype', HALVES, ids=str)
def test_gradients_of_mixed_size(cuda, dtype, shape):
    """A row, a head and an image whose incoming gradients are 2^12 times the others', and an image with a value 2^8
    times the others: the small rows' gradients are as good as if they were alone."""
    q, k, v, grad = inputs(shape, dtype, 44)
    B, Q, N, H, Hk, D = shape
    grad = (grad / 2).view(B, Q, H, D).clone()
    small_q = torch.ones((B, Q, H), dtype=torch.bool, device='cuda')
    small_k = torch.ones((B, N, Hk), dtype=torch.bool, device='cuda')
    small_q[0, 5], small_k[0] = False, False  # a row, which every key of its image has a share of
    small_q[1, :, H - 1], small_k[1, :, Hk - 1] = False, False  # a head
    if B > 2:
        small_q[2], small_k[2] = False, False  # an image
    grad = torch.where(small_q[..., None], grad, grad.float().mul(2.0 ** 12).clamp(-30000, 30000).to(dtype))
    for spread in (1.0, 2.0 ** 8):
        v = v.clone()
        v[0, N // 2] *= spread
        got = run(q, k, v, grad.view(B, Q, H * D))
        want = attention_exact(q, k, v, grad=grad.view(B, Q, H * D))
        for name, a, (b, _), small in zip(NAMES[1:], got[1:], want[1:], (small_q, small_k, small_k)):
            if small.any():
                found = off(a[small], b[small], dtype)
                assert found < LIMIT, (name, spread, found)
            found = off(a, b, dtype)
            assert found < LIMIT, (name, spread, found)


@pytest.mark.parametrize('shape', [(1, 500, 20000, 1, 1, 32), (1, 300, 60000, 1, 1, 64)], ids=str)
@pytest.mark.parametrize('dtype', HALVES, ids=str)
def test_gradients_over_very_long_keys(cuda, dtype, shape):
    """Probabilities near float16's smallest normal number and below (1 / 60000 = 1.7e-5 against 6.1e-5)."""
    q, k, v, grad = inputs(shape, dtype, 45)
    for name, got, want in zip(NAMES, run(q, k, v, grad * 40), attention_exact(q, k, v, grad=grad * 40)):
        found = off(got, want[0], dtype)
        assert found < LIMIT, (name, found)


@pytest.mark.parametrize('kind', ('none', 'pairs', 'causal'))
@pytest.mark.parametrize('shape', SHAPES, ids=str)
@pytest.mark.parametrize('dtype', HALVES, ids=str)
def test_gradients_behind_large_results(cuda, dtype, shape, kind):
    """Values around 16 that differ by about one: what is left of dP - delta is a sixteenth of either, so that a delta
    from rounded results, without what rounding took from them, puts the queries' gradient 20 to 120 times as far off as
    its own rounding does.

    What is allowed follows the result's error into them. A result that is off by a relative x moves delta_i by at most
    t_i = x sum|do_i o_i|, and with it dq_i by scale t_i sum_j P_ij k_j and dk_j by scale sum_i P_ij t_i q_i. Here x is
    u^2 for the result's two parts, u^2 for those of P, and the tensor core's cuts of a sum of values that all have one
    sign: 2^-24 of it for each of two groups of 8 in the 16 terms of a product, so N 2^-24 / 8 for one part of P (the
    other adds u of that)."""
    q, k, v, grad = inputs(shape, dtype, 46)
    v = v + 16
    kw = masks(kind, shape, 46)
    B, Q, N, H, Hk, D = shape
    x, G, scale = 2 * U[dtype] ** 2 + N * 2.0 ** -24 / 8 * (1 + U[dtype]), H // Hk, D ** -0.5
    exact = attention_exact(q, k, v, grad=grad, **kw)
    wide_q, wide_k = q.double().transpose(1, 2), k.double().transpose(1, 2).repeat_interleave(G, 1)
    scores = (wide_q @ wide_k.transpose(2, 3) * scale).masked_fill(
        blocked_pairs(B, Q, N, kw['key_padding_mask'], kw['attn_mask'], kw['causal'], q.device), -float('inf'))
    p = scores.softmax(3).nan_to_num(0.0)
    t = x * (grad.double() * exact[0][0]).abs().view(B, Q, H, D).sum(3).transpose(1, 2)[..., None]
    moved = {'grad_query': scale * t * (p @ wide_k),
             'grad_key': scale * (p.transpose(2, 3) @ (t * wide_q.abs())).view(B, Hk, G, N, D).sum(2)}
    for name, got, (want, _) in zip(NAMES, run(q, k, v, grad, **kw), exact):
        own, found = (want.to(dtype).double() - want).norm().item(), off(got, want, dtype)
        allowed = moved[name].norm().item() / own if name in moved and own > 0 else 0.0
        assert found < LIMIT + allowed, (name, found, allowed)


@pytest.mark.parametrize('kind', ('none', 'pairs', 'causal'))
@pytest.mark.parametrize('N', (2, 3, 5, 8, 17, 32, 33))
@pytest.mark.parametrize('D', (16, 32, 64, 128))
@pytest.mark.parametrize('dtype', HALVES, ids=str)
def test_gradients_of_few_keys(cuda, dtype, D, N, kind):
    """Sums of few terms, where a factor rounded to 16 bits would show in each. Where one key has all the weight, what
    is left of dP - delta is small against both and off by what test_gradients_behind_large_results counts: a few u^2 of
    sum|do_i v_j| for each pair, in proportion to its probability."""
    shape = (2, 150, N, 4, 2, D)
    q, k, v, grad = inputs(shape, dtype, 47)
    kw = masks(kind, shape, 47)
    B, Q, _, H, Hk, _ = shape
    exact = attention_exact(q, k, v, grad=grad, **kw)
    G, scale, x = H // Hk, D ** -0.5, 4 * U[dtype] ** 2 + 16 * 2.0 ** -24
    wide_q, wide_k, wide_v = (t.double().transpose(1, 2) for t in (q, k, v))
    wide_k, wide_v = wide_k.repeat_interleave(G, 1), wide_v.repeat_interleave(G, 1)
    scores = (wide_q @ wide_k.transpose(2, 3) * scale).masked_fill(
        blocked_pairs(B, Q, N, kw['key_padding_mask'], kw['attn_mask'], kw['causal'], q.device), -float('inf'))
    p = scores.softmax(3).nan_to_num(0.0)
    do = grad.double().view(B, Q, H, D).transpose(1, 2)
    t = x * p * (do.abs() @ wide_v.abs().transpose(2, 3)).amax(3, keepdim=True)
    moved = {'grad_query': scale * (t @ wide_k.abs()),
             'grad_key': scale * (t.transpose(2, 3) @ wide_q.abs()).view(B, Hk, G, N, D).sum(2)}
    for name, got, (want, _) in zip(NAMES, run(q, k, v, grad, **kw), exact):
        own, found = (want.to(dtype).double() - want).norm().item(), off(got, want, dtype)
        allowed = moved[name].norm().item() / own if name in moved and own > 0 else 0.0
        assert found < LIMIT + allowed, (name, found, allowed)
