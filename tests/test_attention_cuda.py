"""attention on the GPU, forward and backward, against float64 with counted error bounds: every dtype, head layout and
mask, lengths from one, strided views, streams and graphs."""

import pytest
import torch

from attention_oracle import attention_exact, check
from marearts_tinydeform_b200 import _native, attention

pytestmark = pytest.mark.gpu

DTYPES = (torch.float32, torch.float16, torch.bfloat16, torch.float64)
# B, Q, N, H, Hk, D: one token; fewer than a tile; the decoder's; grouped heads; a tile exactly and one more; widths
# that are no power of two, and no multiple of a 16-byte vector; one and few queries over long keys; one key
SHAPES = [(1, 1, 1, 1, 1, 32), (2, 7, 5, 4, 2, 16), (1, 300, 300, 8, 8, 32), (2, 129, 257, 4, 1, 64),
          (1, 128, 128, 2, 2, 128), (2, 200, 333, 6, 3, 24), (1, 130, 70, 2, 1, 20), (3, 2, 1000, 8, 4, 32),
          (1, 65, 1, 2, 2, 64), (2, 257, 129, 4, 2, 128), (2, 1, 2500, 4, 1, 64), (1, 9, 700, 3, 1, 96),
          (1, 1, 4097, 16, 2, 128), (2, 448, 640, 2, 2, 40), (2, 9, 1500, 6, 2, 32), (1, 40, 2100, 2, 2, 72),
          (2, 260, 300, 4, 2, 60), (1, 300, 390, 2, 1, 124)]
MASKS = ('none', 'padding', 'pairs', 'pairs-all', 'causal', 'everything')
NAMES = ('out', 'grad_query', 'grad_key', 'grad_value')


def inputs(shape, dtype, seed=0, device='cuda'):
    B, Q, N, H, Hk, D = shape
    g = torch.Generator(device=device).manual_seed(seed)
    q, k, v = (torch.randn(s, generator=g, device=device).to(dtype)
               for s in ((B, Q, H, D), (B, N, Hk, D), (B, N, Hk, D)))
    return q, k, v, (torch.randn((B, Q, H * D), generator=g, device=device) * 0.1).to(dtype)


def masks(kind, shape, seed=0, device='cuda'):
    B, Q, N, H, _, _ = shape
    g = torch.Generator(device=device).manual_seed(1000 + seed)
    pad = pairs = None
    if kind in ('padding', 'everything'):
        left = torch.randint(0, N + 1, (B,), generator=g, device=device)
        left[0] = 0 if B > 1 else N // 2  # an image without any key
        pad = torch.arange(N, device=device)[None, :] >= left[:, None]
    if kind == 'pairs':
        pairs = torch.rand((Q, N), generator=g, device=device) < 0.6
        pairs[Q // 2] = True  # a row that is left nothing
    if kind in ('pairs-all', 'everything'):
        pairs = torch.rand((B, H, Q, N), generator=g, device=device) < 0.5
        pairs[:, :, :, N // 3:N // 3 + 150] = True  # whole tiles blocked
    return dict(key_padding_mask=pad, attn_mask=pairs, causal=kind in ('causal', 'everything'))


def run(q, k, v, grad, **kw):
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = attention(*leaves, **kw)
    return [out.detach()] + list(torch.autograd.grad(out, leaves, grad))


@pytest.mark.parametrize('kind', MASKS)
@pytest.mark.parametrize('shape', SHAPES, ids=str)
@pytest.mark.parametrize('dtype', DTYPES, ids=str)
def test_attention(cuda, dtype, shape, kind):
    q, k, v, grad = inputs(shape, dtype)
    kw = masks(kind, shape)
    exact = attention_exact(q, k, v, grad=grad, **kw)
    with torch.inference_mode():
        check(attention(q, k, v, **kw), exact[0], 'out (inference)')
    for name, got, want in zip(NAMES, run(q, k, v, grad, **kw), exact):
        check(got, want, name)
    assert _native.device_error() == 0


# calls of few long rows of work: the forward shares a query tile's keys among CTAs (splits that end inside a tile, and
# of which masks leave some nothing), the backward shares a tile's queries (those of a whole group, too) or keys
@pytest.mark.parametrize('kind', MASKS)
@pytest.mark.parametrize('shape', [(1, 140, 1700, 4, 2, 32), (2, 300, 2049, 2, 1, 128), (1, 1300, 100, 8, 1, 32),
                                   (1, 3, 2600, 2, 2, 64), (1, 900, 20, 3, 1, 48)], ids=str)
@pytest.mark.parametrize('dtype', DTYPES, ids=str)
def test_shared_rows_of_work(cuda, dtype, shape, kind):
    q, k, v, grad = inputs(shape, dtype, 21)
    kw = masks(kind, shape, 21)
    if kind in ('padding', 'pairs'):  # a whole split, and more, without a key
        if kind == 'padding':
            kw['key_padding_mask'][-1, shape[2] // 4:shape[2] * 3 // 4] = True
        else:
            kw['attn_mask'][:, :shape[2] * 2 // 3] = True
    exact = attention_exact(q, k, v, grad=grad, **kw)
    with torch.inference_mode():
        check(attention(q, k, v, **kw), exact[0], 'out (inference)')
    first = run(q, k, v, grad, **kw)
    for name, got, want in zip(NAMES, first, exact):
        check(got, want, name)
    for name, got, again in zip(NAMES, first, run(q, k, v, grad, **kw)):
        assert torch.equal(got, again), name
    assert _native.device_error() == 0


@pytest.mark.parametrize('dtype', (torch.float16, torch.bfloat16), ids=str)
def test_cuda_core_kernels(policy, dtype):
    shape = (2, 150, 200, 4, 2, 64)
    q, k, v, grad = inputs(shape, dtype, 3)
    kw = masks('everything', shape, 3)
    for name, got, want in zip(NAMES, run(q, k, v, grad, **kw), attention_exact(q, k, v, grad=grad, **kw)):
        check(got, want, f'{policy} {name}')


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
def test_packed_and_strided_views(cuda, dtype):
    g = torch.Generator(device='cuda').manual_seed(5)
    packed = torch.randn((2, 190, 3, 4, 32), generator=g, device='cuda').to(dtype)
    q, k, v = packed.unbind(2)
    grad = torch.randn((2, 190, 128), generator=g, device='cuda').to(dtype)
    exact = attention_exact(q, k, v, grad=grad)
    for name, got, want in zip(NAMES, run(q, k, v, grad), exact):
        check(got, want, f'packed {name}')
    # head-major storage, an odd storage offset, a reversed innermost layout, one shared key head
    forms = [tuple(t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)),
             tuple(torch.cat([t.new_zeros(1), t.reshape(-1)])[1:].view(t.shape) for t in (q, k, v)),
             tuple(t.transpose(2, 3).contiguous().transpose(2, 3) for t in (q, k, v))]
    for i, form in enumerate(forms):
        for name, got, want in zip(NAMES, run(*form, grad), exact):
            check(got, want, f'form {i} {name}')
    shared = (q, k[:, :, :1].expand(2, 190, 4, 32), v[:, :, :1].expand(2, 190, 4, 32))
    for name, got, want in zip(NAMES, run(*shared, grad), attention_exact(*shared, grad=grad)):
        check(got, want, f'expanded {name}')
    # a transposed gradient
    strided = grad.transpose(0, 1).contiguous().transpose(0, 1)
    for name, got, want in zip(NAMES, run(q, k, v, strided), exact):
        check(got, want, f'strided gradient {name}')


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('Q', (1, 140))
def test_padded_keys_may_hold_anything(cuda, dtype, Q):
    shape = (2, Q, 300, 4, 2, 32)
    q, k, v, grad = inputs(shape, dtype, 7)
    pad = torch.zeros((2, 300), dtype=torch.bool, device='cuda')
    pad[0, 170:] = True
    pad[1, ::3] = True
    want = run(q, k, v, grad, key_padding_mask=pad)
    for junk in (float('nan'), float('inf'), -float('inf')):
        kj, vj = (t.masked_fill(pad[:, :, None, None], junk) for t in (k, v))
        for name, got, ref in zip(NAMES, run(q, kj, vj, grad, key_padding_mask=pad), want):
            assert torch.equal(got, ref), f'{name} with {junk} in padded rows'


@pytest.mark.parametrize('shape', [(1, 40, 300, 2, 2, 32), (2, 70, 333, 4, 2, 64), (1, 20, 270, 1, 1, 128),
                                   (1, 33, 90, 2, 2, 32), (1, 5, 700, 2, 1, 64), (1, 130, 1700, 2, 1, 24)], ids=str)
@pytest.mark.parametrize('dtype', DTYPES, ids=str)
def test_keys_at_infinity(cuda, dtype, shape):
    """A key whose score is minus infinity for every query has no probability: results are those of a call that pads
    it."""
    q, k, v, _ = inputs(shape, dtype, 14)
    q[..., 0] = q[..., 0].abs() + 0.25
    pad = torch.zeros((shape[0], shape[2]), dtype=torch.bool, device='cuda')
    for j in (0, 7, shape[2] // 2, shape[2] - 1):
        k[:, j, :, 0] = -float('inf')
        pad[:, j] = True
    exact = attention_exact(q, k, v, key_padding_mask=pad)[0]
    with torch.inference_mode():
        check(attention(q, k, v), exact, 'out (inference)')
    check(attention(*(t.detach().requires_grad_() for t in (q, k, v))).detach(), exact, 'out')


@pytest.mark.parametrize('causal', (False, True))
@pytest.mark.parametrize('shape', [(1, 40, 300, 2, 2, 32), (2, 70, 333, 4, 2, 64), (1, 20, 270, 1, 1, 128),
                                   (1, 33, 90, 2, 2, 32), (1, 5, 700, 2, 1, 64), (1, 130, 1700, 2, 1, 24),
                                   (2, 40, 20, 2, 2, 32)], ids=str)
@pytest.mark.parametrize('dtype', DTYPES, ids=str)
def test_gradients_with_keys_at_infinity(cuda, dtype, shape, causal):
    """Such keys' gradients are zero and they take no part in the others', but for the queries' in the infinite column
    (zero times infinity)."""
    q, k, v, grad = inputs(shape, dtype, 15)
    q[..., 0] = q[..., 0].abs() + 0.25
    pad = torch.zeros((shape[0], shape[2]), dtype=torch.bool, device='cuda')
    for j in (0, 7, shape[2] // 2, shape[2] - 1):
        k[:, j, :, 0] = -float('inf')
        pad[:, j] = True
    exact = attention_exact(q, k, v, key_padding_mask=pad, grad=grad, causal=causal)
    got = run(q, k, v, grad, causal=causal)
    B, Q, H, D = q.shape
    exact[1], got[1] = [t.view(B, Q, H, D)[..., 1:] for t in exact[1]], got[1][..., 1:]
    for name, a, b in zip(NAMES, got, exact):
        check(a, b, name)


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
def test_rows_without_keys_are_zero(cuda, dtype):
    shape = (2, 131, 90, 4, 4, 32)
    q, k, v, grad = inputs(shape, dtype, 8)
    pairs = torch.zeros((131, 90), dtype=torch.bool, device='cuda')
    pairs[5] = True
    pairs[128:] = True
    out, dq, dk, dv = run(q, k, v, grad, attn_mask=pairs)
    assert not out[:, 5].any() and not out[:, 128:].any() and not dq[:, 5].any() and not dq[:, 128:].any()
    pairs[:] = True
    assert not any(t.any() for t in run(q, k, v, grad, attn_mask=pairs))
    # more queries than keys under the causal rule: the first Q - N queries have none
    out, dq, _, _ = run(q, k, v, grad, causal=True)
    assert not out[:, :41].any() and not dq[:, :41].any() and out[:, 41].any()


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
def test_large_and_small_magnitudes(cuda, dtype):
    """Sharp rows (scores in the hundreds), a large offset that every key shares, and gradients near the type's
    smallest and largest numbers."""
    shape = (1, 200, 260, 2, 2, 64)
    q, k, v, grad = inputs(shape, dtype, 9)
    cases = [(q * 8, k * 8, v, grad), (q, k + 20, v, grad), (q, k, v * 50, grad * 100)]
    cases.append((q, k, v, grad * (2.0 ** -10 if dtype == torch.float16 else 2.0 ** -60)))
    cases.append((q, k, v * 64, grad * 2000))
    for i, (a, b, c, d) in enumerate(cases):
        for name, got, want in zip(NAMES, run(a, b, c, d), attention_exact(a, b, c, grad=d)):
            check(got, want, f'case {i} {name}')


@pytest.mark.parametrize('dtype', (torch.float32, torch.float16, torch.bfloat16), ids=str)
def test_same_bits_every_time(cuda, dtype):
    shape = (2, 333, 410, 8, 2, 64)
    q, k, v, grad = inputs(shape, dtype, 10)
    kw = masks('everything', shape, 10)
    first = run(q, k, v, grad, **kw)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, run(q, k, v, grad, **kw)))


def test_gradients_against_differences(cuda):
    """float64, by central differences, with shared heads and an expanded key."""
    torch.manual_seed(0)
    q, k, v = (torch.randn(s, dtype=torch.float64, device='cuda', requires_grad=True)
               for s in ((2, 5, 4, 3), (2, 6, 2, 3), (2, 6, 2, 3)))
    pad = torch.zeros((2, 6), dtype=torch.bool, device='cuda')
    pad[1, 4:] = True
    assert torch.autograd.gradcheck(lambda a, b, c: attention(a, b, c, key_padding_mask=pad, causal=True), (q, k, v))
    assert torch.autograd.gradcheck(lambda a, b: attention(a, b.expand(2, 6, 2, 3), b.expand(2, 6, 2, 3)),
                                    (q, k[:, :1].detach().requires_grad_()))


@pytest.mark.parametrize('shape', [(2, 300, 300, 8, 8, 32), (4, 1, 5000, 8, 2, 64)], ids=str)
@pytest.mark.parametrize('dtype', (torch.float32, torch.float16), ids=str)
def test_graph_capture_and_streams(cuda, dtype, shape):
    """Two captured graphs replayed at once on two streams, on inputs rewritten in place, against plain calls."""
    B, Q, N = shape[:3]
    runs = []
    pad = torch.arange(N, device='cuda')[None, :] >= torch.tensor([N, N // 2] * (B // 2), device='cuda')[:, None]
    pairs = torch.rand((Q, N), device='cuda') < 0.3
    for seed in (1, 2):
        stream = torch.cuda.Stream()
        q, k, v, grad = inputs(shape, dtype, seed)
        leaves = [t.requires_grad_() for t in (q, k, v)]
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            for _ in range(2):
                out = attention(*leaves, key_padding_mask=pad, attn_mask=pairs)
                torch.autograd.grad(out, leaves, grad)
                del out
            graph = torch.cuda.CUDAGraph()
            stream.synchronize()
            with torch.cuda.graph(graph, stream=stream):
                out = attention(*leaves, key_padding_mask=pad, attn_mask=pairs)
                grads = torch.autograd.grad(out, leaves, grad)
        runs.append((stream, graph, leaves, grad, [out.detach(), *grads]))
    torch.cuda.synchronize()
    for seed in (3, 4):
        for stream, graph, leaves, grad, _ in runs:
            fresh = inputs(shape, dtype, seed)
            with torch.no_grad():
                for t, x in zip((*leaves, grad), fresh):
                    t.copy_(x)
        torch.cuda.synchronize()
        for stream, graph, *_ in runs:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        q, k, v, grad = inputs(shape, dtype, seed)
        want = run(q, k, v, grad, key_padding_mask=pad, attn_mask=pairs)
        for *_, got in runs:
            for name, a, b in zip(NAMES, got, want):
                assert torch.equal(a, b), name


def test_offsets_beyond_32_bits(cuda):
    """Images more than 2^31 elements apart in one buffer (4.4 GB), read in place."""
    gap = 2 ** 31 + 4096
    buf = torch.empty(gap + 3 * 70 * 64, dtype=torch.float16, device='cuda')
    q, k, v = (buf[i * 70 * 64:].as_strided((2, 70, 2, 32), (gap, 64, 32, 1)) for i in range(3))
    ref = inputs((2, 70, 70, 2, 2, 32), torch.float16, 11)
    for t, x in zip((q, k, v), ref):
        t.copy_(x)
    for name, got, want in zip(NAMES, run(q, k, v, ref[3]), run(*ref)):
        assert torch.equal(got, want), name


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
def test_one_key_has_no_gradient_through_the_scores(cuda, dtype):
    """The probability of an only key is one whatever the scores: gradients of query and key are exactly zero."""
    for shape in ((2, 1, 1, 4, 2, 32), (1, 70, 1, 2, 2, 128), (3, 5, 1, 2, 1, 20)):
        q, k, v, grad = inputs(shape, dtype, 13)
        out, dq, dk, _ = run(q * 5, k, v, grad)
        assert not dq.any() and not dk.any()
        G = shape[3] // shape[4]
        want = v.repeat_interleave(G, 2).expand(shape[0], shape[1], shape[3], shape[5]).reshape(out.shape)
        assert torch.equal(out, want)


def test_no_queries_no_keys(cuda):
    for dtype in DTYPES:
        q, k, v, grad = inputs((2, 0, 5, 2, 2, 32), dtype)
        out, dq, dk, dv = run(q, k, v, grad)
        assert out.shape == (2, 0, 64) and dq.shape == q.shape and not dk.any() and not dv.any()
        q, k, v, grad = inputs((2, 5, 0, 2, 2, 32), dtype)
        out, dq, dk, dv = run(q, k, v, grad)
        assert not out.any() and not dq.any() and dk.shape == k.shape
        q, k, v, grad = inputs((0, 5, 4, 2, 2, 32), dtype)
        assert run(q, k, v, grad)[0].shape == (0, 5, 64)


def test_partial_gradients(cuda):
    q, k, v, grad = inputs((1, 40, 50, 2, 2, 32), torch.float16, 12)
    want = run(q, k, v, grad)
    k2 = k.detach().requires_grad_()
    got, = torch.autograd.grad(attention(q, k2, v), [k2], grad)
    assert torch.equal(got, want[2])
    with pytest.raises(RuntimeError):  # no second derivative: refused, not wrong
        x = q.detach().requires_grad_()
        g, = torch.autograd.grad(attention(x, k, v), [x], grad, create_graph=True)
        g.sum().backward()


@pytest.mark.parametrize('shape', [(2, 1100, 1100, 8, 8, 32), (1, 300, 4200, 4, 4, 32), (1, 700, 1000, 8, 2, 64),
                                   (1, 300, 1000, 4, 1, 128)], ids=str)
def test_float32_is_float32_over_long_keys(cuda, shape):
    """Over whole results, not elements: what roundings leave there does not grow with the keys. Standard normal inputs
    have scores of about one, and a product of three TF32 ones is off by up to 2^-22 of it, the tensor core's cut sums
    (one a group of 8, up to 16 for D = 128) by another 16 x 2^-24 on average: 2^-19.7 in the probabilities; a tile's
    sums add 8 x 2^-24 and its join 2^-24 for each of the tiles, in either direction. Together below 2^-19; sums cut
    over all keys instead would be off by keys / 8 x 3 x 2^-24 on the way, 2.5e-5 here."""
    q, k, v, grad = inputs(shape, torch.float32, 31)
    for name, got, want in zip(NAMES, run(q, k, v, grad), attention_exact(q, k, v, grad=grad)):
        want = want[0] if isinstance(want, tuple) else want
        error = float((got.double() - want).norm() / want.norm())
        assert error < 2.0 ** -19, (name, error)


@pytest.mark.parametrize('causal', (False, True))
@pytest.mark.parametrize('padded', (False, True))
@pytest.mark.parametrize('shape', [(2, 150, 210, 4, 2, 32), (3, 3, 1500, 2, 1, 64)], ids=str)
@pytest.mark.parametrize('dtype', DTYPES, ids=str)
def test_mask_layouts(cuda, dtype, shape, padded, causal):
    """Masks shared by images or heads, expanded, sliced, transposed and of any nonzero bytes, against the same pairs
    written out as a dense [B, H, Q, N] mask: the same bits."""
    B, Q, N, H, _, _ = shape
    q, k, v, grad = inputs(shape, dtype, 51)
    g = torch.Generator(device='cuda').manual_seed(52)
    kw = dict(causal=causal, key_padding_mask=masks('padding', shape, 51)['key_padding_mask'] if padded else None)

    def some(*s):
        m = torch.rand(s, generator=g, device='cuda') < 0.5
        m[..., N // 3:N // 3 + 140] = True
        return m

    wide = some(B, H, Q + 3, N + 13)
    layouts = {'[Q, N]': some(Q, N), '[1, 1, Q, N]': some(1, 1, Q, N), '[B, 1, Q, N]': some(B, 1, Q, N),
               '[1, H, Q, N]': some(1, H, Q, N), 'images expanded': some(1, H, Q, N).expand(B, H, Q, N),
               'heads expanded': some(B, 1, Q, N).expand(B, H, Q, N), 'both expanded': some(Q, N).expand(B, H, Q, N),
               'queries expanded': some(B, H, 1, N).expand(B, H, Q, N), 'one row for all': some(1, N).expand(Q, N),
               'sliced': wide[:, :, 2:Q + 2, 5:N + 5], 'sliced [Q, N]': wide[0, 0, 2:Q + 2, 5:N + 5],
               'every other image': some(2 * B, H, Q, N)[::2], 'heads innermost': some(B, Q, H, N).transpose(1, 2),
               'transposed': some(B, H, Q, N).transpose(2, 3).contiguous().transpose(2, 3),
               'keys expanded': (torch.rand((Q, 1), generator=g, device='cuda') < 0.3).expand(Q, N)}
    for name, m in layouts.items():
        dense = m.expand(B, H, Q, N).contiguous()
        want = run(q, k, v, grad, attn_mask=dense, **kw)
        any_byte = m.to(torch.uint8) * 2 if m.dim() == 2 else torch.where(m, 255, 0).to(torch.uint8)
        for form in (m, any_byte):
            for part, a, b in zip(NAMES, run(q, k, v, grad, attn_mask=form, **kw), want):
                assert torch.equal(a, b), (name, form.dtype, part)
