"""rms_norm, linear_fp8 and the 8-bit conversions without a GPU: the CPU path against float64, refusals, and the C ABI's
argument checks."""

import ctypes
import os

import pytest
import torch

from attention_oracle import check
from fp8_oracle import (E4M3, check_quantized, linear_train_exact, product_exact, quantized, rms_norm_exact, through,
                        worth)
from marearts_tinydeform_b200 import (_native, build, dequantize_fp8, linear_fp8, quantize_fp8, quantize_weight_fp8,
                                      rms_norm)

DTYPES = (torch.float32, torch.float16, torch.bfloat16)


@pytest.fixture(scope='module')
def lib():
    build.build()
    return _native.load()


def normal(*shape, dtype=torch.float32, seed=0, std=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype)


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('shape', [(1, 1), (3, 128), (5, 129), (130, 300)], ids=str)
def test_quantize_reference(dtype, shape):
    x = normal(*shape, dtype=dtype) * torch.exp2(normal(shape[0], 1, dtype=dtype, seed=1) * 4).to(dtype)
    x[0, 0] = 0
    for make, rows in ((quantize_fp8, 1), (quantize_weight_fp8, 128)):
        data, scale = make(x)
        q, s = quantized(x, rows, 128)
        assert data.dtype == E4M3 and torch.equal(data.double(), q) and torch.equal(scale.double(), s)
        assert torch.equal(dequantize_fp8(data, scale, torch.float32).double(), worth(q, s, rows, 128))


def test_quantize_edges():
    x = torch.zeros(6, 130)
    x[1, 3], x[1, 129] = 448.0, 449.0
    x[2, :3] = torch.tensor([float('inf'), float('nan'), 7.0])
    x[3, 0] = 3.4e38
    x[4, 0] = 1e-40
    x[5, :4] = torch.tensor([17.0, 19.0, 21.0, -23.0])  # between 16, 18, 20, 22 and 24: ties go to even
    x[5, 4] = 448.0
    data, scale = quantize_fp8(x)
    q, s = quantized(x, 1, 128)
    assert torch.equal(data.double().nan_to_num(nan=-1), q.nan_to_num(nan=-1)) and torch.equal(scale.double(), s)
    assert scale[1].tolist() == [1.0, 2.0] and scale[0].tolist() == [2.0 ** -126] * 2
    assert data[2].double().isnan().sum() == 2 and scale[2, 0] == 2.0 ** -6
    assert data[5, :4].tolist() == [16.0, 20.0, 20.0, -24.0]
    assert quantize_fp8(x[0])[1].shape == (2,) and quantize_fp8(x[:0])[0].shape == (0, 130)


@pytest.mark.parametrize('dtype', (*DTYPES, torch.float64), ids=str)
def test_rms_norm_reference(dtype):
    x, r, dy, ds = (normal(6, 133, dtype=dtype, seed=i) for i in range(4))
    w = normal(133, dtype=dtype, seed=5)
    leaves = [t.detach().requires_grad_() for t in (x, w, r)]
    y, s = rms_norm(*leaves, return_sum=True)
    got = [y.detach(), s.detach()] + list(torch.autograd.grad((y, s), leaves[:2], (dy, ds)))
    exact = rms_norm_exact(x, w, r, grad=dy, grad_sum=ds)
    for a, e in zip(got, exact):
        check(a, e, 'rms norm')
    if dtype != torch.float64:
        with torch.no_grad():
            check_quantized(rms_norm(x, w, r, quantize=True), exact[0], 'rms norm in 8 bits')


@pytest.mark.parametrize('dtype', DTYPES, ids=str)
def test_linear_reference(dtype):
    x, w, b, g = normal(2, 33, 200, dtype=dtype), normal(140, 200, dtype=dtype, seed=1), \
        normal(140, dtype=dtype, seed=2), normal(2, 33, 140, dtype=dtype, seed=3)
    rows = x.view(66, 200)
    for act in (None, 'relu', 'gelu', 'silu'):
        exact = product_exact(through(rows, 1, 128), through(w, 128, 128), dtype, b, act)
        check(linear_fp8(x, w, b, activation=act).view(66, 140), exact, act)
        check(linear_fp8(quantize_fp8(x), quantize_weight_fp8(w), b, act, dtype=dtype).view(66, 140), exact, act)
        check_quantized(linear_fp8(x, quantize_weight_fp8(w), b, act, quantize=True), exact, act)
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    y = linear_fp8(*leaves)
    got = [y.detach().view(66, 140)] + list(torch.autograd.grad(y, leaves, g))
    got[1] = got[1].view(66, 200)
    for a, e in zip(got, linear_train_exact(rows, w, b, g.view(66, 140))):
        check(a, e, 'training')


def test_activations_keep_their_digits():
    """The lower tails of GELU and SiLU, to two roundings of float32 (computed in 64 bits, rounded once, compared)."""
    v = torch.cat([torch.linspace(-13, 13, 200), torch.tensor([-100., -90, -88.5, -40, -20])])
    w8 = quantize_weight_fp8(torch.zeros(v.numel(), 128))
    d = v.double()
    for act, want in (('gelu', 0.5 * d * torch.erfc(-d / 2 ** 0.5)), ('silu', d * torch.sigmoid(d))):
        off = (linear_fp8(torch.ones(1, 128), w8, v, act)[0].double() - want).abs()
        assert (off <= 2.0 ** -23 * want.abs() + 2.0 ** -149).all(), act


def test_linear_gradients_against_differences():
    """Small whole numbers survive the rounding to 8 bits, so the product is its own formula and linear in each
    operand: differences over a step of 1 are its gradients, exactly."""
    gen = torch.Generator().manual_seed(7)
    x, w, g = (torch.randint(-4, 5, s, generator=gen).float() for s in ((5, 9), (4, 9), (5, 4)))
    b = torch.randint(-4, 5, (4,), generator=gen).float()
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(linear_fp8(*leaves), leaves, g)
    for k in range(3):
        for i in range(leaves[k].numel()):
            moved = [t.clone() for t in (x, w, b)]
            moved[k].view(-1)[i] += 1
            slope = ((linear_fp8(*moved) - linear_fp8(x, w, b)) * g).sum()
            assert slope == grads[k].reshape(-1)[i]


def keeps_what_its_gradients_read(device):
    """Each gradient alone: what the graph holds until the backward, and that the operand which the gradient does not
    read may change in between."""
    gen = torch.Generator().manual_seed(3)
    x, w, b, g = (torch.randint(-4, 5, s, generator=gen).float().to(device) for s in ((6, 20), (7, 20), (7,), (6, 7)))
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    want = torch.autograd.grad(linear_fp8(*leaves), leaves, g)
    for k, held in enumerate(([torch.float32], [E4M3, torch.float32], [])):
        only = [t.clone().requires_grad_(i == k) for i, t in enumerate((x, w, b))]
        y = linear_fp8(*only)
        assert [t.dtype for t in y.grad_fn.saved_tensors if t is not None] == held
        with torch.no_grad():
            for i, t in enumerate(only):
                if i != 1 or k != 0:
                    t.zero_()
        assert torch.equal(torch.autograd.grad(y, only[k], g)[0], want[k])


def test_the_graph_keeps_what_its_gradients_read():
    keeps_what_its_gradients_read('cpu')


def test_rms_norm_refusals():
    x, w = torch.zeros(3, 8), torch.ones(8)
    for args, kw, message in [((x, w[:7]), {}, 'weight'), ((x, w, x[:2]), {}, 'residual'),
                              ((x, w.double()), {}, 'device and dtype'), ((x, w, None, -1.0), {}, 'eps'),
                              ((x.int(), w), {}, 'unsupported dtype'), ((torch.zeros(()), w), {}, 'one dimension'),
                              ((torch.zeros(2, 8193), torch.zeros(8193)), {}, 'channels'),
                              ((x.double(), w.double()), dict(quantize=True), '8-bit result needs'),
                              ((x.clone().requires_grad_(), w), dict(quantize=True), 'no gradient')]:
        with pytest.raises(RuntimeError, match=message):
            rms_norm(*args, **kw)


def test_linear_refusals():
    x, w, b = torch.zeros(3, 200), torch.zeros(150, 200), torch.zeros(150)
    x8, w8 = quantize_fp8(x), quantize_weight_fp8(w)
    wg = w.clone().requires_grad_()
    good = dict(x=x, weight=w8, bias=b)
    linear_fp8(**good)
    for change, message in [
            (dict(x=x.double()), 'float32, float16 or bfloat16'), (dict(x=torch.zeros(())), 'one dimension'),
            (dict(x=x[:, :199]), 'last dimension of x'), (dict(x=torch.zeros(3, 0)), 'between 1 and'),
            (dict(x=x8), 'needs the dtype'), (dict(x=(x8[0], x8[1].double()), dtype=torch.float32), 'float32 scales'),
            (dict(x=(x8[0].float(), x8[1]), dtype=torch.float32), 'float8_e4m3fn'),
            (dict(x=(x8[0], x8[1][:, :1]), dtype=torch.float32), 'scales of x'), (dict(x=x8[0]), 'float32, float16'),
            (dict(x=(x8[0],)), 'pair'), (dict(weight=(w8[0], w8[1][:1])), 'scales of weight'),
            (dict(weight=x8), 'scales of weight'), (dict(weight=w.half()), 'dtype of x'),
            (dict(weight=w[0]), 'weight must be'), (dict(bias=b[:4]), 'bias'), (dict(bias=b.double()), 'bias'),
            (dict(quantize=True, dtype=torch.float32), 'no dtype'), (dict(dtype=torch.float64), 'dtype must be'),
            (dict(x=x.clone().requires_grad_()), 'gradients need'), (dict(x=x8, weight=wg, dtype=x.dtype),
                                                                    'gradients need'),
            (dict(x=(x8[0], x8[1].clone().requires_grad_()), dtype=x.dtype), 'gradients need'),
            (dict(weight=wg, activation='relu'), 'plain product'), (dict(weight=wg, quantize=True), 'plain product'),
            (dict(weight=wg, dtype=torch.float16), 'plain product'), (dict(weight=wg, bias=b.half()), 'bias must'),
            (dict(x=x.to('meta')), 'same device')]:
        with pytest.raises(RuntimeError, match=message):
            linear_fp8(**{**good, **change})
    with pytest.raises(ValueError, match='activation'):
        linear_fp8(**good, activation='tanh')
    with pytest.raises(RuntimeError, match='weight must be'):
        quantize_weight_fp8(x[0])
    with pytest.raises(RuntimeError, match='scales'):
        dequantize_fp8(x8[0], x8[1][:, :1], torch.float32)
    with pytest.raises(RuntimeError, match='dtype'):
        dequantize_fp8(*x8, torch.float64)


def feed_forward(linear1, linear2, gain, out, tgt):
    """A serving layer's feed-forward half from a model's parameters, as a user writes it."""
    w1, w2 = quantize_weight_fp8(linear1.weight), quantize_weight_fp8(linear2.weight)
    with torch.no_grad():
        h, tgt = rms_norm(out, gain, residual=tgt, return_sum=True, quantize=True)
        a = linear_fp8(h, w1, linear1.bias, activation='relu', quantize=True)
        return linear_fp8(a, w2, linear2.bias, dtype=tgt.dtype), tgt


def check_feed_forward(device):
    torch.manual_seed(0)
    layers = [torch.nn.Linear(*s, device=device) for s in ((256, 512), (512, 256))]
    gain = torch.nn.Parameter(torch.rand(256, device=device) + 0.5)
    out, tgt = (torch.randn(3, 20, 256, device=device) for _ in range(2))
    y, s = feed_forward(*layers, gain, out, tgt)
    assert torch.equal(s, out + tgt) and not y.requires_grad
    with torch.no_grad():
        h = s * torch.rsqrt(s.square().mean(-1, keepdim=True) + 1e-6) * gain
        want = layers[1](torch.relu(layers[0](h)))
    # the operands' roundings to 8 bits, 2^-4 at most each: about 3 % of independent terms
    assert (y - want).norm() <= 0.1 * want.norm()
    h8 = rms_norm(out, gain.detach(), residual=tgt, quantize=True)
    with pytest.raises(RuntimeError, match='gradients need'):  # a bias that requires grad, outside no_grad
        linear_fp8(h8, quantize_weight_fp8(layers[0].weight), layers[0].bias, activation='relu', quantize=True)
    with pytest.raises(RuntimeError, match='no gradient'):
        rms_norm(out, gain, residual=tgt, quantize=True)


def test_a_models_feed_forward_half_in_serving():
    check_feed_forward('cpu')


def test_linear_refuses_what_is_no_operand():
    for bad in (None, 3.0):
        with pytest.raises(RuntimeError, match='pair'):
            linear_fp8(bad, torch.zeros(4, 8))
        with pytest.raises(RuntimeError, match='pair'):
            linear_fp8(torch.zeros(4, 8), bad)


def test_quantising_refuses_to_cut_a_graph():
    """A result that looks differentiable and is not would train nothing."""
    x = torch.randn(3, 200, requires_grad=True)
    w8 = quantize_weight_fp8(torch.nn.Parameter(torch.randn(150, 200)))  # laid out once, from a module's parameter
    for make in (quantize_fp8, lambda t: linear_fp8(quantize_fp8(t), w8, dtype=t.dtype), lambda t: quantize_fp8(t * 2)):
        with pytest.raises(RuntimeError, match='no gradient'):
            make(x)
    with torch.no_grad():
        kept = quantize_fp8(x)
    assert torch.equal(kept[0].float(), quantize_fp8(x.detach())[0].float())
    with pytest.raises(RuntimeError, match='no gradient'):
        dequantize_fp8(kept[0], kept[1].requires_grad_(), torch.float32)


def test_rms_norm_abi_refuses_before_any_launch(lib):
    err = ctypes.create_string_buffer(256)
    p = ctypes.c_void_p(16)

    def forward(dtype=0, rows=4, C=8, eps=1e-5, x=p, y=p, q=None, pitch=0, scale=None):
        return lib.td_rms_norm_forward(dtype, x, None, p, y, None, q, pitch, scale, None, rows, C, eps, None, err, 256)

    assert forward(dtype=9) == 1 and forward(rows=-1) == 1 and forward(C=0) == 1 and forward(C=8193) == 1
    assert forward(eps=-1.0) == 1 and forward(x=None) == 1 and forward(y=None) == 1
    q = dict(y=None, q=p, pitch=16, scale=p)
    assert forward(**{**q, 'dtype': 3}) == 1 and forward(**{**q, 'pitch': 8}) == 1 and forward(**{**q, 'pitch': 32}) == 1
    assert forward(**{**q, 'scale': None}) == 1 and forward(**{**q, 'y': p}) == 1
    assert forward(**{**q, 'q': ctypes.c_void_p(24)}) == 1
    assert forward(rows=0, x=None) == 0
    assert lib.td_rms_norm_workspace_bytes(0, 4, 8) == 8 * 4 and lib.td_rms_norm_workspace_bytes(9, 4, 8) == 0
    assert lib.td_rms_norm_backward(0, p, None, p, None, p, p, p, p, 4, 8, p, 3, None, err, 256) == 3
    assert lib.td_rms_norm_backward(0, p, None, p, None, p, None, p, p, 4, 8, p, 1 << 20, None, err, 256) == 1


def test_fp8_abi_refuses_before_any_launch(lib):
    err = ctypes.create_string_buffer(256)
    p, big = ctypes.c_void_p(256), 1 << 30

    def linear(x_dtype=0, x_pitch=0, x_scale=None, w_pitch=128, bias_dtype=0, bias=None, act=0, out_dtype=0, out=p,
               out_pitch=0, out_scale=None, M=4, K=128, N=64, ws=p, ws_bytes=big, x=p):
        return lib.td_fp8_linear(x_dtype, x, x_pitch, x_scale, p, w_pitch, p, bias_dtype, bias, act, out_dtype, out,
                                 out_pitch, out_scale, M, K, N, ws, ws_bytes, None, err, 256)

    for kw in (dict(x_dtype=3), dict(out_dtype=3), dict(bias=p, bias_dtype=4), dict(act=4), dict(act=-1), dict(M=-1),
               dict(M=2 ** 31 - 255), dict(K=0), dict(N=0), dict(K=65537), dict(x=None), dict(w_pitch=127), dict(out=None),
               dict(x_dtype=4, x_pitch=128), dict(x_dtype=4, x_pitch=127, x_scale=p),
               dict(out_dtype=4, out_pitch=80, out_scale=p), dict(out_dtype=4, out_pitch=64)):
        assert linear(**kw) == 1, (kw, err.value)
    assert linear(M=0, x=None) == 0 and linear(ws=None) == 3 and linear(ws_bytes=8) == 3
    assert lib.td_fp8_linear_workspace_bytes(3, 4, 128, 64, 0, 0) == 0
    assert lib.td_fp8_linear_workspace_bytes(4, 4, 128, 64, 0, 0) == 0
    assert linear(w_pitch=136, ws=None) == 3 and linear(w_pitch=1 << 40) == 1

    def backward(dtype=0, g=p, x=p, x_pitch=128, w=p, M=4, K=128, N=64, ws=p, ws_bytes=big):
        return lib.td_fp8_linear_backward(dtype, g, x, x_pitch, p, w, p, p, p, M, K, N, ws, ws_bytes, None, err, 256)

    for kw in (dict(dtype=4), dict(g=None), dict(x=None), dict(w=None), dict(x_pitch=127), dict(M=-1), dict(N=0)):
        assert backward(**kw) == 1, kw
    assert backward(ws=None) == 3 and backward(ws_bytes=8) == 3

    def quantize(dtype=0, x=p, pitch=128, M=4, K=128, q=p, scale=p):
        return lib.td_fp8_quantize(dtype, x, q, pitch, scale, M, K, 0, None, err, 256)

    for kw in (dict(dtype=3), dict(x=None), dict(pitch=112), dict(pitch=144), dict(q=None), dict(scale=None),
               dict(q=ctypes.c_void_p(8)), dict(K=0)):
        assert quantize(**kw) == 1, kw
    assert quantize(M=0, x=None) == 0
    assert lib.td_fp8_dequantize(0, p, 127, p, p, 4, 128, 0, None, err, 256) == 1


def role(file, start):
    """The source of a warp's role, from `start` on."""
    text = open(os.path.join(build.CSRC, file)).read()
    return text[text.index(start):]


def test_bounded_waits_begin_behind_the_kernel_before():
    """A product's CTA may start while the kernel before it in the stream still runs, for longer than its own waits last:
    the issuing thread and the producers count from behind their dependency wait. (Read from the source: a kernel that
    runs for a second after it let the next one start would be needed to see it.)"""
    issuer = role('td_fp8_tc.cuh', 'else if (warp == 9) {')
    assert 0 < issuer.index('grid_dependency_wait()') < issuer.index('mbar_wait_at(')
    producer = role('td_fp8_tc.cuh', 'if (warp == 8) {')
    assert producer.index('grid_dependency_wait()') < producer.index('t0 = clock64()') < producer.index('mbar_test(')
    epilogue = role('td_fp8_tc.cuh', 'setmaxnreg.inc')
    assert epilogue.index('grid_dependency_wait()') < epilogue.index('mbar_wait_at(')
    # the projection's roles wait for the kernel before where their time for a tile runs out, and then once more
    for start, end in (('// MMA issuer.', 'mma_issue<T>'), ('// float32: split every landed slot', 'float4* x')):
        text = role('td_gemm_tc.cuh', start)
        text = text[:text.index(end)]
        assert 'mbar_wait_behind(' in text and 'mbar_wait(&full' not in text and 'mbar_wait(wfull' not in text
    patient = role('td_ptx.cuh', 'bool mbar_wait_behind(')
    assert 0 < patient.index('grid_dependency_wait()') < patient.index('mbar_wait(bar, parity, err_code)')
