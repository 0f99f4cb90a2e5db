"""The 8-bit conversions and products on the GPU, forward and backward, against float64 with counted error bounds, and a
feed-forward half made of norm and products."""

import pytest
import torch

from attention_oracle import check
from fp8_oracle import (E4M3, behind_rows, check_quantized, linear_train_exact, product_exact, quantized,
                        rms_norm_exact, through, worth)
from marearts_tinydeform_b200 import (_native, dequantize_fp8, linear_fp8, quantize_fp8, quantize_fp8_reference,
                                      quantize_weight_fp8, quantize_weight_fp8_reference, rms_norm)

pytestmark = pytest.mark.gpu

DTYPES = (torch.float32, torch.float16, torch.bfloat16)
ACTS = (None, 'relu', 'gelu', 'silu')
# M, K, N: one value; one row; few rows (up to 16 and past it) with short, odd and long sums; edges of a tile of 128
# and 256; odd sizes; a long sum behind few tiles; more tiles than a wave
SHAPES = [(1, 1, 1), (1, 128, 128), (1, 4096, 700), (3, 7, 5), (2, 129, 130), (8, 200, 1000), (9, 256, 64),
          (16, 4100, 512), (17, 256, 64), (33, 4099, 40), (128, 128, 256), (129, 515, 257), (300, 256, 1024),
          (300, 1024, 256), (1000, 1030, 264), (513, 96, 1030), (130, 8200, 130), (5000, 384, 1000)]


def normal(*shape, dtype=torch.float32, seed=0, std=1.0):
    g = torch.Generator(device='cuda').manual_seed(seed)
    return (torch.randn(shape, generator=g, device='cuda') * std).to(dtype)


def spread(M, K, dtype, seed=0):
    """Rows and channels of different sizes."""
    return (normal(M, K, seed=seed) * torch.exp(normal(M, 1, seed=seed + 1)) *
            torch.exp(0.7 * normal(1, K, seed=seed + 2))).to(dtype)


def free_pair(w):
    """w in blocks of 128 x 128 with scales that are no powers of two."""
    N, K = w.shape
    scale = torch.rand((-(-N // 128), -(-K // 128)), device='cuda') * 0.01 + 0.001
    per = scale.repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]
    return (w.float() / per).clamp(-448, 448).to(E4M3), scale


@pytest.mark.parametrize('shape', [(1, 1), (3, 128), (5, 129), (130, 300), (257, 1000), (1000, 256), (3, 8200), (2, 520)],
                         ids=str)
@pytest.mark.parametrize('dtype', DTYPES, ids=str)
def test_quantize(cuda, dtype, shape):
    x = spread(*shape, dtype)
    x[0, 0] = 0
    for make, rows in ((quantize_fp8, 1), (quantize_weight_fp8, 128)):
        data, scale = make(x)
        q, s = quantized(x, rows, 128)
        assert data.dtype == E4M3 and torch.equal(data.double(), q) and torch.equal(scale.double(), s)
        for out in (torch.float32, torch.bfloat16, torch.float16):
            assert torch.equal(dequantize_fp8(data, scale, out), worth(q, s, rows, 128).float().to(out))
    # rows that start anywhere, and a leading shape
    odd = torch.cat([x.new_zeros(1), x.reshape(-1)])[1:].view(1, *shape)
    assert torch.equal(quantize_fp8(odd)[0][0].float(), quantize_fp8(x)[0].float())
    assert torch.equal(quantize_fp8(x.t().contiguous().t())[0].float(), quantize_fp8(x)[0].float())


def test_quantize_edges(cuda):
    for C in (130, 136):  # rows in vectors and without
        x = torch.zeros(6, C)
        x[1, 3], x[1, 129] = 448.0, 449.0
        x[2, :3] = torch.tensor([float('inf'), float('nan'), 7.0])
        x[3, 0] = 3.4e38
        x[4, 0] = 1e-40
        x[5, :4] = torch.tensor([17.0, 19.0, 21.0, -23.0])
        x[5, 4] = 448.0
        for make, ref in ((quantize_fp8, quantize_fp8_reference),
                          (quantize_weight_fp8, quantize_weight_fp8_reference)):
            got, want = make(x.cuda()), ref(x)
            assert torch.equal(got[1].cpu(), want[1])
            assert torch.equal(got[0].float().cpu().nan_to_num(nan=-1), want[0].float().nan_to_num(nan=-1))
    assert quantize_fp8(x.cuda()[:0])[0].shape == (0, 136)


@pytest.mark.parametrize('shape', SHAPES, ids=str)
@pytest.mark.parametrize('dtype', DTYPES, ids=str)
def test_linear(policy, dtype, shape):
    M, K, N = shape
    x, w, b = spread(M, K, dtype), normal(N, K, dtype=dtype, seed=5, std=K ** -0.5), normal(N, dtype=dtype, seed=6)
    x8, w8 = quantize_fp8(x), quantize_weight_fp8(w)
    xd, wd = through(x, 1, 128), through(w, 128, 128)
    free = free_pair(w)
    free_d = worth(*free, 128, 128)
    for act, bias in ((None, None), (None, b), ('relu', b), ('gelu', b), ('silu', None)):
        exact = product_exact(xd, wd, dtype, bias, act)
        check(linear_fp8(x, w8, bias, act), exact, f'{act}')
        check(linear_fp8(x8, w8, bias, act, dtype=dtype), exact, f'{act}, 8-bit input')
        check_quantized(linear_fp8(x, w8, bias, act, quantize=True), exact, f'{act}, 8-bit result')
        check(linear_fp8(x, free, bias, act), product_exact(xd, free_d, dtype, bias, act), f'{act}, other scales')
    check(linear_fp8(x, w, b), product_exact(xd, wd, dtype, b), 'floating weight')
    check(linear_fp8(x, w8, b.float(), dtype=torch.float32), product_exact(xd, wd, torch.float32, b), 'float32 result')
    assert not behind_rows(linear_fp8(x8, w8, b, quantize=True)[0]).any()
    assert _native.device_error() == 0


@pytest.mark.parametrize('shape', SHAPES + [(1, 1, 200), (300, 1, 7), (300, 9, 1), (300, 1, 1), (129, 128, 1)], ids=str)
@pytest.mark.parametrize('dtype', DTYPES, ids=str)
def test_training(policy, dtype, shape):
    M, K, N = shape
    x, w, b = spread(M, K, dtype), normal(N, K, dtype=dtype, seed=5, std=K ** -0.5), normal(N, dtype=dtype, seed=6)
    g = spread(M, N, dtype, 7) * 0.1
    exact = linear_train_exact(x, w, b, g)
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    y = linear_fp8(*leaves)
    got = [y.detach()] + list(torch.autograd.grad(y, leaves, g))
    for name, a, e in zip(('y', 'grad_x', 'grad_weight', 'grad_bias'), got, exact):
        check(a, e, name)
    # one gradient at a time gives the same bits
    for k in range(3):
        only = [t.detach().requires_grad_(i == k) for i, t in enumerate((x, w, b))]
        assert torch.equal(torch.autograd.grad(linear_fp8(*only), only[k], g)[0], got[k + 1])
    assert _native.device_error() == 0


def test_gradients_against_differences(policy):
    """Small whole numbers survive the rounding to 8 bits, so the product is its own formula and linear in each
    operand: differences over a step of 1 are its gradients, exactly."""
    gen = torch.Generator().manual_seed(7)
    x, w, g = (torch.randint(-4, 5, s, generator=gen).float().cuda() for s in ((5, 9), (4, 9), (5, 4)))
    b = torch.randint(-4, 5, (4,), generator=gen).float().cuda()
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(linear_fp8(*leaves), leaves, g)
    for k in range(3):
        for i in range(leaves[k].numel()):
            moved = [t.clone() for t in (x, w, b)]
            moved[k].view(-1)[i] += 1
            assert ((linear_fp8(*moved) - linear_fp8(x, w, b)) * g).sum() == grads[k].reshape(-1)[i]


def test_the_input_is_kept_in_8_bits_alone(cuda):
    x = normal(4096, 1024, dtype=torch.bfloat16).requires_grad_()
    w = normal(128, 1024, dtype=torch.bfloat16, seed=1).requires_grad_()
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    y = linear_fp8(x, w)
    kept = torch.cuda.memory_allocated() - before - y.numel() * 2
    assert 4096 * 1024 <= kept <= 4096 * 1024 * 1.04  # a byte a value and a scale each 128
    saved = [t.dtype for t in y.grad_fn.saved_tensors]
    assert saved == [E4M3, torch.float32, torch.bfloat16]  # (the last is the weight, the caller's own)


def test_strides_and_shapes(policy):
    x, w, b = normal(6, 10, 264, dtype=torch.float16), normal(72, 264, dtype=torch.float16, seed=1), None
    x8, w8 = quantize_fp8(x), quantize_weight_fp8(w)
    want = linear_fp8(x8, w8, b, dtype=torch.float16)
    assert want.shape == (6, 10, 72)

    def same(a, weight=w8):
        assert torch.equal(linear_fp8(a, weight, b, dtype=torch.float16).reshape(60, 72), want.view(60, 72))

    same(x.view(60, 264))
    same(x.transpose(0, 1).contiguous().transpose(0, 1))
    dense = x8[0].contiguous()
    same((dense, x8[1]))                                             # rows 264 bytes apart: no multiple of 16
    wide = torch.zeros(60, 400, dtype=torch.uint8, device='cuda')
    wide[:, 16:280] = dense.view(torch.uint8).view(60, 264)
    wide[:, 280:] = 0x7F                                             # NaN behind the rows: not read
    same((wide[:, 16:280].view(E4M3), x8[1].view(60, -1)))           # aligned rows of a wider tensor
    same((wide[:, 16:280].view(E4M3).view(6, 10, 264), x8[1]))
    odd = torch.zeros(60, 400, dtype=torch.uint8, device='cuda')
    odd[:, 3:267] = dense.view(torch.uint8).view(60, 264)
    same((odd[:, 3:267].view(E4M3), x8[1].view(60, -1)))             # rows that start anywhere
    same((dense.transpose(0, 1).contiguous().transpose(0, 1), x8[1].transpose(0, 1).contiguous().transpose(0, 1)))
    same(x8, (w8[0].t().contiguous().t(), w8[1].t().contiguous().t()))
    one = linear_fp8((x8[0][:1, :1].expand(6, 10, 264), x8[1][:1, :1].expand(6, 10, 3)), w8, dtype=torch.float16)
    assert torch.equal(one, want[:1, :1].expand(6, 10, 72))
    assert torch.equal(linear_fp8(x[0, 0], w8), want[0, 0])          # a single row without a leading dimension
    assert linear_fp8(x[:0], w8).shape == (0, 10, 72)
    empty = [x[:0].detach().requires_grad_(), w.detach().requires_grad_()]
    gx, gw = torch.autograd.grad(linear_fp8(*empty), empty, x.new_zeros(0, 10, 72))
    assert gx.shape == (0, 10, 264) and not gw.any()


@pytest.mark.parametrize('M', (1, 3, 14, 40, 200))
def test_operands_that_start_anywhere(policy, M):
    """x, weight and bias one element behind a boundary, in wide and in 8-bit types."""
    def shifted(t):
        return torch.cat([t.new_zeros(1), t.reshape(-1)])[1:].view(t.shape)

    def shifted8(t):
        return shifted(t.contiguous().view(torch.uint8)).view(E4M3)

    for dtype, K in ((torch.bfloat16, 256), (torch.float32, 136), (torch.float16, 131)):
        x, w = normal(M, K, dtype=dtype), normal(200, K, dtype=dtype, seed=1)
        b = normal(200, dtype=dtype, seed=2)
        x8, w8 = quantize_fp8(x), quantize_weight_fp8(w)
        want, want8 = linear_fp8(x8, w8, b, 'relu', dtype=dtype), linear_fp8(x8, w8, b, quantize=True)
        for a in (x, shifted(x), x8, (shifted8(x8[0]), x8[1]), (x8[0].contiguous(), x8[1])):
            for v in (w8, (shifted8(w8[0]), w8[1]), (w8[0].contiguous(), w8[1])):
                assert torch.equal(linear_fp8(a, v, shifted(b), 'relu', dtype=dtype), want)
                got8 = linear_fp8(a, v, shifted(b), quantize=True)
                assert torch.equal(got8[0].float(), want8[0].float()) and torch.equal(got8[1], want8[1])


@pytest.mark.parametrize('M', (1, 5, 200))
def test_infinities_and_nan_stay_in_their_rows(policy, M):
    x, w = normal(M + 2, 300), normal(140, 300, seed=1)
    clean = linear_fp8(x, quantize_weight_fp8(w))
    x[0, 7], x[M + 1, 299] = float('inf'), float('nan')
    got = linear_fp8(x, quantize_weight_fp8(w))
    assert got[[0, M + 1]].isnan().all() and torch.equal(got[1:M + 1], clean[1:M + 1])
    data, scale = linear_fp8(x, quantize_weight_fp8(w), activation='relu', quantize=True)
    assert data[[0, M + 1]].float().isnan().all() and data[1:M + 1].float().isfinite().all()


@pytest.mark.parametrize('M', (1, 9, 200))
def test_nan_in_a_weight_or_bias_stays_in_its_column(policy, M):
    x, w, b = normal(M, 300), normal(270, 300, seed=1), normal(270, seed=2)
    clean = linear_fp8(x, quantize_weight_fp8(w), b)
    rest = [n for n in range(270) if n not in (5, 140, 269)]
    w[5, 299], w[140, 0], b[269] = float('nan'), float('inf'), float('nan')
    got = linear_fp8(x, quantize_weight_fp8(w), b)
    assert got[:, [5, 140, 269]].isnan().all() and torch.equal(got[:, rest], clean[:, rest])
    data, scale = linear_fp8(x, quantize_weight_fp8(w), b, activation='relu', quantize=True)
    assert data[:, [5, 140, 269]].float().isnan().all() and data[:, rest].float().isfinite().all()
    assert scale.isfinite().all()


def test_infinities_and_nan_in_a_gradient(policy):
    """A row of grad_x and a row of grad_weight go, the rest stays; the bias's sum is the sum, infinity and all."""
    x, w, b, g = normal(300, 200), normal(140, 200, seed=1), normal(140, seed=2), normal(300, 140, seed=3)

    def grads(g):
        leaves = [t.detach().requires_grad_() for t in (x, w, b)]
        return torch.autograd.grad(linear_fp8(*leaves), leaves, g)

    clean = grads(g)
    g[7, 3], g[250, 139] = float('inf'), float('nan')
    gx, gw, gb = grads(g)
    for got, want, bad in ((gx, clean[0], [7, 250]), (gw, clean[1], [3, 139])):
        rest = torch.ones(got.shape[0], dtype=torch.bool, device='cuda')
        rest[bad] = False
        assert got[bad].isnan().all() and torch.isfinite(got[rest]).all()
    keep = [n for n in range(140) if n not in (3, 139)]
    assert gb[3] == float('inf') and gb[139].isnan() and torch.equal(gb[keep], clean[2][keep])


@pytest.mark.parametrize('M', (2, 40))
def test_activations_at_their_ends(policy, M):
    """Arguments from -1000 to 1000 (exact products of powers of two), where exponentials leave float32's range."""
    x = torch.zeros(M, 128, device='cuda')
    x[:, 0] = 1
    v = torch.tensor([-1000., -128, -96, -88, -64, -32, -16, -8, -1, -2.0 ** -6, 0, 2.0 ** -6, 1, 8, 88, 128, 1000],
                     device='cuda')
    w8 = quantize_weight_fp8(torch.zeros(v.numel(), 128, device='cuda'))
    for act in ('relu', 'gelu', 'silu'):
        check(linear_fp8(x, w8, v, act), product_exact(x, torch.zeros(v.numel(), 128, device='cuda'), torch.float32, v,
                                                       act), act)


def test_two_threads_at_once(cuda):
    """Calls from two host threads, each on a stream of its own, give what they give alone."""
    import threading
    w8 = quantize_weight_fp8(normal(512, 256, dtype=torch.bfloat16, seed=1))
    xs = [normal(M, 256, dtype=torch.bfloat16, seed=M) for M in (3, 300)]
    want = [linear_fp8(x, w8, activation='relu') for x in xs]
    torch.cuda.synchronize()
    wrong = []

    def work(x, e):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                outs = [linear_fp8(x, w8, activation='relu') for _ in range(50)]
                torch.cuda.current_stream().synchronize()
            if not all(torch.equal(o, e) for o in outs):
                wrong.append('results differ')
        except Exception as exc:  # a thread's own exception would be lost
            wrong.append(repr(exc))

    threads = [threading.Thread(target=work, args=a) for a in zip(xs, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_rows_behind_the_last_are_left_alone(policy):
    """Results of a smaller call into the front of a larger allocation's neighbours: what lies behind stays."""
    for M, N in ((5, 130), (130, 264), (300, 1024)):
        x, w8 = normal(M, 256, dtype=torch.bfloat16), quantize_weight_fp8(normal(N, 256, dtype=torch.bfloat16, seed=1))
        lib, big = _native.load(), torch.full((M + 140, N), 7.0, dtype=torch.bfloat16, device='cuda')
        ws_bytes = lib.td_fp8_linear_workspace_bytes(_native.TD_BF16, M, 256, N, 0, 0)
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device='cuda')
        _native._launch(lib.td_fp8_linear, x.device, _native.TD_BF16, x.data_ptr(), 0, None, w8[0].data_ptr(),
                        256, w8[1].data_ptr(), 0, None, 0, _native.TD_BF16, big.data_ptr(), 0, None, M, 256, N,
                        ws.data_ptr(), ws_bytes)
        assert (big[M:] == 7).all() and torch.equal(big[:M], linear_fp8(x, w8))


def test_offsets_past_31_bits(cuda):
    """Results and gradients of more than 2^31 values: the last rows, and a weight's gradient that only they feed."""
    M, K, N, last = 530000, 128, 4096, 700
    x, w = normal(M, K, dtype=torch.bfloat16), normal(N, K, dtype=torch.bfloat16, seed=1, std=K ** -0.5)
    end = slice(M - last, M)
    xd, wd = through(x[end], 1, 128), through(w, 128, 128)
    y8, scale = linear_fp8(x, quantize_weight_fp8(w), quantize=True)
    check_quantized((y8[end], scale[end]), product_exact(xd, wd, torch.bfloat16), '8-bit result')
    del y8, scale
    leaves = [x.requires_grad_(), w.requires_grad_()]
    y = linear_fp8(*leaves)
    check(y.detach()[end], product_exact(xd, wd, torch.bfloat16), 'y')
    g = torch.zeros(M, N, dtype=torch.bfloat16, device='cuda')
    first = M // 128 * 128 - 512  # from the beginning of a block of rows
    g[first:] = normal(M - first, N, dtype=torch.bfloat16, seed=2)
    gx, gw = torch.autograd.grad(y, leaves, g)
    del y
    check(gx[first:], product_exact(through(g[first:], 1, 128), wd.t(), torch.bfloat16), 'grad_x')
    cols = through(g[first:], 128, 1).t(), through(through(x.detach()[first:], 1, 128), 128, 1).t()
    check(gw, product_exact(*cols, torch.bfloat16), 'grad_weight')


def test_same_bits_every_time(cuda):
    x, w, b = spread(2400, 256, torch.float16), normal(1024, 256, dtype=torch.float16, seed=1), \
        normal(1024, dtype=torch.float16, seed=2)
    g = normal(2400, 1024, dtype=torch.float16, seed=3)

    def once():
        leaves = [t.detach().requires_grad_() for t in (x, w, b)]
        y = linear_fp8(*leaves)
        return [y.detach()] + list(torch.autograd.grad(y, leaves, g))

    first = once()
    assert all(torch.equal(p, q) for _ in range(3) for p, q in zip(first, once()))


@pytest.mark.parametrize('M', (4, 300))
def test_graph_capture_and_streams(cuda, M):
    """Two captured calls of one shape, replayed in turn on fresh inputs, and eager calls on two streams at once."""
    w8 = quantize_weight_fp8(normal(1024, 512, dtype=torch.bfloat16, seed=1))
    xs = [normal(M, 512, dtype=torch.bfloat16, seed=i) for i in range(4)]
    want = [linear_fp8(x, w8, activation='silu') for x in xs]
    graphs, held = [], [xs[0].clone(), xs[1].clone()]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        linear_fp8(held[0], w8, activation='silu')
        stream.synchronize()
        for x in held:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                out = linear_fp8(x, w8, activation='silu')
            graphs.append((graph, out))
    for turn in (0, 2):
        for x, fresh in zip(held, xs[turn:turn + 2]):
            x.copy_(fresh)
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for (_, out), e in zip(graphs, want[turn:turn + 2]):
            assert torch.equal(out, e)
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[], []]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(10):
        for s, x, o in zip(streams, xs, outs):
            with torch.cuda.stream(s):
                o.append(linear_fp8(x, w8, activation='silu'))
    torch.cuda.synchronize()
    for o, e in zip(outs, want):
        assert all(torch.equal(t, e) for t in o)


def test_training_graph_capture(cuda):
    def fresh(seed):
        return [spread(700, 256, torch.bfloat16, seed), normal(512, 256, dtype=torch.bfloat16, seed=seed + 3),
                normal(512, dtype=torch.bfloat16, seed=seed + 4), normal(700, 512, dtype=torch.bfloat16, seed=seed + 5)]

    def eager(x, w, b, g):
        leaves = [t.detach().requires_grad_() for t in (x, w, b)]
        y = linear_fp8(*leaves)
        return [y.detach()] + list(torch.autograd.grad(y, leaves, g))

    *leaves, g = fresh(0)
    for t in leaves:
        t.requires_grad_()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        torch.autograd.grad(linear_fp8(*leaves), leaves, g)
        graph = torch.cuda.CUDAGraph()
        stream.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            y = linear_fp8(*leaves)
            grads = torch.autograd.grad(y, leaves, g)
    new = fresh(20)
    with torch.no_grad():
        for t, f in zip((*leaves, g), new):
            t.copy_(f)
    graph.replay()
    torch.cuda.synchronize()
    for got, want in zip((y, *grads), eager(*new)):
        assert torch.equal(got, want)


# ---- the operators together: a layer's feed-forward half ----------------------------------------------------------

@pytest.mark.parametrize('dtype', DTYPES, ids=str)
@pytest.mark.parametrize('rows', (1, 16, 300))
def test_feed_forward_serving(policy, dtype, rows):
    """Norm, product with activation, product, each held to float64 on what the one before it gave."""
    C, F = 256, 1024
    x, r, gain = normal(rows, C, dtype=dtype), normal(rows, C, dtype=dtype, seed=1), 1 + normal(C, dtype=dtype, seed=2) / 8
    w1, w2 = normal(F, C, dtype=dtype, seed=3, std=C ** -0.5), normal(C, F, dtype=dtype, seed=4, std=F ** -0.5)
    b1, b2 = normal(F, dtype=dtype, seed=5), normal(C, dtype=dtype, seed=6)
    w1_8, w2_8 = quantize_weight_fp8(w1), quantize_weight_fp8(w2)
    with torch.inference_mode():
        h, s = rms_norm(x, gain, r, return_sum=True, quantize=True)
        a = linear_fp8(h, w1_8, b1, 'relu', quantize=True)
        y = linear_fp8(a, w2_8, b2, dtype=dtype)
    exact = rms_norm_exact(x, gain, r)
    check_quantized(h, exact[0], 'norm')
    check(s, exact[1], 'sum')
    check_quantized(a, product_exact(worth(*h, 1, 128), through(w1, 128, 128), dtype, b1, 'relu'), 'first product')
    check(y, product_exact(worth(*a, 1, 128), through(w2, 128, 128), dtype, b2), 'second product')


def test_feed_forward_training(cuda):
    """The half layer's gradients, composed of the operators' own in float64 along the same values."""
    dtype, rows, C, F = torch.float32, 200, 256, 512
    x, r, gain = normal(rows, C), normal(rows, C, seed=1), 1 + normal(C, seed=2) / 8
    w1, w2 = normal(F, C, seed=3, std=C ** -0.5), normal(C, F, seed=4, std=F ** -0.5)
    g = normal(rows, C, seed=5)
    leaves = [t.requires_grad_() for t in (x, r, gain, w1, w2)]
    h, s = rms_norm(x, gain, r, return_sum=True)
    z = linear_fp8(h, w1)
    a = torch.relu(z)
    y = s + linear_fp8(a, w2)
    inner = torch.autograd.grad(y, [h, z, a], g, retain_graph=True)
    grads = torch.autograd.grad(y, leaves, g)
    h, z, a = (t.detach() for t in (h, z, a))
    second = linear_train_exact(a, w2.detach(), None, g)
    check(inner[2], second[1], 'through the second product')
    check(grads[4], second[2], 'grad of the second weight')
    assert torch.equal(inner[1], inner[2] * (z > 0))
    first = linear_train_exact(h, w1.detach(), None, inner[1])
    check(inner[0], first[1], 'through the first product')
    check(grads[3], first[2], 'grad of the first weight')
    norm = rms_norm_exact(x.detach(), gain.detach(), r.detach(), grad=inner[0], grad_sum=g)
    check(grads[0], norm[2], 'grad_x')
    check(grads[2], norm[3], 'grad of the gain')
    assert torch.equal(grads[0], grads[1])
