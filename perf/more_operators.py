"""Performance cases of the feed-forward half of a layer: root-mean-square norm and products in 8-bit floating point.

``rms_norm`` adds the residual, norms the sum and, for serving, gives its result in 8 bits (e4m3) with a scale for each
block of 128 channels. ``linear`` is the product in 8 bits: the input in blocks of 1 x 128, the weight in blocks of
128 x 128; for serving with a weight that was laid out once, from one row on. ``train`` is the same product with a
floating weight and its three gradients, the input kept for them in 8 bits. ``ffn`` is the three products of a serving
layer in a row: norm, first product with its activation, second product.

Every case is one call a model makes (``ffn``: three); ``run`` computes it in plain torch operations (float32, rounded
once), or, with ``own``, through this package. ``exact`` is the operators' definition in float64; it says nothing of a
result in 8 bits, where a value beside the middle of two numbers may become either.
"""

import math

import torch

own = False

DTYPES = {'float32': torch.float32, 'float16': torch.float16, 'bfloat16': torch.bfloat16}
BLOCK = 128
EPS = 1e-6


def _device():
    return torch.device('cuda' if torch.cuda.is_available() else 'cpu')


# ---- cases --------------------------------------------------------------------------------------------------------

def _norm(dtype, rows, C, train=False, residual=True, total=True, quantize=False):
    """total: the sum x + residual is returned too. quantize: the norm's result in 8 bits."""
    return dict(op='norm', dtype=dtype, rows=rows, C=C, train=train, residual=residual, total=total and residual,
                quantize=quantize)


def _linear(dtype, M, K, N, act='none', bias=True, ready=False, quantize=False, free=False):
    """ready: the input comes in 8 bits already. quantize: the output leaves in 8 bits. free: the weight's scales are
    any numbers, as in a checkpoint from elsewhere, not powers of two."""
    return dict(op='linear', dtype=dtype, M=M, K=K, N=N, act=act, bias=bias, ready=ready, quantize=quantize, free=free)


def _train(dtype, M, K, N, bias=True):
    return dict(op='train', dtype=dtype, M=M, K=K, N=N, bias=bias)


def _ffn(dtype, M, K, N, act='relu'):
    return dict(op='ffn', dtype=dtype, M=M, K=K, N=N, act=act)


def listed():
    named = [
        # a decoder of 300 queries serving one image: the sum kept for the next layer, the norm in 8 bits
        ('norm_decoder_b1', _norm('float16', 300, 256, quantize=True)),
        # an encoder's norm over every token of 8 images of 800 x 1333, in 8 bits for the product behind it
        ('norm_encoder_fp8', _norm('bfloat16', 8 * 22223, 256, total=False, quantize=True)),
        # the same norm in training, with the sum
        ('norm_train_encoder', _norm('bfloat16', 8 * 22223, 256, train=True)),
        # float32 rows of odd width
        ('norm_train_odd', _norm('float32', 8 * 1100, 515, train=True, total=False)),
        # one token against a wide layer's weight
        ('linear_one_row', _linear('bfloat16', 1, 4096, 4096, bias=False, free=True)),
        # the first product of a decoder's feed-forward part, one image, its hidden values leaving in 8 bits
        ('linear_decoder_b1', _linear('float16', 300, 256, 1024, act='relu', quantize=True)),
        # odd sizes in float32
        ('linear_odd', _linear('float32', 8 * 1100, 515, 1030, act='silu')),
        # a wide layer over a long prompt, input in 8 bits
        ('linear_wide', _linear('bfloat16', 8192, 4096, 4096, ready=True, bias=False, free=True)),
        # the second product over every token of 8 images of 800 x 1333
        ('linear_encoder', _linear('bfloat16', 8 * 22223, 1024, 256, ready=True)),
        # a decoder's feed-forward product in training, 8 images of 300 queries
        ('train_decoder', _train('float16', 8 * 300, 256, 1024)),
        # an encoder's, over the three levels (80 x 80, 40 x 40, 20 x 20) of 8 images
        ('train_encoder', _train('bfloat16', 8 * 8400, 256, 1024)),
        # norm and both products of a serving decoder layer, 8 images
        ('ffn_decoder_b8', _ffn('bfloat16', 8 * 300, 256, 1024)),
    ]
    return [dict(case, name=name) for name, case in named]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


# the largest drawn calls: multiply-adds of a product and elements of a norm stay within the listed ones'
_MOST_PRODUCT = {'linear': 8192 * 4096 * 4096, 'train': 8 * 8400 * 256 * 1024, 'ffn': 8 * 8400 * 256 * 1024}
_MOST_ROWS = 8 * 22223


def draw(rng):
    dtype = rng.choice(['float16', 'bfloat16', 'float16', 'bfloat16', 'float32'])
    op = rng.choice(['norm', 'linear', 'linear', 'train', 'train', 'ffn'])
    if op == 'norm':
        C = rng.choice([256, 512, 1024, _log_int(rng, 32, 8192), _log_int(rng, 32, 8192)])
        rows = _log_int(rng, 1, max(1, min(_MOST_ROWS, _MOST_ROWS * 256 // C // (2 if dtype == 'float32' else 1))))
        train = rng.random() < 0.5
        return _norm(dtype, rows, C, train=train, residual=rng.random() < 0.7, total=rng.random() < 0.5,
                     quantize=not train and rng.random() < 0.7)
    K = rng.choice([256, 512, 1024, _log_int(rng, 32, 4096), _log_int(rng, 32, 4096)])
    N = rng.choice([256, 1024, 2048, _log_int(rng, 32, 4096), _log_int(rng, 32, 4096)])
    most = min(_MOST_PRODUCT[op] // (K * N), _MOST_ROWS * 1024 // (K + N))
    if dtype == 'float32':
        most = most // 2
    M = _log_int(rng, 1, max(1, min(_MOST_ROWS, most)))
    bias = rng.random() < 0.7
    if op == 'train':
        return _train(dtype, M, K, N, bias=bias)
    if op == 'ffn':
        return _ffn('bfloat16', M, K, N, act=rng.choice(['relu', 'silu', 'gelu']))
    return _linear(dtype, M, K, N, act=rng.choice(['none', 'relu', 'silu', 'gelu']), bias=bias,
                   ready=rng.random() < 0.4, quantize=rng.random() < 0.4, free=rng.random() < 0.5)


# ---- 8-bit blocks in plain operations -----------------------------------------------------------------------------

def _power_of_two(amax):
    """The smallest 2^e, e >= -126, with amax * 2^-e <= 448 = 0.875 * 2^9."""
    mantissa, exponent = torch.frexp(amax)
    e = (exponent - 9 + (mantissa > 0.875).to(exponent.dtype)).clamp_(min=-126)
    e = torch.where(amax == 0, torch.full_like(e, -126), e)
    return ((e + 127) << 23).to(torch.int32).view(torch.float32)


def _padded(x, rows, cols):
    """x [R, C] in float32 with zeros up to multiples of rows and cols."""
    R, C = x.shape
    return torch.nn.functional.pad(x.float(), (0, -C % cols, 0, -R % rows))


def _quantize(x, rows, cols, scale=None):
    """x [R, C] in blocks of rows x cols: the e4m3 tensor, its scales [R / rows, C / cols] (rounded up)."""
    R, C = x.shape
    p = _padded(x, rows, cols)
    p = p.view(p.shape[0] // rows, rows, p.shape[1] // cols, cols)
    if scale is None:
        scale = _power_of_two(p.abs().amax((1, 3)))
    q = (p / scale[:, None, :, None]).to(torch.float8_e4m3fn)
    return q.view(p.shape[0] * rows, p.shape[2] * cols)[:R, :C].contiguous(), scale


def _dequantize(q, scale, rows, cols):
    R, C = q.shape
    p = _padded(q, rows, cols)
    p = p.view(p.shape[0] // rows, rows, p.shape[1] // cols, cols) * scale[:, None, :, None]
    return p.view(p.shape[0] * rows, -1)[:R, :C]


def _through(x, rows, cols):
    """What x [R, C] is worth after its rounding to 8 bits, in float32."""
    return _dequantize(*_quantize(x, rows, cols), rows, cols)


# ---- inputs -------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    dev, dtype = _device(), DTYPES[case['dtype']]
    gen = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, generator=gen, device=dev) * std).to(dtype)

    def activations(M, K):
        """Rows whose channels differ in size, as behind a norm's weight."""
        size = torch.exp(0.5 * torch.randn(K, generator=gen, device=dev))
        return (torch.randn(M, K, generator=gen, device=dev) * size).to(dtype)

    def laid_out(weight, free=False):
        w = weight.float()
        if not free:
            return _quantize(w, BLOCK, BLOCK)
        p = _padded(w, BLOCK, BLOCK)
        top = p.view(p.shape[0] // BLOCK, BLOCK, p.shape[1] // BLOCK, BLOCK).abs().amax((1, 3))
        return _quantize(w, BLOCK, BLOCK, scale=top.clamp_min(1e-12) / 448)

    state = dict(case=case)
    if case['op'] == 'norm':
        rows, C = case['rows'], case['C']
        state['x'] = normal(rows, C)
        state['residual'] = normal(rows, C, std=2.0) if case['residual'] else None
        state['weight'] = (1 + 0.1 * torch.randn(C, generator=gen, device=dev)).to(dtype)
        if case['train']:
            state['grad'] = normal(rows, C, std=0.1)
            state['grad_total'] = normal(rows, C, std=0.1) if case['total'] else None
        return state
    M, K, N = case['M'], case['K'], case['N']
    if case['op'] == 'ffn':
        state['x'], state['residual'] = normal(M, K), normal(M, K, std=2.0)
        state['gain'] = (1 + 0.1 * torch.randn(K, generator=gen, device=dev)).to(dtype)
        state['w1'], state['b1'] = laid_out(normal(N, K, std=K ** -0.5)), normal(N, std=0.1)
        state['w2'], state['b2'] = laid_out(normal(K, N, std=N ** -0.5)), normal(K, std=0.1)
        return state
    x = activations(M, K)
    state['bias'] = normal(N, std=0.1) if case['bias'] else None
    weight = normal(N, K, std=K ** -0.5)
    if case['op'] == 'train':
        state['x'], state['weight'] = x, weight
        state['grad'] = normal(M, N, std=0.1)
    else:
        state['x'] = _quantize(x, 1, BLOCK) if case['ready'] else x
        state['weight'] = laid_out(weight, case['free'])
    return state


# ---- one pass -----------------------------------------------------------------------------------------------------

def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return {'norm': _plain_norm, 'linear': _plain_linear, 'train': _plain_train,
                'ffn': _plain_ffn}[state['case']['op']](state)


def _run_own(state):
    import marearts_tinydeform_b200 as mt
    case = state['case']
    op, dtype = case['op'], DTYPES[case['dtype']]
    if op == 'norm' and case['train']:
        leaves = [t.detach().requires_grad_() for t in (state['x'], state['weight'], state['residual'])
                  if t is not None]
        out = mt.rms_norm(leaves[0], leaves[1], residual=leaves[2] if case['residual'] else None, eps=EPS,
                          return_sum=case['total'])
        outs = list(out) if case['total'] else [out]
        grads = [state['grad']] + ([state['grad_total']] if case['total'] else [])
        return [t.detach() for t in outs] + list(torch.autograd.grad(outs, leaves, grads))
    if op == 'train':
        leaves = [t.detach().requires_grad_() for t in (state['x'], state['weight'], state['bias']) if t is not None]
        y = mt.linear_fp8(*leaves)
        return [y.detach()] + list(torch.autograd.grad(y, leaves, state['grad']))
    with torch.inference_mode():
        if op == 'norm':
            out = mt.rms_norm(state['x'], state['weight'], residual=state['residual'], eps=EPS,
                              return_sum=case['total'], quantize=case['quantize'])
            if not case['quantize']:
                return out
            y, total = out if case['total'] else (out, None)
            y = mt.dequantize_fp8(*y, dtype=torch.bfloat16)
            return [y] if total is None else [y, total]
        if op == 'ffn':
            h, total = mt.rms_norm(state['x'], state['gain'], residual=state['residual'], eps=EPS, return_sum=True,
                                   quantize=True)
            a = mt.linear_fp8(h, state['w1'], state['b1'], activation=case['act'], quantize=True)
            return [mt.linear_fp8(a, state['w2'], state['b2'], dtype=dtype), total]
        y = mt.linear_fp8(state['x'], state['weight'], state['bias'], quantize=case['quantize'],
                          activation=None if case['act'] == 'none' else case['act'],
                          dtype=None if case['quantize'] else dtype)
        return mt.dequantize_fp8(*y, dtype=torch.bfloat16) if case['quantize'] else y


def _activate(v, act):
    if act == 'relu':
        return v * (v > 0)
    if act == 'silu':
        return v / (1 + torch.exp(-v))
    if act == 'gelu':
        return 0.5 * v * (1 + torch.erf(v * math.sqrt(0.5)))
    return v


def _plain_norm(state):
    case = state['case']
    dtype = DTYPES[case['dtype']]
    s = state['x'].float()
    if state['residual'] is not None:
        s = s + state['residual'].float()
    w = state['weight'].float()
    rstd = torch.rsqrt(s.square().mean(-1, keepdim=True) + EPS)
    z = s * rstd
    y = z * w
    outs = [_through(y, 1, BLOCK).bfloat16() if case['quantize'] else y.to(dtype)]
    if case['total']:
        outs.append(s.to(dtype))
    if not case['train']:
        return outs if len(outs) > 1 or case['quantize'] else outs[0]
    dy = state['grad'].float()
    g = dy * w
    ds = (g - z * (g * z).mean(-1, keepdim=True)) * rstd
    if case['total']:
        ds = ds + state['grad_total'].float()
    ds = ds.to(dtype)
    dw = (dy * z).sum(0, dtype=torch.float64).to(dtype)  # column sums over many rows, in 64 bits
    return outs + [ds, dw] + ([ds] if case['residual'] else [])


def _product(x, weight, bias, act):
    """x [M, K] in float32 against a laid-out weight."""
    y = torch.matmul(x, _dequantize(*weight, BLOCK, BLOCK).t())
    return _activate(y if bias is None else y + bias.float(), act)


def _plain_linear(state):
    case = state['case']
    x = _dequantize(*state['x'], 1, BLOCK) if case['ready'] else _through(state['x'], 1, BLOCK)
    y = _product(x, state['weight'], state['bias'], case['act'])
    return _through(y, 1, BLOCK).bfloat16() if case['quantize'] else y.to(DTYPES[case['dtype']])


def _plain_train(state):
    dtype = DTYPES[state['case']['dtype']]
    x, w = _through(state['x'], 1, BLOCK), _through(state['weight'], BLOCK, BLOCK)
    y = torch.matmul(x, w.t())
    if state['bias'] is not None:
        y = y + state['bias'].float()
    dy = state['grad']
    dx = torch.matmul(_through(dy, 1, BLOCK), w)
    # over the rows: the gradient and the kept input in blocks of 128 rows
    dw = torch.matmul(_through(dy, BLOCK, 1).t(), _through(x, BLOCK, 1))
    outs = [y.to(dtype), dx.to(dtype), dw.to(dtype)]
    if state['bias'] is not None:
        outs.append(dy.sum(0, dtype=torch.float64).to(dtype))
    return outs


def _plain_ffn(state):
    case = state['case']
    dtype = DTYPES[case['dtype']]
    s = state['x'].float() + state['residual'].float()
    h = s * torch.rsqrt(s.square().mean(-1, keepdim=True) + EPS) * state['gain'].float()
    a = _product(_through(h, 1, BLOCK), state['w1'], state['b1'], case['act'])
    y = _product(_through(a, 1, BLOCK), state['w2'], state['b2'], 'none')
    return [y.to(dtype), s.to(dtype)]


# ---- what a pass cannot do without --------------------------------------------------------------------------------

def work(case):
    e = 4 if case['dtype'] == 'float32' else 2
    if case['op'] == 'norm':
        n = case['rows'] * case['C']
        tensors = 1 + case['residual'] + case['total'] + (not case['quantize'])
        if case['train']:  # the gradients read, the input's written (it is the residual's as well)
            return {'bytes': e * ((tensors + 2 + case['total']) * n + 2 * case['C']), 'flops': 16 * n}
        # a block's 128 values and their scale
        return {'bytes': e * (tensors * n + case['C']) + (n + n // 32 if case['quantize'] else 0), 'flops': 6 * n}
    M, K, N = case['M'], case['K'], case['N']
    if case['op'] == 'ffn':  # x, residual, their sum, the result; both weights; the hidden values stay inside
        return {'bytes': 4 * e * M * K + 2 * K * N, 'flops': 4 * M * K * N}
    if case['op'] == 'train':  # x, y, dy, dx, both weights, the input kept in 8 bits: written and read
        return {'bytes': e * (2 * M * (K + N) + 2 * N * K) + 2 * M * K, 'flops': 6 * M * K * N}
    into, out = (1 if case['ready'] else e), (1 if case['quantize'] else e)
    return {'bytes': into * M * K + N * K + out * M * N, 'flops': 2 * M * K * N}


# ---- the definition in 64 bits ------------------------------------------------------------------------------------

def _two_to(e):
    """2^e for whole numbers e in float64, by its bits: exactly that, so that values half way between two stay there."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_scale(top):
    """The power of two that brings `top` to at most 448, from the ratio's own exponent."""
    e = torch.ceil(torch.log2(top.clamp_min(2.0 ** -130) / 448))
    # log2 may be a hair off beside a power of two: the inequality itself decides
    e = torch.where(top * _two_to(-e) > 448, e + 1, e)
    e = torch.where(top * _two_to(1 - e) <= 448, e - 1, e)
    return _two_to(e.clamp_min(-126))


def _exact_e4m3(v):
    """v rounded to the nearest of e4m3's values (3 bits behind the point, steps no finer than 2^-9), ties to even."""
    step = _two_to((torch.frexp(v)[1] - 1).clamp_min(-6) - 3)
    return torch.round(v / step) * step


def _exact_rows(x):
    """x [R, C] rounded in blocks of 1 x 128."""
    parts = []
    for c in range(0, x.shape[1], BLOCK):
        part = x[:, c:c + BLOCK].contiguous()
        scale = _exact_scale(part.abs().amax(1, keepdim=True))
        parts.append(_exact_e4m3(part / scale) * scale)
    return torch.cat(parts, 1)


def _exact_tiles(w):
    out = torch.empty_like(w)
    for r in range(0, w.shape[0], BLOCK):
        for c in range(0, w.shape[1], BLOCK):
            tile = w[r:r + BLOCK, c:c + BLOCK]
            scale = _exact_scale(tile.abs().max())
            out[r:r + BLOCK, c:c + BLOCK] = _exact_e4m3(tile / scale) * scale
    return out


def _exact_worth(q, scale, rows):
    """The values that a laid-out tensor's numbers stand for."""
    per_row = scale.double().repeat_interleave(rows, 0)[:q.shape[0]]
    return q.double() * per_row.repeat_interleave(BLOCK, 1)[:, :q.shape[1]]


def _exact_act(v, act):
    return {'none': lambda t: t, 'relu': lambda t: t.clamp_min(0), 'silu': lambda t: t * torch.sigmoid(t),
            'gelu': lambda t: t * 0.5 * torch.erfc(-t / 2 ** 0.5)}[act](v)


def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        return {'norm': _exact_norm, 'linear': _exact_linear, 'train': _exact_train,
                'ffn': _exact_ffn}[case['op']](state)


def _exact_norm(state):
    case = state['case']
    w, parts, dw = state['weight'].double(), [], 0.0
    for i in range(0, case['rows'], 16384):
        s = state['x'][i:i + 16384].double()
        if case['residual']:
            s = s + state['residual'][i:i + 16384].double()
        n = s.shape[1]
        rms = torch.sqrt(torch.einsum('rc,rc->r', s, s) / n + EPS)[:, None]
        y = s / rms * w
        row = [None if case['quantize'] else y] + ([s] if case['total'] else [])
        if case['train']:
            dy = state['grad'][i:i + 16384].double()
            ds = dy * w / rms - s * torch.einsum('rc,rc->r', dy * w, s)[:, None] / (n * rms ** 3)
            if case['total']:
                ds = ds + state['grad_total'][i:i + 16384].double()
            row.append(ds)
            dw = dw + torch.einsum('rc,rc->c', dy, s / rms)
        parts.append(row)
    whole = [None if col[0] is None else torch.cat(col) for col in zip(*parts)]
    if not case['train']:
        if len(whole) > 1:
            return whole
        return whole[0]
    return whole + [dw] + ([whole[-1]] if case['residual'] else [])


def _exact_linear(state):
    case = state['case']
    if case['quantize']:
        return None
    w = _exact_worth(*state['weight'], BLOCK).t()
    out = []
    for i in range(0, case['M'], 16384):
        if case['ready']:
            x = _exact_worth(state['x'][0][i:i + 16384], state['x'][1][i:i + 16384], 1)
        else:
            x = _exact_rows(state['x'][i:i + 16384].double())
        y = x @ w
        out.append(_exact_act(y if state['bias'] is None else y + state['bias'].double(), case['act']))
    return torch.cat(out)


def _exact_train(state):
    x, dy = _exact_rows(state['x'].double()), state['grad'].double()
    w = _exact_tiles(state['weight'].double())
    y = x @ w.t()
    dw = 0.0
    for i in range(0, x.shape[0], BLOCK):
        dw = dw + _exact_rows(dy[i:i + BLOCK].t()) @ _exact_rows(x[i:i + BLOCK].t()).t()
    if state['bias'] is None:
        return [y, _exact_rows(dy) @ w, dw]
    return [y + state['bias'].double(), _exact_rows(dy) @ w, dw, dy.sum(0)]


def _exact_ffn(state):
    s = state['x'].double() + state['residual'].double()
    h = s / torch.sqrt((s * s).mean(1, keepdim=True) + EPS) * state['gain'].double()
    a = _exact_rows(h) @ _exact_worth(*state['w1'], BLOCK).t() + state['b1'].double()
    a = _exact_rows(_exact_act(a, state['case']['act']))
    return [a @ _exact_worth(*state['w2'], BLOCK).t() + state['b2'].double(), s]
