"""Performance cases of the decoder layer's attention and layer norm operators.

``attention`` is the self attention among a DETR decoder's queries (and any other softmax attention over keys of its
own length): forward, and forward plus backward. ``layer_norm`` is the normalisation behind each attention, with the
residual added inside. Every case is one call a model makes; ``run`` computes it in plain torch operations (float32,
rounded once), or, with ``own``, through this package. ``exact`` is the operators' definition in float64.
"""

import math

import torch

own = False

DTYPES = {'float32': torch.float32, 'float16': torch.float16, 'bfloat16': torch.bfloat16}


def _device():
    return torch.device('cuda' if torch.cuda.is_available() else 'cpu')


# ---- cases --------------------------------------------------------------------------------------------------------

def _attn(dtype, B, Q, N, H, Hk, D, train=False, causal=False, ragged=False, groups=0, packed=False):
    """groups > 0: the first fifth or so of the queries are that many denoising groups, with their mask."""
    return dict(op='attention', dtype=dtype, B=B, Q=Q, N=N, H=H, Hk=Hk, D=D, train=train, causal=causal,
                ragged=ragged, groups=groups, packed=packed)


def _norm(dtype, rows, C, train=False, residual=True):
    return dict(op='layer_norm', dtype=dtype, rows=rows, C=C, train=train, residual=residual)


def listed():
    named = [
        # RT-DETR's decoder serving one image: self attention among 300 queries, read from one packed projection
        ('attn_decoder_b1', _attn('float16', 1, 300, 300, 8, 8, 32, packed=True)),
        # the same in float32, two images
        ('attn_decoder_f32', _attn('float32', 2, 300, 300, 8, 8, 32)),
        # DINO with denoising queries: 900 matching + 200 denoising in 5 groups, under the groups' mask
        ('attn_denoise_b8', _attn('float16', 8, 1100, 1100, 8, 8, 32, groups=5, packed=True)),
        # one query (a tracked object, a single new token) over the tokens of padded 800 x 1333 images
        ('attn_one_query', _attn('bfloat16', 8, 1, 22223, 8, 8, 32, ragged=True)),
        # a causal prompt with grouped heads
        ('attn_causal_grouped', _attn('bfloat16', 2, 4096, 4096, 16, 4, 64, causal=True)),
        # RT-DETR's decoder training, 8 images
        ('attn_train_decoder', _attn('float16', 8, 300, 300, 8, 8, 32, train=True)),
        # DINO's decoder training with denoising queries
        ('attn_train_denoise', _attn('bfloat16', 4, 1100, 1100, 8, 8, 32, train=True, groups=5)),
        # a causal sequence of odd length with grouped wide heads
        ('attn_train_grouped', _attn('float16', 2, 2047, 2047, 8, 2, 128, train=True, causal=True)),
        # full self attention over an RT-DETR image's three levels (80 x 80, 40 x 40, 20 x 20)
        ('attn_train_encoder', _attn('bfloat16', 1, 8400, 8400, 8, 8, 32, train=True)),
        # the decoder's norm serving one image
        ('norm_decoder_b1', _norm('float16', 300, 256)),
        # a training encoder's norm over every token of 8 images of 800 x 1333
        ('norm_train_encoder', _norm('bfloat16', 8 * 22223, 256, train=True)),
        # float32 rows of odd width
        ('norm_train_odd', _norm('float32', 8 * 1100, 515, train=True)),
    ]
    return [dict(case, name=name) for name, case in named]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


# the largest drawn calls: an attention's multiply-adds and a norm's elements stay within the listed ones'
_MOST_PAIRS = {False: 4096 * 4096 * 2 * 16 * 64 // 2, True: 8400 * 8400 * 8 * 32}


def draw(rng):
    if rng.random() < 0.3:
        dtype = rng.choice(['float16', 'bfloat16', 'float32'])
        C = rng.choice([256, 512, 1024, _log_int(rng, 32, 4096), _log_int(rng, 32, 4096)])
        rows = _log_int(rng, 1, min(170000, 8 * 22223 * 256 // C // (2 if dtype == 'float32' else 1)))
        return _norm(dtype, rows, C, train=rng.random() < 0.6, residual=rng.random() < 0.7)
    dtype = rng.choice(['float16', 'bfloat16', 'float16', 'bfloat16', 'float32'])
    D = rng.choice([16, 32, 32, 64, 64, 128])
    Hk = rng.choice([1, 2, 4, 8])
    H = Hk * rng.choice([1, 1, 2, 4])
    B = _log_int(rng, 1, 16)
    kind = rng.choice(['self', 'self', 'denoise', 'causal', 'few'])
    train = kind != 'few' and rng.random() < 0.6
    # float32 runs an eighth of the largest 16-bit work
    pairs = _MOST_PAIRS[train] // (8 if dtype == 'float32' else 1) // (B * H * D)
    if kind == 'few':
        Q, N = _log_int(rng, 1, 16), _log_int(rng, 64, 22223)
        N = min(N, max(64, pairs // Q), max(64, 2 * 8 * 22223 * 8 * 32 // (B * Hk * D)))
        return _attn(dtype, B, Q, N, H, Hk, D, ragged=rng.random() < 0.7)
    N = _log_int(rng, 1, max(1, min(8400, math.isqrt(pairs))))
    if kind == 'denoise' and N >= 20:
        return _attn(dtype, B, N, N, H, Hk, D, train=train, groups=rng.choice([2, 3, 5]))
    return _attn(dtype, B, N, N, H, Hk, D, train=train, causal=kind == 'causal', ragged=rng.random() < 0.4)


def _lengths(case):
    """Keys left in each image under `ragged`: the first whole, the last about half."""
    B, N = case['B'], case['N']
    return [N - (b * N) // (2 * B) for b in range(B)] if case['ragged'] else [N] * B


def _denoise_mask(case):
    """True = blocked: matching queries do not see denoising ones, denoising groups do not see one another."""
    n, groups = case['Q'], case['groups']
    size = max(1, n // 5 // groups)
    pad = size * groups
    mask = torch.zeros(n, n, dtype=torch.bool)
    mask[pad:, :pad] = True
    group = torch.arange(pad) // size
    mask[:pad, :pad] = group[:, None] != group[None, :]
    return mask


# ---- inputs -------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    dev, dtype = _device(), DTYPES[case['dtype']]
    gen = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, generator=gen, device=dev) * std).to(dtype)

    state = dict(case=case)
    if case['op'] == 'layer_norm':
        rows, C = case['rows'], case['C']
        state['x'] = normal(rows, C)
        state['residual'] = normal(rows, C, std=2.0) if case['residual'] else None
        state['weight'] = (1 + 0.1 * torch.randn(C, generator=gen, device=dev)).to(dtype)
        state['bias'] = normal(C, std=0.1)
        leaves = ('x', 'residual', 'weight', 'bias')
        if case['train']:
            state['grad'] = normal(rows, C, std=0.1)
    else:
        B, Q, N, H, Hk, D = (case[k] for k in ('B', 'Q', 'N', 'H', 'Hk', 'D'))
        if case['packed']:
            state['q'], state['k'], state['v'] = normal(B, N, 3, H, D).unbind(2)
        else:
            state['q'], state['k'], state['v'] = normal(B, Q, H, D), normal(B, N, Hk, D), normal(B, N, Hk, D)
        state['padding'] = None
        if case['ragged']:
            left = torch.tensor(_lengths(case), device=dev)
            state['padding'] = torch.arange(N, device=dev)[None, :] >= left[:, None]
        state['mask'] = _denoise_mask(case).to(dev) if case['groups'] else None
        leaves = ('q', 'k', 'v')
        if case['train']:
            state['grad'] = normal(B, Q, H * D, std=0.1)
    state['leaves'] = [state[k] for k in leaves if state[k] is not None]
    if case['train'] and own:
        for t in state['leaves']:
            t.requires_grad_()
    return state


# ---- one pass -----------------------------------------------------------------------------------------------------

def run(state):
    case = state['case']
    if own:
        return _run_own(state)
    with torch.no_grad():
        if case['op'] == 'layer_norm':
            return _plain_norm(state)
        return _plain_attention(state)


def _run_own(state):
    import marearts_tinydeform_b200 as mt
    case = state['case']

    def call():
        if case['op'] == 'layer_norm':
            return mt.layer_norm(state['x'], state['weight'], state['bias'], residual=state['residual'])
        return mt.attention(state['q'], state['k'], state['v'], key_padding_mask=state['padding'],
                            attn_mask=state['mask'], causal=case['causal'])

    if not case['train']:
        with torch.inference_mode():
            return call()
    out = call()
    return [out.detach()] + list(torch.autograd.grad(out, state['leaves'], state['grad']))


def _blocked(state):
    """The pairs that no query may use, broadcastable to [B, 1, Q, N], or None."""
    case = state['case']
    blocked = None
    if state['padding'] is not None:
        blocked = state['padding'][:, None, None, :]
    if state['mask'] is not None:
        blocked = state['mask'] if blocked is None else blocked | state['mask']
    if case['causal']:
        Q, N = case['Q'], case['N']
        late = torch.ones(Q, N, dtype=torch.bool, device=state['q'].device).triu(N - Q + 1)
        blocked = late if blocked is None else blocked | late
    return blocked


def _plain_attention(state):
    case = state['case']
    B, Q, N, H, Hk, D = (case[k] for k in ('B', 'Q', 'N', 'H', 'Hk', 'D'))
    dtype, G, scale = DTYPES[case['dtype']], H // Hk, 1 / math.sqrt(D)
    q = state['q'].float().transpose(1, 2).reshape(B, Hk, G * Q, D)
    k = state['k'].float().transpose(1, 2)
    v = state['v'].float().transpose(1, 2)
    scores = torch.matmul(q, k.transpose(-1, -2)).mul_(scale).view(B, H, Q, N)
    blocked = _blocked(state)
    if blocked is not None:
        scores.masked_fill_(blocked, -math.inf)
        # a row with no key left has no maximum; its probabilities are zero
        top = scores.amax(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).min)
    else:
        top = scores.amax(-1, keepdim=True)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    p.div_(torch.where(total == 0, 1.0, total))
    out = torch.matmul(p.view(B, Hk, G * Q, N), v)

    def to_rows(t):  # [B, Hk, G * Q, D] -> [B, Q, H, D]
        return t.reshape(B, H, Q, D).transpose(1, 2)

    flat = to_rows(out).reshape(B, Q, H * D).to(dtype)
    if not case['train']:
        return flat
    do = state['grad'].float().view(B, Q, H, D).transpose(1, 2).reshape(B, Hk, G * Q, D)
    p = p.view(B, Hk, G * Q, N)
    dv = torch.matmul(p.transpose(-1, -2), do)
    ds = torch.matmul(do, v.transpose(-1, -2)).sub_((do * out).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    dq = torch.matmul(ds, k)
    dk = torch.matmul(ds.transpose(-1, -2), q)
    return [flat, to_rows(dq).to(dtype), dk.transpose(1, 2).to(dtype), dv.transpose(1, 2).to(dtype)]


def _plain_norm(state):
    case = state['case']
    dtype = DTYPES[case['dtype']]
    s = state['x'].float()
    if state['residual'] is not None:
        s = s + state['residual'].float()
    w, b = state['weight'].float(), state['bias'].float()
    centred = s - s.mean(-1, keepdim=True)
    rstd = torch.rsqrt(centred.square().mean(-1, keepdim=True) + 1e-5)
    xhat = centred * rstd
    y = (xhat * w + b).to(dtype)
    if not case['train']:
        return y
    dy = state['grad'].float()
    g = dy * w
    dx = ((g - g.mean(-1, keepdim=True) - xhat * (g * xhat).mean(-1, keepdim=True)) * rstd).to(dtype)
    # column sums over many rows, in 64 bits
    dw = (dy * xhat).sum(0, dtype=torch.float64).to(dtype)
    db = dy.sum(0, dtype=torch.float64).to(dtype)
    return [y, dx] + ([dx] if state['residual'] is not None else []) + [dw, db]


# ---- what a pass cannot do without --------------------------------------------------------------------------------

def _pairs(case):
    """Allowed (query, key) pairs of one head, over all images."""
    Q, N = case['Q'], case['N']
    if case['groups']:
        return case['B'] * int((~_denoise_mask(case)).sum())
    total = 0
    for left in _lengths(case):
        if case['causal']:
            first = N - Q + 1  # keys open to the first query (Q <= N here)
            full = max(0, min(Q, left - first))  # queries that see fewer than `left` keys
            total += full * first + full * (full - 1) // 2 + (Q - full) * left
        else:
            total += Q * left
    return total


def work(case):
    e = 4 if case['dtype'] == 'float32' else 2
    if case['op'] == 'layer_norm':
        n = case['rows'] * case['C']
        tensors = 2 + case['residual']
        if case['train']:
            tensors += 2  # the output's gradient read, the input's written (it is the residual's as well)
            return {'bytes': e * (tensors * n + 4 * case['C']), 'flops': 22 * n}
        return {'bytes': e * (tensors * n + 2 * case['C']), 'flops': 9 * n}
    B, Q, H, Hk, D = (case[k] for k in ('B', 'Q', 'H', 'Hk', 'D'))
    q_bytes, kv_bytes = e * B * Q * H * D, e * sum(_lengths(case)) * Hk * D
    mask = case['Q'] * case['N'] if case['groups'] else 0
    mask += B * case['N'] if case['ragged'] else 0
    pairs = _pairs(case) * H
    if case['train']:
        return {'bytes': 4 * q_bytes + 4 * kv_bytes + mask, 'flops': 14 * D * pairs}
    return {'bytes': 2 * q_bytes + 2 * kv_bytes + mask, 'flops': 4 * D * pairs}


# ---- the definition in 64 bits ------------------------------------------------------------------------------------

def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        return _exact_norm(state) if case['op'] == 'layer_norm' else _exact_attention(state)


def _exact_norm(state):
    case = state['case']
    parts = []
    dw = db = 0.0
    w = state['weight'].double()
    for i in range(0, case['rows'], 16384):
        s = state['x'][i:i + 16384].double()
        if state['residual'] is not None:
            s = s + state['residual'][i:i + 16384].double()
        n = s.shape[1]
        mu = s.sum(1, keepdim=True) / n
        sigma = torch.sqrt(((s - mu) ** 2).sum(1, keepdim=True) / n + 1e-5)
        z = (s - mu) / sigma
        row = [z * w + state['bias'].double()]
        if case['train']:
            dy = state['grad'][i:i + 16384].double()
            dz = dy * w
            row.append((n * dz - dz.sum(1, keepdim=True) - z * (dz * z).sum(1, keepdim=True)) / (n * sigma))
            dw = dw + torch.einsum('rc,rc->c', dy, z)
            db = db + dy.sum(0)
        parts.append(row)
    whole = [torch.cat(col) for col in zip(*parts)]
    if not case['train']:
        return whole[0]
    return whole + ([whole[1]] if state['residual'] is not None else []) + [dw, db]


def _exact_attention(state):
    case = state['case']
    B, Q, N, H, Hk, D = (case[k] for k in ('B', 'Q', 'N', 'H', 'Hk', 'D'))
    dev = state['q'].device
    out = torch.zeros(B, Q, H, D, dtype=torch.float64, device=dev)
    dq = torch.zeros_like(out)
    dk = torch.zeros(B, N, Hk, D, dtype=torch.float64, device=dev)
    dv = torch.zeros_like(dk)
    rows, cols = torch.arange(Q, device=dev)[:, None], torch.arange(N, device=dev)[None, :]
    for b in range(B):
        may = torch.ones(Q, N, dtype=torch.bool, device=dev)
        if case['ragged']:
            may &= cols < _lengths(case)[b]
        if case['causal']:
            may &= cols <= rows + (N - Q)
        if state['mask'] is not None:
            may &= ~state['mask']
        some = may.any(1, keepdim=True)
        for h in range(H):
            qh = state['q'][b, :, h].double()
            kh, vh = state['k'][b, :, h * Hk // H].double(), state['v'][b, :, h * Hk // H].double()
            s = torch.einsum('id,jd->ij', qh, kh) / D ** 0.5
            s = torch.where(may, s, -math.inf)
            log_total = torch.where(some, torch.logsumexp(s, 1, keepdim=True), 0.0)
            p = torch.exp(s - log_total)
            out[b, :, h] = p @ vh
            if case['train']:
                do = state['grad'][b].view(Q, H, D)[:, h].double()
                dp = torch.einsum('id,jd->ij', do, vh)
                ds = p * (dp - (p * dp).sum(1, keepdim=True)) / D ** 0.5
                dq[b, :, h] = ds @ kh
                dk[b, :, h * Hk // H] += ds.T @ qh
                dv[b, :, h * Hk // H] += p.T @ do
    flat = out.view(B, Q, H * D)
    return [flat, dq, dk, dv] if case['train'] else flat
