"""Work that the token operators of the framework are timed on: block_norm (norms before and after a block, gate and residual scale), rotary
(rotary positions) and diff_attention (differential attention, in training, over a prompt and over a cache).

`own` false computes each in elementary torch operations in 32 bits, `own` true through panogrf_amd's entry points."""
import math

import torch

own = False

_TYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}
_SIZE = {'f32': 4, 'bf16': 2, 'f16': 2}


# ------------------------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one new token for each of 16 streams, between two blocks of a served model: latency
        dict(name='norm-token', op='block_norm', dtype='bf16', kind='rms', b=16, n=1, c=1024, gate='channel', scale=0.5, train=False),
        # the ray transformer's 16-channel LayerNorm over a training batch (2 048 rays x 64 samples), ungated residual
        dict(name='norm-rays', op='block_norm', dtype='f32', kind='layer', b=2048, n=64, c=16, gate='none', scale=1.0, train=True),
        # a token net over four panoramas of 512 x 1024 in patches of 8, gated by each panorama's own vector, in training
        dict(name='norm-panorama', op='block_norm', dtype='bf16', kind='rms', b=4, n=8192, c=1024, gate='sample', scale=0.7, train=True),
        # odd rows and channels with a gate for each value, in training
        dict(name='norm-odd', op='block_norm', dtype='f16', kind='layer', b=3, n=1999, c=1001, gate='full', scale=1.0, train=True),
        # one new token for each of 32 streams, far into a long context with scaled frequencies: latency
        dict(name='rotary-token', op='rotary', dtype='bf16', layout='half', b=32, n=1, h=16, hk=4, d=128, rot=128, scaling='parts', factor=8.0,
             first=100000, pos='stream', train=False),
        # queries and keys of a token net over four panoramas (8 192 patches), half of each head rotated, in training
        dict(name='rotary-panorama', op='rotary', dtype='bf16', layout='half', b=4, n=8192, h=16, hk=16, d=64, rot=32, scaling='none', factor=1.0,
             first=0, pos='shared', train=True),
        # the samples of 2 048 rays at their own continuous depths, interleaved pairs, in training
        dict(name='rotary-rays', op='rotary', dtype='f32', layout='interleaved', b=2048, n=64, h=4, hk=4, d=32, rot=32, scaling='linear', factor=4.0,
             first=0, pos='depth', train=True),
        # attention along 2 048 rays of 64 samples, samples that no source view sees masked (some rays wholly), in training
        dict(name='attention-rays', op='attention', mode='train', dtype='f32', b=2048, n=64, m=64, h=4, hk=4, d=32, causal=False, mask='holes'),
        # a token net over two panoramas (8 192 patches each), in training
        dict(name='attention-panorama', op='attention', mode='train', dtype='bf16', b=2, n=8192, m=8192, h=8, hk=8, d=64, causal=False, mask='none'),
        # the second half of a long prompt, odd lengths, four query heads on each key head, views of a fused projection
        dict(name='attention-prompt', op='attention', mode='prompt', dtype='bf16', b=1, n=4001, m=8093, h=16, hk=4, d=128, causal=True, mask='none'),
        # one token for each of 32 streams over caches of up to 16 384 tokens, ragged
        dict(name='attention-cache', op='attention', mode='cache', dtype='bf16', b=32, n=1, m=16384, h=32, hk=8, d=64, causal=True, mask='none'),
        # one token of one stream over a short cache: latency
        dict(name='attention-token', op='attention', mode='cache', dtype='f16', b=1, n=1, m=500, h=8, hk=2, d=64, causal=True, mask='none'),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(['block_norm', 'rotary', 'attention', 'attention'])
    dtype = rng.choice(['f32', 'bf16', 'f16'])
    if op == 'block_norm':
        c = _log(rng, 8, 8192)
        c = c - c % 8 if c > 16 and rng.random() < 0.6 else c
        b = _log(rng, 1, 32)
        n = _log(rng, 1, max(1, min(16384, 4 * 8192 * 1024 // (b * c))))
        kind = rng.choice(['rms', 'layer'])
        return dict(op=op, dtype=dtype, kind=kind, b=b, n=n, c=c, gate=rng.choice(['none', 'channel', 'sample', 'full']),
                    scale=rng.choice([1.0, 0.5, 0.25]), train=rng.random() < 0.6)
    if op == 'rotary':
        d = rng.choice([16, 32, 48, 64, 80, 96, 128, 256])
        rot = d if rng.random() < 0.5 else max(2, 2 * rng.randint(1, d // 2))
        hk = rng.choice([1, 2, 4, 8, 16])
        h = hk * rng.choice([1, 2, 4])
        b = _log(rng, 1, 64)
        n = _log(rng, 1, max(1, min(16384, 4 * 8192 * 32 * 64 // (b * (h + hk) * d))))
        scaling = rng.choice(['none', 'linear', 'ntk', 'parts']) if rot > 2 else 'none'
        return dict(op=op, dtype=dtype, layout=rng.choice(['half', 'interleaved']), b=b, n=n, h=h, hk=hk, d=d, rot=rot, scaling=scaling,
                    factor=1.0 if scaling == 'none' else rng.choice([2.0, 8.0, 32.0]), first=rng.choice([0, 7, 4000, 1000000]),
                    pos=rng.choice(['shared', 'stream', 'depth']), train=rng.random() < 0.5)
    d = rng.choice([32, 64, 64, 128])
    hk = rng.choice([1, 2, 4, 8])
    g = rng.choice([1, 1, 2, 4, 8])
    mode = rng.choice(['train', 'prompt', 'cache'])
    if mode == 'cache':
        b = _log(rng, 1, 64)
        m = _log(rng, 16, max(16, min(16384, 32 * 16384 * 8 * 64 // (b * hk * d))))
        return dict(op=op, mode=mode, dtype=dtype, b=b, n=rng.choice([1, 1, 1, 2, 5]), m=m, h=hk * g, hk=hk, d=d, causal=True, mask='none')
    b = _log(rng, 1, 512)
    pairs = min(2 * 8 * 8192 * 8192, 2 * 8 * 8192 * 8192 * 64 // d // (4 if dtype == 'f32' else 1))
    most = max(8, min(8192, int(math.sqrt(pairs / (b * hk * g)))))
    n = _log(rng, 4, most)
    m = n if rng.random() < 0.5 else min(8192, n + rng.randint(0, n))
    m = m if b * hk * g * n * m <= pairs else n
    return dict(op=op, mode=mode, dtype=dtype, b=b, n=n, m=m, h=hk * g, hk=hk, d=d, causal=rng.random() < 0.5, mask=rng.choice(['none', 'none', 'holes', 'tail']))


def work(case):
    c, e = case, _SIZE[case['dtype']]
    if c['op'] == 'block_norm':
        full = 1 if c['gate'] == 'full' else 0
        values = c['b'] * c['n'] * c['c']
        passes = 4 + full + ((6 + 2 * full) if c['train'] else 0)
        return {'bytes': values * e * passes, 'flops': values * (38 if c['train'] else 14)}
    if c['op'] == 'rotary':
        values = c['b'] * c['n'] * (c['h'] + c['hk']) * c['d']
        turns = 2 if c['train'] else 1
        return {'bytes': 2 * values * e * turns, 'flops': 3 * c['b'] * c['n'] * (c['h'] + c['hk']) * c['rot'] * turns}
    q, kv = c['b'] * c['n'] * c['h'] * 2 * c['d'], c['b'] * c['m'] * c['hk'] * 4 * c['d']
    pairs = c['b'] * c['h'] * c['n'] * c['m']
    if c['mode'] == 'cache':  # lengths are spread evenly over a quarter of the cache to the whole of it
        share = 0.625 if c['b'] > 1 else 1.0
        return {'bytes': e * (2 * q + kv * share), 'flops': 12 * pairs * share * c['d']}
    if c['causal']:
        pairs -= c['b'] * c['h'] * c['n'] * (c['n'] - 1) // 2
    if c['mode'] == 'train':
        return {'bytes': e * (5 * q + 3 * kv), 'flops': 32 * pairs * c['d']}
    return {'bytes': e * (2 * q + kv), 'flops': 12 * pairs * c['d']}


# ----------------------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    c, dt = case, _TYPES[case['dtype']]
    g = torch.Generator(device='cuda').manual_seed(seed)

    def normal(*shape, std=1.0, mean=0.0):
        return (torch.randn(*shape, generator=g, device='cuda') * std + mean).to(dt)

    s = {'case': dict(case)}
    if c['op'] == 'block_norm':
        shape = (c['b'], c['n'], c['c'])
        s['x'] = normal(*shape, std=2.0)
        s['y'] = normal(*shape, std=0.7, mean=0.1)
        gates = {'none': None, 'channel': (c['c'],), 'sample': (c['b'], c['c']), 'full': shape}[c['gate']]
        s['gate'] = None if gates is None else normal(*gates, std=0.3, mean=0.5)
        s['post_w'], s['pre_w'] = normal(c['c'], std=0.1, mean=1.0), normal(c['c'], std=0.1, mean=1.0)
        layer = c['kind'] == 'layer'
        s['post_b'], s['pre_b'] = (normal(c['c'], std=0.1), normal(c['c'], std=0.1)) if layer else (None, None)
        s['leaves'] = [k for k in ('x', 'y', 'gate', 'post_w', 'post_b', 'pre_w', 'pre_b') if s[k] is not None]
        if c['train']:
            s['dx'], s['dz'] = normal(*shape), normal(*shape)
    elif c['op'] == 'rotary':
        s['q'], s['k'] = normal(c['b'], c['n'], c['h'], c['d']), normal(c['b'], c['n'], c['hk'], c['d'])
        if c['pos'] == 'depth':
            s['positions'] = torch.rand(c['b'], c['n'], generator=g, device='cuda').mul_(14.5).add_(0.5 + c['first']).sort(-1)[0]
        elif c['pos'] == 'stream':
            s['positions'] = c['first'] + torch.randint(0, 4096, (c['b'], 1), generator=g, device='cuda') + torch.arange(c['n'], device='cuda')
        else:
            s['positions'] = c['first'] + torch.arange(c['n'], device='cuda')
        s['leaves'] = ['q', 'k']
        if c['train']:
            s['dq'], s['dk'] = normal(c['b'], c['n'], c['h'], c['d']), normal(c['b'], c['n'], c['hk'], c['d'])
    else:
        b, n, m, h, hk, d = (c[x] for x in ('b', 'n', 'm', 'h', 'hk', 'd'))
        s['lam'] = (torch.rand(h, generator=g, device='cuda') * 0.6 + 0.2).to(dt)
        s['mask'] = s['lengths'] = None
        s['q'] = normal(b, n, h, 2, d)
        if c['mode'] == 'prompt':  # a projection makes keys and values side by side
            kv = normal(b, m, hk, 4 * d)
            s['k'], s['v'] = kv[..., :2 * d].unflatten(-1, (2, d)), kv[..., 2 * d:]
        else:
            s['k'], s['v'] = normal(b, m, hk, 2, d), normal(b, m, hk, 2 * d)
        if c['mode'] == 'cache':
            low = max(c['n'], m // 4)
            even = torch.linspace(low, m, b, device='cuda').round().int() if b > 1 else torch.tensor([m], dtype=torch.int32, device='cuda')
            s['lengths'] = even[torch.randperm(b, generator=g, device='cuda')]
        elif c['mask'] == 'holes':
            s['mask'] = torch.rand(b, m, generator=g, device='cuda') > 0.25
            s['mask'][::37] = False
        elif c['mask'] == 'tail':
            s['mask'] = torch.arange(m, device='cuda') < torch.randint(1, m + 1, (b, 1), generator=g, device='cuda')
        s['leaves'] = ['q', 'k', 'v', 'lam']
        if c['mode'] == 'train':
            s['dout'] = normal(b, n, h, 2 * d)
    if c.get('train') or c.get('mode') == 'train':
        for k in s['leaves']:
            s[k].requires_grad_(True)
    return s


# ------------------------------------------------------------------------------------------------------------ plain forms
def _norm(a, w, b, kind, eps=1e-6):
    if kind == 'layer':
        a = a - a.mean(-1, keepdim=True)
    r = a * torch.rsqrt((a * a).mean(-1, keepdim=True) + eps) * w.float()
    return r if b is None else r + b.float()


def _plain_block_norm(s):
    c = s['case']
    x, y = s['x'].float(), _norm(s['y'].float(), s['post_w'], s['post_b'], c['kind'])
    if s['gate'] is not None:
        gate = s['gate'].float()
        y = y * (gate.unsqueeze(1) if c['gate'] == 'sample' else gate)
    x = x + c['scale'] * y
    z = _norm(x, s['pre_w'], s['pre_b'], c['kind'])
    return x.to(s['x'].dtype), z.to(s['x'].dtype)


def _frequencies(c, base=10000.0, trained=4096, low=1.0, high=32.0):
    """Radians by position of each rotated pair, in 64 bits."""
    rot = c['rot']
    if c['scaling'] == 'ntk':
        base = base * c['factor'] ** (rot / (rot - 2))
    f = base ** (-torch.arange(0, rot, 2, dtype=torch.float64, device='cuda') / rot)
    if c['scaling'] == 'linear':
        f = f / c['factor']
    elif c['scaling'] == 'parts':
        keep = ((trained * f / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
        f = f * (keep + (1 - keep) / c['factor'])
    return f


def _turn(x, cos, sin, c):
    rot, v = c['rot'], x.float()
    if c['layout'] == 'half':
        a, b = v[..., :rot // 2], v[..., rot // 2:rot]
        r = torch.cat([a * cos - b * sin, b * cos + a * sin, v[..., rot:]], -1)
    else:
        a, b = v[..., 0:rot:2], v[..., 1:rot:2]
        r = torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2), v[..., rot:]], -1)
    return r.to(x.dtype)


def _plain_rotary(s):
    c = s['case']
    angle = (s['positions'].double().unsqueeze(-1) * _frequencies(c)).unsqueeze(-2)
    cos, sin = angle.cos().float(), angle.sin().float()
    return _turn(s['q'], cos, sin, c), _turn(s['k'], cos, sin, c)


def _allowed(s):
    """Which keys each query may see, broadcast to [b, 1, 1, 1, n, m]; None where it is all of them."""
    c, see = s['case'], None
    n, m = c['n'], c['m']
    j, i = torch.arange(m, device='cuda'), torch.arange(n, device='cuda').unsqueeze(-1)
    if s['lengths'] is not None:
        see = j <= i + (s['lengths'].view(-1, 1, 1) - n)
    elif c['causal']:
        see = (j <= i + (m - n)).unsqueeze(0)
    if s['mask'] is not None:
        see = s['mask'].unsqueeze(1) if see is None else see & s['mask'].unsqueeze(1)
    return None if see is None else see[:, None, None, None]


def _plain_attention(s):
    c = s['case']
    b, n, m, h, hk, d = (c[x] for x in ('b', 'n', 'm', 'h', 'hk', 'd'))
    q = s['q'].float().view(b, n, hk, h // hk, 2, d).permute(0, 2, 4, 3, 1, 5).reshape(b, hk, 2, h // hk * n, d) * d ** -0.5
    k = s['k'].float().permute(0, 2, 3, 4, 1)
    v = s['v'].float().transpose(1, 2)
    scores = torch.matmul(q, k).view(b, hk, 2, h // hk, n, m)
    see = _allowed(s)
    if see is not None:
        scores = scores.masked_fill(~see, -math.inf)
    top = scores.detach().amax(-1, keepdim=True)
    e = torch.exp(scores - top.masked_fill(top == -math.inf, 0.0))
    total = e.sum(-1, keepdim=True)
    p = e / total.masked_fill(total == 0, 1.0)
    p = p[:, :, 0] - s['lam'].float().view(hk, h // hk, 1, 1) * p[:, :, 1]
    out = torch.matmul(p.reshape(b, hk, h // hk * n, m), v)
    return out.view(b, hk, h // hk, n, 2 * d).permute(0, 3, 1, 2, 4).reshape(b, n, h, 2 * d).to(s['q'].dtype)


def run(state):
    s, c = state, state['case']
    leaves = s['leaves']
    if c['op'] == 'block_norm':
        if own:
            from panogrf_amd.block_norm import block_norm
            x, z = block_norm(s['x'], s['y'], gate=s['gate'], post_weight=s['post_w'], post_bias=s['post_b'], pre_weight=s['pre_w'],
                              pre_bias=s['pre_b'], kind=c['kind'], scale=c['scale'], eps=1e-6)
        else:
            x, z = _plain_block_norm(s)
        got, outs, grads = {'x': x, 'z': z}, [x, z], [s.get('dx'), s.get('dz')]
    elif c['op'] == 'rotary':
        if own:
            from panogrf_amd.rotary import rotary
            q, k = rotary(s['q'], s['k'], s['positions'], rotary_dim=c['rot'], layout=c['layout'], base=10000.0,
                          scaling=None if c['scaling'] == 'none' else c['scaling'], factor=c['factor'], trained_length=4096, low=1.0, high=32.0)
        else:
            q, k = _plain_rotary(s)
        got, outs, grads = {'q': q, 'k': k}, [q, k], [s.get('dq'), s.get('dk')]
    else:
        if own:
            from panogrf_amd.attention import diff_attention, diff_attention_cached
            if c['mode'] == 'cache':
                out = diff_attention_cached(s['q'], s['k'], s['v'], s['lam'], s['lengths'])
            else:
                out = diff_attention(s['q'], s['k'], s['v'], s['lam'], causal=c['causal'], key_mask=s['mask'])
        else:
            out = _plain_attention(s)
        got, outs, grads = {'out': out}, [out], [s.get('dout')]
    if grads[0] is None:
        return got
    got = {k: v.detach() for k, v in got.items()}
    for name, grad in zip(leaves, torch.autograd.grad(outs, [s[k] for k in leaves], grads)):
        got['grad_' + name] = grad
    return got


# ------------------------------------------------------------------------------------------------------- in 64 bits, apart
def _exact_norm(a, w, b, kind, g):
    """A norm over the last axis and its gradients for the upstream gradient g (None: the norm alone)."""
    mean = a.mean(-1, keepdim=True) if kind == 'layer' else 0.0
    r = 1.0 / ((a - mean).pow(2).mean(-1, keepdim=True) + 1e-6).sqrt()
    hat = (a - mean) * r
    out = hat * w + (0.0 if b is None else b)
    if g is None:
        return out, None, None
    t = g * w
    da = t - hat * (t * hat).mean(-1, keepdim=True)
    if kind == 'layer':
        da = da - t.mean(-1, keepdim=True)
    return out, da * r, (g * hat).sum((0, 1))


def _exact_block_norm(s):
    c = s['case']
    x, y, pw, qw = (s[k].detach().double() for k in ('x', 'y', 'post_w', 'pre_w'))
    pb, qb = (None if s[k] is None else s[k].detach().double() for k in ('post_b', 'pre_b'))
    gate = torch.ones((), dtype=torch.float64, device='cuda') if s['gate'] is None else s['gate'].detach().double()
    gate = gate[:, None] if c['gate'] == 'sample' else gate
    u = _exact_norm(y, pw, pb, c['kind'], None)[0]
    x1 = x + c['scale'] * gate * u
    if not c['train']:
        return {'x': x1, 'z': _exact_norm(x1, qw, qb, c['kind'], None)[0]}
    dz = s['dz'].double()
    z, dh, dqw = _exact_norm(x1, qw, qb, c['kind'], dz)
    dh = dh + s['dx'].double()
    du = c['scale'] * gate * dh
    _, dy, dpw = _exact_norm(y, pw, pb, c['kind'], du)
    dg = c['scale'] * dh * u
    out = {'x': x1, 'z': z, 'grad_x': dh, 'grad_y': dy, 'grad_post_w': dpw, 'grad_pre_w': dqw}
    if s['gate'] is not None:
        out['grad_gate'] = {'channel': lambda: dg.sum((0, 1)), 'sample': lambda: dg.sum(1), 'full': lambda: dg}[c['gate']]()
    if pb is not None:
        out['grad_post_b'], out['grad_pre_b'] = du.sum((0, 1)), dz.sum((0, 1))
    return out


def _exact_rotary(s):
    c = s['case']
    rot, place = c['rot'], s['positions'].double()
    place = place.expand(c['b'], c['n']) if place.dim() == 1 else place
    base = 10000.0 * (c['factor'] ** (rot / (rot - 2)) if c['scaling'] == 'ntk' else 1.0)
    rates = []
    for i in range(rot // 2):
        f = base ** (-2.0 * i / rot)
        if c['scaling'] == 'linear':
            f /= c['factor']
        elif c['scaling'] == 'parts':
            share = min(1.0, max(0.0, (4096 * f / (2 * math.pi) - 1.0) / 31.0))
            f = f * share + f / c['factor'] * (1 - share)
        rates.append(f)
    z = torch.polar(torch.ones((), dtype=torch.float64, device='cuda'), place[..., None] * torch.tensor(rates, dtype=torch.float64, device='cuda'))
    first = list(range(0, rot // 2)) if c['layout'] == 'half' else list(range(0, rot, 2))
    second = list(range(rot // 2, rot)) if c['layout'] == 'half' else list(range(1, rot, 2))

    def turned(x, phase):
        x = x.detach().double()
        w = torch.complex(x[..., first], x[..., second]) * phase[:, :, None]
        x = x.clone()
        x[..., first], x[..., second] = w.real, w.imag
        return x

    out = {'q': turned(s['q'], z), 'k': turned(s['k'], z)}
    if c['train']:
        out['grad_q'], out['grad_k'] = turned(s['dq'], z.conj()), turned(s['dk'], z.conj())
    return out


def _exact_attention(s):
    c = s['case']
    b, n, m, h, hk, d = (c[x] for x in ('b', 'n', 'm', 'h', 'hk', 'd'))
    train = c['mode'] == 'train'
    f64 = dict(dtype=torch.float64, device='cuda')
    out = torch.zeros(b, n, h, 2 * d, **f64)
    dq, dk, dv, dlam = torch.zeros(b, n, h, 2, d, **f64), torch.zeros(b, m, hk, 2, d, **f64), torch.zeros(b, m, hk, 2 * d, **f64), torch.zeros(h, **f64)
    at_once = max(1, (1 << 26) // (n * m))
    for b0 in range(0, b, at_once):
        rows = slice(b0, min(b, b0 + at_once))
        see = torch.ones(1, n, m, dtype=torch.bool, device='cuda')
        behind = s['lengths'][rows].long().view(-1, 1, 1) if s['lengths'] is not None else torch.full((1, 1, 1), m, device='cuda')
        if c['causal']:
            see = torch.arange(m, device='cuda').view(1, 1, m) - torch.arange(n, device='cuda').view(1, n, 1) <= behind - n
        if s['mask'] is not None:
            see = see & s['mask'][rows][:, None, :]
        for head in range(h):
            at = head // (h // hk)
            v, lam = s['v'][rows, :, at].detach().double(), float(s['lam'][head].detach())
            p, o = [], []
            for i in (0, 1):
                a = torch.bmm(s['q'][rows, :, head, i].detach().double(), s['k'][rows, :, at, i].detach().double().transpose(1, 2)) / math.sqrt(d)
                a = torch.where(see, a, -math.inf)
                w = torch.where(see, (a - a.max(-1, keepdim=True)[0].clamp_min(-1e300)).exp(), 0.0)
                p.append(w / w.sum(-1, keepdim=True).clamp_min(1e-300))
                o.append(torch.bmm(p[i], v))
            out[rows, :, head] = o[0] - lam * o[1]
            if not train:
                continue
            do = s['dout'][rows, :, head].double()
            back = torch.bmm(do, v.transpose(1, 2))
            dv[rows, :, at] += torch.bmm((p[0] - lam * p[1]).transpose(1, 2), do)
            dlam[head] -= (do * o[1]).sum()
            for i, sign in ((0, 1.0), (1, -lam)):
                da = sign * p[i] * (back - (do * o[i]).sum(-1, keepdim=True)) / math.sqrt(d)
                dq[rows, :, head, i] = torch.bmm(da, s['k'][rows, :, at, i].detach().double())
                dk[rows, :, at, i] += torch.bmm(da.transpose(1, 2), s['q'][rows, :, head, i].detach().double())
    if not train:
        return {'out': out}
    return {'out': out, 'grad_q': dq, 'grad_k': dk, 'grad_v': dv, 'grad_lam': dlam}


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {'block_norm': _exact_block_norm, 'rotary': _exact_rotary, 'attention': _exact_attention}[case['op']](s)
