"""block_norm (HIP) against a plain 64-bit form, element by element within first-order bounds; its gradients also against differences."""
import pytest
import torch

from tests import token_ref as R

pytestmark = pytest.mark.gpu
T = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}


def make(shape, dtype, kind, gate, seed, weights=True):
    g = torch.Generator(device='cuda').manual_seed(seed)
    r = lambda *s, std=1.0, mean=0.0: (torch.randn(*s, generator=g, device='cuda') * std + mean).to(T[dtype])
    C = shape[-1]
    gs = {'none': None, 'channel': (C,), 'sample': (shape[0], C), 'full': shape}[gate]
    t = {'x': r(*shape, std=2.0), 'y': r(*shape, std=0.7, mean=0.2), 'gate': None if gs is None else r(*gs, std=0.4, mean=0.5)}
    for n in ('pw', 'qw'):
        t[n] = r(C, std=0.2, mean=1.0) if weights else None
    for n in ('pb', 'qb'):
        t[n] = r(C, std=0.2) if weights and kind == 'layer' else None
    t['dx1'], t['dz'] = r(*shape), r(*shape)
    return t


def call(t, kind, scale, post=True, pre=True):
    from panogrf_amd.block_norm import block_norm
    return block_norm(t['x'], t['y'], t['gate'], t['pw'] if post else None, t['pb'] if post else None, t['qw'] if pre else None,
                      t['qb'] if pre else None, post=post, pre=pre, kind=kind, scale=scale)


def check(t, kind, gate, scale, dtype, post=True, pre=True, use=('dx1', 'dz')):
    names = [n for n in ('x', 'y', 'gate', 'pw', 'pb', 'qw', 'qb') if t[n] is not None and (post or n not in ('pw', 'pb')) and (pre or n not in ('qw', 'qb'))]
    leaves = {n: t[n].detach().clone().requires_grad_(True) for n in names}
    x1, z = call({**t, **leaves}, kind, scale, post, pre)
    with torch.no_grad():
        y1, w = call(t, kind, scale, post, pre)
    assert torch.equal(x1, y1) and (z is None and w is None or torch.equal(z, w))
    outs = [(o, t[n]) for o, n in ((x1, 'dx1'), (z, 'dz')) if o is not None and n in use]
    grads = dict(zip(names, torch.autograd.grad([o for o, _ in outs], [leaves[n] for n in names], [g for _, g in outs], allow_unused=True)))
    again = dict(zip(names, torch.autograd.grad([o for o, _ in [(o, g) for (o, g) in zip(call({**t, **leaves}, kind, scale, post, pre), (t['dx1'], t['dz'])) if o is not None and
                                                                 (g is t['dx1'] and 'dx1' in use or g is t['dz'] and 'dz' in use)]],
                                                [leaves[n] for n in names], [g for _, g in outs], allow_unused=True)))
    gb = t['gate']
    if gb is not None and gate == 'sample':
        gb = gb.view(gb.shape[0], *([1] * (t['x'].dim() - 2)), gb.shape[1])
    ref = R.block_norm(t['x'], t['y'], gb, t['pw'] if post else None, t['pb'] if post else None, t['qw'] if pre else None, t['qb'] if pre else None, kind,
                       scale, 1e-6, post, pre, t['dx1'] if 'dx1' in use else None, t['dz'] if 'dz' in use and pre else None, T[dtype])
    bad = {}
    if t['y'] is not None:
        bad['x1'] = R.worst(x1, *ref['x'])
    if pre:
        bad['z'] = R.worst(z, *ref['z'])
    if 'grad_gate_all' in ref and t['gate'] is not None:
        v, e = ref['grad_gate_all']
        over = {'channel': tuple(range(v.dim() - 1)), 'sample': tuple(range(1, v.dim() - 1)), 'full': ()}[gate]
        v, e = (v.sum(over), e.sum(over)) if over else (v, e)
        ref['grad_gate'] = (v, e * 1.01 + R.HALF[T[dtype]] * v.abs() + 6e-8 * (dtype == 'f16') + 1e-300)
    for n in names:
        if grads[n] is None:
            continue
        assert grads[n].dtype == t[n].dtype and torch.equal(grads[n], again[n]), f'gradient of {n} differs from call to call'
        if 'grad_' + n in ref:
            bad[n] = R.worst(grads[n], *ref['grad_' + n])
    assert all(v <= 1 for v in bad.values()), bad


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('kind', ['rms', 'layer'])
@pytest.mark.parametrize('shape,gate', [((1, 1, 1), 'none'), ((3, 5, 16), 'sample'), ((2, 7, 17), 'full'), ((2, 33, 64), 'channel'), ((5, 3, 250), 'sample'),
                                        ((2, 40, 512), 'none'), ((2, 19, 1001), 'full'), ((3, 11, 1024), 'sample'), ((1, 9, 2048), 'channel'),
                                        ((2, 3, 4096), 'full'), ((1, 2, 8191), 'sample'), ((2, 2, 8192), 'channel'), ((4, 1, 96), 'sample')])
def test_values_and_gradients(shape, gate, kind, dtype):
    check(make(shape, dtype, kind, gate, 3), kind, gate, 0.6, dtype)


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
@pytest.mark.parametrize('post,pre,use', [(True, False, ('dx1',)), (False, True, ('dx1', 'dz')), (False, False, ('dx1',)), (True, True, ('dz',)),
                                          (True, True, ('dx1',))])
def test_parts_left_out(post, pre, use, dtype):
    check(make((3, 21, 136), dtype, 'layer', 'sample', 4), 'layer', 'sample', 1.0, dtype, post, pre, use)
    check(make((3, 21, 136), dtype, 'rms', 'full', 5, weights=False), 'rms', 'full', 0.5, dtype, post, pre, use)


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('kind', ['rms', 'layer'])
@pytest.mark.parametrize('C', [1, 3, 17, 24, 100, 136, 520, 1001, 4104])
def test_without_weights_and_gate(C, kind, dtype):
    check(make((2, 5, C), dtype, kind, 'none', 14, weights=False), kind, 'none', 0.7, dtype)


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('kind', ['rms', 'layer'])
@pytest.mark.parametrize('shape,gate', [((1, 1700, 4104), 'channel'), ((2, 850, 8192), 'full'), ((3, 600, 5001), 'sample'), ((1, 1601, 4097), 'none')])
def test_many_long_rows(shape, gate, kind, dtype):
    """Several rows to a workgroup, whose column sums stand in LDS."""
    check(make(shape, dtype, kind, gate, 15), kind, gate, 0.8, dtype)


@pytest.mark.parametrize('kind', ['rms', 'layer'])
def test_norm_alone(kind):
    t = make((4, 6, 5, 64), 'bf16', kind, 'none', 6)
    t['y'] = None
    check(t, kind, 'none', 1.0, 'bf16', post=False, use=('dz',))
    x1, _ = call(t, kind, 1.0, post=False)
    assert x1 is t['x']


@pytest.mark.parametrize('rows', [1, 255, 4097, 70001])
def test_many_rows_small_channels(rows):
    check(make((rows, 16), 'f32', 'layer', 'channel', 7), 'layer', 'channel', 1.0, 'f32')


def test_no_rows_and_strides_and_alignment():
    t = make((2, 8, 64), 'bf16', 'rms', 'channel', 8)
    e = {k: (v[:0] if v is not None and v.dim() == 3 else v) for k, v in t.items()}
    e = {k: (v.requires_grad_(True) if v is not None and k in ('x', 'pw', 'gate') else v) for k, v in e.items()}
    x1, z = call(e, 'rms', 1.0)
    assert x1.shape == z.shape == (0, 8, 64)
    (x1.sum() + z.sum()).backward()
    assert float(e['pw'].grad.abs().sum()) == 0 and float(e['gate'].grad.abs().sum()) == 0
    t = make((2, 8, 64), 'bf16', 'rms', 'channel', 8)
    want = call(t, 'rms', 0.5)
    wide = torch.zeros(2, 8, 130, dtype=torch.bfloat16, device='cuda')
    wide[..., 1:65], wide[..., 65:129] = t['x'], t['y']
    odd = {**t, 'x': wide[..., 1:65], 'y': wide[..., 65:129]}
    assert all(torch.equal(a, b) for a, b in zip(call(odd, 'rms', 0.5), want))
    flat = torch.zeros(2 * 8 * 64 + 1, dtype=torch.bfloat16, device='cuda')      # rows that start at odd addresses
    flat[1:] = t['x'].reshape(-1)
    got = call({**t, 'x': flat[1:].view(2, 8, 64)}, 'rms', 0.5)
    for a, b in zip(got, want):                                                  # (sums in another order: float arithmetic, one step of the type)
        assert float((a.float() - b.float()).abs().max()) <= 2 ** -7 * float(b.float().abs().max())
    turned = t['x'].transpose(0, 1).contiguous().transpose(0, 1)
    assert all(torch.equal(a, b) for a, b in zip(call({**t, 'x': turned}, 'rms', 0.5), want))


def test_a_row_that_is_not_finite_stays_alone():
    t = make((1, 9, 200), 'f32', 'layer', 'none', 9)
    want = call(t, 'layer', 1.0)
    t['x'][0, 4, 3], t['y'][0, 6, 0] = float('nan'), float('inf')
    got = call(t, 'layer', 1.0)
    keep = [i for i in range(9) if i not in (4, 6)]
    assert all(torch.equal(a[0, keep], b[0, keep]) for a, b in zip(got, want))
    assert torch.isnan(got[1][0, 4]).all() and torch.isnan(got[0][0, 6]).any()


def test_against_differences():
    """Along one direction of every input at once, in float: the difference quotient of a weighted sum of the outputs.  Its truncation error is measured on the 64-bit
    form, its rounding is bounded by the outputs' bounds over the step."""
    t = make((2, 5, 48), 'f32', 'layer', 'sample', 10)
    names = ('x', 'y', 'gate', 'pw', 'pb', 'qw', 'qb')
    g = torch.Generator(device='cuda').manual_seed(1)
    way = {n: torch.randn(t[n].shape, generator=g, device='cuda') for n in names}
    h = 2.0 ** -7
    leaves = {n: t[n].clone().requires_grad_(True) for n in names}
    outs = call({**t, **leaves}, 'layer', 0.5)
    grads = torch.autograd.grad(outs, [leaves[n] for n in names], [t['dx1'], t['dz']])
    slope = sum(float((way[n].double() * d.double()).sum()) for n, d in zip(names, grads))
    quotient, exact, room = 0.0, 0.0, 0.0
    for s in (1, -1):
        m = {**t, **{n: t[n] + s * h * way[n] for n in names}}
        o = call(m, 'layer', 0.5)
        quotient += s * sum(float((a.double() * b.double()).sum()) for a, b in zip(o, (t['dx1'], t['dz']))) / (2 * h)
        r = R.block_norm(m['x'], m['y'], m['gate'][:, None], m['pw'], m['pb'], m['qw'], m['qb'], 'layer', 0.5, 1e-6, True, True, None, None, torch.float32)
        exact += s * sum(float((r[k][0] * t[d].double()).sum()) for k, d in (('x', 'dx1'), ('z', 'dz'))) / (2 * h)
        room += sum(float((r[k][1] * t[d].double().abs()).sum()) for k, d in (('x', 'dx1'), ('z', 'dz'))) / (2 * h)
    assert abs(quotient - exact) <= room
    assert abs(exact - slope) <= 0.02 * abs(slope) + room      # (a central difference's error is of order h^2)


def test_graph_replays():
    t = make((2, 50, 256), 'bf16', 'rms', 'sample', 11)
    names = ('x', 'y', 'gate', 'pw', 'qw')
    fixed = {**t, **{n: t[n].clone().requires_grad_(True) for n in names}}

    def step():
        return list(call(fixed, 'rms', 0.5)), None

    def whole():
        o = call(fixed, 'rms', 0.5)
        return [v.detach() for v in o] + list(torch.autograd.grad(o, [fixed[n] for n in names], [fixed['dx1'], fixed['dz']]))
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        whole()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = whole()
    for seed in (20, 21, 22):
        new = make((2, 50, 256), 'bf16', 'rms', 'sample', seed)
        with torch.no_grad():
            for n in names + ('dx1', 'dz'):
                fixed[n].copy_(new[n])
        graph.replay()
        torch.cuda.synchronize()
        got = [v.clone() for v in held]
        assert all(torch.equal(a, b) for a, b in zip(got, whole()))


def test_on_another_stream():
    t = make((4, 64, 512), 'f16', 'rms', 'channel', 12)
    want = call(t, 'rms', 1.0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call(t, 'rms', 1.0)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
