"""rotary (HIP) against the turn in 64 bits: within half a step of the type and a few of float's."""
import math

import pytest
import torch

from tests import token_ref as R

pytestmark = pytest.mark.gpu
T = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}


def turned(x, positions, rot, layout, back=False, base=10000.0, scaling=None, factor=1.0, trained_length=4096, low=1.0, high=32.0, magnitude=1.0):
    """-> (value, bound): sine and cosine of the double angle reduced to a float fraction of a turn are off by at most 8 U (2 pi / 2 for the fraction, 2 each for
    the function and the products), those of a position p by p 2^-48 more."""
    B, N, D = x.shape[0], x.shape[1], x.shape[-1]
    p = positions.double().expand(B, N)
    b = base * factor ** (rot / (rot - 2)) if scaling == 'ntk' else base
    f = torch.tensor([b ** (-2 * i / rot) for i in range(rot // 2)], dtype=torch.float64, device=x.device)
    if scaling == 'linear':
        f = f / factor
    if scaling == 'parts':
        keep = ((trained_length * f / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
        f = f * keep + f * (1 - keep) / factor
    angle = (p[..., None] * f * (-1 if back else 1)).reshape(B, N, *([1] * (x.dim() - 3)), rot // 2)
    i, j = (torch.arange(rot // 2), torch.arange(rot // 2) + rot // 2) if layout == 'half' else (torch.arange(0, rot, 2), torch.arange(1, rot, 2))
    v = x.detach().double()
    u, w = v[..., i], v[..., j]
    out, bound = v.clone(), torch.zeros_like(v)
    e = (u.abs() + w.abs()) * abs(magnitude) * (8 * R.U + float(p.abs().max() if p.numel() else 0) * 2.0 ** -48)
    out[..., i], out[..., j] = (u * angle.cos() - w * angle.sin()) * magnitude, (w * angle.cos() + u * angle.sin()) * magnitude
    bound[..., i], bound[..., j] = e, e
    return out, bound * 1.01 + R.HALF[x.dtype] * out.abs() * (bound > 0) + (6e-8 if x.dtype == torch.float16 else 0) + 1e-300


def positions_of(kind, B, N, first, g):
    if kind == 'depth':
        return torch.rand(B, N, generator=g, device='cuda') * 15 + first
    p = first + torch.arange(N, device='cuda')
    p = p + torch.randint(0, 999, (B, 1), generator=g, device='cuda') if kind in ('stream', 'stream32') else p
    return p.int() if kind == 'stream32' else p.double() if kind == 'double' else p


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('layout', ['half', 'interleaved'])
@pytest.mark.parametrize('B,N,H,HK,D,rot,kind,first', [(1, 1, 1, 1, 2, 2, 'shared', 0), (2, 1, 4, 1, 64, 64, 'stream', 100000), (3, 17, 2, 2, 48, 22, 'depth', 0),
                                                       (2, 130, 3, 1, 80, 64, 'shared', 1 << 30), (1, 33, 5, 0, 33, 30, 'stream32', 7),
                                                       (2, 2500, 2, 1, 32, 16, 'double', -40), (1, 3, 2, 2, 256, 256, 'stream', 5), (1, 5, 70, 9, 128, 38, 'shared', 9)])
def test_values_and_gradients(B, N, H, HK, D, rot, kind, first, layout, dtype):
    from panogrf_amd.rotary import rotary
    g = torch.Generator(device='cuda').manual_seed(B * 1000 + N + D)
    q = torch.randn(B, N, H, D, generator=g, device='cuda').to(T[dtype]).requires_grad_(True)
    k = torch.randn(B, N, HK, D, generator=g, device='cuda').to(T[dtype]).requires_grad_(True) if HK else None
    p = positions_of(kind, B, N, first, g)
    qo, ko = rotary(q, k, p, rotary_dim=rot, layout=layout)
    assert R.worst(qo, *turned(q, p, rot, layout)) <= 1
    assert torch.equal(qo[..., rot:], q[..., rot:])
    gq = torch.randn(q.shape, generator=g, device='cuda').to(T[dtype])
    if k is None:
        assert ko is None
        qo.backward(gq)
    else:
        assert R.worst(ko, *turned(k, p, rot, layout)) <= 1
        gk = torch.randn(k.shape, generator=g, device='cuda').to(T[dtype])
        torch.autograd.backward([qo, ko], [gq, gk])
        assert R.worst(k.grad, *turned(gk, p, rot, layout, back=True)) <= 1
    assert R.worst(q.grad, *turned(gq, p, rot, layout, back=True)) <= 1


@pytest.mark.parametrize('kw', [dict(scaling='linear', factor=8.0), dict(scaling='ntk', factor=32.0), dict(scaling='parts', factor=8.0, trained_length=512, low=1.0, high=4.0),
                                dict(base=500000.0, magnitude=1.25), dict(scaling='parts', factor=2.0, magnitude=-0.5)])
def test_scaled_for_long_contexts(kw):
    from panogrf_amd.rotary import rotary
    q = torch.randn(2, 40, 4, 64, device='cuda')
    p = torch.arange(40, device='cuda') * 40000
    assert R.worst(rotary(q, None, p, **kw)[0], *turned(q, p, 64, 'half', **kw)) <= 1


def test_views_maps_and_other_strides():
    from panogrf_amd.rotary import rotary
    g = torch.Generator(device='cuda').manual_seed(2)
    fused = torch.randn(2, 9, 3 * 4 * 2 * 32 + 3, generator=g, device='cuda', dtype=torch.float32).to(torch.bfloat16)
    q, k = fused[..., :256].unflatten(-1, (4, 2, 32)), fused[..., 257:513].unflatten(-1, (4, 2, 32))
    p = torch.arange(9, device='cuda')
    qo, ko = rotary(q, k, p, rotary_dim=24)
    assert qo.shape == q.shape and R.worst(qo, *turned(q, p, 24, 'half')) <= 1 and R.worst(ko, *turned(k, p, 24, 'half')) <= 1
    across = torch.randn(2, 4, 9, 64, device='cuda').transpose(1, 2)                      # [B, H, N, D] memory
    assert R.worst(rotary(across, None, p, layout='interleaved')[0], *turned(across, p, 64, 'interleaved')) <= 1
    spread = torch.randn(2, 9, 4, 128, device='cuda')[..., ::2]
    assert R.worst(rotary(spread, None, p)[0], *turned(spread, p, 64, 'half')) <= 1
    once = torch.randn(1, 9, 1, 64, device='cuda', requires_grad=True)
    rotary(once.expand(3, 9, 4, 64), None, p)[0].sum().backward()                          # a broadcast input's gradient is summed
    assert once.grad.shape == once.shape
    want = 12 * turned(torch.ones(1, 9, 1, 64, device='cuda'), p, 64, 'half', back=True)[0]
    assert float((once.grad.double() - want).abs().max()) < 12 * 32 * R.U * 2


def test_one_of_two_gradients_and_empty():
    from panogrf_amd.rotary import rotary
    q, k = (torch.randn(1, 4, 2, 16, device='cuda', requires_grad=True) for _ in range(2))
    p = torch.arange(4, device='cuda')
    qo, ko = rotary(q, k, p)
    ko.sum().backward()
    assert (q.grad is None or float(q.grad.abs().sum()) == 0) and R.worst(k.grad, *turned(torch.ones_like(k), p, 16, 'half', back=True)) <= 1
    e, _ = rotary(q[:, :0], None, p[:0])
    assert e.shape == (1, 0, 2, 16)


def test_products_see_the_difference_of_positions():
    from panogrf_amd.rotary import rotary
    q, k = torch.randn(1, 1, 1, 64, device='cuda').expand(1, 50, 1, 64), torch.randn(1, 1, 1, 64, device='cuda').expand(1, 50, 1, 64)
    p = torch.arange(50, device='cuda')
    a, b = rotary(q, k, p)
    c, d = rotary(q, k, p + 1000003)
    s, t = (torch.matmul(u[0, :, 0].double(), v[0, :, 0].double().t()) for u, v in ((a, b), (c, d)))
    # (each of 64 products of two turned values off by 16 U of them)
    assert float((s - t).abs().max()) <= 2 * 16 * R.U * float(q.abs().max() * k.abs().max()) * 64 * 2


def test_graph_replays():
    from panogrf_amd.rotary import rotary
    q, p = torch.randn(3, 1, 8, 64, device='cuda').to(torch.bfloat16), torch.tensor([[5], [9], [1000]], device='cuda')
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        rotary(q, q, p)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = rotary(q, q, p)
    for step in range(3):
        p += 1
        q.copy_(torch.randn(3, 1, 8, 64, device='cuda'))
        graph.replay()
        torch.cuda.synchronize()
        got = [v.clone() for v in held]
        assert all(torch.equal(a, b) for a, b in zip(got, rotary(q, q, p)))
