"""diff_attention's gradients in f16 where score gradients and maps, taken as they are, leave the type's range: long key axes, the small gradients of mean losses, large ones.

Bounds, element by element, against 64 bits.  What the backward pass rounds is first brought to at most 2^14 by a power of two.  A row's score gradients a (G - delta) (for dq)
are at most 2 |dout_i| max |v_j|, so the factor is at least 2^13 over that, and a rounding off by at most half a step, 2^-11 of the value, or 2^-25 (half the smallest step of the
type) * 2^-13 * 2 |dout_i| max |v_j| = 2^-37 |dout_i| max |v_j|.  For dk the factor is common to a key head: 2^-37 max |dout_i| max |v_j| max(1, |lam|).  For dv: 2^-38 (1 + |lam|).
In the forward pass a map's values are rounded where their sum is at least 1/2: 2^-24 of it.  Nowhere does a floor of the type's own size stand in a bound but for the outputs',
2^-25."""
import pytest
import torch

from tests import token_ref as R

pytestmark = pytest.mark.gpu
HALF = 2.0 ** -11


def bounds(q, k, v, lam, see, scale, do):
    """Gradients and their bounds in 64 bits: {name: (value, bound)}."""
    B, N, H, _, D = q.shape
    M, Hk = k.shape[1], k.shape[2]
    G, U = H // Hk, R.U
    chain = lambda n: (n / 16 + 64) * U
    q, k, v, lam, do = (t.detach().double() for t in (q, k, v, lam, do))
    q = q.view(B, N, Hk, G, 2, D).permute(0, 2, 3, 4, 1, 5)                        # [B, Hk, G, 2, N, D]
    k = k.permute(0, 2, 3, 1, 4).unsqueeze(2)                                      # [B, Hk, 1, 2, M, D]
    v = v.permute(0, 2, 1, 3).unsqueeze(2)                                         # [B, Hk, 1, M, 2D]
    do = do.view(B, N, Hk, G, 2 * D).permute(0, 2, 3, 1, 4)                        # [B, Hk, G, N, 2D]
    lam = lam.view(Hk, G, 1, 1)
    ok = see[:, None, None, None]
    s = torch.matmul(q, k.transpose(-1, -2)) * scale
    es = torch.matmul(q.abs(), k.abs().transpose(-1, -2)) * scale * (D + 8) * U + 8 * U * (1 + s.abs())
    s = s.masked_fill(~ok, -float('inf'))
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - top.masked_fill(top == -float('inf'), 0.0))
    tot = p.sum(-1, keepdim=True)
    p = p / tot.masked_fill(tot == 0, 1.0)
    # (a power of two's argument, score - log sum + its factor's exponent of at most 60, is rounded too)
    es = torch.where(ok, es + 128 * U, torch.zeros_like(s))
    ep = p * (es + (p * es).sum(-1, keepdim=True) + chain(M)) + 2.0 ** -120 * ok
    o = torch.matmul(p, v.unsqueeze(3))
    eo = torch.matmul(ep + p * (HALF + chain(M)) + 2.0 ** -24 * ok, v.abs().unsqueeze(3))
    g = torch.matmul(do, v.transpose(-1, -2))
    eg = torch.matmul(do.abs(), v.abs().transpose(-1, -2)) * chain(2 * D)
    delta = (do.unsqueeze(3) * o).sum(-1, keepdim=True)
    ed = (do.abs().unsqueeze(3) * (eo + o.abs() * chain(2 * D))).sum(-1, keepdim=True)
    sign = torch.stack([torch.ones_like(lam), -lam], 2)                            # [Hk, G, 2, 1, 1]
    ds = sign * p * (g.unsqueeze(3) - delta)
    eds = sign.abs() * (p * (eg.unsqueeze(3) + ed) + ep * (g.unsqueeze(3) - delta).abs()) + (HALF + 8 * U) * ds.abs()
    row = do.norm(dim=-1)[:, :, :, None, :, None] * see.any(2)[:, None, None, None, :, None]
    key = (v.norm(dim=-1)[:, :, 0] * see.any(1)[:, None]).amax(-1)[:, :, None, None, None, None]
    most = lam.abs().amax(1, keepdim=True).clamp_min(1.0)[:, :, None]              # [Hk, 1, 1, 1, 1]
    eq = eds + 2.0 ** -37 * sign.abs() * row * key * ok
    ek = eds + 2.0 ** -37 * most * row.amax((2, 4), keepdim=True) * key * ok
    dq, edq = scale * torch.matmul(ds, k), scale * torch.matmul(eq + chain(M) * ds.abs(), k.abs())
    dk = scale * torch.matmul(ds.transpose(-1, -2), q).sum(2)
    edk = scale * torch.matmul((ek + chain(N * G) * ds.abs()).transpose(-1, -2), q.abs()).sum(2)
    pc = p[:, :, :, 0] - lam * p[:, :, :, 1]
    epc = ep[:, :, :, 0] + lam.abs() * ep[:, :, :, 1] + (HALF + 2 * U) * pc.abs() + 2 * U * p.sum(3) + 2.0 ** -37 * most[:, :, 0] * ok[:, :, :, 0]
    dv = torch.matmul(pc.transpose(-1, -2), do).sum(2)
    edv = torch.matmul((epc + chain(N * G) * pc.abs()).transpose(-1, -2), do.abs()).sum(2)
    t = p[:, :, :, 1] * g
    edl = (ep[:, :, :, 1] * g.abs() + p[:, :, :, 1] * eg + chain(M + B * N) * t.abs()).sum((0, 3, 4)).reshape(H)
    done = lambda x, e: (x, HALF * x.abs() + e * (1 + HALF) + 2.0 ** -25)
    return {'q': done(dq.permute(0, 4, 1, 2, 3, 5).reshape(B, N, H, 2, D), edq.permute(0, 4, 1, 2, 3, 5).reshape(B, N, H, 2, D)),
            'k': done(dk.permute(0, 3, 1, 2, 4), edk.permute(0, 3, 1, 2, 4)), 'v': done(dv.permute(0, 2, 1, 3), edv.permute(0, 2, 1, 3)),
            'lam': done(-t.sum((0, 3, 4)).reshape(H), edl)}


def make(B, N, M, H, Hk, D, small, dout, seed=0):
    """Scores of about 1; with 'q' small, scale * k, what dq is made of, is large (and dk's share, scale * q, small), with 'k' the other way round."""
    g = torch.Generator(device='cuda').manual_seed(seed + N * 5 + M)
    r = lambda *s: torch.randn(*s, generator=g, device='cuda')
    f = 1 / 64 if small == 'q' else 8.0
    q, k = (r(B, N, H, 2, D) * f).half(), (r(B, M, Hk, 2, D) * (1 / 8 / f)).half()
    v, do = r(B, M, Hk, 2 * D).half(), (r(B, N, H, 2 * D) * dout).half()
    lam = (torch.rand(H, generator=g, device='cuda') * 0.8 + 0.1).half()
    return q, k, v, lam, do, 8 * D ** -0.5


def check(q, k, v, lam, do, scale, causal=False, mask=None, names=('q', 'k', 'v', 'lam')):
    from panogrf_amd.attention import diff_attention
    ts = [t.detach().requires_grad_(n in names) for n, t in zip(('q', 'k', 'v', 'lam'), (q, k, v, lam))]
    leaves = [t for t in ts if t.requires_grad]
    grads = torch.autograd.grad(diff_attention(*ts, causal=causal, key_mask=mask, scale=scale), leaves, do)
    again = torch.autograd.grad(diff_attention(*ts, causal=causal, key_mask=mask, scale=scale), leaves, do)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))
    ref = bounds(q, k, v, lam, R.may_see(q.shape[0], q.shape[1], k.shape[1], causal, mask), scale, do)
    bad = {n: R.worst(t, *ref[n]) for n, t in zip(names, grads)}
    assert all(x <= 1 for x in bad.values()), bad
    return grads


SHAPES = [(1, 96, 8192, 2, 1, 64), (1, 1500, 2048, 2, 2, 64), (2, 200, 4096, 2, 2, 32), (1, 300, 3001, 2, 1, 128), (256, 64, 64, 1, 1, 32), (128, 33, 40, 4, 2, 64), (2, 1, 20000, 2, 1, 64),
          (128, 20, 17, 4, 2, 32)]


@pytest.mark.parametrize('B,N,M,H,Hk,D', SHAPES)
@pytest.mark.parametrize('small', ['q', 'k'])
@pytest.mark.parametrize('dout', [1e-5, 1e-4, 1e-2])
def test_small_gradients(B, N, M, H, Hk, D, small, dout):
    q, k, v, lam, do, scale = make(B, N, M, H, Hk, D, small, dout)
    check(q, k, v, lam, do, scale)


@pytest.mark.parametrize('B,N,M,H,Hk,D', SHAPES)
@pytest.mark.parametrize('mask', ['none', 'holes'])
def test_small_gradients_behind_masks(B, N, M, H, Hk, D, mask):
    q, k, v, lam, do, scale = make(B, N, M, H, Hk, D, 'q', 1e-4)
    if mask == 'holes':
        mask = torch.rand(B, M, generator=torch.Generator(device='cuda').manual_seed(3), device='cuda') > 0.4
        v[~mask], k[~mask] = 60000.0, float('nan')       # what hidden keys hold has no part in the range either
        got = check(q, k.where(mask[..., None, None, None], torch.zeros_like(k)), v.where(mask[..., None, None], torch.zeros_like(v)), lam, do, scale, True, mask)
        from panogrf_amd.attention import diff_attention
        ts = [t.requires_grad_(True) for t in (q, k, v, lam)]
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(diff_attention(*ts, causal=True, key_mask=mask, scale=scale), ts, do), got))
    else:
        check(q, k, v, lam, do, scale, True)


@pytest.mark.parametrize('B,N,M,H,Hk,D', [s for s in SHAPES if s[2] < 4000])
@pytest.mark.parametrize('name,small', [('q', 'k'), ('k', 'q')])
def test_large_gradients(B, N, M, H, Hk, D, name, small):
    """Peaked maps under gradients (of a scaled loss, say) whose score gradients are over 65504, while the gradient itself is not."""
    q, k, v, lam, do, scale = make(B, N, M, H, Hk, D, small, 8192.0)
    assert float(do.abs().max()) < 65504
    check(q * 4, k, v, lam, do, scale / 4096, names=(name,))
    check(q * 64, k, v, lam, do / 16, scale / 64, names=(name,))


@pytest.mark.parametrize('B,N,M,H,Hk,D', [(1, 300, 700, 4, 2, 64), (128, 20, 40, 4, 2, 32), (1, 300, 700, 4, 2, 128)])
def test_large_weight_of_the_second_map(B, N, M, H, Hk, D):
    q, k, v, lam, do, scale = make(B, N, M, H, Hk, D, 'q', 1e-4)
    check(q, k, v, lam.float() * 300, do, scale)


def test_rows_of_different_sizes():
    """dq of rows whose gradients are far smaller than those of their neighbours."""
    q, k, v, lam, do, scale = make(1, 256, 4096, 2, 2, 64, 'q', 1.0)
    do = (do * (2.0 ** -(torch.arange(256, device='cuda') % 13))[None, :, None, None]).half()
    check(q, k, v, lam, do, scale)


@pytest.mark.parametrize('B,N,M,H,Hk,D', [(256, 200, 64, 2, 1, 32), (256, 130, 33, 1, 1, 64), (1, 200, 900, 2, 1, 128)])
@pytest.mark.parametrize('turn', [False, True])
def test_blocks_of_growing_size(B, N, M, H, Hk, D, turn):
    q, k, v, lam, do, scale = make(B, N, M, H, Hk, D, 'q', 2e-3)
    do = (do.flip(1) if turn else do) * (1.6 ** (torch.arange(N, device='cuda') / 8))[None, :, None, None]
    do = (do.flip(1) if turn else do).half()
    do[1::2, :40] = 0
    check(q, k, v, lam, do, scale)
