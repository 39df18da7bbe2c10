"""diff_attention's output in 16 bits where its maps have much in common: what cancels must not leave its roundings behind.

Bounds, element by element, against 64 bits.  Up to 32 rows, or 64 keys, of a key head probabilities go into the product with v in two pieces of the type: off by half a step of
a half step, 2^-16 of themselves in bf16 and 2^-22 in f16 (or half f16's smallest step, 2^-25, where the row's sum is at least 1/2).  In bf16 from 2^33 products and 1024 rows on
they are f16, off by 2^-11 of themselves or 2^-24 of the row's sum, beside a v whose values are off by 2^-25 where 2^14 is its key head's largest: 2^-39 of that.  Roundings of many probabilities are independent of each other: of n of them, off by
at most e_i each, no more than 7 sqrt(sum e_i^2) comes together but once in e^24 times (`chance`)."""
import pytest
import torch

from tests import token_ref as R

pytestmark = pytest.mark.gpu
U = R.U


def output(q, k, v, lam, see, scale, piece, floor, off, chance=False):
    """(value, bound) of the queries in q [B, n, H, 2, D], with see [B, n, M]; piece, floor: a probability's rounding, relative and of the row's sum; off [B, Hk]: of v's values."""
    B, n, H, _, D = q.shape
    M, Hk = k.shape[1], k.shape[2]
    G = H // Hk
    half, chain = R.HALF[q.dtype], (M / 16 + 64) * U
    out, err = torch.empty(B, n, H, 2 * D, dtype=torch.float64, device='cuda'), torch.empty(B, n, H, 2 * D, dtype=torch.float64, device='cuda')
    for h in range(H):
        kh, vh = k[:, :, h // G].double(), v[:, :, h // G].double()
        kh, vh = (t.where(see.any(1).view(B, M, *[1] * (t.dim() - 2)), torch.zeros((), dtype=torch.float64, device='cuda')) for t in (kh, vh))
        o = []
        for i in (0, 1):
            s = torch.bmm(q[:, :, h, i].double(), kh[:, :, i].transpose(1, 2).contiguous()) * scale
            es = torch.bmm(q[:, :, h, i].double().abs(), kh[:, :, i].abs().transpose(1, 2).contiguous()) * scale * (D + 8) * U + 4 * U * (1 + s.abs())
            s = s.masked_fill(~see, -float('inf'))
            p = torch.exp(s - s.amax(-1, keepdim=True).clamp_min(-1e300))
            p = p / p.sum(-1, keepdim=True).clamp_min(1e-300)
            es = es.masked_fill(~see, 0.0)
            ep = p * (es + (p * es).sum(-1, keepdim=True) + 2 * chain) + 2.0 ** -126 * see
            rounding = p * piece + floor * see
            r = 7 * torch.bmm(rounding * rounding, vh * vh).sqrt() if chance else torch.bmm(rounding, vh.abs())
            o.append((torch.bmm(p, vh), torch.bmm(ep, vh.abs()) + off[:, h // G].view(B, 1, 1), r))
        w = float(lam[h])
        out[:, :, h] = o[0][0] - w * o[1][0]
        err[:, :, h] = o[0][1] + abs(w) * o[1][1] + 4 * U * (o[0][0].abs() + abs(w) * o[1][0].abs())
        err[:, :, h] += torch.hypot(o[0][2], w * o[1][2]) if chance else o[0][2] + abs(w) * o[1][2]
    return out, half * out.abs() + err * (1 + half) + (2.0 ** -25 if q.dtype == torch.float16 else 1e-300)


def make(B, N, M, H, Hk, D, dtype, seed=0):
    g = torch.Generator(device='cuda').manual_seed(seed + N + M)
    r = lambda *s: torch.randn(*s, generator=g, device='cuda')
    q, k = r(B, N, H, 1, D), r(B, M, Hk, 1, D)
    q, k = torch.cat([q, q + 0.1 * r(B, N, H, 1, D)], 3).to(dtype), torch.cat([k, k + 0.1 * r(B, M, Hk, 1, D)], 3).to(dtype)     # maps that are nearly alike
    return q, k, (r(B, M, Hk, 2 * D) + 0.5).to(dtype), torch.full((H,), 0.9, device='cuda').to(dtype)


def check(q, k, v, lam, causal=False, mask=None, way='two', rows=None, grad=False, chance=False):
    from panogrf_amd.attention import diff_attention
    B, N, H, _, D = q.shape
    M = k.shape[1]
    ts = [t.detach().requires_grad_(grad) for t in (q, k, v, lam)]
    out = diff_attention(*ts, causal=causal, key_mask=mask).detach()
    assert torch.equal(out, diff_attention(q, k, v, lam, causal=causal, key_mask=mask))
    see = torch.ones(B, N, M, dtype=torch.bool, device='cuda') if rows is None else torch.ones(B, len(rows), M, dtype=torch.bool, device='cuda')
    at = torch.arange(N, device='cuda') if rows is None else rows
    if causal:
        see = see & (torch.arange(M, device='cuda') <= (at + M - N)[:, None])
    if mask is not None:
        see = see & mask[:, None]
    if way == 'two':
        piece, floor = (2.0 ** -16, 0.0) if q.dtype == torch.bfloat16 else (2.0 ** -22, 2.0 ** -24)
        off = torch.zeros(B, k.shape[2], dtype=torch.float64, device='cuda')
    else:
        piece, floor = 2.0 ** -11, 2.0 ** -24
        hidden = torch.zeros_like(v) if mask is None else torch.zeros_like(v).masked_fill(~mask[:, :, None, None], 1)
        off = v.masked_fill(hidden > 0, 0).abs().amax((1, 3)).double() * 2.0 ** -39
    ref = output(q[:, at], k, v, lam, see, D ** -0.5, piece, floor, off, chance)
    assert R.worst(out[:, at], *ref) <= 1
    return out


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
@pytest.mark.parametrize('D', [32, 64, 128])
@pytest.mark.parametrize('B,N,M,H,Hk', [(300, 64, 64, 2, 1), (2, 200, 33, 4, 2), (1, 40, 64, 1, 1), (3, 8, 1000, 8, 2), (1, 17, 1, 6, 2)])
@pytest.mark.parametrize('causal', [False, True])
def test_two_pieces(B, N, M, H, Hk, D, dtype, causal):
    q, k, v, lam = make(B, N, M, H, Hk, D, dtype)
    check(q, k, v, lam, causal, grad=True)
    mask = torch.rand(B, M, generator=torch.Generator(device='cuda').manual_seed(1), device='cuda') > 0.3
    k[~mask], v[~mask] = float('nan'), float('inf')
    check(q, k, v, lam, causal, mask)


LONG = [(1, 8192, 8192, 8, 8, 64), (2, 4099, 8195, 16, 4, 64), (1, 4200, 8100, 16, 2, 128), (3, 9000, 5003, 8, 8, 32), (1, 1024, 33000, 16, 1, 64), (1, 64, 33000, 256, 4, 64), (2, 1024, 4096, 16, 16, 64), (2, 1500, 1500, 32, 2, 128)]
ROWS = 40


def some(N, seed):
    return torch.randperm(N, generator=torch.Generator().manual_seed(seed))[:ROWS].sort()[0].cuda()


@pytest.mark.parametrize('B,N,M,H,Hk,D', LONG)
@pytest.mark.parametrize('causal', [False, True])
def test_values_in_f16(B, N, M, H, Hk, D, causal):
    assert B * H * N * M * D >= 1 << 33 and N * H // Hk >= 1024
    q, k, v, lam = make(B, N, M, H, Hk, D, torch.bfloat16)
    check(q, k, v, lam, causal, way='f16', rows=some(N, 0), grad=D == 64)
    mask = torch.rand(B, M, generator=torch.Generator(device='cuda').manual_seed(1), device='cuda') > 0.3
    mask[0, M - 100:] = False
    k[~mask], v[~mask] = float('nan'), float('inf')
    check(q, k, v, lam, causal, mask, way='f16', rows=some(N, 1))


@pytest.mark.parametrize('B,N,M,H,Hk,D', LONG)
@pytest.mark.parametrize('causal', [False, True])
def test_sharp_maps(B, N, M, H, Hk, D, causal):
    """Maps of a few keys, nearly alike, with nearly all of the one taken off: roundings to bf16 are four times the output's own there."""
    q, k, v, lam = make(B, N, M, H, Hk, D, torch.bfloat16)
    check(q * 4, k, v, lam, causal, way='f16', rows=some(N, 6), chance=True)


@pytest.mark.parametrize('size', [1e30, 1e-30, 1e-37])
def test_values_far_from_one(size):
    q, k, v, lam = make(1, 8192, 8192, 8, 8, 64, torch.bfloat16)
    v = (v.float() * size).bfloat16()
    v[:, :, 3] = 0
    out = check(q, k, v, lam, True, way='f16', rows=some(8192, 2))
    assert float(out[:, :, 3].abs().max()) == 0


@pytest.mark.parametrize('far', [1e30, 1e-30, 70000.0])
def test_keys_of_very_different_sizes(far):
    """Those key heads go the other way, and no other does: row 0 .. 3000 do not see the key that is out of line."""
    q, k, v, lam = make(1, 8192, 8192, 8, 8, 64, torch.bfloat16)
    v[:, 3001, 2] = (v[:, 3001, 2].float() * far).bfloat16()
    v[:, 5000, 5] = (v[:, 5000, 5].float() * far).bfloat16()
    rows = torch.cat([some(3000, 3)[:20], some(8192, 4)[:20]]).sort()[0].unique()
    out = check(q, k, v, lam, True, way='f16', rows=rows)                            # (their own bound is the narrower one, below)
    for h in (2, 5):
        ref = output(q[:, rows, h:h + 1], k[:, :, h:h + 1], v[:, :, h:h + 1], lam[h:h + 1], torch.arange(8192, device='cuda') <= rows[None, :, None], 64 ** -0.5, 2.0 ** -16, 0.0,
                     torch.zeros(1, 1, dtype=torch.float64, device='cuda'))
        assert R.worst(out[:, rows, h:h + 1], *ref) <= 1


def test_infinite_values_stay_in_their_columns():
    q, k, v, lam = make(1, 8192, 8192, 8, 8, 64, torch.bfloat16)
    from panogrf_amd.attention import diff_attention
    want = diff_attention(q, k, v, lam, causal=True)
    v[0, 4000, 1, 7], v[0, 5000, 6, 100] = float('inf'), float('nan')
    got = diff_attention(q, k, v, lam, causal=True)
    bad = ~torch.isfinite(got[0])
    assert bad[4000:, 1, 7].all() and bad[5000:, 6, 100].all()
    same = torch.ones_like(bad)
    same[3968:, 1, 7], same[4992:, 6, 100] = False, False                            # (a block of 32 keys may mix a hidden key's infinity into rows that stand in it)
    assert torch.equal(got[0][same], want[0][same])


def test_a_cache_with_many_new_tokens():
    """The form over a cache takes the same ways; what stands behind the lengths may be anything."""
    from panogrf_amd.attention import diff_attention_cached
    B, N, M, H, Hk, D = 2, 2048, 9000, 16, 4, 64
    q, k, v, lam = make(B, N, M, H, Hk, D, torch.bfloat16)
    n = torch.tensor([7001, 8999], dtype=torch.int32, device='cuda')
    for b in range(B):
        k[b, n[b]:], v[b, n[b]:] = float('nan'), 3e38
    out, rows = diff_attention_cached(q, k, v, lam, n), some(N, 5)
    see = torch.arange(M, device='cuda') <= (rows[None, :, None] + (n - N).view(-1, 1, 1))
    off = torch.stack([v[b, :n[b]].abs().amax((0, 2)).double() for b in range(B)]) * 2.0 ** -39
    assert R.worst(out[:, rows], *output(q[:, rows], k, v, lam, see, D ** -0.5, 2.0 ** -11, 2.0 ** -24, off)) <= 1


def test_values_in_f16_captured():
    """Two graphs of the same call, replayed in turn with other inputs and eager work between: what the eager calls give, also where a key head changes its way."""
    from panogrf_amd.attention import diff_attention
    q, k, v, lam = make(2, 1024, 4096, 16, 16, 64, torch.bfloat16)
    with torch.no_grad():
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(2):
                diff_attention(q, k, v, lam)
        torch.cuda.current_stream().wait_stream(side)
        graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
        outs = []
        for graph in graphs:
            with torch.cuda.graph(graph):
                outs.append(diff_attention(q, k, v, lam))
        for i, far in enumerate((1.0, 1e25, 1e-20, 1.0)):
            for t, new in zip((q, k, v), make(2, 1024, 4096, 16, 16, 64, torch.bfloat16, seed=10 + i)):
                t.copy_(new)
            v[1, 77, 3 + i] = (v[1, 77, 3 + i].float() * far).bfloat16()
            want = diff_attention(q, k, v, lam)
            for graph, out in zip(graphs, outs):
                out.zero_()
                graph.replay()
                torch.cuda.synchronize()
                assert torch.equal(out, want), i
