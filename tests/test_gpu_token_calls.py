"""Calls of the token operators that their documentation allows, at the edges of what they took (HIP)."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('kind', ['rms', 'layer'])
def test_a_gate_for_each_of_many_rays(kind, dtype):
    """Over 60 000 shared gate rows: what the gate expanded to every row gives, to the last bit, and a gradient of that form."""
    from panogrf_amd.block_norm import block_norm
    g = torch.Generator(device='cuda').manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g, device='cuda').to(dtype)
    for rays, n, C in ((70001, 3, 16), (60001, 2, 33), (60002, 4, 520)):
        x, y, gate, dx, dz = r(rays, n, C), r(rays, n, C), r(rays, C), r(rays, n, C), r(rays, n, C)
        w = [r(C) for _ in range(4 if kind == 'layer' else 2)]

        def run(gate):
            ts = [t.detach().requires_grad_(True) for t in (x, y, *w)]
            names = ('post_weight', 'pre_weight', 'post_bias', 'pre_bias')
            outs = block_norm(ts[0], ts[1], gate, kind=kind, scale=0.5, **dict(zip(names, ts[2:])))
            return tuple(t.detach() for t in outs) + torch.autograd.grad(outs, ts, (dx, dz))
        got, want = run(gate), run(gate.unsqueeze(1).expand(rays, n, C).contiguous())
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        # no weights: no sums over rows, and no scratch for them
        ts = [t.detach().requires_grad_(True) for t in (x, y)]
        a, b = block_norm(*ts, gate, kind=kind, scale=0.5), block_norm(*ts, gate.unsqueeze(1).expand(rays, n, C), kind=kind, scale=0.5)
        assert all(torch.equal(s, t) for s, t in zip(torch.autograd.grad(a, ts, (dx, dz)), torch.autograd.grad(b, ts, (dx, dz))))
        # the way the refusal names: the expanded gate's gradient, added up outside
        leaf = gate.detach().requires_grad_(True)
        full = torch.autograd.grad(block_norm(x, y, leaf.unsqueeze(1).expand(rays, n, C), kind=kind, scale=0.5), leaf, (dx, dz))[0]
        assert full.shape == gate.shape and torch.isfinite(full).all()


def test_one_query_a_stream_in_sequence_first_memory():
    """[1, B, H, 2, d].transpose(0, 1): contiguous, with over 2^22 values from the only token to the next."""
    from panogrf_amd.attention import diff_attention, diff_attention_cached
    g = torch.Generator(device='cuda').manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g, device='cuda').bfloat16()
    B, H, Hk, D, M = 520, 32, 8, 128, 5
    q = r(1, B, H, 2, D).transpose(0, 1)
    assert q.stride(1) > 1 << 22 and q.is_contiguous()
    k, v, lam, do = r(B, M, Hk, 2, D), r(B, M, Hk, 2 * D), torch.rand(H, generator=g, device='cuda'), r(B, 1, H, 2 * D)
    n = torch.arange(B, device='cuda', dtype=torch.int32) % (M + 1)

    def run(q, k, v):
        ts = [t.detach().requires_grad_(True) for t in (q, k, v, lam)]
        out = diff_attention(*ts)
        return (out.detach(), *torch.autograd.grad(out, ts, do), diff_attention_cached(q, k, v, lam, n))
    one = torch.empty(B * H * 2 * D, device='cuda', dtype=torch.bfloat16).view(B, 1, H, 2, D).copy_(q)
    assert one.stride(1) < 1 << 22
    assert all(torch.equal(a, b) for a, b in zip(run(q, k, v), run(one, k, v)))
    # keys of one token likewise
    k1, v1 = k[:, :1].contiguous().transpose(0, 1).contiguous().transpose(0, 1), r(1, B, 32, 2 * D).transpose(0, 1)[:, :, ::4]
    far = v1.as_strided(v1.shape, (v1.stride(0), 1 << 23, v1.stride(2), 1))
    n.clamp_(max=1)
    assert all(torch.equal(a, b) for a, b in zip(run(q, k1, far), run(one, k[:, :1].clone(), v1.clone(memory_format=torch.contiguous_format))))


@pytest.mark.parametrize('B,H,D,M,dtype', [((1 << 20) + 3, 16, 32, 2, torch.bfloat16), ((1 << 20) + 1, 8, 128, 1, torch.float16)])
def test_more_than_two_to_the_24_tiles(B, H, D, M, dtype):
    """What calls of parts of the batch give, to the last bit (parts of over 1280 key heads: fewer are cut otherwise and take other kernels)."""
    from panogrf_amd.attention import diff_attention
    g = torch.Generator(device='cuda').manual_seed(2)
    r = lambda *s: torch.randn(*s, generator=g, device='cuda', dtype=dtype)
    q, k, v, do, lam = r(B, 1, H, 2, D), r(B, M, H, 2, D), r(B, M, H, 2 * D), r(B, 1, H, 2 * D), torch.rand(H, generator=g, device='cuda')

    def run(*ts):
        ts, do = [t.detach().requires_grad_(True) for t in ts[:4]], ts[4]
        out = diff_attention(*ts)
        return (out.detach(), *torch.autograd.grad(out, ts, do))
    whole, sums = run(q, k, v, lam, do), torch.zeros(H, dtype=torch.float64, device='cuda')
    for i in range(0, B, B // 5 + 1):
        at = slice(i, i + B // 5 + 1)
        part = run(q[at], k[at], v[at], lam, do[at])
        assert all(torch.equal(a[at], b) for a, b in zip(whole[:4], part[:4])), i
        sums += part[4].double()
    # dlam: a float sum over B rows in 4096 chains, each term a sum of 2 D products, on both sides
    most = (do.abs().float() * v.abs().float()).sum(-1).amax(1).sum(0).double()
    assert ((whole[4].double() - sums).abs() <= 2 * 2.0 ** -24 * (B / 4096 + 64 + 2 * D) * most).all()


def test_rotary_of_more_than_two_to_the_24_wide_tokens():
    """Heads so wide that a workgroup would take one token, of one panorama's queries seen by many entries."""
    from panogrf_amd.rotary import rotary
    g = torch.Generator(device='cuda').manual_seed(3)
    B, N, H, D = 4096, 4099, 27, 38
    one = torch.randn(1, N, H, D, generator=g, device='cuda').bfloat16()
    with torch.no_grad():
        want = rotary(one, None, torch.arange(N, device='cuda'))[0][0]
        got = rotary(one.expand(B, N, H, D), None, torch.arange(N, device='cuda'))[0]
        assert all(torch.equal(got[i], want) for i in (0, 1, 2047, 4001, 4094, 4095))
