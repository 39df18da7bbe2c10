"""diff_attention and diff_attention_cached (HIP) against a plain 64-bit form, element by element within first-order bounds."""
import pytest
import torch

from tests import token_ref as R

pytestmark = pytest.mark.gpu
T = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}


def make(B, N, M, H, Hk, D, dtype, seed=0, lam_dtype=None):
    g = torch.Generator(device='cuda').manual_seed(seed + N * 7 + M)
    r = lambda *s: torch.randn(*s, generator=g, device='cuda').to(T[dtype])
    q, k, v, do = r(B, N, H, 2, D), r(B, M, Hk, 2, D), r(B, M, Hk, 2 * D) + 0.25, r(B, N, H, 2 * D)
    lam = (torch.rand(H, generator=g, device='cuda') * 0.8 + 0.1).to(T[lam_dtype or dtype])
    return q, k, v, lam, do


def mask_of(kind, B, M, seed=1):
    if kind == 'none':
        return None
    g = torch.Generator(device='cuda').manual_seed(seed)
    m = torch.rand(B, M, generator=g, device='cuda') > 0.3
    if kind == 'tail':
        m = torch.arange(M, device='cuda') < torch.randint(0, M + 1, (B, 1), generator=g, device='cuda')
    m[0] = False
    return m


def grads(q, k, v, lam, do, **kw):
    from panogrf_amd.attention import diff_attention
    ts = [t.detach().requires_grad_(True) for t in (q, k, v, lam)]
    out = diff_attention(*ts, **kw)
    return (out.detach(),) + torch.autograd.grad(out, ts, do)


def check(q, k, v, lam, do, causal, mask, scale=None):
    B, N, H, _, D = q.shape
    got = grads(q, k, v, lam, do, causal=causal, key_mask=mask, scale=scale)
    from panogrf_amd.attention import diff_attention
    with torch.no_grad():
        assert torch.equal(diff_attention(q, k, v, lam, causal=causal, key_mask=mask, scale=scale), got[0])
    again = grads(q, k, v, lam, do, causal=causal, key_mask=mask, scale=scale)
    assert all(torch.equal(a, b) for a, b in zip(got, again)), 'differs from call to call'
    ref = R.diff_attention(q, k, v, lam, R.may_see(B, N, k.shape[1], causal, mask), D ** -0.5 if scale is None else scale, do, q.dtype)
    lim = ref['lam']
    ref['lam'] = (lim[0], lim[1] + R.HALF[lam.dtype] * lim[0].abs() + 1e-300)
    bad = {n: R.worst(t, *ref[n]) for n, t in zip(('out', 'q', 'k', 'v', 'lam'), got)}
    assert all(x <= 1 for x in bad.values()), bad
    return got


SHAPES = [(1, 1, 1, 1, 1), (2, 3, 5, 2, 2), (1, 17, 33, 4, 2), (3, 64, 64, 2, 2), (2, 65, 40, 3, 1), (1, 130, 300, 8, 1), (2, 200, 129, 4, 4), (1, 31, 512, 6, 2)]


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('D', [32, 64, 128])
@pytest.mark.parametrize('B,N,M,H,Hk', SHAPES)
@pytest.mark.parametrize('causal,mask', [(False, 'none'), (True, 'none'), (False, 'holes'), (True, 'tail')])
def test_values_and_gradients(B, N, M, H, Hk, D, dtype, causal, mask):
    check(*make(B, N, M, H, Hk, D, dtype), causal, mask_of(mask, B, M))


@pytest.mark.parametrize('dtype,D,N,M,G', [('bf16', 64, 1000, 1000, 1), ('f16', 32, 777, 1555, 4), ('f32', 64, 600, 601, 2), ('bf16', 128, 515, 900, 2)])
@pytest.mark.parametrize('causal', [False, True])
def test_longer(dtype, D, N, M, G, causal):
    check(*make(1, N, M, 2 * G, 2, D, dtype), causal, None)


def test_rows_that_see_nothing():
    q, k, v, lam, do = make(2, 9, 4, 2, 2, 32, 'bf16')
    got = check(q, k, v, lam, do, True, None)                       # nine queries, four keys: the first five see none
    assert float(got[0][:, :5].abs().max()) == 0 and float(got[1][:, :5].abs().max()) == 0
    mask = torch.zeros(2, 4, dtype=torch.bool, device='cuda')
    got = check(q, k, v, lam, do, False, mask)
    assert all(float(t.abs().max()) == 0 for t in got)


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
def test_what_masked_places_hold_does_not_matter(dtype):
    q, k, v, lam, do = make(2, 70, 150, 4, 2, 64, dtype)
    mask = mask_of('holes', 2, 150)
    want = check(q, k, v, lam, do, False, mask)
    k2, v2 = k.clone(), v.clone()
    for i, x in enumerate((float('nan'), float('inf'), -float('inf'), torch.finfo(T[dtype]).min)):
        k2[(~mask) & (torch.arange(150, device='cuda') % 4 == i)] = x
        v2[(~mask) & (torch.arange(150, device='cuda') % 4 == (i + 1) % 4)] = x
    got = grads(q, k2, v2, lam, do, key_mask=mask)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize('dtype,D', [('f32', 32), ('bf16', 32), ('f16', 32), ('bf16', 64), ('f16', 64)])
@pytest.mark.parametrize('B,N,M,H,Hk', [(64, 64, 64, 4, 4), (256, 33, 40, 1, 1), (65, 70, 17, 12, 4), (128, 31, 32, 4, 2), (300, 1, 64, 1, 1), (90, 5, 1, 6, 3), (256, 100, 33, 2, 1)])
@pytest.mark.parametrize('causal,mask', [(False, 'none'), (True, 'none'), (False, 'holes'), (True, 'tail')])
def test_many_heads_of_few_keys(B, N, M, H, Hk, dtype, D, causal, mask):
    q, k, v, lam, do = make(B, N, M, H, Hk, D, dtype)
    m = mask_of(mask, B, M)
    check(q, k, v, lam, do, causal, m)
    # what masked keys and queries that see nothing hold does not matter
    see = R.may_see(B, N, M, causal, m)
    blind, hidden = ~see.any(2), torch.zeros(B, M, dtype=torch.bool, device='cuda') if m is None else ~m
    want = grads(q, k, v, lam, do, causal=causal, key_mask=m)
    q, k, v, do = q.clone(), k.clone(), v.clone(), do.clone()
    q[blind], do[blind], k[hidden], v[hidden] = float('nan'), float('inf'), float('nan'), float('nan')
    assert all(torch.equal(a, b) for a, b in zip(grads(q, k, v, lam, do, causal=causal, key_mask=m), want))


def test_few_keys_one_gradient_at_a_time():
    q, k, v, lam, do = make(64, 40, 50, 8, 4, 32, 'f32')
    want = grads(q, k, v, lam, do)
    from panogrf_amd.attention import diff_attention
    for i in range(4):
        ts = [t.clone().requires_grad_(j == i) for j, t in enumerate((q, k, v, lam))]
        assert torch.equal(torch.autograd.grad(diff_attention(*ts), ts[i], do)[0], want[1 + i])


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('D', [32, 64, 128])
@pytest.mark.parametrize('M', [70, 600])
def test_what_queries_that_see_nothing_hold_does_not_matter(M, D, dtype):
    """They give 0 and move nothing, also where a 16-bit gradient overflowed on its way to them."""
    for causal, N in ((False, 40), (True, M + 37)):
        q, k, v, lam, do = make(2, N, M, 4, 2, D, dtype)
        mask = mask_of('none' if causal else 'holes', 2, M)
        blind = (torch.arange(N, device='cuda') < N - M) if causal else slice(None)
        want = grads(q, k, v, lam, do, causal=causal, key_mask=mask)
        q, do = q.clone(), do.clone()
        for b in (0, 1) if causal else (0,):                                       # (the holes leave entry 0 nothing)
            q[b, blind], do[b, blind] = float('nan'), float('inf')
        got = grads(q, k, v, lam, do, causal=causal, key_mask=mask)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize('M', [40, 600])
def test_an_entry_without_keys_reads_nothing_behind_its_rows(M):
    """The last entry's mask leaves nothing: what stands behind its last query (here the next piece of one tensor, not finite) is not read."""
    q, k, v, lam, do = make(2, 41, M, 2, 2, 64, 'bf16')
    room = torch.full((3, 41, 2, 2, 64), float('nan'), device='cuda', dtype=torch.bfloat16)
    room[:2] = q
    mask = torch.ones(2, M, dtype=torch.bool, device='cuda')
    mask[1] = False
    want, got = grads(q, k, v, lam, do, key_mask=mask), grads(room[:2], k, v, lam, do, key_mask=mask)
    assert all(torch.equal(a, b) and torch.isfinite(a).all() for a, b in zip(got, want))
    assert all(float(t[1].abs().sum()) == 0 for t in got[:4])


def test_large_scores():
    q, k, v, lam, do = make(1, 50, 200, 2, 2, 64, 'f32')
    check(q * 20, k * 4, v, lam, do, False, None)                   # maps that are nearly one key
    q, k, v, lam, do = make(1, 50, 200, 2, 2, 64, 'bf16')
    check(torch.zeros_like(q), k, v, lam, do, True, None)           # maps that are even
    check(q, k, v, lam, do, False, None, scale=0.01)


def test_a_single_key_has_no_score_gradient():
    got = grads(*make(2, 1, 1, 2, 2, 64, 'bf16'))
    assert float(got[1].abs().max()) < 1e-5 and float(got[2].abs().max()) < 1e-5


@pytest.mark.parametrize('dtype', ['bf16', 'f16'])
def test_lam_in_float(dtype):
    check(*make(2, 40, 50, 4, 2, 64, dtype, lam_dtype='f32'), True, None)


def test_views_other_orders_and_odd_addresses():
    q, k, v, lam, do = make(2, 33, 47, 4, 2, 32, 'bf16')
    want = grads(q, k, v, lam, do, causal=True)
    fused = torch.empty(2, 47, 2, 2 * 32 + 64 + 8, dtype=torch.bfloat16, device='cuda')
    fused[..., :64], fused[..., 72:] = k.flatten(-2), v
    kv = (fused[..., :64].unflatten(-1, (2, 32)), fused[..., 72:])
    across = q.permute(0, 2, 1, 3, 4).contiguous().permute(0, 2, 1, 3, 4)             # [B, H, N, 2, d] memory
    maps_apart = torch.stack([q[..., 0, :], q[..., 1, :]]).permute(1, 2, 3, 0, 4)     # the two maps far from each other
    odd = torch.empty(q.numel() + 1, dtype=torch.bfloat16, device='cuda')[1:].view(q.shape).copy_(q)
    step = torch.empty(2, 33, 4, 2, 64, dtype=torch.bfloat16, device='cuda')[..., ::2].copy_(q)
    for qq, (kk, vv) in ((across, kv), (maps_apart, (k, v)), (odd, (k, v)), (step, kv)):
        got = grads(qq, kk, vv, lam, do.transpose(0, 1).contiguous().transpose(0, 1), causal=True)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_broadcast_inputs_and_single_gradients():
    from panogrf_amd.attention import diff_attention
    q, k, v, lam, do = make(3, 20, 30, 2, 2, 32, 'f32')
    k1, v1 = k[:1].clone().requires_grad_(True), v[:1].clone().requires_grad_(True)
    out = diff_attention(q, k1.expand(3, -1, -1, -1, -1), v1.expand(3, -1, -1, -1), lam)
    dk, dv = torch.autograd.grad(out, (k1, v1), do)
    full = grads(q, k[:1].repeat(3, 1, 1, 1, 1), v[:1].repeat(3, 1, 1, 1), lam, do)
    for a, b in ((dk, full[2]), (dv, full[3])):                                       # (three float values added)
        assert float((a - b.sum(0, keepdim=True)).abs().max()) <= 4 * R.U * float(b.abs().sum(0).max())
    for i in range(4):
        ts = [t.clone().requires_grad_(j == i) for j, t in enumerate((q, k, v, lam))]
        diff_attention(*ts).backward(do)
        assert torch.equal(ts[i].grad, grads(q, k, v, lam, do)[1 + i]) and all(t.grad is None for j, t in enumerate(ts) if j != i)


def test_no_rows_no_keys():
    q, k, v, lam, do = make(2, 6, 5, 2, 1, 32, 'f16')
    for a, b, c, d in ((q[:, :0], k, v, do[:, :0]), (q, k[:, :0], v[:, :0], do), (q[:0], k[:0], v[:0], do[:0])):
        got = grads(a, b, c, lam, d)
        assert [t.shape for t in got] == [d.shape, a.shape, b.shape, c.shape, lam.shape] and all(float(t.abs().sum()) == 0 for t in got)


def test_against_differences():
    """Along one direction of all inputs at once, in float: the quotient's own error is measured on the 64-bit form, its rounding bounded by the outputs' bounds over the step."""
    from panogrf_amd.attention import diff_attention
    ts = make(1, 12, 20, 2, 1, 32, 'f32')
    q, k, v, lam, do = ts
    way = [torch.randn_like(t) * 0.3 for t in ts[:4]]
    h, see = 2.0 ** -7, R.may_see(1, 12, 20, True)
    slope = sum(float((a.double() * b.double()).sum()) for a, b in zip(way, grads(*ts, causal=True)[1:]))
    quotient = exact = room = 0.0
    for s in (1, -1):
        m = [t + s * h * w for t, w in zip(ts[:4], way)]
        quotient += s * float((diff_attention(*m, causal=True).double() * do.double()).sum()) / (2 * h)
        ref, bound = R.diff_attention(*m, see, 32 ** -0.5, None, torch.float32)['out']
        exact += s * float((ref * do.double()).sum()) / (2 * h)
        room += float((bound * do.double().abs()).sum()) / (2 * h)
    assert abs(quotient - exact) <= room
    assert abs(exact - slope) <= 0.02 * abs(slope) + room            # (a central difference's error is of order h^2)


# ------------------------------------------------------------------------------------------------------------------- cache
@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('D', [32, 64, 128])
@pytest.mark.parametrize('B,N,M,H,Hk,lengths', [(1, 1, 500, 8, 2, (500,)), (4, 1, 300, 4, 4, (0, 1, 300, 77)), (3, 5, 260, 6, 2, (3, 5, 999)), (2, 1, 5000, 8, 1, (4999, 64)),
                                                (1, 40, 2000, 2, 2, (1200,)), (2, 2, 64, 12, 4, (-3, 33))])
def test_cached(B, N, M, H, Hk, D, lengths, dtype):
    from panogrf_amd.attention import diff_attention_cached
    q, k, v, lam, _ = make(B, N, M, H, Hk, D, dtype)
    n = torch.tensor(lengths, dtype=torch.int32, device='cuda')
    ref = R.diff_attention(q, k, v, lam, R.may_see(B, N, M, True, lengths=n), D ** -0.5, None, T[dtype])['out']
    got = diff_attention_cached(q, k, v, lam, n)
    assert R.worst(got, *ref) <= 1
    behind = torch.arange(M, device='cuda') >= n.view(-1, 1)
    k2, v2 = k.clone(), v.clone()
    k2[behind], v2[behind] = float('nan'), float('inf')
    assert torch.equal(diff_attention_cached(q, k2, v2, lam, n), got)


def test_cached_is_the_last_rows_of_the_whole():
    from panogrf_amd.attention import diff_attention, diff_attention_cached
    q, k, v, lam, _ = make(2, 90, 90, 4, 2, 64, 'f32')
    whole = diff_attention(q, k, v, lam, causal=True)
    n = torch.full((2,), 90, dtype=torch.int32, device='cuda')
    for last in (1, 7):
        got = diff_attention_cached(q[:, -last:], k, v, lam, n)
        assert float((got - whole[:, -last:]).abs().max()) < 2e-6        # (two orders of 90 float additions of values near 1: 2 * 90 / 16 U and a few)


def test_cache_behind_2_to_the_32():
    from panogrf_amd.attention import diff_attention_cached
    if torch.cuda.mem_get_info()[0] < 80 << 30:
        pytest.skip('needs 80 GB')
    M, Hk, D = (1 << 23) + 8, 8, 32                                      # an entry of each cache: over 2^32 values
    k = torch.empty(2, M, Hk, 2, D, dtype=torch.bfloat16, device='cuda')
    v = torch.empty(2, M, Hk, 2 * D, dtype=torch.bfloat16, device='cuda')
    q, ks, vs, lam, _ = make(2, 1, 400, 8, 8, D, 'bf16')
    k[:, :400], v[:, :400] = ks, vs
    n = torch.tensor([100, 400], dtype=torch.int32, device='cuda')
    got = diff_attention_cached(q, k, v, lam, n)
    ref = R.diff_attention(q, ks, vs, lam, R.may_see(2, 1, 400, True, lengths=n), D ** -0.5, None, torch.bfloat16)['out']
    assert R.worst(got, *ref) <= 1


def test_captured_steps_follow_the_lengths():
    from panogrf_amd.attention import diff_attention_cached
    q, k, v, lam, _ = make(3, 1, 4000, 8, 2, 64, 'bf16')
    n = torch.tensor([5, 900, 4000], dtype=torch.int32, device='cuda')
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        diff_attention_cached(q, k, v, lam, n)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):                                                   # two graphs, each with a workspace of its own
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = diff_attention_cached(q, k, v, lam, n)
        graphs.append((graph, held))
    for step in range(3):
        n.copy_(torch.tensor([6 + step, 901 + 64 * step, 3990 + step], dtype=torch.int32))
        q.copy_(torch.randn(q.shape, device='cuda'))
        for graph, held in graphs:
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(held.clone(), diff_attention_cached(q, k, v, lam, n))


def test_training_step_in_a_graph():
    q, k, v, lam, do = make(2, 70, 70, 4, 2, 64, 'bf16')
    from panogrf_amd.attention import diff_attention
    ts = [t.clone().requires_grad_(True) for t in (q, k, v, lam)]

    def step():
        out = diff_attention(*ts, causal=True)
        return (out.detach(),) + torch.autograd.grad(out, ts, do)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in range(3):
        new = make(2, 70, 70, 4, 2, 64, 'bf16', seed=seed + 50)
        with torch.no_grad():
            for t, x in zip(ts + [do], new):
                t.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held]
        assert all(torch.equal(a, b) for a, b in zip(got, step()))


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('D', [32, 64, 128])
@pytest.mark.parametrize('N', [20, 50, 140])
def test_partial_last_blocks(N, D, dtype):
    """Workgroups of every size, with a last block of keys that ends at every place of a tile of 64, and what stands behind it not finite."""
    from panogrf_amd.attention import diff_attention_cached
    for M in (20, 40, 84, 116, 148, 212, 257, 300, 383, 447, 511):
        q, k, v, lam, _ = make(2, N, M + 70, 2, 2, D, dtype)
        k[:, M:], v[:, M:] = float('nan'), float('inf')
        n = torch.tensor([M, M + 1 - M % 3], dtype=torch.int32, device='cuda')
        k[1, M:M + 2], v[1, M:M + 2] = 1.0, 1.0
        behind = torch.arange(M + 70, device='cuda') >= n.view(-1, 1)
        kz, vz = k.clone(), v.clone()
        kz[behind], vz[behind] = 0, 0
        ref = R.diff_attention(q, kz, vz, lam, R.may_see(2, N, M + 70, True, lengths=n), D ** -0.5, None, T[dtype])['out']
        assert R.worst(diff_attention_cached(q, k, v, lam, n), *ref) <= 1, M


# one workgroup for all gradients; shares of rows and keys; both with maps kept; the widest heads
WAYS = [(64, 64, 64, 4, 4, 32, 'f32'), (1, 2048, 2048, 4, 2, 64, 'bf16'), (2, 700, 1100, 4, 4, 64, 'f16'), (1, 1100, 1100, 2, 1, 128, 'bf16')]


@pytest.mark.parametrize('B,N,M,H,Hk,D,dtype', WAYS)
def test_training_steps_of_every_way_in_graphs(B, N, M, H, Hk, D, dtype):
    from panogrf_amd.attention import diff_attention
    ts = [t.clone() for t in make(B, N, M, H, Hk, D, dtype)]
    for t in ts[:4]:
        t.requires_grad_(True)
    mask = torch.ones(B, M, dtype=torch.bool, device='cuda')

    def step():
        out = diff_attention(*ts[:4], causal=True, key_mask=mask)
        return (out.detach(),) + torch.autograd.grad(out, ts[:4], ts[4])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in range(3):
        with torch.no_grad():
            for t, x in zip(ts, make(B, N, M, H, Hk, D, dtype, seed=seed + 70)):
                t.copy_(x)
            mask.copy_(torch.arange(M, device='cuda') < M - 13 * seed)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held]
        assert all(torch.equal(a, b) for a, b in zip(got, step()))


def test_calls_beside_each_other():
    """Every way on a stream of its own, all at once: the results of one after the other."""
    args = [make(*w[:7], seed=90) for w in WAYS]
    want = [grads(*a) for a in args]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in WAYS]
    for _ in range(3):
        got = []
        for a, s in zip(args, streams):
            with torch.cuda.stream(s):
                got.append(grads(*a))
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for g, w in zip(got, want) for x, y in zip(g, w))


def test_long_caches_of_one_stream_in_a_graph():
    """The cut of the key axis that a single stream's cache gets, replayed while its length grows."""
    from panogrf_amd.attention import diff_attention_cached
    q, k, v, lam, _ = make(1, 1, 5000, 8, 2, 64, 'bf16')
    n = torch.tensor([4000], dtype=torch.int32, device='cuda')
    diff_attention_cached(q, k, v, lam, n)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = diff_attention_cached(q, k, v, lam, n)
    for length in (4000, 1, 0, 4999, 5000, 33):
        n.fill_(length)
        graph.replay()
        torch.cuda.synchronize()
        got = held.clone()
        assert torch.equal(got, diff_attention_cached(q, k, v, lam, n))
        ref = R.diff_attention(q, k, v, lam, R.may_see(1, 1, 5000, True, lengths=n), 64 ** -0.5, None, T['bf16'])['out']
        assert R.worst(got, *ref) <= 1


def test_on_another_stream():
    q, k, v, lam, do = make(2, 100, 100, 2, 2, 64, 'bf16')
    want = grads(q, k, v, lam, do)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = grads(q, k, v, lam, do)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
