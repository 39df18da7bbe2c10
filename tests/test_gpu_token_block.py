"""The token operators together: a transformer block of block_norm, rotary and diff_attention, its values and gradients against a plain form in 64 bits, as a served model
steps through it, and as the mono-depth net of the framework's own renderer.

Tolerance.  Rounding moves a value by at most half a step of its type (HALF).  The plain form in 64 bits runs again with every intermediate value, and every gradient on its
way back, moved by exactly half a step up or down at random: what that does to a result, in the Euclidean norm, bounds what the roundings of the operators (within half a
step, with a root mean square of 0.58 of it) do to it.  Results of few values (lam) leave more to chance, so the largest of eight such runs counts, twice.  In float the longest
sums, of up to 192 terms, add a deviation of about sqrt(192) < 16 half steps, so values move by 16 there."""
import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

from tests import token_ref as R

pytestmark = pytest.mark.gpu


class _Shake(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, there, back, gen):
        ctx.back, ctx.gen = back, gen
        return _Shake.moved(x, there, gen)

    @staticmethod
    def backward(ctx, g):
        return _Shake.moved(g, ctx.back, ctx.gen), None, None, None

    @staticmethod
    def moved(x, by, gen):
        return x * (1 + by * (2.0 * torch.randint(0, 2, x.shape, generator=gen, device=x.device, dtype=x.dtype) - 1)) if by else x.clone()


class Plain:
    """The operators in 64 bits; step: how far every intermediate value is moved, relative to itself."""

    def __init__(self, step=0.0, seed=0):
        self.step, self.gen = step, torch.Generator(device='cuda').manual_seed(seed)

    def shake(self, x, there=True, back=True):
        return _Shake.apply(x, self.step if there else 0.0, self.step if back else 0.0, self.gen)

    def norm(self, a, w, b, kind, eps):
        return R.norm(a, w, b, kind, eps)[0]

    def block_norm(self, x, y=None, gate=None, post_weight=None, post_bias=None, pre_weight=None, pre_bias=None, kind='rms', scale=1.0, eps=1e-6):
        if y is not None:
            y = self.norm(self.shake(y, False), post_weight, post_bias, kind, eps)
            x = x + scale * (y if gate is None else y * (gate.unsqueeze(1) if gate.dim() == 2 else gate))
        z = self.shake(self.norm(x, pre_weight, pre_bias, kind, eps))
        return self.shake(x), z

    def rotary(self, q, k, positions):
        d = q.shape[-1]
        f = 10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64, device=q.device) / d)
        a = positions.double()[..., None] * f
        a = a if a.dim() == 3 else a[None]

        def turn(x):
            c, s = (t.view(t.shape[0], t.shape[1], *[1] * (x.dim() - 3), d // 2) for t in (a.cos(), a.sin()))
            u, v = x[..., :d // 2], x[..., d // 2:]
            return self.shake(torch.cat([u * c - v * s, v * c + u * s], -1))
        return turn(q), turn(k)

    def diff_attention(self, q, k, v, lam, causal=False, key_mask=None, lengths=None):
        B, N, H, _, d = q.shape
        M, G = k.shape[1], H // k.shape[2]
        see = R.may_see(B, N, M, causal, key_mask, lengths)[:, None]
        k, v = k.repeat_interleave(G, 2), v.repeat_interleave(G, 2).transpose(1, 2)
        out = []
        for i in (0, 1):
            s = self.shake(torch.matmul(q[..., i, :].transpose(1, 2), k[..., i, :].permute(0, 2, 3, 1)) * d ** -0.5, False)      # (scores stay float; their gradients are rounded)
            s = s.masked_fill(~see, -float('inf'))
            top = s.detach().amax(-1, keepdim=True)
            p = torch.exp(s - top.masked_fill(top == -float('inf'), 0.0))
            total = p.sum(-1, keepdim=True)
            out.append(torch.matmul(self.shake(p / total.masked_fill(total == 0, 1.0), True, False), v))
        return self.shake((out[0] - lam[:, None, None] * out[1]).transpose(1, 2))

    def linear(self, x, w):
        return self.shake(x @ w.t())


class Own:
    def __init__(self):
        from panogrf_amd import attention, block_norm, rotary
        self.block_norm, self.rotary, self.diff_attention = block_norm.block_norm, rotary.rotary, attention.diff_attention
        self.cached = attention.diff_attention_cached

    def linear(self, x, w):
        return F.linear(x, w)


def weights(C, H, Hk, d, dtype, kind, seed=0):
    g = torch.Generator(device='cuda').manual_seed(seed)
    r = lambda *s, std=1.0, mean=0.0: (torch.randn(*s, generator=g, device='cuda') * std + mean).to(dtype)
    w = dict(pre=r(C, std=0.1, mean=1.0), qkv=r((2 * H + 4 * Hk) * d, C, std=C ** -0.5), head=r(2 * d, std=0.1, mean=1.0), lam=torch.rand(H, generator=g, device='cuda').to(dtype),
             out=r(C, 2 * d * H, std=(2 * d * H) ** -0.5), post=r(C, std=0.1, mean=1.0), gate=r(C, std=0.3, mean=0.5), next=r(C, std=0.1, mean=1.0))
    if kind == 'layer':
        w.update(pre_b=r(C, std=0.1), post_b=r(C, std=0.1), next_b=r(C, std=0.1))
    return w


def qkv_of(ops, w, z, H, Hk, d):
    qkv = ops.linear(z, w['qkv'])
    q, k, v = qkv.split([2 * H * d, 2 * Hk * d, 2 * Hk * d], -1)                   # (views of one projection)
    return q.unflatten(-1, (H, 2, d)), k.unflatten(-1, (Hk, 2, d)), v.unflatten(-1, (Hk, 2 * d))


def behind(ops, w, x, o, kind, sample_gate=None):
    o = ops.block_norm(o, pre_weight=w['head'])[1]                                 # every head by itself
    y = ops.linear(o.flatten(-2), w['out'])
    return ops.block_norm(x, y, gate=w['gate'] if sample_gate is None else sample_gate, post_weight=w['post'], post_bias=w.get('post_b'), pre_weight=w['next'],
                          pre_bias=w.get('next_b'), kind=kind, scale=0.5)


def block(ops, w, x, positions, sizes, kind, sample_gate, **see):
    z = ops.block_norm(x, pre_weight=w['pre'], pre_bias=w.get('pre_b'), kind=kind)[1]
    q, k, v = qkv_of(ops, w, z, *sizes)
    q, k = ops.rotary(q, k, positions)
    return behind(ops, w, x, ops.diff_attention(q, k, v, w['lam'], **see), kind, sample_gate)


def close(name, got, exact, moved):
    scale = max(float((m - exact).norm()) for m in moved)
    assert torch.isfinite(got).all(), name
    assert float((got.double() - exact).norm()) <= 2 * scale, (name, float((got.double() - exact).norm()), scale)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('B,N,C,H,Hk,d,kind,causal,masked,per_sample', [
    (2, 70, 96, 4, 2, 32, 'rms', True, False, False), (3, 33, 192, 2, 2, 64, 'layer', False, True, True), (1, 130, 136, 4, 1, 32, 'rms', False, True, False)])
def test_a_block_in_training(B, N, C, H, Hk, d, kind, causal, masked, per_sample, dtype):
    g = torch.Generator(device='cuda').manual_seed(5)
    r = lambda *s: torch.randn(*s, generator=g, device='cuda').to(dtype)
    w, x, dx, dz = weights(C, H, Hk, d, dtype, kind), r(B, N, C), r(B, N, C), r(B, N, C)
    sample_gate = r(B, C) if per_sample else None
    mask = None
    if masked:
        mask = torch.rand(B, N, generator=g, device='cuda') > 0.3
        if B > 1:
            mask[0] = False                                                        # a panorama whose tokens see nothing
    positions = torch.rand(B, N, generator=g, device='cuda') * 14.5

    def run(ops, to):
        leaf = lambda t: t.detach().to(to).requires_grad_(True)
        ww, xx, sg = {n: leaf(t) for n, t in w.items()}, leaf(x), None if sample_gate is None else leaf(sample_gate)
        leaves = {**ww, 'x': xx}
        if sg is not None:
            leaves['sample_gate'] = sg
            del leaves['gate']
        x1, z = block(ops, ww, xx, positions, (H, Hk, d), kind, sg, causal=causal, key_mask=mask)
        gs = torch.autograd.grad([x1, z], list(leaves.values()), [dx.to(to), dz.to(to)])
        return {'x1': x1.detach(), 'z': z.detach(), **{'grad_' + n: t for n, t in zip(leaves, gs)}}
    own, exact = run(Own(), dtype), run(Plain(), torch.float64)
    step = R.HALF[dtype] * (16 if dtype == torch.float32 else 1)
    moved = [run(Plain(step, s + 1), torch.float64) for s in range(8)]
    for n in exact:
        close(n, own[n], exact[n], [m[n] for m in moved])
    assert all(torch.equal(a, b) for a, b in zip(own.values(), run(Own(), dtype).values()))


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
def test_a_block_served_token_by_token(dtype):
    """A prompt into the cache, then single tokens of ragged streams in one captured step, against the block over all tokens at once."""
    B, C, H, Hk, d, first, steps, room = 3, 128, 4, 2, 32, (5, 17, 9), 4, 40
    sizes, ops, kind = (H, Hk, d), Own(), 'rms'
    g = torch.Generator(device='cuda').manual_seed(9)
    w, x = weights(C, H, Hk, d, dtype, kind), torch.randn(B, room, C, generator=g, device='cuda').to(dtype)
    kc, vc = (torch.full((B, room, Hk, *s), float('nan'), device='cuda', dtype=dtype) for s in ((2, d), (2 * d,)))
    at = torch.arange(B, device='cuda')
    lengths = torch.zeros(B, dtype=torch.int32, device='cuda')
    rows = torch.empty(B, 1, C, device='cuda', dtype=dtype)
    with torch.no_grad():
        for b, n in enumerate(first):                                              # prompts, one by one
            z = ops.block_norm(x[b:b + 1, :n].contiguous(), pre_weight=w['pre'])[1]
            q, k, v = qkv_of(ops, w, z, *sizes)
            _, kr = ops.rotary(q, k, torch.arange(n, device='cuda'))
            kc[b, :n], vc[b, :n] = kr[0], v[0]
        lengths.copy_(torch.tensor(first, dtype=torch.int32))

        def step():
            z = ops.block_norm(rows, pre_weight=w['pre'])[1]
            q, k, v = qkv_of(ops, w, z, *sizes)
            q, k = ops.rotary(q, k, lengths[:, None])
            kc[at, lengths.long()] = k[:, 0]
            vc[at, lengths.long()] = v[:, 0]
            lengths.add_(1)
            return behind(ops, w, rows, ops.cached(q, kc, vc, w['lam'], lengths), kind)
        held = (kc.clone(), vc.clone(), lengths.clone())
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        rows.copy_(x[:, :1])
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        for t, saved in zip((kc, vc, lengths), held):
            t.copy_(saved)
        got = []
        for i in range(steps):
            rows.copy_(torch.stack([x[b, n + i] for b, n in enumerate(first)])[:, None])
            graph.replay()
            torch.cuda.synchronize()
            got.append([t.clone() for t in out])
    wd = {n: t.double() for n, t in w.items()}

    def whole(step_, seed):
        with torch.no_grad():
            return [block(Plain(step_, seed), wd, x[b:b + 1, :n + steps].double(), torch.arange(n + steps, device='cuda'), sizes, kind, None, causal=True)
                    for b, n in enumerate(first)]
    exact, moved = whole(0.0, 0), [whole(R.HALF[dtype], s + 1) for s in range(8)]
    for b, n in enumerate(first):
        for j, name in enumerate(('x1', 'z')):
            close((name, b), torch.stack([got[i][j][b, 0] for i in range(steps)]), exact[b][j][0, n:], [m[b][j][0, n:] for m in moved])


def test_second_derivatives_are_refused():
    from panogrf_amd import attention, block_norm, rotary
    x = torch.randn(1, 4, 2, 2, 32, device='cuda', requires_grad=True)
    v, lam = torch.randn(1, 4, 2, 64, device='cuda'), torch.rand(2, device='cuda')
    for out in (attention.diff_attention(x, x, v, lam), block_norm.block_norm(x)[1], rotary.rotary(x, None, torch.arange(4, device='cuda'))[0]):
        g, = torch.autograd.grad(out.square().sum(), x, create_graph=True)         # (the gradient itself is given)
        assert torch.isfinite(g).all()
        with pytest.raises(RuntimeError):
            torch.autograd.grad(g.square().sum(), x)


@pytest.fixture
def room():
    """Tensors of over 2^31 values, here and nowhere else."""
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip('needs 60 GB')
    yield
    torch.cuda.empty_cache()


def test_norms_and_rotations_of_over_2_to_the_31_values(room):
    """What stands behind 2^31 values is what the same rows give by themselves."""
    from panogrf_amd.block_norm import block_norm
    from panogrf_amd.rotary import rotary
    rows, C = 265000, 8192
    x = torch.randn(rows, C, device='cuda', dtype=torch.bfloat16)
    y, ends = x.flip(1), (slice(0, 300), slice(rows - 300, rows))
    assert x.numel() > 2 ** 31
    w = torch.rand(C, device='cuda').to(x.dtype)
    for e in ends:
        xs, ys = x[e].clone(), y[e].clone()
        got = block_norm(x, y, post_weight=w, kind='layer')
        assert all(torch.equal(a[e], b) for a, b in zip(got, block_norm(xs, ys, post_weight=w, kind='layer')))
        del got
    xl, yl = x.requires_grad_(True), y.requires_grad_(True)
    out = block_norm(xl, yl, post_weight=w, kind='rms')
    dx, dy = torch.autograd.grad(out, [xl, yl], [x.detach(), y.detach()])
    del out
    for e in ends:
        xs, ys = x.detach()[e].clone().requires_grad_(True), y.detach()[e].clone().requires_grad_(True)
        want = torch.autograd.grad(block_norm(xs, ys, post_weight=w, kind='rms'), [xs, ys], [xs.detach(), ys.detach()])
        assert torch.equal(dx[e], want[0]) and torch.equal(dy[e], want[1])
    del xl, yl, dx, dy, y
    q = x.detach().view(1, rows, 128, 64)
    turned, _ = rotary(q, None, torch.arange(rows, device='cuda'))
    for e in ends:
        assert torch.equal(turned[:, e], rotary(q[:, e].clone(), None, torch.arange(rows, device='cuda')[e])[0])


def test_attention_of_over_2_to_the_31_values(room):
    from panogrf_amd.attention import diff_attention
    B, N, M, H, D = 2, 131100, 33, 64, 64
    q = torch.randn(B, N, H, 2, D, device='cuda', dtype=torch.bfloat16)
    assert q.numel() > 2 ** 31
    k, v, lam = torch.randn(B, M, H, 2, D, device='cuda').to(q.dtype), torch.randn(B, M, H, 2 * D, device='cuda').to(q.dtype), torch.rand(H, device='cuda')
    q.requires_grad_(True)
    out = diff_attention(q, k, v, lam)
    dq, = torch.autograd.grad(out, q, q.detach().view(B, N, H, 2 * D))
    qs = q.detach()[1:, N - 200:].clone().requires_grad_(True)
    alone = diff_attention(qs, k[1:], v[1:], lam)
    ds, = torch.autograd.grad(alone, qs, qs.detach().view(1, 200, H, 2 * D))
    # (which rows share a workgroup does not enter a row's sums)
    assert torch.equal(out[1:, N - 200:], alone) and torch.equal(dq[1:, N - 200:], ds)


class TokenMono(nn.Module):
    """A small mono-depth net over the panorama's patches, behind the renderer's call d_net(erp, cube, dnet=True) -> {'pred_depth', 'mono_feat'}."""

    def __init__(self, ops, C=64, H=2, Hk=1, d=32, patch=8):
        super().__init__()
        self.ops, self.sizes, self.patch = ops, (H, Hk, d), patch
        self.embed = nn.Conv2d(3, C, patch, patch)
        self.w = nn.ParameterDict(weights(C, H, Hk, d, torch.float32, 'layer', seed=3))
        self.depth, self.feat = nn.Conv2d(C, 1, 1), nn.Conv2d(C, 32, 1)

    def forward(self, erp, cube=None, dnet=True):
        e = self.embed(erp)
        n, C, h, w = e.shape
        to = torch.float64 if isinstance(self.ops, Plain) else e.dtype
        x = e.flatten(2).transpose(1, 2).contiguous().to(to)
        ww = {k: t.to(to) for k, t in self.w.items()}
        z = block(self.ops, ww, x, torch.arange(h * w, device=x.device), self.sizes, 'layer', None)[1]
        z = z.to(e.dtype).transpose(1, 2).unflatten(2, (h, w)).contiguous()
        return {'pred_depth': 1.0 + 6.0 * torch.sigmoid(self.depth(z)), 'mono_feat': self.feat(z)}


def test_a_token_net_as_the_renderer_s_mono_depth_net():
    import numpy as np
    from panogrf_amd.imgs_info import build_imgs_info, build_render_imgs_info, imgs_info_to_torch
    from panogrf_amd.renderer import name2network
    from tests import mvs_fixtures as MF
    H, W, dn = 64, 128, 32
    cfg = dict(MF.MVS_ARGS, height=H, width=W, mono_height=64, mono_width=128, depth_height=32, depth_width=64, network='neuray_gen', init_net_type='cost_volume',
               use_wrap_padding=True, seq_len=3, use_disp=True, use_hierarchical_sampling=True, render_depth=True, depth_sample_num=dn, fine_depth_sample_num=dn,
               sample_num=dn, dist_decoder_cfg={'use_vis': False}, fine_dist_decoder_cfg={'use_vis': False}, min_depth=0.5, max_depth=15.0)
    torch.manual_seed(0)
    net = name2network['neuray_gen'](cfg, d_net=TokenMono(Own())).cuda().eval()
    g = torch.Generator().manual_seed(1)
    imgs = torch.rand(2, 3, H, W, generator=g).numpy()
    pose = lambda tx: np.concatenate([np.eye(3), np.array([[tx], [0.0], [0.0]])], 1)
    ref = imgs_info_to_torch(build_imgs_info(imgs, np.stack([pose(0.5), pose(-0.5)]), [[0.5, 15.0]] * 2), 'cuda')
    src = imgs_info_to_torch(build_imgs_info(imgs[::-1].copy(), np.stack([pose(-0.5), pose(0.5)]), [[0.5, 15.0]] * 2), 'cuda')
    que = imgs_info_to_torch(build_render_imgs_info(pose(0.0), (H, W), [0.5, 15.0]), 'cuda')
    frame = lambda: net({'que_imgs_info': dict(que), 'ref_imgs_info': dict(ref), 'src_imgs_info': dict(src), 'eval': True})
    mono = net.init_net.depth_net.d_net
    seen = []
    with torch.no_grad():
        net.cfg['hip_reuse_source_maps'] = False
        frames = [frame(), frame()]                                                # the stage goes into a graph with this net in it, and is replayed
        assert torch.isfinite(frames[0]['pixel_colors_nr_fine']).all()
        for k in ('pixel_colors_nr_fine', 'render_depth_fine'):
            assert torch.equal(frames[0][k], frames[1][k]), k
        replayed = {k: t.clone() for k, t in net._run_init_net(ref, src, False).items()}
        hook = mono.register_forward_hook(lambda m, i, o: seen.append((i[0].clone(), {k: t.clone() for k, t in o.items()})))
        launched = net.__dict__['_hip_init'](ref, src, False)                      # the same stage, launch by launch
        hook.remove()
        assert len(seen) == 1
        for k in ('ray_feats', 'mvs_depth'):
            assert torch.equal(replayed[k], launched[k]), k
        # what the net gave the renderer, against its plain form
        x, out = seen[0]
        plain = lambda step, seed: [setattr(mono, 'ops', Plain(step, seed)), mono(x)][1]
        exact, moved = plain(0.0, 0), [plain(16 * R.U, s + 1) for s in range(8)]
        for k in exact:
            close(k, out[k], exact[k].double(), [m[k].double() for m in moved])
