"""Plain 64-bit forms of the token operators and first-order bounds on what float arithmetic and the output's rounding may add.

HALF[t] = eps(t) / 2 is half a step of the type relative to the value; U = 2^-24 is float's.  A float sum of n terms in a chain of k additions is off by at most
k U times the sum of the magnitudes; K = 64 covers the chains of the operators' row sums (at most 32 values per thread, 8 exchanges) and the few products
around them."""
import torch

U = 2.0 ** -24
HALF = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}
K = 64


def worst(got, ref, bound):
    """The largest error over its bound (<= 1 passes); `got` and `ref` must agree in what is not finite."""
    got, ref, bound = got.detach().double().cpu(), ref.detach().double().cpu(), bound.detach().double().cpu()
    assert got.shape == ref.shape, (got.shape, ref.shape)
    assert torch.equal(torch.isfinite(got), torch.isfinite(ref))
    if not got.numel():
        return 0.0
    f = torch.isfinite(ref)
    return float(((got - ref).abs()[f] / bound.expand(ref.shape)[f].clamp_min(1e-300)).max()) if f.any() else 0.0


def norm(a, w, b, kind, eps):
    """-> (value, normalised, mean, 1 / deviation)"""
    m = a.mean(-1, keepdim=True) if kind == 'layer' else torch.zeros_like(a[..., :1])
    r = ((a - m).pow(2).mean(-1, keepdim=True) + eps) ** -0.5
    hat = (a - m) * r
    v = hat if w is None else hat * w
    return (v if b is None else v + b), hat, m, r


def norm_error(a, w, b, hat, m, r, ea, kind):
    """Bound on the error of a norm's value for an input that is off by up to `ea` and float arithmetic."""
    e = ea + K * U * (a.abs() + m.abs())
    e_hat = r * (e + (e.mean(-1, keepdim=True) if kind == 'layer' else 0.0)) + hat.abs() * ((e * hat.abs()).mean(-1, keepdim=True) * r + K * U)
    ww = 1.0 if w is None else w.abs()
    return e_hat * ww + 4 * U * (hat.abs() * ww + (0.0 if b is None else b.abs())), e_hat


def pull(t, hat, r, kind, et, e_hat):
    """Gradient of a norm for t = g w, and a bound on its error for t off by `et` and hat off by `e_hat`."""
    mean = lambda v: v.mean(-1, keepdim=True)
    d = t - hat * mean(t * hat) - (mean(t) if kind == 'layer' else 0.0)
    e = et + hat.abs() * (mean(et * hat.abs()) + mean(t.abs() * e_hat)) + e_hat * mean(t * hat).abs() + (mean(et) if kind == 'layer' else 0.0)
    e = e + K * U * (t.abs() + hat.abs() * mean((t * hat).abs()) + mean(t.abs()))
    return r * d, r * e + K * U * (r * d).abs()


def block_norm(x, y, gate, pw, pb, qw, qb, kind, scale, eps, post, pre, dx1, dz, dtype):
    """Values and gradients in 64 bits, with bounds: {name: (value, bound)}.  gate already broadcast against x (or None)."""
    D = lambda t: None if t is None else t.detach().double()
    x, y, gate, pw, pb, qw, qb, dx1, dz = map(D, (x, y, gate, pw, pb, qw, qb, dx1, dz))
    half, out = HALF[dtype], {}
    rounded = lambda v, e: (v, half * v.abs() + e * (1 + half) + 1e-300 + (6e-8 if dtype == torch.float16 else 0.0))   # (f16: below 2^-14 steps are 2^-24)
    g = torch.ones((), dtype=torch.float64, device=x.device) if gate is None else gate
    if y is not None:
        if post:
            u, hy, my, ry = norm(y, pw, pb, kind, eps)
            eu, ehy = norm_error(y, pw, pb, hy, my, ry, torch.zeros_like(y), kind)
        else:
            u, hy, eu, ehy = y, y, torch.zeros_like(y), torch.zeros_like(y)
        x1 = x + scale * g * u
        e1 = scale * g.abs() * eu + 4 * U * (x.abs() + (scale * g * u).abs())
        out['x'] = rounded(x1, e1)
    else:
        x1, e1 = x, torch.zeros_like(x)
    if pre:
        z, h1, m1, r1 = norm(x1, qw, qb, kind, eps)
        ez, eh1 = norm_error(x1, qw, qb, h1, m1, r1, e1, kind)
        out['z'] = rounded(z, ez)
    if dx1 is None and dz is None:
        return out
    dh, edh = torch.zeros_like(x) if dx1 is None else dx1, torch.zeros_like(x)
    rows = tuple(range(x.dim() - 1))
    chain = 256 + x.numel() // x.shape[-1] / 256          # additions a column sum goes through one after the other, at most
    if pre and dz is not None:
        t = dz if qw is None else dz * qw
        d, e = pull(t, h1, r1, kind, U * t.abs(), eh1)
        dh, edh = dh + d, edh + e + U * (dh.abs() + d.abs())
        column = lambda v, ev: rounded(v.sum(rows), (ev + chain * U * v.abs()).sum(rows))
        out['grad_qw'], out['grad_qb'] = column(dz * h1, dz.abs() * eh1), column(dz, torch.zeros_like(dz))
    out['grad_x'] = rounded(dh, edh)
    if y is None:
        return out
    du, edu = scale * g * dh, scale * g.abs() * edh + 4 * U * (scale * g * dh).abs()
    if post:
        t, et = (du, edu) if pw is None else (du * pw, edu * pw.abs() + U * (du * pw).abs())
        out['grad_y'] = rounded(*pull(t, hy, ry, kind, et, ehy))
    else:
        out['grad_y'] = rounded(du, edu)
    column = lambda v, ev: rounded(v.sum(rows), (ev + chain * U * v.abs()).sum(rows))
    out['grad_pw'], out['grad_pb'] = column(du * hy, edu * hy.abs() + du.abs() * ehy), column(du, edu)
    out['grad_gate_all'] = (scale * dh * u, scale * (edh * u.abs() + dh.abs() * eu) + chain * U * (scale * dh * u).abs())
    return out


def diff_attention(q, k, v, lam, see, scale, dout=None, dtype=None):
    """Values and gradients in 64 bits with first-order bounds: {name: (value, bound)}.  see [B, N, M] bool.

    A product of D values of the type is exact in float, so a score is off by (D + 8) U of its magnitudes (and the power of two behind it by U of the score); a map's value p by
    that much relative to itself, and by the row sum's chain of at most M / 16 + 64 additions.  For the product with v, p is rounded to the type (half a step; in f16
    not below 2^-25, as the row's largest value is at least 1 when it is rounded); the score gradients and p1 - lam p2 likewise in the backward pass.  A sum over n values adds
    (n / 16 + 64) U of their magnitudes: sixteen places of a matrix instruction are added as one."""
    q, k, v, lam = (t.detach().double() for t in (q, k, v, lam))
    B, N, H, _, D = q.shape
    M, Hk = k.shape[1], k.shape[2]
    G = H // Hk
    half = HALF[dtype]
    inner = 0.0 if dtype == torch.float32 else half
    # below the smallest normal float, 2^-126, a value (and a product with a factor of up to 2^6) keeps fewer bits or none: a map of scores 200 apart has such values
    tiny = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -120
    chain = lambda n: (n / 16 + 64) * U
    q = q.view(B, N, Hk, G, 2, D).permute(0, 2, 3, 4, 1, 5)                        # [B, Hk, G, 2, N, D]
    k = k.permute(0, 2, 3, 1, 4).unsqueeze(2)                                      # [B, Hk, 1, 2, M, D]
    keep = see.any(1)[:, None, None, :, None]
    k, v = k.where(keep[:, :, :, None], torch.zeros((), dtype=torch.float64, device=k.device)), v.permute(0, 2, 1, 3).unsqueeze(2).where(keep, torch.zeros((), dtype=torch.float64, device=v.device))
    lam = lam.view(Hk, G, 1, 1)
    s = torch.matmul(q, k.transpose(-1, -2)) * scale
    es = torch.matmul(q.abs(), k.abs().transpose(-1, -2)) * scale * (D + 8) * U
    ok = see[:, None, None, None]
    s = s.masked_fill(~ok, -float('inf'))
    top = s.amax(-1, keepdim=True)
    top = torch.where(top == -float('inf'), torch.zeros_like(top), top)
    p = torch.exp(s - top)
    tot = p.sum(-1, keepdim=True)
    p = p / torch.where(tot == 0, torch.ones_like(tot), tot)
    es = torch.where(ok, es + 4 * U * (1 + s.abs()), torch.zeros_like(s))
    ep = p * (es + (p * es).sum(-1, keepdim=True) + chain(M)) + 2.0 ** -126 * ok   # error of p, unrounded
    o = torch.matmul(p, v.unsqueeze(3))                                            # [B, Hk, G, 2, N, 2D]
    va = v.abs().unsqueeze(3)
    eo = torch.matmul(ep + p * (inner + chain(M)) + tiny * ok, va)
    out = o[:, :, :, 0] - lam * o[:, :, :, 1]
    e = eo[:, :, :, 0] + lam.abs() * eo[:, :, :, 1]
    back = lambda t: t.permute(0, 3, 1, 2, 4).reshape(B, N, H, -1)
    room = 1e-300 + (6e-8 if dtype == torch.float16 else 0.0)
    done = lambda t, err: (t, half * t.abs() + err * (1 + half) + room)
    res = {'out': done(back(out), back(e))}
    if dout is None:
        return res
    do = dout.detach().double().view(B, N, Hk, G, 2 * D).permute(0, 2, 3, 1, 4)    # [B, Hk, G, N, 2D]
    g = torch.matmul(do, v.transpose(-1, -2))
    eg = torch.matmul(do.abs(), v.abs().transpose(-1, -2)) * chain(2 * D)
    delta = (do.unsqueeze(3) * o).sum(-1, keepdim=True)
    ed = (do.abs().unsqueeze(3) * (eo + o.abs() * chain(2 * D))).sum(-1, keepdim=True)
    sign = torch.stack([torch.ones_like(lam), -lam], 2)                            # [Hk, G, 2, 1, 1]
    ds = sign * p * (g.unsqueeze(3) - delta)
    eds = sign.abs() * (p * (eg.unsqueeze(3) + ed) + ep * (g.unsqueeze(3) - delta).abs())
    eds = eds + inner * ds.abs() + 4 * U * ds.abs() + tiny * ok
    dq = scale * torch.matmul(ds, k)
    edq = scale * torch.matmul(eds + chain(M) * ds.abs(), k.abs())
    dk = scale * torch.matmul(ds.transpose(-1, -2), q).sum(2)                      # [B, Hk, 2, M, D]
    edk = scale * torch.matmul((eds + chain(N * G) * ds.abs()).transpose(-1, -2), q.abs()).sum(2)
    pc = p[:, :, :, 0] - lam * p[:, :, :, 1]
    epc = ep[:, :, :, 0] + lam.abs() * ep[:, :, :, 1] + (inner + 2 * U) * pc.abs() + 2 * U * p.sum(3) + tiny * ok[:, :, :, 0]
    dv = torch.matmul(pc.transpose(-1, -2), do).sum(2)
    edv = torch.matmul((epc + chain(N * G) * pc.abs()).transpose(-1, -2), do.abs()).sum(2)
    t = p[:, :, :, 1] * g
    dlam = -t.sum((0, 3, 4)).reshape(H)
    edl = (ep[:, :, :, 1] * g.abs() + p[:, :, :, 1] * eg + chain(M + B * N) * t.abs()).sum((0, 3, 4)).reshape(H)
    res['q'] = done(dq.permute(0, 4, 1, 2, 3, 5).reshape(B, N, H, 2, D), edq.permute(0, 4, 1, 2, 3, 5).reshape(B, N, H, 2, D))
    res['k'] = done(dk.permute(0, 3, 1, 2, 4), edk.permute(0, 3, 1, 2, 4))
    res['v'] = done(dv.permute(0, 2, 1, 3), edv.permute(0, 2, 1, 3))
    res['lam'] = (dlam, edl)
    return res


def may_see(B, N, M, causal, mask=None, lengths=None, device='cuda'):
    i, j = torch.arange(N, device=device).view(1, N, 1), torch.arange(M, device=device).view(1, 1, M)
    end = torch.full((B, 1, 1), M, device=device) if lengths is None else lengths.clamp(0, M).view(B, 1, 1).long()
    see = (j < end).expand(B, N, M)
    if causal:
        see = see & (j <= i + end - N)
    return see if mask is None else see & mask[:, None]
