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
