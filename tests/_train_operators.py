"""64-bit references of the embedding, gated residual norm and gradient clipping operators, and the error bounds that follow from how
they are specified: fp32 sums, statistics and intermediate values (u = 2^-24 a rounding), one rounding of at most half a step
(finfo.eps / 2) on the way to the output type."""
import torch

U = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half the distance between the smallest values of a type (what rounding costs next to zero)."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def check(got, want, bound, what):
    """|got - want| <= bound element by element; bound may be a tensor."""
    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    assert got.shape == want.shape, f"{what}: shape {tuple(got.shape)}, expected {tuple(want.shape)}"
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in other places"
    bound = torch.as_tensor(bound, dtype=torch.float64).cpu().expand_as(want)
    off = (got - want).abs()
    off = torch.where(torch.isnan(want) | (got == want), torch.zeros_like(off), off)
    bad = off > bound
    assert not bool(bad.any()), (f"{what}: {int(bad.sum())} of {bad.numel()} values off, worst {float((off / bound.clamp(min=1e-300)).max()):.3g} times "
                                 f"the bound, first at {bad.nonzero()[0].tolist()}: {float(got[bad][0])!r} for {float(want[bad][0])!r}")


# ------------------------------------------------------------------------------------------------ embedding
def embedding_reference(ids, weight, scale):
    """(y, bound): one product in fp32 (scale itself rounded to fp32), one rounding."""
    V = weight.shape[0]
    w = torch.cat((weight.double().cpu(), torch.zeros(1, weight.shape[1], dtype=torch.float64)))
    i = ids.cpu().long()
    i = torch.where((i < 0) | (i >= V), V, i)
    y = w[i] * scale
    return y, y.abs() * (half_step(weight.dtype) + 3 * U) + tiny(weight.dtype)


def embedding_gradient(ids, dy, V, scale):
    """(dw, bound): n terms added in fp32 in any order are off by at most (n - 1) u of the sum of their magnitudes."""
    D = dy.shape[-1]
    i = ids.cpu().long().reshape(-1)
    d = dy.double().cpu().reshape(-1, D)
    on = (i >= 0) & (i < V)
    i, d = i[on], d[on]
    dw, mag = torch.zeros(V, D, dtype=torch.float64).index_add_(0, i, d), torch.zeros(V, D, dtype=torch.float64).index_add_(0, i, d.abs())
    n = torch.bincount(i, minlength=V).double()[:, None]
    dw = dw * scale
    return dw, mag * abs(scale) * U * (n + 3) + dw.abs() * half_step(dy.dtype) + tiny(dy.dtype)


# ------------------------------------------------------------------------------------------------ gated residual norm
def _norm64(t, gamma, beta, norm, eps):
    m = t.mean(-1, keepdim=True) if norm == "layer" else torch.zeros_like(t[..., :1])
    r = ((t - m).square().mean(-1, keepdim=True) + eps).rsqrt()
    hat = (t - m) * r
    return hat * gamma + (0 if beta is None else beta), hat, r


def gated_reference(x, u, z, keep, keep_scale, post, scale, pre, norm, eps, dy=None, dn=None):
    """Outputs and gradients in 64 bits by the formulas, and a bound for each: {name: (value, bound)}.

    Bounds.  Let c = 4 (D + 16) u.  A row sum of D terms is off by at most D u of its magnitudes, so mean and deviation are off by c / 4 of
    the row's largest magnitude / of themselves; a normalised value (t - m) r is off by c / 4 times (|t| + max|t|) r + |hat|, which is at most
    c H with H = r max|t| + max|hat| over the row.  That error passes on through every product with the factors it meets there.  A
    gradient row through a norm, r (g - mean g - hat mean(g hat)), is off by c r max|g| (1 + H)^2.  A column sum of R rows adds
    (R + 16) u of the sum of its terms' magnitudes to the terms' own errors.  Every output is rounded once."""
    D = x.shape[-1]
    dtype = x.dtype
    ptype = next((t.dtype for t in (*(post or ()), scale, *(pre or ())) if t is not None), torch.float32)

    def d64(t):
        return None if t is None else t.detach().double().cpu().reshape(-1, D)

    def p64(t):
        return None if t is None else t.detach().double().cpu()

    xs, us, zs, dys, dns = (d64(t) for t in (x, u, z, dy, dn))
    R = xs.shape[0]
    on = torch.ones_like(xs, dtype=torch.bool) if keep is None else keep.cpu().reshape(-1, D) != 0
    ks = keep_scale if keep is not None else 1.0
    c = 4 * (D + 16) * U
    hs, hp = half_step(dtype), half_step(ptype)

    def top(t):
        return t.abs().amax(-1, keepdim=True)

    def rounded(err, value, h=hs, t=dtype):
        return err + (value.abs() + err) * h + tiny(t)

    uu = xs if us is None else us
    if post is not None:
        pg, pb = p64(post[0]), p64(post[1])
        v, uhat, ur = _norm64(uu, pg, pb, norm, eps)
        Hu = ur * top(uu) + top(uhat)
        ev = c * Hu * pg.abs() + 3 * U * v.abs()
    else:
        v, ev = uu, torch.zeros_like(uu)
    sig = torch.ones_like(xs) if zs is None else torch.sigmoid(zs)
    w = torch.where(on, sig * ks, 0.0)
    ew = 6 * U * w                                                       # exp, a division and a product
    dwz = torch.where(on, sig * (1 - sig) * ks, 0.0)
    a = torch.ones(D, dtype=torch.float64) if scale is None else p64(scale)
    step = torch.where(on, v * w * a, 0.0)
    es = torch.where(on, (ev * w + v.abs() * ew) * a.abs() + 3 * U * step.abs(), 0.0)
    y = xs + step
    ey = es + U * (xs.abs() + step.abs())
    out = {"y": (y, rounded(ey, y))}
    if pre is not None:
        ng, nb = p64(pre[0]), p64(pre[1])
        n, yhat, yr = _norm64(y, ng, nb, norm, eps)
        Hy = yr * top(y) + top(yhat)
        eh = c * Hy + 4 * top(ey) * yr * (1 + Hy)                        # (statistics from a y that is off by ey)
        out["n"] = (n, rounded(eh * ng.abs() + 3 * U * (n.abs() + (0 if nb is None else nb.abs())), n))
    if dy is None and dn is None:
        return {k: (t.reshape(x.shape), b.reshape(x.shape)) for k, (t, b) in out.items()}
    t = torch.zeros_like(xs) if dys is None else dys
    et = torch.zeros_like(xs)

    def column(terms, errs):
        s = terms.sum(0)
        return s, rounded(errs.sum(0) + (R + 16) * U * (terms.abs() + errs).sum(0), s, hp, ptype)

    if pre is not None and dns is not None:
        g = dns * ng
        m1 = g.mean(-1, keepdim=True) if norm == "layer" else 0.0
        G = yr * (g - m1 - yhat * (g * yhat).mean(-1, keepdim=True))
        t = t + G
        et = yr * top(g) * (1 + Hy) * (c * (1 + Hy) + 4 * eh.amax(-1, keepdim=True)) + U * (t.abs() + G.abs())
        out["dpre_gamma"] = column(dns * yhat, dns.abs() * eh)
        if nb is not None:
            out["dpre_beta"] = column(dns, torch.zeros_like(dns))
    dv = torch.where(on, t * a * w, 0.0)
    edv = torch.where(on, et * a.abs() * w + t.abs() * a.abs() * ew + 3 * U * dv.abs(), 0.0)
    if scale is not None:
        out["dscale"] = column(torch.where(on, t * w * v, 0.0), torch.where(on, et * w * v.abs() + t.abs() * (ew * v.abs() + w * ev) + 3 * U * (t * w * v).abs(), 0.0))
    if zs is not None:
        dz = torch.where(on, t * a * v * dwz, 0.0)
        out["dz"] = (dz, rounded(torch.where(on, (et * v.abs() + t.abs() * ev) * a.abs() * dwz + 10 * U * dz.abs(), 0.0), dz))
    du, edu = dv, edv
    if post is not None:
        out["dpost_gamma"] = column(dv * uhat, edv * uhat.abs() + dv.abs() * c * Hu)
        if pb is not None:
            out["dpost_beta"] = column(dv, edv)
        g = dv * pg
        m1 = g.mean(-1, keepdim=True) if norm == "layer" else 0.0
        du = ur * (g - m1 - uhat * (g * uhat).mean(-1, keepdim=True))
        edu = ur * (1 + Hu) ** 2 * (c * top(g) + 4 * top(edv) * pg.abs().max())
    if us is None:
        out["dx"] = (t + du, rounded(et + edu + U * (t.abs() + du.abs()), t + du))
    else:
        out["dx"] = (t, rounded(et, t))
        out["du"] = (du, rounded(edu, du))
    return {k: ((v_.reshape(x.shape), b.reshape(x.shape)) if v_.dim() == 2 else (v_, b)) for k, (v_, b) in out.items()}


# ------------------------------------------------------------------------------------------------ gradient clipping
def clip_reference(grads, max_norm, p):
    """(norm, its bound, clipped gradients, their bounds): the norm is rounded once from 64 bits, the factor once, the product once."""
    wide = [g.detach().double().cpu() for g in grads]
    every = torch.cat([w.reshape(-1) for w in wide]) if wide else torch.zeros(1, dtype=torch.float64)
    if every.numel() == 0:
        every = torch.zeros(1, dtype=torch.float64)
    norm = every.abs().max() if p == float("inf") else every.abs().pow(p).sum().pow(1 / p)
    if torch.isnan(every).any():
        norm = norm * float("nan")
    factor = max_norm / (norm + 1e-6)
    factor = torch.where(factor > 1, torch.ones_like(factor), factor)
    outs = [w * factor for w in wide]
    return norm, float(norm.abs()) * 2 * U, outs, [o.abs() * (half_step(g.dtype) + 3 * U) + tiny(g.dtype) for o, g in zip(outs, grads)]
