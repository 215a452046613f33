"""fp64 oracles of the language-model operators, each value with a bound on its rounding error.

U is the unit roundoff of fp32 (2^-24); u(t) that of a stored type.  A kernel sums at most 16 values per
thread serially and then 64 to 1024 threads as a tree (at most 10 levels), with a handful of products and a
square root (or a division) around it: fewer than K = 64 roundings between an input and an output of a row.
Sums over rows are serial in the worst case.  An input held in a type is exact.
"""
import torch

U = 2.0 ** -24
K = 64
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -133, torch.float32: 2.0 ** -149, torch.float64: 0.0}


def u(t):
    return torch.finfo(t).eps / 2


def within(got, ref, bound, what=""):
    """|got - ref| <= bound + the rounding of ref to got's type (places where ref is not finite agree in kind)."""
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    g, ref = got.detach().double(), ref.double()
    fine = torch.isfinite(ref)
    assert torch.equal(torch.isfinite(g), fine) and torch.equal(torch.isnan(g), torch.isnan(ref)), what
    lim = bound * (1 + u(got.dtype)) + u(got.dtype) * ref.abs() + TINY[got.dtype]
    over = ((g - ref).abs() - lim)[fine]
    worst = float(over.max()) if over.numel() else -1.0
    assert worst <= 0, f"{what}: {worst:.3g} over its bound, at most {float(((g - ref).abs() / lim)[fine].max()):.3g} x"


def embedding(ids, weight, scale, pad, dy):
    """y, bound, dw, bound; tokens outside the table give NaN rows and no gradient."""
    rows, d = weight.shape
    flat = ids.reshape(-1).long()
    ok = (flat >= 0) & (flat < rows)
    w = weight.double()
    y = torch.full((flat.numel(), d), float("nan"), dtype=torch.float64, device=weight.device)
    y[ok] = w[flat[ok]] * scale
    yb = y.abs() * 2 * U  # scale to fp32, and the product
    use = ok & (flat != pad) if pad is not None else ok
    g = dy.reshape(-1, d).double()
    at = flat[use]
    dw = torch.zeros(rows, d, dtype=torch.float64, device=weight.device).index_add_(0, at, g[use])
    mass = torch.zeros(rows, d, dtype=torch.float64, device=weight.device).index_add_(0, at, g[use].abs())
    count = torch.zeros(rows, 1, dtype=torch.float64, device=weight.device)
    count.index_add_(0, at, torch.ones(at.numel(), 1, dtype=torch.float64, device=weight.device))
    return y.view(*ids.shape, d), yb.view(*ids.shape, d), dw * scale, mass * abs(scale) * U * (count + 3)


def _norm(v, vb, w, b, rms, eps):
    """hat, its bound, 1 / deviation, out, its bound, for rows v known to vb"""
    m = 0.0 if rms else v.mean(-1, keepdim=True)
    r = 1 / ((v - m).square().mean(-1, keepdim=True) + eps).sqrt()
    hat = (v - m) * r
    size = v.abs() + (0.0 if rms else v.abs().mean(-1, keepdim=True))
    vb = vb + (0.0 if rms else vb.mean(-1, keepdim=True))
    d = (K * U * size + vb) * r  # of (v - m) r with r exact
    hatb = d + hat.abs() * ((d * hat.abs()).mean(-1, keepdim=True) + K * U)  # and r's own
    out = hat * w if w is not None else hat
    outb = hatb * (w.abs() if w is not None else 1.0) + 2 * U * out.abs()
    if b is not None:
        out = out + b
        outb = outb + U * out.abs()
    return hat, hatb, r, out, outb


def _norm_back(hat, hatb, r, a, ab, rms):
    """The gradient of the norm's input for the gradient a of hat, and its bound."""
    c1 = 0.0 if rms else a.mean(-1, keepdim=True)
    c2 = (a * hat).mean(-1, keepdim=True)
    c1b = 0.0 if rms else ab.mean(-1, keepdim=True)
    mass = a.abs() + (0.0 if rms else a.abs().mean(-1, keepdim=True)) + hat.abs() * (a * hat).abs().mean(-1, keepdim=True)
    c2b = (ab * hat.abs() + a.abs() * hatb).mean(-1, keepdim=True)
    g = r * (a - c1 - hat * c2)
    return g, r * (ab + c1b + hatb * c2.abs() + hat.abs() * c2b + K * U * mass) + K * U * g.abs()


def residual_norm(y, x, weight, bias, gate, post_weight, post_bias, rms, eps, alpha, post, dh, ds):
    """{name: (value, bound)} of h, s and the gradients.  dh or ds may be None."""
    wide = [None if t is None else t.double() for t in (y, x, weight, bias, gate, post_weight, post_bias, dh, ds)]
    y_, x_, w, b, g, pw, pb, dh_, ds_ = wide
    zero = torch.zeros_like(y_)
    if post:
        phat, phatb, pr, un, ub = _norm(y_, zero, pw, pb, rms, eps)
    else:
        un, ub = y_, zero
    gu = un if g is None else un * g
    gub = ub if g is None else ub * g.abs() + U * gu.abs()
    s = gu if x is None else alpha * x_ + gu
    sb = gub if x is None else gub + 2 * U * ((alpha * x_).abs() + gu.abs())
    hat, hatb, r, h, hb = _norm(s, sb, w, b, rms, eps)
    out = {"h": (h, hb), "s": (s, sb)}
    if dh is None and ds is None:
        return out
    kept = y.dtype if x is None else x.dtype  # s is read back in its own type
    if not (x is None and g is None and not post):
        hatb = hatb + u(kept) * (s.abs() + (0.0 if rms else s.abs().mean(-1, keepdim=True))) * r
    dh_ = zero if dh is None else dh_
    a = dh_ if w is None else dh_ * w
    S, Sb = _norm_back(hat, hatb, r, a, U * a.abs(), rms)
    if dh is None:
        S, Sb = zero, zero
    if ds is not None:
        S = S + ds_
        Sb = Sb + U * S.abs()
    lead = tuple(range(y.dim() - 1))
    rows = max(1, y.numel() // y.shape[-1])

    def total(v, vb, like):
        """sum over the rows that share one value of `like`"""
        dims = [k for k in lead if like.dim() == 1 or like.shape[k] == 1 and y.shape[k] != 1]
        keep = like.dim() > 1
        both = [(t.sum(dims, keepdim=keep) if dims else t) for t in (v, vb + (rows + 4) * U * v.abs())]
        return tuple(t.reshape(like.shape) for t in both)

    if x is not None:
        out["dx"] = (alpha * S, abs(alpha) * Sb + 2 * U * (alpha * S).abs())
    if w is not None:
        out["dweight"] = total(dh_ * hat, dh_.abs() * hatb, w)
    if b is not None:
        out["dbias"] = total(dh_, zero, b)
    du, dub = (S, Sb) if g is None else (S * g, Sb * g.abs() + U * (S * g).abs())
    if g is not None:
        out["dgate"] = total(S * un, Sb * un.abs() + S.abs() * ub, g)
    if post:
        if pw is not None:
            out["dpost_weight"] = total(du * phat, dub * phat.abs() + du.abs() * phatb, pw)
        if pb is not None:
            out["dpost_bias"] = total(du, dub, pb)
        a = du if pw is None else du * pw
        du, dub = _norm_back(phat, phatb, pr, a, (dub if pw is None else dub * pw.abs()) + U * a.abs(), rms)
    out["dy"] = (du, dub)
    return out
