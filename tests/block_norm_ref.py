"""``block_norm`` and its gradients in 64 bits, and a bound for what fp32 arithmetic may be off.

``exact`` differentiates the definition with autograd.  ``slack`` follows the same formulas with
magnitudes: with u = 2^-24, every element is off by at most a few u of the terms it is made of
(4 u is taken), and the sum of a row's d terms, formed in chains of at most 16 in a thread, 6 levels
across a wave and 16 waves, by 64 u of the sum of the terms' magnitudes.
"""
import torch

U = 2.0 ** -24
ROW = 64 * U
FEW = 4 * U


def norm(v, w, b, eps, rms):
    c = v if rms else v - v.mean(-1, keepdim=True)
    out = c / (c.pow(2).mean(-1, keepdim=True) + eps).sqrt() * w
    return out if b is None else out + b


def exact(t, alpha, eps, rms, dy=None, ds=None):
    """{"y", "s"} and, for the names of `t` given, their gradients "d<name>"."""
    v = {k: x.detach().double().requires_grad_() for k, x in t.items() if x is not None}
    h = v["x"]
    if "post_weight" in v:
        h = norm(h, v["post_weight"], v.get("post_bias"), eps, rms)
    s = v["residual"] + alpha * (h * v["gate"] if "gate" in v else h)
    y = norm(s, v["weight"], v.get("bias"), eps, rms)
    out = {"y": y.detach(), "s": s.detach()}
    outs = [(o, g.double()) for o, g in ((y, dy), (s, ds)) if g is not None]
    if outs:
        grads = torch.autograd.grad([o for o, _ in outs], list(v.values()), [g for _, g in outs], allow_unused=True)
        out.update({"d" + k: g for k, g in zip(v, grads)})
    return out


def _mean(v):
    return v.mean(-1, keepdim=True)


def _normalised(v, e, eps, rms):
    """(n, 1 / deviation, bound of n's error, bound of 1 / deviation's relative error) for v known to within e."""
    m = 0.0 if rms else _mean(v)
    r = (_mean((v - m).pow(2)) + eps).rsqrt()
    n = (v - m) * r
    shift = 0.0 if rms else ROW * _mean(v.abs()) + _mean(e)
    e_c = e + shift + FEW * v.abs()
    rel = ROW + 2 * r * _mean(n.abs() * e_c)
    return n, r, r * e_c + rel * n.abs(), rel


def _transposed(d, e_d, n, e_n, r, rel, w, rms):
    """(value, error bound) of the norm's backward for a gradient d known to within e_d."""
    g, e_g = d * w, e_d * w.abs() + FEW * (d * w).abs()
    p = 0.0 * g if rms else _mean(g)
    e_p = 0.0 if rms else ROW * _mean(g.abs()) + _mean(e_g)
    q = _mean(g * n)
    e_q = ROW * _mean((g * n).abs()) + _mean(e_g * n.abs() + g.abs() * e_n)
    size = g.abs() + (p.abs() + (n * q).abs())
    return r * (g - p - n * q), r * (e_g + e_p + n.abs() * e_q + e_n * q.abs() + (FEW + rel) * size)


def slack(t, alpha, eps, rms, dy=None, ds=None):
    """Bounds of the fp32 errors (before the rounding into the outputs' types), as `exact` is laid out."""
    v = {k: x.detach().double() for k, x in t.items() if x is not None}
    shape = v["x"].shape
    x, zero = v["x"], torch.zeros_like(v["x"])
    n2, r2, e_n2, rel2 = x, 1.0, zero, 0.0
    pw, pb = torch.ones_like(x), zero
    if "post_weight" in v:
        n2, r2, e_n2, rel2 = _normalised(x, zero, eps, rms)
        pw, pb = v["post_weight"], v.get("post_bias", zero)
    h = n2 * pw + pb
    e_h = pw.abs() * e_n2 + FEW * ((n2 * pw).abs() + pb.abs())
    g = v.get("gate", torch.ones_like(x))
    s = v["residual"] + alpha * g * h
    e_s = abs(alpha) * g.abs() * e_h + FEW * (v["residual"].abs() + (alpha * g * h).abs())
    n1, r1, e_n1, rel1 = _normalised(s, e_s, eps, rms)
    w, b = v["weight"], v.get("bias", zero)
    out = {"y": w.abs() * e_n1 + FEW * ((n1 * w).abs() + b.abs()), "s": e_s}
    if dy is None and ds is None:
        return out
    dy_ = zero if dy is None else dy.double()
    d, e = _transposed(dy_, zero, n1, e_n1, r1, rel1, w, rms)
    if ds is not None:
        d, e = d + ds.double(), e + FEW * ds.double().abs()
    e = e + FEW * d.abs()
    out["dresidual"] = e
    dh, e_dh = alpha * g * d, abs(alpha) * g.abs() * e + FEW * (alpha * g * d).abs()
    if "post_weight" in v:
        out["dx"] = _transposed(dh, e_dh, n2, e_n2, r2, rel2, pw, rms)[1]
    else:
        out["dx"] = e_dh
    rows = x.numel() // shape[-1]
    chain = (rows / 256 + 100) * U  # rows of one team, then the teams' and blocks' sums

    def column(value, err, like):
        """A sum over the dimensions in which `like` is broadcast."""
        return (err + (chain + FEW) * value.abs()).sum_to_size(like.shape)

    out["dweight"] = column(dy_ * n1, dy_.abs() * e_n1, w)
    if "bias" in v:
        out["dbias"] = column(dy_, zero, b)
    if "post_weight" in v:
        out["dpost_weight"] = column(dh * n2, e_dh * n2.abs() + dh.abs() * e_n2, pw)
    if "post_bias" in v:
        out["dpost_bias"] = column(dh, e_dh, pb)
    if "gate" in v:
        out["dgate"] = column(alpha * d * h, abs(alpha) * (e * h.abs() + d.abs() * e_h), v["gate"])
    return out
