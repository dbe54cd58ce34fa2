"""The gated residual norm and its gradients in 64 bits, step by step as fp32 code takes them, every value with a bound on
what fp32 arithmetic may be off by.

A Val is a value x and an absolute bound e: what an fp32 computation of it returns lies within e.  With u = 2^-24 a
product of a and b is off by |a| eb + |b| ea + ea eb and a rounding of u; a sum of n terms by the terms' bounds and `depth`
roundings of the sum of their magnitudes, where depth is the longest chain of additions that a term passes.  The bounds
are made of each element's own terms, so a missing or wrong term of any size above the rounding shows
(test_norm_bounds.py breaks the gradients in many ways and has every bound refuse them)."""
import torch

U = 2.0**-24
ROW_DEPTH = 41   # a lane adds at most 32 columns, then 6 steps in a wave and 3 across waves


class Val:
    def __init__(self, x, e=0.0):
        self.x = x
        self.e = e if torch.is_tensor(e) else torch.full_like(x, e)

    def _rounded(self, x, e):
        return Val(x, e + U * (x.abs() + e))

    def __mul__(self, o):
        return self._rounded(self.x * o.x, self.x.abs() * o.e + o.x.abs() * self.e + self.e * o.e)

    def __add__(self, o):
        return self._rounded(self.x + o.x, self.e + o.e)

    def __sub__(self, o):
        return self._rounded(self.x - o.x, self.e + o.e)

    def sum(self, dim, depth, keepdim=True):
        e, mag = self.e.sum(dim, keepdim=keepdim), (self.x.abs() + self.e).sum(dim, keepdim=keepdim)
        g = depth * U
        return Val(self.x.sum(dim, keepdim=keepdim), e + g / (1 - g) * mag)

    def rsqrt(self):
        """The function itself within 2 units in the last place."""
        r = self.x.rsqrt()
        return Val(r, (self.x - self.e).rsqrt() - r + 4 * U * r)


def number(v):
    """A number that the kernel gets in fp32."""
    t = torch.tensor(float(v), dtype=torch.float64)
    return Val(t, U * t.abs())


def _mean(v, C):
    return v.sum(1, ROW_DEPTH) * number(1.0 / C)


def _normalise(v, kind, eps):
    """(v - mean) * rstd and rstd"""
    C = v.x.shape[1]
    d = v - _mean(v, C) if kind == "layer" else v
    r = (_mean(d * d, C) + number(eps)).rsqrt()
    return d * r, r


def _norm_back(gw, vh, kind, rstd, drop):
    C = gw.x.shape[1]
    m2 = _mean(gw * vh, C)
    d = gw
    if kind == "layer" and "mean" not in drop:
        d = d - _mean(gw, C)
    if "projection" not in drop:
        d = d - vh * m2
    return rstd * d


def column_depth(M):
    """Chain of a column sum: a workgroup's rows of a lane (512 workgroups of at least one row slot, several samples in
    turn), 6 + 3 steps in the workgroup, 32 partial rows a wave, 16 waves; rounded up."""
    return 80 + M // 256


def gated_norm(t, dy, dh, alpha, post, pre, rps, eps=1e-5, drop=()):
    """t: f, x, gate (None, [C] or [samples, C]), rs, post_w, post_b, pre_w, pre_b.  Returns {name: Val} of y, h and the
    gradients of those present, for gradients dy and dh (None: zero).  drop: what a broken backward leaves out."""
    M, C = t["f"].shape
    v = {n: None if p is None else Val(p.detach().cpu().double()) for n, p in t.items()}
    one, zero = Val(torch.ones(1, C).double()), Val(torch.zeros(1, C).double())
    gate, samples = v["gate"] or one, 1
    if t["gate"] is not None and t["gate"].ndim == 2:
        samples = t["gate"].shape[0]
        gate = Val(gate.x.repeat_interleave(M // samples, 0))
    rs = Val(torch.ones(M, 1).double()) if v["rs"] is None else Val(v["rs"].x.repeat_interleave(rps)[:M, None])
    w0, b0, w1, b1 = v["post_w"] or one, v["post_b"] or zero, v["pre_w"] or one, v["pre_b"] or zero
    al = number(alpha)
    fh, r0 = _normalise(v["f"], post, eps) if post else (v["f"], None)
    y = rs * gate * (fh * w0 + b0) + al * v["x"]
    out = {"y": y}
    if pre:
        yh, r1 = _normalise(y, pre, eps)
        out["h"] = yh * w1 + b1
    depth = column_depth(M)
    dY = Val(torch.zeros(M, C).double())
    if dh is not None and pre:
        g = Val(dh.detach().cpu().double())
        out["pre_w"], out["pre_b"] = (g * yh).sum(0, depth, False), g.sum(0, depth, False)
        dY = _norm_back(g * w1, yh, pre, r1, drop if "in pre" in drop else ())
    if dy is not None and "dy" not in drop:
        dY = dY + Val(dy.detach().cpu().double())
    out["x"] = dY if "alpha" in drop else al * dY
    dYr = dY if "row scale" in drop else dY * rs
    a, b = dYr * fh, dYr
    if samples > 1:
        # a sample's sums close into its gate's gradient over its row chunks (at most 512 in turn)
        A, B = (Val(p.x.view(samples, -1, C), p.e.view(samples, -1, C)).sum(1, depth, False) for p in (a, b))
        dg = A * w0 + B * b0
        dg = Val(dg.x, dg.e + 512 * U * (a.x.abs() * w0.x.abs() + b.x.abs() * b0.x.abs()).view(samples, -1, C).sum(1))
        gs = v["gate"]
        out["gate"], dw, db = dg, (gs * A).sum(0, 8 + samples // 512, False), (gs * B).sum(0, 8 + samples // 512, False)
    else:
        A, B = a.sum(0, depth, False), b.sum(0, depth, False)
        dg = A * w0 + B * b0
        g1 = Val(gate.x.reshape(-1, C)[0])
        out["gate"], dw, db = Val(dg.x.view(-1, C)[0], dg.e.view(-1, C)[0]), g1 * A, g1 * B
    out["post_w"], out["post_b"] = dw, db
    dn = dYr if "gate" in drop else dYr * gate
    out["f"] = _norm_back(dn * w0, fh, post, r0, drop if "in post" in drop else ()) if post else dn
    for n in ("gate", "post_w", "post_b", "pre_w", "pre_b"):
        if t[n] is None:
            out.pop(n, None)
    if t["gate"] is not None and t["gate"].ndim == 2 and samples == 1:
        out["gate"] = Val(out["gate"].x[None], out["gate"].e[None])
    return out


def excess(got, want, dtype=None):
    """How far got lies outside want's bound (<= 0: inside); dtype: the type that got was rounded to from fp32."""
    tol = want.e
    if dtype is not None and dtype is not torch.float32:
        tol = tol + torch.finfo(dtype).eps / 2 * (want.x.abs() + want.e)
    err = (got.detach().cpu().double() - want.x).abs() - tol
    return float("inf") if err.isnan().any() else err.max().item()


def case(M, C, dtype, post, pre, samples=0, rs=0, bias=True, seed=0):
    """Inputs and the two gradients.  samples: 0 for a gate per channel; rs: rows a row factor (0: none)."""
    g = torch.Generator().manual_seed(1000 * seed + M + C)
    n = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    t = {"f": (2 * n(M, C)).to(dtype), "x": (n(M, C) + 0.5).to(dtype), "gate": n(*((samples, C) if samples else (C,)))}
    for k, kind in (("post", post), ("pre", pre)):
        t[k + "_w"] = 1 + 0.2 * n(C) if kind else None
        t[k + "_b"] = 0.2 * n(C) if kind and bias else None
    t["rs"] = (torch.rand(-(-M // rs), generator=g) < 0.8).float() / 0.8 if rs else None
    return t, n(M, C).to(dtype), n(M, C).to(dtype)


B, F = torch.bfloat16, torch.float32
# (M, C, type, post, pre, samples, rs, alpha): every width class of the kernels (vectors of 4 and 8, single columns; a part
# of a wave, a wave, a workgroup), the norm kinds, more samples than workgroups, more rows than a workgroup takes at once
CASES = ([(9, C, dt, "layer", "layer", 0, 0, 1.0) for C in (8, 48, 130, 264, 331, 520, 768, 776, 1024, 1025, 1032, 2056, 4096, 4099, 8192)
          for dt in (B, F)]
         + [(37, C, dt, post, pre, 0, 5, 0.7) for C in (96, 97, 2000) for dt in (B, F) for post in (None, "layer", "rms")
            for pre in (None, "layer", "rms")]
         + [(M, C, dt, "rms", "layer", samples, rs, 1.0) for M, samples, rs in ((6, 2, 3), (2100, 2100, 1), (4000, 4, 100), (1300, 1300, 7),
                                                                             (5000, 0, 64), (5001, 1, 0)) for C in (40, 45) for dt in (B, F)]
         + [(210, C, B, "layer", "rms", 7, 0, 1.0) for C in (768, 1024, 1030, 4104)])
