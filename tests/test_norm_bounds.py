"""The bounds of the gated residual norm's gradients: right gradients lie inside, broken ones do not."""
import pytest
import torch

import _norm_ref as N
import _packed_ref as R


def _ids(c):
    return "-".join(str(v).replace("torch.", "") for v in c)


def _case(c):
    M, C, dtype, post, pre, samples, rs, alpha = c
    t, dy, dh = N.case(M, C, dtype, post, pre, samples, rs)
    return t, dy, dh, dict(alpha=alpha, post=post, pre=pre, rps=rs or 1)


def _zeroed(v):
    return {n: torch.zeros_like(v[n].x) for n in ("f", "x", "gate", "post_w", "post_b", "pre_w", "pre_b") if n in v}


@pytest.mark.parametrize("c", N.CASES, ids=_ids)
def test_bounds_refuse_broken_gradients(c):
    t, dy, dh, kw = _case(c)
    M, C, dtype, post, pre, samples, rs, _ = c
    want = N.gated_norm(t, dy, dh, **kw)
    for n, z in _zeroed(want).items():   # no gradient at all
        assert N.excess(z, want[n], dtype if n in "fx" else None) > 0, n

    def broken(names, *drop):
        got = N.gated_norm(t, dy, dh, **kw, drop=drop)
        for n in names:
            assert N.excess(got[n].x, want[n], dtype if n in "fx" else None) > 0, (n, drop)

    sums = [n for n in ("gate", "post_w", "post_b") if n in want]
    if pre:
        broken(["f", "x", *sums], "in pre", "projection")
        broken(["f", "x", *sums], "dy")
    if pre == "layer":
        broken(["f", "x", *sums], "in pre", "mean")
    if post:
        broken(["f"], "in post", "projection")
    if post == "layer":
        broken(["f"], "in post", "mean")
    if kw["alpha"] != 1:
        broken(["x"], "alpha")
    if rs:
        broken(["f", *sums], "row scale")
    broken(["f"], "gate")


@pytest.mark.parametrize("use", ["both", "y", "h"])
@pytest.mark.parametrize("c", [c for c in N.CASES if c[2] is torch.float32 and c[0] * c[1] < 100000], ids=_ids)
def test_values_are_the_formulas(c, use):
    """Against automatic differentiation of the formula in 64 bits, and plain fp32 torch within the bounds."""
    t, dy, dh, kw = _case(c)
    M, C, dtype, post, pre, samples, rs, alpha = c
    dy, dh = (None if use == "h" and pre else dy), (dh if use != "y" and pre else None)
    want = N.gated_norm(t, dy, dh, **kw)
    for dt in (torch.float64, torch.float32):
        p = {n: None if v is None else v.to(dt).requires_grad_(n != "rs") for n, v in t.items()}
        y, h = R.gated_norm(p["f"], p["x"], p["gate"], p["rs"], rs or 1, alpha, post, p["post_w"], p["post_b"], pre, p["pre_w"], p["pre_b"])
        wrt = [n for n, v in p.items() if v is not None and n != "rs"]
        outs = [(o, g.to(dt)) for o, g in ((y, dy), (h, dh)) if g is not None]
        grads = dict(zip(wrt, torch.autograd.grad([o for o, _ in outs], [p[n] for n in wrt], [g for _, g in outs], allow_unused=True)))
        grads.update(y=y.detach(), **({"h": h.detach()} if pre else {}))
        for n, g in grads.items():
            if g is None:
                assert n not in want
            elif dt is torch.float64:
                assert (g - want[n].x).abs().max() <= 1e-11 * (1 + want[n].x.abs().max()), n
            else:   # (torch adds in other orders: a row in chains of up to C, columns of up to M)
                assert N.excess(g, N.Val(want[n].x, want[n].e * (1 + C / 41 + M / 80)), None) <= 0, n
