"""Plain 64-bit forms of the packed-sequence operators on the CPU, with bounds on what the kernels may be off by.

u(t) = torch.finfo(t).eps / 2 is the relative error of one rounding to t.  The bounds below add up, term by term,
the roundings that a kernel makes: its output's (u), those of bf16 probabilities on their way into the second
product (u), and fp32 arithmetic (2^-24 per operation, counted)."""
import math

import torch

U32 = 2.0**-24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def offsets(lengths):
    return torch.tensor([0] + list(lengths)).cumsum(0).to(torch.int32)


def attention(q, k, v, lq, lk, causal, scale, dtype, dout=None):
    """fp64 out, lse (and dq, dk, dv) with their tolerances; rows behind the last sequence 0 / -inf."""
    q, k, v = (x.detach().cpu().double() for x in (q, k, v))
    dout = None if dout is None else dout.detach().cpu().double()
    h, hkv, D = q.shape[1], k.shape[1], q.shape[2]
    g = h // hkv
    u = half_step(dtype)
    up = u if dtype == torch.bfloat16 else 0.0   # P and dS are rounded for their products in bf16 only
    out, lse = torch.zeros_like(q), torch.full(q.shape[:2], -math.inf, dtype=torch.float64)
    tol, tol_lse = torch.zeros_like(q), torch.zeros_like(lse)
    grads = {n: torch.zeros_like(x) for n, x in (("dq", q), ("dk", k), ("dv", v))}
    gtol = {n: torch.zeros_like(x) for n, x in grads.items()}
    a0 = b0 = 0
    for a, b in zip(lq, lk):
        qs, ks, vs = q[a0:a0 + a], k[b0:b0 + b], v[b0:b0 + b]
        seen = torch.ones(a, b, dtype=torch.bool)
        if causal:
            seen = torch.arange(b)[None] <= torch.arange(a)[:, None] + (b - a)
        for i in range(h if a and b else 0):
            j = i // g
            s = (qs[:, i] @ ks[:, j].T * scale).masked_fill(~seen, -math.inf)
            some = seen.any(1)
            L = torch.logsumexp(s, 1)
            p = torch.where(seen, torch.exp(s - torch.where(some, L, 0.0)[:, None]), 0.0)
            # a score's error: D + 4 operations on terms adding up to mag; exp, sums and the second product: b + 16
            mag = (qs[:, i].abs() @ ks[:, j].abs().T * scale).where(seen, torch.zeros(())).amax(1)
            e32 = U32 * (2 * (D + 4) * (mag + 1) + 2 * b + 16)
            o = p @ vs[:, j]
            oa = p @ vs[:, j].abs()
            out[a0:a0 + a, i] = o
            lse[a0:a0 + a, i] = L
            tol[a0:a0 + a, i] = (up * (1 + u) + e32[:, None]) * oa + u * o.abs() * (1 + up)
            tol_lse[a0:a0 + a, i] = e32 + 4 * U32 * L.abs().where(some, torch.zeros(()))
            if dout is None:
                continue
            do = dout[a0:a0 + a, i]
            dp = do @ vs[:, j].T
            delta, delta_abs = (do * o).sum(1, keepdim=True), (do * o).abs().sum(1, keepdim=True)
            ds = p * (dp - delta)
            # dS: its rounding, the forward output's error inside delta, and fp32 work on |dp| + |delta|
            ds_err = (up * ds.abs() + p * (do.abs() * tol[a0:a0 + a, i]).sum(1, keepdim=True)
                      + e32[:, None] * p * (do.abs() @ vs[:, j].abs().T + delta_abs))
            grads["dq"][a0:a0 + a, i] = ds @ ks[:, j] * scale
            grads["dk"][b0:b0 + b, j] += ds.T @ qs[:, i] * scale
            grads["dv"][b0:b0 + b, j] += p.T @ do
            sums = U32 * (a * g + b + 8)
            gtol["dq"][a0:a0 + a, i] = (ds_err + sums * ds.abs()) @ ks[:, j].abs() * scale
            gtol["dk"][b0:b0 + b, j] += (ds_err + sums * ds.abs()).T @ qs[:, i].abs() * scale
            gtol["dv"][b0:b0 + b, j] += (p * (up + e32[:, None] + sums)).T @ do.abs()
        a0, b0 = a0 + a, b0 + b
    for n in grads:
        gtol[n] += u * (grads[n].abs() + gtol[n])
    res = {"out": (out, tol), "lse": (lse, tol_lse)}
    if dout is not None:
        res.update({n: (grads[n], gtol[n]) for n in grads})
    return res


def rotary(x, positions, sections, theta, interleaved, inverse=False):
    """fp64 turned x and its tolerance."""
    dtype = x.dtype
    x, P = x.detach().cpu().double(), sum(sections)
    pos = positions.detach().cpu().double()
    angle = torch.cat([pos[:, i:i + 1] * torch.tensor([theta ** (-j / n) for j in range(n)], dtype=torch.float64)
                       for i, n in enumerate(sections)], 1)[:, None] * (-1 if inverse else 1)
    c, s = angle.cos(), angle.sin()
    y, m = x.clone(), torch.zeros_like(x)
    one, two = (slice(0, 2 * P, 2), slice(1, 2 * P, 2)) if interleaved else (slice(0, P), slice(P, 2 * P))
    a, b = x[..., one], x[..., two]
    y[..., one], y[..., two] = a * c - b * s, b * c + a * s
    m[..., one] = m[..., two] = a.abs() + b.abs()
    # turn to float: 2 pi 2^-26; sine and cosine 2 steps of 2^-24; three operations: under 8 * 2^-24 of |a| + |b|;
    # fp64 angles: position * 2^-52 turns
    far = 2.0**-50 * pos.abs().amax(1)[:, None, None]
    tol = (8 * U32 + far) * m + half_step(dtype) * y.abs() * (1 + 1e-6)
    return y, tol


def gated_norm(f, x, gate, rs, rps, alpha, post, post_w, post_b, pre, pre_w, pre_b, eps=1e-5):
    """fp64 (y, h) of tensors that may require gradients (autograd gives the formula's gradients)."""
    def norm(v, kind, w, b):
        d = v - v.mean(1, keepdim=True) if kind == "layer" else v
        d = d / (d.square().mean(1, keepdim=True) + eps).sqrt()
        d = d if w is None else d * w
        return d if b is None else d + b

    M = f.shape[0]
    n = f if post is None else norm(f, post, post_w, post_b)
    if gate is not None:
        n = n * (gate.repeat_interleave(M // gate.shape[0], 0) if gate.ndim == 2 else gate)
    if rs is not None:
        n = n * rs.repeat_interleave(rps)[:M, None]
    y = alpha * x + n
    return y, (None if pre is None else norm(y, pre, pre_w, pre_b))
