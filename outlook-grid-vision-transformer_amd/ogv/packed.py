"""Operators for packed rows: sequences (images, clips) of different lengths laid end to end.

    packed_attention        softmax attention inside each sequence, shared key / value heads, causal or not
    axial_rotary            rotary positions with several axes on q and k
    rotary_attention_rows   both on the rows of one qkv projection
    gated_residual_norm     y = alpha x + s gate N_post(f), h = N_pre(y)

They stand next to ogv.functional's grid attention and LayerNorm and follow its rules: HIP device tensors
only, bf16 or fp32 activations, fp32 parameters, torch's current stream of the tensors' own device, no host
synchronisation (so every call can be captured into a graph), deterministic results.  Forward and backward
call the C-ABI (ogv_packed_attn_*, ogv_axial_rotary, ogv_gated_norm_*).
"""
from __future__ import annotations

import ctypes
import math

import torch

from . import _lib
from ._lib import OGV_BF16, OGV_F32, GatedNormDesc, PackedDesc, RotaryDesc, check
from .functional import _ptr, _vp, f32

NORMS = {None: 0, "none": 0, "layer": 1, "rms": 2}


def _need(ok, what, exc=ValueError):
    if not ok:
        raise exc(what)


def _dtype(what, *ts):
    """The C-ABI's element type of tensors that must agree in it."""
    t = ts[0].dtype
    _need(t in (torch.bfloat16, torch.float32), f"{what}: float32 or bfloat16 activations, got {t}", TypeError)
    for o in ts[1:]:
        _need(o is None or o.dtype == t, f"{what}: mixed activation types {t} and {None if o is None else o.dtype}", TypeError)
    return OGV_BF16 if t == torch.bfloat16 else OGV_F32


def _device(what, first, *ts):
    for t in (first, *ts):
        if t is not None and not t.is_cuda:
            raise RuntimeError(f"{what}: the MI355X kernels need HIP device tensors (got {t.device}); "
                               f"this framework has no CPU execution path")
        _need(t is None or t.device == first.device, f"{what}: tensors on {first.device} and {t.device if t is not None else None}")


class _on:
    """The tensors' device made current; yields its current stream's handle."""

    def __init__(self, t):
        self.guard = torch.cuda.device(t.device)
        self.device = t.device

    def __enter__(self):
        self.guard.__enter__()
        return _vp(torch.cuda.current_stream(self.device).cuda_stream)

    def __exit__(self, *exc):
        return self.guard.__exit__(*exc)


def _ws(nbytes, like):
    return torch.empty(int(nbytes), dtype=torch.uint8, device=like.device) if nbytes else None


def _heads3(t):
    """A [rows, heads, D] tensor the kernels can address (unit last stride, 16-byte rows, heads and base), else a copy."""
    al = 16 // t.element_size()
    if (t.shape[0] > 1 and t.stride(0) % al or t.shape[1] > 1 and t.stride(1) % al or t.stride(2) != 1 and t.shape[2] > 1
            or t.data_ptr() % 16):
        t = t.clone(memory_format=torch.contiguous_format)
    return t


def _strides(t):
    """(row, head) strides; those of a size-1 dim are never used and may be anything in torch."""
    return (t.stride(0) if t.shape[0] > 1 else 0, t.stride(1) if t.shape[1] > 1 else 0)


# ------------------------------------------------------------------------------------------------
# Attention
# ------------------------------------------------------------------------------------------------
def _packed_desc(B, q, k, v, causal, scale, **more):
    d = PackedDesc(B=B, Mq=q.shape[0], Mk=k.shape[0], heads=q.shape[1], kv_heads=k.shape[1], D=q.shape[2],
                   causal=int(causal), scale=scale)
    for i, t in enumerate((q, k, v, more.get("out"), more.get("dout"), more.get("dq"), more.get("dk"), more.get("dv"))):
        if t is not None:
            d.row[i], d.head[i] = _strides(t)
    return d


def _attn_fwd(q, k, v, cu_q, cu_k, causal, scale):
    lib = _lib.load()
    dt = _dtype("ogv.packed_attention", q, k, v)
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device)
    if q.shape[0] == 0:
        return out, lse
    if cu_q.numel() == 1:   # no sequence at all: every row is behind the last one
        return out.zero_(), lse.fill_(-math.inf)
    d = _packed_desc(cu_q.numel() - 1, q, k, v, causal, scale, out=out)
    with _on(q) as stream:
        ws = _ws(lib.ogv_packed_attn_fwd_ws_bytes(ctypes.byref(d), dt), q)
        check(lib.ogv_packed_attn_fwd(_ptr(q), _ptr(k), _ptr(v), _ptr(cu_q), _ptr(cu_k), _ptr(out), _ptr(lse), _ptr(ws),
                                      ctypes.byref(d), dt, stream), "ogv_packed_attn_fwd")
    return out, lse


def _attn_bwd(dout, q, k, v, out, lse, cu_q, cu_k, causal, scale, dq, dk, dv):
    """Writes dq, dk, dv (which may be strided)."""
    lib = _lib.load()
    dt = _dtype("ogv.packed_attention", q, k, v, dout)
    if q.shape[0] == 0 or cu_q.numel() == 1:
        for t in (dq, dk, dv):
            t.zero_()
        return
    d = _packed_desc(cu_q.numel() - 1, q, k, v, causal, scale, out=out, dout=dout, dq=dq, dk=dk, dv=dv)
    with _on(q) as stream:
        ws = _ws(lib.ogv_packed_attn_bwd_ws_bytes(ctypes.byref(d), dt), q)
        check(lib.ogv_packed_attn_bwd(_ptr(dout), _ptr(q), _ptr(k), _ptr(v), _ptr(out), _ptr(lse), _ptr(cu_q), _ptr(cu_k),
                                      _ptr(dq), _ptr(dk), _ptr(dv), _ptr(ws), ctypes.byref(d), dt, stream),
              "ogv_packed_attn_bwd")


class _PackedAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, cu_q, cu_k, causal, scale):
        out, lse = _attn_fwd(q, k, v, cu_q, cu_k, causal, scale)
        ctx.save_for_backward(q, k, v, out, lse, cu_q, cu_k)
        ctx.meta = (causal, scale)
        ctx.mark_non_differentiable(lse)
        return out, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, _dlse):
        q, k, v, out, lse, cu_q, cu_k = ctx.saved_tensors
        dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
        _attn_bwd(_heads3(dout.to(q.dtype)), q, k, v, out, lse, cu_q, cu_k, *ctx.meta, dq, dk, dv)
        return dq, dk, dv, None, None, None, None


def _check_cu(what, cu, like):
    _need(cu.dtype == torch.int32 and cu.ndim == 1 and cu.numel() >= 1, f"{what}: int32 [sequences + 1] expected, got "
          f"{cu.dtype} {tuple(cu.shape)}")
    return cu.contiguous()


def _check_attention(what, D, heads, kv_heads, scale):
    _need(heads > 0 and kv_heads > 0 and heads % kv_heads == 0, f"{what}: heads ({heads}) must be a multiple of kv_heads ({kv_heads})")
    _need(8 <= D <= 128 and D % 8 == 0, f"{what}: head_dim {D} unsupported (a multiple of 8 up to 128)")
    scale = D**-0.5 if scale is None else float(scale)
    _need(0.0 < scale < math.inf, f"{what}: scale must be positive and finite, got {scale}")
    return scale


def packed_attention(q, k, v, cu_q, cu_k=None, causal=False, scale=None, return_lse=False):
    """softmax(scale q k^T) v inside each of the packed sequences.

    q [rows, heads, D]; k, v [key rows, kv_heads, D], heads a multiple of kv_heads (query heads
    h * G .. h * G + G - 1 share key / value head h).  Row and head strides are free (the column slices of one
    projection's rows need no copy).  cu_q int32 [sequences + 1] on the device: sequence b asks with rows
    cu_q[b] .. cu_q[b+1] - 1 of q; cu_k (default: cu_q) likewise for the keys; offsets begin at 0 and do not
    decrease, any length may be 0 or 1.  causal: key j is seen by query i where j <= i + keys - queries.  A row
    that sees no key, and a row behind the last sequence, is 0 (lse -inf) and has zero gradients.
    Returns out [rows, heads, D], with return_lse also the fp32 log-sum-exp [rows, heads] (no gradient).
    A non-finite value in v reaches its own sequence only, also where causal hides it."""
    what = "ogv.packed_attention"
    _need(q.ndim == 3 and k.ndim == 3 and v.ndim == 3, f"{what}: q, k, v must be [rows, heads, head_dim]")
    cu_k = cu_q if cu_k is None else cu_k
    _need(k.shape == v.shape, f"{what}: k {tuple(k.shape)} and v {tuple(v.shape)} differ")
    _need(q.shape[2] == k.shape[2], f"{what}: head_dim of q ({q.shape[2]}) and k ({k.shape[2]}) differ")
    scale = _check_attention(what, q.shape[2], q.shape[1], k.shape[1], scale)
    _dtype(what, q, k, v)
    cu_q, cu_k = _check_cu(f"{what}: cu_q", cu_q, q), _check_cu(f"{what}: cu_k", cu_k, q)
    _need(cu_q.numel() == cu_k.numel(), f"{what}: cu_q has {cu_q.numel()} offsets, cu_k {cu_k.numel()}")
    _device(what, q, k, v, cu_q, cu_k)
    out, lse = _PackedAttention.apply(_heads3(q), _heads3(k), _heads3(v), cu_q, cu_k, bool(causal), scale)
    return (out, lse) if return_lse else out


# ------------------------------------------------------------------------------------------------
# Rotary positions
# ------------------------------------------------------------------------------------------------
def _rotate(xs, outs, positions, meta, inverse):
    """Turn the one or two [M, heads, D] tensors xs into outs."""
    sections, theta, interleaved = meta
    x = xs[0]
    if x.shape[0] == 0:
        return
    lib = _lib.load()
    d = RotaryDesc(M=x.shape[0], D=x.shape[2], axes=len(sections), interleaved=int(interleaved), inverse=int(inverse),
                   pos_float=int(positions.dtype == torch.float32), theta=theta)
    for i, n in enumerate(sections):
        d.pairs[i] = n
    for i, (a, b) in enumerate(zip(xs, outs)):
        d.heads[i] = a.shape[1]
        d.row_in[i], d.head_in[i] = _strides(a)
        d.row_out[i], d.head_out[i] = _strides(b)
    k, k_out = (xs[1], outs[1]) if len(xs) > 1 else (None, None)
    with _on(x) as stream:
        check(lib.ogv_axial_rotary(_ptr(x), _ptr(outs[0]), _ptr(k), _ptr(k_out), _ptr(positions), ctypes.byref(d),
                                   _dtype("ogv.axial_rotary", *xs), stream), "ogv_axial_rotary")


class _AxialRotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, positions, meta, *xs):
        outs = tuple(torch.empty(x.shape, dtype=x.dtype, device=x.device) for x in xs)
        _rotate(xs, outs, positions, meta, False)
        ctx.save_for_backward(positions)
        ctx.meta = meta
        return outs

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, *gs):
        positions, = ctx.saved_tensors
        gs = [_heads3(g) for g in gs]
        outs = tuple(torch.empty(g.shape, dtype=g.dtype, device=g.device) for g in gs)
        _rotate(gs, outs, positions, ctx.meta, True)
        return (None, None, *outs)


def _check_rotary(what, D, positions, sections, theta, interleaved, rows):
    sections = tuple(int(n) for n in sections)
    _need(1 <= len(sections) <= 4 and all(n > 0 for n in sections), f"{what}: sections must be 1 to 4 positive pair counts, got {sections}")
    _need(D % 2 == 0 and D <= 128 and 2 * sum(sections) <= D, f"{what}: {sum(sections)} pairs need an even head_dim of at "
          f"least {2 * sum(sections)} (and at most 128), got {D}")
    _need(positions.dtype in (torch.int32, torch.float32), f"{what}: positions must be int32 or float32, got {positions.dtype}", TypeError)
    _need(positions.shape == (rows, len(sections)), f"{what}: positions [rows, axes] = [{rows}, {len(sections)}] expected, got {tuple(positions.shape)}")
    theta = float(theta)
    _need(0.0 < theta < math.inf, f"{what}: theta must be positive and finite, got {theta}")
    return positions.detach().contiguous(), (sections, theta, bool(interleaved))


def axial_rotary(q, k, positions, sections, theta=10000.0, interleaved=False):
    """Rotary positions with several axes: (q, k) turned, q [rows, heads, D] and k [rows, kv_heads, D] (or None:
    the turned q alone).

    positions [rows, axes] int32 or float32: a token's coordinates, e.g. (height, width) or (time, height,
    width); sections: pairs of head dims per axis, their sum P at most D / 2.  The j-th of an axis' n pairs turns
    by position * theta^(-j / n); pair p is the dims (p, p + P), or (2p, 2p + 1) with interleaved; dims from 2 P
    on pass unchanged.  Angles are reduced in 64 bits.  Positions get no gradient."""
    what = "ogv.axial_rotary"
    _need(q.ndim == 3 and (k is None or k.ndim == 3), f"{what}: q and k must be [rows, heads, head_dim]")
    _need(q.shape[1] > 0 and (k is None or k.shape[1] > 0), f"{what}: no heads")
    _need(k is None or (k.shape[0] == q.shape[0] and k.shape[2] == q.shape[2]),
          f"{what}: q {tuple(q.shape)} and k {None if k is None else tuple(k.shape)} differ in rows or head_dim")
    xs = (q,) if k is None else (q, k)
    _dtype(what, *xs)
    positions, meta = _check_rotary(what, q.shape[2], positions, sections, theta, interleaved, q.shape[0])
    _device(what, q, k, positions)
    outs = _AxialRotary.apply(positions, meta, *(_heads3(x) for x in xs))
    return outs[0] if k is None else outs


class _RotaryAttentionRows(torch.autograd.Function):
    """out = attention of the (turned) column slices of qkv; one gradient buffer, written in place."""

    @staticmethod
    def _split(rows, heads, kv_heads):
        D = rows.shape[1] // (heads + 2 * kv_heads)
        return [x.unflatten(1, (-1, D)) for x in rows.split((heads * D, kv_heads * D, kv_heads * D), 1)]

    @staticmethod
    def forward(ctx, qkv, cu, positions, rot, heads, kv_heads, causal, scale):
        q, k, v = _RotaryAttentionRows._split(qkv, heads, kv_heads)
        if rot is not None:
            turned = torch.empty(q.shape, dtype=q.dtype, device=q.device), torch.empty(k.shape, dtype=k.dtype, device=k.device)
            _rotate((q, k), turned, positions, rot, False)
            q, k = turned
        out, lse = _attn_fwd(q, k, v, cu, cu, causal, scale)
        ctx.save_for_backward(qkv, *((q, k) if rot is not None else (None, None)), out, lse, cu, positions)
        ctx.meta = (rot, heads, kv_heads, causal, scale)
        return out.flatten(1)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        qkv, q, k, out, lse, cu, positions = ctx.saved_tensors
        rot, heads, kv_heads, causal, scale = ctx.meta
        q0, k0, v = _RotaryAttentionRows._split(qkv, heads, kv_heads)
        q, k = (q0, k0) if rot is None else (q, k)
        dqkv = torch.empty(qkv.shape, dtype=qkv.dtype, device=qkv.device)
        dq, dk, dv = _RotaryAttentionRows._split(dqkv, heads, kv_heads)
        _attn_bwd(_heads3(dout.to(qkv.dtype).unflatten(1, (heads, -1))), q, k, v, out, lse, cu, cu, causal, scale, dq, dk, dv)
        if rot is not None:
            _rotate((dq, dk), (dq, dk), positions, rot, True)
        return dqkv, None, None, None, None, None, None, None


def rotary_attention_rows(qkv, cu, heads, kv_heads=None, positions=None, sections=None, theta=10000.0,
                          interleaved=False, causal=False, scale=None):
    """Self-attention of packed sequences on the rows of one projection: qkv [rows, (heads + 2 kv_heads) * D] laid
    out q | k | v, turned by axial_rotary where positions are given -> [rows, heads * D].  The same results as
    packed_attention(*axial_rotary(q, k, ...), v, cu), with one gradient buffer for all three."""
    what = "ogv.rotary_attention_rows"
    kv_heads = heads if kv_heads is None else int(kv_heads)
    _need(qkv.ndim == 2, f"{what}: qkv must be [rows, columns]")
    _need(heads > 0 and kv_heads > 0 and qkv.shape[1] % (heads + 2 * kv_heads) == 0,
          f"{what}: {qkv.shape[1]} columns do not split into {heads} + 2 * {kv_heads} heads")
    D = qkv.shape[1] // (heads + 2 * kv_heads)
    scale = _check_attention(what, D, heads, kv_heads, scale)
    _dtype(what, qkv)
    cu = _check_cu(f"{what}: cu", cu, qkv)
    _need((positions is None) == (sections is None), f"{what}: positions and sections belong together")
    rot = None
    if positions is not None:
        positions, rot = _check_rotary(what, D, positions, sections, theta, interleaved, qkv.shape[0])
    _device(what, qkv, cu, positions)
    al = 16 // qkv.element_size()
    if qkv.stride(1) != 1 or qkv.stride(0) % al or qkv.data_ptr() % 16:
        qkv = qkv.clone(memory_format=torch.contiguous_format)
    return _RotaryAttentionRows.apply(qkv, cu, positions, rot, int(heads), kv_heads, bool(causal), scale)


# ------------------------------------------------------------------------------------------------
# Norms around a gated residual
# ------------------------------------------------------------------------------------------------
class _GatedNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, f, x, gate, rs, post_w, post_b, pre_w, pre_b, meta):
        lib = _lib.load()
        dt = _dtype("ogv.gated_residual_norm", f, x)
        M, C = f.shape
        post, pre, samples, rps, alpha, post_eps, pre_eps = meta
        d = GatedNormDesc(M=M, C=C, post=post, pre=pre, samples=samples, rps=rps, alpha=alpha, post_eps=post_eps,
                          pre_eps=pre_eps)
        y = torch.empty_like(f)
        h = torch.empty_like(f) if pre else None
        stats = torch.empty((M, 4), dtype=torch.float32, device=f.device) if any(ctx.needs_input_grad) else None
        if M:
            with _on(f) as stream:
                check(lib.ogv_gated_norm_fwd(_ptr(f), _ptr(x), _ptr(gate), _ptr(rs), _ptr(post_w), _ptr(post_b),
                                             _ptr(pre_w), _ptr(pre_b), _ptr(y), _ptr(h), _ptr(stats), ctypes.byref(d), dt,
                                             stream), "ogv_gated_norm_fwd")
        ctx.save_for_backward(f, x, gate, rs, post_w, post_b, pre_w, pre_b, stats)
        ctx.meta = d
        ctx.set_materialize_grads(False)
        return (y, h) if pre else y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dh=None):
        f, x, gate, rs, post_w, post_b, pre_w, pre_b, stats = ctx.saved_tensors
        if dy is None and dh is None:
            return (None,) * 9
        d, lib = ctx.meta, _lib.load()
        M, C = f.shape
        dy, dh = (None if g is None else g.to(f.dtype).contiguous() for g in (dy, dh))
        df, dx = torch.empty_like(f), torch.empty_like(f)
        sums = torch.empty((5, C), dtype=torch.float32, device=f.device)
        dgate = torch.empty_like(gate) if d.samples > 1 and gate is not None else None
        if M:
            with _on(f) as stream:
                dt = _dtype("ogv.gated_residual_norm", f)
                ws = _ws(lib.ogv_gated_norm_bwd_ws_bytes(ctypes.byref(d), dt), f)
                check(lib.ogv_gated_norm_bwd(_ptr(dy), _ptr(dh), _ptr(f), _ptr(x), _ptr(gate), _ptr(rs), _ptr(post_w),
                                             _ptr(post_b), _ptr(pre_w), _ptr(pre_b), _ptr(stats), _ptr(df), _ptr(dx),
                                             _ptr(sums), _ptr(dgate), _ptr(ws), ctypes.byref(d), dt, stream),
                      "ogv_gated_norm_bwd")
        else:
            sums.zero_()
            dgate = torch.zeros_like(gate) if dgate is not None else None
        if gate is not None and dgate is None:
            dgate = sums[0].view(gate.shape)
        pick = lambda p, i: None if p is None else sums[i]  # noqa: E731
        return (df, dx, dgate, None, pick(post_w, 3), pick(post_b, 4), pick(pre_w, 1), pick(pre_b, 2), None)


def gated_residual_norm(branch, residual, gate=None, row_scale=None, rps=1, alpha=1.0, post_norm=None, post_weight=None,
                        post_bias=None, pre_norm="layer", pre_weight=None, pre_bias=None, post_eps=1e-5, pre_eps=1e-5):
    """The end of a residual half-block and the norm that begins the next one:

        y = alpha * residual + row_scale * gate * N_post(branch)        h = N_pre(y)

    branch, residual [rows, C] (bf16 or fp32).  post_norm / pre_norm: "layer", "rms" or None, with fp32 weights
    and biases [C] (None: 1 and 0).  gate fp32 [C] (a gate per channel) or [samples, C] with rows / samples rows
    each.  row_scale fp32, one factor per rps rows (DropPath's; it gets no gradient).
    Returns (y, h), or y alone without a pre_norm.  h comes from y before its rounding.  C <= 8192."""
    what = "ogv.gated_residual_norm"
    _need(branch.ndim == 2 and branch.shape == residual.shape, f"{what}: branch {tuple(branch.shape)} and residual "
          f"{tuple(residual.shape)} must be equal [rows, channels]")
    M, C = branch.shape
    _need(post_norm in NORMS and pre_norm in NORMS, f"{what}: norms are 'layer', 'rms' or None, got {post_norm!r}, {pre_norm!r}")
    _need(1 <= C <= 8192, f"{what}: {C} channels unsupported (1 to 8192)")
    _dtype(what, branch, residual)
    post, pre = NORMS[post_norm], NORMS[pre_norm]
    _need(post or (post_weight is None and post_bias is None), f"{what}: weights for an absent post_norm")
    _need(pre or (pre_weight is None and pre_bias is None), f"{what}: weights for an absent pre_norm")
    params = []
    for name, p in (("post_weight", post_weight), ("post_bias", post_bias), ("pre_weight", pre_weight), ("pre_bias", pre_bias)):
        _need(p is None or p.shape == (C,), f"{what}: {name} must be [{C}]")
        params.append(None if p is None else f32(p).contiguous())
    samples = 1
    if gate is not None:
        _need(gate.ndim in (1, 2) and gate.shape[-1] == C, f"{what}: gate must be [{C}] or [samples, {C}], got {tuple(gate.shape)}")
        if gate.ndim == 2:
            samples = gate.shape[0]
            _need(samples >= 1 and M % samples == 0, f"{what}: {M} rows do not divide into {samples} samples")
        gate = f32(gate).contiguous()
    rps = int(rps)
    _need(rps >= 1, f"{what}: rps must be >= 1")
    if row_scale is not None:
        _need(row_scale.numel() * rps >= M, f"{what}: row_scale has {row_scale.numel()} factors of {rps} rows for {M} rows")
        row_scale = row_scale.detach().float().reshape(-1).contiguous()
    _device(what, branch, residual, gate, row_scale, *params)
    meta = (post, pre, samples, rps, float(alpha), float(post_eps), float(pre_eps))
    return _GatedNorm.apply(branch.contiguous(), residual.contiguous(), gate, row_scale, *params, meta)
