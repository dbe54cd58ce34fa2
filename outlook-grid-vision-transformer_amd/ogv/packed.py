"""Operators for packed rows: sequences (images, clips) of different lengths laid end to end.

    packed_attention        softmax attention inside each sequence, shared key / value heads, causal or not
    axial_rotary            rotary positions with several axes on q and k
    rotary_attention_rows   both on the rows of one qkv projection
    gated_residual_norm     y = alpha x + s gate N_post(f), h = N_pre(y)

They stand next to ogv.functional's grid attention and LayerNorm and follow its rules: HIP device tensors
only, bf16 or fp32 activations, fp32 parameters, torch's current stream of the tensors' own device, no host
synchronisation (so every call can be captured into a graph), deterministic results, reverse-mode gradients (forward
mode is refused).  Forward and backward call the C-ABI (ogv_packed_attn_*, ogv_axial_rotary, ogv_gated_norm_*).
"""
from __future__ import annotations

import ctypes
import functools
import math

import torch
from torch.autograd import forward_ad

from . import _lib
from ._lib import OGV_BF16, OGV_F32, GatedNormDesc, PackedDesc, RotaryDesc, check
from .functional import f32

NORMS = {None: 0, "none": 0, "layer": 1, "rms": 2}

# Small calls are bound by the host, so what depends on sizes alone (the C-ABI's descriptors and workspace sizes) is
# looked up by value, the device is only switched where it differs, and calls without gradients skip autograd.
# What a caller passes as a number becomes one first: a tensor as a key would stand for its identity, not its value.


def _dtype(what, first, *ts):
    """The C-ABI's element type of tensors that must agree in it."""
    t = first.dtype
    if t is not torch.bfloat16 and t is not torch.float32:
        raise TypeError(f"{what}: float32 or bfloat16 activations, got {t}")
    for o in ts:
        if o is not None and o.dtype is not t:
            raise TypeError(f"{what}: mixed activation types {t} and {o.dtype}")
    return OGV_BF16 if t is torch.bfloat16 else OGV_F32


def _device(what, first, *ts):
    dev = first.get_device()   # (-1: not on a device)
    for t in (first, *ts):
        if t is not None:
            if t.get_device() < 0:
                raise RuntimeError(f"{what}: the MI355X kernels need HIP device tensors (got {t.device}); "
                                   f"this framework has no CPU execution path")
            if t.get_device() != dev:
                raise ValueError(f"{what}: tensors on {first.device} and {t.device}")


def _rows32(what, *rows):
    """The C-ABI counts rows in 32 bits."""
    for m in rows:
        if m >= 1 << 31:
            raise ValueError(f"{what}: too many rows ({m})")


def _grad(*ts):
    """Whether the call goes through its autograd function.  Inside a forward-mode level every call does (a dual tensor
    does not require gradients by itself, and without gradient mode either): the function refuses dual tensors."""
    if forward_ad._current_level >= 0:
        return True
    if torch.is_grad_enabled():
        for t in ts:
            if t is not None and t.requires_grad:
                return True
    return False


def _ptr(t):
    return None if t is None else t.data_ptr()


def _launch(fn, name, like, *args):
    """Call the C-ABI on the current stream of `like`'s device, with that device current."""
    dev = like.get_device()
    if dev == torch.cuda.current_device():
        check(fn(*args, torch._C._cuda_getCurrentRawStream(dev)), name)
    else:
        with torch.cuda.device(dev):
            check(fn(*args, torch._C._cuda_getCurrentRawStream(dev)), name)


def _ws(nbytes, like):
    return torch.empty(nbytes, dtype=torch.uint8, device=like.device) if nbytes else None


def _addressable(shape, stride, al, group=1):
    """Whether the kernels can address [rows, heads, D] of these strides: unit last stride, rows and heads at multiples of
    al elements (16 bytes), offsets inside a tile and inside a group of query heads within 32 bits."""
    (m, h, d), (sm, sh, sd) = shape, stride
    return not (m > 1 and (sm % al or sm >= 1 << 24) or h > 1 and (sh % al or group > 1 and sh >= (1 << 28) // group)
                or d > 1 and sd != 1)


def _heads3(t, group=1):
    """t, or a contiguous copy where the kernels cannot address it."""
    if t.data_ptr() % 16 or not _addressable(t.shape, t.stride(), 16 // t.element_size(), group):
        t = t.clone(memory_format=torch.contiguous_format)
    return t


def _row_head(shape, stride):
    """(row, head) strides; those of a size-1 dim are never used and may be anything in torch."""
    return (stride[0] if shape[0] > 1 else 0, stride[1] if shape[1] > 1 else 0)


def _strides(t):
    return _row_head(t.shape, t.stride())


# ------------------------------------------------------------------------------------------------
# Attention
# ------------------------------------------------------------------------------------------------
@functools.lru_cache(4096)
def _packed_desc(B, Mq, Mk, heads, kv_heads, D, causal, scale, dt, *strides):
    """(descriptor, forward workspace bytes, backward workspace bytes)."""
    _rows32("ogv.packed_attention", Mq, Mk, B)
    d = PackedDesc(B=B, Mq=Mq, Mk=Mk, heads=heads, kv_heads=kv_heads, D=D, causal=causal, scale=scale)
    for i, (row, head) in enumerate(strides):
        d.row[i], d.head[i] = row, head
    lib = _lib.load()
    r = ctypes.byref(d)
    return r, lib.ogv_packed_attn_fwd_ws_bytes(r, dt), lib.ogv_packed_attn_bwd_ws_bytes(r, dt)


def _attn_fwd(q, k, v, cu_q, cu_k, causal, scale, lo=None, plan=None):
    """out and lse; lo (like out) gets what the rounding took from out."""
    dt = OGV_BF16 if q.dtype is torch.bfloat16 else OGV_F32
    Mq, heads, D = q.shape
    out = q.new_empty((Mq, heads, D))
    lse = q.new_empty((Mq, heads), dtype=torch.float32)
    if Mq == 0:
        return out, lse
    B = cu_q.shape[0] - 1
    if B == 0:   # no sequence at all: every row is behind the last one
        if lo is not None:
            lo.zero_()
        return out.zero_(), lse.fill_(-math.inf)
    d, ws, _ = plan or _packed_desc(B, Mq, k.shape[0], heads, k.shape[1], D, causal, scale, dt, _strides(q), _strides(k),
                                    _strides(v), (heads * D, D))
    ws = _ws(ws, q)
    _launch(_lib.load().ogv_packed_attn_fwd, "ogv_packed_attn_fwd", q, _ptr(q), _ptr(k), _ptr(v), _ptr(cu_q), _ptr(cu_k),
            _ptr(out), _ptr(lo), _ptr(lse), _ptr(ws), d, dt)
    return out, lse


def _lo(q):
    return torch.empty(q.shape, dtype=q.dtype, device=q.device) if q.dtype is torch.bfloat16 else None


def _attn_bwd(dout, q, k, v, out, lo, lse, cu_q, cu_k, causal, scale, dq, dk, dv):
    """Writes dq, dk, dv (which may be strided)."""
    dt = _dtype("ogv.packed_attention", q, k, v, dout)
    Mq, heads, D = q.shape
    B = cu_q.shape[0] - 1
    if Mq == 0 or B == 0:
        for t in (dq, dk, dv):
            t.zero_()
        return
    d, _, ws = _packed_desc(B, Mq, k.shape[0], heads, k.shape[1], D, causal, scale, dt,
                            *(_strides(t) for t in (q, k, v, out, dout, dq, dk, dv)))
    ws = _ws(ws, q)
    _launch(_lib.load().ogv_packed_attn_bwd, "ogv_packed_attn_bwd", q, _ptr(dout), _ptr(q), _ptr(k), _ptr(v), _ptr(out),
            _ptr(lo), _ptr(lse), _ptr(cu_q), _ptr(cu_k), _ptr(dq), _ptr(dk), _ptr(dv), _ptr(ws), d, dt)


class _PackedAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, cu_q, cu_k, causal, scale):
        lo = _lo(q)
        out, lse = _attn_fwd(q, k, v, cu_q, cu_k, causal, scale, lo)
        ctx.save_for_backward(q, k, v, out, lo, lse, cu_q, cu_k)
        ctx.meta = (causal, scale)
        ctx.mark_non_differentiable(lse)
        ctx.set_materialize_grads(False)
        return out, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout, _dlse):
        if dout is None:
            return (None,) * 7
        q, k, v, out, lo, lse, cu_q, cu_k = ctx.saved_tensors
        dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
        _attn_bwd(_heads3(dout.to(q.dtype), q.shape[1] // k.shape[1]), q, k, v, out, lo, lse, cu_q, cu_k, *ctx.meta, dq, dk, dv)
        return dq, dk, dv, None, None, None, None


def _check_cu(what, cu):
    if cu.dtype is not torch.int32 or cu.ndim != 1 or cu.shape[0] < 1:
        raise ValueError(f"{what}: row offsets must be int32 [sequences + 1], got {cu.dtype} {tuple(cu.shape)}")
    return cu if cu.is_contiguous() else cu.contiguous()


def _check_attention(what, D, heads, kv_heads, scale):
    if not (heads > 0 and kv_heads > 0 and heads % kv_heads == 0):
        raise ValueError(f"{what}: heads ({heads}) must be a multiple of kv_heads ({kv_heads})")
    if not (8 <= D <= 128 and D % 8 == 0):
        raise ValueError(f"{what}: head_dim {D} unsupported (a multiple of 8 up to 128)")
    scale = D**-0.5 if scale is None else float(scale)
    if not 0.0 < scale < math.inf:
        raise ValueError(f"{what}: scale must be positive and finite, got {scale}")
    return scale


@functools.lru_cache(4096)
def _attn_plan(what, q, qs, k, ks, v, vs, nq, nk, causal, scale, dt):
    """What follows from shapes and strides: refusals; (scale, descriptor of a call without copies or None, group)."""
    if len(q) != 3 or len(k) != 3 or len(v) != 3:
        raise ValueError(f"{what}: q, k, v must be [rows, heads, head_dim]")
    if k != v:
        raise ValueError(f"{what}: k {tuple(k)} and v {tuple(v)} differ")
    if q[2] != k[2]:
        raise ValueError(f"{what}: head_dim of q ({q[2]}) and k ({k[2]}) differ")
    scale = _check_attention(what, q[2], q[1], k[1], scale)
    if nq != nk:
        raise ValueError(f"{what}: cu_q has {nq} offsets, cu_k {nk}")
    al, group, plan = 8 if dt == OGV_BF16 else 4, q[1] // k[1], None
    if q[0] and nq > 1 and _addressable(q, qs, al, group) and _addressable(k, ks, al) and _addressable(v, vs, al):
        plan = _packed_desc(nq - 1, q[0], k[0], q[1], k[1], q[2], causal, scale, dt, _row_head(q, qs), _row_head(k, ks),
                            _row_head(v, vs), (q[1] * q[2], q[2]))
    return scale, plan, group


def packed_attention(q, k, v, cu_q, cu_k=None, causal=False, scale=None, return_lse=False):
    """softmax(scale q k^T) v inside each of the packed sequences.

    q [rows, heads, D]; k, v [key rows, kv_heads, D], heads a multiple of kv_heads (query heads
    h * G .. h * G + G - 1 share key / value head h).  Row and head strides are free (the column slices of one
    projection's rows need no copy).  cu_q int32 [sequences + 1] on the device: sequence b asks with rows
    cu_q[b] .. cu_q[b+1] - 1 of q; cu_k (default: cu_q) likewise for the keys; offsets begin at 0 and do not
    decrease (they are not checked: of ones that do the results are unspecified), any length may be 0 or 1.  causal: key j is seen by query i where j <= i + keys - queries.  A row
    that sees no key, and a row behind the last sequence, is 0 (lse -inf) and has zero gradients.
    Returns out [rows, heads, D], with return_lse also the fp32 log-sum-exp [rows, heads] (no gradient).
    A non-finite value in v reaches its own sequence only, also where causal hides it; so does, in the backward, one
    in q, k, v or the gradient (a weight of 0 times it is not 0)."""
    what = "ogv.packed_attention"
    dt = _dtype(what, q, k, v)
    causal, scale = bool(causal), None if scale is None else float(scale)
    cu_q = _check_cu(what, cu_q)
    cu_k = cu_q if cu_k is None else _check_cu(what, cu_k)
    scale, plan, group = _attn_plan(what, q.shape, q.stride(), k.shape, k.stride(), v.shape, v.stride(), cu_q.shape[0],
                                    cu_k.shape[0], causal, scale, dt)
    _device(what, q, k, v, cu_q, cu_k)
    if plan is None or (q.data_ptr() | k.data_ptr() | v.data_ptr()) & 15:
        q, k, v, plan = _heads3(q, group), _heads3(k), _heads3(v), None
    if _grad(q, k, v):
        out, lse = _PackedAttention.apply(q, k, v, cu_q, cu_k, causal, scale)
    else:
        out, lse = _attn_fwd(q, k, v, cu_q, cu_k, causal, scale, plan=plan)
    return (out, lse) if return_lse else out


# ------------------------------------------------------------------------------------------------
# Rotary positions
# ------------------------------------------------------------------------------------------------
@functools.lru_cache(4096)
def _rotary_desc(M, D, sections, theta, interleaved, inverse, pos_float, *tensors):
    _rows32("ogv.axial_rotary", M)
    d = RotaryDesc(M=M, D=D, axes=len(sections), interleaved=interleaved, inverse=inverse, pos_float=pos_float, theta=theta)
    for i, n in enumerate(sections):
        d.pairs[i] = n
    for i, (heads, a, b) in enumerate(tensors):
        d.heads[i] = heads
        (d.row_in[i], d.head_in[i]), (d.row_out[i], d.head_out[i]) = a, b
    return ctypes.byref(d)


def _rotate(xs, outs, positions, meta, inverse, desc=None):
    """Turn the one or two [M, heads, D] tensors xs into outs."""
    x = xs[0]
    if x.shape[0] == 0:
        return
    if desc is None:
        desc = _rotary_desc(x.shape[0], x.shape[2], *meta, inverse, positions.dtype is torch.float32,
                            *((a.shape[1], _strides(a), _strides(b)) for a, b in zip(xs, outs)))
    k, k_out = (xs[1], outs[1]) if len(xs) > 1 else (None, None)
    _launch(_lib.load().ogv_axial_rotary, "ogv_axial_rotary", x, _ptr(x), _ptr(outs[0]), _ptr(k), _ptr(k_out), _ptr(positions),
            desc, OGV_BF16 if x.dtype is torch.bfloat16 else OGV_F32)


def _rotate_new(positions, meta, *xs, desc=None):
    outs = tuple([x.new_empty(x.shape) for x in xs])
    _rotate(xs, outs, positions, meta, False, desc)
    return outs


@functools.lru_cache(4096)
def _rotary_plan(what, q, qs, k, ks, positions, pos_float, sections, theta, interleaved, al):
    """What follows from shapes and strides: refusals; (meta, descriptor of a call without copies or None)."""
    if len(q) != 3 or k is not None and len(k) != 3:
        raise ValueError(f"{what}: q and k must be [rows, heads, head_dim]")
    if not (q[1] > 0 and (k is None or k[1] > 0)):
        raise ValueError(f"{what}: no heads")
    if k is not None and (k[0] != q[0] or k[2] != q[2]):
        raise ValueError(f"{what}: q {tuple(q)} and k {tuple(k)} differ in rows or head_dim")
    meta = _rotary_meta(what, q[2], sections, theta, interleaved)
    _positions_shape(what, positions, q[0], meta)
    xs, desc = [(q, qs)] if k is None else [(q, qs), (k, ks)], None
    if q[0] and all(_addressable(x, st, al) for x, st in xs):
        desc = _rotary_desc(q[0], q[2], *meta, False, pos_float,
                            *((x[1], _row_head(x, st), (x[1] * x[2], x[2])) for x, st in xs))
    return meta, desc


class _AxialRotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, positions, meta, *xs):
        ctx.save_for_backward(positions)
        ctx.meta = meta
        return _rotate_new(positions, meta, *xs)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, *gs):
        positions, = ctx.saved_tensors
        gs = [_heads3(g) for g in gs]
        outs = tuple(torch.empty(g.shape, dtype=g.dtype, device=g.device) for g in gs)
        _rotate(gs, outs, positions, ctx.meta, True)
        return (None, None, *outs)


@functools.lru_cache(1024)
def _rotary_meta(what, D, sections, theta, interleaved):
    if not (1 <= len(sections) <= 4 and all(n > 0 for n in sections)):
        raise ValueError(f"{what}: sections must be 1 to 4 positive pair counts, got {sections}")
    if not (D % 2 == 0 and D <= 128 and 2 * sum(sections) <= D):
        raise ValueError(f"{what}: {sum(sections)} pairs need an even head_dim of at "
                         f"least {2 * sum(sections)} (and at most 128), got {D}")
    if not 0.0 < theta < math.inf:
        raise ValueError(f"{what}: theta must be positive and finite, got {theta}")
    return sections, theta, interleaved


def _positions_shape(what, shape, rows, meta):
    if shape != (rows, len(meta[0])):
        raise ValueError(f"{what}: positions [rows, axes] = [{rows}, {len(meta[0])}] expected, got {tuple(shape)}")


def _check_positions(what, positions):
    if positions.dtype is not torch.int32 and positions.dtype is not torch.float32:
        raise TypeError(f"{what}: positions must be int32 or float32, got {positions.dtype}")
    if positions.requires_grad:
        positions = positions.detach()
    return positions if positions.is_contiguous() else positions.contiguous()


def axial_rotary(q, k, positions, sections, theta=10000.0, interleaved=False):
    """Rotary positions with several axes: (q, k) turned, q [rows, heads, D] and k [rows, kv_heads, D] (or None:
    the turned q alone).

    positions [rows, axes] int32 or float32: a token's coordinates, e.g. (height, width) or (time, height,
    width); sections: pairs of head dims per axis, their sum P at most D / 2.  The j-th of an axis' n pairs turns
    by position * theta^(-j / n); pair p is the dims (p, p + P), or (2p, 2p + 1) with interleaved; dims from 2 P
    on pass unchanged.  Angles are reduced in 64 bits.  Positions get no gradient."""
    what = "ogv.axial_rotary"
    dt = _dtype(what, q, k)
    sections = tuple([int(n) for n in sections])
    positions = _check_positions(what, positions)
    meta, desc = _rotary_plan(what, q.shape, q.stride(), None if k is None else k.shape, None if k is None else k.stride(),
                              positions.shape, positions.dtype is torch.float32, sections, float(theta), bool(interleaved),
                              8 if dt == OGV_BF16 else 4)
    _device(what, q, k, positions)
    if desc is None or (q.data_ptr() if k is None else q.data_ptr() | k.data_ptr()) & 15:
        q, k, desc = _heads3(q), None if k is None else _heads3(k), None
    xs = (q,) if k is None else (q, k)
    outs = _AxialRotary.apply(positions, meta, *xs) if _grad(q, k) else _rotate_new(positions, meta, *xs, desc=desc)
    return outs[0] if k is None else outs


class _RotaryAttentionRows(torch.autograd.Function):
    """out [rows, heads, D] = attention of the (turned) column slices of qkv; one gradient buffer, written in place."""

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
        lo = _lo(q) if ctx.needs_input_grad[0] else None
        out, lse = _attn_fwd(q, k, v, cu, cu, causal, scale, lo)
        ctx.save_for_backward(qkv, *((q, k) if rot is not None else (None, None)), out, lo, lse, cu, positions)
        ctx.meta = (rot, heads, kv_heads, causal, scale)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        qkv, q, k, out, lo, lse, cu, positions = ctx.saved_tensors
        rot, heads, kv_heads, causal, scale = ctx.meta
        q0, k0, v = _RotaryAttentionRows._split(qkv, heads, kv_heads)
        q, k = (q0, k0) if rot is None else (q, k)
        dqkv = torch.empty(qkv.shape, dtype=qkv.dtype, device=qkv.device)
        dq, dk, dv = _RotaryAttentionRows._split(dqkv, heads, kv_heads)
        _attn_bwd(_heads3(dout.to(qkv.dtype), heads // kv_heads), q, k, v, out, lo, lse, cu, cu, causal, scale, dq, dk, dv)
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
    if not (qkv.ndim == 2):
        raise ValueError(f"{what}: qkv must be [rows, columns]")
    if not (heads > 0 and kv_heads > 0 and qkv.shape[1] % (heads + 2 * kv_heads) == 0):
        raise ValueError(f"{what}: {qkv.shape[1]} columns do not split into {heads} + 2 * {kv_heads} heads")
    D = qkv.shape[1] // (heads + 2 * kv_heads)
    scale = _check_attention(what, D, heads, kv_heads, scale)
    _dtype(what, qkv)
    cu = _check_cu(what, cu)
    if not ((positions is None) == (sections is None)):
        raise ValueError(f"{what}: positions and sections belong together")
    rot = None
    if positions is not None:
        positions = _check_positions(what, positions)
        rot = _rotary_meta(what, D, tuple([int(n) for n in sections]), float(theta), bool(interleaved))
        _positions_shape(what, positions.shape, qkv.shape[0], rot)
    _device(what, qkv, cu, positions)
    al = 16 // qkv.element_size()
    if qkv.stride(1) != 1 or qkv.stride(0) % al or qkv.stride(0) >= 1 << 24 or qkv.data_ptr() % 16:
        qkv = qkv.clone(memory_format=torch.contiguous_format)
    return _RotaryAttentionRows.apply(qkv, cu, positions, rot, int(heads), kv_heads, bool(causal), scale).flatten(1)


# ------------------------------------------------------------------------------------------------
# Norms around a gated residual
# ------------------------------------------------------------------------------------------------
@functools.lru_cache(4096)
def _norm_desc(M, C, post, pre, samples, rps, alpha, post_eps, pre_eps, dt):
    """(descriptor, backward workspace bytes)."""
    _rows32("ogv.gated_residual_norm", M)
    d = ctypes.byref(GatedNormDesc(M=M, C=C, post=post, pre=pre, samples=samples, rps=rps, alpha=alpha, post_eps=post_eps,
                                   pre_eps=pre_eps))
    return d, _lib.load().ogv_gated_norm_bwd_ws_bytes(d, dt)


def _norm_fwd(f, x, gate, rs, post_w, post_b, pre_w, pre_b, meta, stats=None, desc=None):
    dt = OGV_BF16 if f.dtype is torch.bfloat16 else OGV_F32
    y = torch.empty_like(f)
    h = torch.empty_like(f) if meta[1] else None
    if f.shape[0]:
        _launch(_lib.load().ogv_gated_norm_fwd, "ogv_gated_norm_fwd", f, _ptr(f), _ptr(x), _ptr(gate), _ptr(rs), _ptr(post_w),
                _ptr(post_b), _ptr(pre_w), _ptr(pre_b), _ptr(y), _ptr(h), _ptr(stats), desc or _norm_desc(*f.shape, *meta, dt)[0], dt)
    return y if h is None else (y, h)


def _rows(g, like):
    """A gradient as contiguous rows of the activations' type."""
    if g is None:
        return None
    if g.dtype is not like.dtype:
        g = g.to(like.dtype)
    return g if g.is_contiguous() else g.contiguous()


class _GatedNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, f, x, gate, rs, post_w, post_b, pre_w, pre_b, meta):
        stats = torch.empty((f.shape[0], 4), dtype=torch.float32, device=f.device)
        out = _norm_fwd(f, x, gate, rs, post_w, post_b, pre_w, pre_b, meta, stats)
        ctx.save_for_backward(f, x, gate, rs, post_w, post_b, pre_w, pre_b, stats)
        ctx.meta = meta
        ctx.set_materialize_grads(False)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dh=None):
        f, x, gate, rs, post_w, post_b, pre_w, pre_b, stats = ctx.saved_tensors
        if dy is None and dh is None:
            return (None,) * 9
        M, C = f.shape
        dy, dh = _rows(dy, f), _rows(dh, f)
        df, dx = torch.empty_like(f), torch.empty_like(f)
        sums = torch.empty((5, C), dtype=torch.float32, device=f.device)
        dgate = torch.empty_like(gate) if gate is not None and ctx.meta[2] > 1 else None
        if M:
            dt = _dtype("ogv.gated_residual_norm", f)
            d, ws = _norm_desc(M, C, *ctx.meta, dt)
            ws = _ws(ws, f)
            _launch(_lib.load().ogv_gated_norm_bwd, "ogv_gated_norm_bwd", f, _ptr(dy), _ptr(dh), _ptr(f), _ptr(x), _ptr(gate),
                    _ptr(rs), _ptr(post_w), _ptr(post_b), _ptr(pre_w), _ptr(pre_b), _ptr(stats), _ptr(df), _ptr(dx), _ptr(sums),
                    _ptr(dgate), _ptr(ws), d, dt)
        else:
            sums.zero_()
            dgate = torch.zeros_like(gate) if dgate is not None else None
        g, w1, b1, w0, b0 = sums.unbind(0)
        if gate is not None and dgate is None:
            dgate = g if gate.ndim == 1 else g.view(gate.shape)
        return (df, dx, dgate, None, None if post_w is None else w0, None if post_b is None else b0,
                None if pre_w is None else w1, None if pre_b is None else b1, None)


def _shape(t):
    return None if t is None else t.shape


def _f32c(t):
    """A parameter as contiguous fp32."""
    if t is None:
        return None
    t = f32(t)
    return t if t.is_contiguous() else t.contiguous()


@functools.lru_cache(4096)
def _norm_plan(what, branch, residual, gate, factors, rps, post_norm, post_w, post_b, pre_norm, pre_w, pre_b, alpha, post_eps,
               pre_eps, dt):
    """What follows from shapes: refusals; (meta, descriptor)."""
    if len(branch) != 2 or branch != residual:
        raise ValueError(f"{what}: branch {tuple(branch)} and residual {tuple(residual)} must be equal [rows, channels]")
    M, C = branch
    if post_norm not in NORMS or pre_norm not in NORMS:
        raise ValueError(f"{what}: norms are 'layer', 'rms' or None, got {post_norm!r}, {pre_norm!r}")
    if not 1 <= C <= 8192:
        raise ValueError(f"{what}: {C} channels unsupported (1 to 8192)")
    post, pre = NORMS[post_norm], NORMS[pre_norm]
    if not post and not (post_w is None and post_b is None):
        raise ValueError(f"{what}: weights for an absent post_norm")
    if not pre and not (pre_w is None and pre_b is None):
        raise ValueError(f"{what}: weights for an absent pre_norm")
    for name, p in (("post_weight", post_w), ("post_bias", post_b), ("pre_weight", pre_w), ("pre_bias", pre_b)):
        if p is not None and p != (C,):
            raise ValueError(f"{what}: {name} must be [{C}]")
    samples = 1
    if gate is not None:
        if len(gate) not in (1, 2) or gate[-1] != C:
            raise ValueError(f"{what}: gate must be [{C}] or [samples, {C}], got {tuple(gate)}")
        if len(gate) == 2:
            samples = gate[0]
            if samples < 1 or M % samples:
                raise ValueError(f"{what}: {M} rows do not divide into {samples} samples")
    if rps < 1:
        raise ValueError(f"{what}: rps must be >= 1")
    if factors is not None and factors * rps < M:
        raise ValueError(f"{what}: row_scale has {factors} factors of {rps} rows for {M} rows")
    meta = (post, pre, samples, max(1, min(rps, M)), alpha, post_eps, pre_eps)
    return meta, _norm_desc(M, C, *meta, dt)[0] if M else None


def gated_residual_norm(branch, residual, gate=None, row_scale=None, rps=1, alpha=1.0, post_norm=None, post_weight=None,
                        post_bias=None, pre_norm="layer", pre_weight=None, pre_bias=None, post_eps=1e-5, pre_eps=1e-5):
    """The end of a residual half-block and the norm that begins the next one:

        y = alpha * residual + row_scale * gate * N_post(branch)        h = N_pre(y)

    branch, residual [rows, C] (bf16 or fp32).  post_norm / pre_norm: "layer", "rms" or None, with fp32 weights
    and biases [C] (None: 1 and 0).  gate fp32 [C] (a gate per channel) or [samples, C] with rows / samples rows
    each.  row_scale fp32, one factor per rps rows (DropPath's; it gets no gradient).
    Returns (y, h), or y alone without a pre_norm.  h comes from y before its rounding.  C <= 8192."""
    what = "ogv.gated_residual_norm"
    dt = _dtype(what, branch, residual)
    meta, desc = _norm_plan(what, branch.shape, residual.shape, None if gate is None else gate.shape,
                            None if row_scale is None else row_scale.numel(), int(rps), post_norm, _shape(post_weight),
                            _shape(post_bias), pre_norm, _shape(pre_weight), _shape(pre_bias), float(alpha), float(post_eps),
                            float(pre_eps), dt)
    if row_scale is not None:
        row_scale = _f32c(row_scale.detach().reshape(-1))
    gate = _f32c(gate)
    params = _f32c(post_weight), _f32c(post_bias), _f32c(pre_weight), _f32c(pre_bias)
    _device(what, branch, residual, gate, row_scale, *params)
    if not branch.is_contiguous():
        branch = branch.contiguous()
    if not residual.is_contiguous():
        residual = residual.contiguous()
    if _grad(branch, residual, gate, *params):
        return _GatedNorm.apply(branch, residual, gate, row_scale, *params, meta)
    return _norm_fwd(branch, residual, gate, row_scale, *params, meta, desc=desc)
