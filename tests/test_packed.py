"""Packed-sequence operators, CPU side: what they refuse, before anything reaches a device."""
import ctypes

import pytest
import torch


def _attn(**more):
    a = dict(q=torch.zeros(6, 4, 16), k=torch.zeros(6, 2, 16), v=torch.zeros(6, 2, 16),
             cu_q=torch.tensor([0, 2, 6], dtype=torch.int32))
    a.update(more)
    return a


@pytest.mark.parametrize("more,match", [
    (dict(q=torch.zeros(6, 64)), "rows, heads"),
    (dict(v=torch.zeros(6, 2, 8)), "differ"),
    (dict(k=torch.zeros(6, 2, 8), v=torch.zeros(6, 2, 8)), "head_dim"),
    (dict(k=torch.zeros(6, 3, 16), v=torch.zeros(6, 3, 16)), "multiple of kv_heads"),
    (dict(q=torch.zeros(6, 4, 12), k=torch.zeros(6, 2, 12), v=torch.zeros(6, 2, 12)), "head_dim 12"),
    (dict(q=torch.zeros(6, 4, 136), k=torch.zeros(6, 2, 136), v=torch.zeros(6, 2, 136)), "head_dim 136"),
    (dict(scale=0.0), "scale"),
    (dict(scale=float("inf")), "scale"),
    (dict(cu_q=torch.tensor([0, 2, 6])), "int32"),
    (dict(cu_q=torch.zeros(2, 2, dtype=torch.int32)), "int32"),
    (dict(cu_k=torch.tensor([0, 6], dtype=torch.int32)), "offsets"),
])
def test_attention_refusals(more, match):
    from ogv.packed import packed_attention
    with pytest.raises(ValueError, match=match):
        packed_attention(**_attn(**more))


def test_attention_types_and_device():
    from ogv.packed import packed_attention
    with pytest.raises(TypeError, match="float32 or bfloat16"):
        packed_attention(**{n: t.half() if t.is_floating_point() else t for n, t in _attn().items()})
    with pytest.raises(TypeError, match="mixed"):
        packed_attention(**_attn(v=torch.zeros(6, 2, 16).bfloat16()))
    with pytest.raises(RuntimeError, match="HIP device"):
        packed_attention(**_attn())


@pytest.mark.parametrize("more,match", [
    (dict(q=torch.zeros(5, 16)), "rows, heads"),
    (dict(k=torch.zeros(4, 2, 16)), "differ"),
    (dict(sections=()), "sections"),
    (dict(sections=(4, 0)), "sections"),
    (dict(sections=(4, 5)), "pairs"),
    (dict(sections=(4, 4, 1, 1, 1)), "sections"),
    (dict(positions=torch.zeros(5, 1, dtype=torch.int32)), "positions"),
    (dict(positions=torch.zeros(4, 2, dtype=torch.int32)), "positions"),
    (dict(theta=0.0), "theta"),
    (dict(theta=float("nan")), "theta"),
])
def test_rotary_refusals(more, match):
    from ogv.packed import axial_rotary
    a = dict(q=torch.zeros(5, 3, 16), k=torch.zeros(5, 1, 16), positions=torch.zeros(5, 2, dtype=torch.int32), sections=(4, 4))
    with pytest.raises(ValueError, match=match):
        axial_rotary(**{**a, **more})
    with pytest.raises(TypeError, match="int32 or float32"):
        axial_rotary(**{**a, "positions": torch.zeros(5, 2, dtype=torch.int64)})
    with pytest.raises(RuntimeError, match="HIP device"):
        axial_rotary(**a)


def test_rotary_attention_rows_refusals():
    from ogv.packed import rotary_attention_rows
    cu = torch.tensor([0, 5], dtype=torch.int32)
    with pytest.raises(ValueError, match="columns"):
        rotary_attention_rows(torch.zeros(5, 50), cu, 4)
    with pytest.raises(ValueError, match="belong together"):
        rotary_attention_rows(torch.zeros(5, 48), cu, 2, sections=(2, 2))
    with pytest.raises(ValueError, match="multiple of kv_heads"):
        rotary_attention_rows(torch.zeros(5, 8 * 7), cu, 3, 2)
    with pytest.raises(RuntimeError, match="HIP device"):
        rotary_attention_rows(torch.zeros(5, 48), cu, 2)


@pytest.mark.parametrize("more,match", [
    (dict(residual=torch.zeros(6, 7)), "equal"),
    (dict(pre_norm="batch"), "norms are"),
    (dict(post_weight=torch.ones(8)), "absent post_norm"),
    (dict(pre_norm=None, pre_weight=torch.ones(8)), "absent pre_norm"),
    (dict(pre_weight=torch.ones(7)), "pre_weight"),
    (dict(gate=torch.ones(7)), "gate"),
    (dict(gate=torch.ones(4, 8)), "samples"),
    (dict(rps=0), "rps"),
    (dict(row_scale=torch.ones(2), rps=2), "row_scale"),
    (dict(branch=torch.zeros(1, 8200), residual=torch.zeros(1, 8200)), "8200 channels"),
])
def test_gated_norm_refusals(more, match):
    from ogv.packed import gated_residual_norm
    a = dict(branch=torch.zeros(6, 8), residual=torch.zeros(6, 8))
    with pytest.raises(ValueError, match=match):
        gated_residual_norm(**{**a, **more})
    with pytest.raises(TypeError, match="mixed"):
        gated_residual_norm(torch.zeros(6, 8), torch.zeros(6, 8).bfloat16())
    with pytest.raises(RuntimeError, match="HIP device"):
        gated_residual_norm(**a)


def test_layers_refuse():
    from ogv.layers import GatedResidualNorm, PackedSelfAttention
    with pytest.raises(ValueError, match="divisible"):
        PackedSelfAttention(10, 4)
    with pytest.raises(ValueError, match="multiple"):
        PackedSelfAttention(64, 4, 3)
    with pytest.raises(ValueError, match="packed rows"):
        PackedSelfAttention(64, 4)(torch.zeros(1, 2, 64), None)
    with pytest.raises(KeyError):
        GatedResidualNorm(8, post_norm="batch")
    m = GatedResidualNorm(8, post_norm="rms", pre_norm="layer", gate_init=0.5)
    assert sorted(n for n, _ in m.named_parameters()) == ["gate", "post_weight", "pre_bias", "pre_weight"]


def test_c_abi_refuses_before_any_launch():
    """Every one of these calls returns an error code on a machine without a GPU: nothing was launched."""
    import ogv._lib as L
    lib = L.load()
    x, odd = ctypes.c_void_p(64), ctypes.c_void_p(72)

    def desc(**more):
        d = L.PackedDesc(B=2, Mq=10, Mk=10, heads=4, kv_heads=2, D=16, causal=0, scale=0.25)
        for i in range(8):
            d.row[i], d.head[i] = 64, 16
        for n, v in more.items():
            setattr(d, n, v)
        return ctypes.byref(d)

    def fwd(d, **p):
        a = dict(q=x, k=x, v=x, cu_q=x, cu_k=x, out=x, lse=x, ws=x, dt=1)
        a.update(p)
        rc = lib.ogv_packed_attn_fwd(a["q"], a["k"], a["v"], a["cu_q"], a["cu_k"], a["out"], None, a["lse"], a["ws"], d, a["dt"], None)
        return rc, lib.ogv_last_error().decode()

    for more, match in ((dict(B=0), "bad shape"), (dict(Mq=0), "bad shape"), (dict(Mk=-1), "bad shape"), (dict(heads=3), "multiple"),
                        (dict(D=20), "head_dim"), (dict(D=136), "head_dim"), (dict(scale=-1.0), "scale"), (dict(scale=float("nan")), "scale"),
                        (dict(Mq=(1 << 30)), "too many rows"), (dict(Mk=(1 << 30)), "too many rows")):
        rc, msg = fwd(desc(**more))
        assert rc == L.OGV_ERR_ARG and match in msg, (more, rc, msg)
        assert lib.ogv_packed_attn_fwd_ws_bytes(desc(**more), 1) == 0 and lib.ogv_packed_attn_bwd_ws_bytes(desc(**more), 1) == 0
        assert lib.ogv_packed_attn_bwd(x, x, x, x, x, x, x, x, x, x, x, x, x, desc(**more), 1, None) == L.OGV_ERR_ARG
    assert fwd(desc(), dt=2)[0] == L.OGV_ERR_ARG
    assert "null" in fwd(desc(), lse=None)[1]
    assert "aligned" in fwd(desc(), k=odd)[1]
    assert lib.ogv_packed_attn_fwd(x, x, x, x, x, x, x, x, x, None, 1, None) == L.OGV_ERR_ARG
    d = L.PackedDesc(B=2, Mq=10, Mk=10, heads=4, kv_heads=2, D=16, scale=0.25)
    d.row[1] = 12
    assert "multiples of 16" in fwd(ctypes.byref(d))[1]
    d.row[1] = 1 << 24
    assert "too large" in fwd(ctypes.byref(d))[1]
    d.row[1], d.head[0] = 32, 1 << 28      # two query heads share a key head: their distance is a 32-bit offset
    assert "too large" in fwd(ctypes.byref(d))[1]

    def rot(**more):
        d = L.RotaryDesc(M=4, D=16, axes=2, theta=1e4)
        d.heads[0], d.heads[1], d.pairs[0], d.pairs[1] = 2, 1, 4, 4
        for n, v in more.items():
            if isinstance(v, tuple):
                for i, e in enumerate(v):
                    getattr(d, n)[i] = e
            else:
                setattr(d, n, v)
        rc = lib.ogv_axial_rotary(x, x, x, x, x, ctypes.byref(d), 1, None)
        return rc, lib.ogv_last_error().decode()

    for more in (dict(M=-1), dict(heads=(0, 1)), dict(axes=0), dict(axes=5), dict(pairs=(4, 0)), dict(pairs=(4, 5)), dict(pairs=(60, 60)),
                 dict(D=15), dict(D=130), dict(theta=0.0), dict(row_in=(-8, 0)), dict(interleaved=1, row_in=(33, 0))):
        assert rot(**more)[0] == L.OGV_ERR_ARG, more

    def norm(f=x, **more):
        d = L.GatedNormDesc(M=4, C=16, post=1, pre=1, samples=1, rps=1, alpha=1.0, post_eps=1e-5, pre_eps=1e-5)
        for n, v in more.items():
            setattr(d, n, v)
        a = lib.ogv_gated_norm_fwd(f, x, None, None, None, None, None, None, x, x, x, ctypes.byref(d), 1, None)
        b = lib.ogv_gated_norm_bwd(x, x, f, x, x, None, None, None, None, None, x, x, x, x, None, x, ctypes.byref(d), 1, None)
        return a, b

    for more in (dict(f=None), dict(M=0), dict(C=0), dict(C=8193), dict(post=3), dict(pre=-1), dict(samples=3), dict(samples=0), dict(rps=0)):
        assert norm(**more) == (L.OGV_ERR_ARG, L.OGV_ERR_ARG), more
    assert norm(samples=2)[1] == L.OGV_ERR_ARG   # a gate per sample without a place for its gradient


def test_oracle_forms_against_differences():
    """The 64-bit forms that the kernels are tested against: their gradients against central differences, and the
    rotary against its inverse."""
    import _packed_ref as R
    g = torch.Generator().manual_seed(3)
    q, k, v, do = (torch.randn(7, h, 8, generator=g).double() for h in (4, 2, 2, 4))
    lq, lk = (3, 0, 4), (2, 1, 4)
    args = (lq, lk, True, 0.4, torch.float32)
    res = R.attention(q, k, v, *args, dout=do)
    for name, t in (("dq", q), ("dk", k), ("dv", v)):
        w = torch.randn(t.shape, generator=g).double()
        a, b = ({"q": q, "k": k, "v": v, name[1]: t + s * 1e-5 * w} for s in (1, -1))
        num = sum(s * (R.attention(x["q"], x["k"], x["v"], *args)["out"][0] * do).sum() for s, x in ((1, a), (-1, b))) / 2e-5
        assert abs(num - (res[name][0] * w).sum()) < 1e-7
    x, pos = torch.randn(5, 2, 12, generator=g), torch.randint(0, 99, (5, 2), generator=g)
    y, _ = R.rotary(x, pos, (2, 3), 100.0, True)
    z, _ = R.rotary(y, pos, (2, 3), 100.0, True, inverse=True)
    assert (z - x.double()).abs().max() < 1e-12


def test_numbers_given_as_tensors_count_by_their_value():
    """What is looked up by value must not be found again by the identity of a tensor whose value has changed."""
    from ogv.packed import axial_rotary, gated_residual_norm, packed_attention
    cpu = pytest.raises(RuntimeError, match="HIP device")   # past every check of the arguments
    scale = torch.tensor(0.25)
    with cpu:
        packed_attention(**_attn(scale=scale))
    scale.neg_()
    with pytest.raises(ValueError, match="scale"):
        packed_attention(**_attn(scale=scale))
    theta, n = torch.tensor(1e4), torch.tensor(4)
    rot = dict(q=torch.zeros(5, 3, 16), k=None, positions=torch.zeros(5, 2, dtype=torch.int32))
    with cpu:
        axial_rotary(**rot, sections=(n, 4), theta=theta)
    theta.neg_()
    with pytest.raises(ValueError, match="theta"):
        axial_rotary(**rot, sections=(n, 4), theta=theta)
    theta.neg_()
    n.fill_(5)
    with pytest.raises(ValueError, match="pairs"):
        axial_rotary(**rot, sections=(n, 4), theta=theta)
    x, rs, rps = torch.zeros(4, 8), torch.ones(2), torch.tensor(2)
    with cpu:
        gated_residual_norm(x, x, row_scale=rs, rps=rps)
    rps.fill_(1)
    with pytest.raises(ValueError, match="factors"):
        gated_residual_norm(x, x, row_scale=rs, rps=rps)


def test_rows_beyond_32_bits_are_refused():
    """Row counts are 32-bit in the C-ABI: a larger one is an error, never a smaller call."""
    from ogv.packed import axial_rotary, gated_residual_norm, packed_attention
    big = (1 << 32) + 5

    few = _attn()
    rows = torch.empty(big, 2, 16, device="meta")
    for more in (dict(q=torch.empty(big, 4, 16, device="meta")), dict(k=rows, v=rows)):
        with pytest.raises(ValueError, match="too many rows"):
            packed_attention(**{**few, **more})
    with pytest.raises(ValueError, match="too many rows"):
        axial_rotary(rows, None, torch.empty(big, 1, dtype=torch.int32, device="meta"), (8,))
    x = torch.empty(big, 8, device="meta")
    with pytest.raises(ValueError, match="too many rows"):
        gated_residual_norm(x, x)
    with pytest.raises(RuntimeError, match="HIP device"):   # more rows per factor than rows: one factor, nothing to refuse
        gated_residual_norm(torch.zeros(4, 8), torch.zeros(4, 8), row_scale=torch.ones(1), rps=big)


@pytest.fixture
def no_launch(monkeypatch):
    """The Python side on CPU tensors: nothing is launched, outputs hold zeros."""
    from ogv import packed as P
    monkeypatch.setattr(P, "_device", lambda *a: None)
    monkeypatch.setattr(P, "_launch", lambda *a: None)
    monkeypatch.setattr(torch, "empty", torch.zeros)
    monkeypatch.setattr(torch, "empty_like", torch.zeros_like)
    monkeypatch.setattr(torch.Tensor, "new_empty", torch.Tensor.new_zeros)
    return P


def _forward_mode_calls(P):
    """name -> (call, its differentiable inputs)"""
    g = torch.Generator().manual_seed(0)
    x = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    cu, pos = torch.tensor([0, 2, 6], dtype=torch.int32), torch.zeros(6, 2, dtype=torch.int32)
    return {
        "attention": (lambda q, k, v: P.packed_attention(q, k, v, cu), (x(6, 4, 16), x(6, 2, 16), x(6, 2, 16))),
        "rotary": (lambda q, k: P.axial_rotary(q, k, pos, (4, 4)), (x(6, 4, 16), x(6, 2, 16))),
        "rotary of q": (lambda q: P.axial_rotary(q, None, pos, (4, 4)), (x(6, 4, 16),)),
        "rows": (lambda qkv: P.rotary_attention_rows(qkv, cu, 2), (x(6, 96),)),
        "norm": (lambda f, r, g, w0, b0, w1, b1: P.gated_residual_norm(f, r, gate=g, post_norm="layer", post_weight=w0, post_bias=b0,
                                                                       pre_weight=w1, pre_bias=b1), (x(6, 8), x(6, 8), *(x(8) for _ in range(5)))),
    }


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("name", ["attention", "rotary", "rotary of q", "rows", "norm"])
def test_forward_mode_derivatives_are_refused(no_launch, name, grad):
    """There is no forward-mode formula: a dual input is an error, never a result without its tangent."""
    from torch.autograd import forward_ad
    call, inputs = _forward_mode_calls(no_launch)[name]
    with torch.set_grad_enabled(grad):
        call(*inputs)
        with forward_ad.dual_level():
            call(*inputs)   # no dual input: nothing to refuse
            for i, t in enumerate(inputs):
                dual = forward_ad.make_dual(t, torch.ones_like(t))
                with pytest.raises(NotImplementedError):
                    call(*inputs[:i], dual, *inputs[i + 1:])


def test_rows_attention_result_may_be_changed_in_place(no_launch):
    """As packed_attention's: in-place work on the result is allowed, and a backward that needs the old values says so."""
    qkv, cu = torch.randn(6, 96, requires_grad=True), torch.tensor([0, 2, 6], dtype=torch.int32)
    out = no_launch.rotary_attention_rows(qkv, cu, 2)
    assert out.shape == (6, 32)
    out += 1.0
    with pytest.raises(RuntimeError, match="inplace"):
        out.sum().backward()
    (no_launch.rotary_attention_rows(qkv, cu, 2) + 1.0).sum().backward()
    assert qkv.grad.shape == qkv.shape


@pytest.mark.parametrize("D,pairs,interleaved,M,heads", [(128, 64, 0, 1 << 20, 1 << 25), (128, 64, 1, 8, 1 << 25), (2, 1, 0, 8, 1 << 28),
                                                         (16, 5, 0, 3, 1 << 26), (16, 4, 0, 1, (1 << 31) - 1)])
def test_rotary_refuses_more_heads_than_it_can_count(D, pairs, interleaved, M, heads):
    """A workgroup counts the pieces of its tokens' heads in 32 bits."""
    import ogv._lib as L
    lib, x = L.load(), ctypes.c_void_p(64)
    for split in (0, 5):   # all heads in q, or some of them in k
        d = L.RotaryDesc(M=M, D=D, axes=1, theta=1e4, interleaved=interleaved)
        d.heads[0], d.heads[1], d.pairs[0] = heads - split, split, pairs
        for i in range(2):
            d.row_in[i] = d.row_out[i] = heads * D
            d.head_in[i] = d.head_out[i] = D
        assert lib.ogv_axial_rotary(x, x, x, x, x, ctypes.byref(d), 1, None) == L.OGV_ERR_ARG
        assert "too many heads" in lib.ogv_last_error().decode()
