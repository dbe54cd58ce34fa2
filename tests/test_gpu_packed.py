"""Packed-sequence operators on the device against their plain 64-bit forms (_packed_ref.py, which derives the
tolerances), at the lengths, layouts and masks where they can go wrong."""
import math

import pytest
import torch

import _norm_ref as N
import _packed_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _near(got, want, tol, name=""):
    got = got.detach().double().cpu()
    assert got.shape == want.shape
    inf = ~torch.isfinite(want)
    assert torch.equal(got[inf], want[inf]), name
    err = ((got - want).abs() - tol)[~inf]
    assert torch.isfinite(got[~inf]).all(), name
    assert err.numel() == 0 or err.max() <= 0, f"{name}: off by more than the bound, worst excess {err.max():.3e}"


def _check(q, k, v, lq, lk, causal, scale=None, dout=None, layout=lambda t: t):
    """Kernel against the 64-bit form; returns the kernel's out and gradients."""
    from ogv.packed import packed_attention
    cu_q, cu_k = R.offsets(lq).to(DEV), R.offsets(lk).to(DEV)
    qd, kd, vd = (layout(t.to(DEV)).requires_grad_(dout is not None) for t in (q, k, v))
    out, lse = packed_attention(qd, kd, vd, cu_q, cu_k, causal=causal, scale=scale, return_lse=True)
    ref = R.attention(q, k, v, lq, lk, causal, q.shape[2]**-0.5 if scale is None else scale, q.dtype, dout)
    _near(out, *ref["out"], "out")
    _near(lse, *ref["lse"], "lse")
    if dout is None:
        return (out,)
    grads = torch.autograd.grad(out, (qd, kd, vd), dout.to(DEV))
    for n, g in zip(("dq", "dk", "dv"), grads):
        _near(g, *ref[n], n)
    return (out, *grads)


def _qkv(mq, mk, h, hkv, D, dtype, seed):
    g = _gen(seed)
    return [torch.randn(m, n, D, generator=g).to(dtype) for m, n in ((mq, h), (mk, hkv), (mk, hkv), (mq, h))]


LENGTHS = [(1,), (2, 1), (16, 16), (31, 32, 33), (1, 0, 5, 0, 64, 65), (127, 128, 129), (3,) * 70, (0, 0, 40), (200,)]


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lengths", LENGTHS, ids=str)
@pytest.mark.parametrize("dtype", [BF, F32], ids=str)
def test_attention_lengths(dtype, lengths, causal):
    m = sum(lengths)
    q, k, v, do = _qkv(m, m, 4, 2, 32, dtype, m)
    _check(q, k, v, lengths, lengths, causal, dout=do)


@pytest.mark.parametrize("D", [8, 24, 40, 64, 72, 96, 104, 128])
@pytest.mark.parametrize("dtype", [BF, F32], ids=str)
def test_attention_head_dims(dtype, D):
    lengths = (70, 1, 133)
    q, k, v, do = _qkv(204, 204, 2, 2, D, dtype, D)
    _check(q, k, v, lengths, lengths, True, dout=do)


@pytest.mark.parametrize("h,hkv", [(1, 1), (3, 1), (6, 2), (12, 1), (10, 5)])
@pytest.mark.parametrize("causal", [False, True])
def test_attention_shared_heads(h, hkv, causal):
    lq = lk = (37, 64, 2)
    q, k, v, do = _qkv(103, 103, h, hkv, 48, BF, h)
    _check(q, k, v, lq, lk, causal, dout=do)


@pytest.mark.parametrize("lq,lk", [((1, 1, 1), (1, 300, 0)), ((5, 40, 2), (9, 10, 70)), ((0, 3), (4, 0)), ((130,), (3,)), ((2, 2), (600, 31))],
                         ids=str)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", [BF, F32], ids=str)
def test_attention_other_queries_than_keys(dtype, lq, lk, causal):
    """More queries than keys under the causal mask: the first ones see nothing."""
    q, k, v, do = _qkv(sum(lq), sum(lk), 4, 2, 64, dtype, sum(lk))
    _check(q, k, v, lq, lk, causal, dout=do)


@pytest.mark.parametrize("dtype", [BF, F32], ids=str)
@pytest.mark.parametrize("lq,lk,h,hkv", [((1,), (2500,), 2, 1), ((1, 1, 1, 1), (4000, 3, 900, 1), 8, 1), ((3,), (1999,), 3, 3),
                                         ((40, 1), (1500, 1500), 2, 2), ((130,), (3000,), 1, 1), ((200, 3), (2100, 900), 2, 1)], ids=str)
def test_attention_few_rows_many_keys(dtype, lq, lk, h, hkv):
    """The key axis is split between workgroups and joined."""
    import ctypes

    import ogv._lib as L
    q, k, v, do = _qkv(sum(lq), sum(lk), h, hkv, 64, dtype, 5)
    d = L.PackedDesc(B=len(lq), Mq=sum(lq), Mk=sum(lk), heads=h, kv_heads=hkv, D=64, scale=1.0)
    assert L.load().ogv_packed_attn_fwd_ws_bytes(ctypes.byref(d), 1 if dtype == BF else 0) > 0
    for causal in (False, True):
        _check(q, k, v, lq, lk, causal, dout=do)


@pytest.mark.parametrize("D", [40, 128])
def test_attention_many_single_queries(D):
    """More sequences than a wave has lanes, keys of every length among them 0 and 1, rows behind the last sequence."""
    from ogv.packed import packed_attention
    g = _gen(D)
    lk = [0, 1, 2000] + [int(n) for n in torch.randint(1, 1300, (117,), generator=g)]
    q, k, v, _ = _qkv(130, sum(lk), 2, 1, D, BF, 3)
    out, lse = packed_attention(q.to(DEV), k.to(DEV), v.to(DEV), R.offsets([1] * 120).to(DEV), R.offsets(lk).to(DEV), return_lse=True)
    ref = R.attention(q, k, v, [1] * 120, lk, False, D**-0.5, BF)
    _near(out, *ref["out"])
    _near(lse, *ref["lse"])
    assert (out[120:] == 0).all()


def test_attention_thousands_of_sequences():
    lengths = [int(n) for n in torch.randint(0, 4, (5000,), generator=_gen(0))]
    m = sum(lengths)
    q, k, v, do = _qkv(m, m, 2, 1, 16, BF, 7)
    _check(q, k, v, lengths, lengths, True, dout=do)


@pytest.mark.parametrize("dtype", [BF, F32], ids=str)
@pytest.mark.parametrize("D", [32, 64, 96, 128])
@pytest.mark.parametrize("h,hkv,lengths", [(3, 1, (900, 700)), (4, 1, (1100,)), (2, 2, (1400, 1700)), (2, 1, (40, 70))], ids=str)
def test_attention_rows_split_for_keys(dtype, D, h, hkv, lengths):
    """Few key tiles and many rows: the rows of dk and dv are split between workgroups and their sums joined."""
    import ctypes

    import ogv._lib as L
    m = sum(lengths)
    d = L.PackedDesc(B=len(lengths), Mq=m, Mk=m, heads=h, kv_heads=hkv, D=D, scale=1.0)
    split = L.load().ogv_packed_attn_bwd_ws_bytes(ctypes.byref(d), 1 if dtype == BF else 0) > 8 * m * h + 16
    assert split == (dtype == F32 or m > 1000)
    q, k, v, do = _qkv(m, m, h, hkv, D, dtype, D + h)
    for causal in (False, True):
        _check(q, k, v, lengths, lengths, causal, dout=do)


def test_attention_layouts():
    """Slices of one projection, head-major tensors, unaligned ones, broadcast heads: the same bits as contiguous ones."""
    from ogv.packed import packed_attention
    lengths, h, D = (50, 7, 90), 3, 32
    q, k, v, do = (t.to(DEV) for t in _qkv(147, 147, h, h, D, BF, 1))
    cu = R.offsets(lengths).to(DEV)

    def run(q, k, v, do=do):
        q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
        out = packed_attention(q, k, v, cu, causal=True)
        return (out, *torch.autograd.grad(out, (q, k, v), do))

    want = run(q, k, v)
    cat = torch.cat([t.flatten(1) for t in (q, k, v)], 1)
    odd = torch.empty(cat.numel() + 3, dtype=BF, device=DEV)[3:].view(cat.shape).copy_(cat)
    for rows in (cat, odd):
        got = run(*(t.unflatten(1, (h, D)) for t in rows.split(h * D, 1)))
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    major = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v)]
    got = run(*major, do=do.transpose(0, 1).contiguous().transpose(0, 1))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # one key / value head broadcast to all: the gradient of the one is the sum over the copies
    k1, v1 = k[:, :1].clone().requires_grad_(), v[:, :1].clone().requires_grad_()
    out = packed_attention(q, k1.expand(-1, h, -1), v1.expand(-1, h, -1), cu, causal=True)
    # (as shared heads the rows are grouped into other tiles, of another size: each result is within its bound of the
    # exact one, so they differ by two bounds at most)
    tol = R.attention(q, k1, v1, lengths, lengths, True, D**-0.5, BF)["out"][1]
    shared = packed_attention(q, k1, v1, cu, causal=True)
    assert ((out.double() - shared.double()).abs().cpu() <= 2 * tol).all()
    a = torch.autograd.grad(out, (k1, v1), do)
    b = torch.autograd.grad(packed_attention(q, k1, v1, cu, causal=True), (k1, v1), do)
    for x, y in zip(a, b):   # h rounded gradients added (3 roundings of the sum too) against one rounding
        assert (x.float() - y.float()).abs().max() <= 8 * 2.0**-8 * y.float().abs().max()


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", [BF, F32], ids=str)
def test_attention_rows_behind_the_last_sequence(dtype, causal):
    """Rows that belong to no sequence hold NaN: they give zeros and reach nothing; so does another sequence's NaN."""
    lengths, pad = (33, 70), 150
    q, k, v, do = _qkv(103, 103, 4, 2, 40, dtype, 9)
    from ogv.packed import packed_attention
    cu = R.offsets(lengths).to(DEV)

    def tail(t):
        return torch.cat([t, torch.full((pad, *t.shape[1:]), math.nan, dtype=dtype)]).to(DEV).requires_grad_()

    qd, kd, vd = tail(q), tail(k), tail(v)
    out, lse = packed_attention(qd, kd, vd, cu, causal=causal, return_lse=True)
    got = torch.autograd.grad(out, (qd, kd, vd), tail(do).detach())
    ref = R.attention(q, k, v, lengths, lengths, causal, 40**-0.5, dtype, do)   # (other sizes may take another split)
    for a, n in zip((out, *got), ("out", "dq", "dk", "dv")):
        _near(a[:103], *ref[n], n)
        assert (a[103:] == 0).all()
    want = _check(q, k, v, lengths, lengths, causal, dout=do)
    assert (lse[103:] == -math.inf).all()
    # NaN and infinities in the first sequence stay there
    for t in (q, k, v):
        t[5] = math.nan
        t[7] = math.inf
    qd, kd, vd = (t.to(DEV).requires_grad_() for t in (q, k, v))
    out = packed_attention(qd, kd, vd, cu, causal=causal)
    got = torch.autograd.grad(out, (qd, kd, vd), do.to(DEV))
    for a, b in zip((out, *got), want):
        assert torch.equal(a[33:], b[33:])


def test_attention_masked_keys_of_any_size():
    """Hidden keys with scores beyond every visible one, in both directions, and rows of one huge score."""
    lengths = (90,)
    q, k, v, do = _qkv(90, 90, 1, 1, 32, F32, 4)
    k[60:] *= 1e4          # seen by rows from 60 on only
    k[60:, :, 0] += 1e6
    q[:60, :, 0] = q[:60, :, 0].abs()
    out, dq, dk, dv = _check(q[:60], k[:60], v[:60], (60,), (60,), True, dout=do[:60])
    from ogv.packed import packed_attention
    full = packed_attention(q.to(DEV), k.to(DEV), v.to(DEV), R.offsets(lengths).to(DEV), causal=True)
    assert torch.equal(full[:60], out)
    assert torch.isfinite(full).all()
    # every score near the type's lowest value: the softmax is that of the differences
    q2, k2 = q[:40].clone(), k[:40].clone()
    q2[..., 0], k2[..., 0] = -1e18, 1e18
    out = packed_attention(q2.to(DEV), k2.to(DEV), v[:40].to(DEV), R.offsets((40,)).to(DEV), scale=1.0)
    mean = v[:40].double().mean(0)   # the other dims are lost in the sum: all scores equal
    assert (out.double().cpu() - mean).abs().max() <= 2.0**-24 * 64 * v.abs().max()


@pytest.mark.parametrize("D", [32, 128])
@pytest.mark.parametrize("dtype", [BF, F32], ids=str)
def test_attention_rows_decide_for_themselves(dtype, D):
    """A row of huge or infinite scores (exponents past 2^24) leaves the rows beside it in its tile as they were."""
    from ogv.packed import packed_attention
    q, k, v, _ = (t.to(DEV) for t in _qkv(100, 300, 2, 1, D, dtype, D))
    k[..., 0] = k[..., 0].abs() + 0.5
    cu_q, cu_k = R.offsets((100,)).to(DEV), R.offsets((300,)).to(DEV)
    want = packed_attention(q, k, v, cu_q, cu_k, return_lse=True)
    others = torch.arange(100, device=DEV) != 41
    for huge in (1e9, -1e9, math.inf):
        q2 = q.clone()
        q2[41, 1, 0] = huge
        got = packed_attention(q2, k, v, cu_q, cu_k, return_lse=True)
        for a, b in zip(got, want):
            assert torch.equal(a[others], b[others]) and torch.equal(a[41, 0], b[41, 0])


@pytest.mark.parametrize("scale", [1e-30, 1.5e-38, 1e-38, 2.0**-140])
@pytest.mark.parametrize("lq,lk", [((40, 70), (40, 70)), ((1,), (2500,))], ids=str)
@pytest.mark.parametrize("dtype", [BF, F32], ids=str)
def test_attention_tiny_scales(dtype, lq, lk, scale):
    """All weights of a row are equal then, however small the scale: a row that sees keys is never one that sees none."""
    from ogv.packed import packed_attention
    q, k, v, do = _qkv(sum(lq), sum(lk), 2, 1, 32, dtype, 3)
    ts = [t.to(DEV).requires_grad_() for t in (q, k, v)]
    out, lse = packed_attention(*ts, R.offsets(lq).to(DEV), R.offsets(lk).to(DEV), causal=True, scale=scale, return_lse=True)
    dq, dk, dv = torch.autograd.grad(out, ts, do.to(DEV))
    ref = R.attention(q, k, v, lq, lk, True, scale, dtype, do)
    for got, n in ((out, "out"), (lse, "lse"), (dv, "dv")):
        _near(got, *ref[n], n)
    for got, n in ((dq, "dq"), (dk, "dk")):   # below the smallest normal number a result may be flushed to zero
        _near(got, ref[n][0], ref[n][1] + 2.0**-126, n)


@pytest.mark.parametrize("D", [24, 32, 72])
@pytest.mark.parametrize("dtype", [BF, F32], ids=str)
def test_attention_key_of_minus_infinity(dtype, D):
    """A key whose score is -inf for every query weighs nothing, with every head size (padded or not)."""
    from ogv.packed import packed_attention
    q, k, v, _ = _qkv(50, 50, 2, 1, D, dtype, D)
    q[..., 0] = q[..., 0].abs() + 0.5
    keep = torch.arange(50) != 5
    ref = R.attention(q, k[keep], v[keep], (50,), (49,), False, D**-0.5, dtype)
    k[5, :, 0] = -math.inf
    out = packed_attention(q.to(DEV), k.to(DEV), v.to(DEV), R.offsets((50,)).to(DEV))
    _near(out, *ref["out"])


def test_attention_bad_offsets_stay_inside():
    """Offsets past the rows are clamped, a decreasing pair is an empty sequence: no row outside is read or written."""
    from ogv.packed import packed_attention
    q, k, v, _ = (t.to(DEV) for t in _qkv(40, 40, 2, 2, 32, BF, 2))
    got = packed_attention(q, k, v, torch.tensor([0, 10, 1000], dtype=torch.int32, device=DEV))
    assert torch.equal(got, packed_attention(q, k, v, torch.tensor([0, 10, 40], dtype=torch.int32, device=DEV)))
    got = packed_attention(q, k, v, torch.tensor([5, 10, 40], dtype=torch.int32, device=DEV))
    assert torch.equal(got, packed_attention(q, k, v, torch.tensor([0, 10, 40], dtype=torch.int32, device=DEV)))


@pytest.mark.parametrize("h,hkv", [(2, 2), (2, 1), (4, 1), (6, 2)])
@pytest.mark.parametrize("offsets", [(0, 60, 5, 60), (0, 60, *(5,) * 70, 60), (0, 3, 1, 500, -4, 20), (0, *(60, 0) * 40)], ids=lambda o: str(len(o)))
@pytest.mark.parametrize("causal", [False, True])
def test_attention_decreasing_offsets_stay_inside(h, hkv, offsets, causal):
    """Offsets that decrease are the caller's error: the results are unspecified, nothing beside them is written."""
    import ogv._lib as L
    from ogv import packed as P
    m, D, edge, boxes = 60, 32, 4096, []
    q, k, v, do = (t.to(DEV) for t in _qkv(m, m, h, hkv, D, BF, 2))
    cu = torch.tensor(offsets, dtype=torch.int32, device=DEV)

    def boxed(*shape, dtype=BF):
        n = math.prod(shape)
        box = torch.full((n + 2 * edge,), 7.0, dtype=dtype, device=DEV)
        boxes.append(box)
        return box[edge:edge + n].view(shape)

    out, lo, dq = (boxed(m, h, D) for _ in range(3))
    dk, dv = (boxed(m, hkv, D) for _ in range(2))
    lse = boxed(m, h, dtype=F32)
    d, ws, _ = P._packed_desc(len(offsets) - 1, m, m, h, hkv, D, causal, D**-0.5, L.OGV_BF16, *(P._strides(t) for t in (q, k, v, out)))
    ws = P._ws(ws, q)
    P._launch(L.load().ogv_packed_attn_fwd, "ogv_packed_attn_fwd", q, *map(P._ptr, (q, k, v, cu, cu, out, lo, lse, ws)), d, L.OGV_BF16)
    P._attn_bwd(do, q, k, v, out, lo, lse, cu, cu, causal, D**-0.5, dq, dk, dv)
    torch.cuda.synchronize()
    for box in boxes:
        assert (box[:edge] == 7).all() and (box[-edge:] == 7).all()


def test_attention_no_rows():
    from ogv.packed import packed_attention
    z = torch.zeros(0, 2, 16, device=DEV, requires_grad=True)
    cu = torch.zeros(3, dtype=torch.int32, device=DEV)
    assert packed_attention(z, z, z, cu).shape == (0, 2, 16)
    q = torch.ones(4, 2, 16, device=DEV, requires_grad=True)
    none = torch.zeros(1, dtype=torch.int32, device=DEV)
    out, lse = packed_attention(q, q, q, none, return_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all()
    assert (torch.autograd.grad(out.sum(), q)[0] == 0).all()
    out, lse = packed_attention(q, z, z, torch.tensor([0, 1, 4], dtype=torch.int32, device=DEV), cu, return_lse=True)   # no key anywhere
    assert (out == 0).all() and (lse == -math.inf).all()
    dq, dk, dv = torch.autograd.grad(out.sum(), (q, z, z))[0], None, None
    assert (dq == 0).all()


def test_attention_far_rows():
    """Row offsets past 32 bits: a key cache whose rows are 4 Mi elements apart."""
    from ogv.packed import packed_attention
    n, stride = 700, 1 << 22
    big = torch.empty(n * stride, dtype=BF, device=DEV)
    q, k, v, do = _qkv(3, n, 2, 1, 64, BF, 8)
    kd = big.as_strided((n, 1, 64), (stride, 64, 1)).copy_(k)
    vd = big.as_strided((n, 1, 64), (stride, 64, 1), 4096).copy_(v)
    cu_q, cu_k = R.offsets((3,)).to(DEV), R.offsets((n,)).to(DEV)
    got = packed_attention(q.to(DEV), kd, vd, cu_q, cu_k)
    assert torch.equal(got, packed_attention(q.to(DEV), k.to(DEV), v.to(DEV), cu_q, cu_k))


@pytest.mark.parametrize("dtype", [BF, F32], ids=str)
def test_attention_is_deterministic(dtype):
    q, k, v, do = _qkv(700, 700, 4, 2, 64, dtype, 6)
    a, b = (_check(q, k, v, (400, 300), (400, 300), True, dout=do) for _ in range(2))
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_attention_gradient_against_differences():
    from ogv.packed import packed_attention
    lengths = (40, 23)
    q, k, v, do = (t.to(DEV) for t in _qkv(63, 63, 4, 2, 32, F32, 12))
    cu = R.offsets(lengths).to(DEV)
    ts = [t.requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(packed_attention(*ts, cu, causal=True), ts, do)
    g = _gen(1)
    e = 2.0**-6
    for i, (t, gr) in enumerate(zip(ts, grads)):
        w = torch.randn(t.shape, generator=g).to(DEV)
        w /= w.norm()
        loss = []
        for s in (1, -1, 2, -2):
            a = [x.detach() for x in ts]
            a[i] = a[i] + s * e * w
            loss.append((packed_attention(*a, cu, causal=True).double() * do.double()).sum().item())
        num = (8 * (loss[0] - loss[1]) - (loss[2] - loss[3])) / (12 * e)   # error e^4 f''''' / 30
        # each loss is a sum of 63 * 4 * 32 products whose fp32 outputs are off by under 2^-20 relative
        noise = 2.0**-20 * do.double().abs().sum().item() * 3 * 18 / (12 * e) / math.sqrt(do.numel())
        assert abs(num - (gr.double() * w.double()).sum().item()) <= noise + 30 * e**4


# ------------------------------------------------------------------------------------------------ rotary
@pytest.mark.parametrize("dtype", [BF, F32], ids=str)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("M,h,hkv,D,sections,far", [
    (1, 1, 1, 2, (1,), 9), (3, 2, 1, 6, (1, 1), 99), (17, 3, 3, 24, (6, 6), 28), (50, 12, 4, 64, (16, 16), 32), (33, 4, 1, 128, (16, 24, 24), 100000),
    (9, 2, 2, 40, (8,), 50), (65, 5, 5, 128, (8, 8, 8, 8), 1000), (7, 2, 1, 64, (5, 6), 10), (300, 8, 2, 96, (48,), 1 << 30)])
def test_rotary(dtype, interleaved, M, h, hkv, D, sections, far):
    from ogv.packed import axial_rotary
    g = _gen(D + M)
    q, k, dq, dk = (torch.randn(M, n, D, generator=g).to(dtype) for n in (h, hkv, h, hkv))
    pos = torch.randint(-far, far, (M, len(sections)), generator=g).int()
    qd, kd = q.to(DEV).requires_grad_(), k.to(DEV).requires_grad_()
    a, b = axial_rotary(qd, kd, pos.to(DEV), sections, theta=500.0, interleaved=interleaved)
    ga, gb = torch.autograd.grad((a, b), (qd, kd), (dq.to(DEV), dk.to(DEV)))
    for got, x, inv in ((a, q, False), (b, k, False), (ga, dq, True), (gb, dk, True)):
        _near(got, *R.rotary(x, pos, sections, 500.0, interleaved, inv))
    only = axial_rotary(q.to(DEV), None, pos.to(DEV), sections, theta=500.0, interleaved=interleaved)
    assert torch.equal(only, a)


def test_rotary_positions_and_layouts():
    """Fractional positions, slices of one projection, unaligned rows, a broadcast head, no rows."""
    from ogv.packed import axial_rotary
    g = _gen(2)
    M, h, D, sec = 31, 3, 32, (8, 8)
    qkv = torch.randn(M, 3 * h * D + 8, generator=g).to(BF).to(DEV)
    pos = torch.rand(M, 2, generator=g).to(DEV) * 14
    q, k = (qkv[:, i * h * D:(i + 1) * h * D].unflatten(1, (h, D)) for i in (0, 1))
    a, b = axial_rotary(q, k, pos, sec)
    _near(a, *R.rotary(q, pos, sec, 1e4, False))
    c, d = axial_rotary(q.contiguous(), k.contiguous(), pos, sec)
    assert torch.equal(a, c) and torch.equal(b, d)
    odd = torch.empty(q.numel() + 1, dtype=BF, device=DEV)[1:].view(q.shape).copy_(q)
    assert torch.equal(axial_rotary(odd, None, pos, sec), a)
    one = q[:, :1].detach().clone().requires_grad_()
    e = axial_rotary(one.expand(-1, h, -1), None, pos, sec)
    assert torch.equal(e[:, 0], e[:, 2])
    torch.autograd.grad(e.sum(), one)
    assert axial_rotary(q[:0], k[:0], pos[:0], sec)[1].shape == (0, h, D)


# ------------------------------------------------------------------------------------------------ norms
def _norm_case(M, C, dtype, post, pre, gate, samples, rs, bias, seed):
    g = _gen(seed)
    t = {"f": torch.randn(M, C, generator=g).to(dtype) * 2, "x": torch.randn(M, C, generator=g).to(dtype) + 0.5}
    t["gate"] = torch.randn(*((samples, C) if samples else (C,)), generator=g) if gate else None
    for n, kind in (("post", post), ("pre", pre)):
        t[n + "_w"] = 1 + 0.2 * torch.randn(C, generator=g) if kind else None
        t[n + "_b"] = 0.2 * torch.randn(C, generator=g) if kind and bias else None
    t["rs"] = (torch.rand(-(-M // rs), generator=g) < 0.8).float() / 0.8 if rs else None
    return t, torch.randn(M, C, generator=g).to(dtype), torch.randn(M, C, generator=g).to(dtype)


def _norm_check(M, C, dtype, post, pre, gate=True, samples=0, rs=0, bias=True, alpha=1.0, use=("y", "h"), seed=0):
    from ogv.packed import gated_residual_norm
    t, dy, dh = _norm_case(M, C, dtype, post, pre, gate, samples, rs, bias, seed + M + C)
    wrt = [n for n, v in t.items() if v is not None and n != "rs"]
    dev = {n: None if v is None else v.to(DEV).requires_grad_(n in wrt) for n, v in t.items()}
    ref = {n: None if v is None else v.double().requires_grad_(n in wrt) for n, v in t.items()}
    got = gated_residual_norm(dev["f"], dev["x"], gate=dev["gate"], row_scale=dev["rs"], rps=rs or 1, alpha=alpha, post_norm=post,
                              post_weight=dev["post_w"], post_bias=dev["post_b"], pre_norm=pre, pre_weight=dev["pre_w"], pre_bias=dev["pre_b"])
    y, h = R.gated_norm(ref["f"], ref["x"], ref["gate"], ref["rs"], rs or 1, alpha, post, ref["post_w"], ref["post_b"], pre, ref["pre_w"],
                        ref["pre_b"])
    got = dict(zip("yh", got if pre else (got,)))
    want = {"y": y, "h": h}
    u = R.half_step(dtype)
    # fp32 arithmetic: a row's sums add at most 8 columns a lane (32 past 4096) and 8 steps across lanes; with the
    # dozen operations of a value, and of the values it is made from, under K = 256 roundings of 2^-24, each of a
    # number bounded by the row's largest (the norm magnifies by rstd, and its own output by 1 + max |vhat|)
    K = 256 * R.U32

    def amp(v, kind):
        if kind is None:
            return torch.ones(M, 1, dtype=torch.float64), torch.ones(M, 1, dtype=torch.float64)
        d = v - v.mean(1, keepdim=True) if kind == "layer" else v
        rstd = 1 / (d.square().mean(1, keepdim=True) + 1e-5).sqrt()
        return rstd, 1 + (d * rstd).abs().amax(1, keepdim=True)

    with torch.no_grad():
        rows = torch.arange(M)
        sg = (ref["gate"][rows // (M // samples)] if samples else ref["gate"][None]).abs() if gate else torch.ones(1, 1).double()
        if rs:
            sg = sg * ref["rs"][rows // rs][:, None]
        wb = {n: (ref[n + "_w"].abs().amax() + (ref[n + "_b"].abs().amax() if ref[n + "_b"] is not None else 0)) if ref[n + "_w"] is not None else 1.0
              for n in ("post", "pre")}
        fmax = ref["f"].abs().amax(1, keepdim=True)
        rf, af = amp(ref["f"], post)
        n_mag = (af * (1 + rf * fmax) * wb["post"]) if post else fmax
        sgm = sg.amax(1, keepdim=True)
        y_mag = abs(alpha) * ref["x"].abs().amax(1, keepdim=True) + sgm * n_mag
        ry, ay = amp(y, pre)
        h_mag = ay * (1 + ry * y_mag) * wb["pre"]
    _near(got["y"], y.detach(), u * y.detach().abs() * (1 + K) + K * y_mag, "y")
    if pre:
        _near(got["h"], h.detach(), u * h.detach().abs() * (1 + K) + K * h_mag, "h")
    use = [n for n in use if n in got]
    given = {"y": dy, "h": dh}
    ga = torch.autograd.grad([got[n] for n in use], [dev[n] for n in wrt], [given[n].to(DEV) for n in use], allow_unused=True)
    gr = torch.autograd.grad([want[n] for n in use], [ref[n] for n in wrt], [given[n].double() for n in use], allow_unused=True)
    with torch.no_grad():
        dyv = dy.double().abs().amax(1, keepdim=True) if "y" in use else 0.0
        dhv = dh.double().abs().amax(1, keepdim=True) * wb["pre"] if "h" in use and pre else torch.zeros(M, 1).double()
        dY_mag = dyv + (ay**2 * (1 + ry * y_mag) * ry * dhv if pre else 0.0)
        dn_mag = sgm * dY_mag
        mags = {"x": abs(alpha) * dY_mag, "f": af**2 * (1 + rf * fmax) * rf * dn_mag * wb["post"] if post else dn_mag}
        # column sums: at most M further additions of terms bounded by the rows' magnitudes
        S = K + M * R.U32
        rs_row = ref["rs"][rows // rs][:, None] if rs else torch.ones(M, 1).double()
        gm = rs_row * n_mag * dY_mag
        mags["gate"] = (gm.view(samples, -1).sum(1, keepdim=True) if samples else gm.sum()) if gate else None
        mags["pre_w"], mags["pre_b"] = (dhv * ay * (1 + ry * y_mag)).sum(), dhv.sum()
        mags["post_w"], mags["post_b"] = (dn_mag * af * (1 + rf * fmax)).sum(), dn_mag.sum()
    for n, a, b in zip(wrt, ga, gr):
        if b is None:   # the formula does not reach it: zeros, or no gradient
            assert a is None or (a == 0).all(), n
        elif n in ("f", "x"):
            _near(a, b, u * b.abs() * (1 + K) + K * mags[n], n)
        else:
            assert a.dtype == F32
            _near(a, b, (S * mags[n]).expand_as(b) + R.U32 * b.abs(), n)
    return got, ga


@pytest.mark.parametrize("dtype", [BF, F32], ids=str)
@pytest.mark.parametrize("C", [1, 3, 8, 24, 48, 130, 264, 331, 512, 520, 768, 776, 1024, 1025, 1032, 2048, 2056, 4096, 4099, 8192])
def test_norm_channels(dtype, C):
    _norm_check(9, C, dtype, "layer" if C > 1 else "rms", "layer" if C > 1 else "rms")


@pytest.mark.parametrize("post", [None, "layer", "rms"])
@pytest.mark.parametrize("pre", [None, "layer", "rms"])
@pytest.mark.parametrize("C", [96, 97, 2000])
def test_norm_kinds(post, pre, C):
    _norm_check(37, C, BF, post, pre, rs=5, alpha=0.7)
    _norm_check(37, C, F32, post, pre, gate=False, bias=False)


@pytest.mark.parametrize("M,samples,rs", [(1, 1, 1), (6, 2, 3), (2100, 2100, 1), (4000, 4, 100), (1300, 1300, 7), (5000, 0, 64), (3, 0, 8)])
@pytest.mark.parametrize("C", [40, 45])
def test_norm_samples(M, samples, rs, C):
    """A gate per sample, more samples than workgroups, more rows than a workgroup takes at once."""
    _norm_check(M, C, F32, "rms", "layer", samples=samples, rs=rs)


@pytest.mark.parametrize("use", ["both", "y", "h"])
@pytest.mark.parametrize("c", N.CASES, ids=lambda c: "-".join(str(v).replace("torch.", "") for v in c))
def test_norm_values_and_gradients(c, use):
    """Every output and gradient within a bound made of its own terms' roundings (test_norm_bounds.py: broken gradients
    do not lie within them)."""
    from ogv.packed import gated_residual_norm
    M, C, dtype, post, pre, samples, rs, alpha = c
    t, dy, dh = N.case(M, C, dtype, post, pre, samples, rs)
    dy, dh = (None if use == "h" and pre else dy), (dh if use != "y" and pre else None)
    want = N.gated_norm(t, dy, dh, alpha, post, pre, rs or 1)
    p = {n: None if v is None else v.to(DEV).requires_grad_(n != "rs") for n, v in t.items()}
    out = gated_residual_norm(p["f"], p["x"], gate=p["gate"], row_scale=p["rs"], rps=rs or 1, alpha=alpha, post_norm=post, post_weight=p["post_w"],
                              post_bias=p["post_b"], pre_norm=pre, pre_weight=p["pre_w"], pre_bias=p["pre_b"])
    y, h = out if pre else (out, None)
    wrt = [n for n, v in p.items() if v is not None and n != "rs"]
    outs = [(o, g.to(DEV)) for o, g in ((y, dy), (h, dh)) if g is not None]
    got = dict(zip(wrt, torch.autograd.grad([o for o, _ in outs], [p[n] for n in wrt], [g for _, g in outs])))
    got.update(y=y, **({"h": h} if pre else {}))
    for n, g in got.items():
        if n not in want:   # (no gradient reaches the pre norm without dh)
            assert (g == 0).all(), n
            continue
        assert g.shape == want[n].x.shape and g.dtype == (dtype if n in "yhfx" else F32)
        assert N.excess(g, want[n], g.dtype) <= 0, n


@pytest.mark.parametrize("use", [("y",), ("h",)])
def test_norm_one_gradient(use):
    _norm_check(50, 64, BF, "layer", "layer", use=use)


def test_norm_edges():
    from ogv.packed import gated_residual_norm
    # constant rows: variance 0, h = bias; no rows; strided and broadcast operands
    f = torch.full((4, 64), 3.0, device=DEV)
    y, h = gated_residual_norm(f, f, post_norm="layer", pre_norm="layer")
    assert torch.equal(y, f) and (h == 0).all()
    w = torch.ones(64, device=DEV, requires_grad=True)
    y, h = gated_residual_norm(f[:0], f[:0], gate=w, pre_weight=w)
    assert y.shape == (0, 64)
    assert (torch.autograd.grad(h.sum(), w)[0] == 0).all()
    x = torch.randn(10, 130, device=DEV)
    a = gated_residual_norm(x[:, 1:65], x[:, 65:129], gate=w)
    b = gated_residual_norm(x[:, 1:65].contiguous(), x[:, 65:129].contiguous(), gate=w)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    row = torch.randn(1, 64, device=DEV, requires_grad=True)
    y, h = gated_residual_norm(row.expand(5, -1), x[:5, :64])
    g, = torch.autograd.grad(y.sum(), row)
    torch.testing.assert_close(g, torch.full_like(g, 5.0))
    # a row of NaN stays alone
    f2 = torch.randn(6, 64, device=DEV)
    f3 = f2.clone()
    f3[2] = math.nan
    for p, q in zip(gated_residual_norm(f2[:4], f, gate=w, post_norm="rms"), gated_residual_norm(f3[:4], f, gate=w, post_norm="rms")):
        assert torch.equal(p[[0, 1, 3]], q[[0, 1, 3]]) and q[2].isnan().all()


def test_norm_gradient_against_differences():
    from ogv.packed import gated_residual_norm
    g = _gen(4)
    t = [torch.randn(s, generator=g).to(DEV).requires_grad_() for s in ((12, 40), (12, 40), (3, 40), (40,), (40,))]
    dy, dh = (torch.randn(12, 40, generator=g).to(DEV) for _ in range(2))

    def loss(f, x, gate, w0, w1):
        return gated_residual_norm(f, x, gate=gate, post_norm="rms", post_weight=w0, pre_norm="layer", pre_weight=w1)

    grads = torch.autograd.grad(loss(*t), t, (dy, dh))
    e = 2.0**-7
    for i, gr in enumerate(grads):
        w = torch.randn(t[i].shape, generator=g).to(DEV)
        w /= w.norm()
        v = []
        for s in (1, -1, 2, -2):
            a = [p.detach() for p in t]
            a[i] = a[i] + s * e * w
            y, h = loss(*a)
            v.append((y.double() * dy.double()).sum().item() + (h.double() * dh.double()).sum().item())
        num = (8 * (v[0] - v[1]) - (v[2] - v[3])) / (12 * e)
        # outputs off by under 2^-20 of numbers up to 8, 960 of them, independent; truncation e^4 of a norm's fifth derivative
        noise = 2.0**-20 * 8 * math.sqrt(960) * 3 * 18 / (12 * e)
        assert abs(num - (gr.double() * w.double()).sum().item()) <= noise + 300 * e**4


# ------------------------------------------------------------------------------------------------ together
def _block(dtype, dim=96, heads=4, kv=2):
    from ogv.layers import GatedResidualNorm, PackedSelfAttention
    torch.manual_seed(0)
    attn = PackedSelfAttention(dim, heads, kv, sections=(6, 6), causal=False).to(DEV)
    norm = GatedResidualNorm(dim, post_norm="rms", pre_norm="layer", gate_init=0.3).to(DEV)
    return attn, norm


LENS = (49, 16, 100, 1)


def _block_inputs(dtype, dim=96):
    g = _gen(77)
    m = sum(LENS)
    x, h = torch.randn(m, dim, generator=g), torch.randn(m, dim, generator=g)
    pos = torch.cat([torch.stack([torch.arange(n) // 7, torch.arange(n) % 7], 1) for n in LENS]).int()
    return x.to(dtype).to(DEV), h.to(dtype).to(DEV), pos.to(DEV), R.offsets(LENS).to(DEV)


def test_rotary_attention_rows_is_the_two_operators():
    from ogv.packed import axial_rotary, packed_attention, rotary_attention_rows
    _, _, pos, cu = _block_inputs(BF)
    h, hkv, D = 4, 2, 24
    for dtype in (BF, F32):
        qkv = torch.randn(sum(LENS), (h + 2 * hkv) * D, generator=_gen(1)).to(dtype).to(DEV).requires_grad_()
        do = torch.randn(sum(LENS), h * D, generator=_gen(2)).to(dtype).to(DEV)
        for with_pos in (True, False):
            out = rotary_attention_rows(qkv, cu, h, hkv, positions=pos if with_pos else None, sections=(6, 6) if with_pos else None, causal=True)
            got, = torch.autograd.grad(out, qkv, do)
            q, k, v = (t.unflatten(1, (-1, D)) for t in qkv.split((h * D, hkv * D, hkv * D), 1))
            if with_pos:
                q, k = axial_rotary(q, k, pos, (6, 6))
            want = packed_attention(q, k, v, cu, causal=True).flatten(1)
            assert torch.equal(out, want)
            assert torch.equal(got, torch.autograd.grad(want, qkv, do)[0])


@pytest.mark.parametrize("dtype", [BF, F32], ids=str)
def test_block_of_all_three(dtype):
    """h -> qkv -> rotary -> packed attention -> proj -> gated residual norm, against the 64-bit composition."""
    attn, norm = _block(dtype)
    x, h, pos, cu = _block_inputs(dtype)
    params = [*attn.parameters(), *norm.parameters()]
    xs, hs = x.detach().requires_grad_(), h.detach().requires_grad_()
    y, z = norm(attn(hs, cu, pos), xs)
    g = _gen(5)
    dy, dz = (torch.randn(y.shape, generator=g).to(dtype).to(DEV) for _ in range(2))
    got = (y, z, *torch.autograd.grad((y, z), (xs, hs, *params), (dy, dz)))

    P = [p.detach().double().cpu().requires_grad_() for p in params]
    wq, bq, wp, bp = P[:4]
    names = [n for n, _ in norm.named_parameters()]
    N = dict(zip(names, P[4:]))
    xd, hd = (t.detach().double().cpu().requires_grad_() for t in (x, h))
    q, k, v = ((hd @ wq.T + bq).split((96, 48, 48), 1))
    q, k, v = (t.unflatten(1, (-1, 24)) for t in (q, k, v))
    ang = torch.cat([pos[:, a:a + 1].double().cpu() * torch.tensor([1e4 ** (-j / 6) for j in range(6)], dtype=torch.float64) for a in (0, 1)], 1)[:, None]
    turn = lambda t: torch.cat((t[..., :12] * ang.cos() - t[..., 12:] * ang.sin(), t[..., 12:] * ang.cos() + t[..., :12] * ang.sin()), -1)  # noqa: E731
    q, k = turn(q), turn(k)
    outs, a = [], 0
    for n in LENS:
        s = torch.einsum("ihd,jhd->hij", q[a:a + n], k[a:a + n].repeat_interleave(2, 1)) * 24**-0.5
        outs.append(torch.einsum("hij,jhd->ihd", s.softmax(-1), v[a:a + n].repeat_interleave(2, 1)).flatten(1))
        a += n
    o = torch.cat(outs) @ wp.T + bp
    yr, zr = R.gated_norm(o, xd, N["gate"], None, 1, 1.0, "rms", N["post_weight"], None, "layer", N["pre_weight"], N["pre_bias"])
    want = (yr, zr, *torch.autograd.grad((yr, zr), (xd, hd, *P), (dy.double().cpu(), dz.double().cpu())))
    # eight stages, each with at most three roundings to the type on its path (input, product, output; weights are
    # split in two in the forward and rounded in the backward): in 2-norm at most 24 u, and 2^-16 of fp32 sums
    u = R.half_step(dtype)
    for i, (p, r) in enumerate(zip(got, want)):
        rel = (p.detach().double().cpu() - r.detach()).norm() / r.detach().norm()
        assert rel <= 24 * u + 2.0**-16, (i, rel)


def test_captured_blocks_replay():
    """Forward and backward of the three operators in two graphs, replayed in turn with eager work between them on
    another stream: every replay gives the eager bits."""
    attn, norm = _block(BF)
    for p in (*attn.parameters(), *norm.parameters()):
        p.requires_grad_(False)

    def step(x, h, pos, cu, dy, dz):
        xs, hs = x.detach().requires_grad_(), h.detach().requires_grad_()
        y, z = norm(attn(hs, cu, pos), xs)
        return (y, z, *torch.autograd.grad((y, z), (xs, hs), (dy, dz)))

    sets = []
    for seed in (1, 2):
        g = _gen(seed)
        x, h, pos, cu = _block_inputs(BF)
        dy, dz = (torch.randn(x.shape, generator=g).to(BF).to(DEV) for _ in range(2))
        sets.append([x * seed, h / seed, pos, cu, dy, dz])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = [step(*s) for s in sets]
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for s in sets:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(step(*s))
        graphs.append(gr)
    for n in range(4):
        for gr in graphs if n % 2 else graphs[::-1]:
            gr.replay()
        with torch.cuda.stream(side):
            again = step(*sets[n % 2])
        torch.cuda.synchronize()
        for got, w in zip(outs, want):
            assert all(torch.equal(a, b) for a, b in zip(got, w))
        assert all(torch.equal(a, b) for a, b in zip(again, want[n % 2]))
    # new lengths in the same offsets tensor reach the replay: nothing is kept from one call for the next
    new = R.offsets((100, 1, 16, 49)).to(DEV)
    sets[0][3].copy_(new)
    graphs[0].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs[0], step(*sets[0])))
