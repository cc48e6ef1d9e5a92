"""Attention over packed sequences (detrpose_amd.attention) against its definition in 64 bits.

Tolerances, per element, from the operator's own roundings (h: half a step of the type, u = 2^-24):
a weight p carries a relative error ep from f32 scores (dim products, the bias), the exponential and the
sum, and one rounding h for its product; the result one rounding h of itself and n u from the f32 sum of
its n terms. D = sum dO O inherits the stored output's error; ds = p (dp - D) that of p, dp and D, and
one rounding h for its products. _reference() adds these up term by term in magnitudes."""
import math

import pytest
import torch

from detrpose_amd import attention as A

U = 2.0 ** -24
HALF = {torch.float32: U, torch.bfloat16: 2.0 ** -8}
F = torch.float64


def _bucket(rel, buckets, max_distance, both):
    """One distance's bucket from the formula, in whole numbers."""
    nb = buckets // 2 if both else buckets
    base = buckets // 2 if both and rel > 0 else 0
    n = abs(rel) if both else max(0, -rel)
    e = nb // 2
    if n < e:
        return base + n
    j = 0
    while j + 1 < nb - e and n ** (nb - e) >= e ** (nb - e - j - 1) * max_distance ** (j + 1):
        j += 1
    return base + e + j


def _reference(q, k, v, ql, kl, causal, scale, table=None, max_distance=128, both=True, dout=None):
    """{name: (value, bound)} in 64 bits."""
    h = HALF[q.dtype]
    tb = 0.0 if table is None else HALF[table.dtype]
    H, hk, d = q.shape[1], k.shape[1], q.shape[2]
    z = lambda t: [torch.zeros(t.shape, dtype=F, device=t.device) for _ in range(2)]  # noqa: E731
    out, dq, dk, dv = z(q), z(q), z(k), z(v)
    dt = None if table is None else z(table)
    dkr, dvr = z(k), z(v)   # magnitudes before the last rounding
    dtr = None if table is None else torch.zeros(table.shape, dtype=F, device=q.device)
    q0 = k0 = 0
    for a, b in zip(ql, kl):
        qs, ks = slice(q0, q0 + a), slice(k0, k0 + b)
        q0, k0 = q0 + a, k0 + b
        if not a or not b:
            continue
        rel = torch.arange(b, device=q.device)[None] - torch.arange(a, device=q.device)[:, None] - (b - a)
        see = rel <= 0 if causal else torch.ones_like(rel, dtype=torch.bool)
        if table is not None:
            far = a + b
            lut = torch.tensor([_bucket(r, table.shape[0], max_distance, both) for r in range(-far, far + 1)],
                               device=q.device)
            which = lut[rel + far]
        for n in range(H):
            m = n // (H // hk)
            qh, kh, vh = q[qs, n].to(F), k[ks, m].to(F), v[ks, m].to(F)
            s = scale * (qh @ kh.t())
            es = U * (d + 3) * scale * (qh.abs() @ kh.abs().t())
            if table is not None:
                s = s + table[:, n].to(F)[which]
            s = s.masked_fill(~see, -math.inf)
            top = s.amax(1, keepdim=True)
            top = torch.where(top == -math.inf, torch.zeros_like(top), top)
            x = (s - top).exp()
            l = x.sum(1, keepdim=True)
            p = x / torch.where(l > 0, l, torch.ones_like(l))
            mag = torch.where(s.isinf(), torch.zeros_like(s), s).abs()
            lm = torch.log(l.clamp(min=1e-300)).abs() + top.abs()
            ep = es + es.amax(1, keepdim=True) + 8 * U * (mag + mag.amax(1, keepdim=True) + lm) + (b + 32) * U
            ep = ep * (p > 0)
            o = p @ vh
            po = ((h + ep + (b + 8) * U) * p) @ vh.abs() + ((ep * p).sum(1, keepdim=True)) * (p @ vh.abs())
            eo = po + h * (o.abs() + po)
            out[0][qs, n], out[1][qs, n] = o, eo
            if dout is None:
                continue
            g = dout[qs, n].to(F)
            dvr[0][ks, m] += p.t() @ g
            dvr[1][ks, m] += ((h + ep + (a * H // hk + 8) * U) * p).t() @ g.abs()
            dp = g @ vh.t()
            D = (g * o).sum(1, keepdim=True)
            eD = (g.abs() * (eo + (d + 2) * U * o.abs())).sum(1, keepdim=True)
            edp = (d + 3) * U * (g.abs() @ vh.abs().t())
            ds = p * (dp - D)
            eds = p * (edp + eD + (ep + 4 * U) * (dp - D).abs())
            eds = eds * (1 + ep)
            full = eds + (h + (b + 8) * U) * (ds.abs() + eds)
            dqv = scale * (ds @ kh)
            edq = scale * (full @ kh.abs())
            dq[0][qs, n], dq[1][qs, n] = dqv, edq + (h + 2 * U) * (dqv.abs() + edq)
            dkr[0][ks, m] += scale * (ds.t() @ qh)
            dkr[1][ks, m] += scale * ((full + a * H // hk * U * ds.abs()).t() @ qh.abs())
            if table is not None:
                cnt = table.shape[0]
                dtr[:, n] += torch.bincount(which.flatten(), ds.flatten(), cnt)
                dt[1][:, n] += torch.bincount(which.flatten(), (eds + (a + b + 64) * U * ds.abs()).flatten(), cnt)
    got = {"out": out}
    if dout is not None:
        got["dq"] = dq
        for nm, raw in (("dk", dkr), ("dv", dvr)):
            got[nm] = (raw[0], raw[1] + (h + 2 * U) * (raw[0].abs() + raw[1]))
        if table is not None:
            got["dtable"] = (dtr, dt[1] + tb * (dtr.abs() + dt[1]))
    return got


def _check(got, want, name):
    value, bound = want
    err = (got.to(F) - value).abs()
    assert torch.isfinite(got).all(), name
    bad = err > bound + 1e-37
    assert not bad.any(), f"{name}: {int(bad.sum())} of {bad.numel()} off, worst {float((err / (bound + 1e-37)).max()):.3g} x the bound"


def _cu(lens):
    return torch.tensor([0] + list(lens)).cumsum(0).to(torch.int32).cuda()


def _inputs(seed, dtype, heads, hk, d, ql, kl, table=0, tdtype=None, extra=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g).to(dtype).cuda()  # noqa: E731
    q, k, v = r(sum(ql) + extra, heads, d), r(sum(kl) + extra, hk, d), r(sum(kl) + extra, hk, d)
    dout = r(sum(ql) + extra, heads, d)
    t = (0.8 * torch.randn(table, heads, generator=g)).to(tdtype or dtype).cuda() if table else None
    return q, k, v, dout, t


def _run(q, k, v, dout, ql, kl, table=None, **kw):
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    if table is not None:
        leaves.append(table.detach().requires_grad_())
        kw["bias_table"] = leaves[3]
    out = A.packed_attention(*leaves[:3], _cu(ql), _cu(kl), **kw)
    names = ["dq", "dk", "dv"] + (["dtable"] if table is not None else [])
    return {"out": out.detach(), **dict(zip(names, torch.autograd.grad(out, leaves, dout)))}


# ------------------------------------------------------------------------------------------- on the CPU
def test_bucket_edges():
    for nb, md, both in ((32, 128, True), (32, 128, False), (16, 64, True), (64, 300, False), (8, 5, True), (2, 2, False),
                         (32, 4096, True), (6, 100, True)):
        edges = A.bucket_edges(nb, md, both)
        assert list(edges) == sorted(edges) and edges[-1] <= md
        for n in list(range(0, 3 * min(md, 400))) + [md - 1, md, md + 1, 10 ** 6]:
            assert sum(e <= n for e in edges) == _bucket(-n, nb, md, both), (nb, md, both, n)
    # borders that are exact powers: 16 = 8 x 16^(2/8)
    assert 16 in A.bucket_edges(16, 128, False)
    for bad in ((31, 128, True), (1, 128, False), (66, 128, False), (2, 128, True), (32, 8, True), (32, 5000, True)):
        with pytest.raises(ValueError):
            A.bucket_edges(*bad)


def test_refusals_without_gpu():
    q, k = torch.zeros(4, 4, 32), torch.zeros(4, 2, 32)
    cu = torch.tensor([0, 4], dtype=torch.int32)
    call = lambda *a, **kw: A.packed_attention(*a, **kw)  # noqa: E731
    with pytest.raises(RuntimeError, match="GPU"):
        call(q, k, k, cu)
    with pytest.raises(TypeError, match="q dtype"):
        call(q.half(), k.half(), k.half(), cu)
    with pytest.raises(TypeError, match="k dtype"):
        call(q, k.bfloat16(), k, cu)
    with pytest.raises(ValueError, match="not match"):
        call(q, k, k[:3], cu)
    with pytest.raises(ValueError, match="not match"):
        call(q, k[..., :16], k[..., :16], cu)
    with pytest.raises(ValueError, match="heads"):
        call(q, torch.zeros(4, 3, 32), torch.zeros(4, 3, 32), cu)
    for d in (4, 12, 136):
        with pytest.raises(ValueError, match="head dim"):
            call(*(torch.zeros(4, 2, d),) * 3, cu)
    with pytest.raises(ValueError, match=r"rows, heads, dim"):
        call(q[0], k, k, cu)
    for bad in (cu.long(), cu[None], cu[:0]):
        with pytest.raises(ValueError, match="int32"):
            call(q, k, k, bad)
    with pytest.raises(ValueError, match="sequences"):
        call(q, k, k, cu, torch.tensor([0, 2, 4], dtype=torch.int32))
    for s in (0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(ValueError, match="scale"):
            call(q, k, k, cu, scale=s)


def test_c_entry_refusals():
    import ctypes as C
    from detrpose_amd import _lib
    lib = _lib.load()

    def desc(**kw):
        a = _lib.PackedAttn()
        for n in ("q", "k", "v", "out", "cu_q", "cu_k", "dout", "dq", "dk", "dv", "lse", "ws"):
            setattr(a, n, 4096)   # never dereferenced: the calls end before a launch
        for n in ("q", "k", "v", "o", "g"):
            setattr(a, n + "_row", 64)
            setattr(a, n + "_head", 32)
        a.nseq, a.tq, a.tk, a.heads, a.kv_heads, a.dim, a.scale, a.dtype, a.ws_bytes = 1, 4, 4, 2, 2, 32, 1.0, 1, 1 << 20
        for n, x in kw.items():
            if n == "edge":
                a.edge[:len(x)] = x
            else:
                setattr(a, n, x)
        return a

    table = dict(bias=4096, bias_dtype=0, buckets=4, both=0, dbias=4096, edge=[1, 2, 5])
    bad = [dict(dtype=2), dict(dim=12), dict(dim=136), dict(kv_heads=3), dict(scale=0.0), dict(scale=float("nan")),
           dict(q=4104), dict(k_row=60), dict(v_row=1 << 24), dict(tq=-1), dict(nseq=-1), dict(out=None), dict(k=None),
           dict(cu_q=None), dict(tq=1 << 30), {**table, "edge": [2, 1, 5]}, {**table, "edge": [1, 2, 5000]},
           {**table, "edge": [0, 2, 5]}, {**table, "buckets": 65}, {**table, "bias_dtype": 3}, {**table, "both": 1, "buckets": 3}]
    for kw in bad:
        for fn in (lib.dp_packed_attn_fwd, lib.dp_packed_attn_bwd):
            assert fn(C.byref(desc(**kw)), None) == 1000, kw
    for kw in (dict(lse=None), dict(dout=None), dict(dk=None), dict(ws_bytes=8), dict(dq=4104), {**table, "dbias": None},
               dict(g_row=4)):
        assert lib.dp_packed_attn_bwd(C.byref(desc(**kw)), None) == 1000, kw
    assert lib.dp_packed_attn_fwd(C.byref(desc(tq=0)), None) == 0


# ------------------------------------------------------------------------------------------- on the GPU
# heads, key heads, dim, query lengths, key lengths (None: the same), causal
SHAPES = [
    (1, 1, 8, [1], None, False),
    (8, 8, 32, [18, 60, 1, 0, 33], None, False),
    (4, 2, 64, [130, 1, 257], None, True),
    (6, 2, 40, [65, 31], None, True),
    (5, 1, 80, [40, 100], None, False),
    (8, 1, 128, [129, 7], None, True),
    (4, 4, 96, [64, 128, 3], None, True),
    (8, 2, 64, [1, 1, 1, 1], [70, 1, 300, 129], True),
    (4, 2, 32, [17, 5, 40], [100, 5, 333], True),
    (2, 1, 128, [50, 20, 9], [3, 0, 9], True),        # more queries than keys: rows that see nothing
    (3, 3, 16, [20, 0, 4], [0, 7, 65], False),        # no keys, no queries
    (2, 2, 24, [i % 6 for i in range(150)], None, True),   # more sequences than a wave has lanes
    (16, 4, 128, [700], None, True),
]


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"h{s[0]}k{s[1]}d{s[2]}n{len(s[3])}q{max(s[3])}")
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_forward_backward(shape, dtype):
    heads, hk, d, ql, kl, causal = shape
    kl = kl or ql
    q, k, v, dout, _ = _inputs(d + len(ql), dtype, heads, hk, d, ql, kl)
    got = _run(q, k, v, dout, ql, kl, causal=causal)
    want = _reference(q, k, v, ql, kl, causal, d ** -0.5, dout=dout)
    for n in want:
        _check(got[n], want[n], n)


# keys cut into parts that are joined: single tokens and chunks over long caches, few long sequences
LONG = [
    (8, 2, 128, [1, 1, 0, 1, 3], [5000, 1, 40, 2311, 700], True, 0),
    (4, 4, 64, [1, 2], [3001, 1500], True, 16),
    (2, 1, 32, [1], [9000], False, 0),
    (8, 2, 128, [200, 3], [4100, 1700], True, 0),
    (4, 2, 64, [300], [2500], False, 32),
    (2, 2, 96, [1300], [1300], True, 0),
    (6, 2, 64, [3, 2100], [10, 2100], True, 8),
]


@pytest.mark.gpu
@pytest.mark.parametrize("shape", LONG, ids=lambda s: f"h{s[0]}k{s[1]}d{s[2]}b{s[6]}q{max(s[3])}k{max(s[4])}")
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_long_keys(shape, dtype):
    heads, hk, d, ql, kl, causal, nb = shape
    q, k, v, dout, t = _inputs(d + nb, dtype, heads, hk, d, ql, kl, nb, extra=5)
    got = _run(q, k, v, dout, ql, kl, t, causal=causal)
    want = _reference(q, k, v, ql, kl, causal, d ** -0.5, t, 128, not causal, dout)
    for n in want:
        _check(got[n], want[n], n)
    n, m = sum(ql), sum(kl)
    out = torch.full_like(q, 3.0)
    with torch.no_grad():
        A.packed_attention(q, k, v, _cu(ql), _cu(kl), causal=causal, bias_table=t, out=out)
    assert torch.equal(out[:n], got["out"][:n]) and (out[n:] == 3).all()
    assert not got["out"][n:].any() and not got["dk"][m:].any() and not got["dv"][m:].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("nb", [0, 8])
def test_hidden_values_with_long_keys(dtype, nb):
    """The last key, seen by the last query alone, is inf: the other queries do not change (their rows
    are computed again key by key, which moves them by roundings only)."""
    for ql, kl in (([3], [3000]), ([150], [3000])):
        q, k, v, _, t = _inputs(12, dtype, 4, 2, 64, ql, kl, nb)
        kw = dict(causal=True, bias_table=t)
        base = A.packed_attention(q, k, v, _cu(ql), _cu(kl), **kw)
        v[-1] = float("inf")
        got = A.packed_attention(q, k, v, _cu(ql), _cu(kl), **kw)
        lim = 4 * HALF[dtype] * base.double().abs() + 2e-5 * (dtype == torch.float32) + 2e-2 * (dtype != torch.float32)
        assert ((got.double() - base.double()).abs() <= lim)[:-1].all()
        assert got[-1].isinf().all()


BIASED = [
    (4, 4, 32, [18, 300, 1, 77], None, False, 32, 128, None),
    (4, 2, 64, [200, 65, 129], None, True, 32, 128, None),
    (6, 2, 64, [90, 33], [150, 33], True, 16, 20, True),          # causal with a two-way table
    (2, 2, 128, [140, 10], [100, 50], False, 8, 40, False),       # both directions seen, a one-way table
    (3, 1, 48, [400], None, False, 64, 300, None),
    (2, 1, 32, [5, 1, 3], [40, 200, 3], True, 2, 2, None),
]


@pytest.mark.gpu
@pytest.mark.parametrize("shape", BIASED, ids=lambda s: f"h{s[0]}k{s[1]}d{s[2]}b{s[6]}m{s[7]}")
@pytest.mark.parametrize("dtype,tdtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16),
                                          (torch.bfloat16, torch.float32)], ids=["f32", "bf16", "bf16-f32table"])
def test_bias(shape, dtype, tdtype):
    heads, hk, d, ql, kl, causal, nb, md, both = shape
    kl = kl or ql
    q, k, v, dout, t = _inputs(d + nb, dtype, heads, hk, d, ql, kl, nb, tdtype)
    got = _run(q, k, v, dout, ql, kl, t, causal=causal, max_distance=md, bidirectional=both, scale=0.3)
    want = _reference(q, k, v, ql, kl, causal, 0.3, t, md, not causal if both is None else both, dout)
    for n in want:
        _check(got[n], want[n], n)


@pytest.mark.gpu
def test_gradients_against_differences():
    """Central differences of the f32 operator along random directions, step 2^-7 of values of order 1: the
    loss is about 10, its f32 rounding over the step 10 x 2^-24 x 64 x sqrt(terms) ~ 1e-3, the third
    derivative's share 2^-14 of the gradient."""
    ql, kl = [9, 30], [20, 30]
    q, k, v, dout, t = _inputs(3, torch.float32, 4, 2, 32, ql, kl, 8)
    kw = dict(causal=True, max_distance=16)
    got = _run(q, k, v, dout, ql, kl, t, **kw)
    loss = lambda a: (A.packed_attention(*a[:3], _cu(ql), _cu(kl), bias_table=a[3], **kw).double() * dout.double()).sum()  # noqa: E731
    g = torch.Generator().manual_seed(1)
    for i, n in enumerate(("dq", "dk", "dv", "dtable")):
        x = [q, k, v, t]
        way = torch.randn(x[i].shape, generator=g).cuda()
        way /= way.norm()
        h = 2.0 ** -5
        up, dn = list(x), list(x)
        up[i], dn[i] = x[i] + h * way, x[i] - h * way
        num = ((loss(up) - loss(dn)) / (2 * h)).item()
        ana = (got[n].double() * way.double()).sum().item()
        assert abs(num - ana) < 5e-3 * max(1.0, abs(ana)), (n, num, ana)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_strides(dtype):
    """Slices of one fused projection, a cache laid out head first, rows that are no 16-byte pieces, one
    gradient row for all: the same bits as contiguous tensors."""
    ql = [33, 70, 1]
    g = torch.Generator().manual_seed(2)
    qkv = torch.randn(104, (4 + 2 + 2) * 40, generator=g).to(dtype).cuda()
    q, k, v = (t.unflatten(1, (-1, 40)) for t in qkv.split([160, 80, 80], 1))
    dout = torch.randn(104, 4, 40, generator=g).to(dtype).cuda()
    base = _run(q.contiguous(), k.contiguous(), v.contiguous(), dout, ql, ql, causal=True)
    odd = torch.zeros(104, 2, 43, dtype=dtype, device="cuda")
    odd[..., 1:41] = k
    first = v.transpose(0, 1).contiguous().transpose(0, 1)
    for a, b, c in ((q, k, v), (q, odd[..., 1:41], first)):
        got = _run(a, b, c, dout, ql, ql, causal=True)
        for n in base:
            assert torch.equal(got[n], base[n]), n
    one = _run(q, k, v, dout[:1, :1].expand(104, 4, 40), ql, ql, causal=True)
    two = _run(q, k, v, dout[:1, :1].expand(104, 4, 40).contiguous(), ql, ql, causal=True)
    assert all(torch.equal(one[n], two[n]) for n in one)
    cu = torch.stack([_cu(ql), _cu(ql)], 1)[:, 0]   # strided offsets
    assert torch.equal(A.packed_attention(q, k, v, cu, causal=True), base["out"])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_rows_behind_the_last_sequence(dtype):
    ql, kl = [40, 3], [50, 130]
    q, k, v, dout, t = _inputs(4, dtype, 4, 2, 64, ql, kl, 8, extra=150)
    n, m = sum(ql), sum(kl)
    for x in (q, dout):
        x[n:] = float("nan")
    for x in (k, v):
        x[m:] = float("nan")
    got = _run(q, k, v, dout, ql, kl, t, max_distance=30)
    clean = _run(q[:n], k[:m], v[:m], dout[:n], ql, kl, t, max_distance=30)
    for name, rows in (("out", n), ("dq", n), ("dk", m), ("dv", m)):
        assert torch.equal(got[name][:rows], clean[name]), name
        assert not got[name][rows:].any() and got[name][rows:].shape[0] == 150, name
    assert torch.equal(got["dtable"], clean["dtable"])
    out = torch.full_like(q, 7.0)
    with torch.no_grad():
        same = A.packed_attention(q, k, v, _cu(ql), _cu(kl), out=out, bias_table=t, max_distance=30)
    assert same is out and torch.equal(out[:n], clean["out"]) and (out[n:] == 7).all()
    # no sequence at all, and offsets past the rows: cut there
    none = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert not A.packed_attention(q, k, v, none).any()
    far = torch.tensor([0, n, 10 ** 9], dtype=torch.int32, device="cuda")
    kfar = torch.tensor([0, m, 10 ** 9], dtype=torch.int32, device="cuda")
    cut = A.packed_attention(q[:n + 2].nan_to_num(), k[:m + 5].nan_to_num(), v[:m + 5].nan_to_num(), far, kfar)
    same = A.packed_attention(q[:n + 2].nan_to_num(), k[:m + 5].nan_to_num(), v[:m + 5].nan_to_num(),
                              _cu([n, 2]), _cu([m, 5]))
    assert torch.equal(cut, same)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_hidden_values(dtype, value):
    """What causal order hides, or belongs to another sequence, does not reach a query."""
    ql = [100, 140]
    q, k, v, _, _ = _inputs(5, dtype, 4, 2, 64, ql, ql)
    cu = _cu(ql)
    base = A.packed_attention(q, k, v, cu, causal=True)
    for bad in ("k", "v", "both"):
        k2, v2 = k.clone(), v.clone()
        if bad != "v":
            k2[70] = value
        if bad != "k":
            v2[70, :, 5] = value
        got = A.packed_attention(q, k2, v2, cu, causal=True)
        # the tile's other rows are computed again key by key: the same value within f32 and one rounding
        lim = 4 * HALF[dtype] * base.double().abs() + 2e-5 * (dtype == torch.float32) + 2e-2 * (dtype != torch.float32)
        assert ((got.double() - base.double()).abs() <= lim)[:70].all(), bad
        assert torch.equal(got[100:], base[100:]), bad
        if bad != "k":
            assert not torch.isfinite(got[70:100, :, 5]).any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_bias_of_extreme_values(dtype):
    """A bucket of -inf hides its keys, a table of -inf everything; one of the lowest value of the type
    leaves equal weights where nothing else is seen."""
    ql = [70]
    q, k, v, dout, t = _inputs(6, dtype, 2, 2, 32, ql, ql, 4)
    t[0] = -math.inf                                     # the query's own key and those behind it
    kw = dict(max_distance=3, bidirectional=False)
    got = _run(q, k, v, dout, ql, ql, t, causal=True, **kw)
    want = _reference(q, k, v, ql, ql, True, 32 ** -0.5, t, 3, False, dout)
    for n in want:
        _check(got[n], want[n], n)
    assert not got["out"][0].any()                       # the first query sees only its own key
    none = _run(q, k, v, dout, ql, ql, torch.full_like(t, -math.inf), **kw)
    assert all(not x.any() for x in none.values())
    low = _run(q, k, v, dout, ql, ql, torch.full_like(t, torch.finfo(dtype).min), **kw)["out"]
    mean = v.double().mean(0)
    assert ((low.double() - mean).abs() <= HALF[dtype] * (2 * mean.abs() + v.double().abs().mean(0)) + 80 * U).all()


@pytest.mark.gpu
def test_large_scores():
    """One key far above the others, and all scores far below zero."""
    q, k, v, _, _ = _inputs(7, torch.bfloat16, 2, 1, 64, [200], [200])
    k[:] = -k.abs()
    q[:] = q.abs() * 30
    k[77] = 3.0
    want = _reference(q, k, v, [200], [200], False, 1.0)
    _check(A.packed_attention(q, k, v, _cu([200]), scale=1.0), want["out"], "out")


@pytest.mark.gpu
def test_equal_bits_and_streams():
    """Repeated, on another stream, and with other sequences beside it, a result has the same bits."""
    ql = [200, 77]
    q, k, v, dout, t = _inputs(8, torch.bfloat16, 8, 2, 64, ql, ql, 32)
    base = _run(q, k, v, dout, ql, ql, t, causal=True)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        other = _run(q, k, v, dout, ql, ql, t, causal=True)
    s.synchronize()
    for n in base:
        assert torch.equal(base[n], other[n]), n
    alone = _run(q[200:], k[200:], v[200:], dout[200:], ql[1:], ql[1:], t, causal=True)
    for n in ("out", "dq", "dk", "dv"):
        assert torch.equal(alone[n], base[n][200:]), n


@pytest.mark.gpu
def test_captured_and_replayed_with_other_lengths():
    """Two graphs, forward and backward, replayed in turn on new inputs and new lengths."""
    total = 300
    g = torch.Generator().manual_seed(9)
    new = lambda h: torch.randn(total, h, 64, generator=g).bfloat16().cuda()  # noqa: E731
    q, k, v, dout = new(4), new(2), new(2), new(4)
    t = torch.randn(16, 4, generator=g).cuda()
    cu = _cu([100, 150, 50])

    def step(causal):
        a = [x.detach().requires_grad_() for x in (q, k, v, t)]
        o = A.packed_attention(*a[:3], cu, causal=causal, bias_table=a[3], max_distance=40)
        return (o.detach(), *torch.autograd.grad(o, a, dout))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(True), step(False)
    torch.cuda.current_stream().wait_stream(s)
    graphs, outs = [], []
    for causal in (True, False):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(causal))
        graphs.append(graph)
    for lens in ([100, 150, 50], [1, 0, 299], [300, 0, 0], [10, 20, 30]):
        cu.copy_(_cu(lens))
        for x in (q, k, v, dout):
            x.copy_(torch.randn(x.shape, generator=g))
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for causal, got in zip((True, False), outs):
            for i, (x, y) in enumerate(zip(got, step(causal))):
                assert torch.equal(x, y), (lens, causal, i)


@pytest.mark.gpu
def test_gpu_refusals():
    q, k, v, _, t = _inputs(10, torch.bfloat16, 4, 2, 64, [5], [5], 8)
    cu = _cu([5])
    with pytest.raises(RuntimeError, match="same GPU"):
        A.packed_attention(q, k, v, cu.cpu())
    with pytest.raises(ValueError, match="bias_table"):
        A.packed_attention(q, k, v, cu, bias_table=t[:, :3])
    with pytest.raises(TypeError, match="bias_table"):
        A.packed_attention(q, k, v, cu, bias_table=t.half())
    with pytest.raises(ValueError, match="max_distance"):
        A.packed_attention(q, k, v, cu, bias_table=t, max_distance=1)
    with pytest.raises(ValueError, match="out"):
        A.packed_attention(q, k, v, cu, out=torch.empty_like(q)[:3])
    with pytest.raises(RuntimeError, match="no gradient"):
        A.packed_attention(q.requires_grad_(), k, v, cu, out=torch.empty_like(q))


@pytest.mark.gpu
def test_only_some_gradients():
    ql = [30]
    q, k, v, dout, t = _inputs(11, torch.bfloat16, 2, 2, 32, ql, ql, 8)
    full = _run(q, k, v, dout, ql, ql, t)
    v.requires_grad_()
    out = A.packed_attention(q, k, v, _cu(ql), bias_table=t)
    assert torch.equal(torch.autograd.grad(out, v, dout)[0], full["dv"])
    with torch.no_grad():
        assert not A.packed_attention(q, k, v, _cu(ql), bias_table=t).requires_grad


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_strides_of_dimensions_of_one(dtype):
    """One row or one head: whatever stride that dimension has, the rows are read and written."""
    e = 16 // torch.empty(0, dtype=dtype).element_size()
    base = torch.randn(1 << 16, generator=torch.Generator().manual_seed(3)).to(dtype).cuda()
    row = lambda h: base.as_strided((1, h, 32), (3 * e + 1, 32, 1))  # noqa: E731
    head = lambda n: base.as_strided((n, 1, 32), (64, 5, 1), 64 * e)  # noqa: E731
    far = base.as_strided((1, 2, 32), (1 << 30, 32, 1))
    for q, k in ((row(4), row(2)), (head(50), head(50)), (far, far)):
        lens = [q.shape[0]]
        dout = torch.ones_like(q)
        got, want = _run(q, k, k, dout, lens, lens), _run(q.clone(), k.clone(), k.clone(), dout, lens, lens)
        assert all(torch.equal(got[n], want[n]) for n in want)
        out = torch.zeros(1 << 16, device="cuda", dtype=dtype).as_strided(q.shape, q.stride())
        with torch.no_grad():
            A.packed_attention(q, k, k, _cu(lens), out=out)
        assert torch.equal(out, want["out"])


@pytest.mark.gpu
def test_out_apart_from_what_is_read():
    """out= across an input, or across itself, is refused; a tensor that autograd holds is known as changed."""
    q, k, v, _, _ = _inputs(13, torch.float32, 2, 2, 32, [6], [6])
    cu = _cu([6])
    for bad in (q, k, v):
        with pytest.raises(ValueError, match="lies across"):
            A.packed_attention(q, k, v, cu, out=bad)
    with pytest.raises(ValueError, match="lies across k"):
        both = torch.zeros(6, 4, 32, device="cuda")
        A.packed_attention(q, both[:, :2], v, cu, out=both[:, 2:])
    flat = torch.zeros(4096, device="cuda")
    for strides in ((0, 32, 1), (64, 0, 1), (32, 32, 1), (64, 16, 1)):
        with pytest.raises(ValueError, match="overlap"):
            A.packed_attention(q, k, v, cu, out=flat.as_strided((6, 2, 32), strides))
    want = A.packed_attention(q, k, v, cu)
    for strides in ((32, 192, 1), (128, 32, 1), (64, 32, 1)):   # head first, gaps, plain
        assert torch.equal(A.packed_attention(q, k, v, cu, out=flat.as_strided((6, 2, 32), strides)), want)
    x = torch.ones(6, 2, 32, device="cuda", requires_grad=True)
    out = torch.ones(6, 2, 32, device="cuda")
    y = (x * out).sum()
    A.packed_attention(q, k, v, cu, out=out)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.backward()


def test_two_way_buckets_need_two_a_direction():
    import ctypes as C
    from detrpose_amd import _lib
    a = _lib.PackedAttn()
    for n in ("q", "k", "v", "out", "cu_q", "cu_k", "bias"):
        setattr(a, n, 4096)   # never dereferenced
    for n in ("q", "k", "v", "o"):
        setattr(a, n + "_row", 64)
        setattr(a, n + "_head", 32)
    a.nseq, a.tq, a.tk, a.heads, a.kv_heads, a.dim, a.scale, a.dtype = 1, 4, 4, 2, 2, 32, 1.0, 1
    a.buckets, a.both = 2, 1
    assert _lib.load().dp_packed_attn_fwd(C.byref(a), None) == 1000
    # more blocks than a grid takes threads for
    a.bias, a.nseq, a.tq, a.tk, a.heads, a.kv_heads = None, 1 << 24, 1 << 24, 1 << 24, 2, 2
    a.ws_bytes, a.ws = 1 << 60, 4096
    assert _lib.load().dp_packed_attn_fwd(C.byref(a), None) == 1000


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("lens", [[150], [1, 300], [40, 2100]], ids=str)
def test_where_nan_is_seen(dtype, lens):
    """NaN or inf in q, k, v: exactly the outputs that see one are not finite, however many rows do."""
    n = sum(lens)
    for case in ("q", "k", "v", "all", "column", "late"):
        q, k, v, _, _ = _inputs(14, dtype, 2, 1, 64, lens, lens)
        want = torch.zeros(n, 2, 64, dtype=torch.bool, device="cuda")
        s0 = n - lens[-1]
        if case == "q":
            q[n - 5, 1] = float("nan")
            want[n - 5, 1] = True
        elif case == "k":
            k[s0] = float("nan")
            want[s0:] = True
        elif case == "v":
            v[n - 30] = float("inf")
            want[n - 30:] = True
        elif case == "all":
            q[:], k[:], v[:] = (float("nan"),) * 3
            want[:] = True
        elif case == "column":
            v[:, :, 9] = float("nan")
            want[:, :, 9] = True
        else:
            v[s0 + 100:, :, 3] = float("nan")
            k[s0 + 120:] = float("inf")
            want[s0 + 100:, :, 3] = True
            want[s0 + 120:] = True
        got = A.packed_attention(q, k, v, _cu(lens), causal=True)
        if case == "late":   # q k is inf or NaN by its signs: -inf hides the key again
            got, want = got[:s0 + 120], want[:s0 + 120]
        assert torch.equal(~torch.isfinite(got), want), case


# dk and dv in shares that begin and end anywhere in a tile's walk: many key heads, so few shares a head
SHARES = [
    (32, 32, 32, [700, 1, 260, 0, 90], None, True, 0),
    (32, 32, 128, [400, 33, 129], None, True, 0),
    (64, 32, 64, [300, 7, 500], [500, 0, 400], True, 8),       # queries over more, no and fewer keys
    (32, 32, 64, [257, 100], [130, 513], False, 0),
    (64, 64, 16, [(i * 37) % 90 for i in range(150)], None, True, 0),
]


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHARES, ids=lambda s: f"h{s[0]}k{s[1]}d{s[2]}n{len(s[3])}b{s[6]}")
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_shares(shape, dtype):
    heads, hk, d, ql, kl, causal, nb = shape
    kl = kl or ql
    q, k, v, dout, t = _inputs(d + nb + len(ql), dtype, heads, hk, d, ql, kl, nb, extra=140)
    got = _run(q, k, v, dout, ql, kl, t, causal=causal)
    want = _reference(q, k, v, ql, kl, causal, d ** -0.5, t, 128, not causal, dout)
    for n in want:
        _check(got[n], want[n], n)
    again = _run(q, k, v, dout, ql, kl, t, causal=causal)
    assert all(torch.equal(again[n], got[n]) for n in got)


@pytest.mark.gpu
@pytest.mark.parametrize("nb", [0, 8])
def test_no_queries_or_no_keys(nb):
    for n, m in ((0, 150), (150, 0), (0, 0)):
        q, k, v, dout, t = _inputs(15, torch.bfloat16, 4, 2, 64, [n], [m], nb)
        got = _run(q, k, v, dout, [n], [m], t, causal=True)
        assert got["out"].shape == q.shape and got["dk"].shape == k.shape
        assert all(not x.any() for x in got.values())


def test_forward_mode_is_refused():
    """A tangent is never dropped: the call says that it has no forward-mode derivative."""
    from torch.autograd import forward_ad
    q, cu = torch.zeros(4, 2, 32), torch.tensor([0, 4], dtype=torch.int32)
    table = torch.zeros(8, 2)
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        for args, kw in (((dual(q), q, q), {}), ((q, dual(q), q), {}), ((q, q, dual(q)), {}),
                         ((q, q, q), dict(bias_table=dual(table))), ((q, q, q), dict(out=dual(torch.zeros(4, 2, 32)))),
                         ((dual(q), q, q), dict(out=torch.zeros(4, 2, 32)))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                A.packed_attention(*args, cu, **kw)
        with pytest.raises(RuntimeError, match="on the GPU"):   # none of them has a tangent
            A.packed_attention(q, q, q, cu)


def _host_desc(**kw):
    """A descriptor of four rows at addresses that the call never gets to."""
    from detrpose_amd import _lib
    a = _lib.PackedAttn()
    for n in ("q", "k", "v", "out", "cu_q", "cu_k", "dout", "dq", "dk", "dv", "lse", "ws"):
        setattr(a, n, 4096)
    for n in ("q", "k", "v", "o", "g"):
        setattr(a, n + "_row", 64)
        setattr(a, n + "_head", 32)
    a.nseq, a.tq, a.tk, a.heads, a.kv_heads, a.dim, a.scale, a.dtype, a.ws_bytes = 1, 4, 4, 2, 2, 32, 1.0, 1, 1 << 60
    for n, x in kw.items():
        setattr(a, n, x)
    return a


def test_offsets_are_needed_without_sequences():
    import ctypes as C
    from detrpose_amd import _lib
    lib = _lib.load()
    for kw in (dict(cu_q=None), dict(cu_k=None), dict(cu_q=None, cu_k=None)):
        for fill in (0, 1):
            for fn in (lib.dp_packed_attn_fwd, lib.dp_packed_attn_bwd):
                assert fn(C.byref(_host_desc(nseq=0, fill_tail=fill, **kw)), None) == 1000
                assert b"no sequence offsets" in lib.dp_last_error()
    assert lib.dp_packed_attn_fwd(C.byref(_host_desc(nseq=0, tq=0, cu_q=None, cu_k=None)), None) == 0


def test_grids_of_the_backward():
    """A grid of 2^32 threads is refused before anything is launched, that of the keys' join too."""
    import ctypes as C
    from detrpose_amd import _lib
    lib = _lib.load()
    many = dict(nseq=1 << 20, tq=1 << 16, kv_heads=1, heads=1)
    for kw in (dict(dim=128, tk=1 << 27), dict(dim=64, tk=1 << 28), dict(dim=8, tk=1 << 29),
               dict(dim=8, tk=1 << 27, heads=4, kv_heads=4)):
        assert lib.dp_packed_attn_bwd(C.byref(_host_desc(**{**many, **kw})), None) == 1000, kw
        assert b"too many tiles" in lib.dp_last_error(), kw


# A bias that is the same everywhere changes no weight. With q or k of zeros every score is exactly the bias, so the
# reference with a table of zeros is the answer, to the same bounds, however large the bias is: the scores'
# differences and the exponentials carry no error of its size.
ALIKE = [(2, 2, 32, [70], [70], True), (4, 2, 64, [33, 5], [200, 1], False), (4, 1, 128, [300, 1], [300, 40], True)]


def _alike(dtype, heads, hk, d, ql, kl, causal, bias):
    q, k, v, dout, t = _inputs(21, dtype, heads, hk, d, ql, kl, 8)
    for zero in ("q", "k"):
        x = {"q": q, "k": k, zero: torch.zeros_like(q if zero == "q" else k)}
        want = _reference(x["q"], x["k"], v, ql, kl, causal, d ** -0.5, torch.zeros_like(t), 128, not causal, dout)
        got = _run(x["q"], x["k"], v, dout, ql, kl, torch.full_like(t, bias), causal=causal)
        for n in want:
            _check(got[n], want[n], (zero, n))


@pytest.mark.gpu
@pytest.mark.parametrize("shape", ALIKE, ids=lambda s: f"h{s[0]}k{s[1]}d{s[2]}")
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("bias", [-1e4, -1e9, "lowest", 1e6])
def test_gradients_under_a_large_bias(shape, dtype, bias):
    """Weights and their gradients where all that a query sees has one bias, small or as low as the type goes."""
    _alike(dtype, *shape, torch.finfo(dtype).min if bias == "lowest" else bias)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_gradients_beside_the_lowest_bias(dtype):
    """The lowest value hides as -inf does what stands beside other keys."""
    ql = [150, 3]
    q, k, v, dout, t = _inputs(22, dtype, 4, 2, 64, ql, ql, 8)
    t[2:] = -math.inf
    want = _reference(q, k, v, ql, ql, True, 0.125, t, 20, False, dout)
    t[2:] = torch.finfo(dtype).min
    got = _run(q, k, v, dout, ql, ql, t, causal=True, max_distance=20)
    for n in want:
        _check(got[n], want[n], n)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(4, 2, 64, [1, 2], [5000, 1300], True), (2, 1, 128, [3], [9001], True),
                                   (4, 4, 32, [200, 3], [4100, 1700], False)], ids=lambda s: f"h{s[0]}k{s[1]}d{s[2]}")
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("bias", [-1e4, "lowest", 1e6])
def test_cut_keys_under_a_large_bias(shape, dtype, bias):
    """Few queries over many keys, which are cut into parts of unequal length: each part weighs as its keys do."""
    _alike(dtype, *shape, torch.finfo(dtype).min if bias == "lowest" else bias)
    heads, hk, d, ql, kl, causal = shape
    q, k, v, _, t = _inputs(23, dtype, heads, hk, d, ql, kl, 8)
    v[kl[0] - 60:kl[0]] += 30                                # in the last part of the first sequence
    q.zero_()
    want = _reference(q, k, v, ql, kl, causal, d ** -0.5, torch.zeros_like(t), 128, not causal)
    t.fill_(torch.finfo(dtype).min if bias == "lowest" else bias)
    _check(A.packed_attention(q, k, v, _cu(ql), _cu(kl), causal=causal, bias_table=t), want["out"], "out")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_bias_without_lse_lo(dtype, monkeypatch):
    """A caller of the C entries may leave lse_lo out: ordinary biases keep their bounds."""
    desc = A._desc

    def without(*args):
        a = desc(*args)
        a.lse_lo = None
        return a
    monkeypatch.setattr(A, "_desc", without)
    ql, kl = [130, 1, 20], [200, 300, 20]
    q, k, v, dout, t = _inputs(24, dtype, 4, 2, 64, ql, kl, 8)
    got = _run(q, k, v, dout, ql, kl, t, causal=True)
    want = _reference(q, k, v, ql, kl, True, 0.125, t, 128, False, dout)
    for n in want:
        _check(got[n], want[n], n)


def test_lse_lo_needs_lse():
    import ctypes as C
    from detrpose_amd import _lib
    lib = _lib.load()
    for fn in (lib.dp_packed_attn_fwd, lib.dp_packed_attn_bwd):
        assert fn(C.byref(_host_desc(lse=None, lse_lo=4096)), None) == 1000
        assert b"lse_lo" in lib.dp_last_error()
