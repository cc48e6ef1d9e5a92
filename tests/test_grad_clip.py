"""Clipping of many gradients by their global norm (detrpose_amd.gradients) against 64-bit sums.

Tolerances. The squares are added in 64 bits and the norm is rounded to f32 once: 2^-24 of it. The
coefficient is rounded to f32 once and each product once: 2 x 2^-24 of the value in f32, 2^-8 more in
bf16."""
import math

import pytest
import torch

from detrpose_amd import gradients as G

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def _set(seed, sizes, dtypes=(torch.float32, torch.bfloat16), level=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(level * torch.randn(n, generator=g)).to(dtypes[i % len(dtypes)]).cuda() for i, n in enumerate(sizes)]


def _norm(ts):
    return math.sqrt(sum(float(t.double().square().sum()) for t in ts))


def _check(got, grads, coef):
    for a, b in zip(got, grads):
        want = b.double() * coef
        assert ((a.double() - want).abs() <= (HALF[a.dtype] * (a.dtype != torch.float32) + 2.1 * 2.0 ** -24) * want.abs()
                + 2.0 ** -149).all()


def test_refusals_without_gpu():
    t = torch.zeros(3)
    with pytest.raises(RuntimeError, match="one GPU"):
        G.clip_grad_norm_([t], 1.0)
    with pytest.raises(ValueError, match="max_norm"):
        G.clip_grad_norm_([t], -1.0)
    with pytest.raises(ValueError, match="max_norm"):
        G.clip_grad_norm_([t], float("nan"))
    with pytest.raises(TypeError, match="dtypes"):
        G.clip_grad_norm_([t.half()], 1.0)
    with pytest.raises(TypeError, match="sparse"):
        G.clip_grad_norm_([t.to_sparse()], 1.0)
    assert G.clip_grad_norm_([], 1.0) == 0
    assert G.clip_grad_norm_([torch.zeros(3, requires_grad=True)], 1.0) == 0   # no .grad yet
    with pytest.raises(ValueError, match="out holds"):
        G.clip_grad_norm_([], 1.0, out=torch.zeros(3))


def test_c_entry_refusals():
    import ctypes as C
    from detrpose_amd import _lib
    lib = _lib.load()
    one, sh = (C.c_void_p * 2)(4096, 8192), (C.c_void_p * 2)(4096, 4100)
    n, dt = (C.c_int64 * 2)(4, 4), (C.c_int32 * 2)(0, 0)
    need = lib.dp_grad_clip_ws_bytes(2)
    call = lambda p, m, w, out=None, k=0: lib.dp_grad_clip(p, n, dt, 2, m, 64, out, k, 0, 64, w, None)  # noqa: E731
    assert call(one, 1.0, need - 1) == 1000 and b"workspace" in lib.dp_last_error()
    assert call(one, -1.0, need) == 1000
    assert call(sh, 1.0, need) == 1000 and b"share memory" in lib.dp_last_error()
    assert call(one, 1.0, need, 4104, 8) == 1000        # the output lies over the first tensor
    assert call(one, 1.0, need, 1 << 20, 7) == 1000 and b"output holds" in lib.dp_last_error()
    assert lib.dp_grad_clip_ws_bytes(0) == 0


SETS = [[1], [7, 1, 300, 8192], [8193, 8191, 5, 16384, 3], [1 + (i * 37) % 900 for i in range(300)], [2_000_003, 17, 65]]


@pytest.mark.gpu
@pytest.mark.parametrize("sizes", SETS, ids=lambda s: f"{len(s)}x{sum(s)}")
@pytest.mark.parametrize("dtypes", [(torch.float32,), (torch.bfloat16,), (torch.float32, torch.bfloat16)],
                         ids=["f32", "bf16", "mixed"])
def test_clip(sizes, dtypes):
    grads = _set(len(sizes), sizes, dtypes, 0.3)
    true = _norm(grads)
    for max_norm in (0.1 * true, 10 * true):
        coef = min(1.0, max_norm / (true + 1e-6))
        mine = [g.clone() for g in grads]
        norm = G.clip_grad_norm_(mine, max_norm)
        assert norm.dtype == torch.float32 and norm.shape == ()
        assert abs(norm.item() - true) <= 1.1 * 2.0 ** -24 * true
        _check(mine, grads, coef)
        for odt in (torch.float32, torch.bfloat16):
            out = torch.full((sum(sizes) + 2,), 7.0, device="cuda", dtype=odt)[1:-1]   # an odd offset
            kept = [g.clone() for g in grads]
            assert torch.equal(G.clip_grad_norm_(kept, max_norm, out=out), norm)
            assert all(torch.equal(a, b) for a, b in zip(kept, grads))
            _check(out.split(sizes), grads, coef)


@pytest.mark.gpu
def test_offsets_empty_and_parameters():
    base = torch.randn(1000, device="cuda")
    views = [base[1:4], base[4:4], base[5:700], base[701:]]          # odd offsets, one of no elements
    ref = [v.clone() for v in views]
    true = _norm(ref)
    gap = base[700].clone()
    G.clip_grad_norm_(views, 0.5 * true)
    _check(views, ref, 0.5 * true / (true + 1e-6))
    assert base[700] == gap
    p = [torch.nn.Parameter(torch.zeros(5, device="cuda")) for _ in range(3)]
    p[0].grad, p[2].grad = torch.full((5,), 2.0, device="cuda"), torch.full((5,), -1.0, device="cuda")
    n = G.clip_grad_norm_(iter(p), 1.0)
    assert abs(n.item() - 5.0) < 1e-6 and p[1].grad is None
    assert abs(_norm([p[0].grad, p[2].grad]) - 1.0) < 1e-5
    assert G.clip_grad_norm_(torch.zeros(0, device="cuda"), 1.0).item() == 0


@pytest.mark.gpu
def test_layouts_and_refusals():
    w = torch.randn(8, 3, 5, 7, device="cuda").to(memory_format=torch.channels_last)
    ref = w.clone()
    n = _norm([ref])
    G.clip_grad_norm_([w], 0.5 * n)                                   # dense in another order: in place
    _check([w], [ref], 0.5 * n / (n + 1e-6))
    out = torch.empty(w.numel(), device="cuda")
    G.clip_grad_norm_([ref], 0.5 * n, out=out)
    _check([out], [ref.contiguous().flatten()], 0.5 * n / (n + 1e-6))
    with pytest.raises(ValueError, match="one span"):
        G.clip_grad_norm_([torch.zeros(4, 6, device="cuda")[:, :3]], 1.0)
    t = torch.ones(10, device="cuda")
    from detrpose_amd._lib import HipError
    with pytest.raises(HipError, match="share memory"):
        G.clip_grad_norm_([t, t], 1.0)
    with pytest.raises(HipError, match="share memory"):
        G.clip_grad_norm_([t[:5], t[5:]], 1.0, out=t)
    with pytest.raises(ValueError, match="contiguous row"):
        G.clip_grad_norm_([t], 1.0, out=torch.empty(9, device="cuda"))
    with pytest.raises(ValueError, match="contiguous row"):
        G.clip_grad_norm_([t], 1.0, out=torch.empty(20, device="cuda")[::2])
    with pytest.raises(RuntimeError, match="one GPU"):
        G.clip_grad_norm_([t, torch.ones(3)], 1.0)


@pytest.mark.gpu
def test_range_and_unusual_values():
    big = [torch.full((1000,), 1e30, device="cuda"), torch.full((5,), 1e-30, device="cuda")]
    n = G.clip_grad_norm_(big, 1.0)                                   # squares past f32
    true = math.sqrt(1000) * float(torch.tensor(1e30))
    assert abs(n.item() - true) <= 1e-6 * true
    assert abs(_norm(big) - 1.0) < 1e-6
    tiny = [torch.full((1000,), 1e-30, device="cuda")]
    assert abs(G.clip_grad_norm_(tiny, 1.0).item() / (math.sqrt(1000) * 1e-30) - 1) < 1e-6
    assert (tiny[0] == 1e-30).all()
    bad = [torch.ones(3, device="cuda"), torch.tensor([float("nan"), 1.0], device="cuda")]
    assert G.clip_grad_norm_(bad, 1.0).isnan() and bad[0].isnan().all()
    inf = [torch.ones(3, device="cuda"), torch.tensor([float("inf"), 1.0], device="cuda")]
    assert G.clip_grad_norm_(inf, 1.0).isinf() and not inf[0].any() and inf[1][0].isnan()
    z = [torch.ones(7, device="cuda")]
    G.clip_grad_norm_(z, 0.0)
    assert not z[0].any()


@pytest.mark.gpu
def test_captured_and_replayed():
    """One graph of the clipping, replayed on new gradients with eager calls between: equal bits."""
    g = torch.Generator().manual_seed(3)
    grads = _set(1, [50, 9000, 3, 77_777])
    out = torch.empty(sum(t.numel() for t in grads), device="cuda")
    G.clip_grad_norm_(grads, 1.0, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = G.clip_grad_norm_(grads, 1.0, out=out)
    for k in range(4):
        for t in grads:
            t.copy_(torch.randn(t.numel(), generator=g).to(t.dtype))
        graph.replay()
        torch.cuda.synchronize()
        other = torch.empty_like(out)
        assert torch.equal(G.clip_grad_norm_(grads, 1.0, out=other), norm) and torch.equal(out, other), k


@pytest.mark.gpu
def test_autograd_sees_what_was_written():
    """Tensors that a graph holds are known as changed, clipped in place or gathered into."""
    x = torch.ones(9, device="cuda", requires_grad=True)
    for out in (None, torch.ones(9, device="cuda")):
        g = torch.ones(9, device="cuda")
        y = (x * (g if out is None else out)).sum()
        G.clip_grad_norm_([g], 0.5, out=out)
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            y.backward()


def test_frozen_parameters_are_not_gradients():
    """A parameter stands for its .grad whether it asks for one or not: without one it is passed over."""
    from detrpose_amd import build_model
    model, _ = build_model("n")
    frozen = {n: p.detach().clone() for n, p in model.named_parameters() if not p.requires_grad}
    assert {"transformer.up", "transformer.reg_scale"} <= frozen.keys()
    assert G.clip_grad_norm_(model.parameters(), 0.1) == 0            # no gradients yet
    assert G.clip_grad_norm_(model.parameters(), 0.1, out=torch.zeros(0)) == 0
    assert all(torch.equal(p, frozen[n]) for n, p in model.named_parameters() if n in frozen)
    late = torch.ones(3, requires_grad=True)                          # frozen after its backward pass
    late.sum().backward()
    late.requires_grad_(False)
    with pytest.raises(RuntimeError, match="one GPU"):                # its .grad, which is on the CPU
        G.clip_grad_norm_([late, *model.parameters()], 0.1)
    with pytest.raises(ValueError, match="pass parameters or gradients"):
        G.clip_grad_norm_([*model.parameters(), torch.ones(3)], 0.1)


@pytest.mark.gpu
def test_frozen_parameters_of_the_model():
    from detrpose_amd import build_model
    model = build_model("n")[0].cuda()
    model.backbone.requires_grad_(False)
    kept = {n: p.detach().clone() for n, p in model.named_parameters()}
    gen = torch.Generator("cuda").manual_seed(5)
    trained = [p for p in model.parameters() if p.requires_grad]
    assert 0 < len(trained) < len(kept) - 2
    for p in trained:
        p.grad = torch.randn(p.shape, generator=gen, device="cuda")
    ref = [p.grad.clone() for p in trained]
    true = _norm(ref)
    flat = torch.empty(sum(g.numel() for g in ref), device="cuda")
    norm = G.clip_grad_norm_(model.parameters(), 0.5 * true, out=flat)
    assert abs(norm.item() - true) <= 1.1 * 2.0 ** -24 * true
    _check([t.view_as(g) for t, g in zip(flat.split([g.numel() for g in ref]), ref)], ref, 0.5 * true / (true + 1e-6))
    assert torch.equal(G.clip_grad_norm_(model.parameters(), 0.5 * true), norm)
    _check([p.grad for p in trained], ref, 0.5 * true / (true + 1e-6))
    for n, p in model.named_parameters():
        assert torch.equal(p, kept[n]), n
        assert p.requires_grad or p.grad is None, n


def test_norm_of_no_gradients():
    """0 as f32, on the device of the parameters that have no gradient (of out, when it is given)."""
    torch.set_default_dtype(torch.float64)
    try:
        bare = [torch.nn.Parameter(torch.zeros(3, device="meta")) for _ in range(2)]
        n = G.clip_grad_norm_(bare, 1.0)
        assert n.device.type == "meta" and n.dtype == torch.float32 and n.shape == ()
        assert G.clip_grad_norm_(bare, 1.0, out=torch.zeros(0)).device.type == "cpu"
        assert G.clip_grad_norm_([], 1.0).dtype == torch.float32
    finally:
        torch.set_default_dtype(torch.float32)


def test_forward_mode_is_refused():
    """Gradients with a tangent are not clipped behind its back, nor gathered into a tensor with one."""
    from torch.autograd import forward_ad
    g = torch.ones(4)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(torch.ones(4), torch.ones(4))
        for call in (lambda: G.clip_grad_norm_([g, dual], 1.0), lambda: G.clip_grad_norm_([g], 1.0, out=dual)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
