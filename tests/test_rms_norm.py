"""RMS norm with the residual's addition (detrpose_amd.norm) against its definition in 64 bits.

Tolerances. y, dx in bf16: one rounding of the result, 2^-8 of its value, plus f32 work (2^-24 x a
few). r is one rounding of an exact sum of two values. f32: the row sum of c squares in f32 has a
relative error of at most c 2^-24 (all terms positive), half of it in rstd; dweight's terms have any
sign, so its error is bounded by (rows + 8) 2^-24 times the sum of the terms' magnitudes."""
import pytest
import torch

from detrpose_amd import norm as N

EPS = 1e-6
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def _ref(x, w, res, eps=EPS):
    r = x if res is None else (x.double() + res.double()).float().to(x.dtype)
    r64 = r.double()
    rstd = 1 / (r64.square().mean(-1, keepdim=True) + eps).sqrt()
    return r, r64 * rstd * w.double(), rstd


def _close(got, want, rel, scale=None):
    """|got - want| <= rel x max(|want|, scale) everywhere."""
    want = want.double()
    lim = rel * (want.abs() if scale is None else torch.maximum(want.abs(), scale.expand_as(want)))
    bad = (got.double() - want).abs() > lim + 1e-300
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {(got.double() - want).abs().max().item():.3g}"


def test_refusals_without_gpu():
    x = torch.zeros(3, 8)
    w = torch.ones(8)
    with pytest.raises(RuntimeError, match="GPU"):
        N.rms_norm(x, w)
    with pytest.raises(TypeError, match="x dtype"):
        N.rms_norm(x.half(), w)
    with pytest.raises(TypeError, match="weight dtype"):
        N.rms_norm(x, w.bfloat16())
    with pytest.raises(ValueError, match="weight"):
        N.rms_norm(x, torch.ones(7))
    with pytest.raises(ValueError, match="residual"):
        N.rms_norm(x, w, residual=torch.zeros(2, 8))
    with pytest.raises(ValueError, match="residual"):
        N.rms_norm(x, w, residual=torch.zeros(3, 8, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="eps"):
        N.rms_norm(x, w, eps=-1.0)
    with pytest.raises(ValueError, match="rows of 1 to 8192"):
        N.rms_norm(torch.zeros(1, 8193), torch.ones(8193))
    with pytest.raises(ValueError, match="rows of 1"):
        N.rms_norm(torch.zeros(3, 0), torch.ones(0))


def test_c_entry_refusals():
    from detrpose_amd import _lib
    lib = _lib.load()
    p = 4096   # never dereferenced: the calls end before a launch
    assert lib.dp_rms_norm(None, None, None, p, 8, None, 0, p, 0, EPS, 1, 8, 0, None) == 1000
    assert lib.dp_rms_norm(p, p, None, p, 8, None, 0, p, 0, EPS, 1, 8, 0, None) == 1000      # r without res
    assert lib.dp_rms_norm(p, None, None, p, 8, None, 0, p, 1, EPS, 1, 8, 0, None) == 1000   # bf16 weight, f32 x
    assert lib.dp_rms_norm(p, None, None, p, 8, None, 0, p, 0, EPS, 1, 16385, 1, None) == 1000
    assert lib.dp_rms_norm(p, None, None, p, 8, None, 0, p, 0, EPS, 0, 8, 0, None) == 0      # no rows
    need = lib.dp_rms_norm_bwd_ws_floats(100, 300, 1)
    assert need >= 300
    assert lib.dp_rms_norm_bwd(p, p, p, 300, p, p, 300, None, 0, p, 0, p, need - 1, 100, 300, 1, None) == 1000


CASES = [(1, 1), (3, 7), (5, 64), (2, 255), (18, 256), (9, 511), (7, 1000), (4, 1024), (6, 2049), (3, 4100), (2, 8192),
         (1200, 384)]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,c", CASES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("residual", [False, True])
def test_forward_backward(rows, c, dtype, residual):
    g = torch.Generator().manual_seed(rows * 7919 + c)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    x, res = r(rows, c).to(dtype).cuda(), (2 * r(rows, c)).to(dtype).cuda() if residual else None
    wt = dtype if c % 2 else torch.float32
    w = (1 + 0.2 * r(c)).to(wt).cuda()
    dy, dr = r(rows, c).to(dtype).cuda(), r(rows, c).to(dtype).cuda()
    leaves = [t.clone().requires_grad_() for t in (x, w)] + ([res.clone().requires_grad_()] if residual else [])
    got = N.rms_norm(leaves[0], leaves[1], residual=leaves[2] if residual else None, eps=EPS)
    y, rr = got if residual else (got, None)
    grads = torch.autograd.grad([y, rr] if residual else [y], leaves, [dy, dr] if residual else [dy])
    r0, y0, rstd = _ref(x, w, res)
    if residual:
        assert torch.equal(rr, r0)
    h = HALF[dtype]
    f32 = (c + 8) * 2.0 ** -24
    _close(y, y0, h + f32)
    xh = r0.double() * rstd
    wdy = dy.double() * w.double()
    dot = (wdy * xh).mean(-1, keepdim=True)
    dx0 = rstd * (wdy - xh * dot) + (dr.double() if residual else 0)
    # the terms that dx is the difference of, and the dot's own terms
    size = rstd * (wdy.abs() + xh.abs() * (wdy * xh).abs().mean(-1, keepdim=True)) + (dr.double().abs() if residual else 0)
    assert ((grads[0].double() - dx0).abs() <= h * dx0.abs() + 2 * f32 * size).all()
    terms = (dy.double() * xh).abs().sum(0)
    dw0 = (dy.double() * xh).sum(0)
    assert ((grads[1].double() - dw0).abs() <= HALF[wt] * dw0.abs() + ((rows + 8) * 2.0 ** -24 + f32) * terms).all()
    if residual:
        assert torch.equal(grads[2], grads[0])


@pytest.mark.gpu
def test_gradient_against_differences():
    """Central differences of the f32 operator: their own error is the values' rounding over the step
    (2^-24 x |loss| / h, |loss| ~ 10) plus the third derivative (h^2); h = 2^-6."""
    g = torch.Generator().manual_seed(5)
    x, w, res = (torch.randn(4, 33, generator=g).cuda(), torch.rand(33, generator=g).cuda() + 0.5,
                 torch.randn(4, 33, generator=g).cuda())
    cy, cr = torch.randn(4, 33, generator=g).cuda(), torch.randn(4, 33, generator=g).cuda()

    def loss(a, b, c):
        y, r = N.rms_norm(a, b, residual=c, eps=EPS)
        return (y.double() * cy.double()).sum() + (r.double() * cr.double()).sum()

    leaves = [t.clone().requires_grad_() for t in (x, w, res)]
    grads = torch.autograd.grad(loss(*leaves), leaves)
    h = 2.0 ** -6
    for i, at in ((0, (0, 0)), (0, (3, 32)), (0, (2, 17)), (1, (0,)), (1, (32,)), (2, (1, 5))):
        up, dn = [t.clone() for t in (x, w, res)], [t.clone() for t in (x, w, res)]
        up[i][at] += h
        dn[i][at] -= h
        step = (up[i][at] - dn[i][at]).double()
        num = ((loss(*up) - loss(*dn)) / step).item()
        assert abs(num - grads[i][at].item()) < 2e-3 * max(1.0, abs(num)), (i, at, num, grads[i][at].item())


@pytest.mark.gpu
def test_strides_shapes_and_parts():
    """Rows of a wider tensor, odd offsets, leading dimensions, expanded gradients, unused outputs."""
    g = torch.Generator().manual_seed(6)
    wide = torch.randn(6, 5, 301, generator=g).bfloat16().cuda()
    x, res = wide[..., 1:150], wide[..., 150:299]
    w = torch.rand(149, generator=g).cuda()
    y, r = N.rms_norm(x, w, residual=res, eps=EPS)
    r0, y0, _ = _ref(x, w, res)
    assert torch.equal(r, r0)
    _close(y, y0, HALF[torch.bfloat16] + 160 * 2.0 ** -24)
    yt = N.rms_norm(x.transpose(0, 1), w)   # a copy is taken
    assert torch.equal(yt, N.rms_norm(x.contiguous(), w).transpose(0, 1))
    a = x.float().contiguous().requires_grad_()
    N.rms_norm(a, w).sum().backward()       # expanded gradient
    b = x.float().contiguous().requires_grad_()
    N.rms_norm(b, w).backward(torch.ones(6, 5, 149, device="cuda"))
    assert torch.equal(a.grad, b.grad)
    c = x.float().contiguous().requires_grad_()
    q = res.float().contiguous().requires_grad_()
    wg = w.clone().requires_grad_()
    N.rms_norm(c, wg, residual=q)[1].sum().backward()   # only the sum is used
    assert torch.equal(c.grad, torch.ones_like(c)) and torch.equal(q.grad, torch.ones_like(q))
    assert not wg.grad.any()
    e = torch.zeros(0, 149, device="cuda", requires_grad=True)
    wz = w.clone().requires_grad_()
    N.rms_norm(e, wz).sum().backward()
    assert e.grad.shape == (0, 149) and not wz.grad.any()


@pytest.mark.gpu
@pytest.mark.parametrize("rows,c", [(1, 1), (3, 7), (18, 256), (5, 1001), (4, 5120), (2, 8192)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_e4m3(rows, c, dtype):
    """y * scale is the norm within one e4m3 rounding (2^-4 of the value, half the least step 2^-10 of the
    scale) and the f32 work's error; the scale is max |norm| / 448."""
    g = torch.Generator().manual_seed(rows + 31 * c)
    x, res = torch.randn(rows, c, generator=g).to(dtype).cuda(), torch.randn(rows, c, generator=g).to(dtype).cuda()
    w = (1 + 0.2 * torch.randn(c, generator=g)).cuda()
    y, scale, r = N.rms_norm_e4m3(x, w, residual=res, eps=EPS)
    assert y.dtype == torch.float8_e4m3fn and scale.shape == (rows,)
    r0, y0, _ = _ref(x, w, res)
    assert torch.equal(r, r0)
    f32 = (c + 8) * 2.0 ** -24
    s0 = y0.abs().amax(-1) / 448
    _close(scale, s0, f32)
    back = y.double() * scale.double()[:, None]
    assert ((back - y0).abs() <= (2.0 ** -4 + f32) * y0.abs() + 2.0 ** -10 * scale.double()[:, None]).all()
    assert (y.float().abs().amax(-1) == 448).all()
    y2, s2, none = N.rms_norm_e4m3(r0, w, eps=EPS)
    assert none is None and torch.equal(y2.view(torch.uint8), y.view(torch.uint8)) and torch.equal(s2, scale)
    with pytest.raises(RuntimeError, match="no gradient"):
        N.rms_norm_e4m3(x.clone().requires_grad_(), w)


@pytest.mark.gpu
def test_unusual_values():
    w = torch.ones(40, device="cuda")
    x = torch.zeros(4, 40, device="cuda")
    x[1] = 3e38          # the square overflows: rstd is 0
    x[2, 3] = float("nan")
    x[3, 5] = float("inf")
    y = N.rms_norm(x, w, eps=EPS)
    assert not y[0].any() and not y[1].any() and y[2].isnan().all()
    assert y[3, 5].isnan() and not y[3, :5].any()
    y8, s, _ = N.rms_norm_e4m3(x, w, eps=EPS)
    assert not y8[0].float().any() and s[0] == 0 and y8[2].float().isnan().all()


@pytest.mark.gpu
def test_captured_and_replayed():
    """Forward and backward in a graph, replayed on new inputs with eager work between."""
    g = torch.Generator().manual_seed(8)
    x, dy = torch.randn(70, 640, generator=g).bfloat16().cuda(), torch.randn(70, 640, generator=g).bfloat16().cuda()
    w = torch.rand(640, generator=g).cuda()

    def step(a, b, d):
        a, b = a.detach().requires_grad_(), b.detach().requires_grad_()
        y = N.rms_norm(a, b)
        return (y.detach(), *torch.autograd.grad(y, [a, b], d))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(x, w, dy)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(x, w, dy)
    for k in range(4):
        x.copy_(torch.randn(70, 640, generator=g).bfloat16())
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, step(x, w, dy)):
            assert torch.equal(a, b), k


@pytest.mark.gpu
def test_e4m3_rows_below_the_normal_numbers():
    """A norm whose 448th part is no normal f32 keeps finite values: the scale stays at 2^-126, and a value is off
    by at most half the least step 2^-10 of it or 2^-4 of itself, and the f32 product's half step 2^-150."""
    x = torch.randn(6, 300, generator=torch.Generator().manual_seed(4)).cuda()
    for tiny in (1e-36, 1e-38, 1e-40, 1e-42, 1e-44):
        w = torch.full((300,), tiny, device="cuda")
        y, s, _ = N.rms_norm_e4m3(x, w, eps=EPS)
        assert torch.isfinite(y.float()).all() and (s >= 2.0 ** -126).all()
        y0 = x.double() * (x.double().pow(2).mean(-1, keepdim=True) + EPS).rsqrt() * w.double()
        err = (y.double() * s.double()[:, None] - y0).abs()
        lim = (2.0 ** -4 + 310 * 2.0 ** -24) * y0.abs() + 2.0 ** -10 * s.double()[:, None] + 2.0 ** -149
        assert (err <= lim).all(), tiny


@pytest.mark.gpu
def test_same_tensor_twice_and_modes():
    """x as its own residual, with gradients from both uses; no graph in no_grad and inference_mode."""
    x = torch.randn(5, 64, generator=torch.Generator().manual_seed(5)).cuda().requires_grad_()
    w = torch.ones(64, device="cuda", requires_grad=True)
    y, r = N.rms_norm(x, w, residual=x)
    assert torch.equal(r, 2 * x)
    gx, gw = torch.autograd.grad(y.sum() + r.sum(), [x, w])
    x2 = x.detach().clone().requires_grad_()
    y2, r2 = N.rms_norm(2 * x2, w, residual=torch.zeros_like(x2))
    gx2, gw2 = torch.autograd.grad(y2.sum() + r2.sum(), [x2, w])
    assert torch.equal(gx, gx2) and torch.equal(gw, gw2)
    for mode in (torch.no_grad, torch.inference_mode):
        with mode():
            y3, r3 = N.rms_norm(x, w, residual=x)
            y8, s8, r8 = N.rms_norm_e4m3(x, w, residual=x)
        assert torch.equal(y3, y) and not y3.requires_grad and torch.equal(r8, r3)


@pytest.mark.gpu
def test_more_rows_than_a_grid_has_threads():
    """2^32 threads of 256 a row: the rows behind them are computed by a second launch."""
    rows, c = (1 << 24) + 5, 1032
    if torch.cuda.mem_get_info()[0] < 80 << 30:
        pytest.skip("80 GiB of memory")
    x = torch.zeros(rows, c, device="cuda", dtype=torch.bfloat16)
    x[-9:] = torch.randn(9, c, generator=torch.Generator().manual_seed(6)).bfloat16()
    x[0] = x[-1]
    w = torch.linspace(0.5, 2, c, device="cuda")
    y = N.rms_norm(x, w)
    assert torch.equal(y[-9:], N.rms_norm(x[-9:].clone(), w)) and torch.equal(y[0], y[-1])
    assert not y[1000].any() and not y[-10].any()


def test_forward_mode_is_refused():
    """A tangent is never dropped: the calls say that they have no forward-mode derivative."""
    from torch.autograd import forward_ad
    x, w = torch.zeros(3, 8), torch.ones(8)
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        for f in (N.rms_norm, N.rms_norm_e4m3):
            for args in ((dual(x), w), (x, dual(w)), (x, w, dual(x))):
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    f(*args)
