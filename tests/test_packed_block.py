"""Blocks of a transformer over packed sequences, from the operators together: the norm with the residual's
addition, attention with grouped heads and a bias table, the gradients' clipping.

Tolerances are relative to a tensor's norm. A step is a chain of about 20 stages from the input to a gradient (per
block and direction: norm, projection, attention, projection, norm, two products). In f32 a stage errs by
its sums' terms x 2^-24 at most, 512 x 2^-24 = 3e-5, so 20 of them by 6e-4; in bf16 each stage rounds its
result by 2^-8 at most, 20 x 2^-8 = 0.08. Scores of order 1 and norms over 64 elements pass errors on by
factors about 1: 1e-3 and 0.1 allow 1.3 to 1.6 for them."""
import pytest
import torch

from detrpose_amd import attention as A
from detrpose_amd import gradients as G
from detrpose_amd import norm as N

pytestmark = pytest.mark.gpu

HEADS, KV, DIM, WIDE, BUCKETS, FAR = 4, 2, 16, 64, 16, 40
TOL = {torch.float32: 1e-3, torch.bfloat16: 0.1}


def _parameters(seed, dtype, blocks=2):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: (torch.randn(*s, generator=g) * s[0] ** -0.5).to(dtype).cuda()  # noqa: E731
    p = []
    for _ in range(blocks):
        p += [1 + 0.1 * r(WIDE), r(WIDE, (HEADS + 2 * KV) * DIM), r(BUCKETS, HEADS), r(HEADS * DIM, WIDE),
              1 + 0.1 * r(WIDE), r(WIDE, 2 * WIDE), r(2 * WIDE, WIDE)]
    return p


def _blocks(x, p, norm, attend):
    r = None
    for i in range(0, len(p), 7):
        n1, qkv, table, proj, n2, up, down = p[i:i + 7]
        y, r = norm(x, n1, torch.zeros_like(x) if r is None else r)
        q, k, v = (t.unflatten(1, (-1, DIM)) for t in (y @ qkv).split([HEADS * DIM, KV * DIM, KV * DIM], 1))
        y, r = norm(attend(q, k, v, table).flatten(1) @ proj, n2, r)
        x = torch.tanh(y @ up) @ down
    return x + r


def _plain(x, p, lens, causal):
    def norm(x, w, r):
        r = x + r
        return r * (r.pow(2).mean(-1, keepdim=True) + 1e-6).rsqrt() * w, r

    def attend(q, k, v, table):
        out, at = [], 0
        edges = torch.tensor(A.bucket_edges(BUCKETS, FAR, not causal), device=q.device)
        for n in lens:
            a, b, c = q[at:at + n], k[at:at + n], v[at:at + n]
            at += n
            rel = torch.arange(n, device=q.device)[None] - torch.arange(n, device=q.device)[:, None]
            dist = rel.abs() if not causal else (-rel).clamp(min=0)
            which = torch.bucketize(dist, edges, right=True) + (BUCKETS // 2 * (rel > 0) if not causal else 0)
            s = torch.einsum("ihd,jhd->hij", a, b.repeat_interleave(HEADS // KV, 1)) * DIM ** -0.5
            s = s + table[which].permute(2, 0, 1)
            if causal:
                s = s.masked_fill(rel > 0, -torch.inf)
            out.append(torch.einsum("hij,jhd->ihd", s.softmax(-1), c.repeat_interleave(HEADS // KV, 1)))
        out.append(torch.zeros_like(q[at:]))
        return torch.cat(out)

    return _blocks(x, p, norm, attend)


def _own(x, p, cu, causal):
    return _blocks(x, p, lambda x, w, r: N.rms_norm(x, w, residual=r),
                   lambda q, k, v, t: A.packed_attention(q, k, v, cu, causal=causal, bias_table=t, max_distance=FAR))


def _cu(lens):
    return torch.tensor([0] + list(lens)).cumsum(0).int().cuda()


def _near(a, b, tol, name):
    err = (a.double() - b).norm() / b.norm()
    assert err <= tol, f"{name}: {float(err):.3g}"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("causal", [False, True])
def test_training_step(dtype, causal):
    """Loss, gradients and clipped gradients of two blocks; a padded batch: rows behind the last sequence."""
    lens, pad = [60, 1, 18, 0, 101], 13
    n = sum(lens)
    g = torch.Generator().manual_seed(1)
    x, way = torch.randn(n + pad, WIDE, generator=g).to(dtype).cuda(), torch.randn(n + pad, WIDE, generator=g).cuda()
    way[n:] = 0
    p = [torch.nn.Parameter(t) for t in _parameters(2, dtype)]
    out = _own(x, p, _cu(lens), causal)
    (out.float() * way).sum().backward()
    ref = [t.detach().double().requires_grad_() for t in p]
    want = _plain(x.double(), ref, lens, causal)
    (want * way.double()).sum().backward()
    _near(out[:n], want[:n].detach(), TOL[dtype], "out")
    for i, (a, b) in enumerate(zip(p, ref)):
        _near(a.grad, b.grad, TOL[dtype], f"parameter {i}")
    before = [t.grad.double().clone() for t in p]
    true = torch.cat([t.flatten() for t in before]).norm()
    flat = torch.empty(sum(t.numel() for t in p), device="cuda", dtype=torch.float32)
    norm = G.clip_grad_norm_(p, 1.0, out=flat)
    assert abs(norm.double() - true) <= 1e-6 * true
    _near(flat, torch.cat([t.flatten() for t in before]) / (true + 1e-6), 1e-6, "gathered")
    G.clip_grad_norm_(p, 1.0)
    for t, b in zip(p, before):
        _near(t.grad, b / (true + 1e-6), 2.0 ** -23 if dtype == torch.float32 else 2.0 ** -8, "clipped")


def test_captured_step_on_two_streams():
    """A whole step, forward, backward and clipping, captured and replayed with new lengths between eager steps;
    and two steps at once on two streams. The products are the library's: within the f32 tolerance."""
    total, dtype = 200, torch.float32
    g = torch.Generator().manual_seed(3)
    x, way = (torch.randn(total, WIDE, generator=g).cuda() for _ in range(2))
    base = _parameters(4, dtype)
    cu = _cu([100, 60, 40])

    def step():
        p = [t.detach().requires_grad_() for t in base]
        grads = list(torch.autograd.grad((_own(x, p, cu, True) * way).sum(), p))
        return G.clip_grad_norm_(grads, 1.0), grads

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm, grads = step()
    for lens in ([100, 60, 40], [1, 0, 199], [200, 0, 0], [20, 5, 3]):
        cu.copy_(_cu(lens))
        x.copy_(torch.randn(total, WIDE, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        n0, g0 = step()
        assert abs(n0 - norm) <= 1e-3 * n0
        for a, b in zip(grads, g0):
            _near(a, b.double(), 1e-3, lens)
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        n1, g1 = step()
    n2, g2 = step()
    torch.cuda.synchronize()
    assert abs(n1 - n2) <= 1e-3 * n2
    for a, b in zip(g1, g2):
        _near(a, b.double(), 1e-3, "streams")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
def test_prompt_chunks_and_tokens(dtype):
    """A causal prompt at once, in chunks and token by token over the keys so far: the same rows."""
    lens = [70, 33]
    n = sum(lens)
    x = torch.randn(n, WIDE, generator=torch.Generator().manual_seed(5)).to(dtype).cuda()
    p = _parameters(6, dtype, 1)
    want = _plain(x.double(), [t.double() for t in p], lens, True)
    with torch.no_grad():
        _near(_own(x, p, _cu(lens), True), want, TOL[dtype], "at once")
        for size in (16, 1):
            cache, got = [[], []], [[], []]
            for at in range(0, max(lens), size):
                part = [x[s + min(at, m):s + min(at + size, m)] for s, m in ((0, lens[0]), (lens[0], lens[1]))]

                def attend(q, k, v, t):
                    a = 0
                    for b, xs in enumerate(part):
                        cache[b].append((k[a:a + len(xs)], v[a:a + len(xs)]))
                        a += len(xs)
                    keys, values = (torch.cat([kv[i] for c in cache for kv in c]) for i in (0, 1))
                    ck = _cu([sum(len(kv[0]) for kv in c) for c in cache])
                    return A.packed_attention(q, keys, values, _cu(map(len, part)), ck, causal=True, bias_table=t,
                                              max_distance=FAR)

                y = _blocks(torch.cat(part), p, lambda a, w, r: N.rms_norm(a, w, residual=r), attend)
                got[0].append(y[:len(part[0])])
                got[1].append(y[len(part[0]):])
            _near(torch.cat(got[0] + got[1]), want, TOL[dtype], size)
