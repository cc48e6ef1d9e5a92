"""Cases of the token-sequence and gradient operators: attention over packed sequences (grouped
heads, causal order, a learned relative position bias by buckets, with gradients), root-mean-square
norm with the residual's addition (with gradients, and with an 8-bit output), and the clipping of
many gradients by their global norm.

A case is a dict of plain values; sequence lengths are a text of comma-separated numbers.
`run` computes a case's plain form with elementary torch operations in 32 bits, or, where `own`
is set, through the framework's entry points."""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
E4M3_MAX = 448.0


def _lens(text):
    return [int(x) for x in text.split(",")]


# ------------------------------------------------------------------------------------- the cases
def _attn(name, dtype, heads, kv_heads, dim, q_lens, k_lens="", causal=False, train=False, buckets=0,
          max_distance=128, fused=False):
    return {"name": name, "op": "attention", "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "q_lens": q_lens, "k_lens": k_lens or q_lens, "causal": causal, "train": train, "buckets": buckets,
            "max_distance": max_distance, "fused": fused}


def _norm(name, dtype, rows, width, residual, form):
    return {"name": name, "op": "norm", "dtype": dtype, "rows": rows, "width": width, "residual": residual, "form": form}


def _clip(name, dtype, tensors, total, max_norm):
    return {"name": name, "op": "clip", "dtype": dtype, "tensors": tensors, "total": total, "max_norm": max_norm}


def listed():
    return [
        # one new token of each of four short sequences: what it takes is latency
        _attn("attention_token", "bf16", 16, 4, 64, "1,1,1,1", "65,130,7,257"),
        # one new token of each of sixteen sequences over long caches of different lengths
        _attn("attention_token_long", "bf16", 32, 8, 128, ",".join(["1"] * 16),
              "32768,20011,16384,12001,9000,8192,7777,6000,4097,4000,3001,2047,1500,1024,333,1"),
        # prompts of different lengths in one pass, q, k and v as slices of one fused projection
        _attn("attention_prompt", "bf16", 32, 8, 128, "4096,2049,1023,517,260,129,1", causal=True, fused=True),
        # a chunk of new tokens of each sequence behind what its cache holds
        _attn("attention_chunk", "bf16", 32, 8, 128, "512,65,17,1", "8192,4001,1025,333", causal=True),
        # a training step's attention over packed sequences, forward and backward
        _attn("attention_train", "bf16", 16, 4, 128, "4096,1537,1024,333,64,1", causal=True, train=True),
        # the token counts of a pose decoder's images (instances x 18 tokens, 20 x 20 map), exact precision
        _attn("attention_train_f32", "f32", 8, 8, 32, "1080,400,396,90,18,18", train=True),
        # an encoder with a learned relative position bias, both directions
        _attn("bias_prompt", "bf16", 16, 16, 64, "2048,1025,511,130,17", buckets=32),
        # its training step, causal, with the gradient of the table
        _attn("bias_train", "bf16", 16, 8, 64, "2048,1111,640,200,31,1", causal=True, train=True, buckets=32),
        # a block's norm in training: the residual stream's sum, its norm, and all gradients
        _norm("norm_train", "bf16", 8192, 4096, True, "train"),
        # serving: the norm before an 8-bit product, each row with its scale
        _norm("norm_e4m3", "bf16", 515, 5120, True, "e4m3"),
        # every gradient of a small pose model: many tensors, most of them tiny
        _clip("clip_small", "f32", 368, 4_100_000, 0.1),
        # the gradients of a large model, in two types
        _clip("clip_large", "mixed", 600, 320_000_000, 1.0),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["token", "chunk", "prompt", "train", "train", "bias", "norm", "clip"])
    if kind in ("norm",):
        form = rng.choice(["train", "e4m3", "forward"])
        width = rng.choice([128, 256, 384, 1000, 1024, 2048, 2560, 4096, 4100, 5120, 8192, _log_int(rng, 33, 8192)])
        return _norm("", rng.choice(["bf16", "bf16", "f32"]), _log_int(rng, 1, max(2, 16_000_000 // width)), width,
                     rng.random() < 0.7, form)
    if kind == "clip":
        total = _log_int(rng, 100_000, 250_000_000)
        return _clip("", rng.choice(["f32", "bf16", "mixed"]), _log_int(rng, 20, 700), total, rng.choice([0.1, 0.5, 1.0]))
    dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
    dim = rng.choice([32, 64, 80, 96, 128])
    kv = rng.choice([2, 4, 8])
    heads = kv * rng.choice([1, 2, 3, 4, 8 if kv < 8 else 4])
    if kind == "token":
        n = _log_int(rng, 1, 64)
        ks = [_log_int(rng, 1, max(2, min(32768, 131072 // n))) for _ in range(n)]
        return _attn("", dtype, heads, kv, dim, ",".join(["1"] * n), ",".join(map(str, ks)))
    most = 4096 if dtype == "bf16" else 1500
    n = _log_int(rng, 1, 8)
    qs = [_log_int(rng, 1, most // (1 if n < 3 else 2)) for _ in range(n)]
    if kind == "chunk":
        qs = [min(q, 512) for q in qs]
        ks = [q + _log_int(rng, 1, 8000 // (1 if n < 4 else 2)) for q in qs]
        return _attn("", dtype, heads, kv, dim, ",".join(map(str, qs)), ",".join(map(str, ks)), causal=True)
    lens = ",".join(map(str, qs))
    if kind == "prompt":
        return _attn("", dtype, heads, kv, dim, lens, causal=rng.random() < 0.7, fused=rng.random() < 0.5)
    heads, kv = min(heads, 16), min(kv, 4) if heads > 16 else kv
    if kind == "train":
        return _attn("", dtype, heads, kv, dim, lens, causal=rng.random() < 0.6, train=True)
    return _attn("", dtype, heads, kv, min(dim, 96), lens, causal=rng.random() < 0.5, train=rng.random() < 0.6,
                 buckets=rng.choice([16, 32, 32, 64]), max_distance=rng.choice([64, 128, 128, 300]))


# ------------------------------------------------------------------------------------- the inputs
def _clip_sizes(case, gen):
    """Tensor sizes as a model's: a few large ones, many small, adding up to `total`."""
    n, total = case["tensors"], case["total"]
    u = torch.exp(torch.rand(n, generator=gen) * 9.0)
    sizes = torch.clamp((u / u.sum() * total).long(), min=1)
    sizes[0] += total - int(sizes.sum())
    return [int(max(1, s)) for s in sizes]


def _cu(lens):
    return torch.tensor([0] + lens).cumsum(0).to(torch.int32).cuda()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(1000 + int(seed))
    s = dict(case)
    if case["op"] == "attention":
        dt = DTYPES[case["dtype"]]
        ql, kl = _lens(case["q_lens"]), _lens(case["k_lens"])
        tq, tk, h, hk, d = sum(ql), sum(kl), case["heads"], case["kv_heads"], case["dim"]
        r = lambda *shape: torch.randn(*shape, generator=gen, device="cuda").to(dt)  # noqa: E731
        if case["fused"]:
            qkv = r(tq, (h + 2 * hk) * d)
            q, k, v = (t.unflatten(1, (-1, d)) for t in qkv.split([h * d, hk * d, hk * d], 1))
        else:
            q, k, v = r(tq, h, d), r(tk, hk, d), r(tk, hk, d)
        s.update(q=q, k=k, v=v, cu_q=_cu(ql), cu_k=_cu(kl), ql=ql, kl=kl)
        if case["buckets"]:
            s["table"] = (torch.randn(case["buckets"], h, generator=gen, device="cuda") * 0.7).to(dt)
        if case["train"]:
            s["dout"] = r(tq, h, d)
            for n in ("q", "k", "v", "table"):
                if n in s:
                    s[n] = s[n].requires_grad_()
    elif case["op"] == "norm":
        dt = DTYPES[case["dtype"]]
        shape = (case["rows"], case["width"])
        r = lambda: torch.randn(*shape, generator=gen, device="cuda").to(dt)  # noqa: E731
        s["x"] = r()
        s["weight"] = 1 + 0.2 * torch.randn(case["width"], generator=gen, device="cuda")
        if case["residual"]:
            s["res"] = (2 * torch.randn(*shape, generator=gen, device="cuda")).to(dt)
        if case["form"] == "train":
            s["dy"] = r()
            if case["residual"]:
                s["dr"] = r()
            for n in ("x", "weight", "res"):
                if n in s:
                    s[n] = s[n].requires_grad_()
    else:
        host = torch.Generator().manual_seed(77)
        sizes = _clip_sizes(case, host)
        flat = torch.randn(sum(sizes), generator=gen, device="cuda")
        level = torch.exp(torch.randn(len(sizes), generator=gen, device="cuda") - 5)
        grads = []
        for i, (g, lv) in enumerate(zip(flat.split(sizes), level)):
            low = case["dtype"] == "bf16" or (case["dtype"] == "mixed" and i % 2 == 0)
            grads.append((g * lv).to(torch.bfloat16 if low else torch.float32))
        s.update(grads=grads, out=torch.empty_like(flat))
    return s


# ------------------------------------------------------------------------------------- one pass
def _edges(buckets, max_distance, both):
    """The least distance of every bucket behind the first one, as whole numbers: the first half of
    the buckets holds one distance each, bucket e + j of the other half (e of them, K in all) begins at
    the least n with n >= e (max_distance / e)^(j / K)."""
    nb = buckets // 2 if both else buckets
    e = nb // 2
    edges = list(range(1, e + 1))
    for j in range(1, nb - e):
        n = e
        while n ** (nb - e) < e ** (nb - e - j) * max_distance ** j:
            n += 1
        edges.append(n)
    return edges


def _buckets(rel, buckets, max_distance, both):
    edges = torch.tensor(_edges(buckets, max_distance, both), device=rel.device)
    n = rel.abs() if both else (-rel).clamp(min=0)
    b = torch.bucketize(n, edges, right=True)
    return b + (rel > 0) * (buckets // 2) if both else b


def _pad(x, cu, longest):
    """Packed rows (T, heads, dim) -> (sequences, heads, longest, dim) in 32 bits, zeros behind each."""
    at = cu[:-1].long()[:, None] + torch.arange(longest, device=x.device)
    ok = at < cu[1:].long()[:, None]
    y = x[at.clamp(max=max(0, x.shape[0] - 1))].float() * ok[..., None, None]
    return y.transpose(1, 2).contiguous()


def _unpad(y, cu, rows, dtype):
    """(sequences, heads, longest, dim) -> packed rows of `dtype`."""
    at = torch.arange(rows, device=y.device)
    seq = torch.bucketize(at, cu[1:].long(), right=True)
    return y[seq, :, at - cu.long()[seq]].to(dtype).contiguous()


def _plain_attention(s):
    q, k, v, cu_q, cu_k = (s[n].detach() for n in ("q", "k", "v", "cu_q", "cu_k"))
    lq, lk, g, scale = max(s["ql"]), max(s["kl"]), s["heads"] // s["kv_heads"], s["dim"] ** -0.5
    qp, kp, vp = _pad(q, cu_q, lq), _pad(k, cu_k, lk), _pad(v, cu_k, lk)
    b, hk, _, d = kp.shape
    qp = qp.view(b, hk, g * lq, d)  # query heads of one key head side by side
    nq, nk = (cu_q[1:] - cu_q[:-1]).long(), (cu_k[1:] - cu_k[:-1]).long()
    pos = torch.arange(lq, device=q.device)[None] + (nk - nq)[:, None]
    rel = torch.arange(lk, device=q.device)[None, None] - pos[..., None]
    see = torch.arange(lk, device=q.device)[None, None] < nk[:, None, None]
    if s["causal"]:
        see = see & (rel <= 0)
    x = (torch.matmul(qp, kp.transpose(2, 3).contiguous()) * scale).view(b, hk, g, lq, lk)
    if s["buckets"]:
        which = _buckets(rel, s["buckets"], s["max_distance"], not s["causal"])
        x = x + s["table"].detach().float()[which].permute(0, 3, 1, 2).reshape(b, hk, g, lq, lk)
    see = see[:, None, None]
    x = torch.where(see, x, torch.full_like(x, -math.inf))
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    p = (p / torch.where(total > 0, total, torch.ones_like(total))).view(b, hk, g * lq, lk)
    del x
    o = torch.matmul(p, vp)
    out = {"out": _unpad(o.view(b, hk * g, lq, d), cu_q, q.shape[0], q.dtype)}
    if s["train"]:
        do = _pad(s["dout"], cu_q, lq).view(b, hk, g * lq, d)
        out["dv"] = _unpad(torch.matmul(p.transpose(2, 3).contiguous(), do), cu_k, k.shape[0], k.dtype)
        dp = torch.matmul(do, vp.transpose(2, 3).contiguous())
        ds = p * (dp - (do * o).sum(-1, keepdim=True))
        del dp, p
        out["dq"] = _unpad((torch.matmul(ds, kp) * scale).view(b, hk * g, lq, d), cu_q, q.shape[0], q.dtype)
        out["dk"] = _unpad(torch.matmul(ds.transpose(2, 3).contiguous(), qp) * scale, cu_k, k.shape[0], k.dtype)
        if s["buckets"]:  # sums along the diagonals first, then by bucket
            skew = torch.nn.functional.pad(ds.view(b, hk * g, lq, lk).flip(2), (0, lq)).flatten(2)
            diag = skew[..., :lq * (lq + lk - 1)].reshape(b, hk * g, lq, lq + lk - 1).sum(2, dtype=torch.float64)
            rel = torch.arange(lq + lk - 1, device=q.device)[None] - (lq - 1) - (nk - nq)[:, None]
            which = _buckets(rel, s["buckets"], s["max_distance"], not s["causal"])
            hot = (which[..., None] == torch.arange(s["buckets"], device=q.device)).double()
            out["dtable"] = torch.matmul(diag, hot).sum(0).t().to(s["table"].dtype).contiguous()
    return out


def _plain_norm(s):
    x, w = s["x"].detach(), s["weight"].detach()
    out = {}
    if s["residual"]:
        x = (x.float() + s["res"].detach().float()).to(x.dtype)
        out["r"] = x
    if s["form"] == "e4m3":  # 64 bits: values next to a border between two 8-bit values
        x64 = x.double()
        y = x64 * torch.rsqrt(x64.square().mean(-1, keepdim=True) + 1e-6) * w.double()
        scale = (y.abs().amax(-1, keepdim=True) / E4M3_MAX).float()
        out["y"] = (y / scale.double()).float().to(torch.float8_e4m3fn).to(torch.bfloat16)
        out["scale"] = scale.squeeze(-1)
        return out
    xf = x.float()
    rstd = torch.rsqrt(xf.square().mean(-1, keepdim=True) + 1e-6)
    xh = xf * rstd
    out["y"] = (xh * w).to(x.dtype)
    if s["form"] == "train":
        dy = s["dy"].float()
        wdy = dy * w
        dx = rstd * (wdy - xh * (wdy * xh).mean(-1, keepdim=True))
        out["dx"] = (dx + s["dr"].float() if s["residual"] else dx).to(x.dtype)
        out["dweight"] = (dy * xh).sum(0)
    return out


def _plain_clip(s):
    norm = torch.stack([g.double().square().sum() for g in s["grads"]]).sum().sqrt()
    coef = torch.clamp(s["max_norm"] / (norm + 1e-6), max=1.0).float()
    torch.cat([(g.float() * coef) for g in s["grads"]], out=s["out"])
    return {"norm": norm.float(), "out": s["out"]}


def run(s):
    if not own:
        if s["op"] == "attention":
            return _plain_attention(s)
        return _plain_norm(s) if s["op"] == "norm" else _plain_clip(s)
    if s["op"] == "attention":
        from detrpose_amd.attention import packed_attention
        extra = {}
        if s["buckets"]:
            extra = dict(bias_table=s["table"], max_distance=s["max_distance"], bidirectional=not s["causal"])
        out = packed_attention(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], causal=s["causal"], **extra)
        if not s["train"]:
            return {"out": out}
        names = ["q", "k", "v"] + (["table"] if s["buckets"] else [])
        grads = torch.autograd.grad(out, [s[n] for n in names], s["dout"])
        return {"out": out, **{"d" + n: g for n, g in zip(names, grads)}}
    if s["op"] == "norm":
        from detrpose_amd.norm import rms_norm, rms_norm_e4m3
        if s["form"] == "e4m3":
            y, scale, r = rms_norm_e4m3(s["x"], s["weight"], residual=s.get("res"), eps=1e-6)
            out = {"y": y.to(torch.bfloat16), "scale": scale}
            return {**out, "r": r} if s["residual"] else out
        got = rms_norm(s["x"], s["weight"], residual=s.get("res"), eps=1e-6)
        y, r = got if s["residual"] else (got, None)
        out = {"y": y, "r": r} if s["residual"] else {"y": y}
        if s["form"] == "train":
            ends, tops = ([y, r], [s["dy"], s["dr"]]) if s["residual"] else ([y], [s["dy"]])
            out["dx"], out["dweight"] = torch.autograd.grad(ends, [s["x"], s["weight"]], tops)
        return out
    from detrpose_amd.gradients import clip_grad_norm_
    return {"norm": clip_grad_norm_(s["grads"], s["max_norm"], out=s["out"]), "out": s["out"]}


# ------------------------------------------------------------------------------------- what it needs
def _pairs(q, k, causal):
    """Query-key pairs that see each other in one sequence."""
    if not causal:
        return q * k
    first = max(0, q - k)  # queries in front of every key see nothing
    n = q - first
    lo = k - q + first + 1
    return n * (2 * lo + n - 1) // 2


def work(case):
    if case["op"] == "attention":
        e = 2 if case["dtype"] == "bf16" else 4
        ql, kl = _lens(case["q_lens"]), _lens(case["k_lens"])
        h, hk, d = case["heads"], case["kv_heads"], case["dim"]
        pairs = sum(_pairs(a, b, case["causal"]) for a, b in zip(ql, kl))
        nq, nk = sum(ql) * h * d * e, sum(kl) * hk * d * e
        table = case["buckets"] * h * e
        if case["train"]:
            return {"bytes": 4 * nq + 4 * nk + 2 * table, "flops": 14 * d * h * pairs}
        return {"bytes": 2 * nq + 2 * nk + table, "flops": 4 * d * h * pairs}
    if case["op"] == "norm":
        e = 2 if case["dtype"] == "bf16" else 4
        n = case["rows"] * case["width"]
        res = 1 if case["residual"] else 0
        if case["form"] == "train":  # forward: x (res) -> y (r); backward: dy (dr) -> dx, the saved row is one of these
            return {"bytes": n * e * (4 + 3 * res) + 8 * case["width"], "flops": 14 * n}
        out = n + 4 * case["rows"] if case["form"] == "e4m3" else n * e
        return {"bytes": n * e * (1 + 2 * res) + out + 4 * case["width"], "flops": 5 * n}
    share = {"f32": 4.0, "bf16": 2.0, "mixed": 3.0}[case["dtype"]]
    return {"bytes": int(case["total"] * (share + 4)), "flops": 3 * case["total"]}


# ------------------------------------------------------------------------------------- in 64 bits
def _exact_bucket(rel, buckets, max_distance, both):
    """One distance's bucket, by whole-number powers."""
    nb, base = buckets, 0
    if both:
        nb, base = buckets // 2, buckets // 2 if rel > 0 else 0
    n = abs(rel) if both else max(0, -rel)
    e = nb // 2
    if n < e:
        return base + n
    j = 0
    while j + 1 < nb - e and n ** (nb - e) >= e ** (nb - e - j - 1) * max_distance ** (j + 1):
        j += 1
    return base + e + j


def exact(case, seed):
    s = prepare(case, seed)
    f = torch.float64
    if case["op"] == "attention":
        ql, kl, h, hk, d = s["ql"], s["kl"], s["heads"], s["kv_heads"], s["dim"]
        q, k, v = (s[n].detach().to(f) for n in ("q", "k", "v"))
        out = torch.zeros_like(q, memory_format=torch.contiguous_format)
        dq, dk, dv = (torch.zeros(t.shape, dtype=f, device=t.device) for t in (q, k, v))
        dtable = torch.zeros(max(1, case["buckets"]), h, dtype=f, device=q.device)
        q0 = k0 = 0
        for a, b in zip(ql, kl):
            i = torch.arange(a, device=q.device)[:, None] + (b - a)
            j = torch.arange(b, device=q.device)[None]
            seen = (j <= i) if case["causal"] else torch.ones(a, b, dtype=torch.bool, device=q.device)
            if case["buckets"]:
                far = max(a, b)
                both = not case["causal"]
                lut = torch.tensor([_exact_bucket(r, case["buckets"], case["max_distance"], both)
                                    for r in range(-far, far + 1)], device=q.device)
                which = lut[j - i + far]
            for n in range(h):
                m = n * hk // h
                qh, kh, vh = q[q0:q0 + a, n], k[k0:k0 + b, m], v[k0:k0 + b, m]
                x = qh @ kh.t() / math.sqrt(d)
                if case["buckets"]:
                    x = x + s["table"].detach().to(f)[:, n][which]
                x = x.masked_fill(~seen, -math.inf)
                top = x.max(1, keepdim=True).values
                x = (x - top.masked_fill(top == -math.inf, 0)).exp()
                p = x / x.sum(1, keepdim=True).clamp(min=1e-300)
                out[q0:q0 + a, n] = p @ vh
                if case["train"]:
                    g = s["dout"].to(f)[q0:q0 + a, n]
                    dv[k0:k0 + b, m] += p.t() @ g
                    dp = g @ vh.t()
                    ds = p * (dp - (dp * p).sum(1, keepdim=True))
                    dq[q0:q0 + a, n] = ds @ kh / math.sqrt(d)
                    dk[k0:k0 + b, m] += ds.t() @ qh / math.sqrt(d)
                    if case["buckets"]:
                        dtable[:, n] += torch.bincount(which.flatten(), ds.flatten(), case["buckets"])
            q0, k0 = q0 + a, k0 + b
        if not case["train"]:
            return {"out": out}
        got = {"out": out, "dq": dq, "dk": dk, "dv": dv}
        return {**got, "dtable": dtable} if case["buckets"] else got
    if case["op"] == "norm":
        x, w = s["x"].detach(), s["weight"].detach().to(f)
        got = {}
        if case["residual"]:
            x = (x.to(f) + s["res"].detach().to(f)).to(x.dtype)
            got["r"] = x.to(f)
        x = x.to(f)
        inv = 1 / ((x ** 2).sum(1, keepdim=True) / case["width"] + 1e-6).sqrt()
        y = x * inv * w
        if case["form"] == "e4m3":
            return {**got, "y": None, "scale": y.abs().max(1).values / E4M3_MAX}
        got["y"] = y
        if case["form"] == "train":
            dy = s["dy"].to(f)
            dot = (dy * w * x).sum(1, keepdim=True) / case["width"]
            got["dx"] = inv * dy * w - x * dot * inv ** 3 + (s["dr"].to(f) if case["residual"] else 0)
            got["dweight"] = (dy * x * inv).sum(0)
        return got
    norm = math.sqrt(sum(float(g.to(f).square().sum()) for g in s["grads"]))
    coef = min(1.0, case["max_norm"] / (norm + 1e-6))
    return {"norm": torch.tensor(norm, dtype=f), "out": torch.cat([g.to(f) * coef for g in s["grads"]])}
