"""Attention over packed sequences, on the HIP kernels.

`packed_attention` takes sequences of different lengths row behind row instead of padded batches (images
with different numbers of instances, prompts, cached tokens), with grouped heads, causal order and a
learned relative position bias by buckets; it is differentiable in q, k, v and the bias table. The
model's own attention (fixed lengths, equal heads) stays with `dp_attention`, `dp_mha_layernorm` and
`dp_attn_fwd` / `dp_attn_bwd`.

There is no CPU path: the HIP library must load (see _lib.load()).
"""
from __future__ import annotations

import ctypes as C
import functools

import torch

from . import _lib

_DT = {torch.float32: _lib.DP_F32, torch.bfloat16: _lib.DP_BF16}


@functools.lru_cache(maxsize=64)
def bucket_edges(num_buckets, max_distance, bidirectional):
    """The distances at which the next bucket of one direction begins: distance n falls into the bucket
    numbered by how many edges are <= n. Of a direction's nb buckets (num_buckets, or half of them when
    bidirectional) the first e = nb // 2 hold one distance each; bucket e + j, j < K = nb - e, begins at the
    least n >= e (max_distance / e)^(j / K), compared in whole numbers (n^K against e^(K - j)
    max_distance^j), so no rounding decides a border."""
    if bidirectional and num_buckets % 2:
        raise ValueError(f"packed_attention: {num_buckets} buckets for two directions")
    nb = num_buckets // 2 if bidirectional else num_buckets
    e = nb // 2
    if not (2 <= num_buckets <= 64 and nb >= 2):
        raise ValueError(f"packed_attention: {num_buckets} buckets (2 to 64, at least 2 a direction)")
    if not e < max_distance <= 4096:
        raise ValueError(f"packed_attention: max_distance {max_distance} ({e + 1} to 4096 with {num_buckets} buckets)")
    k = nb - e
    edges = list(range(1, e + 1))
    n = e
    for j in range(1, k):
        bound = e ** (k - j) * max_distance ** j
        while n ** k < bound:
            n += 1
        edges.append(n)
    return tuple(edges)


def _check(q, k, v, cu_q, cu_k, scale, bias_table, out):
    for n, t in (("q", q), ("k", k), ("v", v)):
        if t.dtype not in _DT or t.dtype != q.dtype:
            raise TypeError(f"packed_attention: {n} dtype {t.dtype} (f32 / bf16, all three alike)")
        if t.dim() != 3:
            raise ValueError(f"packed_attention: {n} {tuple(t.shape)} is not (rows, heads, dim)")
    (_, h, d), (tk, hk, dk) = q.shape, k.shape
    if v.shape != k.shape or dk != d:
        raise ValueError(f"packed_attention: q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)} do not match")
    if hk == 0 or h == 0 or h % hk:
        raise ValueError(f"packed_attention: {h} heads over {hk} key heads")
    if not (0 < d <= 128 and d % 8 == 0):
        raise ValueError(f"packed_attention: head dim {d} (multiples of 8 up to 128)")
    for n, c in (("cu_seqlens_q", cu_q), ("cu_seqlens_k", cu_k)):
        if c.dtype != torch.int32 or c.dim() != 1 or c.numel() < 1:
            raise ValueError(f"packed_attention: {n} is a row of int32, one more than the sequences")
    if cu_q.numel() != cu_k.numel():
        raise ValueError(f"packed_attention: {cu_q.numel() - 1} query sequences, {cu_k.numel() - 1} key sequences")
    if not 0 < scale < float("inf"):
        raise ValueError(f"packed_attention: scale {scale}")
    if not q.is_cuda:
        raise RuntimeError("packed_attention: tensors must be on the GPU (no CPU path)")
    for n, t in (("k", k), ("v", v), ("cu_seqlens_q", cu_q), ("cu_seqlens_k", cu_k), ("bias_table", bias_table),
                 ("out", out)):
        if t is not None and t.device != q.device:
            raise RuntimeError(f"packed_attention: q on {q.device}, {n} on {t.device}: all must be on the same GPU")
    if bias_table is not None:
        if bias_table.dtype not in (torch.float32, q.dtype):
            raise TypeError(f"packed_attention: bias_table dtype {bias_table.dtype} (f32, or q's {q.dtype})")
        if bias_table.dim() != 2 or bias_table.shape[1] != h:
            raise ValueError(f"packed_attention: bias_table {tuple(bias_table.shape)} is not (buckets, {h} heads)")
        if h // hk * bias_table.shape[0] > 4096:
            raise ValueError(f"packed_attention: {h // hk} heads a group x {bias_table.shape[0]} buckets (4096 at most)")
    if q.shape[0] * h >= 2 ** 31 - 128 or tk >= 2 ** 31 - 128:
        raise ValueError(f"packed_attention: q {tuple(q.shape)}, k {tuple(k.shape)}: too many rows")


def _ready(t):
    """The tensor, or a contiguous copy where its rows cannot be read in 16-byte pieces."""
    if t.numel() == 0 or (t.is_contiguous() and t.data_ptr() % 16 == 0):
        return t
    e, (row, head) = t.element_size(), _strides(t)
    ok = (t.stride(2) == 1 and t.data_ptr() % 16 == 0 and row * e % 16 == 0 and head * e % 16 == 0
          and row * e < 1 << 24 and head * e * t.shape[1] < 1 << 28)
    return t if ok else t.contiguous()


def _strides(t):
    """(row, head) in elements; a tensor may have any stride along a dimension of one."""
    return (t.stride(0) if t.shape[0] > 1 else t.shape[2]), (t.stride(1) if t.shape[1] > 1 else t.shape[2])


def _span(t):
    """First byte and the one behind the last of a tensor that is not empty."""
    return t.data_ptr(), t.data_ptr() + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()


def _check_out(q, k, v, cu_q, cu_k, table, out):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, v, table, out)):
        raise RuntimeError("packed_attention: out= has no gradient (call it under torch.no_grad())")
    if out.shape != q.shape or out.dtype != q.dtype or (out.numel() and _ready(out) is not out):
        raise ValueError(f"packed_attention: out {tuple(out.shape)} {out.dtype} with strides {out.stride()} does not "
                         f"match q {tuple(q.shape)} {q.dtype} in rows of 16-byte pieces")
    if not out.numel():
        return
    (row, head), (n, h, d) = _strides(out), out.shape
    if not ((head >= d or h == 1) and (row >= (h - 1) * head + d or n == 1)
            or (row >= d or n == 1) and (head >= (n - 1) * row + d or h == 1)):
        raise ValueError(f"packed_attention: rows of out {tuple(out.shape)} with strides {out.stride()} overlap")
    a, b = _span(out)
    for name, t in (("q", q), ("k", k), ("v", v), ("cu_seqlens_q", cu_q), ("cu_seqlens_k", cu_k), ("bias_table", table)):
        if t is not None and t.numel() and a < _span(t)[1] and _span(t)[0] < b:
            raise ValueError(f"packed_attention: out lies across {name}, which is read while out is written")


def _ptr(t):
    return None if t is None else t.data_ptr()


def _desc(q, k, v, out, lse, lo, cu_q, cu_k, causal, scale, table, edges, both, fill_tail):
    a = _lib.PackedAttn()
    a.q, a.k, a.v, a.out, a.lse, a.out_lo = _ptr(q), _ptr(k), _ptr(v), _ptr(out), _ptr(lse), _ptr(lo)
    if lse is not None and lse.shape[0] == 2 and lse.numel():
        a.lse_lo = lse.data_ptr() + 4 * lse.stride(0)
    (a.q_row, a.q_head), (a.k_row, a.k_head) = _strides(q), _strides(k)
    (a.v_row, a.v_head), (a.o_row, a.o_head) = _strides(v), _strides(out)
    a.cu_q, a.cu_k, a.nseq = _ptr(cu_q), _ptr(cu_k), cu_q.numel() - 1
    a.tq, a.tk, a.heads, a.kv_heads, a.dim = q.shape[0], k.shape[0], q.shape[1], k.shape[1], q.shape[2]
    a.causal, a.fill_tail, a.scale, a.dtype = int(causal), int(fill_tail), scale, _DT[q.dtype]
    if table is not None:
        a.bias, a.bias_dtype, a.buckets, a.both = _ptr(table), _DT[table.dtype], table.shape[0], int(both)
        a.edge[:len(edges)] = edges
    return a


def _forward(q, k, v, cu_q, cu_k, causal, scale, table, edges, both, out, need_lse):
    """(out, lse, what out's rounding left off, and the tensors as the kernels read them)."""
    q, k, v, cu_q, cu_k = _ready(q), _ready(k), _ready(v), cu_q.contiguous(), cu_k.contiguous()
    table = None if table is None else table.contiguous()
    fill = out is None
    if fill:
        out = torch.empty(q.shape, device=q.device, dtype=q.dtype)
    lib = _lib.load()
    with _lib.device_of(q):
        lse = None   # with a bias also what its rounding left off
        if need_lse:
            lse = torch.empty((1 if table is None else 2, *q.shape[:2]), device=q.device, dtype=torch.float32)
        lo = torch.empty(q.shape, device=q.device, dtype=q.dtype) if need_lse and q.dtype == torch.bfloat16 else None
        a = _desc(q, k, v, out, lse, lo, cu_q, cu_k, causal, scale, table, edges, both, fill)
        nb = int(lib.dp_packed_attn_ws_bytes(C.byref(a), 0))
        ws = torch.empty(nb, device=q.device, dtype=torch.uint8) if nb else None
        a.ws, a.ws_bytes = _ptr(ws), nb
        s = torch.cuda.current_stream().cuda_stream
        _lib.check(lib.dp_packed_attn_fwd(C.byref(a), C.c_void_p(s)), "dp_packed_attn_fwd")
    return out, lse, lo, (q, k, v, cu_q, cu_k, table)


class PackedAttentionFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, table, cu_q, cu_k, causal, scale, edges, both):
        need = any(ctx.needs_input_grad[:4])
        out, lse, lo, read = _forward(q, k, v, cu_q, cu_k, causal, scale, table, edges, both, None, need)
        if need:
            ctx.save_for_backward(*read, out, lse, lo)
            ctx.how = (causal, scale, edges, both)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        q, k, v, cu_q, cu_k, table, out, lse, lo = ctx.saved_tensors
        causal, scale, edges, both = ctx.how
        dout = _ready(dout.to(q.dtype))
        lib = _lib.load()
        with _lib.device_of(q):
            dq, dk, dv = (torch.empty(t.shape, device=t.device, dtype=t.dtype) for t in (q, k, v))
            dtable = None if table is None else torch.empty_like(table)
            a = _desc(q, k, v, out, lse, lo, cu_q, cu_k, causal, scale, table, edges, both, False)
            a.dout, (a.g_row, a.g_head) = _ptr(dout), _strides(dout)
            a.dq, a.dk, a.dv, a.dbias = _ptr(dq), _ptr(dk), _ptr(dv), _ptr(dtable)
            nb = int(lib.dp_packed_attn_ws_bytes(C.byref(a), 1))
            ws = torch.empty(nb, device=q.device, dtype=torch.uint8)
            a.ws, a.ws_bytes = _ptr(ws), nb
            s = torch.cuda.current_stream().cuda_stream
            _lib.check(lib.dp_packed_attn_bwd(C.byref(a), C.c_void_p(s)), "dp_packed_attn_bwd")
        return dq, dk, dv, dtable, None, None, None, None, None, None


def packed_attention(q, k, v, cu_seqlens_q, cu_seqlens_k=None, *, causal=False, scale=None, bias_table=None,
                     max_distance=128, bidirectional=None, out=None):
    """softmax(scale q k^T + bias) v within each of the sequences packed row behind row.

    q (Tq, heads, dim), k and v (Tk, kv_heads, dim), f32 or bf16, strided as they come (rows that are no
    multiples of 16 bytes are copied); dim a multiple of 8 up to 128, kv_heads a divisor of heads: query head h
    reads key head h // (heads // kv_heads). cu_seqlens_q / cu_seqlens_k (sequences + 1) int32 on the GPU:
    sequence b has the query rows cu_seqlens_q[b] : cu_seqlens_q[b + 1] and the key rows of cu_seqlens_k
    (None: the same), beginning at 0, rising; nothing reads them on the host, so a captured call replays with
    other lengths. Query i of a sequence of lq queries and lk keys stands at position i + lk - lq: a new token
    or a chunk of them sits behind what a cache holds. causal: it sees the keys up to its position.
    A query that sees no key (an empty sequence, lk < lq under causal, every bias -inf) gives zeros.
    scale: dim ** -0.5 by default, positive.

    bias_table (buckets, heads), f32 or q's type: a learned bias by relative position j - position, in
    the buckets of `bucket_edges(buckets, max_distance, bidirectional)`; when bidirectional (by default:
    unless causal) keys behind the position take the upper half of the buckets, otherwise they count as
    distance 0. It differs by head, and its gradient is summed in f32. Where all that a query sees has the
    type's lowest value (or any bias that swallows the scores), its weights are equal, in the gradients too.

    Returns (Tq, heads, dim) of q's type; rows behind the last sequence are zeros. Differentiable (once, in
    reverse) in q, k, v and bias_table, with equal bits for equal inputs; gradients of rows behind the last sequence are
    zeros. How long walks are cut goes by the whole call's sizes, so a sequence's last bits may change with what
    is packed beside it. Scores and sums are f32; in bf16 the weights (and their gradients) are rounded to bf16 for the
    products with v, q and k. out: the result is written here instead, rows behind the last sequence are left
    as they are; without gradients only, and in memory apart from what is read.
    Values that causal order hides from a query do not reach its output, be they inf or NaN; its gradients
    need finite ones."""
    if cu_seqlens_k is None:
        cu_seqlens_k = cu_seqlens_q
    if scale is None:
        scale = float(q.shape[-1] or 1) ** -0.5 if q.dim() == 3 else 1.0
    scale = float(scale)
    _lib.refuse_tangents("packed_attention", q, k, v, bias_table, out)
    _check(q, k, v, cu_seqlens_q, cu_seqlens_k, scale, bias_table, out)
    both = not causal if bidirectional is None else bool(bidirectional)
    edges = () if bias_table is None else bucket_edges(bias_table.shape[0], int(max_distance), both)
    if out is not None:
        _check_out(q, k, v, cu_seqlens_q, cu_seqlens_k, bias_table, out)
        torch.autograd.graph.increment_version(out)
        return _forward(q, k, v, cu_seqlens_q, cu_seqlens_k, causal, scale, bias_table, edges, both, out, False)[0]
    if not (torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or
                                         (bias_table is not None and bias_table.requires_grad))):
        return _forward(q, k, v, cu_seqlens_q, cu_seqlens_k, causal, scale, bias_table, edges, both, None, False)[0]
    return PackedAttentionFunction.apply(q, k, v, bias_table, cu_seqlens_q, cu_seqlens_k, bool(causal), scale, edges, both)
