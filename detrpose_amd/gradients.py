"""The global norm of many gradient tensors, and their clipping by it, on the HIP kernels.

`clip_grad_norm_` is the step between `loss.backward()` and an optimizer over separate parameter
tensors (the reference's torch.nn.utils.clip_grad_norm_, src/solver/engine.py:78-89); the Trainer's
own step keeps one flat gradient buffer instead and clips inside its AdamW (`dp_grad_sqnorm`,
`dp_adamw`). With `out` the clipped gradients are gathered into such a flat buffer.

There is no CPU path: the HIP library must load (see _lib.load()).
"""
from __future__ import annotations

import array
import ctypes as C

import torch

from . import _lib

_DT = {torch.float32: _lib.DP_F32, torch.bfloat16: _lib.DP_BF16}


def _dense(t):
    """Whether the tensor's elements fill one span of memory in some order of its dimensions."""
    want = 1
    for st, n in sorted((st, n) for st, n in zip(t.stride(), t.shape) if n != 1):
        if st != want:
            return False
        want *= n
    return True


def _holds(tensors):
    """Which tensors stand for their .grad: parameters, frozen or not, and leaves that have one or ask for one. (The
    whole list at once: hundreds of tensors are looked at in front of a few launches.)"""
    kinds = set(map(type, tensors))
    if kinds == {torch.nn.Parameter}:
        return [True] * len(tensors)
    holds = [t.requires_grad or t.grad is not None for t in tensors]
    if True in holds:   # what a graph computed is a gradient itself
        holds = [h and t.is_leaf for h, t in zip(holds, tensors)]
    if kinds != {torch.Tensor}:
        holds = [h or isinstance(t, torch.nn.Parameter) for h, t in zip(holds, tensors)]
    return holds


def clip_grad_norm_(parameters, max_norm, out=None):
    """Clip gradients by their global 2-norm: g * min(1, max_norm / (norm + 1e-6)) for every tensor.

    parameters: a tensor or an iterable of tensors, either parameters or gradients. A torch.nn.Parameter, frozen
    or not, and a leaf that requires a gradient or has one stand for their .grad, and are passed over while
    that is None; other tensors are gradients themselves. Both kinds in one call are refused: a frozen weight that
    is a plain tensor could not be told from a gradient. Gradients are f32 or bf16, mixed as they come, all
    on one GPU; no two of them share memory.
    out: None clips in place. A contiguous 1-d f32 or bf16 tensor of as many elements as the
    gradients together takes the clipped gradients one behind the other, in their order, and the
    gradients are left as they are.
    Returns the norm (before clipping) as an f32 scalar on the GPU: nothing waits for it. Where there is no gradient
    it is 0, on the device of out or of the first tensor (an empty list: on the CPU). A norm that is not
    finite makes the clipped gradients NaN (or 0 for finite ones under an infinite norm), as
    torch.nn.utils.clip_grad_norm_ without error_if_nonfinite. Deterministic: equal gradients give equal bits."""
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    max_norm = float(max_norm)
    if not max_norm >= 0:
        raise ValueError(f"clip_grad_norm_: max_norm {max_norm}")
    tensors = list(parameters)
    holds = _holds(tensors)
    if True in holds:
        if False in holds:
            raise ValueError(f"clip_grad_norm_: parameters and, at {holds.index(False)}, a tensor that neither is one nor "
                             "requires a gradient: pass parameters or gradients")
        grads = [g for g in (p.grad for p in tensors) if g is not None]
    else:
        grads = tensors
    if not grads:
        if out is not None and out.numel():
            raise ValueError(f"clip_grad_norm_: out holds {out.numel()} elements, the gradients 0")
        at = out if out is not None else tensors[0] if tensors else None
        return torch.zeros((), device=None if at is None else at.device, dtype=torch.float32)
    _lib.refuse_tangents("clip_grad_norm_", out, *grads)
    device = grads[0].device
    kinds = {g.dtype for g in grads}
    if kinds - _DT.keys():
        raise TypeError(f"clip_grad_norm_: gradient dtypes {sorted(map(str, kinds))} (f32 / bf16)")
    if len(set(map(torch.Tensor.get_device, grads))) != 1 or device.type != "cuda" or grads[0].layout != torch.strided:
        if any(g.layout != torch.strided for g in grads):
            raise TypeError("clip_grad_norm_: sparse gradients")
        raise RuntimeError("clip_grad_norm_: gradients must be on one GPU (no CPU path)")
    sizes = list(map(torch.Tensor.numel, grads))
    if out is not None:
        if out.dtype not in _DT:
            raise TypeError(f"clip_grad_norm_: out dtype {out.dtype} (f32 / bf16)")
        if out.device != device:
            raise RuntimeError(f"clip_grad_norm_: gradients on {device}, out on {out.device}")
        if out.dim() != 1 or not out.is_contiguous() or out.numel() != sum(sizes):
            raise ValueError(f"clip_grad_norm_: out {tuple(out.shape)} is not a contiguous row of {sum(sizes)} elements")
        if out.requires_grad and torch.is_grad_enabled():
            raise RuntimeError("clip_grad_norm_: out requires a gradient")
    try:
        plain = list(map(torch.Tensor.is_contiguous, grads))
    except RuntimeError:   # a sparse tensor has no strides
        raise TypeError("clip_grad_norm_: sparse gradients") from None
    for i in (i for i, ok in enumerate(plain) if not ok) if not all(plain) else ():
        if out is not None:
            grads[i] = grads[i].contiguous()   # out takes the elements in their logical order
        elif not _dense(grads[i]):
            raise ValueError(f"clip_grad_norm_: gradient {i} {tuple(grads[i].shape)} with strides {grads[i].stride()} "
                             "does not fill one span of memory: clip a contiguous copy")
    n = len(grads)
    ptrs = array.array("Q", map(torch.Tensor.data_ptr, grads))
    nums = array.array("q", sizes)
    dts = array.array("i", [_DT[g.dtype] for g in grads] if len(kinds) > 1 else [_DT[grads[0].dtype]]) * (n if len(kinds) == 1 else 1)
    lib = _lib.load()
    with _lib.device_of(grads[0]):
        norm = torch.empty((), device=device, dtype=torch.float32)
        nb = int(lib.dp_grad_clip_ws_bytes(n))
        ws = torch.empty(nb, device=device, dtype=torch.uint8)
        s = torch.cuda.current_stream().cuda_stream
        _lib.check(lib.dp_grad_clip(ptrs.buffer_info()[0], nums.buffer_info()[0], dts.buffer_info()[0], n, max_norm,
                                    norm.data_ptr(), None if out is None else out.data_ptr(),
                                    0 if out is None else out.numel(),
                                    _lib.DP_F32 if out is None else _DT[out.dtype], ws.data_ptr(), nb,
                                    C.c_void_p(s)), "dp_grad_clip")
    torch.autograd.graph.increment_version(grads if out is None else [out])
    return norm
