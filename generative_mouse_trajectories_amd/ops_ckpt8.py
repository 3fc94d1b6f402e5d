"""8-bit activation checkpoints (csrc/ckpt8.hip): an activation kept for the backward pass as int8 codes and one exponent per
32 channels, a quarter of its fp32 bytes, and the weight gradient that reads it.

A block of 32 neighbouring channels of one row stands for q 2^e with |q| <= 127 and the smallest e in -118 .. 121 that reaches
its largest magnitude: an element is off by at most 2^(e-1) (2^e next to fp32's largest number, where 127 2^121 is the last value).  A block
that holds an infinity or a NaN stands for NaN.  `ops.linear`,
`ops_ssm.causal_conv` and `ops_ssm.selective_scan` take `ckpt8=True`: their gradients are then those at the values that the
checkpoints stand for (the outputs are computed from the inputs themselves).
"""
from __future__ import annotations

import contextlib
import ctypes
from typing import NamedTuple, Optional, Tuple

import torch
from torch.autograd import forward_ad

from . import _lib as L_

BLOCK = 32
DTYPES = (torch.float32, torch.bfloat16)
MAX_SIZE = (1 << 31) - (1 << 18)             # the kernels' sizes are 32-bit, and so are their sums with a tile's or a segment's

FAR = 1 << 24                                # elements from row to row that the weight gradient's 32-bit offsets do not reach


def fits(shape, name: str) -> None:
    """GmtError if one of these sizes would not arrive at the kernels as it is."""
    if max(shape) > MAX_SIZE:
        raise L_.GmtError(f'{name}: sizes of at most 2^31 - 2^18 expected, got {tuple(shape)}')


class Ckpt8(NamedTuple):
    """codes int8 [..., C], exponents uint8 [..., ceil(C / 32)] (255: the block stands for NaN), dtype of what was packed."""
    codes: torch.Tensor
    exponents: torch.Tensor
    dtype: torch.dtype


_HERE = contextlib.nullcontext()


def on_device(*tensors) -> int:
    """Index of the one GPU that all of them (None: left out) are on.  Every entry point passes its tensors through here: one with a
    forward-mode tangent is refused, which a kernel called beside autograd would drop without a word."""
    if forward_ad._current_level >= 0:                   # (looked at only within a dual level: 0.5 us a tensor)
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise L_.GmtError(f'a tensor of shape {tuple(t.shape)} has a forward-mode tangent: these operators have no forward-mode derivatives')
    dev = None
    for t in tensors:
        if t is not None:
            d = t.get_device()
            if d != dev:
                L_.require_cuda(t)
                if dev is not None:
                    raise L_.GmtError(f'tensors on different devices: cuda:{dev} and cuda:{d}')
                dev = d
    return dev


def on(dev: int):
    """Context in which `dev` is the current device (nothing to do where it is already: a device switch costs microseconds)."""
    return _HERE if dev == torch.cuda.current_device() else torch.cuda.device(dev)


def time_major(t: torch.Tensor) -> torch.Tensor:
    """`t` itself when its last axis is contiguous (rows may have any pitch), else a contiguous copy."""
    return t if t.stride()[-1] == 1 or t.shape[-1] == 1 else t.contiguous()


# Autograd brings a leaf's gradient to the stream on which the first graph of that leaf was made.  While such a graph from the default
# stream lives, a captured backward pass would have the default stream wait for the capture, which breaks it beyond an ordinary error.
_DEFAULT = 'gmt_default_stream'
with torch.inference_mode(False), torch.enable_grad():     # (whatever mode the package is imported in)
    _LEAF = type(torch.autograd.graph.get_gradient_edge(torch.zeros(1, requires_grad=True)).node)


def refuse_capture_beside(tensors) -> None:
    """Before a pass that may be differentiated is captured: GmtError if a leaf behind it has a live graph from the default stream."""
    todo = [torch.autograd.graph.get_gradient_edge(t).node for t in tensors if torch.is_tensor(t) and t.requires_grad]
    seen = set(todo)
    while todo:
        node = todo.pop()
        if type(node) is _LEAF and node.metadata.get(_DEFAULT):
            raise L_.GmtError(f'a leaf of shape {tuple(node.variable.shape)} has a graph that was made eagerly on the default stream and is still '
                              'alive: its backward pass cannot be captured.  Drop that graph (its outputs), run it under another '
                              'stream, or capture under torch.no_grad()')
        for n, _ in node.next_functions:
            if n is not None and n not in seen:
                seen.add(n)
                todo.append(n)


def apply(fn, dev: int, *args):
    """fn.apply(*args) for a differentiable operator of device `dev`, which must not be captured beside an eager graph of its leaves."""
    default = L_.stream_of(dev) == 0
    if not default and torch.cuda.is_current_stream_capturing():
        refuse_capture_beside(args)
    out = fn.apply(*args)
    # the leaves that the operator reads directly are marked with the stream of their first graph, until their last graph has gone
    for node, _ in (out[0] if type(out) is tuple else out).grad_fn.next_functions:
        if type(node) is _LEAF:
            node.metadata.setdefault(_DEFAULT, default)
    return out


def pack(x: torch.Tensor) -> Ckpt8:
    """x [..., C] fp32 or bf16 -> its 8-bit checkpoint."""
    dev = on_device(x)
    if x.dtype not in DTYPES:
        raise L_.GmtError(f'ckpt8 packs float32 and bfloat16, not {x.dtype}')
    if x.dim() < 1 or x.numel() == 0:
        raise L_.GmtError(f'ckpt8: nothing to pack in a tensor of shape {tuple(x.shape)}')
    fits(x.shape[-2:] if x.dim() == 3 else x.shape[-1:], 'ckpt8')
    x = time_major(x.detach()) if x.requires_grad else time_major(x)
    C = x.shape[-1]
    if x.dim() == 3:
        T, B, st, sb = x.shape[0], x.shape[1], x.stride(0), x.stride(1)
    else:
        x = x if x.dim() <= 2 else x.contiguous()
        T, B, st, sb = x.numel() // C, 1, (x.stride(0) if x.dim() == 2 else C), C
    with on(dev):
        codes = x.new_empty(x.shape, dtype=torch.int8)
        exps = x.new_empty((*x.shape[:-1], (C + BLOCK - 1) // BLOCK), dtype=torch.uint8)
        L_.call('gmt_ckpt8_pack', x.data_ptr(), st, sb, codes.data_ptr(), exps.data_ptr(), T, B, C, int(x.dtype == torch.bfloat16),
                L_.stream_of(dev), nbytes=float(x.numel() * (x.element_size() + 1)))
    return Ckpt8(codes, exps, x.dtype)


def check(p: Ckpt8) -> int:
    dev = on_device(p.codes, p.exponents)
    C = p.codes.shape[-1]
    fits((C,), 'ckpt8')
    if (p.codes.dtype != torch.int8 or p.exponents.dtype != torch.uint8 or p.codes.numel() == 0 or not p.codes.is_contiguous()
            or not p.exponents.is_contiguous() or p.exponents.shape != (*p.codes.shape[:-1], (C + BLOCK - 1) // BLOCK)):
        raise L_.GmtError('not an 8-bit checkpoint: contiguous int8 codes [..., C] and uint8 exponents [..., ceil(C / 32)] expected')
    return dev


def unpack(p: Ckpt8, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """The values that a checkpoint stands for, as `dtype` (default: what was packed; both types hold them exactly)."""
    dev = check(p)
    dtype = p.dtype if dtype is None else dtype
    if dtype not in DTYPES:
        raise L_.GmtError(f'ckpt8 unpacks to float32 and bfloat16, not {dtype}')
    C = p.codes.shape[-1]
    with on(dev):
        out = p.codes.new_empty(p.codes.shape, dtype=dtype)
        L_.call('gmt_ckpt8_unpack', p.codes.data_ptr(), p.exponents.data_ptr(), out.data_ptr(), out.numel() // C, C,
                int(dtype == torch.bfloat16), L_.stream_of(dev), nbytes=float(out.numel() * (out.element_size() + 1)))
    return out


def wgrad(dY: torch.Tensor, p: Ckpt8, want_db: bool = False) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """dW = dY^T X over the rows, X [..., I] given as its checkpoint and dY [..., N] (fp32 or bf16) with as many rows: fp32 [N, I];
    with want_db also db = dY.sum over the rows.  The products are exact (for an fp32 dY from 2^-102 on, below to 2^-126 in dY), the sums fp32
    (csrc/ckpt8.hip); `ops.wgrad` is the same for an fp32 X."""
    dev = check(p)
    if on_device(dY) != dev:
        raise L_.GmtError('wgrad: dY and the checkpoint are on different devices')
    if dY.dtype not in DTYPES:
        raise L_.GmtError(f'wgrad: dY must be float32 or bfloat16, not {dY.dtype}')
    N, I = dY.shape[-1], p.codes.shape[-1]
    R = p.codes.numel() // I
    fits((N,), 'wgrad')
    if N == 0 or dY.numel() // N != R:
        raise L_.GmtError(f'wgrad: dY {tuple(dY.shape)} and the checkpoint {tuple(p.codes.shape)} have different rows')
    dY = time_major(dY.detach()) if dY.requires_grad else time_major(dY)
    if dY.dim() != 2:
        dY = dY.reshape(R, N)
    if R > 1 and not N <= dY.stride(0) < FAR:            # (an expanded gradient, whose rows share memory, or rows out of reach)
        dY = dY.contiguous()
    with on(dev):
        need = ctypes.c_longlong(0)
        L_.call('gmt_ckpt8_wgrad_workspace_floats', R, N, I, ctypes.addressof(need), label='skip')
        ws = dY.new_empty(need.value, dtype=torch.float32)
        out = dY.new_empty(N * I + N, dtype=torch.float32)
        L_.call('gmt_ckpt8_wgrad', dY.data_ptr(), dY.stride(0) if R > 1 else N, p.codes.data_ptr(), p.exponents.data_ptr(), out.data_ptr(), R,
                N, I, int(dY.dtype == torch.bfloat16), int(want_db), L_.ptr(ws), need.value, L_.stream_of(dev),
                label=f'wgrad8_N{N}_I{I}', flops=2.0 * R * N * I)
    return out[:N * I].view(N, I), (out[N * I:] if want_db else None)
