"""Selective state-space operators (csrc/ssm_conv.hip, ssm_scan_fwd.hip, ssm_scan_bwd.hip): recurrent layers over time-major
sequences [L, B, ...] whose recurrence is a diagonal of N states per channel, beside the LSTM layers of `ops`, with the short
causal convolution in front of them and the single-step forms of both for sampling.

    past = [state; x];  pre[t] = bias + sum_k weight[:, k] past[t + k];  y[t] = silu(pre[t])                    causal_conv
    step = softplus(dt + dt_bias);  h[t] = exp(step A) h[t-1] + step x B;  y = (sum_n C h + D x) silu(z)        selective_scan

Sequences are fp32 or bf16 (all of one call alike); parameters, the scan's states and every sum are fp32.  The last axis is
contiguous (it is copied if not), steps and rows may have any pitch: slices of one projection's output go in without a copy.
`lengths` [B] are the rows' numbers of steps, 0 .. L: what lies behind them may hold anything, outputs and gradients there are zero,
and the final state is the one after the row's last step.  Gradients are first-order.  GPU only.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib as L_
from . import ops_ckpt8
from .ops_ckpt8 import Ckpt8, on_device, time_major

MAX_STATES = 32


def _fail(msg: str):
    raise L_.GmtError(msg)


def _want(t: Optional[torch.Tensor], name: str, shape, dtype) -> None:
    if t is not None and (tuple(t.shape) != tuple(shape) or t.dtype != dtype):
        _fail(f'{name}: {dtype} {tuple(shape)} expected, got {t.dtype} {tuple(t.shape)}')


def _seq(x: torch.Tensor, name: str, dims: int) -> None:
    if x.dim() != dims or x.numel() == 0:
        _fail(f'{name}: a {dims}-dimensional tensor with at least one element expected, got {tuple(x.shape)}')
    if x.dtype not in ops_ckpt8.DTYPES:
        _fail(f'{name}: float32 or bfloat16 expected, got {x.dtype}')


def _lengths(lengths: Optional[torch.Tensor], B: int, L: int, dev) -> Optional[torch.Tensor]:
    if lengths is None:
        return None
    if lengths.dtype not in (torch.int32, torch.int64) or tuple(lengths.shape) != (B,):
        _fail(f'lengths: an int32 or int64 tensor of {B} rows expected, got {lengths.dtype} {tuple(lengths.shape)}')
    if lengths.dtype == torch.int64:
        lengths = lengths.clamp(0, L)
    return lengths.to(device=dev, dtype=torch.int32).contiguous()


def _active(active: Optional[torch.Tensor], B: int, dev) -> Optional[torch.Tensor]:
    if active is None:
        return None
    if active.dtype not in (torch.bool, torch.uint8) or tuple(active.shape) != (B,):
        _fail(f'active: a bool tensor of {B} rows expected, got {active.dtype} {tuple(active.shape)}')
    return active.to(dev).contiguous()


def _step_states(state: torch.Tensor, state_out: Optional[torch.Tensor], name: str, shape, dtype) -> torch.Tensor:
    """The buffer of the updated state: `state` itself, or one that does not overlap it."""
    _want(state, name, shape, dtype)
    out = state if state_out is None else state_out
    _want(out, f'{name}_out', shape, dtype)
    if not state.is_contiguous() or not out.is_contiguous():
        _fail(f'{name}: states of a single step are updated where they are and must be contiguous')
    if out.data_ptr() != state.data_ptr():
        n = state.numel() * state.element_size()
        if abs(out.data_ptr() - state.data_ptr()) < n:
            _fail(f'{name}_out overlaps {name}')
    return out


def _no_grad_only(name: str, *tensors) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        _fail(f'{name} has no backward pass: call it under torch.no_grad() (for training, {name[:-5]} over whole sequences)')


# ----------------------------------------------------------------------------------------
# short causal convolution
# ----------------------------------------------------------------------------------------
def _conv_args(x, weight, bias, state, lengths, silu, **more) -> L_.ConvArgs:
    p = L_.ptr
    shape = (x.codes if isinstance(x, Ckpt8) else x).shape
    a = L_.ConvArgs(w=p(weight), bias=p(bias), state=p(state), lengths=p(lengths), L=shape[0], B=shape[1], C=shape[2],
                    K=weight.shape[1], silu=int(silu), **more)
    if isinstance(x, Ckpt8):
        a.x, a.x_scale, a.bf16 = p(x.codes), p(x.exponents), int(x.dtype == torch.bfloat16)
    else:
        a.x, a.x_t, a.x_b, a.bf16 = x.data_ptr(), x.stride(0), x.stride(1), int(x.dtype == torch.bfloat16)
    return a


class CausalConvFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, state, lengths, silu, ckpt8, keep):
        L, B, C = x.shape
        K = weight.shape[1]
        y = torch.empty(L, B, C, device=x.device, dtype=x.dtype)
        last = torch.empty(K - 1, B, C, device=x.device, dtype=x.dtype)
        a = _conv_args(x, weight, bias, state, lengths, silu, y=L_.ptr(y), state_out=L_.ptr(last))
        L_.call('gmt_causal_conv_fwd', ctypes.addressof(a), L_.stream(), nbytes=2.0 * x.numel() * x.element_size())
        if keep:
            packed = ops_ckpt8.pack(x) if ckpt8 else None
            ctx.save_for_backward(*((packed.codes, packed.exponents) if ckpt8 else (x, None)), weight, bias, state, lengths)
            ctx.silu, ctx.dtype, ctx.ckpt8 = silu, x.dtype, ckpt8
            ctx.set_materialize_grads(False)
        return y, last

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dlast):
        x, exps, weight, bias, state, lengths = ctx.saved_tensors
        if ctx.ckpt8:
            x = Ckpt8(x, exps, ctx.dtype)
        L, B, C = (x.codes if ctx.ckpt8 else x).shape
        K, dev = weight.shape[1], weight.device
        with torch.cuda.device(dev):
            dy = torch.zeros(L, B, C, device=dev, dtype=ctx.dtype) if dy is None else time_major(dy)
            dlast = None if dlast is None else dlast.contiguous()
            dx = torch.empty(L, B, C, device=dev, dtype=ctx.dtype)
            dparam = torch.empty(K + 1, C, device=dev, dtype=torch.float32)
            dstate = None if state is None else torch.empty_like(state)
            a = _conv_args(x, weight, bias, state, lengths, ctx.silu, dy=dy.data_ptr(), dstate_out=L_.ptr(dlast), dx=L_.ptr(dx),
                           dparam=L_.ptr(dparam), dstate=L_.ptr(dstate), dy_t=dy.stride(0), dy_b=dy.stride(1))
            need = ctypes.c_longlong(0)
            L_.call('gmt_causal_conv_bwd_workspace_floats', ctypes.addressof(a), ctypes.addressof(need), label='skip')
            ws = torch.empty(need.value, device=dev, dtype=torch.float32)
            a.workspace, a.workspace_floats = L_.ptr(ws), need.value
            L_.call('gmt_causal_conv_bwd', ctypes.addressof(a), L_.stream(), nbytes=3.0 * dx.numel() * dx.element_size())
        return dx, dparam[:K].t().contiguous(), (None if bias is None else dparam[K]), dstate, None, None, None, None


def _conv_checks(x, weight, bias, dims: int):
    _seq(x, 'x', dims)
    C = x.shape[-1]
    if weight.dim() != 2 or not 2 <= weight.shape[1] <= 4:
        _fail(f'weight: [{C}, K] with K = 2 .. 4 taps expected, got {tuple(weight.shape)}')
    _want(weight, 'weight', (C, weight.shape[1]), torch.float32)
    _want(bias, 'bias', (C,), torch.float32)
    return C, weight.shape[1]


def causal_conv(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None,
                state: Optional[torch.Tensor] = None, silu: bool = True, ckpt8: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """x [L, B, C], weight [C, K] (K = 2 .. 4, the last tap meets the step itself), bias [C], state [K-1, B, C]: the inputs before
    the first step (None: zeros) -> (y [L, B, C], the last K-1 inputs of each row, as `state` of the next call or of
    causal_conv_step).  ckpt8: x is kept in 8 bits for the backward pass."""
    dev = on_device(x, weight, bias, state)
    C, K = _conv_checks(x, weight, bias, 3)
    L, B = x.shape[:2]
    _want(state, 'state', (K - 1, B, C), x.dtype)
    keep = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias, state))
    lengths = _lengths(lengths, B, L, dev)
    with torch.cuda.device(dev):
        return CausalConvFn.apply(time_major(x), weight.contiguous(), None if bias is None else bias.contiguous(),
                                  None if state is None else state.contiguous(), lengths, bool(silu), bool(ckpt8), keep)


def causal_conv_step(x: torch.Tensor, state: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, silu: bool = True,
                     active: Optional[torch.Tensor] = None, state_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One step: x [B, C], state [K-1, B, C] -> y [B, C].  The updated state goes to state_out (None: in place).  Rows whose `active`
    is false keep their state and give zeros."""
    dev = on_device(x, state, weight, bias, state_out)
    C, K = _conv_checks(x, weight, bias, 2)
    B = x.shape[0]
    out = _step_states(state, state_out, 'state', (K - 1, B, C), x.dtype)
    _no_grad_only('causal_conv_step', x, state, weight, bias, state_out)
    x, active = time_major(x), _active(active, B, dev)
    with torch.cuda.device(dev):
        weight, bias = weight.contiguous(), None if bias is None else bias.contiguous()
        y = torch.empty(B, C, device=dev, dtype=x.dtype)
        a = L_.ConvArgs(x=x.data_ptr(), w=L_.ptr(weight), bias=L_.ptr(bias), state=L_.ptr(state), y=L_.ptr(y), state_out=L_.ptr(out),
                        x_b=x.stride(0), L=1, B=B, C=C, K=K, bf16=int(x.dtype == torch.bfloat16), silu=int(silu))
        L_.call('gmt_causal_conv_step', ctypes.addressof(a), L_.ptr(active), L_.stream(),
                nbytes=float(2 * K * x.numel() * x.element_size()))
    torch.autograd.graph.increment_version(out)
    return y


# ----------------------------------------------------------------------------------------
# selective scan
# ----------------------------------------------------------------------------------------
def _scan_args(x, dt, z, A, B, C, D, dt_bias, state, lengths, **more) -> L_.ScanArgs:
    p = L_.ptr
    q8 = isinstance(x, Ckpt8)
    shape = (x.codes if q8 else x).shape
    a = L_.ScanArgs(A=p(A), Bm=B.data_ptr(), Cm=C.data_ptr(), D=p(D), dt_bias=p(dt_bias), state=p(state), lengths=p(lengths),
                    B_t=B.stride(0), B_b=B.stride(1), B_g=B.stride(2), C_t=C.stride(0), C_b=C.stride(1), C_g=C.stride(2),
                    L=shape[0], B=shape[1], C=shape[2], N=A.shape[1], G=B.shape[2], bf16=int(B.dtype == torch.bfloat16), **more)
    for name, t in (('x', x), ('dt', dt), ('z', z)):
        if t is None:
            continue
        if q8:
            setattr(a, name, p(t.codes))
            setattr(a, name + '_scale', p(t.exponents))
        else:
            setattr(a, name, t.data_ptr())
            setattr(a, name + '_t', t.stride(0))
            setattr(a, name + '_b', t.stride(1))
    return a


def _workspace(a) -> Tuple[int, int, int]:
    n = [ctypes.c_longlong(0) for _ in range(3)]
    L_.call('gmt_selective_scan_workspace', ctypes.addressof(a), *(ctypes.addressof(v) for v in n), label='skip')
    return tuple(v.value for v in n)


class SelectiveScanFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, dt, A, B, C, D, z, dt_bias, state, lengths, ckpt8, keep):
        L, Bt, Ch = x.shape
        dev = x.device
        y = torch.empty(L, Bt, Ch, device=dev, dtype=x.dtype)
        last = torch.empty(Bt, Ch, A.shape[1], device=dev, dtype=torch.float32)
        a = _scan_args(x, dt, z, A, B, C, D, dt_bias, state, lengths, y=L_.ptr(y), state_out=L_.ptr(last))
        n_ck, n_fwd, _ = _workspace(a)
        # the states before every eighth step; from 8-bit checkpoints the backward pass finds them itself
        ck = torch.empty(n_ck if keep and not ckpt8 else 0, device=dev, dtype=torch.float32)
        ws = torch.empty(n_fwd, device=dev, dtype=torch.float32)
        a.ck, a.workspace, a.workspace_floats = L_.ptr(ck), L_.ptr(ws), n_fwd
        L_.call('gmt_selective_scan_fwd', ctypes.addressof(a), L_.stream(),
                nbytes=float((3 + (z is not None)) * x.numel() * x.element_size()))
        if keep:
            seqs = []
            for t in (x, dt, z):
                p = ops_ckpt8.pack(t) if ckpt8 and t is not None else None
                seqs += [t, None] if p is None else [p.codes, p.exponents]
            ctx.save_for_backward(*seqs, A, B, C, D, dt_bias, state, lengths, ck)
            ctx.dtype, ctx.ckpt8 = x.dtype, ckpt8
            ctx.set_materialize_grads(False)
        return y, last

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dlast):
        x, xe, dt, dte, z, ze, A, B, C, D, dt_bias, state, lengths, ck = ctx.saved_tensors
        L, Bt, Ch = x.shape
        N, dev, dtype = A.shape[1], A.device, ctx.dtype
        if ctx.ckpt8:
            x, dt = Ckpt8(x, xe, dtype), Ckpt8(dt, dte, dtype)
            z = None if z is None else Ckpt8(z, ze, dtype)
        with torch.cuda.device(dev):
            dy = torch.zeros(L, Bt, Ch, device=dev, dtype=dtype) if dy is None else time_major(dy)
            dlast = None if dlast is None else dlast.contiguous()
            dx, ddt, dz = (torch.empty(L, Bt, Ch, device=dev, dtype=dtype) for _ in range(3)) if z is not None else \
                (torch.empty(L, Bt, Ch, device=dev, dtype=dtype), torch.empty(L, Bt, Ch, device=dev, dtype=dtype), None)
            dB, dC = (torch.empty(B.shape, device=dev, dtype=dtype) for _ in range(2))
            dparam = torch.empty(Ch * (N + 2), device=dev, dtype=torch.float32)
            dstate = None if state is None else torch.empty_like(state)
            p = L_.ptr
            a = _scan_args(x, dt, z, A, B, C, D, dt_bias, state, lengths, dy=dy.data_ptr(), dstate_out=p(dlast), dx=p(dx), ddt=p(ddt),
                           dz=p(dz), dB=p(dB), dC=p(dC), dparam=p(dparam), dstate=p(dstate), dy_t=dy.stride(0), dy_b=dy.stride(1))
            n_ck, _, n_bwd = _workspace(a)
            if ctx.ckpt8:
                ck = torch.empty(n_ck, device=dev, dtype=torch.float32)
            ws = torch.empty(n_bwd, device=dev, dtype=torch.float32)
            a.ck, a.workspace, a.workspace_floats = p(ck), p(ws), n_bwd
            L_.call('gmt_selective_scan_bwd', ctypes.addressof(a), L_.stream(),
                    nbytes=float((5 + 2 * (z is not None)) * dx.numel() * dx.element_size()))
        dA = dparam[:Ch * N].view(Ch, N)
        return (dx, ddt, dA, dB, dC, None if D is None else dparam[Ch * N:Ch * (N + 1)], dz,
                None if dt_bias is None else dparam[Ch * (N + 1):], dstate, None, None, None)


def _scan_checks(x, dt, A, B, C, D, z, dt_bias, state, lead):
    """Shapes and types of a scan over `lead` = (L, B) or (B,) -> B and C with their group axis."""
    Ch = x.shape[-1]
    if A.dim() != 2 or not 1 <= A.shape[1] <= MAX_STATES:
        _fail(f'A: [{Ch}, N] with N = 1 .. {MAX_STATES} states expected, got {tuple(A.shape)}')
    N = A.shape[1]
    _want(A, 'A', (Ch, N), torch.float32)
    _want(dt, 'dt', x.shape, x.dtype)
    _want(z, 'z', x.shape, x.dtype)
    _want(D, 'D', (Ch,), torch.float32)
    _want(dt_bias, 'dt_bias', (Ch,), torch.float32)
    _want(state, 'state', (lead[-1], Ch, N), torch.float32)
    maps = []
    for name, m in (('B', B), ('C', C)):
        if m.dim() == len(lead) + 1:
            m = m.unsqueeze(-2)
        if m.dim() != len(lead) + 2 or m.shape[-2] < 1 or Ch % m.shape[-2]:
            _fail(f'{name}: {(*lead, N)} or {(*lead, "G", N)} with G dividing {Ch} channels expected, got {tuple(m.shape)}')
        _want(m, name, (*lead, m.shape[-2], N), x.dtype)
        maps.append(time_major(m))
    if maps[0].shape != maps[1].shape:
        _fail(f'B and C have different groups: {maps[0].shape[-2]} and {maps[1].shape[-2]}')
    return maps


def selective_scan(x: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor, D: Optional[torch.Tensor] = None,
                   z: Optional[torch.Tensor] = None, dt_bias: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None,
                   state: Optional[torch.Tensor] = None, ckpt8: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """x, dt [L, B, C] (and the gate z, or None), A [C, N] (N <= 32), B and C [L, B, N] or [L, B, G, N] (G groups of C / G neighbouring
    channels share them), D and dt_bias [C], state [B, C, N] fp32 (None: zeros) -> (y [L, B, C], the state after each row's
    last step).  ckpt8: x, dt and z are kept in 8 bits for the backward pass, which then finds the states again."""
    dev = on_device(x, dt, A, B, C, D, z, dt_bias, state)
    _seq(x, 'x', 3)
    L, Bt, _ = x.shape
    Bm, Cm = _scan_checks(x, dt, A, B, C, D, z, dt_bias, state, (L, Bt))
    keep = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, dt, A, B, C, D, z, dt_bias, state))
    whole = lambda t: None if t is None else t.contiguous()  # noqa: E731
    lengths = _lengths(lengths, Bt, L, dev)
    with torch.cuda.device(dev):
        return SelectiveScanFn.apply(time_major(x), time_major(dt), whole(A), Bm, Cm, whole(D), None if z is None else time_major(z),
                                     whole(dt_bias), whole(state), lengths, bool(ckpt8), keep)


def selective_scan_step(x: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor, state: torch.Tensor,
                        D: Optional[torch.Tensor] = None, z: Optional[torch.Tensor] = None, dt_bias: Optional[torch.Tensor] = None,
                        active: Optional[torch.Tensor] = None, state_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One step: x, dt (z) [B, C], B and C [B, N] or [B, G, N], state [B, C, N] fp32 -> y [B, C].  The updated state goes to state_out
    (None: in place).  Rows whose `active` is false keep their state and give zeros."""
    dev = on_device(x, dt, A, B, C, state, D, z, dt_bias, state_out)
    _seq(x, 'x', 2)
    Bt, Ch = x.shape
    Bm, Cm = _scan_checks(x, dt, A, B, C, D, z, dt_bias, None, (Bt,))
    N = A.shape[1]
    out = _step_states(state, state_out, 'state', (Bt, Ch, N), torch.float32)
    _no_grad_only('selective_scan_step', x, dt, A, B, C, state, D, z, dt_bias, state_out)
    active = _active(active, Bt, dev)
    with torch.cuda.device(dev):
        y = torch.empty(Bt, Ch, device=dev, dtype=x.dtype)
        up = lambda t: None if t is None else time_major(t).unsqueeze(0)  # noqa: E731
        whole = lambda t: None if t is None else t.contiguous()  # noqa: E731
        A, D, dt_bias, x, dt, z = whole(A), whole(D), whole(dt_bias), up(x), up(dt), up(z)
        a = _scan_args(x, dt, z, A, Bm.unsqueeze(0), Cm.unsqueeze(0), D, dt_bias, state, None, y=L_.ptr(y), state_out=L_.ptr(out))
        L_.call('gmt_selective_scan_step', ctypes.addressof(a), L_.ptr(active), L_.stream(), nbytes=float(8 * state.numel()))
    torch.autograd.graph.increment_version(out)
    return y
