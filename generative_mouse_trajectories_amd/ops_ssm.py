"""Selective state-space operators (csrc/ssm_conv.hip, ssm_scan_fwd.hip, ssm_scan_bwd.hip): recurrent layers over time-major
sequences [L, B, ...] whose recurrence is a diagonal of N states per channel, beside the LSTM layers of `ops`, with the short
causal convolution in front of them and the single-step forms of both for sampling.

    past = [state; x];  pre[t] = bias + sum_k weight[:, k] past[t + k];  y[t] = silu(pre[t])                    causal_conv
    step = softplus(dt + dt_bias);  h[t] = exp(step A) h[t-1] + step x B;  y = (sum_n C h + D x) silu(z)        selective_scan

Sequences are fp32 or bf16 (all of one call alike); parameters, the scan's states and every sum are fp32.  The last axis is
contiguous (it is copied if not), steps and rows may have any pitch: slices of one projection's output go in without a copy (but for the scan's
sequences whose steps lie 2^27 elements or more apart, and its maps B and C from 2^26 on).
`lengths` [B] are the rows' numbers of steps, 0 .. L: what lies behind them may hold anything, outputs and gradients there are zero,
and the final state is the one after the row's last step.  Gradients are first-order and reverse-mode.  GPU only.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _lib as L_
from . import ops_ckpt8
from .ops_ckpt8 import Ckpt8, on, on_device, time_major

MAX_STATES = 32
FAR_SEQ, FAR_MAP = 1 << 27, 1 << 26          # elements from one step to the next that the scan's 32-bit offsets within a chunk do not reach


def _fail(msg: str):
    raise L_.GmtError(msg)


def _want(t: Optional[torch.Tensor], name: str, shape: tuple, dtype) -> None:
    if t is not None and (t.shape != shape or t.dtype != dtype):
        _fail(f'{name}: {dtype} {shape} expected, got {t.dtype} {tuple(t.shape)}')


def _seq(x: torch.Tensor, name: str, dims: int) -> None:
    if x.dim() != dims or x.numel() == 0:
        _fail(f'{name}: a {dims}-dimensional tensor with at least one element expected, got {tuple(x.shape)}')
    if x.dtype not in ops_ckpt8.DTYPES:
        _fail(f'{name}: float32 or bfloat16 expected, got {x.dtype}')
    ops_ckpt8.fits(x.shape, name)


def _lengths(lengths: Optional[torch.Tensor], B: int, L: int, x: torch.Tensor) -> Optional[torch.Tensor]:
    if lengths is None:
        return None
    if lengths.dtype not in (torch.int32, torch.int64) or lengths.shape != (B,):
        _fail(f'lengths: an int32 or int64 tensor of {B} rows expected, got {lengths.dtype} {tuple(lengths.shape)}')
    if lengths.dtype == torch.int64:
        lengths = lengths.clamp(0, L)
    return lengths.to(device=x.device, dtype=torch.int32).contiguous()


def _active(active: Optional[torch.Tensor], B: int, x: torch.Tensor) -> Optional[torch.Tensor]:
    if active is None:
        return None
    if active.dtype not in (torch.bool, torch.uint8) or active.shape != (B,):
        _fail(f'active: a bool tensor of {B} rows expected, got {active.dtype} {tuple(active.shape)}')
    return active.to(x.device).contiguous()


def _step_states(state: torch.Tensor, state_out: Optional[torch.Tensor], shape: tuple, dtype) -> torch.Tensor:
    """The buffer of the updated state: `state` itself, or one that does not overlap it."""
    _want(state, 'state', shape, dtype)
    if not state.is_contiguous():
        _fail('state: the state of a single step is updated where it is and must be contiguous')
    if state_out is None:
        return state
    _want(state_out, 'state_out', shape, dtype)
    if not state_out.is_contiguous():
        _fail('state_out: must be contiguous')
    apart = abs(state_out.data_ptr() - state.data_ptr())
    if 0 < apart < state.numel() * state.element_size():
        _fail('state_out overlaps state')
    return state_out


def _no_grad_only(name: str, *tensors) -> None:
    for t in tensors:
        if t is not None and t.requires_grad:
            _fail(f'{name} has no backward pass: call it under torch.no_grad() (for training, {name[:-5]} over whole sequences)')


def _any_grad(*tensors) -> bool:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


def _whole(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    return t if t is None or t.is_contiguous() else t.contiguous()


def _at(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _near(t: torch.Tensor, far: int) -> torch.Tensor:
    """time_major(t), as a contiguous copy if its steps lie `far` or more apart."""
    t = time_major(t)
    return t if t.stride(0) < far or t.shape[0] == 1 else t.contiguous()


def _space(n: int, like: torch.Tensor) -> Optional[torch.Tensor]:
    return like.new_empty(n, dtype=torch.float32) if n else None


# ----------------------------------------------------------------------------------------
# short causal convolution
# ----------------------------------------------------------------------------------------
def _conv_args(x, weight, bias, state, lengths, silu, **more) -> L_.ConvArgs:
    if isinstance(x, Ckpt8):
        shape = x.codes.shape
        more.update(x=x.codes.data_ptr(), x_scale=x.exponents.data_ptr(), bf16=x.dtype == torch.bfloat16)
    else:
        shape, st = x.shape, x.stride()
        more.update(x=x.data_ptr(), x_t=st[0], x_b=st[1], bf16=x.dtype == torch.bfloat16)
    return L_.ConvArgs(w=weight.data_ptr(), bias=_at(bias), state=_at(state), lengths=_at(lengths), L=shape[0], B=shape[1], C=shape[2],
                       K=weight.shape[1], silu=silu, **more)


def _conv_forward(x, weight, bias, state, lengths, silu):
    y = x.new_empty(x.shape)
    last = x.new_empty((weight.shape[1] - 1, x.shape[1], x.shape[2]))
    a = _conv_args(x, weight, bias, state, lengths, silu, y=y.data_ptr(), state_out=last.data_ptr())
    L_.call('gmt_causal_conv_fwd', ctypes.addressof(a), L_.stream_of(x.get_device()), nbytes=2.0 * x.numel() * x.element_size())
    return y, last


class CausalConvFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, state, lengths, silu, ckpt8):
        y, last = _conv_forward(x, weight, bias, state, lengths, silu)
        packed = ops_ckpt8.pack(x) if ckpt8 else None
        ctx.save_for_backward(*((packed.codes, packed.exponents) if ckpt8 else (x, None)), weight, bias, state, lengths)
        ctx.silu, ctx.dtype, ctx.ckpt8 = silu, x.dtype, ckpt8
        ctx.set_materialize_grads(False)
        return y, last

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dlast):
        x, exps, weight, bias, state, lengths = ctx.saved_tensors
        shape, dtype, K = x.shape, ctx.dtype, weight.shape[1]
        if ctx.ckpt8:
            x = Ckpt8(x, exps, dtype)
        dev = weight.get_device()
        with on(dev):
            dy = weight.new_zeros(shape, dtype=dtype) if dy is None else time_major(dy)
            dlast = _whole(dlast)
            dx = weight.new_empty(shape, dtype=dtype)
            dparam = weight.new_empty((K + 1, shape[2]))
            dstate = None if state is None else torch.empty_like(state)
            st = dy.stride()
            a = _conv_args(x, weight, bias, state, lengths, ctx.silu, dy=dy.data_ptr(), dstate_out=_at(dlast), dx=dx.data_ptr(),
                           dparam=dparam.data_ptr(), dstate=_at(dstate), dy_t=st[0], dy_b=st[1])
            need = ctypes.c_longlong(0)
            L_.call('gmt_causal_conv_bwd_workspace_floats', ctypes.addressof(a), ctypes.addressof(need), label='skip')
            ws = _space(need.value, weight)
            a.workspace, a.workspace_floats = _at(ws), need.value
            L_.call('gmt_causal_conv_bwd', ctypes.addressof(a), L_.stream_of(dev), nbytes=3.0 * dx.numel() * dx.element_size())
        return dx, dparam[:K].t().contiguous(), (None if bias is None else dparam[K]), dstate, None, None, None


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
    lengths = _lengths(lengths, B, L, x)
    args = time_major(x), _whole(weight), _whole(bias), _whole(state), lengths, bool(silu)
    with on(dev):
        if _any_grad(x, weight, bias, state):
            return ops_ckpt8.apply(CausalConvFn, dev, *args, bool(ckpt8))
        return _conv_forward(*args)


def causal_conv_step(x: torch.Tensor, state: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, silu: bool = True,
                     active: Optional[torch.Tensor] = None, state_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One step: x [B, C], state [K-1, B, C] -> y [B, C].  The updated state goes to state_out (None: in place).  Rows whose `active`
    is false keep their state and give zeros."""
    dev = on_device(x, state, weight, bias, state_out)
    C, K = _conv_checks(x, weight, bias, 2)
    B = x.shape[0]
    out = _step_states(state, state_out, (K - 1, B, C), x.dtype)
    if torch.is_grad_enabled():
        _no_grad_only('causal_conv_step', x, state, weight, bias, state_out)
    active = _active(active, B, x)
    x, weight, bias = time_major(x), _whole(weight), _whole(bias)
    with on(dev):
        y = x.new_empty((B, C))
        a = L_.ConvArgs(x=x.data_ptr(), w=weight.data_ptr(), bias=_at(bias), state=state.data_ptr(), y=y.data_ptr(), state_out=out.data_ptr(),
                        x_b=x.stride()[0], L=1, B=B, C=C, K=K, bf16=x.dtype == torch.bfloat16, silu=bool(silu))
        L_.call('gmt_causal_conv_step', ctypes.addressof(a), _at(active), L_.stream_of(dev), nbytes=2.0 * K * B * C * x.element_size())
    torch.autograd.graph.increment_version(out)
    return y


# ----------------------------------------------------------------------------------------
# selective scan
# ----------------------------------------------------------------------------------------
def _map_pitches(m: torch.Tensor, lead: int):
    """Pitches of B or C [.., N] or [.., G, N]: (step, row, group), the step's 0 without a second step."""
    st = m.stride()
    return (st[0] if lead == 2 and m.shape[0] > 1 else 0), st[lead - 1], (st[lead] if m.dim() == lead + 2 else 0)


def _scan_args(x, dt, z, A, B, C, D, dt_bias, state, lengths, **more) -> L_.ScanArgs:
    if isinstance(x, Ckpt8):
        shape = x.codes.shape
        more.update(x=x.codes.data_ptr(), x_scale=x.exponents.data_ptr(), dt=dt.codes.data_ptr(), dt_scale=dt.exponents.data_ptr())
        if z is not None:
            more.update(z=z.codes.data_ptr(), z_scale=z.exponents.data_ptr())
    else:
        shape, xs, ds = x.shape, x.stride(), dt.stride()
        steps = shape[0] > 1                             # (the pitch of a single step may be anything)
        more.update(x=x.data_ptr(), x_t=xs[0] if steps else 0, x_b=xs[1], dt=dt.data_ptr(), dt_t=ds[0] if steps else 0, dt_b=ds[1])
        if z is not None:
            zs = z.stride()
            more.update(z=z.data_ptr(), z_t=zs[0] if steps else 0, z_b=zs[1])
    Bp, Cp = _map_pitches(B, 2), _map_pitches(C, 2)
    return L_.ScanArgs(A=A.data_ptr(), Bm=B.data_ptr(), Cm=C.data_ptr(), D=_at(D), dt_bias=_at(dt_bias), state=_at(state), lengths=_at(lengths),
                       B_t=Bp[0], B_b=Bp[1], B_g=Bp[2], C_t=Cp[0], C_b=Cp[1], C_g=Cp[2], L=shape[0], B=shape[1], C=shape[2], N=A.shape[1],
                       G=1 if B.dim() == 3 else B.shape[2], bf16=B.dtype == torch.bfloat16, **more)


def _workspace(a):
    """Floats of (the kept states, a forward call's workspace, a backward call's)."""
    n = (ctypes.c_longlong * 3)()
    at = ctypes.addressof(n)
    L_.call('gmt_selective_scan_workspace', ctypes.addressof(a), at, at + 8, at + 16, label='skip')
    return n


def _scan_forward(x, dt, A, B, C, D, z, dt_bias, state, lengths, keep):
    y = x.new_empty(x.shape)
    last = A.new_empty((x.shape[1], *A.shape))
    a = _scan_args(x, dt, z, A, B, C, D, dt_bias, state, lengths, y=y.data_ptr(), state_out=last.data_ptr())
    n_ck, n_fwd, n_bwd = _workspace(a)
    ck, ws = _space(n_ck if keep else 0, A), _space(n_fwd, A)
    a.ck, a.workspace, a.workspace_floats = _at(ck), _at(ws), n_fwd
    L_.call('gmt_selective_scan_fwd', ctypes.addressof(a), L_.stream_of(x.get_device()), nbytes=float((3 + (z is not None)) * x.numel() * x.element_size()))
    return y, last, ck, (n_ck, n_bwd)


class SelectiveScanFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, dt, A, B, C, D, z, dt_bias, state, lengths, ckpt8):
        # the state before every eighth step; from 8-bit checkpoints the backward pass finds them itself
        y, last, ck, ctx.floats = _scan_forward(x, dt, A, B, C, D, z, dt_bias, state, lengths, not ckpt8)
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
        shape, dtype, (Ch, N) = x.shape, ctx.dtype, A.shape
        if ctx.ckpt8:
            x, dt = Ckpt8(x, xe, dtype), Ckpt8(dt, dte, dtype)
            z = None if z is None else Ckpt8(z, ze, dtype)
        dev = A.get_device()
        with on(dev):
            dy = A.new_zeros(shape, dtype=dtype) if dy is None else _near(dy, FAR_SEQ)
            dlast = _whole(dlast)
            dx, ddt = A.new_empty(shape, dtype=dtype), A.new_empty(shape, dtype=dtype)
            dz = None if z is None else A.new_empty(shape, dtype=dtype)
            dB, dC = B.new_empty(B.shape), C.new_empty(C.shape)
            dparam = A.new_empty(Ch * (N + 2))
            dstate = None if state is None else torch.empty_like(state)
            st = dy.stride()
            a = _scan_args(x, dt, z, A, B, C, D, dt_bias, state, lengths, dy=dy.data_ptr(), dstate_out=_at(dlast), dx=dx.data_ptr(),
                           ddt=ddt.data_ptr(), dz=_at(dz), dB=dB.data_ptr(), dC=dC.data_ptr(), dparam=dparam.data_ptr(), dstate=_at(dstate),
                           dy_t=st[0] if shape[0] > 1 else 0, dy_b=st[1])
            n_ck, n_bwd = ctx.floats
            if ctx.ckpt8:
                ck = _space(n_ck, A)
            ws = _space(n_bwd, A)
            a.ck, a.workspace, a.workspace_floats = ck.data_ptr(), _at(ws), n_bwd
            L_.call('gmt_selective_scan_bwd', ctypes.addressof(a), L_.stream_of(dev),
                    nbytes=float((5 + 2 * (z is not None)) * dx.numel() * dx.element_size()))
        return (dx, ddt, dparam[:Ch * N].view(Ch, N), dB, dC, None if D is None else dparam[Ch * N:Ch * (N + 1)], dz,
                None if dt_bias is None else dparam[Ch * (N + 1):], dstate, None, None)


def _scan_checks(x, dt, A, B, C, D, z, dt_bias, lead: tuple):
    """Shapes and types of a scan over `lead` = (L, B) or (B,)."""
    shape, dtype = x.shape, x.dtype
    Ch = shape[-1]
    if A.dim() != 2 or not 1 <= A.shape[1] <= MAX_STATES:
        _fail(f'A: [{Ch}, N] with N = 1 .. {MAX_STATES} states expected, got {tuple(A.shape)}')
    N = A.shape[1]
    _want(A, 'A', (Ch, N), torch.float32)
    _want(dt, 'dt', shape, dtype)
    _want(z, 'z', shape, dtype)
    _want(D, 'D', (Ch,), torch.float32)
    _want(dt_bias, 'dt_bias', (Ch,), torch.float32)
    groups = []
    for name, m in (('B', B), ('C', C)):
        G = m.shape[-2] if m.dim() == len(lead) + 2 else 1
        if G < 1 or Ch % G or m.shape != ((*lead, N) if m.dim() == len(lead) + 1 else (*lead, G, N)) or m.dtype != dtype:
            _fail(f'{name}: {dtype} {(*lead, N)} or {(*lead, "G", N)} with G dividing {Ch} channels expected, got {m.dtype} {tuple(m.shape)}')
        groups.append(G)
    if groups[0] != groups[1]:
        _fail(f'B and C have different groups: {groups[0]} and {groups[1]}')


def selective_scan(x: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor, D: Optional[torch.Tensor] = None,
                   z: Optional[torch.Tensor] = None, dt_bias: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None,
                   state: Optional[torch.Tensor] = None, ckpt8: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """x, dt [L, B, C] (and the gate z, or None), A [C, N] (N <= 32), B and C [L, B, N] or [L, B, G, N] (G groups of C / G neighbouring
    channels share them), D and dt_bias [C], state [B, C, N] fp32 (None: zeros) -> (y [L, B, C], the state after each row's
    last step).  ckpt8: x, dt and z are kept in 8 bits for the backward pass, which then finds the states again."""
    dev = on_device(x, dt, A, B, C, D, z, dt_bias, state)
    _seq(x, 'x', 3)
    L, Bt, Ch = x.shape
    _scan_checks(x, dt, A, B, C, D, z, dt_bias, (L, Bt))
    _want(state, 'state', (Bt, Ch, A.shape[1]), torch.float32)
    lengths = _lengths(lengths, Bt, L, x)
    args = (_near(x, FAR_SEQ), _near(dt, FAR_SEQ), _whole(A), _near(B, FAR_MAP), _near(C, FAR_MAP), _whole(D), None if z is None else _near(z, FAR_SEQ),
            _whole(dt_bias), _whole(state), lengths)
    with on(dev):
        if _any_grad(x, dt, A, B, C, D, z, dt_bias, state):
            return ops_ckpt8.apply(SelectiveScanFn, dev, *args, bool(ckpt8))
        return _scan_forward(*args, False)[:2]


def selective_scan_step(x: torch.Tensor, dt: torch.Tensor, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor, state: torch.Tensor,
                        D: Optional[torch.Tensor] = None, z: Optional[torch.Tensor] = None, dt_bias: Optional[torch.Tensor] = None,
                        active: Optional[torch.Tensor] = None, state_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One step: x, dt (z) [B, C], B and C [B, N] or [B, G, N], state [B, C, N] fp32 -> y [B, C].  The updated state goes to state_out
    (None: in place).  Rows whose `active` is false keep their state and give zeros."""
    dev = on_device(x, dt, A, B, C, state, D, z, dt_bias, state_out)
    _seq(x, 'x', 2)
    Bt, Ch = x.shape
    _scan_checks(x, dt, A, B, C, D, z, dt_bias, (Bt,))
    N = A.shape[1]
    out = _step_states(state, state_out, (Bt, Ch, N), torch.float32)
    if torch.is_grad_enabled():
        _no_grad_only('selective_scan_step', x, dt, A, B, C, state, D, z, dt_bias, state_out)
    active = _active(active, Bt, x)
    x, dt, B, C = time_major(x), time_major(dt), time_major(B), time_major(C)
    A, D, dt_bias = _whole(A), _whole(D), _whole(dt_bias)
    z = None if z is None else time_major(z)
    Bp, Cp = _map_pitches(B, 1), _map_pitches(C, 1)
    with on(dev):
        y = x.new_empty((Bt, Ch))
        a = L_.ScanArgs(x=x.data_ptr(), dt=dt.data_ptr(), z=_at(z), Bm=B.data_ptr(), Cm=C.data_ptr(), A=A.data_ptr(), D=_at(D),
                        dt_bias=_at(dt_bias), state=state.data_ptr(), y=y.data_ptr(), state_out=out.data_ptr(), x_b=x.stride()[0],
                        dt_b=dt.stride()[0], z_b=0 if z is None else z.stride()[0], B_b=Bp[1], B_g=Bp[2], C_b=Cp[1], C_g=Cp[2],
                        L=1, B=Bt, C=Ch, N=N, G=1 if B.dim() == 2 else B.shape[1], bf16=x.dtype == torch.bfloat16)
        L_.call('gmt_selective_scan_step', ctypes.addressof(a), _at(active), L_.stream_of(dev), nbytes=8.0 * Bt * Ch * N)
    torch.autograd.graph.increment_version(out)
    return y
