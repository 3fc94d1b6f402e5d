"""Plain definitions of the selective state-space operators and of the 8-bit checkpoints in float64 on the CPU: one step after the
other, gradients by autograd.  Tolerances (derived from the number of roundings) for the GPU tests."""
import torch
import torch.nn.functional as F

U32 = 2.0 ** -24                                          # half a step of fp32, relative
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def d(t):
    return None if t is None else t.detach().double().cpu()


def stands_for(x):
    """The values of the 8-bit checkpoint of x [..., C]: an independent search for the smallest power of two per block of 32."""
    C = x.shape[-1]
    rows = F.pad(x.double(), (0, -C % 32)).reshape(-1, 32)
    out = torch.empty_like(rows)
    for i, r in enumerate(rows):
        if not torch.isfinite(r).all():
            out[i] = float('nan')
            continue
        e = -118
        while e < 121 and float(r.abs().max()) > 127 * 2.0 ** e:
            e += 1
        out[i] = torch.clamp(torch.round(r / 2.0 ** e), -127, 127) * 2.0 ** e
    return out.reshape(*x.shape[:-1], -1)[..., :C]


def conv(x, w, b, lengths, state, silu=True):
    L, B, C = x.shape
    K = w.shape[1]
    n = torch.full((B,), L) if lengths is None else lengths.long().cpu().clamp(0, L)
    window = [torch.zeros(B, C, dtype=x.dtype)] * (K - 1) if state is None else list(state)
    ys = []
    for t in range(L):
        on = (t < n)[:, None]
        window = window + [torch.where(on, x[t], torch.zeros_like(x[t]))]
        pre = sum(window[k] * w[:, k] for k in range(K)) + (0 if b is None else b)
        ys.append(torch.where(on, F.silu(pre) if silu else pre, torch.zeros_like(pre)))
        window = [torch.where(on, window[k + 1], window[k]) for k in range(K - 1)]
    return torch.stack(ys), torch.stack(window)


def scan(x, dt, A, B, C, D, z, dt_bias, lengths, state):
    L, Bt, Ch = x.shape
    if B.dim() == 3:
        B, C = B.unsqueeze(2), C.unsqueeze(2)
    per = Ch // B.shape[2]
    n = torch.full((Bt,), L) if lengths is None else lengths.long().cpu().clamp(0, L)
    h = torch.zeros(Bt, Ch, A.shape[1], dtype=x.dtype) if state is None else state
    zero = torch.zeros((), dtype=x.dtype)
    ys = []
    for t in range(L):
        on = (t < n)[:, None]
        xt, dtt = torch.where(on, x[t], zero), torch.where(on, dt[t], zero)
        Bv, Cv = (torch.where(on[:, :, None], m[t], zero).repeat_interleave(per, 1) for m in (B, C))
        step = F.softplus(dtt if dt_bias is None else dtt + dt_bias, threshold=1e9)
        new = torch.exp(step[..., None] * A) * h + (step * xt)[..., None] * Bv
        y = (new * Cv).sum(-1) + (0 if D is None else D * xt)
        if z is not None:
            y = y * F.silu(torch.where(on, z[t], zero))
        ys.append(torch.where(on, y, zero))
        h = torch.where(on[:, :, None], new, h)
    return torch.stack(ys), h


def close(got, want, roundings, what):
    """Largest error <= (roundings of fp32 arithmetic + one of the output's type) half steps of the largest magnitude."""
    assert got.shape == want.shape, f'{what}: shape {tuple(got.shape)}, not {tuple(want.shape)}'
    tol = roundings * U32 + (HALF_STEP[got.dtype] if got.dtype != torch.float32 else 0.0)
    g, w = d(got), d(want)
    assert torch.isfinite(g).all(), f'{what}: not finite'
    scale = max(float(w.abs().max()), 1e-30) if w.numel() else 1.0
    err = float((g - w).abs().max()) / scale if w.numel() else 0.0
    assert err <= tol, f'{what}: error {err:.3e} of the largest magnitude, {tol:.3e} allowed'
