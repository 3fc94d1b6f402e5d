"""GPU tests of the short causal convolution and the selective scan against their definitions in float64 (tests/ssm_reference.py).

Tolerance: half steps of fp32 (2^-24) of the largest magnitude, counted along the longest chain of roundings: a state passes 3 a step
(exponent, product, sum) and its input 40 (softplus, silu), a sum over N states or K taps N or K, a parameter's gradient one per
step and one per partial sum; a gradient passes the chain forwards and backwards.  A bf16 output adds its own half step, 2^-8."""
import pytest
import torch

import ssm_reference as R

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'


def ragged(L, B):
    """Lengths that end before, at and behind chunk borders, with an empty row and one of a single step."""
    some = [L, 0, 1, L // 2, max(L - 1, 0), min(8, L), min(9, L), min(L, 3)]
    return torch.tensor([some[i % len(some)] for i in range(B)], dtype=torch.int32)


def grads(outs, leaves, adj):
    return torch.autograd.grad(outs, leaves, adj, allow_unused=True)


CONV = [  # L, B, C, K, dtype, bias, ragged, state, silu, ckpt8
    (1, 1, 1, 2, 'fp32', True, False, False, True, False),
    (1, 3, 33, 4, 'bf16', True, False, True, True, False),
    (2, 5, 64, 4, 'fp32', False, True, True, True, False),
    (7, 9, 40, 3, 'bf16', True, True, False, True, True),
    (17, 4, 250, 3, 'fp32', True, True, True, False, False),
    (129, 33, 96, 4, 'fp32', True, True, True, True, True),
    (200, 3, 512, 4, 'bf16', True, True, True, True, False),
    (300, 2, 7, 2, 'bf16', True, True, True, True, True),
    (50, 700, 24, 4, 'bf16', True, False, False, True, False),
]


@pytest.mark.parametrize('L,B,C,K,dtype,with_bias,rag,with_state,silu,ckpt8', CONV)
def test_conv_forward_backward(L, B, C, K, dtype, with_bias, rag, with_state, silu, ckpt8):
    from generative_mouse_trajectories_amd import ops_ssm
    dt = {'fp32': torch.float32, 'bf16': torch.bfloat16}[dtype]
    gen = torch.Generator().manual_seed(L * 1000 + C)
    x = torch.randn(L, B, C, generator=gen).to(dt)
    w, b = torch.randn(C, K, generator=gen), torch.randn(C, generator=gen) if with_bias else None
    state = torch.randn(K - 1, B, C, generator=gen).to(dt) if with_state else None
    lengths = ragged(L, B) if rag else None
    ay, al = torch.randn(L, B, C, generator=gen).to(dt), torch.randn(K - 1, B, C, generator=gen).to(dt)

    leaves = [t.to(DEV).requires_grad_(True) for t in (x, w, b, state) if t is not None]
    it = iter(leaves)
    gx, gw, gb, gs = (next(it) if t is not None else None for t in (x, w, b, state))
    dirty = gx
    if rag:                                               # what lies behind a row's end may hold anything
        behind = (torch.arange(L)[:, None] >= lengths[None, :])[:, :, None].to(DEV)
        dirty = torch.where(behind, torch.full_like(gx, float('nan')), gx)
        ay_dirty = torch.where(behind, torch.full_like(ay.to(DEV), float('nan')), ay.to(DEV))
    else:
        ay_dirty = ay.to(DEV)
    y, last = ops_ssm.causal_conv(dirty, gw, gb, lengths=None if lengths is None else lengths.to(DEV), state=gs, silu=silu, ckpt8=ckpt8)
    got = grads([y, last], leaves, [ay_dirty, al.to(DEV)])

    ref = [R.d(t).requires_grad_(True) for t in (x, w, b, state) if t is not None]
    it = iter(ref)
    rx, rw, rb, rs = (next(it) if t is not None else None for t in (x, w, b, state))
    with torch.no_grad():
        wy, wl = R.conv(rx, rw, rb, lengths, rs, silu)
    n = 45 + K
    R.close(y, wy, n, 'y')
    assert torch.equal(R.d(last), wl), 'the final state is a copy of inputs'
    if ckpt8:
        rx = R.stands_for(x).requires_grad_(True)
        ref[0] = rx
    outs = R.conv(rx, rw, rb, lengths, rs, silu)
    want = grads(outs, ref, [R.d(ay), R.d(al)])
    for name, g, v in zip([k for k, t in (('x', x), ('weight', w), ('bias', b), ('state', state)) if t is not None], got, want):
        R.close(g, torch.zeros_like(R.d(g)) if v is None else v, 90 + 2 * K + (L * 4 + 64 if name in ('weight', 'bias') else 0), 'd' + name)


SCAN = [  # L, B, C, N, G, dtype, gate, D and bias, ragged, state, ckpt8
    (1, 1, 1, 1, 1, 'fp32', False, False, False, False, False),
    (1, 3, 64, 16, 1, 'bf16', True, True, False, True, False),
    (2, 4, 65, 5, 1, 'fp32', True, True, True, True, False),
    (8, 2, 32, 8, 2, 'fp32', True, False, False, False, False),
    (9, 9, 100, 16, 1, 'bf16', False, True, True, True, True),
    (31, 8, 48, 32, 3, 'fp32', True, True, True, True, False),
    (40, 5, 128, 17, 1, 'bf16', True, True, True, False, True),
    (129, 9, 96, 16, 2, 'fp32', True, True, True, True, False),        # cut into segments from here on
    (129, 3, 300, 16, 1, 'fp32', True, True, True, True, True),        # two workgroups across the channels
    (300, 8, 40, 7, 1, 'bf16', True, True, True, True, False),
    (257, 2, 600, 16, 2, 'bf16', False, True, False, True, False),
    (200, 1, 64, 32, 1, 'fp32', True, True, False, False, True),
    (20, 300, 130, 16, 1, 'fp32', True, True, True, False, False),     # many rows: not cut, several rows a workgroup
]


def scan_inputs(L, B, C, N, G, dt, gate, extras, with_state, seed):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    t = {'x': r(L, B, C).to(dt), 'dt': (0.7 * r(L, B, C)).to(dt), 'A': -torch.exp(0.5 * r(C, N)) * torch.arange(1, N + 1) ** 0.5,
         'B': r(L, B, G, N).to(dt), 'C': r(L, B, G, N).to(dt), 'D': 1 + 0.3 * r(C) if extras else None,
         'z': r(L, B, C).to(dt) if gate else None, 'dt_bias': r(C) - 3 if extras else None, 'state': r(B, C, N) if with_state else None}
    return t, r(L, B, C).to(dt), r(B, C, N)


NAMES = ('x', 'dt', 'A', 'B', 'C', 'D', 'z', 'dt_bias', 'state')


@pytest.mark.parametrize('L,B,C,N,G,dtype,gate,extras,rag,with_state,ckpt8', SCAN)
def test_scan_forward_backward(L, B, C, N, G, dtype, gate, extras, rag, with_state, ckpt8):
    from generative_mouse_trajectories_amd import ops_ssm
    dt = {'fp32': torch.float32, 'bf16': torch.bfloat16}[dtype]
    t, ay, al = scan_inputs(L, B, C, N, G, dt, gate, extras, with_state, L * 7 + C)
    lengths = ragged(L, B) if rag else None
    names = [k for k in NAMES if t[k] is not None]
    leaves = {k: t[k].to(DEV).requires_grad_(True) for k in names}
    call = {k: leaves.get(k) for k in NAMES}
    ayd = ay.to(DEV)
    if rag:
        behind = (torch.arange(L)[:, None] >= lengths[None, :])[:, :, None].to(DEV)
        for k in ('x', 'dt', 'z'):
            if call[k] is not None:
                call[k] = torch.where(behind, torch.full_like(call[k], float('nan')), call[k])
        for k in ('B', 'C'):
            call[k] = torch.where(behind[..., None], torch.full_like(call[k], float('inf')), call[k])
        ayd = torch.where(behind, torch.full_like(ayd, float('nan')), ayd)
    y, last = ops_ssm.selective_scan(call['x'], call['dt'], call['A'], call['B'], call['C'], D=call['D'], z=call['z'],
                                     dt_bias=call['dt_bias'], state=call['state'], ckpt8=ckpt8,
                                     lengths=None if lengths is None else lengths.to(DEV))
    got = dict(zip(names, grads([y, last], [leaves[k] for k in names], [ayd, al.to(DEV)])))

    ref = {k: R.d(t[k]) for k in NAMES}
    with torch.no_grad():
        wy, wl = R.scan(*(ref[k] for k in NAMES[:8]), lengths, ref['state'])
    chain = 3 * L + N + 45
    R.close(y, wy, chain, 'y')
    R.close(last, wl, chain, 'final state')
    if ckpt8:
        for k in ('x', 'dt', 'z'):
            if ref[k] is not None:
                ref[k] = R.stands_for(t[k])
    rl = {k: ref[k].clone().requires_grad_(True) for k in names}
    outs = R.scan(*(rl.get(k) for k in NAMES[:8]), lengths, rl.get('state'))
    want = dict(zip(names, grads(outs, [rl[k] for k in names], [R.d(ay), R.d(al)])))
    for k in names:
        extra = {'A': L + 80, 'D': L + 80, 'dt_bias': L + 80, 'B': C, 'C': C}.get(k, 0)
        assert got[k].dtype == t[k].dtype
        R.close(got[k], torch.zeros_like(R.d(t[k])) if want[k] is None else want[k], 2 * chain + 45 + extra, 'd' + k)


@pytest.mark.parametrize('B,C,N,G,ckpt8', [(600, 256, 3, 1, False), (1024, 250, 2, 1, True), (1025, 256, 2, 1, False), (700, 512, 2, 2, False)])
def test_many_rows_of_unequal_length(B, C, N, G, ckpt8):
    """Rows are taken in another order than they are stored in, several to a workgroup; the inputs of equal and empty rows stay apart; a
    workgroup sums the parameters' gradients over at most two or three rows."""
    from generative_mouse_trajectories_amd import ops_ssm
    L = 10
    t, ay, al = scan_inputs(L, B, C, N, G, torch.float32, True, True, True, B + N)
    if ckpt8:                                                # values that 8-bit checkpoints hold exactly
        t.update({k: (t[k] * 32).round().clamp(-100, 100) / 32 for k in ('x', 'dt', 'z')})
    lengths = torch.randint(0, L + 1, (B,), generator=torch.Generator().manual_seed(B), dtype=torch.int32)
    lengths[0], lengths[1], lengths[B - 2], lengths[B - 1] = 0, L, L, 0
    leaves = {k: t[k].to(DEV).requires_grad_(True) for k in NAMES}
    outside = lengths.clone()
    outside[0], outside[1] = -7, L + 100                     # read as 0 and L
    y, last = ops_ssm.selective_scan(*(leaves[k] for k in ('x', 'dt', 'A', 'B', 'C')), D=leaves['D'], z=leaves['z'],
                                     dt_bias=leaves['dt_bias'], state=leaves['state'], ckpt8=ckpt8, lengths=outside.to(DEV))
    got = dict(zip(NAMES, grads([y, last], [leaves[k] for k in NAMES], [ay.to(DEV), al.to(DEV)])))
    ref = {k: R.d(t[k]) for k in NAMES}
    chain = 3 * L + N + 45
    with torch.no_grad():
        wy, wl = R.scan(*(ref[k] for k in NAMES[:8]), lengths, ref['state'])
    R.close(y, wy, chain, 'y')
    R.close(last, wl, chain, 'final state')
    rl = {k: ref[k].clone().requires_grad_(True) for k in NAMES}
    outs = R.scan(*(rl[k] for k in NAMES[:8]), lengths, rl['state'])
    want = dict(zip(NAMES, grads(outs, [rl[k] for k in NAMES], [R.d(ay), R.d(al)])))
    for k in NAMES:
        extra = {'A': 3 * L + 80, 'D': 3 * L + 80, 'dt_bias': 3 * L + 80, 'B': C // G, 'C': C // G}.get(k, 0)
        R.close(got[k], want[k], 2 * chain + 45 + extra, 'd' + k)


def test_states_found_again_in_segments_that_the_backward_pass_does_not_have():
    """38 rows of 273 channels: the forward pass is cut into segments, the backward pass from 8-bit checkpoints is not."""
    from generative_mouse_trajectories_amd import ops_ssm
    L, B, C, N = 197, 38, 273, 2
    t, ay, al = scan_inputs(L, B, C, N, 1, torch.float32, True, True, True, 5)
    t.update({k: (t[k] * 32).round().clamp(-100, 100) / 32 for k in ('x', 'dt', 'z')})       # held exactly by the checkpoints
    lengths = ragged(L, B)
    leaves = {k: t[k].to(DEV).requires_grad_(True) for k in NAMES}
    outs = ops_ssm.selective_scan(*(leaves[k] for k in ('x', 'dt', 'A', 'B', 'C')), D=leaves['D'], z=leaves['z'], dt_bias=leaves['dt_bias'],
                                  state=leaves['state'], lengths=lengths.to(DEV), ckpt8=True)
    got = grads(outs, list(leaves.values()), [ay.to(DEV), al.to(DEV)])
    rl = {k: R.d(t[k]).requires_grad_(True) for k in NAMES}
    want = grads(R.scan(*(rl[k] for k in NAMES[:8]), lengths, rl['state']), list(rl.values()), [R.d(ay), R.d(al)])
    chain = 3 * L + N + 45
    for k, g, w in zip(NAMES, got, want):
        extra = {'A': L + 80, 'D': L + 80, 'dt_bias': L + 80, 'B': C, 'C': C}.get(k, 0)
        R.close(g, w, 2 * chain + 45 + extra, 'd' + k)


def test_gradients_against_differences():
    """Directional derivatives of the operators' own outputs (fp32, summed in float64): central differences of width h err by
    h^2 / 6 of the third derivative plus the outputs' rounding over h; h = 2^-6 and outputs of size 1 leave under 2e-3."""
    from generative_mouse_trajectories_amd import ops_ssm
    L, B, C, N = 12, 3, 33, 6
    t, ay, al = scan_inputs(L, B, C, N, 1, torch.float32, True, True, True, 5)
    gen = torch.Generator().manual_seed(9)
    w, b = torch.randn(C, 4, generator=gen).to(DEV), torch.randn(C, generator=gen).to(DEV)
    vals = {k: v.to(DEV) for k, v in t.items()}
    lengths = torch.tensor([12, 7, 1], dtype=torch.int32, device=DEV)

    def loss(v):
        u, _ = ops_ssm.causal_conv(v['x'], w, b, lengths=lengths)
        y, last = ops_ssm.selective_scan(u, v['dt'], v['A'], v['B'], v['C'], D=v['D'], z=v['z'], dt_bias=v['dt_bias'], lengths=lengths,
                                         state=v['state'])
        return (y.double() * ay.to(DEV).double()).sum() + (last.double() * al.to(DEV).double()).sum()

    leaves = {k: v.clone().requires_grad_(True) for k, v in vals.items()}
    got = torch.autograd.grad(loss(leaves), list(leaves.values()))
    h = 2.0 ** -6
    for k, g in zip(leaves, got):
        dirn = torch.randn(vals[k].shape, generator=gen).to(DEV)
        dirn = dirn / dirn.norm()
        with torch.no_grad():
            num = (loss({**vals, k: vals[k] + h * dirn}) - loss({**vals, k: vals[k] - h * dirn})) / (2 * h)
        ana = (g.double() * dirn.double()).sum()
        scale = max(float(g.norm()), 1.0)
        assert abs(float(num - ana)) <= 2e-3 * scale, (k, float(num), float(ana))


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('C,N,G', [(64, 16, 1), (33, 5, 1), (100, 12, 2), (40, 32, 4), (7, 1, 7)])
def test_prompt_and_single_steps_agree(C, N, G, dtype):
    """The first steps in one call, the rest one by one from its states, against one call over all steps; the single steps also
    against the definition.  Inactive rows keep their states and give zeros."""
    from generative_mouse_trajectories_amd import ops_ssm
    L, B, K, P = 21, 5, 4, 13
    t, _, _ = scan_inputs(L, B, C, N, G, dtype, True, True, True, C)
    v = {k: a.to(DEV) for k, a in t.items()}
    gen = torch.Generator().manual_seed(3)
    w, b = torch.randn(C, K, generator=gen).to(DEV), torch.randn(C, generator=gen).to(DEV)
    with torch.no_grad():
        wu, wc = ops_ssm.causal_conv(v['x'], w, b)
        wy, wh = ops_ssm.selective_scan(wu, v['dt'], v['A'], v['B'], v['C'], D=v['D'], z=v['z'], dt_bias=v['dt_bias'], state=v['state'])
        u, cs = ops_ssm.causal_conv(v['x'][:P], w, b)
        y, h = ops_ssm.selective_scan(u, v['dt'][:P], v['A'], v['B'][:P], v['C'][:P], D=v['D'], z=v['z'][:P], dt_bias=v['dt_bias'],
                                      state=v['state'])
        ys = [y]
        for s in range(P, L):
            if s == P + 2:                                # a step in which only rows 1 and 3 are active, undone afterwards
                act = torch.tensor([False, True, False, True, False], device=DEV)
                c0, h0 = cs.clone(), h.clone()
                uu = ops_ssm.causal_conv_step(v['x'][s], cs, w, b, active=act)
                yy = ops_ssm.selective_scan_step(uu, v['dt'][s], v['A'], v['B'][s], v['C'][s], h, D=v['D'], z=v['z'][s],
                                                 dt_bias=v['dt_bias'], active=act)
                off = ~act
                assert torch.equal(cs[:, off], c0[:, off]) and torch.equal(h[off], h0[off]) and not torch.equal(h[act], h0[act])
                assert float(uu[off].abs().max()) == 0 and float(yy[off].abs().max()) == 0
                cs, h = c0, h0
            if s % 2:                                     # in place, and into another buffer
                us = ops_ssm.causal_conv_step(v['x'][s], cs, w, b)
                yn = ops_ssm.selective_scan_step(us, v['dt'][s], v['A'], v['B'][s], v['C'][s], h, D=v['D'], z=v['z'][s], dt_bias=v['dt_bias'])
            else:
                c2, h2 = torch.empty_like(cs), torch.empty_like(h)
                before = h.clone()
                us = ops_ssm.causal_conv_step(v['x'][s], cs, w, b, state_out=c2)
                yn = ops_ssm.selective_scan_step(us, v['dt'][s], v['A'], v['B'][s], v['C'][s], h, D=v['D'], z=v['z'][s], dt_bias=v['dt_bias'],
                                                 state_out=h2)
                assert torch.equal(h, before)
                cs, h = c2, h2
            ys.append(yn[None])
    chain = 3 * L + N + 45
    got = torch.cat(ys)
    # both sides carry the chain's roundings, and in bf16 the convolution's output may round to either neighbour
    slack = chain + (2.0 ** 17 if dtype == torch.bfloat16 else 0)
    R.close(got, wy, slack, 'y')
    R.close(h, wh, slack, 'state')
    assert torch.equal(cs, wc)


def test_rows_do_not_depend_on_each_other():
    """A row of a batch equals the row alone, to the bit, where both run uncut; lengths beyond 0 .. L are taken as 0 and L."""
    from generative_mouse_trajectories_amd import ops_ssm
    L, B, C, N = 40, 6, 64, 16
    t, _, _ = scan_inputs(L, B, C, N, 1, torch.float32, True, True, True, 2)
    v = {k: a.to(DEV) for k, a in t.items()}
    names = ('x', 'dt', 'B', 'C', 'z')

    def run(rows, lengths):
        s = {k: v[k][:, rows] for k in names}
        return ops_ssm.selective_scan(s['x'], s['dt'], v['A'], s['B'], s['C'], D=v['D'], z=s['z'], dt_bias=v['dt_bias'],
                                      state=v['state'][rows], lengths=lengths)
    y, h = run(slice(0, B), None)
    y1, h1 = run(slice(2, 3), None)
    assert torch.equal(y[:, 2:3], y1) and torch.equal(h[2:3], h1)
    y2, h2 = run(slice(0, B), torch.tensor([L, L + 5, 2 ** 31 - 1, L, L, -4], dtype=torch.int32, device=DEV))
    assert torch.equal(y2[:, :5], y[:, :5]) and torch.equal(h2[:5], h[:5])
    assert float(y2[:, 5].abs().max()) == 0 and torch.equal(h2[5], v['state'][5])
    y3, _ = run(slice(0, B), torch.tensor([L, 2 ** 40, L, L, L, -2 ** 40], dtype=torch.int64, device=DEV))
    assert torch.equal(y3, y2)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_strided_inputs(dtype):
    """Slices of one projection's output, batch-first tensors and expanded maps give what contiguous copies give, to the bit."""
    from generative_mouse_trajectories_amd import ops_ssm
    L, B, C, N = 19, 6, 40, 8
    gen = torch.Generator().manual_seed(4)
    wide = torch.randn(B, L, 3 * C + 2 * N + 1, generator=gen).to(DEV, dtype).requires_grad_(True)      # batch-first, odd pitch
    A = -torch.exp(torch.randn(C, N, generator=gen)).to(DEV)
    w = torch.randn(C, 3, generator=gen).to(DEV)
    one = torch.randn(1, 1, 1, N, generator=gen).to(DEV, dtype).requires_grad_(True)

    def parts(t):
        t = t.transpose(0, 1)
        return t[..., 1:C + 1], t[..., C + 1:2 * C + 1], t[..., 2 * C + 1:3 * C + 1], t[..., 3 * C + 1:3 * C + 1 + N], t[..., 3 * C + 1 + N:]

    def run(copy):
        x, dt, z, Bm, Cm = (p.contiguous() if copy else p for p in parts(wide))
        Cm = Cm.unsqueeze(2) * 0 + one if copy else one.expand(L, B, 1, N)
        u, last = ops_ssm.causal_conv(x, w)
        y, h = ops_ssm.selective_scan(u, dt, A, Bm, Cm if copy else Cm.squeeze(2), z=z) if not copy else \
            ops_ssm.selective_scan(u, dt, A, Bm, Cm, z=z)
        g = torch.autograd.grad((y.float() ** 2).sum() + (h ** 2).sum(), [wide, one])
        with torch.no_grad():
            ys = ops_ssm.selective_scan_step(x[3], dt[3], A, Bm[3], (Cm[3] if copy else Cm.squeeze(2)[3]), h.clone(), z=z[3])
        return (y, h, last, ys, *g)
    for a, b in zip(run(False), run(True)):
        assert torch.equal(a, b)
    # an input whose last axis is not contiguous is copied
    xt = torch.randn(C, L, B, generator=gen).to(DEV, dtype).permute(1, 2, 0)
    assert torch.equal(ops_ssm.causal_conv(xt, w)[0], ops_ssm.causal_conv(xt.contiguous(), w)[0])


def test_adjoints_of_one_output_and_no_grad():
    """Only y or only the final state differentiated; an expanded adjoint; no graph under no_grad."""
    from generative_mouse_trajectories_amd import ops_ssm
    L, B, C, N = 11, 3, 33, 4
    t, _, _ = scan_inputs(L, B, C, N, 1, torch.float32, True, True, True, 8)
    leaves = {k: a.to(DEV).requires_grad_(True) for k, a in t.items()}
    ref = {k: R.d(a).requires_grad_(True) for k, a in t.items()}

    def both(pick):
        y, h = ops_ssm.selective_scan(*(leaves[k] for k in NAMES[:5]), **{k: leaves[k] for k in NAMES[5:]})
        ry, rh = R.scan(*(ref[k] for k in NAMES[:8]), None, ref['state'])
        g = torch.autograd.grad(pick(y, h), list(leaves.values()), allow_unused=True)
        w = torch.autograd.grad(pick(ry, rh), list(ref.values()), allow_unused=True)
        for k, a, b in zip(leaves, g, w):
            R.close(a, torch.zeros_like(R.d(a)) if b is None else b, 2 * (3 * L + N + 45) + 45 + L + 80 + C, k)
    both(lambda y, h: y.sum())
    both(lambda y, h: h.sum())
    with torch.no_grad():
        y, h = ops_ssm.selective_scan(*(leaves[k] for k in NAMES[:5]), **{k: leaves[k] for k in NAMES[5:]})
        assert not y.requires_grad and not h.requires_grad
        cy, _ = ops_ssm.causal_conv(leaves['x'], torch.ones(C, 2, device=DEV).requires_grad_(True))
        assert not cy.requires_grad


def test_repeatable_to_the_bit():
    from generative_mouse_trajectories_amd import ops_ssm
    L, B, C, N = 150, 40, 300, 16
    t, ay, al = scan_inputs(L, B, C, N, 1, torch.bfloat16, True, True, True, 6)
    leaves = {k: a.to(DEV).requires_grad_(True) for k, a in t.items()}

    def run():
        y, h = ops_ssm.selective_scan(*(leaves[k] for k in NAMES[:5]), **{k: leaves[k] for k in NAMES[5:]})
        return (y, h, *torch.autograd.grad([y, h], list(leaves.values()), [ay.to(DEV), al.to(DEV)]))
    first = run()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, run()))


def test_other_stream_and_graph_replays():
    """On a side stream; a captured training pass and a captured single step, replayed between eager work on other inputs."""
    from generative_mouse_trajectories_amd import ops_ssm
    L, B, C, N = 130, 4, 64, 16
    t, ay, al = scan_inputs(L, B, C, N, 1, torch.float32, True, True, True, 12)
    t2, _, _ = scan_inputs(L, B, C, N, 1, torch.float32, True, True, True, 13)
    gen = torch.Generator().manual_seed(1)
    w = torch.randn(C, 4, generator=gen).to(DEV).requires_grad_(True)
    ay, al = ay.to(DEV), al.to(DEV)
    leaves = {k: a.to(DEV).requires_grad_(True) for k, a in t.items()}

    def train(ckpt8):
        u, last = ops_ssm.causal_conv(leaves['x'], w, ckpt8=ckpt8)
        y, h = ops_ssm.selective_scan(u, *(leaves[k] for k in NAMES[1:5]), **{k: leaves[k] for k in NAMES[5:]}, ckpt8=ckpt8)
        return (y.detach(), h.detach(), last.detach(), *torch.autograd.grad([y, h], [w, *leaves.values()], [ay, al]))

    state_c, state_h = torch.zeros(3, B, C, device=DEV), torch.zeros(B, C, N, device=DEV)

    def token():
        with torch.no_grad():
            u = ops_ssm.causal_conv_step(leaves['x'][0], state_c, w)
            return ops_ssm.selective_scan_step(u, leaves['dt'][0], leaves['A'], leaves['B'][0], leaves['C'][0], state_h, D=leaves['D'],
                                               z=leaves['z'][0], dt_bias=leaves['dt_bias'])
    side = torch.cuda.Stream()
    for ckpt8 in (False, True):
        eager = train(ckpt8)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            there = train(ckpt8)
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, b) for a, b in zip(eager, there))
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            captured = train(ckpt8)
        for other in (t2, t, t2):
            with torch.no_grad():
                for k in leaves:
                    leaves[k].copy_(other[k].to(DEV))
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(captured, train(ckpt8)))
        with torch.no_grad():
            for k in leaves:
                leaves[k].copy_(t[k].to(DEV))
        del g, captured
    token()
    state_c.zero_(); state_h.zero_()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = token()
    state_c.zero_(); state_h.zero_()
    got = []
    for _ in range(4):
        g.replay()
        torch.cuda.synchronize()
        got.append((out.clone(), state_h.clone()))
        train(False)
    state_c.zero_(); state_h.zero_()
    for y, h in got:
        assert torch.equal(token(), y) and torch.equal(state_h, h)


def test_capture_beside_a_live_eager_graph_is_refused():
    """... before anything is captured; once the eager graph has gone the same pass is captured and replayed."""
    from generative_mouse_trajectories_amd import ops, ops_ssm
    from generative_mouse_trajectories_amd._lib import GmtError
    t, ay, al = scan_inputs(9, 3, 40, 5, 1, torch.float32, True, True, True, 21)
    leaves = {k: a.to(DEV).requires_grad_(True) for k, a in t.items()}
    w, conv = (torch.randn(40, n, generator=torch.Generator().manual_seed(n)).to(DEV).requires_grad_(True) for n in (40, 4))
    ay = ay.to(DEV)

    def passes():
        u, _ = ops_ssm.causal_conv(ops.linear(leaves['x'], w, None, ckpt8=True), conv)
        return ops_ssm.selective_scan(u, *(leaves[k] for k in NAMES[1:5]), **{k: leaves[k] for k in NAMES[5:]})[0]

    def train():
        return torch.autograd.grad(passes(), [w, conv, *leaves.values()], ay)
    eager = passes()
    for call in (passes, lambda: ops.linear(leaves['x'].detach(), w, None, ckpt8=True), lambda: ops_ssm.causal_conv(leaves['z'] * 2, conv)):
        with pytest.raises(GmtError, match='eagerly on the default stream'):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                call()
    want = torch.autograd.grad(eager, [w, conv, *leaves.values()], ay)
    del eager
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = train()
    for _ in range(3):
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        want = train()


def test_two_streams_at_once_and_inference_mode():
    """Training passes on two streams without a wait between them; the same call under inference_mode."""
    from generative_mouse_trajectories_amd import ops_ssm
    L, B, C, N = 150, 6, 96, 16
    runs = []
    for seed in (31, 32):
        t, ay, al = scan_inputs(L, B, C, N, 1, torch.float32, True, True, True, seed)
        runs.append(({k: a.to(DEV).requires_grad_(True) for k, a in t.items()}, ay.to(DEV), al.to(DEV)))

    def run(leaves, ay, al):
        y, h = ops_ssm.selective_scan(*(leaves[k] for k in NAMES[:5]), **{k: leaves[k] for k in NAMES[5:]})
        return (y, h, *torch.autograd.grad([y, h], list(leaves.values()), [ay, al]))
    alone = [run(*r) for r in runs]
    streams = [torch.cuda.Stream() for _ in runs]
    torch.cuda.synchronize()
    both = [[], []]
    for _ in range(3):
        for s, r, out in zip(streams, runs, both):
            with torch.cuda.stream(s):
                out.append(run(*r))
    torch.cuda.synchronize()
    for want, outs in zip(alone, both):
        for got in outs:
            assert all(torch.equal(a, b) for a, b in zip(want, got))
    leaves = runs[0][0]
    with torch.inference_mode():
        y, h = ops_ssm.selective_scan(*(leaves[k] for k in NAMES[:5]), **{k: leaves[k] for k in NAMES[5:]})
        assert torch.equal(y, alone[0][0]) and torch.equal(h, alone[0][1])
        ops_ssm.selective_scan_step(*(leaves[k][0] if k in 'xBC' or k == 'dt' else leaves[k] for k in NAMES[:5]), h, D=leaves['D'],
                                    z=leaves['z'][0], dt_bias=leaves['dt_bias'])


def test_second_derivatives_are_refused_and_changed_inputs_noticed():
    from generative_mouse_trajectories_amd import ops, ops_ssm
    x = torch.randn(5, 2, 8, device=DEV, requires_grad=True)
    w = torch.randn(8, 3, device=DEV, requires_grad=True)
    A, Bm = -torch.ones(8, 4, device=DEV), torch.randn(5, 2, 4, device=DEV)
    h0 = torch.randn(2, 8, 4, device=DEV)
    lin = torch.randn(6, 8, device=DEV, requires_grad=True)
    for y in (ops_ssm.causal_conv(x, w)[0], ops_ssm.selective_scan(x, x, A, Bm, Bm)[0], ops.linear(x, lin, None, ckpt8=True)):
        g, = torch.autograd.grad((y ** 2).sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match='once_differentiable'):
            g.sum().backward()
    y, _ = ops_ssm.selective_scan(x, x, A, Bm, Bm, state=h0)
    with torch.no_grad():                                 # a single step in place on a state that the backward pass needs
        ops_ssm.selective_scan_step(x[0].detach(), x[0].detach(), A, Bm[0], Bm[0], h0)
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        y.sum().backward()


@pytest.mark.parametrize('B,C,N', [(70000, 3, 2), (3, 2050, 16)])
def test_many_rows_and_wide_rows(B, C, N):
    from generative_mouse_trajectories_amd import ops_ssm
    L = 3
    t, ay, al = scan_inputs(L, B, C, N, 1, torch.float32, True, True, True, 4)
    w = torch.randn(C, 4, generator=torch.Generator().manual_seed(2))
    leaves = {k: a.to(DEV).requires_grad_(True) for k, a in t.items()}
    gw = w.to(DEV).requires_grad_(True)
    u, _ = ops_ssm.causal_conv(leaves['x'], gw)
    y, h = ops_ssm.selective_scan(u, *(leaves[k] for k in NAMES[1:5]), **{k: leaves[k] for k in NAMES[5:]})
    got = torch.autograd.grad([y, h], [gw, *leaves.values()], [ay.to(DEV), al.to(DEV)])
    ref = {k: R.d(a).requires_grad_(True) for k, a in t.items()}
    rw = R.d(w).requires_grad_(True)
    ru, _ = R.conv(ref['x'], rw, None, None, None)
    ry, rh = R.scan(ru, *(ref[k] for k in NAMES[1:8]), None, ref['state'])
    want = torch.autograd.grad([ry, rh], [rw, *ref.values()], [R.d(ay), R.d(al)])
    R.close(y, ry, 200, 'y')
    R.close(h, rh, 200, 'state')
    for k, a, b in zip(('weight', *leaves), got, want):
        # sums over B * L rows: partial sums over at most 1024 slabs of the rows, B / 1024 rows each and then 64 + 16 slabs
        R.close(a, b, 400 + (L * (B // 256 + 2) + 80 if k in ('weight', 'A', 'D', 'dt_bias') else 0) + (C if k in 'BC' else 0), k)


def test_offsets_beyond_32_bits():
    """2.2e9 elements a sequence: the last steps agree with calls on the last steps alone."""
    from generative_mouse_trajectories_amd import ops_ckpt8, ops_ssm
    L, B, C, N = 70000, 32, 1000, 4
    x = torch.empty(L, B, C, device=DEV, dtype=torch.bfloat16).normal_(generator=torch.Generator(DEV).manual_seed(1))
    assert x.numel() > 2 ** 31
    w = torch.randn(C, 4, generator=torch.Generator().manual_seed(2)).to(DEV)
    y, last = ops_ssm.causal_conv(x, w)
    y2, last2 = ops_ssm.causal_conv(x[-64:], w, state=x[-67:-64])
    assert torch.equal(y[-64:], y2) and torch.equal(last, last2) and torch.equal(last, x[-3:])
    del y
    p = ops_ckpt8.pack(x)
    q = ops_ckpt8.pack(x[-64:])
    assert torch.equal(p.codes[-64:], q.codes) and torch.equal(p.exponents[-64:], q.exponents)
    del p, q
    A = -torch.rand(C, N, generator=torch.Generator().manual_seed(3)).to(DEV) * 4
    Bm = torch.randn(L, B, N, generator=torch.Generator(DEV).manual_seed(4), device=DEV).to(torch.bfloat16)
    y, h = ops_ssm.selective_scan(x, x, A, Bm, Bm)
    _, h1 = ops_ssm.selective_scan(x[:-640], x[:-640], A, Bm[:-640], Bm[:-640])
    y2, h2 = ops_ssm.selective_scan(x[-640:], x[-640:], A, Bm[-640:], Bm[-640:], state=h1)
    # two partitions of the same recurrence; the memory of a state is 1 / (step A), at most a few hundred steps of 3 roundings
    R.close(h, R.d(h2), 2000, 'state')
    R.close(y[-640:], R.d(y2), 2000, 'y')


def test_layer_run_training_prompt_and_sampling():
    """The operators as they are used together: projection -> convolution -> maps and steps -> scan -> projection, trained with its
    activations in 8 bits and whole, against float64; then a prompt and single steps."""
    from generative_mouse_trajectories_amd import ops, ops_ssm
    L, B, H, E, N, K = 33, 16, 32, 64, 8, 4
    gen = torch.Generator().manual_seed(21)
    r = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    P = {'w_in': r(2 * E, H) / H ** 0.5, 'b_in': 0.1 * r(2 * E), 'w_c': 0.5 * r(E, K), 'b_c': 0.1 * r(E), 'w_x': r(2 * N + E, E) / E ** 0.5,
         'A': -torch.exp(0.3 * r(E, N)) * torch.arange(1, N + 1), 'D': 1 + 0.1 * r(E), 'dt_bias': r(E) * 0.5 - 3,
         'w_out': r(H, E) / E ** 0.5}
    x, adj = r(L, B, H), r(L, B, H)
    lengths = torch.randint(1, L + 1, (B,), generator=gen).to(torch.int32)
    lengths[0] = L

    def layer(P, x, lin, conv, scan):
        xz = lin(x, P['w_in'], P['b_in'])
        u, cs = conv(xz[..., :E], P)
        m = lin(u, P['w_x'], None)
        y, h = scan(u, m[..., 2 * N:], m[..., :N], m[..., N:2 * N], xz[..., E:], P)
        return lin(y, P['w_out'], None), cs, h

    def gpu(ckpt8):
        p = {k: v.to(DEV).requires_grad_(True) for k, v in P.items()}
        xg, ln = x.to(DEV).requires_grad_(True), lengths.to(DEV)
        out, _, _ = layer(p, xg, lambda a, w, b: ops.linear(a, w, b, ckpt8=ckpt8),
                          lambda u, q: ops_ssm.causal_conv(u, q['w_c'], q['b_c'], lengths=ln, ckpt8=ckpt8),
                          lambda u, dt, Bm, Cm, z, q: ops_ssm.selective_scan(u, dt, q['A'], Bm, Cm, D=q['D'], z=z, dt_bias=q['dt_bias'],
                                                                             lengths=ln, ckpt8=ckpt8))
        return out, dict(zip((*P, 'x'), torch.autograd.grad(out, (*p.values(), xg), adj.to(DEV))))

    q = {k: v.double().requires_grad_(True) for k, v in P.items()}
    x64 = x.double().requires_grad_(True)
    import torch.nn.functional as F
    want, _, _ = layer(q, x64, F.linear, lambda u, q: R.conv(u, q['w_c'], q['b_c'], lengths, None),
                       lambda u, dt, Bm, Cm, z, q: R.scan(u, dt, q['A'], Bm, Cm, q['D'], z, q['dt_bias'], lengths, None))
    wg = dict(zip((*P, 'x'), torch.autograd.grad(want, (*q.values(), x64), adj.double())))
    out, got = gpu(False)
    # four operators in a row: four chains of roundings, each through sums of up to L * B = 528 rows
    R.close(out, want, 4 * (3 * L + E + 45), 'out')
    for k in wg:
        R.close(got[k], wg[k], 8 * (3 * L + E + 45) + L * B, 'd' + k)
    out8, got8 = gpu(True)
    assert torch.equal(out8, out), 'the outputs do not depend on what is kept'
    # 8-bit checkpoints: an element is off by at most half a unit, a unit at most 1/63.5 of its block's largest magnitude; six kept
    # activations enter a gradient, in relative terms and to first order at most once each
    for k in wg:
        err = float((R.d(got8[k]) - wg[k]).norm() / wg[k].norm())
        assert err <= 6 / 127, (k, err)

    p = {k: v.to(DEV) for k, v in P.items()}
    with torch.no_grad():
        S = 20
        full, _, _ = layer(p, x.to(DEV), ops.linear, lambda u, q: ops_ssm.causal_conv(u, q['w_c'], q['b_c']),
                           lambda u, dt, Bm, Cm, z, q: ops_ssm.selective_scan(u, dt, q['A'], Bm, Cm, D=q['D'], z=z, dt_bias=q['dt_bias']))
        head, cs, h = layer(p, x[:S].to(DEV), ops.linear, lambda u, q: ops_ssm.causal_conv(u, q['w_c'], q['b_c']),
                            lambda u, dt, Bm, Cm, z, q: ops_ssm.selective_scan(u, dt, q['A'], Bm, Cm, D=q['D'], z=z, dt_bias=q['dt_bias']))
        steps = [head]
        for t in range(S, L):
            o, _, _ = layer(p, x[t].to(DEV), ops.linear, lambda u, q: (ops_ssm.causal_conv_step(u, cs, q['w_c'], q['b_c']), cs),
                            lambda u, dt, Bm, Cm, z, q: (ops_ssm.selective_scan_step(u, dt, q['A'], Bm, Cm, h, D=q['D'], z=z,
                                                                                     dt_bias=q['dt_bias']), h))
            steps.append(o[None])
        R.close(torch.cat(steps), full, 8 * (3 * L + E + 45), 'prompt and single steps')


def test_growing_states_in_segments():
    """A > 0: over a segment the decay exp(A S) exceeds fp32, but a state that is zero (or tiny) there stays finite, as it does step by step."""
    from generative_mouse_trajectories_amd import ops_ssm
    L, B, C, N = 260, 2, 40, 4
    t, ay, _ = scan_inputs(L, B, C, N, 1, torch.float32, True, False, True, 3)
    t['A'] = 0.5 + torch.rand(C, N, generator=torch.Generator().manual_seed(1))
    t['dt'] = t['dt'] + 2.0
    t['x'][:L - 4] = 0                                       # nothing enters before the last steps, no adjoint behind the first ones
    ay[4:] = 0
    for state in (None, torch.full((B, C, N), 1e-30)):
        t['state'] = state
        if state is not None:                                # a small state that grows by up to e^128
            t['dt'] = torch.full_like(t['dt'], -5.0)
            t['dt'][:40] = 2.0
        ref = {k: R.d(t[k]) for k in NAMES}
        wy, wl = R.scan(*(ref[k] for k in NAMES[:8]), None, ref['state'])
        assert float(wl.abs().max()) < 1e38
        leaves = {k: t[k].to(DEV).requires_grad_(True) for k in NAMES if t[k] is not None}
        y, h = ops_ssm.selective_scan(*(leaves[k] for k in NAMES[:5]), z=leaves['z'], state=leaves.get('state'))
        # on top of the chain: an exponent of up to 128 with 40 roundings of a segment's sum of steps and 8 of softplus, scale and product
        assert torch.isfinite(h).all() and torch.isfinite(y).all()
        _, mag = R.scan(ref['x'].abs(), ref['dt'], ref['A'], ref['B'].abs(), *(ref[k] for k in NAMES[4:8]), None, ref['state'])
        rel = ((R.d(h) - wl).abs() / mag).max()
        assert float(rel) <= (3 * L + N + 45 + 128 * 48) * R.U32, float(rel)
        if state is None:
            gx, = torch.autograd.grad(y, leaves['x'], ay.to(DEV))
            rx = ref['x'].clone().requires_grad_(True)
            ry, _ = R.scan(rx, *(ref[k] for k in NAMES[1:8]), None, None)
            want, = torch.autograd.grad(ry, rx, R.d(ay))
            assert torch.isfinite(gx).all()
            R.close(gx, want, 2 * (3 * L + N + 45) + 45, 'dx')


@pytest.mark.parametrize('L,B', [(13, 9), (150, 9), (13, 2100)])
def test_states_without_memory(L, B):
    """A = -inf (or so low that base 2 takes it there): a state holds the last step alone, and what lies behind a row's end leaves it as it is."""
    from generative_mouse_trajectories_amd import ops_ssm
    C, N = 40, 6
    t, ay, al = scan_inputs(L, B, C, N, 1, torch.float32, True, True, True, 4)
    t['A'][3, 2], t['A'][7], t['A'][11, 0] = -float('inf'), -float('inf'), -3e38
    lengths = ragged(L, B)
    ref = {k: R.d(t[k]) for k in NAMES}
    wy, wl = R.scan(*(ref[k] for k in NAMES[:8]), lengths, ref['state'])
    leaves = {k: t[k].to(DEV).requires_grad_(True) for k in NAMES}
    y, h = ops_ssm.selective_scan(*(leaves[k] for k in NAMES[:5]), D=leaves['D'], z=leaves['z'], dt_bias=leaves['dt_bias'], state=leaves['state'],
                                  lengths=lengths.to(DEV))
    R.close(y, wy, 3 * L + N + 45, 'y')
    R.close(h, wl, 3 * L + N + 45, 'final state')
    rx = ref['x'].clone().requires_grad_(True)
    want, = torch.autograd.grad(R.scan(rx, *(ref[k] for k in NAMES[1:8]), lengths, ref['state']), rx, [R.d(ay), R.d(al)])
    got = torch.autograd.grad([y, h], list(leaves.values()), [ay.to(DEV), al.to(DEV)])
    R.close(got[0], want, 2 * (3 * L + N + 45) + 45, 'dx')
    assert all(torch.isfinite(g).all() for g in got)


@pytest.mark.parametrize('seq,maps', [(2 ** 27 - 24, 2 ** 26 - 1), (2 ** 27 + 8, 2 ** 26 + 3)])
def test_steps_far_apart(seq, maps):
    """Steps at the largest pitch that is read in place, and beyond it (copied): what contiguous sequences give, to the bit."""
    from generative_mouse_trajectories_amd import ops_ssm
    L, B, C, N = 11, 2, 40, 5
    t, ay, al = scan_inputs(L, B, C, N, 1, torch.bfloat16, True, True, True, 6)
    far = torch.zeros(10 * max(seq, maps) + 2 * B * C, device=DEV, dtype=torch.bfloat16)

    def apart(a, pitch, at):
        v = far[at:].as_strided(a.shape, (pitch, *a.stride()[1:]))
        v.copy_(a)
        return v
    flat = {k: v.to(DEV) for k, v in t.items()}
    for name in ('x', 'dt', 'z', 'B', 'C', 'ay'):
        near, adj = dict(flat), ay.to(DEV)
        if name == 'ay':
            adj = apart(adj, seq, 0)
        else:
            near[name] = apart(flat[name], maps if name in 'BC' else seq, 3)
        out = []
        for vals, a in ((near, adj), (flat, ay.to(DEV))):
            v = [vals[k].detach().requires_grad_(True) for k in NAMES]
            y, h = ops_ssm.selective_scan(*v[:5], D=v[5], z=v[6], dt_bias=v[7], state=v[8])
            out.append((y, h, *torch.autograd.grad([y, h], v, [a, al.to(DEV)])))
        assert all(torch.equal(p, q) for p, q in zip(*out)), name


def test_more_than_four_million_workgroups():
    """A group per channel and 4100 rows: 2^22 + 4096 workgroups in the forward pass."""
    from generative_mouse_trajectories_amd import ops_ssm
    L, B, C, N = 2, 4100, 1024, 2
    t, ay, al = scan_inputs(L, B, C, N, C, torch.float32, True, True, True, 9)
    leaves = {k: t[k].to(DEV).requires_grad_(True) for k in NAMES}
    outs = ops_ssm.selective_scan(*(leaves[k] for k in NAMES[:5]), D=leaves['D'], z=leaves['z'], dt_bias=leaves['dt_bias'], state=leaves['state'])
    got = grads(outs, list(leaves.values()), [ay.to(DEV), al.to(DEV)])
    rl = {k: R.d(t[k]).requires_grad_(True) for k in NAMES}
    want = R.scan(*(rl[k] for k in NAMES[:8]), None, rl['state'])
    for what, g, w in zip(('y', 'state'), outs, want):
        R.close(g, w, 3 * L + N + 45, what)
    for k, g, w in zip(NAMES, got, grads(want, list(rl.values()), [R.d(ay), R.d(al)])):
        # a workgroup sums the parameters' gradients over 1025 rows of L steps
        R.close(g, w, 2 * (3 * L + N + 45) + 45 + (1025 * L + 80 if k in ('A', 'D', 'dt_bias') else 0), 'd' + k)


@pytest.mark.parametrize('B,C,N,dtype', [(2 ** 22 + 3, 16, 8, 'fp32'), (2 ** 20 + 1, 256, 2, 'bf16')])
def test_single_steps_of_millions_of_rows(B, C, N, dtype):
    """The last and the first rows of a step are what a step on these rows alone gives."""
    from generative_mouse_trajectories_amd import ops_ssm
    dt = {'fp32': torch.float32, 'bf16': torch.bfloat16}[dtype]
    gen = torch.Generator(DEV).manual_seed(1)
    r = lambda *s: torch.randn(*s, device=DEV, generator=gen)  # noqa: E731
    x, d, z, Bm, Cm, h = r(B, C).to(dt), r(B, C).to(dt), r(B, C).to(dt), r(B, N).to(dt), r(B, N).to(dt), r(B, C, N)
    A, D, bias = -torch.exp(r(C, N)), r(C), r(C)
    ends = [h[s].clone() for s in (slice(0, 5), slice(B - 77, B))]
    y = ops_ssm.selective_scan_step(x, d, A, Bm, Cm, h, D=D, z=z, dt_bias=bias)
    for s, h0 in zip((slice(0, 5), slice(B - 77, B)), ends):
        want = ops_ssm.selective_scan_step(x[s], d[s], A, Bm[s], Cm[s], h0, D=D, z=z[s], dt_bias=bias)
        assert torch.equal(y[s], want) and torch.equal(h[s], h0)


def test_convolution_step_of_more_than_2_31_elements():
    from generative_mouse_trajectories_amd import ops_ssm
    B, C, K = 2 ** 21 + 5, 1024, 2
    gen = torch.Generator(DEV).manual_seed(1)
    x, state = (torch.randn(*s, device=DEV, generator=gen, dtype=torch.bfloat16) for s in ((B, C), (K - 1, B, C)))
    w, b = torch.randn(C, K, device=DEV, generator=gen), torch.randn(C, device=DEV, generator=gen)
    ends = (slice(0, 5), slice(B - 77, B))
    kept = [state[:, s].clone() for s in ends]
    y = ops_ssm.causal_conv_step(x, state, w, b)
    for s, c0 in zip(ends, kept):
        assert torch.equal(y[s], ops_ssm.causal_conv_step(x[s], c0, w, b)) and torch.equal(state[:, s], c0) and torch.equal(c0[-1], x[s])


def test_parameter_gradients_of_more_than_2_27_elements():
    """4 M channels x 32 states, and a convolution of 33 M channels: a step each, against the formulas in float64."""
    from generative_mouse_trajectories_amd import ops_ssm
    gen = torch.Generator(DEV).manual_seed(1)
    r = lambda *s: torch.randn(*s, device=DEV, generator=gen)  # noqa: E731

    def close(got, want, what):
        err = float((got.double() - want).abs().max()) / float(want.abs().max())
        assert got.shape == want.shape and err <= 200 * R.U32, (what, err)
    C, N = 2 ** 22, 32
    x, dt, A, D, h0 = r(1, 1, C), r(1, 1, C), -torch.exp(r(C, N)), r(C), r(1, C, N)
    Bm, Cm, ay, al = r(1, 1, N), r(1, 1, N), r(1, 1, C), r(1, C, N)
    leaves = [t.requires_grad_(True) for t in (x, dt, A, D, h0)]
    y, h = ops_ssm.selective_scan(x, dt, A, Bm, Cm, D=D, state=h0)
    dx, ddt, dA, dD, dh = torch.autograd.grad([y, h], leaves, [ay, al])
    with torch.no_grad():
        step = torch.log1p(torch.exp(dt.double())).view(C, 1)
        e = torch.exp(step * A.double())
        g = Cm.double().view(1, N) * ay.double().view(C, 1) + al.double()[0]
        close(dh[0], g * e, 'dstate')
        q = g * e * h0.double()[0]
        close(dA, q * step, 'dA')
        gB = (g * Bm.double().view(1, N)).sum(1)
        close(ddt.view(C), ((q * A.double()).sum(1) + x.double().view(C) * gB) * torch.sigmoid(dt.double()).view(C), 'ddt')
        close(dx.view(C), step.view(C) * gB + D.double() * ay.double().view(C), 'dx')
        close(dD, (ay.double() * x.double()).view(C), 'dD')
    del x, dt, A, D, h0, leaves, y, h, dx, ddt, dA, dD, dh, e, g, q, al
    C, K = 2 ** 25 + 65, 3
    x, w, b, s, ay = r(1, 1, C), r(C, K), r(C), r(K - 1, 1, C), r(1, 1, C)
    assert (K + 1) * C > 2 ** 27
    leaves = [t.requires_grad_(True) for t in (x, w, b, s)]
    y, _ = ops_ssm.causal_conv(x, w, b, state=s)
    dx, dw, db, ds = torch.autograd.grad(y, leaves, ay)
    with torch.no_grad():
        past = torch.cat([s, x]).double().view(K, C)
        pre = (past * w.double().t()).sum(0) + b.double()
        sig = torch.sigmoid(pre)
        g = ay.double().view(C) * sig * (1 + pre * (1 - sig))
        close(db, g, 'db')
        close(dw, (g * past).t(), 'dw')
        close(dx.view(C), g * w.double()[:, K - 1], 'dx')
        close(ds.view(K - 1, C), g * w.double().t()[:K - 1], 'dstate')


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('B,C,N,G,aligned', [(8203, 130, 16, 1, True), (8203, 130, 16, 2, False), (8195, 64, 5, 1, True), (2051, 520, 32, 4, True),
                                             (16389, 33, 8, 3, True), (9000, 260, 4, 1, True)])
def test_single_steps_of_many_rows(B, C, N, G, aligned, dtype):
    """Four rows at a time, several groups of them a workgroup, the last of one to three rows; states aligned to 4 bytes; inactive rows."""
    from generative_mouse_trajectories_amd import ops_ssm
    t, _, _ = scan_inputs(1, B, C, N, G, dtype, True, True, True, B + C)
    gen = torch.Generator().manual_seed(2)
    w, b, cs = torch.randn(C, 4, generator=gen), torch.randn(C, generator=gen), torch.randn(3, B, C, generator=gen).to(dtype)
    act = torch.rand(B, generator=gen) < 0.8
    act[-3:] = torch.tensor([True, False, True])
    ref = {k: R.d(t[k]) for k in NAMES}
    wu, wc = R.conv(ref['x'], R.d(w), R.d(b), None, R.d(cs))
    wy, wh = R.scan(*(ref[k] for k in NAMES[:8]), None, ref['state'])
    v = {k: a.to(DEV) for k, a in t.items()}
    one = [v[k][0] if k in ('x', 'dt', 'B', 'C') else v[k] for k in NAMES[:5]]
    for active, aside in ((None, False), (act, True), (act, False)):
        h = v['state'].clone() if aligned else torch.empty(B * C * N + 1, device=DEV)[1:].view(B, C, N).copy_(v['state'])
        c = cs.to(DEV)
        h2 = torch.full_like(h, 7.0) if aside else None
        c2 = torch.full_like(c, 7.0) if aside else None
        a = None if active is None else active.to(DEV)
        y = ops_ssm.selective_scan_step(*one, h, D=v['D'], z=v['z'][0], dt_bias=v['dt_bias'], active=a, state_out=h2)
        u = ops_ssm.causal_conv_step(one[0], c, w.to(DEV), b.to(DEV), active=a, state_out=c2)
        h, c = (h2, c2) if aside else (h, c)
        on = torch.ones(B, dtype=torch.bool) if active is None else act
        R.close(h[on.to(DEV)], wh[on], N + 48, 'state')
        R.close(y[on.to(DEV)], wy[0][on], N + 48, 'y')
        R.close(u[on.to(DEV)], wu[0][on], 49, 'u')
        assert torch.equal(R.d(c)[:, on], wc[:, on])
        if active is not None:
            off = ~act
            assert torch.equal(R.d(h)[off], ref['state'][off]) and torch.equal(R.d(c)[:, off], R.d(cs)[:, off])
            assert float(y[off.to(DEV)].abs().max()) == 0 and float(u[off.to(DEV)].abs().max()) == 0


@pytest.mark.parametrize('B,C,N,G,dtype,gate,ckpt8', [(300, 256, 16, 1, 'bf16', True, False), (300, 128, 32, 1, 'fp32', False, False),
                                                      (600, 256, 16, 2, 'fp32', False, True), (300, 128, 20, 1, 'bf16', True, True)])
def test_many_rows_of_unequal_length_and_many_states(B, C, N, G, dtype, gate, ckpt8):
    """Rows taken by length with two and four lanes a channel, in both types."""
    from generative_mouse_trajectories_amd import ops_ssm
    L, dt = 20, {'fp32': torch.float32, 'bf16': torch.bfloat16}[dtype]
    t, ay, al = scan_inputs(L, B, C, N, G, dt, gate, True, True, B + N)
    if ckpt8:                                                # values that 8-bit checkpoints hold exactly
        t.update({k: (t[k].float() * 32).round().clamp(-100, 100).div(32).to(dt) for k in ('x', 'dt', 'z') if t[k] is not None})
    lengths = torch.randint(0, L + 1, (B,), generator=torch.Generator().manual_seed(B), dtype=torch.int32)
    names = [k for k in NAMES if t[k] is not None]
    leaves = {k: t[k].to(DEV).requires_grad_(True) for k in names}
    y, last = ops_ssm.selective_scan(*(leaves[k] for k in NAMES[:5]), D=leaves['D'], z=leaves.get('z'), dt_bias=leaves['dt_bias'],
                                     state=leaves['state'], ckpt8=ckpt8, lengths=lengths.to(DEV))
    got = dict(zip(names, grads([y, last], [leaves[k] for k in names], [ay.to(DEV), al.to(DEV)])))
    rl = {k: R.d(t[k]).requires_grad_(True) for k in names}
    outs = R.scan(*(rl.get(k) for k in NAMES[:8]), lengths, rl['state'])
    chain = 3 * L + N + 45
    R.close(y, outs[0], chain, 'y')
    R.close(last, outs[1], chain, 'final state')
    want = dict(zip(names, grads(outs, [rl[k] for k in names], [R.d(ay), R.d(al)])))
    for k in names:
        extra = {'A': 3 * L + 80, 'D': 3 * L + 80, 'dt_bias': 3 * L + 80, 'B': C // G, 'C': C // G}.get(k, 0)
        R.close(got[k], want[k], 2 * chain + 45 + extra, 'd' + k)


def test_backward_offsets_beyond_32_bits():
    """2.2e9 elements a sequence, backward: the gradients of the last steps agree with those of calls on the last steps alone (whose adjoint
    is all there is), from kept states and from 8-bit checkpoints, which hold these inputs exactly; unpacking and the weight gradient."""
    from generative_mouse_trajectories_amd import ops_ckpt8, ops_ssm
    L, B, C, N, T = 70000, 32, 1000, 4, 640
    x = (torch.randint(-100, 101, (L, B, C), device=DEV, dtype=torch.int8, generator=torch.Generator(DEV).manual_seed(1)).to(torch.bfloat16) / 32)
    assert x.numel() > 2 ** 31
    x.requires_grad_(True)
    dy = torch.zeros(L, B, C, device=DEV, dtype=torch.bfloat16)
    dy[-T:] = torch.randn(T, B, C, generator=torch.Generator(DEV).manual_seed(2), device=DEV).to(torch.bfloat16)
    w = torch.randn(C, 4, generator=torch.Generator().manual_seed(2)).to(DEV).requires_grad_(True)
    tail = x.detach()[-T:].clone().requires_grad_(True)
    for ckpt8 in (False, True):
        y, _ = ops_ssm.causal_conv(x, w, ckpt8=ckpt8)
        dx, dw = torch.autograd.grad(y, [x, w], dy)
        y2, _ = ops_ssm.causal_conv(tail, w, state=x.detach()[-T - 3:-T])
        dx2, dw2 = torch.autograd.grad(y2, [tail, w], dy[-T:])
        assert torch.equal(dx[-T:], dx2) and float(dx[:-T - 3].abs().max()) == 0
        R.close(dw, R.d(dw2), T * B * 2, 'dw')               # the same terms in another order
        del y, dx, y2, dx2
    A = -torch.rand(C, N, generator=torch.Generator().manual_seed(3)).to(DEV) * 4
    Bm = torch.randn(L, B, N, generator=torch.Generator(DEV).manual_seed(4), device=DEV).to(torch.bfloat16)
    Bt = Bm[-T:].clone()
    with torch.no_grad():
        _, h1 = ops_ssm.selective_scan(x[:-T], x[:-T], A, Bm[:-T], Bm[:-T], z=x[:-T])
    for ckpt8 in (False, True):
        both = []
        for seq, m, adj, state in ((x, Bm, dy, None), (tail, Bt, dy[-T:], h1)):
            v = [t.detach().requires_grad_(True) for t in (seq, seq, m, m, seq)]
            y, _ = ops_ssm.selective_scan(v[0], v[1], A, v[2], v[3], z=v[4], state=state, ckpt8=ckpt8)
            both.append([g[-T:].clone() for g in torch.autograd.grad(y, v, adj)])
            del y, v
        for name, g, want in zip(('x', 'dt', 'B', 'C', 'z'), *both):
            # two partitions of one recurrence (a memory of a few hundred steps of 3 roundings), each rounded to bf16: at most a whole step apart
            R.close(g.float(), R.d(want), 2000 + 2 * 2 ** 16, 'd' + name)
    p = ops_ckpt8.pack(x)
    out = ops_ckpt8.unpack(p)
    assert torch.equal(out[-T:], x[-T:]) and torch.equal(out[:T], x[:T])
    del out
    rows = L * B
    dz = torch.zeros(rows, 8, device=DEV)
    dz[-100:] = torch.randn(100, 8, generator=torch.Generator(DEV).manual_seed(5), device=DEV)
    dW, db = ops_ckpt8.wgrad(dz, p, want_db=True)
    last = x.detach().reshape(rows, C)[-100:]
    dW2, db2 = dz[-100:].double().t() @ last.double(), dz.double().sum(0)
    R.close(dW, dW2, 200, 'dW')
    R.close(db, db2, 200, 'db')
