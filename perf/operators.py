"""The selective state-space operators and the 8-bit activation checkpoints at the sizes they are used at: one pass of
each, in plain torch operations (`own` false) or through the package's entry points (`own` true).

Sequences are time-major [L, B, C]: L steps of B trajectories with C channels.  N states per channel, G groups of channels
that share their input and output maps, K taps of the short convolution.
"""
import torch

own = False

DTYPES = {'fp32': torch.float32, 'bf16': torch.bfloat16}
BLOCK = 32                       # channels that share one scale of an 8-bit checkpoint


def case(op, form, dtype, L=1, B=1, C=1, N=16, G=1, K=4, ragged=False, carried=False, gated=True, ckpt8=False, name=None):
    c = dict(op=op, form=form, dtype=dtype, L=L, B=B, C=C, N=N, G=G, K=K, ragged=ragged, carried=carried, gated=gated, ckpt8=ckpt8)
    if name is not None:
        c['name'] = name
    return c


def listed():
    return [
        # one trajectory continued by one step: the latency of interactive sampling
        case('conv', 'token', 'fp32', B=1, C=256, name='conv_token_one'),
        # the convolution of a training step over a large batch of 128-step trajectories, activations in bf16
        case('conv', 'train', 'bf16', L=128, B=1024, C=512, name='conv_train'),
        # recorded beginnings of 33 trajectories of different lengths, continued from kept inputs; a width that is no multiple of 4
        case('conv', 'prompt', 'fp32', L=200, B=33, C=250, K=3, ragged=True, carried=True, name='conv_prompt_ragged'),
        # one trajectory continued by one step
        case('scan', 'token', 'fp32', B=1, C=256, name='scan_token_one'),
        # sampling of 4096 trajectories side by side, one step of all of them: the state is read and written whole
        case('scan', 'token', 'bf16', B=4096, C=512, name='scan_token_batch'),
        # one long recording read in a single call: few rows, a long axis
        case('scan', 'prompt', 'bf16', L=8192, B=1, C=1024, name='scan_prompt_long'),
        # a training step of a critic in fp32 on ragged trajectories (T + 1 = 129 points)
        case('scan', 'train', 'fp32', L=129, B=512, C=256, ragged=True, name='scan_train_ragged'),
        # a training step in bf16 at twice the length, two groups of input and output maps
        case('scan', 'train', 'bf16', L=256, B=256, C=512, G=2, name='scan_train'),
        # the same kind of step with its activations kept in 8 bits for the backward pass
        case('scan', 'train', 'bf16', L=129, B=256, C=512, ckpt8=True, name='scan_train_ckpt8'),
        # an activation of 200 steps x 512 rows kept in 8 bits and read back
        case('pack', 'train', 'bf16', L=200, B=512, C=512, name='pack'),
        # the weight gradient of a 128 -> 512 projection over all steps of a large fp32 batch, its input kept in 8 bits (N outputs)
        case('wgrad', 'train', 'fp32', L=128, B=4096, C=128, N=512, name='wgrad_fp32'),
        # the same for a small bf16 batch with odd widths
        case('wgrad', 'train', 'bf16', L=129, B=33, C=250, N=515, name='wgrad_odd'),
    ]


def draw(rng):
    def log(lo, hi):
        return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))

    dtype = rng.choice(['fp32', 'bf16'])
    op = rng.choice(['conv', 'scan', 'scan', 'pack', 'wgrad'])
    if op in ('pack', 'wgrad'):
        C, N = log(9, 1024), log(9, 1024)
        rows = log(64, min(1 << 20, (1 << 26) // C))
        if op == 'wgrad':
            rows = min(rows, (1 << 35) // (C * N), (1 << 28) // N)
        L = log(1, min(256, rows))
        return case(op, 'train', dtype, L=L, B=max(1, rows // L), C=C, N=N)
    form = rng.choice(['token', 'prompt', 'train', 'train'])
    C = log(16, 1024)
    N = rng.choice([5, 8, 16, 16, 16, 24, 32])
    G = rng.choice([1, 1, 2, 4])
    if op == 'conv':
        N, G = 16, 1
    C = max(G, C // G * G)
    budget = (1 << 28) // (C * N) if op == 'scan' else (1 << 25) // C
    if form == 'token':
        L, B = 1, log(1, min(4096, budget))
    else:
        L = log(1, min(8192 if form == 'prompt' else 512, budget))
        B = log(1, max(1, min(4096, budget // L)))
    return case(op, form, dtype, L=L, B=B, C=C, N=N, G=G, K=rng.choice([2, 3, 4]), ragged=form != 'token' and rng.random() < 0.5,
                carried=rng.random() < 0.5, gated=rng.random() < 0.7, ckpt8=form == 'train' and rng.random() < 0.3)


def prepare(case, seed):
    dev = 'cuda' if torch.cuda.is_available() else 'cpu'
    gen = torch.Generator(device=dev).manual_seed(int(seed))
    dtype = DTYPES[case['dtype']]
    L, B, C, N, G, K = (case[k] for k in 'LBCNGK')
    train = case['form'] == 'train'

    def normal(*shape, scale=1.0, dt=torch.float32):
        return (torch.randn(*shape, device=dev, generator=gen) * scale).to(dt)

    def uniform(*shape, lo=0.0, hi=1.0):
        return torch.rand(*shape, device=dev, generator=gen) * (hi - lo) + lo

    s = {'case': dict(case)}
    if case['op'] in ('pack', 'wgrad'):
        # activations whose rows differ in size, as those behind a gate do
        s['x'] = (normal(L * B, C) * torch.exp(normal(L * B, 1))).to(dtype)
        if case['op'] == 'wgrad':
            s['dy'] = normal(L * B, N, scale=1e-2, dt=dtype)
        return s
    lead = (B,) if case['form'] == 'token' else (L, B)
    s['lengths'] = None
    if case['ragged']:
        lengths = (L // 2 + torch.rand(B, device=dev, generator=gen) * (L - L // 2 + 1)).to(torch.int32).clamp(max=L)
        lengths[0] = L
        s['lengths'] = lengths
    s['x'] = normal(*lead, C, dt=dtype)
    if case['op'] == 'conv':
        s['weight'] = uniform(C, K, lo=-K ** -0.5, hi=K ** -0.5)
        s['bias'] = uniform(C, lo=-K ** -0.5, hi=K ** -0.5)
        s['state'] = normal(K - 1, B, C, dt=dtype) if case['carried'] or case['form'] == 'token' else None
        if train:
            s['dy'] = normal(L, B, C, dt=dtype)
        else:
            s['state_out'] = normal(K - 1, B, C, dt=dtype)
        return _leaves(s, ('x', 'weight', 'bias', 'state')) if train else s
    step = torch.exp(uniform(C, lo=-6.9, hi=-2.3))                  # steps of 0.001 .. 0.1 at a zero projection
    s['dt'] = normal(*lead, C, scale=0.5, dt=dtype)
    s['dt_bias'] = step + torch.log(-torch.expm1(-step))
    s['A'] = -(torch.arange(1, N + 1, device=dev, dtype=torch.float32) * torch.exp(normal(C, N, scale=0.1)))
    s['B'], s['C'] = normal(*lead, G, N, dt=dtype), normal(*lead, G, N, dt=dtype)
    s['D'] = 1.0 + normal(C, scale=0.1)
    s['z'] = normal(*lead, C, dt=dtype) if case['gated'] else None
    s['state'] = normal(B, C, N) if case['carried'] or case['form'] == 'token' else None
    if train:
        s['dy'], s['dstate'] = normal(L, B, C, dt=dtype), normal(B, C, N, scale=0.1)
        return _leaves(s, SCAN_LEAVES)
    s['state_out'] = normal(B, C, N)
    return s


SCAN_LEAVES = ('x', 'dt', 'A', 'B', 'C', 'D', 'z', 'dt_bias', 'state')


def _leaves(s, names):
    s['leaves'] = [k for k in names if s[k] is not None]
    for k in s['leaves']:
        s[k].requires_grad_(True)
    return s


def run(state):
    c = state['case']
    if own:
        return _run_own(state, c)
    with torch.no_grad():
        return {'conv': _conv, 'scan': _scan, 'pack': _pack, 'wgrad': _wgrad}[c['op']](state, c)


def work(case):
    size = 4 if case['dtype'] == 'fp32' else 2
    L, B, C, N, G, K = (case[k] for k in 'LBCNGK')
    rows, train = L * B, case['form'] == 'train'
    if case['op'] == 'pack':
        return {'bytes': rows * C * (2 * size), 'flops': 4 * rows * C}
    if case['op'] == 'wgrad':
        return {'bytes': rows * (C + N) * size + 4 * N * (C + 1), 'flops': 2 * rows * C * N}
    part = 0.75 if case['ragged'] else 1.0                           # the steps within the trajectories' lengths
    n = rows * C
    kept = case['carried'] or case['form'] == 'token'
    if case['op'] == 'conv':
        states = size * (K - 1) * B * C * (1 + kept)
        by = size * n * (1 + part) + states + 4 * C * (K + 1)
        fl = part * n * (2 * K + 6)
        if train:
            by, fl = by + size * n * (1 + part) + states, fl + part * n * (4 * K + 8)
        return {'bytes': int(by), 'flops': int(fl)}
    ins = 2 + case['gated']
    states, maps = 4 * B * C * N, 2 * rows * G * N * size
    by = size * n * (ins * part + 1) + states * (1 + kept) + part * maps + 4 * C * (N + 2)
    fl = part * n * (7 * N + 20)
    if train:
        by, fl = by + size * n * (part + ins) + states * (1 + kept) + maps + 4 * C * (N + 2), fl + part * n * (20 * N + 40)
    return {'bytes': int(by), 'flops': int(fl)}


# ---- through the package ------------------------------------------------------------------------------------------------
def _run_own(s, c):
    from generative_mouse_trajectories_amd import ops_ckpt8, ops_ssm
    if c['op'] == 'pack':
        return ops_ckpt8.unpack(ops_ckpt8.pack(s['x']))
    if c['op'] == 'wgrad':
        return ops_ckpt8.wgrad(s['dy'], ops_ckpt8.pack(s['x']), want_db=True)
    if c['op'] == 'conv':
        if c['form'] == 'token':
            return ops_ssm.causal_conv_step(s['x'], s['state'], s['weight'], s['bias'], state_out=s['state_out']), s['state_out']
        y, last = ops_ssm.causal_conv(s['x'], s['weight'], s['bias'], lengths=s['lengths'], state=s['state'], ckpt8=c['ckpt8'])
        if c['form'] == 'prompt':
            return y, last
        return (y.detach(), last.detach(), *torch.autograd.grad([y], [s[k] for k in s['leaves']], [s['dy']]))
    if c['form'] == 'token':
        return ops_ssm.selective_scan_step(s['x'], s['dt'], s['A'], s['B'], s['C'], s['state'], D=s['D'], z=s['z'],
                                           dt_bias=s['dt_bias'], state_out=s['state_out']), s['state_out']
    y, last = ops_ssm.selective_scan(s['x'], s['dt'], s['A'], s['B'], s['C'], D=s['D'], z=s['z'], dt_bias=s['dt_bias'],
                                     lengths=s['lengths'], state=s['state'], ckpt8=c['ckpt8'])
    if c['form'] == 'prompt':
        return y, last
    return (y.detach(), last.detach(), *torch.autograd.grad([y, last], [s[k] for k in s['leaves']], [s['dy'], s['dstate']]))


# ---- plain forms, in 32 bits --------------------------------------------------------------------------------------------
def _valid(lengths, L, device):
    """[L, B, 1] truth values: the steps within each trajectory's length (None: all of them)."""
    return None if lengths is None else (torch.arange(L, device=device)[:, None] < lengths[None, :])[:, :, None]


def _within(valid, t):
    return t if valid is None else torch.where(valid, t, torch.zeros((), device=t.device, dtype=t.dtype))


def _sigmoid(v):
    return 1.0 / (1.0 + torch.exp(-v))


def _quantised(x):
    """The values that an 8-bit checkpoint of x [..., C] stands for: whole multiples q 2^e, |q| <= 127, of the smallest 2^e
    (e >= -118) that reaches a block of 32 channels."""
    C = x.shape[-1]
    blocks = torch.nn.functional.pad(x.float(), (0, -C % BLOCK)).unflatten(-1, (-1, BLOCK))
    frac, exp = torch.frexp(blocks.abs().amax(-1, keepdim=True))
    e = torch.where(frac <= 127 / 128, exp - 7, exp - 6).clamp(-118, 121)
    return torch.ldexp(torch.ldexp(blocks, -e).round().clamp(-127, 127), e).flatten(-2)[..., :C]


def _pack(s, c):
    return _quantised(s['x']).to(s['x'].dtype)


def _wgrad(s, c):
    dy = s['dy'].float()
    return dy.t() @ _quantised(s['x']), dy.sum(0)


def _recur(a, b):
    """h[t] = a[t] h[t-1] + b[t] along the first axis, from h[-1] = 0: spans of doubling length are joined."""
    n = 1
    while n < a.shape[0]:
        b = torch.cat([b[:n], torch.addcmul(b[n:], a[n:], b[:-n])])
        a = torch.cat([a[:n], a[n:] * a[:-n]])
        n *= 2
    return b


def _conv(s, c):
    x, w, b = s['x'].float(), s['weight'], s['bias']
    B, C, K = c['B'], c['C'], c['K']
    if c['form'] == 'token':
        past = torch.cat([s['state'].float(), x[None]])
        pre = (past * w.t()[:, None]).sum(0) + b
        return (pre * _sigmoid(pre)).to(s['x'].dtype), past[1:].to(s['x'].dtype)
    L = c['L']
    valid = _valid(s['lengths'], L, x.device)
    head = torch.zeros(K - 1, B, C, device=x.device) if s['state'] is None else s['state'].float()

    def before(x):
        past = torch.cat([head, _within(valid, x)])
        return past, sum(past[k:k + L] * w[:, k] for k in range(K)) + b

    past, pre = before(x)
    y = _within(valid, pre * _sigmoid(pre)).to(s['x'].dtype)
    if s['lengths'] is None:
        last = past[L:]
    else:
        at = s['lengths'].long()[None, :, None] + torch.arange(K - 1, device=x.device)[:, None, None]
        last = torch.gather(past, 0, at.expand(K - 1, B, C))
    last = last.to(s['x'].dtype)
    if c['form'] == 'prompt':
        return y, last
    if c['ckpt8']:
        past, pre = before(_quantised(x))
    sig = _sigmoid(pre)
    g = _within(valid, s['dy'].float() * sig * (1 + pre * (1 - sig)))
    grads = {'weight': torch.stack([(g * past[k:k + L]).sum((0, 1)) for k in range(K)], 1), 'bias': g.sum((0, 1))}
    dpast = sum(torch.nn.functional.pad(g * w[:, k], (0, 0, 0, 0, k, K - 1 - k)) for k in range(K))
    grads['x'], grads['state'] = _within(valid, dpast[K - 1:]).to(s['x'].dtype), dpast[:K - 1].to(s['x'].dtype)
    return (y, last, *(grads[k] for k in s['leaves']))


def _spread(m, C):
    """[..., G, N] maps of the groups -> [..., C, N] of the channels."""
    return m.float().repeat_interleave(C // m.shape[-2], dim=-2)


def _scan(s, c):
    A, D, C, L, B, N, G = s['A'], s['D'], c['C'], c['L'], c['B'], c['N'], c['G']
    dtype = s['x'].dtype
    z = None if s['z'] is None else s['z'].float()
    valid = None if c['form'] == 'token' else _valid(s['lengths'], L, A.device)
    Bm, Cm = _spread(s['B'], C), _spread(s['C'], C)

    def states(x, dt):
        v = dt + s['dt_bias']
        step = _within(valid, torch.where(v > 0, v, torch.zeros_like(v)) + torch.log1p(torch.exp(-v.abs())))
        a = torch.exp(step[..., None] * A)
        b = (step * x)[..., None] * Bm
        if c['form'] == 'token':
            return v, step, a, a * s['state'] + b
        if s['state'] is not None:
            b[0] += a[0] * s['state']
        return v, step, a, _recur(a, b)

    x, dt = _within(valid, s['x'].float()), s['dt'].float()
    v, step, a, h = states(x, dt)
    raw = (h * Cm).sum(-1) + D * x
    y = _within(valid, raw if z is None else raw * z * _sigmoid(z)).to(dtype)
    if c['form'] == 'token':
        return y, h
    last = h[-1].clone()
    if c['form'] == 'prompt':
        return y, last
    if c['ckpt8']:
        x, dt = _within(valid, _quantised(x)), _quantised(dt)
        z = None if z is None else _quantised(z)
        v, step, a, h = states(x, dt)
        raw = (h * Cm).sum(-1) + D * x
    dy = _within(valid, s['dy'].float())
    grads = {}
    if z is not None:
        sig = _sigmoid(z)
        grads['z'] = (dy * raw * sig * (1 + z * (1 - sig))).to(dtype)
        dy = dy * z * sig
    g = dy[..., None] * Cm
    g[-1] += s['dstate']
    g = _recur(torch.cat([torch.ones_like(a[:1]), a.flip(0)[:-1]]), g.flip(0)).flip(0)
    before = torch.zeros_like(h[:1]) if s['state'] is None else s['state'][None]
    ga = g * a * torch.cat([before, h[:-1]])                          # the adjoint of a, times a
    gb = (g * Bm).sum(-1)
    dstep = (ga * A).sum(-1) + gb * x
    dv = _within(valid, dstep * _sigmoid(v))
    grads['x'] = _within(valid, gb * step + D * dy).to(dtype)
    grads['dt'], grads['dt_bias'] = dv.to(dtype), dv.sum((0, 1))
    grads['A'], grads['D'] = (ga * step[..., None]).sum((0, 1)), (dy * x).sum((0, 1))
    grads['B'] = (g * (step * x)[..., None]).unflatten(2, (G, C // G)).sum(3).to(dtype)
    grads['C'] = (h * dy[..., None]).unflatten(2, (G, C // G)).sum(3).to(dtype)
    grads['state'] = g[0] * a[0]
    return (y, last, *(grads[k] for k in s['leaves']))


# ---- from the definitions, in 64 bits -----------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    c = s['case']
    f = {k: t.detach().double() for k, t in s.items() if isinstance(t, torch.Tensor) and t.is_floating_point()}

    def stands_for(t):
        rows = torch.nn.functional.pad(t, (0, -t.shape[-1] % BLOCK)).reshape(-1, BLOCK)
        most = rows.abs().max(1, keepdim=True).values
        unit = torch.exp2(torch.floor(torch.log2(most.clamp(min=2.0 ** -140) / 127)) - 1)
        for _ in range(3):                                            # the smallest power of two that reaches the block
            unit = torch.where(most > 127 * unit, 2 * unit, unit)
        unit = unit.clamp(2.0 ** -118, 2.0 ** 121)
        q = torch.clamp(torch.round(rows / unit), -127, 127) * unit
        return q.reshape(*t.shape[:-1], -1)[..., :t.shape[-1]]

    if c['op'] == 'pack':
        return stands_for(f['x'])
    if c['op'] == 'wgrad':
        return f['dy'].t() @ stands_for(f['x']), f['dy'].sum(0)
    steps = 1 if c['form'] == 'token' else c['L']
    rows = c['B']
    live = torch.full((rows,), steps, device=f['x'].device) if s.get('lengths') is None else s['lengths'].long()
    if c['form'] == 'token':
        f.update({k: f[k][None] for k in ('x', 'dt', 'B', 'C', 'z') if k in f})

    def conv(f):
        K = c['K']
        window = list(f['state']) if 'state' in f else [torch.zeros_like(f['x'][0])] * (K - 1)
        out = []
        for t in range(steps):
            on = (t < live)[:, None]
            window = window + [f['x'][t]]
            pre = f['bias'] + sum(window[k] * f['weight'][:, k] for k in range(K))
            out.append(torch.where(on, torch.nn.functional.silu(pre), 0.0))
            window = [torch.where(on, window[k + 1], window[k]) for k in range(K - 1)]
        return torch.stack(out), torch.stack(window)

    def scan(f):
        per = c['C'] // c['G']
        h = f['state'] if 'state' in f else torch.zeros(rows, c['C'], c['N'], device=f['x'].device, dtype=torch.float64)
        out = []
        for t in range(steps):
            on = (t < live)[:, None]
            d = torch.logaddexp(f['dt'][t] + f['dt_bias'], torch.zeros((), device=h.device, dtype=h.dtype))
            Bt, Ct = (f[k][t].repeat_interleave(per, 1) for k in 'BC')
            new = (d[:, :, None] * f['A']).exp() * h + d[:, :, None] * Bt * f['x'][t][:, :, None]
            y = torch.linalg.vecdot(new, Ct) + f['D'] * f['x'][t]
            if 'z' in f:
                y = y * torch.nn.functional.silu(f['z'][t])
            out.append(torch.where(on, y, 0.0))
            h = torch.where(on[:, :, None], new, h)
        return torch.stack(out), h

    path = conv if c['op'] == 'conv' else scan
    with torch.no_grad():
        y, last = path(f)
    if c['form'] != 'train':
        return (y[0] if c['form'] == 'token' else y), last
    if c['ckpt8']:
        for k in ('x',) if c['op'] == 'conv' else ('x', 'dt', 'z'):
            if k in f:
                f[k] = stands_for(f[k])
    leaves = [f[k].requires_grad_(True) for k in s['leaves']]
    outs = path(f)
    if c['op'] == 'conv':
        return (y, last, *torch.autograd.grad(outs[:1], leaves, [f['dy']]))
    return (y, last, *torch.autograd.grad(outs, leaves, [f['dy'], f['dstate']]))
