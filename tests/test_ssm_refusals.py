"""What the selective state-space operators and the 8-bit checkpoints refuse: every check runs on the host before a launch (CPU)."""
import pytest
import torch

from generative_mouse_trajectories_amd import _lib, ops, ops_ckpt8, ops_ssm
from generative_mouse_trajectories_amd._lib import GmtError


@pytest.fixture
def no_launch(monkeypatch):
    """CPU tensors past the device check; reaching a launch fails the test."""
    def launch(name, *a, **k):
        raise AssertionError(f'{name} was launched')
    monkeypatch.setattr(_lib, 'call', launch)
    monkeypatch.setattr(_lib, 'require_cuda', lambda *t: None)


def seq(L=4, B=3, C=8, dtype=torch.float32):
    return torch.zeros(L, B, C, dtype=dtype)


def scan_call(**over):
    L, B, C, N = 4, 3, 8, 5
    a = dict(x=seq(), dt=seq(), A=torch.zeros(C, N), B=torch.zeros(L, B, N), C=torch.zeros(L, B, N))
    a.update(over)
    return ops_ssm.selective_scan(**a)


def step_call(**over):
    B, C, N = 3, 8, 5
    a = dict(x=torch.zeros(B, C), dt=torch.zeros(B, C), A=torch.zeros(C, N), B=torch.zeros(B, N), C=torch.zeros(B, N), state=torch.zeros(B, C, N))
    a.update(over)
    return ops_ssm.selective_scan_step(**a)


def test_cpu_tensors():
    for call in (scan_call, step_call, lambda: ops_ssm.causal_conv(seq(), torch.zeros(8, 4)), lambda: ops_ckpt8.pack(seq()),
                 lambda: ops_ssm.causal_conv_step(torch.zeros(3, 8), torch.zeros(3, 3, 8), torch.zeros(8, 4))):
        with pytest.raises(GmtError, match='GPU only'):
            call()


@pytest.mark.parametrize('over', [
    dict(x=torch.zeros(4, 3)), dict(x=seq(0)), dict(x=seq(B=0)), dict(x=seq(dtype=torch.float16)), dict(x=seq(dtype=torch.float64)),
    dict(x=seq(dtype=torch.bfloat16)), dict(dt=seq(5)), dict(dt=seq(dtype=torch.bfloat16)), dict(A=torch.zeros(7, 5)), dict(A=torch.zeros(8, 0)),
    dict(A=torch.zeros(8, 33), B=torch.zeros(4, 3, 33), C=torch.zeros(4, 3, 33)), dict(A=torch.zeros(8, 5, dtype=torch.bfloat16)),
    dict(B=torch.zeros(4, 3, 6)), dict(B=torch.zeros(4, 3, 3, 5)), dict(B=torch.zeros(4, 3, 2, 5)), dict(C=torch.zeros(4, 2, 5)),
    dict(C=torch.zeros(4, 3, 5, dtype=torch.bfloat16)), dict(C=torch.zeros(3, 5)), dict(D=torch.zeros(7)), dict(D=torch.zeros(8, dtype=torch.float64)),
    dict(z=seq(C=9)), dict(dt_bias=torch.zeros(1)), dict(state=torch.zeros(3, 5, 8)), dict(state=torch.zeros(3, 8, 5, dtype=torch.bfloat16)),
    dict(lengths=torch.zeros(3)), dict(lengths=torch.zeros(4, dtype=torch.int32)), dict(lengths=torch.zeros(3, 1, dtype=torch.int32))])
def test_scan(no_launch, over):
    with pytest.raises(GmtError):
        scan_call(**over)


@pytest.mark.parametrize('over', [
    dict(x=seq()), dict(dt=torch.zeros(3, 9)), dict(B=torch.zeros(3, 4)), dict(B=torch.zeros(3, 3, 5)), dict(state=torch.zeros(3, 8, 4)),
    dict(state=torch.zeros(3, 5, 8).transpose(1, 2)), dict(state=torch.zeros(3, 8, 5, dtype=torch.bfloat16)),
    dict(state_out=torch.zeros(3, 8, 5)[:2]), dict(active=torch.zeros(3)), dict(active=torch.zeros(2, dtype=torch.bool)),
    dict(x=torch.zeros(3, 8, requires_grad=True))])
def test_scan_step(no_launch, over):
    with pytest.raises(GmtError):
        step_call(**over)


def test_overlapping_state_buffers(no_launch):
    pool = torch.zeros(4 * 8 * 5)
    with pytest.raises(GmtError, match='overlaps'):
        step_call(state=pool[:120].view(3, 8, 5), state_out=pool[40:].view(3, 8, 5))
    pool = torch.zeros(4 * 24)
    with pytest.raises(GmtError, match='overlaps'):
        ops_ssm.causal_conv_step(torch.zeros(3, 8), pool[:72].view(3, 3, 8), torch.zeros(8, 4), state_out=pool[24:].view(3, 3, 8))


@pytest.mark.parametrize('over', [
    dict(x=torch.zeros(4, 8)), dict(x=seq(0)), dict(x=seq(dtype=torch.float16)), dict(weight=torch.zeros(8, 1)), dict(weight=torch.zeros(8, 5)),
    dict(weight=torch.zeros(7, 4)), dict(weight=torch.zeros(8, 4, dtype=torch.bfloat16)), dict(bias=torch.zeros(7)),
    dict(state=torch.zeros(4, 3, 8)), dict(state=torch.zeros(3, 3, 8, dtype=torch.bfloat16)), dict(lengths=torch.zeros(2, dtype=torch.int32))])
def test_conv(no_launch, over):
    a = dict(x=seq(), weight=torch.zeros(8, 4))
    a.update(over)
    with pytest.raises(GmtError):
        ops_ssm.causal_conv(**a)


def test_ckpt8(no_launch):
    for bad in (torch.zeros(3, 4, dtype=torch.float16), torch.zeros(0, 4), torch.zeros(())):
        with pytest.raises(GmtError):
            ops_ckpt8.pack(bad)
    good = ops_ckpt8.Ckpt8(torch.zeros(6, 40, dtype=torch.int8), torch.zeros(6, 2, dtype=torch.uint8), torch.float32)
    with pytest.raises(GmtError):
        ops_ckpt8.unpack(good, torch.float16)
    for p in (good._replace(codes=good.codes.t()), good._replace(exponents=good.exponents[:, :1]), good._replace(codes=good.codes.to(torch.uint8)),
              good._replace(exponents=good.exponents.to(torch.int8))):
        with pytest.raises(GmtError):
            ops_ckpt8.unpack(p)
    for dy in (torch.zeros(5, 8), torch.zeros(6, 8, dtype=torch.float16), torch.zeros(6, 0)):
        with pytest.raises(GmtError):
            ops_ckpt8.wgrad(dy, good)


def test_library_entry_points_check_their_arguments():
    """The C entries return codes for what they cannot run; no launch happens."""
    import ctypes
    L = _lib.lib()
    assert L.gmt_causal_conv_fwd(None, None) == -1 and L.gmt_selective_scan_fwd(None, None) == -1
    a = _lib.ConvArgs(x=16, w=16, L=1, B=1, C=4, K=5, y=16)
    assert L.gmt_causal_conv_fwd(ctypes.addressof(a), None) == -2
    a = _lib.ConvArgs(x=16, w=16, L=64, B=2, C=4, K=4, dy=16, dx=16, dparam=16, workspace=16, workspace_floats=1)
    need = ctypes.c_longlong(0)
    assert L.gmt_causal_conv_bwd_workspace_floats(ctypes.addressof(a), ctypes.addressof(need)) == 0 and need.value > 1
    assert L.gmt_causal_conv_bwd(ctypes.addressof(a), None) == -4
    s = _lib.ScanArgs(x=16, dt=16, A=16, Bm=16, Cm=16, y=16, L=4, B=2, C=6, N=33, G=1)
    assert L.gmt_selective_scan_fwd(ctypes.addressof(s), None) == -2
    s.N, s.G = 16, 4
    assert L.gmt_selective_scan_fwd(ctypes.addressof(s), None) == -1
    s.G, s.L, s.x_scale = 1, 300, 16
    assert L.gmt_selective_scan_fwd(ctypes.addressof(s), None) == -1
    s.x_scale = None
    sizes = [ctypes.c_longlong(-1) for _ in range(3)]
    assert L.gmt_selective_scan_workspace(ctypes.addressof(s), *(ctypes.addressof(v) for v in sizes)) == 0
    assert all(v.value > 0 for v in sizes)
    assert L.gmt_selective_scan_fwd(ctypes.addressof(s), None) == -4      # cut into segments: needs its workspace
    s.dy = s.dx = s.ddt = s.dB = s.dC = s.dparam = s.workspace = 16
    assert L.gmt_selective_scan_bwd(ctypes.addressof(s), None) == -1      # no kept states
    s.ck = 16
    assert L.gmt_selective_scan_bwd(ctypes.addressof(s), None) == -4
    assert L.gmt_ckpt8_pack(None, 1, 1, None, None, 1, 1, 1, 0, None) == -1
    assert L.gmt_ckpt8_wgrad(16, 128, 16, 16, 16, 1 << 20, 128, 128, 0, 0, None, 0, None) == -4
    assert L.gmt_ckpt8_wgrad(16, 4, 16, 16, 16, 1, 8, 8, 0, 0, None, 0, None) == -1


@pytest.mark.parametrize('L', [1, 130, 197, 5000])
def test_a_backward_workspace_holds_what_finding_the_states_again_takes(L):
    """From 8-bit checkpoints the backward call runs the forward pass's segments in its own workspace."""
    import ctypes
    lib, n = _lib.lib(), [ctypes.c_longlong(0) for _ in range(3)]
    for B in (1, 3, 17, 33, 38, 42, 43, 130, 600):
        for C in (1, 40, 96, 128, 273, 520, 1000):
            for N in (2, 8, 16, 32):
                a = _lib.ScanArgs(x=16, dt=16, A=16, Bm=16, Cm=16, L=L, B=B, C=C, N=N, G=1)
                assert lib.gmt_selective_scan_workspace(ctypes.addressof(a), *(ctypes.addressof(v) for v in n)) == 0
                assert n[2].value >= n[1].value, (B, C, N)


def test_capture_beside_a_live_eager_graph(monkeypatch):
    """A pass that may be differentiated is not captured while a graph from the default stream holds one of its leaves."""
    stream, capturing = [0], [False]
    monkeypatch.setattr(_lib, 'stream_of', lambda dev: stream[0])
    monkeypatch.setattr(torch.cuda, 'is_current_stream_capturing', lambda: capturing[0])

    class Twice(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, w):
            return x * w, x + w

        @staticmethod
        def backward(ctx, a, b):
            return a, b

    def run(where, captured, x, w):
        stream[0], capturing[0] = where, captured
        return ops_ckpt8.apply(Twice, 0, x, w)

    x, w = torch.ones(3, requires_grad=True), torch.ones(3, requires_grad=True)
    run(7, True, x, w)                                       # nothing lives: captured
    eager = run(0, False, x, w)
    for inputs in ((x, w), (x.detach(), w), (x * 2, torch.ones(3)), ((x * 2).view(3) + 1, torch.ones(3))):
        with pytest.raises(GmtError, match='eagerly on the default stream'):
            run(7, True, *inputs)
        run(7, False, *inputs)                               # another stream, no capture
    run(7, True, x.detach(), torch.ones(3, requires_grad=True))
    assert eager[0].grad_fn is not None
    del eager, inputs
    beside = run(5, False, x, w)                             # the first graph of its leaves is another stream's
    run(0, False, x, w)
    assert len(run(7, True, x, w)) == len(beside) == 2


@pytest.mark.parametrize('grad', [False, True])
def test_forward_mode_tangents(no_launch, grad):
    """A dual tensor is refused by every entry, with and without a leaf that requires a gradient, rather than come back without its tangent."""
    from torch.autograd import forward_ad
    w, lin = torch.zeros(8, 4, requires_grad=grad), torch.zeros(5, 8, requires_grad=True)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(seq(), torch.ones(4, 3, 8))
        one = forward_ad.make_dual(torch.zeros(3, 8), torch.ones(3, 8))
        A = forward_ad.make_dual(torch.zeros(8, 5), torch.ones(8, 5))
        for call in (lambda: ops_ssm.causal_conv(dual, w), lambda: ops_ssm.causal_conv(seq(), w, bias=one[0]),
                     lambda: scan_call(z=dual), lambda: scan_call(A=A, D=torch.zeros(8, requires_grad=grad)), lambda: step_call(dt=one),
                     lambda: ops_ssm.causal_conv_step(one, torch.zeros(3, 3, 8), w.detach()), lambda: ops_ckpt8.pack(dual),
                     lambda: ops_ckpt8.wgrad(one, ops_ckpt8.Ckpt8(torch.zeros(3, 40, dtype=torch.int8), torch.zeros(3, 2, dtype=torch.uint8), torch.float32)),
                     lambda: ops.linear(dual, lin, None, ckpt8=True)):
            with pytest.raises(GmtError, match='forward-mode'):
                call()


def test_import_under_inference_mode():
    """The package can be imported (first) within torch.inference_mode() or no_grad()."""
    import os
    import subprocess
    import sys
    code = 'import torch\nwith torch.{}():\n    import generative_mouse_trajectories_amd as g\nprint(g.ops_ckpt8._LEAF.__name__)'
    for mode in ('inference_mode', 'no_grad'):
        r = subprocess.run([sys.executable, '-c', code.format(mode)], capture_output=True, text=True, timeout=300,
                           cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
        assert r.returncode == 0 and r.stdout.strip() == 'AccumulateGrad', r.stderr[-500:]


def test_sizes_beyond_32_bits(no_launch):
    """The kernels' sizes are 32-bit: a larger one is refused (taken modulo 2^32 it would be a much smaller call that succeeds)."""
    big = 2 ** 32 + 64
    one = torch.zeros(1)
    codes, scale = torch.zeros(1, dtype=torch.int8), torch.zeros(1, dtype=torch.uint8)
    wide = one.expand(1, big)                               # (one element: every call is refused by its shape)
    for call in (lambda: ops_ckpt8.pack(wide[0]), lambda: ops_ckpt8.pack(wide), lambda: ops_ckpt8.pack(wide.view(1, big, 1)),
                 lambda: ops_ckpt8.pack(wide.view(1, 1, big)),
                 lambda: ops_ckpt8.unpack(ops_ckpt8.Ckpt8(codes.expand(1, big), scale.expand(1, big // 32), torch.float32)),
                 lambda: ops_ckpt8.wgrad(wide, ops_ckpt8.Ckpt8(codes.view(1, 1), scale.view(1, 1), torch.float32)),
                 lambda: ops_ssm.causal_conv(wide.view(big, 1, 1), torch.zeros(1, 4)), lambda: ops_ssm.causal_conv(wide.view(1, big, 1), torch.zeros(1, 4)),
                 lambda: ops_ssm.causal_conv(wide.view(1, 1, big), one.expand(big, 4)),
                 lambda: ops_ssm.causal_conv_step(wide.view(big, 1), one.expand(3, big, 1), torch.zeros(1, 4)),
                 lambda: scan_call(x=wide.view(big, 1, 1), dt=wide.view(big, 1, 1), A=torch.zeros(1, 1), B=wide.view(big, 1, 1), C=wide.view(big, 1, 1)),
                 lambda: step_call(x=wide.view(big, 1), dt=wide.view(big, 1), A=torch.zeros(1, 1), B=wide.view(big, 1), C=wide.view(big, 1),
                                   state=wide.view(big, 1, 1))):
        with pytest.raises(GmtError, match='2\\^31'):
            call()


def test_library_entry_points_check_the_number_of_steps():
    """... whose sums with a segment's length must stay within 32 bits."""
    import ctypes
    lib, n = _lib.lib(), ctypes.c_longlong(0)
    for L, want in ((2 ** 31 - 2 ** 18, 0), (2 ** 31 - 2 ** 18 + 1, -2), (2 ** 31 - 1, -2)):
        a = _lib.ConvArgs(x=16, w=16, L=L, B=1, C=4, K=4, dy=16, dx=16, dparam=16)
        assert lib.gmt_causal_conv_bwd_workspace_floats(ctypes.addressof(a), ctypes.addressof(n)) == want
        s = _lib.ScanArgs(x=16, dt=16, A=16, Bm=16, Cm=16, y=16, L=L, B=1, C=1, N=1, G=1)
        sizes = [ctypes.c_longlong(0) for _ in range(3)]
        assert lib.gmt_selective_scan_workspace(ctypes.addressof(s), *(ctypes.addressof(v) for v in sizes)) == want


def scan_sizes(**over):
    """Return code of the workspace entry (which makes the checks of forward and backward calls) and the sizes."""
    import ctypes
    a = dict(x=16, dt=16, A=16, Bm=16, Cm=16, L=2, B=1, C=1, N=1, G=1)
    a.update(over)
    s = _lib.ScanArgs(**a)
    n = [ctypes.c_longlong(0) for _ in range(3)]
    return _lib.lib().gmt_selective_scan_workspace(ctypes.addressof(s), *(ctypes.addressof(v) for v in n))


@pytest.mark.parametrize('inside,outside', [
    (dict(B=2 ** 17, C=2 ** 10 - 1), dict(B=2 ** 17, C=2 ** 10)),                                      # B C < 2^27
    (dict(C=2 ** 24 - 1), dict(C=2 ** 24)),                                                            # C < 2^24
    (dict(B=2 ** 16, C=64, G=64, N=15), dict(B=2 ** 16, C=64, G=64, N=16)),                            # B G N < 2^26
    (dict(B=4, N=16, B_t=2 ** 26 - 1, C_t=2 ** 26 - 1), dict(B=4, N=16, B_t=2 ** 26)),                 # pitches of a step
    (dict(x_t=2 ** 27 - 1, dt_t=2 ** 27 - 1, z=16, z_t=2 ** 27 - 1, dy_t=2 ** 27 - 1), dict(dy_t=2 ** 27)),
    (dict(B=4096, C=1024, G=1024, N=8), dict(B=4096, C=1024, G=1024, N=16)),                           # a workgroup per row and group: no limit of its own
    (dict(B=2 ** 25, C=2), dict(B=2 ** 26, C=2))])
def test_the_limits_of_a_scan_are_the_documented_ones(inside, outside):
    assert scan_sizes(**inside) == 0
    assert scan_sizes(**outside) == -2


def test_sequences_with_far_steps_are_copied(no_launch, monkeypatch):
    """A pitch of a step that the kernels do not reach is no refusal: the sequence is copied, and the pitch of a single step does not count."""
    seen = {}

    def launch(name, args, *a, **k):
        if name == 'gmt_selective_scan_fwd':
            s = _lib.ScanArgs.from_address(args)
            seen.update({n: getattr(s, n) for n in ('x_t', 'dt_t', 'z_t', 'B_t', 'C_t', 'x_b', 'B_b')})
    monkeypatch.setattr(_lib, 'call', launch)
    monkeypatch.setattr(_lib, 'stream_of', lambda dev: 0)
    monkeypatch.setattr(ops_ssm, 'on', lambda dev: ops_ckpt8._HERE)
    far = torch.empty(2 ** 27 + 64)                         # (untouched memory but for its ends)
    far[:64] = 1
    far[-64:] = 2

    def steps(L, pitch, *rest):
        t = torch.zeros(rest)
        return far.as_strided((L, *rest), (pitch, *t.stride()))
    with torch.no_grad():
        for L, pitch, mapped in ((2, 2 ** 27, 2 ** 26), (2, 2 ** 27 - 1, 2 ** 26 - 1), (1, 2 ** 27, 2 ** 27)):
            x, m = steps(L, pitch, 3, 8), steps(L, mapped, 3, 5)
            ops_ssm.selective_scan(x, x, torch.zeros(8, 5), m, m, z=x)
            want = dict(x_t=24, B_t=15) if pitch == 2 ** 27 and L > 1 else dict(x_t=pitch, B_t=mapped) if L > 1 else dict(x_t=0, B_t=0)
            assert seen == dict(x_t=want['x_t'], dt_t=want['x_t'], z_t=want['x_t'], B_t=want['B_t'], C_t=want['B_t'], x_b=8, B_b=5), (L, pitch)


def test_the_limits_of_a_single_scan_step_are_its_own():
    """64-bit indexing over rows: neither a whole sequence's limits nor its workgroups' count.  (-1: past the limits, the output is missing.)"""
    import ctypes
    for want, over in ((-1, dict(B=2 ** 20, C=256)), (-1, dict(B=2 ** 22, C=16, N=8)), (-1, dict(B=2 ** 31 - 2 ** 18, C=1, N=32)),
                       (-1, dict(B=1, C=2 ** 26 - 1, N=32)), (-2, dict(B=1, C=2 ** 26)), (-2, dict(B=1, C=4, N=33)), (-1, dict(B=1, C=4, G=3))):
        a = dict(x=16, dt=16, A=16, Bm=16, Cm=16, state=16, state_out=16, L=1, N=16, G=1)
        a.update(over)
        s = _lib.ScanArgs(**a)
        assert _lib.lib().gmt_selective_scan_step(ctypes.addressof(s), None, None) == want, over


def test_the_limits_of_the_convolution():
    """Whole sequences: B C < 2^31, C <= 2^30 - 64; a single step: neither.  (-1: past the limits, the output is missing.)"""
    import ctypes
    lib, n = _lib.lib(), ctypes.c_longlong(0)
    for want, over in ((0, dict(B=2 ** 21, C=1023)), (-2, dict(B=2 ** 21, C=1024)), (0, dict(B=2 ** 30 - 1, C=2)), (-2, dict(B=2 ** 30, C=2)),
                       (0, dict(B=1, C=2 ** 30 - 64)), (-2, dict(B=1, C=2 ** 30 - 63))):
        a = dict(x=16, w=16, L=1, K=4, dy=16, dx=16, dparam=16, bf16=1)
        a.update(over)
        a = _lib.ConvArgs(**a)
        assert lib.gmt_causal_conv_bwd_workspace_floats(ctypes.addressof(a), ctypes.addressof(n)) == want, over
        assert lib.gmt_causal_conv_fwd(ctypes.addressof(a), None) == (want or -1), over
        assert lib.gmt_causal_conv_bwd(ctypes.addressof(a), None) == (want or -1), over
    for want, over in ((-1, dict(B=2 ** 22, C=1024)), (-1, dict(B=2 ** 31 - 2 ** 18, C=4)), (-2, dict(B=1, C=4, K=5))):
        a = dict(x=16, w=16, state=16, state_out=16, L=1, K=4, bf16=1)
        a.update(over)
        a = _lib.ConvArgs(**a)
        assert lib.gmt_causal_conv_step(ctypes.addressof(a), None, None) == want, over


def test_weight_gradient_of_rows_far_apart(no_launch, monkeypatch):
    """A row pitch that the kernel's 32-bit offsets do not reach is copied, and the pitch of a single row does not count."""
    seen = []
    monkeypatch.setattr(_lib, 'call', lambda name, *a, **k: seen.append(a[1]) if name == 'gmt_ckpt8_wgrad' else None)
    monkeypatch.setattr(_lib, 'stream_of', lambda dev: 0)
    monkeypatch.setattr(ops_ckpt8, 'on', lambda dev: ops_ckpt8._HERE)
    far = torch.empty(2 ** 24 + 64)
    for R, pitch, want in ((2, 2 ** 24 - 1, 2 ** 24 - 1), (2, 2 ** 24, 8), (1, 2 ** 24, 8), (1, 3, 8)):
        p = ops_ckpt8.Ckpt8(torch.zeros(R, 40, dtype=torch.int8), torch.zeros(R, 2, dtype=torch.uint8), torch.float32)
        ops_ckpt8.wgrad(far.as_strided((R, 8), (pitch, 1)), p)
        assert seen.pop() == want and not seen, (R, pitch)


def test_the_limits_of_the_weight_gradient():
    """-4: past the limits, the workspace is missing."""
    lib = _lib.lib()
    for want, over in ((-4, dict(ldy=2 ** 24 - 1)), (-2, dict(ldy=2 ** 24)), (-2, dict(N=1, I=2 ** 24))):
        a = dict(ldy=128, R=1 << 20, N=128, I=128)
        a.update(over)
        assert lib.gmt_ckpt8_wgrad(16, max(a['ldy'], a['N']), 16, 16, 16, a['R'], a['N'], a['I'], 0, 0, None, 0, None) == want, over
