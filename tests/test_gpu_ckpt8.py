"""GPU tests of the 8-bit activation checkpoints: the values they stand for, to the bit, and the weight gradient that reads them."""
import pytest
import torch

import ssm_reference as R

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'


def spread(rows, C, dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, C, generator=gen) * torch.exp(3 * torch.randn(rows, 1, generator=gen))
    return x.to(dtype)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('shape', [(1, 1), (3, 31), (5, 32), (4, 33), (7, 64), (2, 250), (3, 5, 40), (2, 3, 2, 36), (130, 512)])
def test_pack_unpack(shape, dtype):
    from generative_mouse_trajectories_amd import ops_ckpt8
    x = spread(1, 1, torch.float32, 1).new_empty(0)
    C = shape[-1]
    x = spread(int(torch.tensor(shape[:-1]).prod()), C, dtype, C).reshape(shape)
    p = ops_ckpt8.pack(x.to(DEV))
    assert p.codes.shape == x.shape and p.exponents.shape == (*shape[:-1], (C + 31) // 32) and p.dtype == dtype
    want = R.stands_for(x)
    for out in (None, torch.float32, torch.bfloat16):
        got = ops_ckpt8.unpack(p, out)
        assert got.dtype == (out or dtype) and torch.equal(R.d(got), want)
    assert float((x.double() - want).abs().max()) <= float(x.abs().max()) / 127


def test_pack_at_the_borders():
    """Zeros, denormals, the largest numbers, ties, exact multiples of 127, infinities and NaN."""
    from generative_mouse_trajectories_amd import ops_ckpt8
    big = torch.finfo(torch.float32).max
    rows = [torch.zeros(32), torch.full((32,), 2.0 ** -149), torch.full((32,), 2.0 ** -126), torch.full((32,), big), torch.full((32,), -big),
            torch.arange(32) + 0.5, torch.full((32,), 127.0), torch.full((32,), 127.0 * (1 + 2 ** -23)), 127.0 * 2.0 ** torch.arange(-16, 16),
            torch.tensor([1.0] * 31 + [float('inf')]), torch.tensor([float('nan')] + [2.0] * 31), torch.tensor([-float('inf')] * 32),
            torch.tensor([127.0] + [0.5, 1.5, 2.5, -0.5, -1.5, -2.5, 126.5, -126.5] + [0.0] * 23), torch.full((32,), 127 * 2.0 ** -118)]
    x = torch.stack(rows)
    p = ops_ckpt8.pack(x.to(DEV))
    got, want = R.d(ops_ckpt8.unpack(p)), R.stands_for(x)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))
    assert int((p.exponents.cpu() == 255).sum()) == 3


def test_pack_of_views():
    from generative_mouse_trajectories_amd import ops_ckpt8
    x = spread(6 * 9, 70, torch.float32, 3).reshape(6, 9, 70).to(DEV)
    for v in (x.transpose(0, 1), x[:, ::2, 3:51], x[..., 1:33], x[0].t(), x[2, :, :64]):
        assert torch.equal(ops_ckpt8.unpack(ops_ckpt8.pack(v)), ops_ckpt8.unpack(ops_ckpt8.pack(v.contiguous())))


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('Rows,N,I', [(1, 1, 1), (5, 3, 33), (32, 128, 128), (33, 129, 127), (257, 515, 250), (1000, 64, 9), (4096, 96, 160),
                                      (20000, 130, 64), (700, 2100, 2001), (90, 4000, 3000)])
def test_weight_gradient(Rows, N, I, dtype):
    """Products are exact: the error is that of fp32 sums.  A slab adds its rows 16 at a time (Rows / 16 + 16 roundings at most),
    then slabs add up (512 / 16 + 16 at most), each a half step of the sum of magnitudes."""
    from generative_mouse_trajectories_amd import ops_ckpt8
    x = spread(Rows, I, torch.float32, Rows + I)
    gen = torch.Generator().manual_seed(N)
    dy = torch.randn(Rows, N, generator=gen).to(dtype)
    p = ops_ckpt8.pack(x.to(DEV))
    dW, db = ops_ckpt8.wgrad(dy.to(DEV), p, want_db=True)
    xs = R.stands_for(x) if Rows <= 300 else R.d(ops_ckpt8.unpack(p))      # (checked above; the plain search is slow)
    want, mag = R.d(dy).t() @ xs, R.d(dy).abs().t() @ xs.abs()
    n = Rows / 16 + 16 + 48
    assert dW.shape == (N, I) and dW.dtype == torch.float32
    assert bool(((R.d(dW) - want).abs() <= n * R.U32 * mag + 1e-30).all()), float(((R.d(dW) - want).abs() / mag.clamp(min=1e-30)).max())
    n_db = Rows / 8 + 8 + 48
    assert bool(((R.d(db) - R.d(dy).sum(0)).abs() <= n_db * R.U32 * R.d(dy).abs().sum(0) + 1e-30).all())
    again, none = ops_ckpt8.wgrad(dy.to(DEV), p)
    assert none is None and torch.equal(again, dW)


def test_weight_gradient_of_views_and_wide_range():
    """dY as a slice with an odd pitch, batch-shaped and expanded; magnitudes from 1e-30 to 1e30; a NaN block spoils its columns only."""
    from generative_mouse_trajectories_amd import ops_ckpt8
    x = spread(66, 40, torch.float32, 2)
    p = ops_ckpt8.pack(x.to(DEV))
    p3 = ops_ckpt8.pack(x.reshape(11, 6, 40).to(DEV))
    wide = torch.randn(66, 101, generator=torch.Generator().manual_seed(1)).to(DEV)
    dy = wide[:, 3:51]
    whole = ops_ckpt8.wgrad(dy.contiguous(), p, want_db=True)
    for a in (ops_ckpt8.wgrad(dy, p, want_db=True), ops_ckpt8.wgrad(dy.reshape(11, 6, 48), p3, want_db=True)):
        assert torch.equal(a[0], whole[0]) and torch.equal(a[1], whole[1])
    ones = torch.ones(1, 1, device=DEV).expand(66, 48)
    got, _ = ops_ckpt8.wgrad(ones, p)
    assert torch.equal(got, ops_ckpt8.wgrad(ones.contiguous(), p)[0])
    gen = torch.Generator().manual_seed(7)
    dy = torch.randn(66, 16, generator=gen) * 10.0 ** torch.randint(-30, 30, (1, 16), generator=gen)
    dW, _ = ops_ckpt8.wgrad(dy.to(DEV), p)
    want, mag = R.d(dy).t() @ R.stands_for(x), R.d(dy).abs().t() @ R.stands_for(x).abs()
    assert bool(((R.d(dW) - want).abs() <= 64 * R.U32 * mag).all())
    x[7, 35] = float('nan')
    dW, _ = ops_ckpt8.wgrad(dy.to(DEV), ops_ckpt8.pack(x.to(DEV)))
    bad = torch.isnan(dW).any(0).cpu()
    assert bool(bad[32:].all()) and not bool(bad[:32].any())


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_linear_with_checkpointed_input(dtype):
    from generative_mouse_trajectories_amd import ops, ops_ckpt8
    gen = torch.Generator().manual_seed(3)
    x = torch.randn(9, 16, 70, generator=gen).to(DEV, dtype).requires_grad_(True)
    w = torch.randn(50, 70, generator=gen).to(DEV, dtype).requires_grad_(True)
    b = torch.randn(50, generator=gen).to(DEV, dtype).requires_grad_(True)
    dy = torch.randn(9, 16, 50, generator=gen).to(DEV, dtype)
    y = ops.linear(x, w, b, ckpt8=True)
    assert torch.equal(y, ops.linear(x, w, b))
    gx, gw, gb = torch.autograd.grad(y, (x, w, b), dy)
    wx, = torch.autograd.grad(ops.linear(x, w, b), x, dy)
    assert torch.equal(gx, wx)
    xs = R.stands_for(x.detach().cpu()).reshape(-1, 70)
    R.close(gw, R.d(dy).reshape(-1, 50).t() @ xs, 200, 'dW')
    R.close(gb, R.d(dy).reshape(-1, 50).sum(0), 200, 'db')
    with torch.no_grad():
        assert torch.equal(ops.linear(x, w, b, ckpt8=True), y)
    assert ops.linear(x, w.detach(), None, ckpt8=True).requires_grad


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_weight_gradient_of_infinite_and_tiny_dy(dtype):
    """An infinite dY gives what the definition gives: an infinity, NaN where x is zero or infinities of both signs meet, and NaN gives NaN
    (also one whose mark is in the low half of an fp32 number).  The three bf16 numbers that an fp32 dY is cut into reach down to 2^-24 of it:
    from 2^-102 on all of them are normal, below each (and each product and sum) may lose 2^-126."""
    from generative_mouse_trajectories_amd import ops_ckpt8
    Rows, N, I = 70, 16, 40
    gen = torch.Generator().manual_seed(11)
    x = torch.randint(-100, 101, (Rows, I), generator=gen).float() / 32               # held exactly
    x[3, 4] = x[9, 35] = 0
    p = ops_ckpt8.pack(x.to(DEV))
    dy = torch.randn(Rows, N, generator=gen).to(dtype)
    dy[3, 5], dy[9, 7], dy[20, 9], dy[30, 11], dy[31, 11] = float('inf'), -float('inf'), float('nan'), float('inf'), -float('inf')
    if dtype == torch.float32:
        dy.view(torch.int32)[40, 13] = 0x7f800001
    dW, db = ops_ckpt8.wgrad(dy.to(DEV), p, want_db=True)
    want = (R.d(dy)[:, :, None] * x.double()[:, None, :]).sum(0)
    for got, ref in ((R.d(dW), want), (R.d(db), R.d(dy).sum(0))):
        assert torch.equal(torch.isnan(got), torch.isnan(ref))
        assert torch.equal(torch.isinf(got), torch.isinf(ref)) and torch.equal(got[torch.isinf(got)], ref[torch.isinf(ref)])
    assert int(torch.isinf(want[5]).sum()) > 30 and int(torch.isnan(want[5]).sum()) >= 1 and bool(torch.isnan(want[11]).any())
    fin = torch.isfinite(want)
    mag = torch.nan_to_num(R.d(dy), 0.0, 0.0, 0.0).abs().t() @ x.double().abs()
    assert bool(((R.d(dW) - want)[fin].abs() <= (Rows / 16 + 64) * R.U32 * mag[fin]).all())
    for scale in (2.0 ** -100, 2.0 ** -120):
        small = (torch.randn(Rows, N, generator=gen).double().clamp(0.25, 4.0) * scale).to(dtype)
        dW, _ = ops_ckpt8.wgrad(small.to(DEV), p)
        mag = R.d(small).abs().t() @ x.double().abs()
        lost = 3 * 2.0 ** -126 * (x.double().abs().sum(0) + Rows) if scale < 2.0 ** -102 else 0.0
        assert bool(((R.d(dW) - R.d(small).t() @ x.double()).abs() <= (Rows / 16 + 64) * R.U32 * mag + lost).all()), scale


def test_weight_gradient_of_rows_far_apart():
    from generative_mouse_trajectories_amd import ops_ckpt8
    p = ops_ckpt8.pack(spread(7, 40, torch.float32, 2).to(DEV))
    dy = torch.randn(7, 9, device=DEV)
    far = torch.zeros(8 * 2 ** 24, device=DEV)
    for pitch in (2 ** 24 - 1, 2 ** 24 + 3):
        v = far.as_strided((7, 9), (pitch, 1)).copy_(dy)
        assert torch.equal(ops_ckpt8.wgrad(v, p)[0], ops_ckpt8.wgrad(dy, p)[0])
    one = far.as_strided((1, 9), (2 ** 24, 1)).copy_(dy[:1])
    q = ops_ckpt8.pack(spread(1, 40, torch.float32, 2).to(DEV))
    assert torch.equal(ops_ckpt8.wgrad(one, q)[0], ops_ckpt8.wgrad(dy[:1], q)[0])
