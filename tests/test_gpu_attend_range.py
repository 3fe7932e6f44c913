"""GPU parity of attention where one token outweighs the others by far, so that
what the light ones add lies at the low end of a 16-bit weight's range."""
import numpy as np
import pytest
import torch

from oracle import attend as oatt
from tests.test_gpu_attend import E, U, Case

pytestmark = pytest.mark.gpu


def want(c):
    return oatt.attend_matrix(c.layer, c.pf, c.bt, c.q, c.seqs, c.mask, c.scale, c.ks, c.vs)


def check(c, out):
    """The bound of tests/test_gpu_attend.py with what fp16 weights lose named by where
    they stand: the heaviest token that a sum has met weighs 2^14 at least in it (to
    half a step), so a weight is rounded to half a step relative, or below fp16's
    normal range, 2^-14, by 2^-25: 2^-39 of the heaviest. Sums of n weights over
    their largest: n 2^-39 max |V|."""
    ref, _, mag, amax, vmax, n = want(c)
    d = (c.q.shape[2] + 10) * E * amax + 24 * E
    u = U[c.qtype]
    tol = (u + 2 * d + 2 * n * E)[..., None] * mag + u * np.abs(ref) + 2.0 ** -25
    if c.qtype == torch.float16:
        tol += (n * vmax)[..., None] * 2.0 ** -39
    err = np.abs(out.double().cpu().numpy() - ref)
    assert (err <= tol).all(), f"out off by {(err / tol).max():.2f} of its tolerance"


def spread(c, nats, every):
    """Token j's score is 0, or a little more, or (one in `every`) `nats`; V of the heavy
    ones is 0, of the light ones large."""
    f8 = c.layer.dtype == torch.uint8
    code = (lambda x: x.to(torch.float8_e4m3fn).view(torch.uint8)) if f8 else (lambda x: x.to(c.layer.dtype))
    big = 256.0 if f8 else 2048.0
    gen = torch.Generator().manual_seed(3)
    c.layer[0] = 0
    c.q[:] = 0
    c.q[..., 0] = 8.0
    c.scale = nats / 8.0
    if f8:
        c.ks[:] = 1.0
        c.vs[:] = 8.0
    for bo, _, n, ctx, _ in c.seqs:
        j = torch.arange(n + ctx)
        heavy = j % every == 5 % every
        k = torch.where(heavy, 1.0, (j % 3) / 64.0)
        v = big * (0.5 + 0.5 * torch.rand(n + ctx, c.layer.shape[-1], generator=gen))
        v[heavy] = 0
        page, slot = torch.from_numpy(c.bt[bo + (j // 16).numpy()]).long(), j % 16
        c.layer[0, page, slot, :, 0] = code(k)[:, None]
        c.layer[1, page, slot] = code(v)[:, None]


@pytest.mark.parametrize("dtype,qtype", [(torch.float16, None), (torch.uint8, torch.float16), (torch.bfloat16, None)])
@pytest.mark.parametrize("rows,ctx,g,d", [(1, 3000, 4, 64), (40, 1000, 2, 128), (300, 700, 1, 128), (70, 500, 2, 64),
                                          (40, 700, 1, 256)])
@pytest.mark.parametrize("nats,every", [(12.0, 31), (15.5, 31), (17.0, 31), (17.0, 1000), (19.0, 500)])
def test_light_tokens_beside_heavy_ones(dev, dtype, qtype, rows, ctx, g, d, nats, every):
    c = Case(dev, [(rows, ctx)], dtype=dtype, qtype=qtype, g=g, h=1, d=d, seed=95)
    spread(c, nats, every)
    out, lse = c.run()
    check(c, out)


def test_a_long_light_context(dev):
    """One sequence of 60000 light tokens whose heavy one stands in each part."""
    c = Case(dev, [(1, 60000)] * 4, dtype=torch.float16, g=4, h=8, d=64, seed=96)
    spread(c, 17.0, 300)
    out, lse = c.run()
    check(c, out)


@pytest.mark.parametrize("rows", [1, 40])
def test_scores_that_rise_by_little(dev, rows):
    """A maximum passed again and again, by less than a power of 2 and by more."""
    for step in (0.01, 0.5, 3.0, 30.0):
        c = Case(dev, [(rows, 1500)], dtype=torch.float16, g=2, h=1, d=64, seed=97)
        spread(c, 1.0, 10 ** 6)
        j = torch.arange(1500)
        rise = ((j // 32) * step / 8).to(torch.float16)
        c.layer[0, torch.from_numpy(c.bt[(j // 16).numpy()]).long(), j % 16, :, 0] = rise[:, None]
        c.scale = 1.0
        out, lse = c.run()
        check(c, out)
        c.check(out, lse, want(c))


@pytest.mark.parametrize("dtype,top", [(torch.float16, 6e4), (torch.bfloat16, 6e4), (torch.bfloat16, 1e7)])
@pytest.mark.parametrize("rows,d", [(1, 64), (40, 64), (40, 128), (300, 128), (40, 256)])
@pytest.mark.parametrize("late", [False, True])
def test_huge_scores_choose_one_token(dev, dtype, top, rows, d, late):
    """Scores up to 10^14, further apart than 100 each: a row's output is V of the
    heaviest token that it sees, whatever fp32 makes of the others."""
    c = Case(dev, [(rows, 700)], dtype=dtype, g=2, h=1, d=d, seed=98)
    c.layer[0] = 0
    c.q[:] = 0
    c.q[..., 0] = top
    c.q[1::3, :, 0] = -top
    c.scale = 0.3
    n = rows + 700
    heavy, light = (690, 3) if late else (3, 690)        # of positive, of negative q
    gen = torch.Generator().manual_seed(1)
    k = top * (0.1 + 0.3 * torch.rand(n, generator=gen)) * torch.sign(torch.randn(n, generator=gen))
    k[heavy], k[light] = top * 0.9, -top * 0.9
    j = torch.arange(n)
    c.layer[0, torch.from_numpy(c.bt[(j // 16).numpy()]).long(), j % 16, :, 0] = k.to(dtype)[:, None]
    out, lse = c.run()
    for sign, at in ((1, heavy), (-1, light)):
        mine = [i for i in range(rows) if (sign < 0) == (i % 3 == 1)]
        v = c.layer[1, int(c.bt[at // 16]), at % 16, 0]
        if mine:
            assert torch.equal(out[mine].cpu(), v.expand(len(mine), 2, d))
    assert torch.isfinite(lse).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,ctx", [(1, 0), (1, 6), (7, 0), (60, 0), (1, 900), (30, 900)])
def test_lse_of_equal_scores(dev, dtype, rows, ctx):
    """Scores of 0 over n tokens: log n. The logarithm in powers of 2 is good to an ulp,
    2 e of a value of up to 10 (e = 2^-24), and the parts' sums (of ones) are exact; with the
    product by log 2 and its constant, 4 e of the larger of 1 and log n."""
    c = Case(dev, [(rows, ctx)], dtype=dtype, g=2, h=1, d=64, seed=99)
    c.q[:] = 0
    _, lse = c.run()
    ref = np.log(ctx + 1.0 + np.arange(rows))[:, None]
    assert (np.abs(lse.double().cpu().numpy() - ref) <= 4 * E * np.maximum(1.0, ref)).all()


@pytest.mark.parametrize("dtype,top", [(torch.float16, 2.0 ** 15), (torch.bfloat16, 2.0 ** 17)])
@pytest.mark.parametrize("rows,d", [(1, 64), (40, 64), (40, 128), (300, 128), (40, 256)])
def test_huge_scores_an_ulp_apart(dev, dtype, top, rows, d):
    """Scores of 2^30 and 2^34 that rise token by token by the least that fp32 holds
    there, far more than a weight's range: whichever of them fp32 tells apart, the output
    lies between V's smallest and largest value (half a step of it each, for the weights
    and the result)."""
    c = Case(dev, [(rows, 700)], dtype=dtype, g=2, h=1, d=d, seed=100)
    n = rows + 700
    c.layer[0] = 0
    c.layer[1] = (1 + torch.rand(c.layer[1].shape, generator=torch.Generator().manual_seed(2))).to(dtype)
    c.q[:] = 0
    c.q[..., 0] = top
    c.q[..., 1] = top * top * 2.0 ** -23 / 8               # times 8 steps: an ulp of top * top
    c.q[1::3] *= 0.5
    c.scale = 0.3
    j = torch.arange(n)
    page, slot = torch.from_numpy(c.bt[(j // 16).numpy()]).long(), j % 16
    c.layer[0, page, slot, :, 0] = top
    c.layer[0, page, slot, :, 1] = ((j // 20) * 8.0).to(dtype)[:, None]
    out, lse = c.run()
    assert torch.isfinite(lse).all()
    u = U[dtype]
    assert (out >= 1 - 2 * u).all() and (out <= 2 * (1 + 2 * u)).all()


@pytest.mark.parametrize("dtype,qtype", [(torch.float16, None), (torch.uint8, torch.float16)])
@pytest.mark.parametrize("rows,ctx", [(1, 3000), (40, 1000), (300, 700)])
@pytest.mark.parametrize("nats", [20.5, 21.5, 22.5])
def test_weights_below_the_normal_range(dev, dtype, qtype, rows, ctx, nats):
    """Light tokens whose weights are subnormal in fp16, 2^-15.6 to 2^-18.5: they lose
    bits, not all."""
    c = Case(dev, [(rows, ctx)], dtype=dtype, qtype=qtype, g=2, h=1, d=64, seed=101)
    spread(c, nats, 500)
    out, lse = c.run()
    check(c, out)
    assert (out[..., 0] > 0).float().mean() > 0.9
