"""GPU parity of the forms that attention, weights and eviction take for large
calls: many rows under wide heads, windows of rows over long contexts, and
selections of many long sequences. Against oracle/attend.py's definitions over
whole matrices; tolerances as in tests/test_gpu_attend.py."""
import numpy as np
import pytest
import torch

from daric_amd import cache_ops
from oracle import attend as oatt
from tests.gpu_util import make_layer, same_bytes, to_dev
from tests.test_gpu_attend import E, Case

pytestmark = pytest.mark.gpu
BF, FP, F8 = torch.bfloat16, torch.float16, torch.uint8


def want(c):
    return oatt.attend_matrix(c.layer, c.pf, c.bt, c.q, c.seqs, c.mask, c.scale, c.ks, c.vs)


def check_weigh(c, lse, weights=None):
    """weigh_tokens against its definition, and a second call against the first."""
    a = c.on_gpu()
    start = np.zeros((c.h, c.columns)) if weights is None else weights.double().numpy()
    got = []
    for _ in range(2):
        w = weights.to(c.dev) if weights is not None else None
        got.append(cache_ops.weigh_tokens(a["layer"], c.pf, a["block_table"], a["q"], lse, c.seqs, weights=w,
                                          tree_mask=a["tree_mask"], scale=c.scale, k_scale=a["k_scale"]))
    assert torch.equal(*got)
    ref, size, amax, rows = oatt.weigh_matrix(c.layer, c.pf, c.bt, c.q, lse.cpu(), c.seqs, start, c.mask, c.scale, c.ks)
    tol = (ref - start) * ((c.q.shape[2] + 10) * E * amax + 24 * E + 4 * E * size + rows * E) + 2 * E * np.abs(ref) + 1e-37
    err = np.abs(got[0].double().cpu().numpy() - ref)
    assert (err <= tol).all(), f"weights off by {(err / tol).max():.2f} of their tolerance"


# --------------------------------------------------------------- weights
# 128 workgroups of 256 tokens and more, of up to 1024 rows of a KV head, or 512 of any
# (weigh_rows_kernel).
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("dtype,qtype,layout,d,ps", [
    (BF, None, "nhd", 128, 16), (FP, None, "hnd", 128, 32), (F8, BF, "nhd", 128, 16), (F8, FP, "packed", 64, 16),
    (BF, None, "pf", 96, 16), (FP, None, "nhd", 72, 5), (F8, BF, "hnd", 80, 24), (BF, None, "nhd", 128, 5),
    (BF, None, "nhd", 256, 16), (F8, FP, "nhd", 200 - 8, 5), (FP, None, "nhd_pad", 136, 16)])
def test_windows_of_rows(dev, tree, dtype, qtype, layout, d, ps):
    c = Case(dev, [(40, 6000), (1, 70), (20, 3001)], layout, dtype, qtype, ps=ps, h=8, g=2, d=d, tree=tree, seed=70)
    c.bt[c.seqs[0][0] + 7] = 0
    c.bt[c.seqs[2][0] + 3] = -5
    if tree:
        c.mask[5::9] = 0
    out, lse = c.run()
    c.check(out, lse, want(c))
    check_weigh(c, lse)
    check_weigh(c, lse, torch.rand(8, c.columns))


@pytest.mark.parametrize("dtype", [BF, F8])
@pytest.mark.parametrize("rows,ctx,h", [(700, 4000, 8), (1100, 15300, 8), (1030, 100, 128)])
def test_windows_whose_own_rows_span_workgroups(dev, dtype, rows, ctx, h):
    """The rows that see the last tokens only are passed over for the others."""
    c = Case(dev, [(rows, ctx)], dtype=dtype, h=h, g=1, d=64, seed=71)
    _, lse = c.run()
    check_weigh(c, lse)


def test_window_of_rows_that_see_nothing(dev):
    c = Case(dev, [(40, 6000), (30, 500)], h=8, g=2, d=64, tree=True, seed=72)
    c.bt[:c.seqs[1][0]] = 0
    c.mask[:] = 0
    out, lse = c.run()
    c.check(out, lse, want(c))
    assert (lse[:40] == -torch.inf).all()
    check_weigh(c, lse)


# ------------------------------------------------- many rows of wide heads
WIDE = [(BF, None, 136, "packed"), (BF, None, 200, "nhd"), (BF, None, 256, "nhd"), (FP, None, 192, "hnd"),
        (FP, None, 256, "pf"), (F8, BF, 192, "nhd"), (F8, FP, 256, "hnd"), (F8, BF, 256, "packed"), (BF, None, 150, "nhd")]


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("ps", [5, 16])
@pytest.mark.parametrize("dtype,qtype,d,layout", WIDE)
def test_many_rows_of_wide_heads(dev, dtype, qtype, d, layout, ps, tree):
    c = Case(dev, [(20, 300), (70, 900), (1, 65), (33, 0)], layout, dtype, qtype, ps=ps, h=2, g=2, d=d, tree=tree, seed=73)
    c.bt[c.seqs[1][0] + 2] = 0
    out, lse = c.run()
    c.check(out, lse, want(c))
    check_weigh(c, lse)


@pytest.mark.parametrize("dtype,qtype", [(BF, None), (FP, None), (F8, BF)])
def test_wide_heads_in_parts(dev, dtype, qtype):
    c = Case(dev, [(17, 9000), (300, 2000)], dtype=dtype, qtype=qtype, h=2, g=1, d=256, seed=74)
    out, lse = c.run()
    c.check(out, lse, want(c))


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("d", [136, 256])
def test_rising_scores_of_wide_heads(dev, dtype, d):
    """Maxima of the first tiles that do not hold, for some rows only."""
    c = Case(dev, [(70, 1500)], dtype=dtype, d=d, g=2, h=2, seed=75)
    c.layer[0, ..., 0] = 0
    for j in range(1500):
        c.layer[0, int(c.bt[j // 16]), j % 16, :, 0] = 8.0 * (j // 400) + (40.0 if j == 1497 else 0.0)
    c.q[..., 0] = 0
    c.q[::3, :, 0] = 30.0
    c.q[1::5, :, 0] = -20.0
    out, lse = c.run()
    c.check(out, lse, want(c))
    check_weigh(c, lse)


def test_values_that_are_no_numbers_of_wide_heads(dev):
    c = Case(dev, [(60, 45)], d=256, g=1, h=2, seed=76)
    clean = want(c)
    c.layer[1, int(c.bt[50 // 16]), 50 % 16, :, 3::16] = float("inf")       # draft 5: rows from 5 on see it
    out, lse = c.run()
    bad = np.zeros(clean[0].shape, bool)
    bad[5:, :, 3::16] = True
    got = out.double().cpu()
    assert torch.isposinf(got[torch.from_numpy(bad)]).all()
    c.check(torch.where(torch.from_numpy(bad), torch.from_numpy(clean[0]), got), lse, clean)


# ------------------------------------------------------------- evictions
def evict(dev, L, h, tokens, keep, seed, shared=False, first=1, recent=2, decimals=2):
    """Sequences of these lengths over layers of small rows; many equal weights."""
    g = torch.Generator().manual_seed(seed)
    nb = sum(-(-n // 16) for n in tokens) + 1
    layers = [make_layer("nhd", nb, 16, h, 2, torch.float16, g, kind="bytes")[0] for _ in range(L)]
    bt = np.random.default_rng(seed).permutation(np.arange(1, nb)).astype(np.int32)
    ev, at, col = [], 0, 0
    for n, k in zip(tokens, keep):
        k = max(min(n, first + recent), k)
        ev.append((at, col, n, k, min(first, k), min(recent, k - min(first, k))))
        at, col = at + -(-n // 16), col + n
    w = torch.randn(L, 1 if shared else h, col, generator=g).round(decimals=decimals)
    gl, gw = [to_dev(t, dev) for t in layers], w.to(dev)
    kept = cache_ops.evict_tokens(gl, False, torch.from_numpy(bt).to(dev), gw, ev)
    torch.cuda.synchronize()
    wn = w.numpy().copy()
    ref = oatt.evict_matrix(layers, False, bt, wn, ev, kept.shape[3])
    np.testing.assert_array_equal(kept.cpu().numpy(), ref)
    np.testing.assert_array_equal(gw.cpu().numpy().view(np.uint32), wn.view(np.uint32))
    assert all(same_bytes(a, b) for a, b in zip(gl, layers))


# More than 256 selections of a call, the longest from 2049 to 16384 tokens, shorter ones
# beside it, and more than 1024 with a longer one.
@pytest.mark.parametrize("longest", [2052, 8192, 8195, 8196, 16384, 16387])
@pytest.mark.parametrize("frac", [0.1, 0.8])
def test_many_selections_of_long_sequences(dev, longest, frac):
    tokens = [longest, 20, 255, 2049, 300, 1, 2051, 64, 1500, 259, 17, 33, 700, 128, 31, 5, 2050]
    evict(dev, 2, 8, tokens, [int(n * frac) for n in tokens], 80 + longest)


@pytest.mark.parametrize("keep", [12291, 12292, 16000])
def test_many_selections_beside_the_lds(dev, keep):
    """As many chosen as a workgroup's LDS holds, and more."""
    tokens = [16384] + [40] * 16
    evict(dev, 2, 8, tokens, [keep] + [9] * 16, keep)


@pytest.mark.parametrize("n,keep", [(9000, 8500), (20000, 12291), (20000, 12292), (32771, 30000), (32772, 13000)])
def test_few_selections_beside_the_lds(dev, n, keep):
    evict(dev, 1, 2, [n, 300], [keep, 100], n)


@pytest.mark.parametrize("keep", [2000, 20000])
def test_very_many_selections_with_a_long_one(dev, keep):
    tokens = [32772] + [24 + i % 50 for i in range(31)] + [2500]
    evict(dev, 2, 16, tokens, [keep] + [11] * 31 + [1200], 90, decimals=1)


def test_many_selections_for_all_heads(dev):
    tokens = [9000, 2500] + [100] * 15
    evict(dev, 16, 2, tokens, [4000, 100] + [30] * 15, 91, shared=True)


def test_longest_sequences_need_no_selection(dev):
    """All but the recent tokens are chosen, or none is, of more than 256 sequences' heads."""
    tokens = [3000] * 17
    evict(dev, 2, 8, tokens, [2999, 3, 3000] + [4] * 14, 92)


# ------------------------------------------------------------- alignment
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("sizes,d", [([(2, 100)], 64), ([(30, 20), (1, 300)], 64), ([(300, 50)], 128), ([(40, 2000)], 256)])
def test_out_at_an_odd_element(dev, dtype, sizes, d):
    """Any element of a larger buffer may be out's first; what lies beside stays."""
    c = Case(dev, sizes, dtype=dtype, g=2, h=2, d=d, seed=77)
    plain, pl = c.run()
    for at in (1, 2, 3):
        flat = torch.full((plain.numel() + 8,), 7.0, dtype=dtype, device=dev)
        out = flat[at:at + plain.numel()].view(plain.shape)
        got, lse = c.run(out=out)
        assert got is out and torch.equal(out, plain) and torch.equal(lse, pl)
        assert (flat[:at] == 7).all() and (flat[at + plain.numel():] == 7).all()
