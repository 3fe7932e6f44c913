"""GPU parity of attend_pages, weigh_tokens and evict_tokens against their
definitions in 64 bits (oracle/attend.py), and the loop of the three.

Tolerances. u is half a step of q's type relative to the value
(finfo(t).eps / 2), e = 2^-24 that of fp32. A score is a sum of D products
exact in fp32, so it is off by at most (D + 8) e A, A the row's largest sum of
|q k| times the scale (8: the scale's and the logarithms' conversions); a
weight's exponential by 4 e more, plus the exponent's own rounding, |x| e for
an exponent x of at most 2 A + 16 (the running maximum is within 8 of the true one
in powers of 2): d = (D + 8 + 2) e A + 24 e relative, twice in the quotient.
The weights are then rounded to q's type (u relative; fp16 below its normal
range 2^-25 absolute, where the largest weight is at least 1), summed with V over n
tokens in fp32, and the result rounded once more:
  out: (u + 2 d + 2 n e) sum P |V| + u |out| (+ n 2^-25 max |V| in fp16, and 2^-25)
  lse: d + 4 e (|lse| + 1) + n e
A token's weight over R rows: w (d + 4 e (|x| + |lse|) + R e)."""
import numpy as np
import pytest
import torch

from daric_amd import cache_ops
from oracle import attend as oatt
from tests.gpu_util import make_layer, same_bytes, to_dev

pytestmark = pytest.mark.gpu
E = 2.0 ** -24
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


class Case:
    """Sequences of (rows, context) over one layer of random pages."""

    def __init__(self, dev, sizes, layout="nhd", dtype=torch.bfloat16, qtype=None, ps=16, h=2, g=4, d=64, tree=False,
                 seed=0, words=None, spare=3):
        gen = torch.Generator().manual_seed(seed)
        rng = np.random.default_rng(seed)
        pages = [-(-(n + c) // ps) for n, c in sizes]
        nb = sum(pages) + spare + 1
        self.layer, self.pf = make_layer(layout, nb, ps, h, d, dtype, gen)
        ids = rng.permutation(np.arange(1, nb))
        self.bt = ids[:max(sum(pages), 1)].astype(np.int32)
        self.seqs, at, row, col = [], 0, 0, 0
        for (n, c), p in zip(sizes, pages):
            self.seqs.append((at, row, n, c, col))
            at, row, col = at + p, row + n, col + n + c
        self.T, self.columns, self.h = row, col, h
        self.qtype = qtype or (dtype if dtype != torch.uint8 else torch.bfloat16)
        self.q = (2 * torch.randn(self.T, h * g, d, generator=gen)).to(self.qtype)
        self.mask = None
        if tree:
            longest = max(n for n, _ in sizes)
            w = words or max(1, -(-longest // 64))
            self.mask = torch.from_numpy(rng.integers(0, 2 ** 64, (self.T, w), dtype=np.uint64).view(np.int64))
        self.ks = self.vs = None
        if dtype == torch.uint8:
            self.ks = torch.from_numpy(rng.uniform(0.1, 1, h).astype(np.float32))
            self.vs = torch.from_numpy(rng.uniform(0.1, 1, h).astype(np.float32))
        self.scale = d ** -0.5
        self.dev = dev

    def on_gpu(self):
        m = lambda t: t.to(self.dev) if t is not None else None
        return dict(layer=to_dev(self.layer, self.dev), page_first=self.pf,
                    block_table=torch.from_numpy(self.bt).to(self.dev), q=m(self.q), seqs=self.seqs,
                    tree_mask=m(self.mask), scale=self.scale, k_scale=m(self.ks))

    def want(self):
        return oatt.attend(self.layer, self.pf, self.bt, self.q, self.seqs, self.mask, self.scale, self.ks, self.vs)

    def check(self, out, lse, want=None):
        ref, rlse, mag, amax, vmax, seen = want or self.want()
        n, D = seen.astype(float), self.q.shape[2]
        u = U[self.qtype]
        got, glse = out.double().cpu().numpy(), lse.double().cpu().numpy()
        d = (D + 10) * E * amax + 24 * E
        tol = (u + 2 * d + 2 * n * E)[..., None] * mag + u * np.abs(ref) + 2.0 ** -25
        if self.qtype == torch.float16:
            tol += (n * vmax)[..., None] * 2.0 ** -25
        rows = ~np.isnan(ref)
        err = np.abs(got - ref)
        assert (err[rows] <= tol[rows]).all(), f"out off by {np.nanmax(err[rows] / tol[rows]):.2f} of its tolerance"
        dead = rlse == -np.inf
        assert (glse[dead] == -np.inf).all() and (got[dead] == 0).all()
        live = ~dead & ~np.isnan(rlse)
        tl = d + 4 * E * (np.abs(rlse) + 1) + n * E
        assert (np.abs(glse - rlse)[live] <= tl[live]).all()

    def run(self, **more):
        a = self.on_gpu()
        a["v_scale"] = self.vs.to(self.dev) if self.vs is not None else None
        a.update(more)
        r = cache_ops.attend_pages(a.pop("layer"), a.pop("page_first"), a.pop("block_table"), a.pop("q"), a.pop("seqs"), **a)
        torch.cuda.synchronize()
        return r

    def check_weigh(self, lse, weights=None, **more):
        a = self.on_gpu()
        a.update(more)
        start = np.zeros((self.h, self.columns)) if weights is None else weights.double().numpy()
        w = weights.to(self.dev) if weights is not None else None
        got = cache_ops.weigh_tokens(a["layer"], self.pf, a["block_table"], a["q"], lse, self.seqs, weights=w,
                                     tree_mask=a["tree_mask"], scale=self.scale, k_scale=a["k_scale"])
        torch.cuda.synchronize()
        assert w is None or got is w
        self.weights = got
        ref, size, amax, rows = oatt.weigh(self.layer, self.pf, self.bt, self.q, lse.cpu(), self.seqs, start, self.mask,
                                           self.scale, self.ks)
        D = self.q.shape[2]
        tol = (ref - start) * ((D + 10) * E * amax + 24 * E + 4 * E * size + rows * E) + 2 * E * np.abs(ref) + 1e-37
        err = np.abs(got.double().cpu().numpy() - ref)
        assert (err <= tol).all(), f"weights off by {(err / tol).max():.2f} of their tolerance"


LAYOUTS = ["nhd", "hnd", "pf", "pf_hnd", "packed", "nhd_pad"]
TYPES = [(torch.bfloat16, None), (torch.float16, None), (torch.uint8, torch.bfloat16), (torch.uint8, torch.float16)]


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("dtype,qtype", TYPES)
def test_layouts_and_types(dev, layout, dtype, qtype):
    c = Case(dev, [(1, 37), (5, 200), (1, 0), (33, 1)], layout, dtype, qtype, seed=1)
    out, lse = c.run()
    c.check(out, lse)
    c.check_weigh(lse)


@pytest.mark.parametrize("d", [2, 6, 8, 24, 40, 64, 72, 80, 96, 128, 136, 192, 200, 256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.uint8])
def test_head_sizes(dev, d, dtype):
    c = Case(dev, [(3, 70), (1, 129)], "packed" if d % 16 else "hnd", dtype, d=d, seed=2)
    out, lse = c.run()
    c.check(out, lse)
    c.check_weigh(lse)


@pytest.mark.parametrize("ps", [1, 2, 5, 8, 16, 48, 64, 256])
@pytest.mark.parametrize("g", [1, 3, 5, 16, 21])
def test_pages_and_groups(dev, ps, g):
    c = Case(dev, [(1, 301), (7, 64), (2, 31)], ps=ps, g=g, h=3, d=128, seed=ps + g)
    out, lse = c.run()
    c.check(out, lse)
    c.check_weigh(lse, torch.rand(3, c.columns))


@pytest.mark.parametrize("ctx", [0, 1, 15, 16, 31, 32, 33, 127, 128, 129, 255, 1000])
def test_single_tokens(dev, ctx):
    c = Case(dev, [(1, ctx)], d=128, h=8, seed=ctx)
    out, lse = c.run()
    c.check(out, lse)
    c.check_weigh(lse)


@pytest.mark.parametrize("sizes", [[(5, 40), (64, 7), (65, 0), (130, 513)], [(1, 0)], [(200, 95), (1, 33)]])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.uint8])
def test_trees(dev, sizes, dtype):
    # random bits, rows whose mask leaves nothing among them
    c = Case(dev, sizes, dtype=dtype, tree=True, seed=5, words=4)
    c.mask[::7] = 0
    c.mask[3::11] = -1
    out, lse = c.run()
    c.check(out, lse)
    c.check_weigh(lse)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.uint8])
def test_long_context_in_parts(dev, dtype):
    c = Case(dev, [(1, 20011), (2, 40), (17, 5000)], dtype=dtype, d=128, seed=6)
    out, lse = c.run()
    c.check(out, lse)
    c.check_weigh(lse)


@pytest.mark.parametrize("rows,ctx", [(300, 0), (257, 100), (1000, 31), (129, 2000)])
@pytest.mark.parametrize("dtype,qtype", TYPES)
def test_runs_of_rows(dev, rows, ctx, dtype, qtype):
    c = Case(dev, [(rows, ctx), (3, 50)], dtype=dtype, qtype=qtype, d=128, g=2, h=1, seed=7)
    out, lse = c.run()
    c.check(out, lse)
    c.check_weigh(lse)


def poison(layer):
    """NaN (or e4m3 NaN) everywhere."""
    if layer.dtype == torch.uint8:
        layer.fill_(0x7F)
    else:
        layer.fill_(float("nan"))
    return layer


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.uint8])
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("ps", [5, 16])
def test_what_is_not_seen_has_no_effect(dev, dtype, tree, ps):
    """Null and out-of-range pages, slots behind the last token and other
    pages hold NaN; the result is that of the clean cache."""
    c = Case(dev, [(3, 100), (40, 33), (2, 200)], dtype=dtype, d=96, tree=tree, ps=ps, seed=8)
    pages = [c.seqs[1][0], c.seqs[2][0] - c.seqs[1][0], 0]
    c.bt[c.seqs[0][0] + 1] = 0                          # the null block
    c.bt[c.seqs[2][0] + 2] = c.layer.shape[1]           # past the pool
    c.bt[c.seqs[2][0] + 4] = -7
    clean = c.layer
    dirty = poison(clean.clone())
    ps_ = c.layer.shape[2]
    for bo, _, n, ctx, _ in c.seqs:
        for j in range(n + ctx):
            b = int(c.bt[bo + j // ps_])
            if 0 < b < clean.shape[1]:
                dirty[:, b, j % ps_] = clean[:, b, j % ps_]
    assert pages
    want = c.want()
    c.layer = dirty
    out, lse = c.run()
    c.check(out, lse, want)
    assert torch.isfinite(out.float()).all()
    c.layer = clean
    ref_w = None
    for layer in (clean, dirty):
        a = c.on_gpu()
        w = cache_ops.weigh_tokens(to_dev(layer, dev), c.pf, a["block_table"], a["q"], lse, c.seqs,
                                   tree_mask=a["tree_mask"], scale=c.scale, k_scale=a["k_scale"])
        assert torch.isfinite(w).all()
        assert ref_w is None or torch.equal(w, ref_w)
        ref_w = w


@pytest.mark.parametrize("dtype,bad", [(torch.bfloat16, float("inf")), (torch.float16, float("-inf")),
                                       (torch.bfloat16, float("nan")), (torch.uint8, 0x7F)])
def test_unseen_drafts_with_infinities(dev, dtype, bad):
    """A draft's K and V that some rows see and others do not: those that do get
    what the formula gives, the others nothing of it."""
    c = Case(dev, [(20, 45), (6, 3)], dtype=dtype, d=64, tree=True, seed=9)
    c.mask[:] = -1
    c.mask[:10] &= ~((1 << 4) | (1 << 11))               # rows 0..9 do not see drafts 4 and 11
    clean = c.layer.clone()
    ps = c.layer.shape[2]
    hit = []
    for j in (45 + 4, 45 + 11):
        b = int(c.bt[c.seqs[0][0] + j // ps])
        c.layer[1, b, j % ps, :, 3::16] = bad            # some dims of V
        hit.append((b, j % ps))
    with np.errstate(all="ignore"):
        want = c.want()
    dirty, c.layer = c.layer, clean
    wclean = c.want()
    c.layer = dirty
    out, lse = c.run()
    got = out.double().cpu().numpy()
    finite = np.isfinite(want[0])
    assert not finite.all() and finite[:10].all() and finite[20:].all() and not finite[10:20, :, 3::16].any()
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want[0]))
    np.testing.assert_array_equal(got[~finite], want[0][~finite])
    # all that is finite is the clean cache's
    out2 = torch.where(torch.from_numpy(finite).to(dev), out.double(), torch.from_numpy(wclean[0]).to(dev))
    c.check(out2, lse, wclean)


@pytest.mark.parametrize("rows", [3, 20, 150])
def test_infinities_that_are_seen(dev, rows):
    """Values of V that are no numbers, in cached tokens and among the run's own, reach
    every row that sees them."""
    c = Case(dev, [(rows, 45), (2, 3)], d=64, seed=29)
    clean = c.layer.clone()
    for j, bad in ((7, float("inf")), (45 + 1, float("-inf")), (45 + rows - 1, float("nan"))):
        c.layer[1, int(c.bt[j // 16]), j % 16, :, 3::16] = bad
    with np.errstate(all="ignore"):
        want = c.want()
    dirty, c.layer = c.layer, clean
    wclean = c.want()
    c.layer = dirty
    out, lse = c.run()
    got, finite = out.double().cpu().numpy(), np.isfinite(want[0])
    np.testing.assert_array_equal(got[~finite], want[0][~finite])
    assert np.isnan(want[0][1:rows, :, 3]).all() and np.isposinf(want[0][0, :, 3]).all()
    out2 = torch.where(torch.from_numpy(finite).to(dev), out.double(), torch.from_numpy(wclean[0]).to(dev))
    c.check(out2, lse, wclean)


def test_rows_that_see_nothing(dev):
    c = Case(dev, [(4, 0), (3, 50)], tree=True, seed=10)
    c.mask[:] = 0
    c.bt[c.seqs[1][0]:] = 0
    out, lse = c.run()
    assert (out == 0).all() and (lse == -torch.inf).all()
    c.check_weigh(lse)


def test_scores_of_all_sizes(dev):
    """Rising, falling and huge scores, a negative and a zero scale."""
    for scale, f in ((0.125, 30.0), (-0.125, 30.0), (0.0, 1.0), (4.0, 100.0)):
        c = Case(dev, [(1, 700), (9, 64), (40, 20)], d=64, seed=11)
        ramp = torch.linspace(-f, f, 64 * 16).view(1, -1, 1, 1)
        for bo, _, n, ctx, _ in c.seqs:
            for j in range(n + ctx):
                c.layer[0, int(c.bt[bo + j // 16]), j % 16] = ramp[0, j % ramp.shape[1], 0, 0]
        c.scale = scale
        out, lse = c.run()
        c.check(out, lse)
        c.check_weigh(lse)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,ctx", [(1, 2000), (70, 1500), (300, 700)])
def test_rising_scores(dev, dtype, rows, ctx):
    """Scores that rise by hundreds along the context, for some rows only, late and
    more than once: maxima taken early do not hold."""
    c = Case(dev, [(rows, ctx)], dtype=dtype, d=64, g=2, h=2, seed=28)
    c.layer[0, ..., 0] = 0
    for j in range(ctx):
        b = int(c.bt[j // 16])
        c.layer[0, b, j % 16, :, 0] = 8.0 * (j // 400) + (40.0 if j == ctx - 3 else 0.0)
    c.q[..., 0] = 0
    c.q[::3, :, 0] = 30.0
    c.q[1::5, :, 0] = -20.0
    out, lse = c.run()
    c.check(out, lse)
    c.check_weigh(lse)


def test_given_outputs_and_rows_of_no_sequence(dev):
    c = Case(dev, [(3, 40), (2, 17)], seed=12)
    seqs = [(s[0], s[1] + 1 + i, *s[2:]) for i, s in enumerate(c.seqs)]     # a row free before each
    T = c.T + 3
    q = torch.zeros(T, *c.q.shape[1:], dtype=c.qtype)
    for s, t in zip(c.seqs, seqs):
        q[t[1]:t[1] + t[2]] = c.q[s[1]:s[1] + s[2]]
    out = torch.full(q.shape, 7.0, dtype=c.qtype, device=dev)
    lse = torch.full(q.shape[:2], 7.0, device=dev)
    r = c.run(q=q.to(dev), seqs=seqs, out=out, lse=lse)
    assert r[0] is out and r[1] is lse
    want, wl = c.run()
    for s, t in zip(c.seqs, seqs):
        assert torch.equal(out[t[1]:t[1] + t[2]], want[s[1]:s[1] + s[2]])
        assert torch.equal(lse[t[1]:t[1] + t[2]], wl[s[1]:s[1] + s[2]])
    free = [0, 1 + 3, T - 1]
    assert (out[free] == 7).all() and (lse[free] == 7).all()
    w = torch.full((c.h, c.columns + 5), 2.0, device=dev)
    a = c.on_gpu()
    got = cache_ops.weigh_tokens(a["layer"], c.pf, a["block_table"], a["q"], wl, c.seqs, weights=w[:, 2:-3], scale=c.scale)
    assert (w[:, :2] == 2).all() and (w[:, -3:] == 2).all() and got.data_ptr() == w[:, 2:].data_ptr()
    fresh = cache_ops.weigh_tokens(a["layer"], c.pf, a["block_table"], a["q"], wl, c.seqs, scale=c.scale)
    assert torch.allclose(w[:, 2:-3], fresh + 2, rtol=2e-7, atol=0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.uint8])
def test_strides_and_alignment(dev, dtype):
    """q as a slice of a wider projection, heads transposed, and caches that start
    at odd addresses (other kernels): the same bits as the plain call where the
    rows stay whole units, the same result within the tolerance elsewhere."""
    c = Case(dev, [(2, 100), (30, 20)], dtype=dtype, d=64, seed=13)
    want, wl = c.run()
    q = c.q.to(dev)
    wide = torch.zeros(c.T, 3, *q.shape[1:], dtype=c.qtype, device=dev)
    wide[:, 1] = q
    turned = q.transpose(0, 1).contiguous().transpose(0, 1)
    odd = torch.zeros(q.numel() + 1, dtype=c.qtype, device=dev)[1:].view(q.shape).copy_(q)
    a = c.on_gpu()
    flat = torch.zeros(a["layer"].numel() + 3, dtype=dtype, device=dev)
    shifted = flat[3:].view(a["layer"].shape).copy_(a["layer"])
    for same, more in ((True, dict(q=wide[:, 1])), (True, dict(q=turned)), (False, dict(q=odd)),
                       (False, dict(layer=shifted))):
        out, lse = c.run(**more)
        c.check(out, lse)
        assert not same or (torch.equal(out, want) and torch.equal(lse, wl))
    c.check_weigh(wl)
    w = c.weights
    c.check_weigh(wl, q=wide[:, 1])
    assert torch.equal(w, c.weights)
    c.check_weigh(wl, q=odd, layer=shifted)


def test_many_sequences(dev):
    """More sequences than travel in the kernel arguments, some without rows."""
    rng = np.random.default_rng(14)
    sizes = [(int(n), int(c)) for n, c in zip(rng.integers(0, 3, 200), rng.integers(0, 60, 200))]
    c = Case(dev, sizes, h=1, g=2, d=64, seed=14)
    out, lse = c.run()
    c.check(out, lse)
    c.check_weigh(lse)


def test_sequences_in_any_order(dev):
    c = Case(dev, [(2, 90), (1, 5), (12, 40)], seed=15)
    out, lse = c.run()
    again = c.run(seqs=[c.seqs[2], c.seqs[0], c.seqs[1]])
    assert torch.equal(out, again[0]) and torch.equal(lse, again[1])


def test_shared_pages(dev):
    """Two sequences over the same prefix pages."""
    c = Case(dev, [(1, 64), (1, 64)], seed=16)
    per = -(-65 // 16)
    c.bt[per:per + 4] = c.bt[:4]
    out, lse = c.run()
    c.check(out, lse)


def test_cache_past_32_bits(dev):
    """Pages whose bytes, and whose elements, lie past 2^32 in the layer."""
    ps, h, d = 16, 8, 128
    nb = 140000                                        # 4.27 GiB of K, then V
    layer = torch.empty(2, nb, ps, h, d, dtype=torch.bfloat16, device=dev)
    gen = torch.Generator().manual_seed(17)
    ids = [nb - 1, 5, 131072, 70001, nb - 2, 99999]
    small = torch.randn(2, len(ids) + 1, ps, h, d, generator=gen).to(torch.bfloat16)
    layer[:, ids] = small[:, 1:].to(dev)
    c = Case(dev, [(2, 6 * ps - 2)], h=h, d=d, seed=17)
    c.layer, c.bt = small, np.arange(1, 7, dtype=np.int32)
    bt = torch.tensor(ids, dtype=torch.int32, device=dev)
    out, lse = c.run(layer=layer, block_table=bt)
    c.check(out, lse)
    w = cache_ops.weigh_tokens(layer, False, bt, c.q.to(dev), lse, c.seqs, scale=c.scale)
    c2 = c.on_gpu()
    w2 = cache_ops.weigh_tokens(c2["layer"], False, c2["block_table"], c2["q"], lse, c.seqs, scale=c.scale)
    assert torch.equal(w, w2)
    before = layer[:, ids].cpu()
    wt = torch.rand(1, h, 6 * ps, device=dev)
    ref = wt.cpu().numpy()
    kept = cache_ops.evict_tokens([layer], False, bt, wt, [(0, 0, 6 * ps, 40, 2, 3)])
    ol = torch.cat([before[:, :1], before], 1)
    want = oatt.evict([ol], False, np.arange(1, 7), ref, [(0, 0, 6 * ps, 40, 2, 3)], 40)
    assert np.array_equal(kept.cpu().numpy(), want) and np.array_equal(wt.cpu().numpy(), ref)
    assert same_bytes(layer[:, ids], ol[:, 1:])


# ---------------------------------------------------------------- streams, graphs
def test_other_stream_and_repeats(dev):
    c = Case(dev, [(1, 3000), (60, 700)], d=128, seed=18)
    want, wl = c.run()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    for st in (0, s.cuda_stream, s.cuda_stream):
        out, lse = c.run(stream=st)
        assert torch.equal(out, want) and torch.equal(lse, wl)
    with torch.cuda.stream(s):
        out, lse = c.run()
    assert torch.equal(out, want) and torch.equal(lse, wl)


def test_two_calls_at_once(dev):
    cs = [Case(dev, [(1, 9000 + 500 * i), (40, 900)], d=128, seed=19 + i) for i in range(2)]
    want = [c.run() for c in cs]
    args = [c.on_gpu() for c in cs]
    streams = [torch.cuda.Stream() for _ in cs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(4):
        for i, a in enumerate(args):
            got[i].append(cache_ops.attend_pages(a["layer"], False, a["block_table"], a["q"], a["seqs"],
                                                 scale=a["scale"], stream=streams[i].cuda_stream))
    torch.cuda.synchronize()
    for i in range(2):
        for out, lse in got[i]:
            assert torch.equal(out, want[i][0]) and torch.equal(lse, want[i][1])


def test_captured_loop_replays(dev):
    """attend -> weigh -> evict captured together, replayed with other inputs and
    eager work between; each replay equals the eager calls."""
    c = Case(dev, [(1, 3000), (3, 700)], d=128, h=2, seed=21)
    a = c.on_gpu()
    ev = [(s[0], s[4], s[2] + s[3], (s[2] + s[3]) // 2, 4, 8) for s in c.seqs]
    base = a["layer"].clone()

    def loop(layer, q, w):
        out, lse = cache_ops.attend_pages(layer, c.pf, a["block_table"], q, c.seqs)
        cache_ops.weigh_tokens(layer, c.pf, a["block_table"], q, lse, c.seqs, weights=w)
        return out, lse, cache_ops.evict_tokens([layer], c.pf, a["block_table"], w[None], ev)

    layer, q, w = base.clone(), a["q"].clone(), torch.zeros(c.h, c.columns, device=dev)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        loop(layer, q, w)
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = loop(layer, q, w)
    for rep in range(3):
        nq = torch.randn(c.q.shape, generator=torch.Generator().manual_seed(rep)).to(c.qtype).to(dev)
        l2, w2 = base.clone(), torch.full_like(w, float(rep))
        layer.copy_(base), q.copy_(nq), w.copy_(w2)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = loop(l2, nq, w2)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want)), rep
        assert torch.equal(layer, l2) and torch.equal(w, w2), rep
        _ = float(torch.randn(4096, device=dev).abs().sum())


@pytest.mark.filterwarnings("ignore:The CUDA Graph is empty")
def test_large_calls_refuse_capture(dev):
    c = Case(dev, [(1, 4)] * 100, h=1, g=1, d=64, seed=22)
    c.run()
    g = torch.cuda.CUDAGraph()
    a = c.on_gpu()
    with pytest.raises(RuntimeError, match="cannot be captured in a graph"):
        with torch.cuda.graph(g):
            cache_ops.attend_pages(a["layer"], c.pf, a["block_table"], a["q"], c.seqs)
    torch.cuda.synchronize()
    out, lse = c.run()
    c.check(out, lse)


# ------------------------------------------------------------------------ evict
@pytest.mark.parametrize("layout", ["nhd", "hnd", "pf", "packed", "mla", "nhd_pad"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.uint8, torch.float32])
@pytest.mark.parametrize("shared", [False, True])
def test_eviction(dev, layout, dtype, shared):
    g = torch.Generator().manual_seed(30)
    L, ps, h, d = 3, 16, 1 if layout == "mla" else 4, 40
    sizes = [(100, 50, 4, 10), (37, 37, 0, 5), (64, 1, 0, 0), (257, 256, 0, 0), (300, 7, 3, 4), (20, 30, 10, 10),
             (90, 0, 0, 0), (0, 0, 0, 0), (129, 100, 100, 0), (129, 100, 0, 100), (513, 200, 0, 1)]
    layers = [make_layer(layout, 130, ps, h, d, dtype, g, kind="bytes") for _ in range(L)]
    pf, layers = layers[0][1], [t for t, _ in layers]
    ids = np.random.default_rng(0).permutation(np.arange(1, 130)).astype(np.int32)
    ev, at, col = [], 0, 3
    for n, keep, first, recent in sizes:
        ev.append((at, col, n, keep, first, recent))
        at, col = at + -(-n // ps), col + n + 2
    ids[ev[4][0] + 3] = 0
    ids[ev[4][0] + 0] = 500
    w = torch.randn(L, 1 if shared else h, col, generator=g).round(decimals=1)      # many ties
    w[0, 0, 20:40] = float("nan")
    w[1, 0, ev[10][1]:ev[10][1] + 513] = 0.0
    w[1, 0, ev[10][1] + 5] = -0.0
    w[2, 0, ev[10][1]:ev[10][1] + 400] = float("inf")
    gl = [to_dev(t, dev) for t in layers]
    gw = w.to(dev)
    kept = cache_ops.evict_tokens(gl, pf, torch.from_numpy(ids).to(dev), gw, ev)
    torch.cuda.synchronize()
    wn = w.numpy().copy()
    want = oatt.evict(layers, pf, ids, wn, ev, kept.shape[3])
    np.testing.assert_array_equal(kept.cpu().numpy(), want)
    np.testing.assert_array_equal(gw.cpu().numpy().view(np.uint32), wn.view(np.uint32))
    for a, b in zip(gl, layers):
        assert same_bytes(a, b)


@pytest.mark.parametrize("n", [255, 256, 257, 2047, 2048, 2049, 8191, 8193, 40000])
@pytest.mark.parametrize("frac", [0.01, 0.5, 0.97])
def test_eviction_lengths(dev, n, frac):
    g = torch.Generator().manual_seed(n)
    layer, pf = make_layer("nhd", -(-n // 16) + 1, 16, 2, 8, torch.float16, g, kind="bytes")
    bt = np.random.default_rng(n).permutation(np.arange(1, layer.shape[1])).astype(np.int32)
    w = torch.rand(1, 2, n, generator=g)
    w[0, 1] = torch.linspace(1, 0, n)                   # the head of the sequence is the heaviest: nothing moves,
    if frac == 0.5:
        w[0, 1] = torch.linspace(0, 1, n)               # or its tail: everything does, from one long gap
    ev = [(0, 0, n, max(1, int(n * frac)), 1, 0)]
    gl, gw = to_dev(layer, dev), w.to(dev)
    kept = cache_ops.evict_tokens([gl], pf, torch.from_numpy(bt).to(dev), gw, ev)
    torch.cuda.synchronize()
    wn = w.numpy().copy()
    want = oatt.evict([layer], pf, bt, wn, ev, kept.shape[3])
    np.testing.assert_array_equal(kept.cpu().numpy(), want)
    np.testing.assert_array_equal(gw.cpu().numpy(), wn)
    assert same_bytes(gl, layer)


def test_eviction_many(dev):
    """More sequences and layers than travel in the kernel arguments."""
    g = torch.Generator().manual_seed(33)
    layers = [make_layer("nhd", 301, 8, 1, 16, torch.bfloat16, g)[0] for _ in range(9)]
    ev = [(i * 3, i * 24, 20 + i % 5, 9, 1, 2) for i in range(100)]
    bt = np.random.default_rng(3).permutation(np.arange(1, 301)).astype(np.int32)
    w = torch.rand(9, 1, 2400, generator=g)
    gl, gw = [to_dev(t, dev) for t in layers], w.to(dev)
    kept = cache_ops.evict_tokens(gl, False, torch.from_numpy(bt).to(dev), gw, ev)
    wn = w.numpy().copy()
    want = oatt.evict(layers, False, bt, wn, ev, 9)
    np.testing.assert_array_equal(kept.cpu().numpy(), want)
    np.testing.assert_array_equal(gw.cpu().numpy(), wn)
    assert all(same_bytes(a, b) for a, b in zip(gl, layers))


# --------------------------------------------------------------------- together
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.uint8])
def test_serving_loop(dev, dtype):
    """Decoding under a budget: each step attends, adds the weights, and evicts down
    to the budget; against the same loop in 64 bits fed with the GPU's lse and
    kept choices (the weights' last bits decide ties the oracle cannot know)."""
    c = Case(dev, [(1, 90), (1, 61)], dtype=dtype, d=64, h=2, seed=40, spare=0)
    budget, steps, H = 64, 5, 2
    # room for the tokens to come: two more pages a sequence
    ps, nb = 16, c.layer.shape[1]
    grown, _ = make_layer("nhd", nb + 4, ps, H, 64, dtype, torch.Generator().manual_seed(41))
    grown[:, :nb] = c.layer
    p0 = c.seqs[1][0]
    bt = np.concatenate([c.bt[:p0], [nb, nb + 1], c.bt[p0:], [nb + 2, nb + 3]]).astype(np.int32)
    starts, lens = [0, p0 + 2], [91, 62]
    cpu, gpu, btd = grown.clone(), to_dev(grown, dev), torch.from_numpy(bt).to(dev)
    cols, wd = [0, 200], torch.zeros(1, H, 400, device=dev)
    ks = c.ks.to(dev) if c.ks is not None else None
    vs = c.vs.to(dev) if c.vs is not None else None
    for step in range(steps):
        q = torch.randn(2, c.q.shape[1], 64, generator=torch.Generator().manual_seed(step)).to(c.qtype)
        seqs = [(starts[i], i, 1, lens[i] - 1, cols[i]) for i in range(2)]
        out, lse = cache_ops.attend_pages(gpu, False, btd, q.to(dev), seqs, k_scale=ks, v_scale=vs)
        c.layer, c.bt, c.seqs, c.q, c.mask, c.T, c.scale = cpu, bt, seqs, q, None, 2, 64 ** -0.5
        c.check(out, lse)
        before = wd[0].cpu()
        cache_ops.weigh_tokens(gpu, False, btd, q.to(dev), lse, seqs, weights=wd[0], k_scale=ks)
        ref, size, amax, rows = oatt.weigh(cpu, False, bt, q, lse.cpu(), seqs, before.double().numpy(), None,
                                           64 ** -0.5, c.ks)
        tol = (ref - before.double().numpy()) * (74 * E * amax + 24 * E + 4 * E * size + rows * E) + 2 * E * ref + 1e-37
        assert (np.abs(wd[0].double().cpu().numpy() - ref) <= tol).all()
        ev = [(starts[i], cols[i], lens[i], budget, 2, 8) for i in range(2)]
        wn = wd.cpu().numpy().copy()
        kept = cache_ops.evict_tokens([gpu], False, btd, wd, ev)
        want = oatt.evict([cpu], False, bt, wn, ev, kept.shape[3])
        np.testing.assert_array_equal(kept.cpu().numpy(), want)
        np.testing.assert_array_equal(wd.cpu().numpy(), wn)
        assert same_bytes(gpu, cpu)
        # the next token's K and V stand behind what stayed
        for i in range(2):
            lens[i] = min(lens[i], budget) + 1
            j = lens[i] - 1
            row = make_layer("nhd", 1, 1, H, 64, dtype, torch.Generator().manual_seed(100 + step))[0]
            cpu[:, int(bt[starts[i] + j // ps]), j % ps] = row[:, 0, 0]
            gpu[:, int(bt[starts[i] + j // ps]), j % ps] = row[:, 0, 0].to(dev)


def test_nothing_to_do(dev):
    """No rows, no kept tokens, no sequences, a q without rows."""
    c = Case(dev, [(2, 30)], seed=51)
    a = c.on_gpu()
    out, lse = cache_ops.attend_pages(a["layer"], False, a["block_table"], a["q"][:0], [])
    assert out.shape == (0, 8, 64) and lse.shape == (0, 8)
    w = cache_ops.weigh_tokens(a["layer"], False, a["block_table"], a["q"], torch.zeros(2, 8, device=dev), [(0, 0, 0, 30, 4)])
    assert w.shape == (2, 34) and (w == 0).all()
    assert cache_ops.weigh_tokens(a["layer"], False, a["block_table"], a["q"], torch.zeros(2, 8, device=dev), []).shape == (2, 0)
    before = a["layer"].clone()
    w = torch.rand(1, 2, 32, device=dev)
    kept = cache_ops.evict_tokens([a["layer"]], False, a["block_table"], w, [(0, 1, 30, 0, 0, 0)])
    assert kept.shape == (1, 2, 1, 0) and (w[:, :, 1:31] == 0).all() and (w[:, :, [0, 31]] > 0).all()
    assert torch.equal(before, a["layer"])
    assert cache_ops.evict_tokens([a["layer"]], False, a["block_table"], w, []).shape == (1, 2, 0, 0)


@pytest.mark.filterwarnings("ignore:The CUDA Graph is empty")
def test_mixed_large_call_refuses_capture_whole(dev):
    """Few sequences of many rows beside more of one row than a capture allows: no
    part of the call is enqueued."""
    c = Case(dev, [(20, 4)] + [(1, 4)] * 100, h=1, g=1, d=64, seed=52)
    out, lse = c.run()
    c.check(out, lse)
    a = c.on_gpu()
    out.fill_(3.0)
    g = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="cannot be captured in a graph"):
        with torch.cuda.graph(g):
            cache_ops.attend_pages(a["layer"], c.pf, a["block_table"], a["q"], c.seqs, out=out, lse=lse)
    torch.cuda.synchronize()
    assert (out == 3.0).all()


def test_refusals_on_the_gpu(dev):
    c = Case(dev, [(2, 30)], seed=50)
    a = c.on_gpu()
    call = lambda **k: c.run(**k)
    with pytest.raises(ValueError, match="sequences must be"):
        call(seqs=[(0, 0, 1)])
    with pytest.raises(RuntimeError, match="block_table must be on"):
        call(block_table=a["block_table"].cpu())
    with pytest.raises(RuntimeError, match="rows exceed q"):
        call(seqs=[(0, 0, 3, 10)])
    with pytest.raises(RuntimeError, match="reads past the end of block_table"):
        call(seqs=[(0, 0, 2, 47)])
    with pytest.raises(RuntimeError, match="multiple of the cache's 2 heads"):
        cache_ops.weigh_tokens(a["layer"], False, a["block_table"], a["q"][:, 0], a["q"][:, 0].float(), c.seqs)
    with pytest.raises(ValueError, match="MLA"):
        cache_ops.attend_pages(torch.zeros(4, 16, 64, dtype=torch.bfloat16, device=dev), True, a["block_table"], a["q"],
                               c.seqs)
    with pytest.raises(RuntimeError, match="weights must be"):
        cache_ops.evict_tokens([a["layer"]], False, a["block_table"], torch.zeros(1, 5, 32, device=dev),
                               [(0, 0, 32, 5, 0, 0)])
    assert cache_ops.attend_pages(a["layer"], False, a["block_table"], a["q"], [])[0].shape == a["q"].shape
