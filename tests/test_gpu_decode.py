"""GPU parity of rotate_rows, append_tokens, select_beams and reorder_beams against
their definitions in 64 bits (oracle/decode.py), and a beam search of all of them
with attend_pages.

Tolerances. A rotated value's fp32 arithmetic may be off by the oracle's bound
(oracle.decode.rotate: a few 2^-24 of the pair's size); its rounding by half a step of
the type it is stored in, u = finfo(t).eps / 2 relative, and by half a subnormal
step (fp16 2^-25, e4m3 2^-10; bf16 and fp32 far below). A copied value is exact. An e4m3 code
is within half a step, 2^-4 relative, of the quotient, whose own rounding is 2^-24. A score of a
candidate is rounded to fp32 once, 2^-24 of it, and its row's log-sum is off by at
most (V / 8192 + 48) 2^-24: 8192 fp32 terms of a split summed 32 to a chain and then
as a tree (40 roundings), each exponential off by 2^-23 and the rounding of its
argument, whose weight |x| exp(x) is below 1; tokens and parents are equal where the
data keep candidates apart, which the seeds here do (asserted on the oracle's scores)."""
import numpy as np
import pytest
import torch

from daric_amd import cache_ops
from oracle import decode as odec
from oracle import fp8 as ofp8
from oracle import rope as orope
from oracle.attend import _f64
from oracle.select import k_rows_view, v_view
from tests.gpu_util import make_layer, same_bytes, to_dev

pytestmark = pytest.mark.gpu
E = 2.0 ** -24
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: E}
SUB = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}


def close(got, want, off, dtype):
    got, tol = got.double().cpu().numpy(), U[dtype] * np.abs(want) + off * (1 + U[dtype]) + SUB[dtype] * (off > 0)
    tol = np.where(off > 0, tol, 0)
    bad = np.abs(got - want) > tol
    assert not bad.any(), f"{bad.sum()} of {bad.size} off, by up to {np.max(np.abs(got - want)[bad] / np.maximum(tol[bad], 1e-300)):.2f} of the tolerance"


# ------------------------------------------------------------------- rotation
FAR = np.array([0, 1, 2, 777, 4095, 131071, 1048575, -1, -4096, 2 ** 24 + 1, 2 ** 31 - 5], np.int64)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("heads,dim,rotary,neox", [(40, 128, 128, True), (1, 64, 64, False), (5, 80, 32, False), (3, 80, 20, True),
                                                   (7, 6, 6, True), (2, 10, 2, False), (2, 9, 6, False), (1, 512, 512, True), (3, 100, 36, True)])
def test_rotate(dev, dtype, heads, dim, rotary, neox):
    g = torch.Generator().manual_seed(heads * dim)
    x = torch.randn(len(FAR), heads, dim, generator=g).to(dtype)
    f = orope.default_inv_freq(rotary, 10000.0)
    want, off = odec.rotate(x, FAR, f, rotary, neox, 1.0)
    xd, pos, fd = x.to(dev), torch.from_numpy(FAR).to(dev), torch.from_numpy(np.asarray(f)).to(dev)
    out = cache_ops.rotate_rows(xd, pos, fd, rotary, neox)
    torch.cuda.synchronize()
    assert same_bytes(xd, x) and out.is_contiguous()
    close(out, want, off, dtype)
    assert same_bytes(out[..., rotary:], x[..., rotary:])
    again = cache_ops.rotate_rows(xd, pos, fd, rotary, neox, out=xd)
    torch.cuda.synchronize()
    assert again is xd and same_bytes(xd, out)


@pytest.mark.parametrize("rows", [1, 2, 3, 257, 1023, 2049, 4100, 9001])
def test_rotate_many_rows(dev, rows):
    """Tiles of one to eight rows, the last of them short; a table's scale."""
    g = torch.Generator().manual_seed(rows)
    for dim in (64, 128):
        x = torch.randn(rows, 2, dim, generator=g).to(torch.bfloat16)
        pos = torch.randint(0, 10 ** 6, (rows,), generator=g)
        f = orope.default_inv_freq(dim, 500000.0)
        want, off = odec.rotate(x, pos.numpy(), f, dim, True, 1.2)
        out = cache_ops.rotate_rows(x.to(dev), pos.to(dev), torch.from_numpy(np.asarray(f)).to(dev), dim, attention_scale=1.2)
        close(out, want, off, torch.bfloat16)


@pytest.mark.parametrize("pad,first", [(0, 0), (8, 8), (4, 4), (2, 2), (1, 1), (3, 0)])
def test_rotate_strided_and_misaligned(dev, pad, first):
    """Heads of a joint projection at every alignment, in place: what is beside them stays."""
    g = torch.Generator().manual_seed(5)
    joint = torch.randn(33, 6 * 64 + pad + first, generator=g).to(torch.float16).to(dev)
    before = joint.clone()
    x = joint[:, first: first + 4 * 64].view(33, 4, 64)
    pos = torch.arange(33, device=dev) * 1000
    f = torch.from_numpy(np.asarray(orope.default_inv_freq(64, 10000.0))).to(dev)
    want, off = odec.rotate(x.cpu(), pos.cpu().numpy(), f.cpu().numpy(), 64)
    apart = cache_ops.rotate_rows(x, pos, f, 64)
    close(apart, want, off, torch.float16)
    assert torch.equal(joint, before)
    cache_ops.rotate_rows(x, pos, f, 64, out=x)
    torch.cuda.synchronize()
    assert torch.equal(x, apart)
    assert torch.equal(joint[:, :first], before[:, :first]) and torch.equal(joint[:, first + 256:], before[:, first + 256:])
    # broadcast rows into a tensor of their own
    one = joint[:1, first: first + 256].view(1, 4, 64).expand(33, 4, 64)
    got = cache_ops.rotate_rows(one, pos, f, 64)
    close(got, *odec.rotate(one.cpu(), pos.cpu().numpy(), f.cpu().numpy(), 64), torch.float16)


def test_rotation_by_the_negative_position_is_the_gradient(dev):
    """<rotate(x, p), y> = <x, rotate(y, -p)>, and both agree with differences."""
    g = torch.Generator().manual_seed(9)
    x, y, d = (torch.randn(6, 2, 32, generator=g) for _ in range(3))
    pos = torch.tensor([0, 5, 100, 9999, 1048575, 3])
    f = torch.from_numpy(np.asarray(orope.default_inv_freq(16, 10000.0)))
    for neox in (True, False):
        r = lambda t, p: cache_ops.rotate_rows(t.to(dev), p.to(dev), f.to(dev), 16, neox, attention_scale=1.5).double().cpu()
        grad = r(y, -pos)
        # values of the call are off by at most 8 e of the pair's size (the oracle's 6 e and a rounding)
        size = (x.abs().double().sum() * y.abs().double().max() + x.abs().double().max() * y.abs().double().sum()) * 1.5 * 2
        assert abs(float((r(x, pos) * y.double()).sum() - (x.double() * grad).sum())) <= 8 * E * float(size)
        step = (r(x + d, pos) - r(x, pos)).mul(y.double()).sum()
        moved = ((x + d).double() - x.double())
        size = size + ((x + d).abs().double().sum() * y.abs().double().max()) * 3
        assert abs(float(step - (moved * grad).sum())) <= 8 * E * float(size)


# --------------------------------------------------------------------- append
class Step:
    """Rows of sequences (n_rows, n_ctx) over one layer of random pages, in a joint
    projection; `lost` pages of every sequence are the null page or no page."""

    def __init__(self, sizes, layout="nhd", dtype=torch.bfloat16, qtype=None, ps=16, h=2, g=3, d=64, rotary=None, neox=True,
                 seed=0, scales=True, gap=0, lost=False, m=1.0):
        gen = torch.Generator().manual_seed(seed)
        rng = np.random.default_rng(seed)
        self.pages = [-(-(n + c) // ps) for n, c in sizes]
        nb = sum(self.pages) + 4
        self.layer, self.pf = make_layer(layout, nb, ps, h, d, dtype, gen)
        if layout == "mla":
            h, d = 1, self.layer.shape[2]
        self.bt = rng.permutation(np.arange(1, nb))[:max(1, sum(self.pages))].astype(np.int32)
        self.seqs, at, row = [], 0, gap
        for (n, c), p in zip(sizes, self.pages):
            self.seqs.append((at, row, n, c))
            if lost and p > 1:
                self.bt[at + p // 2] = rng.choice([0, -3, nb])
            at, row = at + p, row + n + gap
        self.T = row
        self.qtype = qtype or (dtype if dtype != torch.uint8 else torch.bfloat16)
        joint = torch.randn(self.T, (g + 2) * h, d, generator=gen).to(self.qtype)
        self.joint, self.h, self.g, self.d = joint, h, g, d
        self.R = d if rotary is None else rotary
        self.rope = (orope.default_inv_freq(self.R, 10000.0), self.R, neox, m) if self.R else None
        self.mla = layout == "mla"
        self.ks = self.vs = None
        if dtype == torch.uint8 and scales:
            self.ks = rng.uniform(0.01, 0.3, h).astype(np.float32)
            self.vs = rng.uniform(0.001, 0.3, h).astype(np.float32)

    def parts(self, joint):
        a, b = self.g * self.h, (self.g + 1) * self.h
        return joint[:, :a], joint[:, a:b], None if self.mla else joint[:, b:]

    def run(self, dev, positions=None, in_place=False, layer=None, with_q=True, stream=0):
        joint = self.joint.to(dev)
        q, k, v = self.parts(joint)
        layer = to_dev(self.layer, dev) if layer is None else layer
        more = {}
        if self.rope:
            more = dict(inv_freq=torch.from_numpy(np.asarray(self.rope[0])).to(dev), rotary_dim=self.R, is_neox_style=self.rope[2],
                        attention_scale=self.rope[3])
            if with_q:
                more.update(q=q, q_out=q if in_place else torch.full(q.shape, 7.0, dtype=q.dtype, device=dev))
        s = lambda x: None if x is None else torch.from_numpy(x).to(dev)
        torch.cuda.synchronize()
        out = cache_ops.append_tokens(layer, self.pf, torch.from_numpy(self.bt).to(dev), k, v, self.seqs, k_scale=s(self.ks),
                                      v_scale=s(self.vs), positions=None if positions is None else positions.to(dev),
                                      stream=stream, **more)
        torch.cuda.synchronize()
        return out, layer, joint

    def check(self, out, layer, positions=None):
        q, k, v = self.parts(self.joint)
        where, pos, kk, vv, off = odec.append(self.layer, self.pf, self.bt, k, v, self.seqs, positions, self.rope, self.ks, self.vs)
        got = layer.cpu()
        fp8 = self.layer.dtype == torch.uint8
        want = self.layer.clone()
        for row, page, slot in where:
            # what was written is compared here and put into the expectation, so that the rest must be as it was
            for view, x, err in ((k_rows_view, kk, off),) + (() if self.mla else ((v_view, vv, np.zeros_like(vv)),)):
                cell = view(got, self.pf)[page, slot]
                if fp8:
                    code, ref = _f64(cell), x[row]
                    ref = np.clip(ref, -448, 448)
                    tol = 2.0 ** -4 * np.abs(ref) + 2.0 ** -10 + (err[row] + E * np.abs(ref)) * 1.0625
                    assert (np.abs(code - ref) <= tol).all()
                else:
                    close(cell[None], x[row][None], err[row][None], self.qtype)
                view(want, self.pf)[page, slot] = cell
        assert same_bytes(got, want)
        if out is not None:
            mine = np.zeros(self.T, bool)
            for _, r0, n, _ in self.seqs:
                mine[r0: r0 + n] = True
            qq, qoff = odec.rotate(q, pos, *self.rope)
            close(out[torch.from_numpy(mine).to(out.device)], qq[mine], qoff[mine], self.qtype)
            return mine


LAYOUTS = ["nhd", "hnd", "pf", "pf_hnd", "packed", "nhd_pad"]


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("dtype,qtype", [(torch.bfloat16, None), (torch.float16, None), (torch.uint8, torch.bfloat16), (torch.uint8, torch.float16)])
def test_append_layouts(dev, layout, dtype, qtype):
    s = Step([(1, 0), (5, 3), (0, 7), (40, 30), (1, 15), (17, 16)], layout, dtype, qtype, gap=2)
    out, layer, joint = s.run(dev)
    mine = s.check(out, layer)
    assert (out[torch.from_numpy(~mine).to(dev)] == 7).all()
    assert same_bytes(joint, s.joint)


@pytest.mark.parametrize("d,rotary,neox,ps", [(80, 32, False, 32), (80, 20, True, 8), (6, 6, True, 4), (10, 2, False, 1), (9, 4, True, 3),
                                              (256, 128, True, 64), (128, 128, True, 16), (12, 0, True, 16), (36, 12, False, 5)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.uint8])
def test_append_sizes(dev, dtype, d, rotary, neox, ps):
    s = Step([(3, 0), (1, 63), (70, 1)], "hnd" if d % 4 == 0 else "nhd", dtype, ps=ps, d=d, rotary=rotary, neox=neox, lost=True, m=1.3)
    out, layer, _ = s.run(dev)
    s.check(out, layer)


@pytest.mark.parametrize("sizes", [[(1, 0)], [(1, c) for c in range(100)], [(1, c % 40) for c in range(700)], [(5000, 3)],
                                   [(2100, 0), (1, 5), (0, 3), (4000, 70)], [(8, 0)] * 300, [(2000, 0), (2500, 17), (1, 0)] * 2])
def test_append_forms(dev, sizes):
    """One tile a sequence and many, found by place or by search; descriptors in the
    arguments, in the pinned slot and uploaded; tiles of one to eight rows."""
    s = Step(sizes, h=1, g=1, d=64, ps=16)
    out, layer, _ = s.run(dev)
    s.check(out, layer)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.uint8])
def test_append_mla(dev, dtype):
    s = Step([(3, 5), (1, 0), (33, 1)], "mla", dtype, h=1, d=96, rotary=32, g=2)
    out, layer, _ = s.run(dev)
    s.check(out, layer)


def test_append_in_place_and_positions(dev):
    s = Step([(7, 20), (1, 3)], gap=1, lost=True)
    pos = torch.randint(-100, 2 ** 20, (s.T,), generator=torch.Generator().manual_seed(3))
    out, layer, _ = s.run(dev, positions=pos)
    mine = s.check(out, layer, pos.numpy())
    again, layer2, joint = s.run(dev, positions=pos, in_place=True)
    sel = torch.from_numpy(mine).to(dev)
    assert torch.equal(again[sel], out[sel]) and same_bytes(layer, layer2)
    want = s.joint.clone().to(dev)
    want[sel, : s.g * s.h] = out[sel]
    assert torch.equal(joint, want)
    # without q the cache is the same
    _, layer3, joint = s.run(dev, positions=pos, with_q=False)
    assert same_bytes(layer, layer3) and same_bytes(joint, s.joint)


def test_append_values_at_the_ends(dev):
    """Saturation, infinities and NaN into e4m3; rows are copied bit by bit into their own type."""
    s = Step([(4, 0)], dtype=torch.uint8, rotary=0, d=16, h=2, g=1)
    k = s.parts(s.joint)[1]
    k[0, 0] = torch.tensor([1e30, -1e30, float("inf"), -float("inf"), float("nan"), 0.0, -0.0, 1e-30] * 2)
    k[1, 1, :4] = torch.tensor([448.0, 464.0, 2.0 ** -10, 3 * 2.0 ** -10]) * float(s.ks[1])
    _, layer, _ = s.run(dev)
    with np.errstate(all="ignore"):
        want = ofp8.encode((k.float().numpy() / s.ks[None, :, None]).astype(np.float32))
    got = k_rows_view(layer.cpu(), s.pf)[int(s.bt[0]), :4].numpy()
    nan = np.isnan(k.float().numpy())
    assert (got[~nan] == want[~nan]).all() and ((got[nan] & 127) == 127).all()
    s = Step([(4, 0)], dtype=torch.bfloat16, rotary=0, d=16, h=2, g=1)
    s.joint.view(torch.int16).random_(generator=torch.Generator().manual_seed(1))
    _, layer, _ = s.run(dev)
    q, k, v = s.parts(s.joint)
    assert torch.equal(layer.cpu()[0, int(s.bt[0]), :4].view(torch.int16), k.contiguous().view(torch.int16))
    assert torch.equal(layer.cpu()[1, int(s.bt[0]), :4].view(torch.int16), v.contiguous().view(torch.int16))


def test_append_on_another_stream_and_twice_at_once(dev):
    a, b = Step([(1, 5)] * 40, seed=1), Step([(600, 0)], seed=2)
    la, lb = to_dev(a.layer, dev), to_dev(b.layer, dev)
    sa, sb = torch.cuda.Stream(), torch.cuda.Stream()
    oa, _, _ = a.run(dev, layer=la, stream=sa.cuda_stream)
    a.check(oa, la)
    f = torch.from_numpy(np.asarray(a.rope[0])).to(dev)
    args = []
    for s, lay in ((a, la), (b, lb)):
        q, k, v = s.parts(s.joint.to(dev))
        args.append((lay, s.pf, torch.from_numpy(s.bt).to(dev), k, v, s.seqs, f, s.R, True, q))
    torch.cuda.synchronize()
    outs = []
    for _ in range(3):
        for st, x in ((sa, args[0]), (sb, args[1])):
            outs.append(cache_ops.append_tokens(*x[:-1], q=x[-1], stream=st.cuda_stream))
    torch.cuda.synchronize()
    for i, o in enumerate(outs):
        (a, b)[i % 2].check(o, (la, lb)[i % 2])


def test_append_at_once_each_to_a_cache_of_its_own(dev):
    """Calls on two streams, each with other rows and another cache: what any of them did not
    write, or wrote elsewhere, is seen."""
    steps = [Step([(1, 5 + i)] * 40 if i % 2 == 0 else [(600, i)], seed=10 + i) for i in range(6)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    f = torch.from_numpy(np.asarray(steps[0].rope[0])).to(dev)
    layers, args = [to_dev(s.layer, dev) for s in steps], []
    for s, layer in zip(steps, layers):
        q, k, v = s.parts(s.joint.to(dev))
        args.append((layer, s.pf, torch.from_numpy(s.bt).to(dev), k, v, s.seqs, f, s.R, True, q))
    torch.cuda.synchronize()
    outs = [cache_ops.append_tokens(*x[:-1], q=x[-1], stream=streams[i % 2].cuda_stream) for i, x in enumerate(args)]
    torch.cuda.synchronize()
    for s, out, layer in zip(steps, outs, layers):
        assert not same_bytes(layer, s.layer)
        s.check(out, layer)


def test_append_mla_rows_that_are_rotated_at_their_end(dev):
    """Rows whose rotated part stands last: turned in place by rotate_rows, then appended as they are."""
    s = Step([(3, 5), (1, 0), (33, 1)], "mla", torch.bfloat16, rotary=0, d=96, g=2)
    R, pos = 32, torch.cat([torch.arange(c, c + n) for n, c in ((3, 5), (1, 0), (33, 1))])
    f = orope.default_inv_freq(R, 10000.0)
    joint = s.joint.to(dev)
    k = s.parts(joint)[1]
    end = k[..., -R:]
    cache_ops.rotate_rows(end, pos.to(dev), torch.from_numpy(np.asarray(f)).to(dev), R, out=end)
    want, off = odec.rotate(s.parts(s.joint)[1][..., -R:], pos.numpy(), f, R)
    close(end, want, off, torch.bfloat16)
    layer = to_dev(s.layer, dev)
    cache_ops.append_tokens(layer, s.pf, torch.from_numpy(s.bt).to(dev), k, None, s.seqs)
    torch.cuda.synchronize()
    before = s.joint.clone()
    s.parts(before)[1][..., -R:] = end.cpu()
    assert same_bytes(joint, before)
    s.joint = before
    s.check(None, layer)


# ------------------------------------------------------------------ selection
def select_case(B, W, V, dtype, seed=0, likely=8):
    g = torch.Generator().manual_seed(seed)
    x = 2 * torch.randn(B, W, V, generator=g)
    x.view(B * W, V).scatter_add_(1, torch.randint(0, V, (B * W, likely), generator=g), 6 + torch.randn(B * W, likely, generator=g))
    return x.to(dtype), (-5 - 3 * torch.rand(B, W, generator=g)).float()


def check_select(got, x, scores, k, ended=None, end_token=-1):
    want = odec.select(x, scores.numpy(), k, None if ended is None else ended.numpy(), end_token)
    V = x.shape[2]
    s, p, t = (v.cpu().numpy() for v in got)
    live = np.isfinite(want[0])
    assert (s[want[0] == np.inf] == np.inf).all()
    with np.errstate(all="ignore"):
        tol = 2 * E * np.abs(want[0]) + (V / 8192 + 48) * E
        # candidates of different beams are further apart than their scores may be off
        apart = np.abs(np.diff(want[0], axis=1))
        close_by = live[:, 1:] & (want[1][:, 1:] != want[1][:, :-1]) & (apart < 2 * tol[:, 1:]) & (apart > 0)
    assert not close_by.any(), "the case's candidates are too close for a comparison"
    assert (p == want[1]).all() and (t == want[2]).all()
    assert (np.abs(s[live] - want[0][live]) <= tol[live]).all() and (s[want[0] == -np.inf] == -np.inf).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,W,V,k", [(1, 4, 32000, 8), (1, 1, 1, 1), (2, 3, 5, 9), (3, 5, 2048, 10), (1, 2, 2049, 4), (7, 4, 8191, 8),
                                     (1, 1, 8193, 64), (2, 32, 1000, 64), (1, 64, 300, 64), (40, 8, 20011, 16), (1, 3, 128000, 33)])
def test_select(dev, dtype, B, W, V, k):
    x, s = select_case(B, W, V, dtype, seed=B * V + k)
    got = cache_ops.select_beams(x.to(dev), s.to(dev), k)
    torch.cuda.synchronize()
    check_select(got, x, s, k)


def test_select_the_largest_vocabulary(dev):
    """As many pieces of rows as a request may have: 64 beams of 2^20 fp32 logits."""
    W, V, k = 64, 2 ** 20, 64
    g = torch.Generator().manual_seed(9)
    x = torch.randn(1, W, V, generator=g)
    s = -torch.rand(1, W, generator=g)
    got = cache_ops.select_beams(x.to(dev), s.to(dev), k)
    torch.cuda.synchronize()
    total = s.double()[0, :, None] + torch.log_softmax(x[0].double(), 1)
    best, at = total.flatten().topk(k)
    sc, par, tok = (v.cpu()[0] for v in got)
    tol = 2 * E * best.abs() + (V / 8192 + 48) * E
    assert (best[:-1] - best[1:] > 2 * tol[1:]).all(), "the case's candidates are too close for a comparison"
    assert (par.long() == at // V).all() and (tok.long() == at % V).all()
    assert ((sc.double() - best).abs() <= tol).all()


def test_select_defaults_and_repeats(dev):
    x, s = select_case(3, 4, 5000, torch.bfloat16, 3)
    a = cache_ops.select_beams(x.to(dev), s.to(dev))
    assert a[0].shape == (3, 4)
    check_select(a, x, s, 4)
    for _ in range(3):
        assert all(torch.equal(u, v) for u, v in zip(a, cache_ops.select_beams(x.to(dev), s.to(dev))))
    none = cache_ops.select_beams(torch.empty(0, 4, 10, device=dev), torch.empty(0, 4, device=dev), 3)
    assert none[0].shape == (0, 3)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [7, 700, 9000, 70000])
def test_select_ties(dev, dtype, V):
    """All logits alike, in one beam and in all; two values; equal beams."""
    for W, k in ((1, 5), (4, 9), (8, 64), (64, 64)):
        x = torch.full((2, W, V), -0.5, dtype=dtype)
        x[1, :, ::3] = 1.5
        s = torch.zeros(2, W)
        check_select(cache_ops.select_beams(x.to(dev), s.to(dev), k), x, s, k)
    row = torch.randn(1, 1, V, generator=torch.Generator().manual_seed(1)).to(dtype)
    x, s = row.expand(3, 6, V).contiguous(), torch.full((3, 6), -2.0)
    check_select(cache_ops.select_beams(x.to(dev), s.to(dev), 20), x, s, 20)
    x = torch.zeros(1, 1, V, dtype=dtype)
    x[0, 0, 1::2] = -0.0                                     # equal values
    check_select(cache_ops.select_beams(x.to(dev), torch.zeros(1, 1, device=dev), 6), x, torch.zeros(1, 1), 6)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("V,spread", [(4096, 0.0), (4096, 8.0), (128000, 2.0), (128000, 0.01), (2 ** 20, 4.0)])
def test_select_scores_within_the_sums_roundings(dev, dtype, V, spread):
    """A row's log-sum is off by its splits' alone, which are joined in 64 bits. A split of 4096
    values (2048 of fp32) is summed in chains of 16 (8) to a lane and 8 more steps of a tree: 24 e at
    most. A term is off by 2 e of the exponential, e |d| of its argument's rounding and e |d| of the
    difference d to the maximum itself; weighted by the terms |d| is 5.6 at most (one value at 0, the
    others at -t: t - 1 where t - 1 = 4095 exp(-t)). In all 38 e, and e of the score for its rounding."""
    g = torch.Generator().manual_seed(V)
    x = (spread * torch.randn(2, 2, V, generator=g)).to(dtype)
    s = torch.tensor([[-1.5, -torch.inf], [-torch.inf, -3.0]])
    got = cache_ops.select_beams(x.to(dev), s.to(dev), 4)[0].double().cpu().numpy()
    want = odec.select(x, s.numpy(), 4)[0]
    assert (np.abs(got - want) <= E * np.abs(want) + 38 * E).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("V", [600, 20000])
def test_select_best_in_few_lanes(dev, dtype, V):
    """A run of neighbouring likely tokens, more than a wavefront ranks at once."""
    g = torch.Generator().manual_seed(V)
    x = torch.randn(2, 2, V, generator=g)
    x[0, 0, 100: 600] += 20 + torch.arange(500) * 0.125
    x[1, 1, V - 70:] += torch.linspace(30, 20, 70)
    x = x.to(dtype)
    s = torch.tensor([[-1.0, -2.0], [-3.0, -1.5]])
    for k in (1, 4, 64):
        check_select(cache_ops.select_beams(x.to(dev), s.to(dev), k), x, s, k)


def test_select_masks_and_numbers(dev):
    """-inf and the type's lowest value in masked places, rows of nothing, infinities and NaN."""
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        x, s = select_case(6, 3, 9000, dtype, 5)
        lowest = torch.finfo(dtype).min
        x[0, :, 10:] = -torch.inf                 # ten tokens left
        x[1, 1] = -torch.inf                      # a beam whose mask leaves nothing
        x[2] = -torch.inf                         # none at all
        x[3, :, 5:] = lowest
        x[4, 0, 4000] = torch.nan
        x[4, 1, 8999] = torch.inf
        x[5, 2, :] = torch.nan
        s[5, 0] = -torch.inf
        s[5, 1] = torch.nan
        check_select(cache_ops.select_beams(x.to(dev), s.to(dev), 40), x, s, 40)
    x = torch.full((1, 2, 300), -1000.0)          # far below 0, where splits of -inf must not stand in
    x[0, :, 3] = -999.0
    x = torch.nn.functional.pad(x, (0, 20000), value=-torch.inf)
    s = torch.tensor([[0.0, -0.25]])
    check_select(cache_ops.select_beams(x.to(dev), s.to(dev), 5), x, s, 5)


def test_select_signed_zeros_and_infinite_scores(dev):
    """Scores of -0 and +0 are alike, and +inf is a score."""
    x = torch.zeros(2, 4, 50)
    s = torch.tensor([[0.0, -0.0, 0.0, -0.0], [torch.inf, -1.0, -torch.inf, torch.inf]])
    ended = torch.tensor([[True, True, True, True], [False, False, False, True]])
    for k in (3, 6, 64):
        check_select(cache_ops.select_beams(x.to(dev), s.to(dev), k, ended=ended.to(dev), end_token=7), x, s, k, ended, 7)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("V", [1, 50, 9000, 50021])
def test_select_rows_of_huge_logits(dev, dtype, V):
    """A mask of the type's lowest value that leaves nothing of a row, and logits as large: the beam's
    score and the number of tokens are what remains."""
    low, high = torch.finfo(dtype).min, torch.finfo(dtype).max
    x, s = select_case(5, 3, V, dtype, seed=V)
    x[0, 1] = low                                 # beside beams with logits
    x[1] = low
    x[2] = high
    x[3, :, ::3] = high / 4
    x[3, :, 1::3] = high / 2
    x[4, 0] = high / 2
    x[4, 0, V // 2] = high
    s[1:4] = torch.tensor([-1.5, -2.0, -2.5])
    s[0, 2] = s[3, 1:] = s[4, 2] = -torch.inf     # no two beams whose candidates may come close
    for k in (3, 20, 64):
        check_select(cache_ops.select_beams(x.to(dev), s.to(dev), k), x, s, k)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V", [50, 9000])
def test_select_scores_below_their_range(dev, dtype, V):
    """Masked logits of a masked beam: their sum is -inf in fp32, and no candidate."""
    low = torch.finfo(torch.float32).min
    x, s = select_case(3, 2, V, dtype, seed=V)
    x[:, :, 5:] = torch.finfo(dtype).min
    s[:, 0] = low
    s[1, 1], s[2, 1] = low / 2, -torch.inf
    for k in (4, 30, 64):
        got = cache_ops.select_beams(x.to(dev), s.to(dev), k)
        check_select(got, x, s, k)
        assert ((got[1] < 0) == (got[0] == -torch.inf)).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("W,V,k", [(4, 50, 3), (4, 50, 40), (3, 9000, 8), (4, 20011, 64), (32, 20000, 40), (64, 70000, 64)])
def test_select_scores_that_swallow_the_logits(dev, dtype, W, V, k):
    """Beams masked by the type's lowest value, -1e18 or +inf: in 64 bits all their candidates are
    alike, and stay in the order of their logits. Few lists and many, joined each way."""
    low = torch.finfo(torch.float32).min
    B = 4 if W * V < 10 ** 6 else 1
    x, _ = select_case(B, W, V, dtype, seed=V + k)
    x[:, :, ::7] = -0.0
    x[:, :, 3::7] = 0.0
    s = torch.full((B, W), low)
    if B == 4:
        s[1, 1:] = -1e18
        s[2, W // 2:] = torch.inf
        s[3, W - 1] = -2.0
    for ended in (None, torch.rand(B, W, generator=torch.Generator().manual_seed(1)) < 0.3):
        got = cache_ops.select_beams(x.to(dev), s.to(dev), k, ended=None if ended is None else ended.to(dev), end_token=V - 1)
        check_select(got, x, s, k, ended, V - 1)


def test_select_ended_beams(dev):
    for W, k in ((4, 8), (1, 3), (32, 64)):
        x, s = select_case(5, W, 3001, torch.bfloat16, W)
        ended = torch.rand(5, W, generator=torch.Generator().manual_seed(2)) < 0.5
        ended[1], ended[2] = True, False
        x[0][ended[0]] = torch.nan                # logits of beams at their end are not looked at
        s[3, 0] = -torch.inf
        got = cache_ops.select_beams(x.to(dev), s.to(dev), k, ended=ended.to(dev), end_token=2999)
        check_select(got, x, s, k, ended, 2999)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("pad,first", [(1, 0), (3, 1), (8, 5)])
def test_select_strided(dev, dtype, pad, first):
    """Rows of a padded vocabulary at any element; the padding holds what would win."""
    B, W, V = 3, 4, 4097
    wide = torch.full((B, W + 1, V + pad + first), 99.0).to(dtype)
    x, s = select_case(B, W, V, dtype, 11)
    wide[:, :W, first: first + V] = x
    d = wide.to(dev)
    got = cache_ops.select_beams(d[:, :W, first: first + V], s.to(dev), 8)
    check_select(got, x, s, 8)
    one = d[:1, :1, first: first + V].expand(B, W, V)
    check_select(cache_ops.select_beams(one, s.to(dev), 8), one.cpu(), s, 8)


def test_select_on_another_stream(dev):
    st = torch.cuda.Stream()
    cases = [select_case(2, 4, 40000, torch.bfloat16, i) for i in range(4)]
    on = [(x.to(dev), s.to(dev)) for x, s in cases]
    torch.cuda.synchronize()
    got = [cache_ops.select_beams(x, s, 8, stream=(st.cuda_stream if i % 2 else 0)) for i, (x, s) in enumerate(on)]
    torch.cuda.synchronize()
    for g, (x, s) in zip(got, cases):
        check_select(g, x, s, 8)


# -------------------------------------------------------------------- reorder
def reorder_case(sizes, layout="nhd", dtype=torch.bfloat16, ps=16, h=2, d=16, L=3, seed=0, parents=None, spare=0):
    """sizes: (beams, tokens) of each request; half of the full pages are shared."""
    rng = np.random.default_rng(seed)
    gen = torch.Generator().manual_seed(seed)
    bt, beams, nxt = [], [], 1
    for W, n in sizes:
        pages = -(-n // ps)
        stride = pages + spare
        beams.append((len(bt), stride, W, n))
        shared = list(range(nxt, nxt + (n // ps) // 2))
        nxt += len(shared)
        for _ in range(W):
            own = list(range(nxt, nxt + pages - len(shared)))
            nxt += len(own)
            bt += shared + own + [-7] * spare
    ids = rng.permutation(np.arange(1, nxt)).tolist() if nxt > 1 else []
    bt = np.array([ids[i - 1] if i > 0 else i for i in bt] + [0], np.int32)
    layers = [make_layer(layout, nxt + 2, ps, h, d, dtype, gen, kind="bytes")[0] for _ in range(L)]
    pf = make_layer(layout, 1, ps, h, d, dtype, gen)[1]
    most = max(W for W, _ in sizes)
    p = rng.integers(-1, most + 1, (len(sizes), most)) if parents is None else parents
    return layers, pf, bt, p.astype(np.int32), beams


def check_reorder(dev, case, stream=0, columns=None):
    layers, pf, bt, p, beams = case
    on = [to_dev(t, dev) for t in layers]
    bd, pd = torch.from_numpy(bt).to(dev), torch.from_numpy(p).to(dev)
    if columns is not None:
        pd = torch.cat([pd, torch.full((len(p), columns), 0, dtype=torch.int32, device=dev)], 1)[:, : p.shape[1]]
    torch.cuda.synchronize()
    cache_ops.reorder_beams(on, pf, bd, pd, beams, stream=stream)
    torch.cuda.synchronize()
    odec.reorder(layers, pf, bt, p, beams)
    assert (bd.cpu().numpy() == bt).all()
    for got, want in zip(on, layers):
        assert same_bytes(got, want)


@pytest.mark.parametrize("layout", LAYOUTS + ["mla"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.uint8, torch.float32])
def test_reorder_layouts(dev, layout, dtype):
    check_reorder(dev, reorder_case([(4, 37), (3, 16), (4, 5), (2, 79)], layout, dtype))


@pytest.mark.parametrize("W", [1, 2, 4, 5, 8, 9, 16, 17, 31, 32])
def test_reorder_beams(dev, W):
    check_reorder(dev, reorder_case([(W, 40), (max(1, W - 1), 21)], seed=W, spare=1))
    turn = np.roll(np.arange(W), 1)[None, :]                  # every beam exchanges its place
    check_reorder(dev, reorder_case([(W, 30)], seed=W, parents=turn))
    check_reorder(dev, reorder_case([(W, 30)], seed=W, parents=np.zeros((1, W), int)))


@pytest.mark.parametrize("ps,h,d,layout", [(1, 1, 8, "nhd"), (3, 3, 5, "hnd"), (64, 1, 2, "packed"), (16, 8, 128, "nhd"), (16, 8, 128, "packed"),
                                           (256, 2, 12, "hnd"), (5, 1, 1, "nhd")])
def test_reorder_sizes(dev, ps, h, d, layout):
    if d == 1:                                                # no pairs: refused
        with pytest.raises(RuntimeError, match="head_dim from 2 on"):
            check_reorder(dev, reorder_case([(3, 4)], layout, torch.uint8, ps=ps, h=h, d=d, L=2))
        return
    for n in (1, ps - 1, ps, ps + 1, 3 * ps + ps // 2):
        if n > 0:
            check_reorder(dev, reorder_case([(3, n), (4, 2 * ps)], layout, torch.uint8, ps=ps, h=h, d=d, L=2, seed=n))


def test_reorder_missing_pages_and_long_lists(dev):
    layers, pf, bt, p, beams = reorder_case([(4, 50), (4, 90)], seed=4, parents=np.array([[1, 2, 3, 0], [3, 3, 1, 1]]))
    for w, bad in ((0, 0), (2, -5), (3, 10 ** 6)):
        bt[beams[0][0] + w * beams[0][1] + 3] = bad           # last pages: not moved, from nor to
    bt[beams[1][0] + 2] = 0                                    # a full page's id moves as any
    check_reorder(dev, (layers, pf, bt, p, beams))
    # thousands of pages, hundreds of requests, more layers than fit in the arguments
    check_reorder(dev, reorder_case([(3, 20001)], ps=2, h=1, d=4, L=2))
    check_reorder(dev, reorder_case([(2, 9)] * 300, ps=4, h=1, d=8, L=3), columns=3)
    check_reorder(dev, reorder_case([(2, 9)] * 3, ps=4, h=1, d=8, L=70), stream=torch.cuda.Stream().cuda_stream)


def test_reorder_rows_and_lists_of_more_than_a_launch(dev):
    """520000 requests of 32 workgroups of rows each, and one for their lists: 2^24 together
    and more. The last pages are missing, which moves no rows."""
    n, PS, H, D = 520000, 2, 256, 128
    layer = torch.full((2, 4, PS, H, D), 7, dtype=torch.bfloat16, device=dev)
    bt = torch.tensor([2, 0, 3, 0], dtype=torch.int32, device=dev).repeat(n)
    parents = torch.tensor([[1, 0]], dtype=torch.int32, device=dev).expand(n, 2).contiguous()
    parents[::2] = -1
    beams = np.empty((n, 4), np.int64)
    beams[:] = (0, 2, 2, 3)
    beams[:, 0] = 4 * np.arange(n)
    torch.cuda.synchronize()
    cache_ops.reorder_beams([layer], False, bt, parents, beams)
    torch.cuda.synchronize()
    got = bt.view(-1, 2, 4).cpu()
    assert (got[:, 0] == torch.tensor([2, 0, 3, 0])).all() and (got[:, 1] == torch.tensor([3, 0, 2, 0])).all()
    assert (layer == 7).all()


# ------------------------------------------------------------- far offsets
def test_offsets_past_32_bits(dev):
    """Rows, pages and logits more than 2^32 elements into their tensors."""
    f = torch.from_numpy(np.asarray(orope.default_inv_freq(64, 10000.0))).to(dev)
    g = torch.Generator().manual_seed(3)
    # rows far apart: element 2^32 is in row 4096
    T, stride = 4200, 2 ** 20
    wide = torch.empty(T * stride, dtype=torch.bfloat16, device=dev)
    x = wide.as_strided((T, 2, 64), (stride, 64, 1))
    host = torch.randn(T, 2, 64, generator=g).to(torch.bfloat16)
    x.copy_(host)
    pos = torch.arange(T, device=dev) * 3
    out = cache_ops.rotate_rows(x, pos, f, 64)
    want, off = odec.rotate(host, pos.cpu().numpy(), f.cpu().numpy(), 64)
    close(out, want, off, torch.bfloat16)
    cache_ops.rotate_rows(x, pos, f, 64, out=x)
    assert torch.equal(x, out)
    # the same memory as a paged cache: its last blocks' V lie past 2^32 values
    NB, PS, H, D = 537000, 16, 4, 64
    layer = wide[: 2 * NB * PS * H * D].view(2, NB, PS, H, D)
    assert layer.stride(0) + (NB - 2) * layer.stride(1) > 2 ** 32
    bt = torch.tensor([NB - 1, 5, NB - 2], dtype=torch.int32, device=dev)
    layer[:, bt.long()] = 0
    k, v = (torch.randn(40, H, D, generator=g).to(torch.bfloat16).to(dev) for _ in range(2))
    cache_ops.append_tokens(layer, False, bt, k, v, [(0, 0, 40, 2)])
    got = layer[:, bt.long()].flatten(1, 2)
    assert torch.equal(got[0, 2:42], k) and torch.equal(got[1, 2:42], v)
    assert not got[:, :2].any() and not got[:, 42:].any()
    # two beams exchange the rows of their last pages, one at each end
    lists = torch.tensor([NB - 1, 5], dtype=torch.int32, device=dev)
    before = layer[:, lists.long()].clone()
    cache_ops.reorder_beams([layer], False, lists, torch.tensor([[1, 0]], dtype=torch.int32, device=dev), [(0, 1, 2, 9)])
    after = layer[:, lists.long()]
    assert torch.equal(after[:, 0, :9], before[:, 1, :9]) and torch.equal(after[:, 1, :9], before[:, 0, :9])
    assert torch.equal(after[:, :, 9:], before[:, :, 9:])
    # logits of beams far apart
    logits = wide.as_strided((2, 3, 5000), (2 ** 31 + 8, 2 ** 29 + 1, 1))
    y, s = select_case(2, 3, 5000, torch.bfloat16, 4)
    logits.copy_(y)
    check_select(cache_ops.select_beams(logits, s.to(dev), 6), y, s, 6)


# ------------------------------------------------------------- graphs, the loop
def test_captured_steps_replay(dev):
    """A captured step of all four calls, replayed with other inputs and eager work between."""
    s = Step([(1, 5), (1, 20), (1, 15), (1, 16)], h=2, g=2)
    layer = to_dev(s.layer, dev)
    f = torch.from_numpy(np.asarray(s.rope[0])).to(dev)
    bt, joint = torch.from_numpy(s.bt).to(dev), s.joint.to(dev)
    q, k, v = s.parts(joint)
    x, sc = select_case(1, 4, 9000, torch.bfloat16, 1)
    xd, scd = x.to(dev), sc.to(dev)
    pos = torch.zeros(s.T, dtype=torch.int64, device=dev)
    lists = [(0, 2, 2, 21)]
    par_in = torch.zeros(1, 2, dtype=torch.int32, device=dev)
    bt2 = torch.tensor([1, 2, 3, 4], dtype=torch.int32, device=dev)
    l2 = to_dev(make_layer("nhd", 6, 16, 2, 64, torch.bfloat16, torch.Generator().manual_seed(8))[0], dev)

    def step():
        out = cache_ops.append_tokens(layer, s.pf, bt, k, v, s.seqs, f, s.R, q=q, positions=pos)
        rot = cache_ops.rotate_rows(q, pos, f, s.R)
        sel = cache_ops.select_beams(xd, scd, 8)
        cache_ops.reorder_beams([l2], False, bt2, par_in, lists)
        return out, rot, sel

    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            out, rot, sel = step()
    for i in range(4):
        s.joint.normal_(generator=torch.Generator().manual_seed(i))
        joint.copy_(s.joint)
        s.layer.copy_(layer.cpu())
        pos.copy_(torch.tensor([i, 100 * i, 7, 10 ** 6]))
        x, sc = select_case(1, 4, 9000, torch.bfloat16, 10 + i)
        xd.copy_(x)
        scd.copy_(sc)
        par_in.copy_(torch.tensor([[1, 0]] if i % 2 else [[0, 0]]))
        want_l2, want_bt = l2.cpu(), bt2.cpu().numpy().copy()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        s.check(out, layer, pos.cpu().numpy())
        assert torch.equal(out, rot)
        check_select(sel, x, sc, 8)
        odec.reorder([want_l2], False, want_bt, par_in.cpu().numpy(), lists)
        assert same_bytes(l2, want_l2) and (bt2.cpu().numpy() == want_bt).all()
        eager = cache_ops.select_beams(xd, scd, 8)
        assert all(torch.equal(a, b) for a, b in zip(sel, eager))
    big = [(0, i, 1, 0) for i in range(100)]
    qb = torch.zeros(100, 2, 64, dtype=torch.bfloat16, device=dev)
    with pytest.raises(RuntimeError, match="cannot be captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            cache_ops.append_tokens(layer, s.pf, bt, qb, qb, big, f, s.R)
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.uint8])
def test_a_beam_search_over_the_paged_cache(dev, dtype):
    """Prompt, then steps of append, attention, choice and reordering, without the host
    looking: at its end each beam's pages hold the rows of its own tokens, bit by bit,
    and its attention is that over a cache that was filled with them alone."""
    W, V, H, G, D, PS, prompt, steps, L = 4, 503, 2, 2, 64, 8, 13, 21, 2
    g = torch.Generator().manual_seed(6)
    qtype = torch.bfloat16
    emb = torch.randn(L, V, (G + 2) * H, D, generator=g).to(qtype).to(dev)
    head = torch.randn(G * H * D, V, generator=g).to(dev) * 0.5
    f = torch.from_numpy(np.asarray(orope.default_inv_freq(D, 10000.0))).to(dev)
    pages = -(-(prompt + steps) // PS)
    # one prompt in shared full pages; each beam has its own page at every other place of its list
    shared = prompt // PS
    own = [[shared + w * (pages - shared) + i + 1 for i in range(pages - shared)] for w in range(W)]
    bt = torch.tensor([list(range(1, shared + 1)) + own[w] for w in range(W)], dtype=torch.int32).flatten().to(dev)
    nb = shared + W * (pages - shared) + 1
    layers = [to_dev(make_layer("hnd", nb, PS, H, D, dtype, g)[0], dev) for _ in range(L)]
    ks = torch.tensor([0.05, 0.1], device=dev) if dtype == torch.uint8 else None
    parts = lambda e: (e[:, : G * H], e[:, G * H: (G + 1) * H], e[:, (G + 1) * H:])
    tokens = torch.randint(0, V, (prompt,), generator=g).to(dev)

    def forward(caches, table, seqs, toks, pos=None):
        """Layers do not feed each other here; the last layer's attention makes the logits."""
        for l, layer in enumerate(caches):
            q, k, v = parts(emb[l, toks])
            q = cache_ops.append_tokens(layer, False, table, k, v, seqs, f, D, q=q, positions=pos, k_scale=ks, v_scale=ks)
            out, _ = cache_ops.attend_pages(layer, False, table, q, seqs, k_scale=ks, v_scale=ks)
        return out

    out = forward(layers, bt, [(0, 0, prompt, 0)], tokens)
    logits = (out[-1:].float().flatten(1) @ head)[None].expand(1, W, V).contiguous()
    scores = torch.tensor([[0.0] + [-torch.inf] * (W - 1)], device=dev)
    history = tokens.view(1, -1).expand(W, -1)
    n = prompt
    for step in range(steps):
        scores, parents, toks = cache_ops.select_beams(logits, scores)
        check_select((scores, parents, toks), logits.cpu(), last if step else torch.tensor([[0.0] + [-torch.inf] * (W - 1)]), W)
        cache_ops.reorder_beams(layers, False, bt, parents, [(0, pages, W, n)])
        history = torch.cat([history[parents[0].long()], toks[0].long()[:, None]], 1)
        out = forward(layers, bt, [(w * pages, w, 1, n) for w in range(W)], toks[0].long())
        logits = (out.float().flatten(1) @ head)[None]
        last = scores.cpu()
        n += 1
    # the same tokens of each beam into a cache of its own
    alone = [to_dev(make_layer("hnd", W * pages + 1, PS, H, D, dtype, torch.Generator().manual_seed(9))[0], dev) for _ in range(L)]
    table = (torch.arange(W * pages, dtype=torch.int32) + 1).to(dev)
    for w in range(W):
        forward(alone, table, [(w * pages, 0, n - 1, 0)], history[w, : n - 1])
    ref = forward(alone, table, [(w * pages, w, 1, n - 1) for w in range(W)], history[:, n - 1])
    assert torch.equal(out, ref)
    for a, b in zip(layers, alone):
        for view in (k_rows_view, v_view):
            x, y = view(a, False), view(b, False)
            for w in range(W):
                for t in range(n):
                    assert same_bytes(x[int(bt[w * pages + t // PS]), t % PS], y[w * pages + 1 + t // PS, t % PS])
