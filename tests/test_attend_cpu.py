"""Attention, weighing and eviction without a GPU: the oracle against torch and
brute force, and every refusal of the C ABI and the Python layer (fake device
pointers; each case fails before any device call)."""
import ctypes

import numpy as np
import pytest
import torch

from daric_amd import _lib, cache_ops
from oracle import attend as oatt
from tests.gpu_util import make_layer
from tests.test_capi_cpu import fake

lib = pytest.fixture(scope="module")(lambda: _lib.load())


# ------------------------------------------------------------------ the oracle
@pytest.mark.parametrize("layout", ["nhd", "hnd", "pf", "packed"])
def test_oracle_attention_is_softmax_attention(layout):
    g = torch.Generator().manual_seed(3)
    layer, pf = make_layer(layout, 9, 4, 2, 8, torch.float16, g)
    bt = np.array([5, 3, 8, 1], np.int32)
    q = torch.randn(5, 4, 8, generator=g).to(torch.float16)
    out, lse, *_ = oatt.attend(layer, pf, bt, q, [(0, 0, 5, 9)], scale=0.3)
    k = torch.from_numpy(oatt.gather(oatt.k_rows_view(layer, pf), bt, 0, 14)[0]).repeat_interleave(2, 1).transpose(0, 1)
    v = torch.from_numpy(oatt.gather(oatt.v_view(layer, pf), bt, 0, 14)[0]).repeat_interleave(2, 1).transpose(0, 1)
    see = torch.arange(14)[None, :] <= torch.arange(5)[:, None] + 9
    s = (q.double().transpose(0, 1) @ k.transpose(1, 2) * 0.3).masked_fill(~see, -torch.inf)
    want = (s.softmax(-1) @ v).transpose(0, 1)
    assert torch.allclose(torch.from_numpy(out), want, atol=1e-12)
    assert torch.allclose(torch.from_numpy(lse), s.logsumexp(-1).t(), atol=1e-12)
    w, *_ = oatt.weigh(layer, pf, bt, q, torch.from_numpy(lse), [(0, 0, 5, 9, 2)], np.ones((2, 17)), scale=0.3)
    p = s.softmax(-1).sum(1).view(2, 2, 14).sum(1).numpy()
    assert np.allclose(w[:, 2:16], 1 + p, atol=1e-12) and (w[:, [0, 1, 16]] == 1).all()


def test_oracle_tree_and_missing_pages():
    # draft 2 sees drafts 0 and 2; the null page's tokens are not there
    assert oatt.sees(2, 3, 3, [0b101]).tolist() == [True] * 3 + [True, False, True]
    wide = [1 << 63, 1]
    assert np.nonzero(oatt.sees(0, 0, 70, wide))[0].tolist() == [63, 64]
    layer, pf = make_layer("nhd", 4, 2, 1, 2, torch.float16, torch.Generator().manual_seed(0))
    assert oatt.gather(oatt.k_rows_view(layer, pf), [1, 0, 9, 3], 0, 8)[1].tolist() == [True] * 2 + [False] * 4 + [True] * 2


def test_oracle_eviction_keeps_the_heaviest_and_moves_few():
    layer, pf = make_layer("nhd", 8, 2, 1, 2, torch.float16, torch.Generator().manual_seed(1))
    before = layer.clone()
    bt = [4, 2, 7, 1, 5]
    w = np.array([[[0, 5, 1, 7, 2, 9, 2, 0, 3, 8]]], np.float32)
    kept = oatt.evict([layer], pf, bt, w, [(0, 0, 10, 5, 1, 1)], 5)
    # stay: 0 (first), 9 (recent), 5 (9), 3 (7), 1 (5); slots 2 and 4 are free, taken by 5 and 9
    assert kept[0, 0, 0].tolist() == [0, 1, 5, 3, 9]
    assert w[0, 0].tolist() == [0, 5, 9, 7, 8, 0, 0, 0, 0, 0]
    k, kb = layer[0], before[0]
    assert torch.equal(k[2, 0], kb[7, 1]) and torch.equal(k[7, 0], kb[5, 1]) and torch.equal(k[5], kb[5])


# ------------------------------------------------------------------ the C ABI
def seqs(*s):
    a = np.array(s, np.int64).reshape(-1, 5)
    return a.ctypes.data, len(a), a


def test_attention_refusals(lib):
    layer = fake((2, 8, 16, 4, 64), torch.bfloat16)
    f8 = fake((2, 8, 16, 4, 64), torch.uint8)
    bt = fake((8,), torch.int32, ptr=0x20000000)
    q = fake((10, 8, 64), torch.bfloat16, ptr=0x30000000)
    out = fake((10, 8, 64), torch.bfloat16, ptr=0x40000000)
    lse = fake((10, 8), torch.float32, ptr=0x50000000)
    w = fake((4, 200), torch.float32, ptr=0x60000000)
    ok = (0, 0, 10, 100, 0)

    def run(lay=layer, s=(ok,), q_=q, bt_=bt, mask=None, scale=1.0, ks=None, vs=None, out_=out, lse_=lse, w_=w, pf=0,
            weigh=False):
        ref = lambda t: ctypes.byref(t) if t is not None else None
        addr, n, _k = seqs(*s)
        if weigh:
            st = lib.daric_weigh_tokens(ref(lay), pf, ref(bt_), ref(q_), ref(lse_), addr, n, ref(mask), scale, ref(ks),
                                        ref(w_), 1, ctypes.c_uint64(0))
        else:
            need = ctypes.c_int64()
            if lib.daric_attend_workspace(ref(lay), pf, ref(q_), addr, n, ctypes.byref(need)) == 0:
                st = lib.daric_attend_pages(ref(lay), pf, ref(bt_), ref(q_), addr, n, ref(mask), scale, ref(ks), ref(vs),
                                            ref(out_), ref(lse_), 0x70000000, need.value, ctypes.c_uint64(0))
            else:
                st = 1
        assert st != 0
        return lib.daric_last_error().decode()

    for weigh in (False, True):
        r = lambda **k: run(weigh=weigh, **k)
        assert "unsupported KV cache dtype" in r(lay=fake((2, 8, 16, 4, 64), torch.float32))
        assert "3-D (MLA) cache" in r(lay=fake((8, 16, 64), torch.bfloat16), pf=1)
        assert "head_dim up to 256" in r(lay=fake((2, 8, 16, 4, 288), torch.bfloat16))
        assert "q must have the cache's element type" in r(q_=fake((10, 8, 64), torch.float16))
        assert "q must have the cache's element type" in r(q_=fake((10, 8, 64), torch.float32))
        assert "multiple of the cache's 4 heads" in r(q_=fake((10, 6, 64), torch.bfloat16))
        assert "multiple of the cache's 4 heads" in r(q_=fake((10, 8, 32), torch.bfloat16))
        assert "multiple of the cache's 4 heads" in r(q_=fake((10, 512), torch.bfloat16))
        assert "q must be on the layer's device" in r(q_=fake((10, 8, 64), torch.bfloat16, device=-1))
        assert "negative field of sequence 0" in r(s=((0, 0, -1, 4, 0),))
        assert "negative field of sequence 1" in r(s=((0, 0, 1, 4, 0), (0, 1, 1, -4, 50)))
        assert "rows exceed q" in r(s=((0, 5, 6, 4, 0),))
        assert "is too long" in r(s=((0, 0, 1, 2 ** 31, 0),))
        assert "is too long" in r(s=((0, 0, 1, 2 ** 62, 0),))
        assert "row 4 is in two sequences" in r(s=((0, 4, 2, 4, 50), (0, 0, 5, 4, 0)))
        assert "reads past the end of block_table" in r(s=((2, 0, 10, 100, 0),))
        assert "reads past the end of block_table" in r(s=((2 ** 62, 0, 1, 0, 0),))
        assert "block_table must be a 1-D contiguous int32" in r(bt_=fake((8,), torch.int64))
        assert "scale must be finite" in r(scale=float("nan"))
        assert "tree_mask must be" in r(mask=fake((9, 1), torch.int64))
        assert "tree_mask must be" in r(mask=fake((10, 1), torch.int32))
        assert "tree_mask has 0 words for 10 rows" in r(mask=fake((10, 0), torch.int64))
        assert "k_scale applies to fp8" in r(ks=fake((4,), torch.float32))
        assert "k_scale must be a contiguous float32 [H]" in r(lay=f8, ks=fake((5,), torch.float32))
        assert "lse must be" in r(lse_=fake((10, 4), torch.float32))
    assert "v_scale applies to fp8" in run(vs=fake((4,), torch.float32))
    assert "out must be" in run(out_=fake((10, 8, 64), torch.float16))
    assert "weights must be" in run(weigh=True, w_=fake((8, 200), torch.float32))
    assert "columns exceed weights" in run(weigh=True, s=((0, 0, 10, 100, 91),))
    assert "column 60 is in two sequences" in run(weigh=True, s=((0, 0, 4, 70, 0), (0, 4, 2, 10, 60)))


def test_attention_needs_its_workspace(lib):
    layer = fake((2, 4000, 16, 4, 64), torch.bfloat16)
    q, out = fake((1, 8, 64), torch.bfloat16), fake((1, 8, 64), torch.bfloat16, ptr=0x40000000)
    bt, lse = fake((4000,), torch.int32), fake((1, 8), torch.float32, ptr=0x50000000)
    addr, n, _k = seqs((0, 0, 1, 60000, 0))
    need = ctypes.c_int64()
    r = ctypes.byref
    assert lib.daric_attend_workspace(r(layer), 0, r(q), addr, n, r(need)) == 0 and need.value > 0
    for ptr, size in ((None, 0), (0x70000000, need.value - 1), (0x70000004, need.value)):
        assert lib.daric_attend_pages(r(layer), 0, r(bt), r(q), addr, n, None, 1.0, None, None, r(out), r(lse), ptr, size,
                                      ctypes.c_uint64(0)) == 1
        assert b"workspace must be 16-byte aligned" in lib.daric_last_error()


def test_nothing_to_attend_makes_no_device_call(lib):
    layer = fake((2, 8, 16, 4, 64), torch.bfloat16)
    bt, q = fake((8,), torch.int32), fake((10, 8, 64), torch.bfloat16)
    out, lse = fake((10, 8, 64), torch.bfloat16), fake((10, 8), torch.float32)
    w = fake((4, 200), torch.float32)
    r = ctypes.byref
    for s in ((), ((0, 0, 0, 100, 0),)):
        addr, n, _k = seqs(*s)
        need = ctypes.c_int64(7)
        assert lib.daric_attend_workspace(r(layer), 0, r(q), addr, n, r(need)) == 0 and need.value == 0
        assert lib.daric_attend_pages(r(layer), 0, r(bt), r(q), addr, n, None, 1.0, None, None, r(out), r(lse), None, 0,
                                      ctypes.c_uint64(0)) == 0
        assert lib.daric_weigh_tokens(r(layer), 0, r(bt), r(q), r(lse), addr, n, None, 1.0, None, r(w), 1,
                                      ctypes.c_uint64(0)) == 0


def test_eviction_refusals(lib):
    layers = (_lib.DaricTensor * 2)(*[fake((2, 8, 16, 4, 64), torch.bfloat16, ptr=0x10000000 * (i + 1)) for i in range(2)])
    bt = fake((8,), torch.int32)
    w = fake((2, 4, 200), torch.float32)
    kept = fake((2, 4, 1, 50), torch.int32)

    def run(s=((0, 0, 100, 50, 0, 0),), w_=w, kept_=kept, ws=None, lay=layers, bt_=bt):
        a = np.array(s, np.int64).reshape(-1, 6)
        r = ctypes.byref
        st = lib.daric_evict_tokens(lay, 2, 0, r(bt_), r(w_), a.ctypes.data, len(a), r(kept_), r(ws or kept_),
                                    ctypes.c_uint64(0))
        assert st != 0
        return lib.daric_last_error().decode()

    two = fake((2, 4, 2, 50), torch.int32)
    assert "weights must be" in run(w_=fake((2, 2, 200), torch.float32))
    assert "weights must be" in run(w_=fake((1, 4, 200), torch.float32))
    assert "weights must be" in run(w_=fake((2, 4, 200), torch.float16))
    assert "negative field of eviction 0" in run(s=((0, 0, 100, 50, -1, 0),))
    assert "n_first + n_recent must not exceed keep" in run(s=((0, 0, 100, 50, 26, 25),))
    assert "n_first + n_recent must not exceed keep" in run(s=((0, 0, 100, 50, 1, 2 ** 62),))
    assert "columns exceed weights" in run(s=((0, 101, 100, 50, 0, 0),))
    assert "reads past the end of block_table" in run(s=((3, 0, 100, 50, 0, 0),))
    assert "is too long" in run(s=((0, 0, 2 ** 31, 50, 0, 0),))
    assert "column 60 is in two sequences" in run(s=((0, 0, 64, 50, 0, 0), (4, 60, 64, 50, 0, 0)), kept_=two)
    assert "kmax at least 50" in run(kept_=fake((2, 4, 1, 49), torch.int32))
    assert "workspace must have kept's shape" in run(ws=fake((2, 4, 1, 51), torch.int32))
    assert "kept must be" in run(kept_=fake((2, 1, 1, 50), torch.int32))
    other = (_lib.DaricTensor * 2)(layers[0], fake((2, 8, 16, 4, 32), torch.bfloat16))
    assert "must share shape" in run(lay=other)
    # evictions of nothing need no device
    a = np.zeros((0, 6), np.int64)
    none = fake((2, 4, 0, 0), torch.int32)
    r = ctypes.byref
    assert lib.daric_evict_tokens(layers, 2, 0, r(bt), r(w), a.ctypes.data, 0, r(none), r(none), ctypes.c_uint64(0)) == 0


def test_memory_that_is_read_and_written(lib):
    """Written memory that other workgroups of the call read or write is refused
    before any device call."""
    r = ctypes.byref
    layer, bt = fake((2, 8, 16, 4, 64), torch.bfloat16, ptr=0x10000000), fake((8,), torch.int32, ptr=0x20000000)
    lse = fake((10, 8), torch.float32, ptr=0x50000000)
    q = fake((10, 8, 64), torch.bfloat16, ptr=0x40000000)
    addr, n, _k = seqs((0, 0, 10, 50, 0))
    for ptr in (0x40000000, 0x40000000 + 10 * 8 * 64 * 2 - 2, 0x40000000 - 10 * 8 * 64 * 2 + 2):
        out = fake((10, 8, 64), torch.bfloat16, ptr=ptr)
        assert lib.daric_attend_pages(r(layer), 0, r(bt), r(q), addr, n, None, 1.0, None, None, r(out), r(lse), None, 0,
                                      ctypes.c_uint64(0)) == 1
        assert b"out must not overlap q" in lib.daric_last_error()

    def evict(ptrs, ws):
        layers = (_lib.DaricTensor * 2)(*[fake((2, 8, 16, 4, 64), torch.bfloat16, ptr=p) for p in ptrs])
        w = fake((2, 4, 200), torch.float32, ptr=0x50000000)
        kept, work = fake((2, 4, 1, 50), torch.int32, ptr=0x60000000), fake((2, 4, 1, 50), torch.int32, ptr=ws)
        a = np.array([(0, 0, 100, 50, 0, 0)], np.int64)
        assert lib.daric_evict_tokens(layers, 2, 0, r(bt), r(w), a.ctypes.data, 1, r(kept), r(work), ctypes.c_uint64(0)) == 1
        return lib.daric_last_error().decode()

    assert "a layer is given twice" in evict((0x10000000, 0x10000000), 0x70000000)
    assert "workspace must not overlap kept" in evict((0x10000000, 0x18000000), 0x60000000 + 2 * 4 * 50 * 4 - 4)


def test_python_lists_of_sequences():
    good = [(0, 0, 1, 5), (1, 1, 2, 6)]
    addr, n, a = cache_ops._sequences(good)
    assert n == 2 and a.shape == (2, 5) and a.tolist() == [[0, 0, 1, 5, 0], [1, 1, 2, 6, 0]]
    assert cache_ops._sequences([])[1] == 0
    assert cache_ops._sequences(np.array(good, np.int32))[2].dtype == np.int64
    for bad in ([(0, 0, 1)], [(0, 0, 1.5, 2)], [("a", 0, 1, 2)]):
        with pytest.raises(ValueError):
            cache_ops._sequences(bad)


# ------------------------------------------------------ the oracle over matrices
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.uint8])
def test_oracle_matrices_are_its_rows(tree, dtype):
    from tests.test_gpu_attend import Case
    c = Case(None, [(5, 40), (0, 3), (70, 9)], dtype=dtype, qtype=torch.float16, h=2, g=2, d=16, tree=tree, seed=60)
    c.bt[c.seqs[2][0] + 1] = 0
    if tree:
        c.mask[3] = 0
        c.bt[:c.seqs[1][0]] = 0                          # rows that see nothing
    args = (c.layer, c.pf, c.bt, c.q, c.seqs, c.mask, c.scale, c.ks)
    want, got = oatt.attend(*args, c.vs), oatt.attend_matrix(*args, c.vs)
    for x, y in zip(want, got):
        np.testing.assert_allclose(y, x, rtol=1e-11, atol=1e-13)
    lse = torch.from_numpy(want[1]).float()
    w0 = np.random.default_rng(0).random((2, c.columns))
    wargs = (c.layer, c.pf, c.bt, c.q, lse, c.seqs, w0, c.mask, c.scale, c.ks)
    for x, y in zip(oatt.weigh(*wargs), oatt.weigh_matrix(*wargs)):
        np.testing.assert_allclose(y, x, rtol=1e-11, atol=1e-13)


@pytest.mark.parametrize("layout,shared", [("nhd", False), ("hnd", True), ("packed", False), ("mla", True)])
def test_oracle_eviction_over_matrices(layout, shared):
    g = torch.Generator().manual_seed(61)
    h = 1 if layout == "mla" else 3
    layers = [make_layer(layout, 40, 4, h, 8, torch.uint8, g, kind="bytes") for _ in range(2)]
    pf, a = layers[0][1], [t for t, _ in layers]
    b = [t.clone() for t in a]
    bt = np.random.default_rng(1).permutation(np.arange(1, 40)).astype(np.int32)
    bt[[2, 20]] = 0, 99
    ev = [(0, 1, 50, 20, 2, 3), (13, 60, 30, 30, 0, 0), (21, 100, 60, 11, 0, 5)]
    w = torch.randn(2, 1 if shared else h, 170, generator=g).round(decimals=1).numpy()
    w[0, 0, 5:9] = np.nan
    v = w.copy()
    np.testing.assert_array_equal(oatt.evict(a, pf, bt, w, ev, 30), oatt.evict_matrix(b, pf, bt, v, ev, 30))
    np.testing.assert_array_equal(w, v)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


# --------------------------------------------- memory that a call writes, and sizes
def test_written_memory_overlaps_nothing(lib):
    """Each pair of an argument that is written and another one, by its last or first
    bytes; refused before any device call."""
    r = ctypes.byref
    at = dict(layer=0x10000000, bt=0x20000000, q=0x30000000, out=0x40000000, lse=0x50000000, mask=0x60000000,
              ks=0x70000000, vs=0x80000000, work=0x90000000, w=0xa0000000)
    shape = dict(layer=((2, 40, 16, 4, 64), torch.uint8), bt=((40,), torch.int32), q=((1, 64, 64), torch.bfloat16),
                 out=((1, 64, 64), torch.bfloat16), lse=((1, 64), torch.float32), mask=((1, 1), torch.int64),
                 ks=((4,), torch.float32), vs=((4,), torch.float32), w=((4, 640), torch.float32))
    size = {k: int(np.prod(s)) * torch.empty(0, dtype=t).element_size() for k, (s, t) in shape.items()}
    names = dict(layer="the layer", bt="block_table", mask="tree_mask", ks="k_scale", vs="v_scale", work="workspace", w="weights")
    addr, n, _k = seqs((0, 0, 1, 639, 0))
    need = ctypes.c_int64()
    t = {k: fake(*shape[k], ptr=at[k]) for k in shape}
    assert lib.daric_attend_workspace(r(t["layer"]), 0, r(t["q"]), addr, n, r(need)) == 0
    size["work"] = need.value
    assert need.value > 0

    def call(weigh, moved):
        p = dict(at, **moved)
        t = {k: fake(*shape[k], ptr=p[k]) for k in shape}
        if weigh:
            st = lib.daric_weigh_tokens(r(t["layer"]), 0, r(t["bt"]), r(t["q"]), r(t["lse"]), addr, n, r(t["mask"]), 1.0,
                                        r(t["ks"]), r(t["w"]), 1, ctypes.c_uint64(0))
        else:
            st = lib.daric_attend_pages(r(t["layer"]), 0, r(t["bt"]), r(t["q"]), addr, n, r(t["mask"]), 1.0, r(t["ks"]),
                                        r(t["vs"]), r(t["out"]), r(t["lse"]), p["work"], need.value, ctypes.c_uint64(0))
        assert st == 1
        return lib.daric_last_error().decode()

    reads = ["q", "layer", "bt", "mask", "ks"]
    for weigh, pairs in ((True, [("w", x) for x in reads + ["lse"]]),
                         (False, [(w, x) for w in ("out", "lse", "work") for x in reads + ["vs"]] +
                                 [("out", "lse"), ("out", "work"), ("lse", "work")])):
        for w, x in pairs:
            unit = 16 if w == "work" else 2 if w == "out" else 4
            ends = [at[x] + size[x] - unit, at[x] - size[w] + unit]
            for ptr in ends if w != "work" else [(p // 16) * 16 for p in (at[x] + size[x] - 1, at[x])]:
                assert f"{names.get(w, w)} must not overlap {names.get(x, x)}" in call(weigh, {w: ptr}), (w, x)


def test_evictions_write_apart(lib):
    r = ctypes.byref
    at = dict(l0=0x10000000, l1=0x18000000, bt=0x20000000, w=0x50000000, kept=0x60000000, work=0x70000000)
    shape = dict(l0=((2, 8, 16, 4, 64), torch.bfloat16), l1=((2, 8, 16, 4, 64), torch.bfloat16), bt=((8,), torch.int32),
                 w=((2, 4, 200), torch.float32), kept=((2, 4, 1, 50), torch.int32), work=((2, 4, 1, 50), torch.int32))
    size = {k: int(np.prod(s)) * torch.empty(0, dtype=t).element_size() for k, (s, t) in shape.items()}
    a = np.array([(0, 0, 100, 50, 0, 0)], np.int64)
    names = dict(l0="a layer", l1="a layer", bt="block_table", w="weights", work="workspace")
    for x, y in [("work", "kept"), ("work", "w"), ("work", "bt"), ("kept", "w"), ("kept", "bt"), ("w", "bt"), ("l0", "bt"),
                 ("l1", "w"), ("l0", "kept"), ("l1", "work")]:
        for ptr in (at[y] + size[y] - 4, at[y] - size[x] + 4):
            p = dict(at, **{x: ptr})
            t = {k: fake(*shape[k], ptr=p[k]) for k in shape}
            layers = (_lib.DaricTensor * 2)(t["l0"], t["l1"])
            assert lib.daric_evict_tokens(layers, 2, 0, r(t["bt"]), r(t["w"]), a.ctypes.data, 1, r(t["kept"]), r(t["work"]),
                                          ctypes.c_uint64(0)) == 1, (x, y)
            assert f"{names.get(x, x)} must not overlap {names.get(y, y)}" in lib.daric_last_error().decode(), (x, y)


def test_rows_past_32_bits_are_refused(lib):
    """The kernels count rows of q in 32 bits."""
    layer, bt = fake((2, 8, 16, 1, 2), torch.bfloat16), fake((8,), torch.int32)
    T = 2 ** 31 + 50
    q, lse = fake((T, 1, 2), torch.bfloat16, ptr=2 ** 40), fake((T, 1), torch.float32, ptr=2 ** 41)
    out, w = fake((T, 1, 2), torch.bfloat16, ptr=2 ** 42), fake((1, 100), torch.float32, ptr=2 ** 43)
    need = ctypes.c_int64()
    r = ctypes.byref
    for start in (2 ** 31 - 8, 2 ** 31 - 1, 2 ** 31, 2 ** 31 + 40):
        addr, n, _k = seqs((0, start, 9, 20, 0))
        assert lib.daric_attend_workspace(r(layer), 0, r(q), addr, n, r(need)) == 1
        assert b"reaches too far into q" in lib.daric_last_error()
        assert lib.daric_attend_pages(r(layer), 0, r(bt), r(q), addr, n, None, 1.0, None, None, r(out), r(lse), None, 0,
                                      ctypes.c_uint64(0)) == 1
        assert b"reaches too far into q" in lib.daric_last_error()
        assert lib.daric_weigh_tokens(r(layer), 0, r(bt), r(q), r(lse), addr, n, None, 1.0, None, r(w), 1,
                                      ctypes.c_uint64(0)) == 1
        assert b"reaches too far into q" in lib.daric_last_error()
    addr, n, _k = seqs((0, 2 ** 31 - 10, 9, 20, 0))
    assert lib.daric_attend_workspace(r(layer), 0, r(q), addr, n, r(need)) == 0


def test_scales_whose_power_of_2_is_infinite_are_refused(lib):
    layer, bt = fake((2, 8, 16, 4, 64), torch.bfloat16), fake((8,), torch.int32, ptr=0x20000000)
    q, lse = fake((10, 8, 64), torch.bfloat16, ptr=0x30000000), fake((10, 8), torch.float32, ptr=0x50000000)
    out, w = fake((10, 8, 64), torch.bfloat16, ptr=0x40000000), fake((4, 200), torch.float32, ptr=0x60000000)
    addr, n, _k = seqs((0, 0, 10, 50, 0))
    r = ctypes.byref
    for scale in (2.5e38, -3.4e38, float("inf"), float("nan")):
        assert lib.daric_attend_pages(r(layer), 0, r(bt), r(q), addr, n, None, scale, None, None, r(out), r(lse), None, 0,
                                      ctypes.c_uint64(0)) == 1
        assert b"scale must be finite" in lib.daric_last_error()
        assert lib.daric_weigh_tokens(r(layer), 0, r(bt), r(q), r(lse), addr, n, None, scale, None, r(w), 1,
                                      ctypes.c_uint64(0)) == 1
        assert b"scale must be finite" in lib.daric_last_error()


def test_inputs_that_require_a_gradient_are_refused():
    """No output silently without a gradient; under no_grad, and for detached inputs, the
    calls go on (here to the refusal of tensors that are not on a GPU)."""
    layer, bt = torch.zeros(2, 4, 16, 2, 64), torch.ones(4, dtype=torch.int32)
    q, lse, w, s = torch.zeros(1, 4, 64), torch.zeros(1, 4), torch.zeros(2, 40), torch.ones(2)
    want = lambda t: t.clone().requires_grad_()
    attend = lambda l=layer, q=q, **k: cache_ops.attend_pages(l, False, bt, q, [(0, 0, 1, 20)], **k)
    weigh = lambda l=layer, q=q, lse=lse, w=w, **k: cache_ops.weigh_tokens(l, False, bt, q, lse, [(0, 0, 1, 20, 0)], weights=w, **k)
    evict = lambda l=layer, w=w: cache_ops.evict_tokens([l], False, bt, w[None], [(0, 0, 20, 10, 0, 0)])
    for call in (lambda: attend(q=want(q)), lambda: attend(want(layer)), lambda: attend(k_scale=want(s)),
                 lambda: attend(v_scale=want(s)), lambda: weigh(q=want(q)), lambda: weigh(lse=want(lse)),
                 lambda: weigh(w=want(w)), lambda: weigh(k_scale=want(s)), lambda: evict(w=want(w)), lambda: evict(want(layer))):
        with pytest.raises(RuntimeError, match="has no backward pass"):
            call()
        with torch.no_grad(), pytest.raises(RuntimeError, match="must be on CUDA"):
            call()
    for call in (attend, weigh, evict):
        with pytest.raises(RuntimeError, match="must be on CUDA"):
            call()
