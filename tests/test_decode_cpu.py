"""New rows and beam search without a GPU: the oracle against facts that do not
restate its formulas, the rotary frequencies, and every refusal of the C ABI and the
Python layer (fake device pointers; each case fails before any device call)."""
import ctypes
import math

import numpy as np
import pytest
import torch

from daric_amd import _lib, cache_ops, rotary
from oracle import decode as odec
from oracle import rope as orope
from tests.gpu_util import make_layer
from tests.test_capi_cpu import fake

lib = pytest.fixture(scope="module")(lambda: _lib.load())
r = ctypes.byref


# ------------------------------------------------------------------ the oracle
@pytest.mark.parametrize("neox", [True, False])
def test_oracle_rotation_is_a_complex_product(neox):
    rng = np.random.default_rng(1)
    f = orope.default_inv_freq(12, 10000.0)
    x = rng.normal(size=(5, 2, 16))
    p = np.array([0, 1, 777, -3, 10 ** 6])
    out, off = odec.rotate(x, p, f, 12, neox, 1.25)
    z = x[..., :6] + 1j * x[..., 6:12] if neox else x[..., 0:12:2] + 1j * x[..., 1:12:2]
    z = z * 1.25 * np.exp(1j * p[:, None, None].astype(float) * np.asarray(f, np.float64))
    got = out[..., :6] + 1j * out[..., 6:12] if neox else out[..., 0:12:2] + 1j * out[..., 1:12:2]
    assert np.allclose(got, z, atol=1e-12) and (out[..., 12:] == x[..., 12:]).all()
    assert (off[..., :12] > 0).all() and (off[..., 12:] == 0).all()
    back, _ = odec.rotate(out, -p, f, 12, neox, 0.8)
    assert np.allclose(back, x, atol=1e-9)
    # the rotation by positions agrees with the cached rows' rotation by a shift
    two, _ = odec.rotate(odec.rotate(x, p, f, 12, neox)[0], np.full(5, 40), f, 12, neox)
    assert np.allclose(two, odec.rotate(x, p + 40, f, 12, neox)[0], atol=1e-9)


def test_oracle_append_places_rows():
    layer, pf = make_layer("nhd", 6, 4, 1, 2, torch.float16, torch.Generator().manual_seed(0))
    k = torch.arange(12, dtype=torch.float16).view(6, 1, 2)
    where, pos, kk, vv, _ = odec.append(layer, pf, [3, 0, 5, 9], k, k, [(0, 1, 3, 2), (2, 4, 2, 3)])
    assert where == [(1, 3, 2), (2, 3, 3), (4, 5, 3)]            # token 4 is on the null page, 9 is no page
    assert pos.tolist() == [0, 2, 3, 4, 3, 4] and (kk == k.double().numpy()).all() and (vv == kk).all()


def test_oracle_selection_is_a_search_over_log_softmax():
    g = torch.Generator().manual_seed(2)
    x = torch.randn(2, 3, 40, generator=g)
    s = torch.randn(2, 3, generator=g)
    got = odec.select(x, s, 5)
    flat = (x.double().log_softmax(-1) + s.double()[..., None]).flatten(1)
    best, at = flat.topk(5)
    assert np.allclose(got[0], best.numpy()) and (got[1] == at.numpy() // 40).all() and (got[2] == at.numpy() % 40).all()
    # ties: the lower beam, then the lower token; an ended beam's one candidate; nothing behind
    x = torch.zeros(1, 2, 4)
    assert odec.select(x, [[0.0, 0.0]], 5)[1:][0].tolist() == [[0, 0, 0, 0, 1]]
    assert odec.select(x, [[0.0, 0.0]], 5)[2].tolist() == [[0, 1, 2, 3, 0]]
    got = odec.select(x, [[-1.0, -math.inf]], 3, ended=[[True, False]], end_token=2)
    assert got[0].tolist() == [[-1.0, -math.inf, -math.inf]] and got[1].tolist() == [[0, -1, -1]] and got[2].tolist() == [[2, -1, -1]]
    x[0, 0, 1] = math.nan
    assert odec.select(x, [[0.0, 0.0]], 1)[1].tolist() == [[1]]


def test_oracle_selection_of_huge_logits():
    """Rows of the type's lowest value alone are rows of equal logits, and so are those of 1e30."""
    for level in (torch.finfo(torch.float32).min, 1e30, torch.finfo(torch.float32).max):
        x = torch.full((1, 2, 10), level)
        got = odec.select(x, [[-1.5, -2.0]], 12)
        assert np.allclose(got[0][0], [-1.5 - math.log(10)] * 10 + [-2.0 - math.log(10)] * 2, rtol=1e-14)
        assert got[1].tolist() == [[0] * 10 + [1] * 2] and got[2].tolist() == [[*range(10), 0, 1]]


def test_oracle_selection_below_the_scores_range():
    """A candidate whose score is -inf in the fp32 that scores are given in is not there."""
    low = torch.finfo(torch.float32).min
    assert np.float32(odec.LEAST) == -np.inf and np.float32(np.nextafter(odec.LEAST, 0)) == low
    x = torch.tensor([[[0.0, low, low / 2, -1.0]]])
    got = odec.select(x, [[low / 2]], 4)
    assert got[2].tolist() == [[0, 3, 2, -1]] and got[1].tolist() == [[0, 0, 0, -1]] and got[0][0, 3] == -np.inf
    assert (got[0][0, :3].astype(np.float32) > -np.inf).all()


def test_oracle_selection_of_swallowed_logits():
    """Where the score leaves nothing of the logits in 64 bits they still order their beam's tokens."""
    x = torch.tensor([[[0.0, 3.0, -1.0, 3.0], [5.0, 9.0, 7.0, 8.0]]])
    low = torch.finfo(torch.float32).min
    for first, second in ((low, low), (-1e18, -1e18), (math.inf, math.inf)):
        got = odec.select(x, [[first, second]], 7)
        assert got[1].tolist() == [[0, 0, 0, 0, 1, 1, 1]] and got[2].tolist() == [[1, 3, 0, 2, 1, 3, 2]]
    got = odec.select(x, [[low, -1.0]], 6)
    assert got[1].tolist() == [[1, 1, 1, 1, 0, 0]] and got[2].tolist() == [[1, 3, 2, 0, 1, 3]]


def test_oracle_reorder_follows_parents():
    layer, pf = make_layer("nhd", 9, 2, 1, 2, torch.float16, torch.Generator().manual_seed(1))
    before = layer.clone()
    bt = np.array([1, 2, 3, 1, 4, 5, 1, 6, 7], np.int32)         # three beams of five tokens, page 1 shared
    odec.reorder([layer], pf, bt, [[1, 0, -1]], [(0, 3, 3, 5)])
    assert bt.tolist() == [1, 4, 3, 1, 2, 5, 1, 6, 7]            # full pages exchanged, last pages stay
    k, kb = layer[0], before[0]
    assert torch.equal(k[3, 0], kb[5, 0]) and torch.equal(k[5, 0], kb[3, 0]) and torch.equal(k[3, 1], kb[3, 1])
    assert torch.equal(k[7], kb[7]) and torch.equal(k[2], kb[2])


# ------------------------------------------------------------- frequencies
def test_frequencies_of_scaled_models():
    f, m = rotary.rotary_frequencies(128, 500000.0)
    assert m == 1.0 and f.dtype == torch.float32
    want = 500000.0 ** (-np.arange(0, 128, 2) / 128)
    assert np.allclose(f.numpy(), want, rtol=2.0 ** -24, atol=0)
    lin, _ = rotary.rotary_frequencies(128, 500000.0, {"type": "linear", "factor": 4.0})
    assert torch.equal(lin, f / 4)
    dyn = {"type": "dynamic", "factor": 2.0, "original_max_position_embeddings": 2048}
    assert torch.equal(rotary.rotary_frequencies(64, 10000.0, dyn, seq_len=2048)[0], rotary.rotary_frequencies(64)[0])
    longer = rotary.rotary_frequencies(64, 10000.0, dyn, seq_len=4096)[0]
    # the slowest pair is stretched by the whole ratio, 2 * 4096 / 2048 - 1 = 3, the fastest not at all
    plain = rotary.rotary_frequencies(64)[0]
    assert longer[0] == 1 and np.isclose(float(plain[-1] / longer[-1]), 3.0, rtol=1e-6)
    l3 = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
          "original_max_position_embeddings": 8192}
    g, m = rotary.rotary_frequencies(128, 500000.0, l3)
    wave = 2 * np.pi / want
    ratio = f.numpy() / g.numpy()
    assert m == 1.0 and np.allclose(ratio[wave < 8192 / 4], 1) and np.allclose(ratio[wave > 8192], 8)
    mid = (wave >= 8192 / 4) & (wave <= 8192)
    assert mid.any() and (ratio[mid] >= 1).all() and (ratio[mid] <= 8).all() and (np.diff(ratio) >= -1e-6).all()
    y, m = rotary.rotary_frequencies(64, 10000.0, {"type": "yarn", "factor": 4.0, "original_max_position_embeddings": 4096})
    p = rotary.rotary_frequencies(64)[0]
    assert np.isclose(m, 0.1 * math.log(4.0) + 1) and y[0] == p[0] and np.isclose(float(p[-1] / y[-1]), 4.0)
    assert rotary.rotary_frequencies(64, 10000.0, {"type": "yarn", "factor": 4.0, "attention_factor": 1.5,
                                                   "original_max_position_embeddings": 4096})[1] == 1.5


@pytest.mark.parametrize("R,base,factor,n", [(64, 150000.0, 32.0, 4096), (128, 10000.0, 4.0, 4096), (64, 10000.0, 40.0, 4096),
                                             (8, 1000.0, 4.0, 512), (16, 10.0, 2.0, 10 ** 6)])
@pytest.mark.parametrize("given", [{}, {"truncate": True}, {"truncate": False}])
def test_yarn_ramp(R, base, factor, n, given):
    """Every pair, by the turns that it makes over n positions: its share of the stretched frequency
    is linear in their logarithm from beta_fast down to beta_slow, and where the ends are whole dims
    from the last dim of at least beta_fast turns to the first of at most beta_slow."""
    got, _ = rotary.rotary_frequencies(R, base, {"type": "yarn", "factor": factor, "original_max_position_embeddings": n, **given})
    dims = np.arange(-300, 300)
    turns = n * base ** (-2.0 * dims / R) / (2 * np.pi)
    if given.get("truncate", True):
        first, last = max(dims[turns >= 32][-1], 0), min(dims[turns <= 1][0], R - 1)
    else:
        first, last = (np.interp(-np.log(t), -np.log(turns), dims) for t in (32.0, 1.0))
        first, last = max(first, 0), min(last, R - 1)
    i = np.arange(R // 2)
    share = np.clip((i - first) / max(last - first, 1e-3), 0, 1)
    f = base ** (-2.0 * i / R)
    # a rounding to fp32, and a few of 64 bits
    assert np.allclose(got.double().numpy(), f * (1 - share) + f / factor * share, rtol=2.0 ** -24 + 1e-11, atol=0)


@pytest.mark.parametrize("scale,part,whole,want", [
    (40.0, 1.0, 1.0, 1.0), (40.0, 0.707, 0.707, 1.0), (16.0, 1.0, 0.5, (0.1 * math.log(16) + 1) / (0.05 * math.log(16) + 1)),
    (16.0, None, None, 0.1 * math.log(16) + 1), (16.0, 1.0, None, 0.1 * math.log(16) + 1), (16.0, 1, 0, 0.1 * math.log(16) + 1),
    (16.0, 0.0, 0.0, 0.1 * math.log(16) + 1), (1.0, 0.5, None, 1.0), (0.5, 2.0, 3.0, 1.0)])
def test_yarn_scale_of_two_parts(scale, part, whole, want):
    """The table's scale is the ratio of the two parts' scales, which is 1 where they are alike."""
    given = {k: v for k, v in (("mscale", part), ("mscale_all_dim", whole)) if v is not None}
    yarn = {"type": "yarn", "factor": scale, "original_max_position_embeddings": 4096, **given}
    assert np.isclose(rotary.rotary_frequencies(64, 10000.0, yarn)[1], want, rtol=1e-14, atol=0)
    null = {**{"mscale": None, "mscale_all_dim": None, "truncate": None, "attention_factor": None}, **yarn}      # as left out
    assert np.isclose(rotary.rotary_frequencies(64, 10000.0, null)[1], want, rtol=1e-14, atol=0)
    assert torch.equal(rotary.rotary_frequencies(64, 10000.0, null)[0], rotary.rotary_frequencies(64, 10000.0, yarn)[0])
    assert rotary.rotary_frequencies(64, 10000.0, {**yarn, "attention_factor": 1.5})[1] == 1.5


@pytest.mark.parametrize("given", [{"mscale": 0.707}, {"mscale_all_dim": 1.0}, {"mscale": 0.707, "mscale_all_dim": 0.0},
                                   {"mscale": "1"}, {"mscale": math.nan, "mscale_all_dim": 1.0}])
def test_yarn_scale_refusals(given):
    yarn = {"type": "yarn", "factor": 16.0, "original_max_position_embeddings": 4096, **given}
    with pytest.raises(ValueError, match="mscale"):
        rotary.rotary_frequencies(64, 10000.0, yarn)


@pytest.mark.parametrize("kind", [{"type": "linear"}, {"rope_type": None, "type": "linear"}, {"rope_type": "linear", "type": "yarn"}])
def test_scaling_names(kind):
    """What changes no frequency may stand in a scaling, what may change one is refused if it is not known."""
    plain = rotary.rotary_frequencies(64, 5e5)[0]
    assert torch.equal(rotary.rotary_frequencies(64, 5e5, {**kind, "factor": 2.0, "rope_theta": 500000, "mrope_section": [16, 8, 8],
                                                           "partial_rotary_factor": 0.5})[0], plain / 2)
    assert torch.equal(rotary.rotary_frequencies(64, 5e5, {"rope_type": "default", "rope_theta": 5e5})[0], plain)
    assert torch.equal(rotary.rotary_frequencies(64, 5e5, {})[0], plain)
    for name in ("alpha", "extrapolation_factor", "long_factor", "attn_factor"):
        with pytest.raises(ValueError, match=name):
            rotary.rotary_frequencies(64, 5e5, {**kind, "factor": 2.0, name: 1.0})
    with pytest.raises(ValueError, match="rope_theta 10000"):
        rotary.rotary_frequencies(64, 5e5, {**kind, "factor": 2.0, "rope_theta": 10000.0})


@pytest.mark.parametrize("args,text", [
    ((7,), "positive and even"), ((0,), "positive and even"), ((8, -1.0), "base must be"),
    ((8, 10000.0, {"type": "linear"}), "finite factor"), ((8, 10000.0, {"type": "linear", "factor": 0}), "must be positive"),
    ((8, 10000.0, {"type": "spiral", "factor": 2.0}), "unknown rotary scaling"),
    ((8, 10000.0, {"type": "llama3", "factor": 2.0, "low_freq_factor": 4.0, "high_freq_factor": 1.0,
                   "original_max_position_embeddings": 64}), "below high_freq_factor"),
    ((8, 10000.0, {"type": "yarn", "factor": 2.0}), "original_max_position_embeddings")])
def test_frequency_refusals(args, text):
    with pytest.raises(ValueError, match=text):
        rotary.rotary_frequencies(*args)


# ------------------------------------------------------------------ the C ABI
def rope(R=64, ptr=0x90000000, neox=1):
    x = _lib.DaricRope()
    x.inv_freq, x.rotary_dim, x.is_neox = ptr, R, neox
    return x


def ref(t):
    return r(t) if t is not None else None


def test_rotation_refusals(lib):
    rows = fake((10, 8, 64), torch.bfloat16, ptr=0x30000000)
    out = fake((10, 8, 64), torch.bfloat16, ptr=0x40000000)
    pos = fake((10,), torch.int64, ptr=0x50000000)

    def run(x=rows, p=pos, ro=rope(), m=1.0, o=out):
        st = lib.daric_rotate_rows(ref(x), ref(p), ref(ro), m, ref(o), ctypes.c_uint64(0))
        assert st != 0
        return lib.daric_last_error().decode()

    assert "bfloat16, float16 or float32" in run(x=fake((10, 8, 64), torch.uint8))
    assert "must be [T, H, D]" in run(x=fake((10, 512), torch.bfloat16))
    assert "must be [T, H, D]" in run(x=fake((10, 8, 64), torch.bfloat16, strides=(512, 1, 8)))
    assert "negative strides" in run(x=fake((10, 8, 64), torch.bfloat16, strides=(-512, 64, 1)))
    assert "too large" in run(x=fake((10, 2 ** 20, 64), torch.bfloat16))
    assert "rows must be on CUDA" in run(x=fake((10, 8, 64), torch.bfloat16, device=-1))
    assert "positions must be" in run(p=fake((10,), torch.int32))
    assert "positions must be" in run(p=fake((9,), torch.int64))
    assert "positions must be" in run(p=fake((10,), torch.int64, device=1))
    assert "rope parameters" in run(ro=None)
    assert "inv_freq must not be null" in run(ro=rope(ptr=None))
    assert "rotary_dim must be" in run(ro=rope(66)) and "rotary_dim must be" in run(ro=rope(7)) and "rotary_dim must be" in run(ro=rope(0))
    assert "at most 512" in run(ro=rope(1024))
    assert "attention_scale must be finite" in run(m=math.nan) and "attention_scale must be finite" in run(m=math.inf)
    assert "out must be rows itself or" in run(o=fake((10, 8, 64), torch.float16, ptr=0x40000000))
    assert "out must be rows itself or" in run(o=fake((10, 8, 64), torch.bfloat16, ptr=0x40000000, strides=(1024, 64, 1)))
    assert "out must be rows itself or" in run(o=fake((10, 4, 64), torch.bfloat16, ptr=0x40000000))
    assert "out must not overlap rows" in run(o=fake((10, 8, 64), torch.bfloat16, ptr=0x30000080))
    assert "out must not overlap positions" in run(o=fake((10, 8, 64), torch.bfloat16, ptr=0x50000000))
    assert "out must not overlap inv_freq" in run(o=fake((10, 8, 64), torch.bfloat16, ptr=0x8fffffe0))
    one = fake((10, 8, 64), torch.bfloat16, ptr=0x30000000, strides=(0, 64, 1))
    assert "share memory" in run(x=one, o=one)
    none = fake((0, 8, 64), torch.bfloat16)
    assert lib.daric_rotate_rows(r(none), r(fake((0,), torch.int64)), r(rope()), 1.0, r(none), ctypes.c_uint64(0)) == 0


def test_append_refusals(lib):
    layer, f8 = fake((2, 8, 16, 4, 64), torch.bfloat16), fake((2, 8, 16, 4, 64), torch.uint8)
    bt = fake((8,), torch.int32, ptr=0x20000000)
    k, v = fake((10, 4, 64), torch.bfloat16, ptr=0x30000000), fake((10, 4, 64), torch.bfloat16, ptr=0x38000000)
    q, out = fake((10, 8, 64), torch.bfloat16, ptr=0x40000000), fake((10, 8, 64), torch.bfloat16, ptr=0x48000000)
    ok = (0, 0, 10, 100, 0)

    def run(lay=layer, pf=0, bt_=bt, k_=k, v_=v, s=(ok,), pos=None, ro=rope(), m=1.0, q_=None, o=None, ks=None, vs=None):
        a = np.array(s, np.int64).reshape(-1, 5)
        st = lib.daric_append_tokens(ref(lay), pf, ref(bt_), ref(k_), ref(v_), a.ctypes.data, len(a), ref(pos), ref(ro), m,
                                     ref(q_), ref(o), ref(ks), ref(vs), ctypes.c_uint64(0))
        assert st != 0
        return lib.daric_last_error().decode()

    assert "unsupported KV cache dtype" in run(lay=fake((2, 8, 16, 4, 64), torch.float32))
    assert "Unsupported KV cache rank" in run(lay=fake((8, 64), torch.bfloat16))
    assert "must not be empty" in run(lay=fake((2, 0, 16, 4, 64), torch.bfloat16))
    assert "head_dim from 2 on" in run(lay=fake((2, 8, 16, 4, 1), torch.bfloat16))
    assert "block_table must be a 1-D contiguous int32" in run(bt_=fake((8,), torch.int64))
    assert "k must have the cache's element type" in run(k_=fake((10, 4, 64), torch.float16))
    assert "k must have the cache's element type" in run(k_=fake((10, 4, 64), torch.float32))
    assert "k must be [T, 4, 64] rows" in run(k_=fake((10, 8, 64), torch.bfloat16))
    assert "k must be [T, 4, 64] rows" in run(k_=fake((10, 4, 32), torch.bfloat16))
    assert "v must be [T, 4, 64] rows" in run(v_=fake((9, 4, 64), torch.bfloat16))
    assert "v must be [T, 4, 64] rows" in run(lay=f8, v_=fake((10, 4, 64), torch.float16))
    assert "v must not be null" in run(v_=None)
    assert "v must be None" in run(lay=fake((8, 16, 64), torch.bfloat16), pf=1, k_=fake((10, 1, 64), torch.bfloat16),
                                   v_=fake((10, 1, 64), torch.bfloat16))
    assert "negative field of sequence 1" in run(s=((0, 0, 1, 4, 0), (0, 1, 1, -4, 50)))
    assert "rows exceed k" in run(s=((0, 5, 6, 4, 0),))
    assert "is too long" in run(s=((0, 0, 1, 2 ** 31, 0),)) and "is too long" in run(s=((0, 0, 1, 2 ** 62, 0),))
    assert "row 4 is in two sequences" in run(s=((0, 4, 2, 4, 50), (0, 0, 5, 4, 0)))
    assert "reaches past the end of block_table" in run(s=((2, 0, 10, 100, 0),))
    assert "reaches past the end of block_table" in run(s=((2 ** 62, 0, 1, 0, 0),))
    assert "positions must be" in run(pos=fake((9,), torch.int64))
    assert "no greater than head_dim" in run(ro=rope(66))
    assert "attention_scale must be finite" in run(m=math.nan)
    assert "q needs inv_freq" in run(ro=None, q_=q, o=out)
    assert "q must be [T, Hq, 64] rows" in run(q_=fake((10, 8, 32), torch.bfloat16), o=out)
    assert "q must be [T, Hq, 64] rows" in run(q_=fake((10, 8, 64), torch.float16), o=out)
    assert "q_out must not be null" in run(q_=q)
    assert "q_out must be q itself or" in run(q_=q, o=fake((10, 8, 64), torch.bfloat16, strides=(1024, 64, 1)))
    assert "k_scale applies to fp8" in run(ks=fake((4,), torch.float32)) and "v_scale applies to fp8" in run(vs=fake((4,), torch.float32))
    assert "k_scale must be a contiguous float32 [H]" in run(lay=f8, ks=fake((5,), torch.float32))
    # written memory that the call reads or writes elsewhere
    assert "the layer must not overlap k" in run(k_=fake((10, 4, 64), torch.bfloat16, ptr=0x10000100))
    assert "the layer must not overlap v" in run(v_=fake((10, 4, 64), torch.bfloat16, ptr=0x10000100))
    assert "the layer must not overlap block_table" in run(bt_=fake((8,), torch.int32, ptr=0x10000100))
    assert "the layer must not overlap q_out" in run(q_=q, o=fake((10, 8, 64), torch.bfloat16, ptr=0x10000100))
    assert "q_out must not overlap q" in run(q_=q, o=fake((10, 8, 64), torch.bfloat16, ptr=0x40000080))
    assert "q_out must not overlap k" in run(q_=q, o=fake((10, 8, 64), torch.bfloat16, ptr=0x30000080))
    assert "q_out must not overlap positions" in run(q_=q, o=out, pos=fake((10,), torch.int64, ptr=0x48000010))
    # q in place in a joint projection is apart from k and v beside it, not from what overlaps it
    joint = [fake((10, n, 64), torch.bfloat16, ptr=0x50000000 + 128 * at, strides=(1024, 64, 1)) for n, at in ((8, 0), (4, 8), (4, 12))]
    a = np.array([(0, 0, 0, 100, 0)], np.int64)
    assert lib.daric_append_tokens(r(layer), 0, r(bt), r(joint[1]), r(joint[2]), a.ctypes.data, 1, None, r(rope()), 1.0,
                                   r(joint[0]), r(joint[0]), None, None, ctypes.c_uint64(0)) == 0      # no rows: no device call
    over = fake((10, 4, 64), torch.bfloat16, ptr=0x50000000 + 128 * 7, strides=(1024, 64, 1))
    assert "q_out must not overlap k" in run(k_=over, v_=joint[2], q_=joint[0], o=joint[0])
    wraps = fake((10, 4, 64), torch.bfloat16, ptr=0x50000000 + 128 * 14, strides=(1024, 64, 1))
    assert "q_out must not overlap v" in run(k_=joint[1], v_=wraps, q_=joint[0], o=joint[0])


def test_optional_tensors_without_dimensions_or_values_are_there(lib):
    """A tensor of no dimensions, or of no values, is refused where one may be left out: it was
    asked for, and is not what the call takes."""
    layer, bt = fake((2, 8, 16, 4, 64), torch.uint8), fake((8,), torch.int32, ptr=0x20000000)
    k, v = fake((10, 4, 64), torch.bfloat16, ptr=0x30000000), fake((10, 4, 64), torch.bfloat16, ptr=0x38000000)
    a = np.array([(0, 0, 0, 100, 0)], np.int64)               # no rows: a call that is accepted ends before the device

    def run(lay=layer, k_=k, v_=v, q=None, ks=None, vs=None, ro=rope(), pf=0):
        if lib.daric_append_tokens(r(lay), pf, r(bt), r(k_), ref(v_), a.ctypes.data, 1, None, ref(ro), 1.0, ref(q), ref(q), ref(ks),
                                   ref(vs), ctypes.c_uint64(0)) == 0:
            return "taken"
        return lib.daric_last_error().decode()

    def none(dtype):
        t = fake((0,), dtype)
        t.data = None
        return t

    assert run() == "taken"
    point = fake((), torch.bfloat16, ptr=0x40000000)
    assert "q must be [T, H, D]" in run(q=point) and "q needs inv_freq" in run(q=point, ro=None)
    assert "k_scale must be a contiguous" in run(ks=none(torch.float32)) and "v_scale must be a contiguous" in run(vs=none(torch.float32))
    assert "v must be None" in run(lay=fake((8, 16, 64), torch.uint8), pf=1, k_=fake((10, 1, 64), torch.bfloat16), v_=none(torch.bfloat16))
    x, sc = fake((0, 4, 1000), torch.bfloat16, ptr=0x30000000), fake((0, 4), torch.float32, ptr=0x40000000)
    outs = [fake((0, 6), t, ptr=0x50000000) for t in (torch.float32, torch.int32, torch.int32)]
    choose = lambda e: lib.daric_select_beams(r(x), r(sc), ref(e), 2, r(outs[0]), r(outs[1]), r(outs[2]), None, 0, ctypes.c_uint64(0))
    assert choose(None) == 0 and choose(fake((0, 4), torch.uint8)) == 0
    assert choose(fake((), torch.uint8, ptr=0x53000000)) != 0 and "ended must be" in lib.daric_last_error().decode()


def test_tensors_without_memory_are_refused(lib):
    """Such as a traced program's, whose address is null: no kernel is given one."""
    def run(call, tensors, name):
        args = {k: (fake(*t, ptr=0x10000000 * (i + 1)) if t is not None else None) for i, (k, t) in enumerate(tensors.items())}
        args[name].data = None
        assert call(**{k: ref(t) for k, t in args.items()}) != 0
        assert "has no memory" in lib.daric_last_error().decode(), (name, lib.daric_last_error())

    st, a = ctypes.c_uint64(0), np.array([(0, 0, 10, 100, 0)], np.int64)
    bf, f32, i32 = torch.bfloat16, torch.float32, torch.int32
    rows = lambda x, p, o: lib.daric_rotate_rows(x, p, r(rope()), 1.0, o, st)
    for name in "xpo":
        run(rows, dict(x=((10, 8, 64), bf), p=((10,), torch.int64), o=((10, 8, 64), bf)), name)
    append = lambda l, b, k, v, p, q, o, s, z: lib.daric_append_tokens(l, 0, b, k, v, a.ctypes.data, 1, p, r(rope()), 1.0, q, o, s, z, st)
    for name in "lbkvpqosz":
        run(append, dict(l=((2, 8, 16, 4, 64), torch.uint8), b=((8,), i32), k=((10, 4, 64), bf), v=((10, 4, 64), bf), p=((10,), torch.int64),
                         q=((10, 8, 64), bf), o=((10, 8, 64), bf), s=((4,), f32), z=((4,), f32)), name)
    choose = lambda x, s, e, o, p, t: lib.daric_select_beams(x, s, e, 2, o, p, t, 0x70000000, 2 ** 20, st)
    for name in "xseopt":
        run(choose, dict(x=((2, 4, 1000), bf), s=((2, 4), f32), e=((2, 4), torch.uint8), o=((2, 6), f32), p=((2, 6), i32), t=((2, 6), i32)), name)
    beams = np.array([(0, 10, 4, 100)], np.int64)
    move = lambda l, b, p: lib.daric_reorder_beams(ctypes.cast(l, ctypes.POINTER(_lib.DaricTensor)), 1, 0, b, p, beams.ctypes.data, 1, st)
    for name in "lbp":
        run(move, dict(l=((2, 8, 16, 4, 64), bf), b=((40,), i32), p=((1, 4), i32)), name)


def test_selection_refusals(lib):
    x = fake((2, 4, 1000), torch.bfloat16, ptr=0x30000000)
    sc, out = fake((2, 4), torch.float32, ptr=0x40000000), fake((2, 6), torch.float32, ptr=0x50000000)
    par, tok = fake((2, 6), torch.int32, ptr=0x51000000), fake((2, 6), torch.int32, ptr=0x52000000)
    end = fake((2, 4), torch.uint8, ptr=0x53000000)

    def run(x_=x, sc_=sc, end_=None, et=2, out_=out, par_=par, tok_=tok, work=0x60000000, size=None):
        need = ctypes.c_int64(0)
        if size is None and lib.daric_select_workspace(ref(x_), par_.sizes[1], r(need)) != 0:
            return lib.daric_last_error().decode()
        st = lib.daric_select_beams(ref(x_), ref(sc_), ref(end_), et, ref(out_), ref(par_), ref(tok_), work,
                                    need.value if size is None else size, ctypes.c_uint64(0))
        assert st != 0
        return lib.daric_last_error().decode()

    assert "bfloat16, float16 or float32" in run(x_=fake((2, 4, 1000), torch.uint8))
    assert "must be [requests, beams, vocabulary]" in run(x_=fake((8, 1000), torch.bfloat16))
    assert "must be [requests, beams, vocabulary]" in run(x_=fake((2, 4, 1000), torch.bfloat16, strides=(1, 2, 8)))
    assert "must be [requests, beams, vocabulary]" in run(x_=fake((2, 4, 1000), torch.bfloat16, strides=(-4000, 1000, 1)))
    assert "must be [requests, beams, vocabulary]" in run(x_=fake((2, 4, 0), torch.bfloat16))
    assert "logits must be on CUDA" in run(x_=fake((2, 4, 1000), torch.bfloat16, device=-1))
    assert "up to 64 beams" in run(x_=fake((2, 65, 1000), torch.bfloat16))
    for k in (0, 65):
        wide = [fake((2, k), t, ptr=0x55000000) for t in (torch.float32, torch.int32, torch.int32)]
        assert "1 to 64 candidates" in run(out_=wide[0], par_=wide[1], tok_=wide[2])
    assert "vocabulary is too large" in run(x_=fake((2, 64, 2 ** 24), torch.bfloat16))
    assert "too many rows" in run(x_=fake((2 ** 24, 4, 100000), torch.bfloat16))
    assert "too many rows" in run(x_=fake((2 ** 62, 4, 8), torch.bfloat16, strides=(0, 8, 1)))
    assert "scores must be" in run(sc_=fake((2, 3), torch.float32)) and "scores must be" in run(sc_=fake((2, 4), torch.float16))
    assert "ended must be" in run(end_=fake((2, 4), torch.int32)) and "ended must be" in run(end_=fake((4,), torch.uint8))
    assert "end_token must be in the vocabulary" in run(end_=end, et=1000)
    assert "end_token must be in the vocabulary" in run(end_=end, et=-1)
    assert "out_scores must be" in run(out_=fake((2, 5), torch.float32))
    assert "tokens must be" in run(tok_=fake((2, 6), torch.int64))
    assert "workspace must be 16-byte aligned" in run(work=None) and "workspace must be 16-byte aligned" in run(work=0x60000004)
    assert "workspace must be 16-byte aligned" in run(size=16)
    assert "parents must not overlap tokens" in run(tok_=fake((2, 6), torch.int32, ptr=0x51000010))
    assert "out_scores must not overlap scores" in run(out_=fake((2, 6), torch.float32, ptr=0x40000010))
    assert "workspace must not overlap logits" in run(work=0x30000010)
    none = [fake((0, 6), t) for t in (torch.float32, torch.int32, torch.int32)]
    assert lib.daric_select_beams(r(fake((0, 4, 10), torch.float32)), r(fake((0, 4), torch.float32)), None, 0, r(none[0]),
                                  r(none[1]), r(none[2]), None, 0, ctypes.c_uint64(0)) == 0


def test_selection_of_as_many_requests_as_a_launch_holds(lib):
    """2^23 workgroups of 512 lanes are 2^32 lanes, one launch too large."""
    need = ctypes.c_int64(0)
    for B, fits in ((2 ** 23 - 1, True), (2 ** 23, False)):
        x = fake((B, 1, 8), torch.bfloat16, strides=(0, 8, 1))
        assert (lib.daric_select_workspace(r(x), 1, r(need)) == 0) is fits
    assert "too many rows" in lib.daric_last_error().decode()
    assert need.value == (2 ** 23 - 1) * 16               # a candidate, a maximum and a sum each


def test_reorder_refusals(lib):
    layers = (_lib.DaricTensor * 2)(*[fake((2, 8, 16, 4, 64), torch.bfloat16, ptr=0x10000000 * (i + 1)) for i in range(2)])
    bt = fake((40,), torch.int32, ptr=0x30000000)
    par = fake((1, 4), torch.int32, ptr=0x40000000)

    def run(s=((0, 10, 4, 100),), lay=layers, bt_=bt, par_=par, pf=0, n=None):
        a = np.array(s, np.int64).reshape(-1, 4)
        st = lib.daric_reorder_beams(lay, 2, pf, r(bt_), ref(par_), a.ctypes.data, len(a), ctypes.c_uint64(0))
        assert st != 0
        return lib.daric_last_error().decode()

    assert "negative field of request 0" in run(s=((0, 10, 4, -1),))
    assert "up to 32 beams" in run(s=((0, 10, 33, 5),))
    assert "more beams than parents has columns" in run(s=((0, 10, 5, 5),))
    assert "is too long" in run(s=((0, 10, 4, 2 ** 31),))
    assert "block lists of its beams overlap" in run(s=((0, 6, 4, 100),))
    assert "reaches past the end of block_table" in run(s=((5, 10, 4, 100),))
    assert "reaches past the end of block_table" in run(s=((0, 2 ** 62, 4, 100),))
    assert "reaches past the end of block_table" in run(s=((2 ** 62, 10, 4, 100),))
    assert "reaches past the end of block_table" in run(s=((2 ** 63 - 1, 2 ** 31, 2, 2 ** 31 - 2000),))
    two = fake((2, 4), torch.int32, ptr=0x40000000)
    assert "block list 20 is in two sequences" in run(s=((0, 10, 3, 40), (20, 10, 2, 30)), par_=two)
    assert "parents must be" in run(par_=two) and "parents must be" in run(par_=fake((1, 4), torch.int64))
    assert "parents must be" in run(par_=fake((1, 4), torch.int32, device=1)) and "parents must be" in run(par_=fake((4,), torch.int32))
    assert "parents must be" in run(par_=fake((1, 4), torch.int32, strides=(4, 2)))
    assert "block_table must be a 1-D contiguous int32" in run(bt_=fake((40,), torch.int64))
    assert "block_table must not overlap parents" in run(par_=fake((1, 4), torch.int32, ptr=0x30000010))
    assert "a layer must not overlap block_table" in run(bt_=fake((40,), torch.int32, ptr=0x10000010))
    twice = (_lib.DaricTensor * 2)(layers[0], layers[0])
    assert "a layer is given twice" in run(lay=twice)
    other = (_lib.DaricTensor * 2)(layers[0], fake((2, 8, 16, 4, 32), torch.bfloat16))
    assert "must share shape" in run(lay=other)
    # nothing to move: no beams, one beam, no tokens
    for s in ((), ((0, 10, 0, 100),), ((0, 10, 1, 100),), ((0, 10, 4, 0),)):
        a = np.array(s, np.int64).reshape(-1, 4)
        p = fake((len(a), 4), torch.int32, ptr=0x40000000)
        assert lib.daric_reorder_beams(layers, 2, 0, r(bt), r(p), a.ctypes.data, len(a), ctypes.c_uint64(0)) == 0


# ------------------------------------------------------------ the Python layer
def test_views_of_tensors_are_their_attributes():
    """Through torch's own function and one by one: the same bytes."""
    base = torch.zeros(4, 40, 2, 16)
    ts = [base, None, base[:, ::2, 1:, 3], base.permute(2, 0, 3, 1), base[:0], torch.zeros(()), torch.zeros(3, 3, requires_grad=True).t(),
          base[:1].expand(5, 40, 2, 16)] + [torch.zeros(1, 3, 1, dtype=t)[:, 1:] for t in (*_lib.DTYPE_CODES, torch.bool, torch.float64)]
    for some in (ts[:8], ts[8:], [None] * 3, []):
        at, arr = _lib.views(*some)
        assert len(at) == len(some)
        for i, (a, t) in enumerate(zip(at, some)):
            assert (a is None) == (t is None)
            if t is not None:
                assert a == ctypes.addressof(arr[i]) and bytes(arr[i]) == _lib.packed(t), (t.dtype, t.shape, t.stride())
    slow = _lib._Views()
    assert slow.fill is not None or not hasattr(torch.Tensor, "__dlpack_c_exchange_api__")
    slow.fill = None
    one = [t for t in ts if t is not None]
    assert bytes(slow.of(one)) == bytes(_lib.layer_views(one))
    for bad in (3, "x", np.zeros(3)):
        with pytest.raises(Exception):
            _lib.views(torch.zeros(3), bad)
    with pytest.raises(RuntimeError, match="rank"):
        _lib.views(torch.zeros([1] * 9))


def test_views_without_the_exchange_tables_function(monkeypatch):
    """An exchange table that leaves the function out, or of another version, is not called."""
    if not hasattr(torch.Tensor, "__dlpack_c_exchange_api__"):
        pytest.skip("this torch has no exchange table")
    name, c = b"dlpack_exchange_api", ctypes.pythonapi
    get = ctypes.PYFUNCTYPE(ctypes.c_void_p, ctypes.py_object, ctypes.c_char_p)(("PyCapsule_GetPointer", c))
    new = ctypes.PYFUNCTYPE(ctypes.py_object, ctypes.c_void_p, ctypes.c_char_p, ctypes.c_void_p)(("PyCapsule_New", c))
    real = ctypes.string_at(get(torch.Tensor.__dlpack_c_exchange_api__, name), 48)
    t = torch.zeros(2, 3)
    for at, number, fits in ((40, 0, False), (0, 2, False), (40, int.from_bytes(real[40:], "little"), True)):
        table = ctypes.create_string_buffer(real, 48)
        ctypes.c_uint64.from_buffer(table, at).value = number
        monkeypatch.setattr(torch.Tensor, "__dlpack_c_exchange_api__", new(ctypes.addressof(table), name, None))
        views = _lib._Views()
        assert (views.fill is not None) is fits
        assert bytes(views.of([t])) == _lib.packed(t)


def test_rows_of_ints():
    take = lambda e: cache_ops._rows_of_ints(e, (5, 4), "refused")
    def values(e):
        at, n, keep = take(e)
        if isinstance(at, bytes):
            return np.frombuffer(at, np.int64).reshape(n, 5).tolist()
        return keep.tolist() if n else []
    assert values([(1, 2, 3, 4), (5, 6, 7, 2 ** 62)]) == [[1, 2, 3, 4, 0], [5, 6, 7, 2 ** 62, 0]]
    assert values([(1, 2, 3, 4, 5)] * 2000) == [[1, 2, 3, 4, 5]] * 2000
    assert values([[1, 2, 3, 4]]) == values(np.array([[1, 2, 3, 4]])) == values(((1, 2, 3, np.int64(4)),)) == [[1, 2, 3, 4, 0]]
    assert values([]) == values(()) == []
    for bad in ([(1, 2, 3)], [(1, 2, 3, 4.0)], [(1, 2, 3, 4), (1, 2, 3)], [(1, 2, 3, "4")], [1, 2], [(1, 2, 3, 4), (1, 2, 3, 4, 5)], [None]):
        with pytest.raises((ValueError, TypeError)):
            take(bad)


def test_python_refusals():
    x = torch.zeros(2, 2, 8, dtype=torch.bfloat16)
    f, p = torch.ones(4), torch.zeros(2, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="inv_freq must be a float32 device tensor"):
        cache_ops.rotate_rows(x, p, f, 8)
    layer, bt = torch.zeros(2, 3, 4, 2, 8, dtype=torch.bfloat16), torch.ones(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="sequences must be"):
        cache_ops.append_tokens(layer, False, bt, x, x, [(0, 0)])
    with pytest.raises(RuntimeError, match="must be on CUDA"):
        cache_ops.append_tokens(layer, False, bt, x, x, [(0, 0, 2, 0)])
    with pytest.raises(RuntimeError, match="q_out needs q"):
        cache_ops.append_tokens(layer, False, bt, x, x, [(0, 0, 2, 0)], q_out=x)
    with pytest.raises(RuntimeError, match="logits must be on CUDA"):
        cache_ops.select_beams(torch.zeros(1, 2, 8), torch.zeros(1, 2))
    with pytest.raises(ValueError, match="beams must be"):
        cache_ops.reorder_beams([layer], False, bt, torch.zeros(1, 2, dtype=torch.int32), [(0, 1, 2)])
    with pytest.raises(RuntimeError, match="must be on CUDA"):
        cache_ops.reorder_beams([layer], False, bt, torch.zeros(1, 2, dtype=torch.int32), [(0, 1, 2, 1)])
    g = torch.zeros(2, 2, 8, requires_grad=True)
    for call in (lambda: cache_ops.rotate_rows(g, p, f, 8), lambda: cache_ops.append_tokens(layer, False, bt, g, x, [(0, 0, 2, 0)]),
                 lambda: cache_ops.select_beams(g, torch.zeros(2, 2))):
        with pytest.raises(RuntimeError, match="has no backward pass"):
            call()


def test_forward_mode_tangents_are_refused():
    """By every call that refuses a gradient; outside of a dual level nothing is asked."""
    x = torch.zeros(2, 2, 8, dtype=torch.bfloat16)
    f, p, bt = torch.ones(4), torch.zeros(2, dtype=torch.int64), torch.ones(2, dtype=torch.int32)
    layer, w = torch.zeros(2, 3, 4, 2, 8, dtype=torch.bfloat16), torch.zeros(1, 2, 8)
    seqs = [(0, 0, 2, 0)]
    with torch.autograd.forward_ad.dual_level():
        dual = lambda t: torch.autograd.forward_ad.make_dual(t, torch.ones_like(t))
        calls = [lambda: cache_ops.rotate_rows(dual(x), p, f, 8), lambda: cache_ops.rotate_rows(x, p, dual(f), 8),
                 lambda: cache_ops.rotate_rows(x, p, f, 8, out=dual(x)),
                 lambda: cache_ops.append_tokens(layer, False, bt, dual(x), x, seqs), lambda: cache_ops.append_tokens(layer, False, bt, x, dual(x), seqs),
                 lambda: cache_ops.append_tokens(dual(layer), False, bt, x, x, seqs), lambda: cache_ops.append_tokens(layer, False, bt, x, x, seqs, q=dual(x)),
                 lambda: cache_ops.select_beams(dual(w), torch.zeros(1, 2)), lambda: cache_ops.select_beams(w, dual(torch.zeros(1, 2))),
                 lambda: cache_ops.reorder_beams([layer, dual(layer)], False, bt, torch.zeros(1, 2, dtype=torch.int32), [(0, 1, 2, 1)]),
                 lambda: cache_ops.attend_pages(layer, False, bt, dual(x), seqs), lambda: cache_ops.weigh_tokens(layer, False, bt, dual(x), w[0, 0], seqs),
                 lambda: cache_ops.evict_tokens([dual(layer)], False, bt, w, [(0, 0, 1, 1, 0, 0)])]
        for call in calls:
            for mode in (torch.enable_grad, torch.no_grad):        # tangents do not heed no_grad
                with mode(), pytest.raises(RuntimeError, match="forward-mode tangents"):
                    call()
        with pytest.raises(RuntimeError, match="must be on CUDA"):  # primals pass on to the checks behind
            cache_ops.append_tokens(layer, False, bt, x, x, seqs)
        with pytest.raises(RuntimeError, match="must be on CUDA"):
            cache_ops.reorder_beams([layer], False, bt, torch.zeros(1, 2, dtype=torch.int32), [(0, 1, 2, 1)])
