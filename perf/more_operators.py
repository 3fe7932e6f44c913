"""A decoding loop's work around attention on the paged cache: rotary positions of
new rows, their way into the pages, the choice of beam search and the reordering
of its paged states, over the range of sizes, layouts and data types that a
serving program meets.

A case is a dict of plain values. `rows` and `ctx` list, as text, the new rows of a
call's sequences and the tokens that stand in the cache before them; `tokens` the
length of each request's beams. Page ids are a random choice of the pool's blocks.

With `own` false every pass is computed from elementary torch operations in 32
bits, in 64 where a position's angle or the order of candidates is at stake; with
`own` true by the package's entry points.
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32, "e4m3": torch.float8_e4m3fn}
SIZES = {"bf16": 2, "fp16": 2, "fp32": 4, "e4m3": 1}
MAX_ARENAS = 32             # allocations that the layers of a cache share


def _text(values):
    return ",".join(str(int(n)) for n in values)


def _ints(text):
    return [int(n) for n in text.split(",")]


def _rotate(name, rows, heads=40, dim=128, rotary=128, neox=True, dtype="bf16", far=8192, factor=1.0, m=1.0, inside=0):
    """far: positions below it; factor, m: the frequencies' and the table's scale
    of a long-context model; inside: heads that stand behind these in a token's row
    (V of a joint projection)."""
    return dict(name=name, op="rotate", rows=rows, heads=heads, dim=dim, rotary=rotary, neox=neox, dtype=dtype,
                far=far, factor=factor, m=m, inside=inside)


def _append(name, ctx, rows, heads=32, kv=8, dim=128, rotary=128, neox=True, page=16, dtype="bf16", qtype="bf16",
            layout="nhd", shift=0, factor=1.0, m=1.0):
    """shift: positions run ahead of the slots by it (as after an eviction), 0: they
    are the slots."""
    return dict(name=name, op="append", ctx=_text(ctx), rows=_text(rows), heads=heads, kv=kv, dim=dim, rotary=rotary,
                neox=neox, page=page, dtype=dtype, qtype=qtype, layout=layout, shift=shift, factor=factor, m=m)


def _select(name, requests, beams, vocab, k, dtype="bf16", ended=0.0, first=0.0):
    """k candidates of every request; ended: share of beams that are at their end;
    first: share of requests at their first step, with one live beam."""
    return dict(name=name, op="select", requests=requests, beams=beams, vocab=vocab, k=k, dtype=dtype, ended=ended,
                first=first)


def _reorder(name, layers, tokens, beams, kv=8, dim=128, page=16, dtype="bf16", layout="nhd"):
    return dict(name=name, op="reorder", layers=layers, tokens=_text(tokens), beams=beams, kv=kv, dim=dim, page=page,
                dtype=dtype, layout=layout)


# A batch of requests as a serving loop holds them.
BATCH = [310, 555, 780, 901, 1024, 1187, 1350, 1499, 1600, 1777, 1801, 2048, 12, 1345, 471, 600,
         777, 950, 1100, 1333, 500, 750, 1001, 96, 444, 800, 120, 1555, 1000, 789, 1500, 191,
         64, 65, 1, 1999, 2000, 1023, 333, 911, 1212, 1313, 1414, 1515, 1616, 17, 18, 190]


def listed():
    return [
        # One request's next token, queries and keys together: latency.
        _rotate("rotate_one", 1),
        # A prompt's queries and keys where a joint projection left them, V behind.
        _rotate("rotate_prompt", 16384, inside=8, far=131072),
        # Odd sizes: interleaved pairs of part of the head, positions of a long-context
        # model with a scaled table.
        _rotate("rotate_odd", 2511, heads=25, dim=80, rotary=32, neox=False, dtype="fp16", far=1048576, factor=8.0, m=1.2),
        # The next token of one request: the smallest call of a decoding step.
        _append("append_one", [777], [1]),
        # A decoding step of a batch on an fp8 cache of Llama-3-70B's KV shape.
        _append("append_batch_fp8", BATCH, [1] * len(BATCH), heads=64, dtype="e4m3"),
        # Prompts behind reused prefixes at Llama-3-8B's KV shape.
        _append("append_prompts", [0, 2048, 512], [8192, 5000, 3111]),
        # Ragged rows after an eviction: head-major pages of 32, half of the head rotated.
        _append("append_odd", [5, 0, 1023, 64, 97], [700, 33, 1, 64, 1301], heads=20, kv=4, dim=80, rotary=40, page=32,
                dtype="fp16", qtype="fp16", layout="hnd", shift=5003),
        # One request of four beams: latency.
        _select("select_one", 1, 4, 128000, 8),
        # A batch of requests of eight beams, twice as many candidates as beams.
        _select("select_batch", 32, 8, 128000, 16, ended=0.05, first=0.1),
        # Odd sizes, logits in 32 bits, many beams at their end.
        _select("select_odd", 7, 5, 50021, 9, dtype="fp32", ended=0.3),
        # One request of four beams, 32 layers.
        _reorder("reorder_one", 32, [777], 4),
        # A batch of requests of eight beams on an fp8 cache of 80 layers.
        _reorder("reorder_batch_fp8", 80, [1500, 2047, 3001, 4095, 513, 610, 7321, 808], 8, dtype="e4m3"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotate", "append", "append", "select", "select", "reorder"])
    dim = rng.choice([64, 64, 80, 96, 128, 128, 128, 256])
    rotary = rng.choice([dim, dim, dim, dim // 2, dim // 4])
    neox = rng.random() < 0.7
    factor, m = rng.choice([(1.0, 1.0), (1.0, 1.0), (4.0, 1.0), (8.0, 1.2)])
    if op == "rotate":
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        heads = rng.choice([1, 4, 8, 20, 25, 40, 72])
        # below the largest listed call's bytes
        rows = _log(rng, 1, 1.6e8 / (heads * dim * SIZES[dtype]))
        c = _rotate("", rows, heads, dim, rotary, neox, dtype, rng.choice([512, 8192, 131072, 1048576]), factor, m,
                    rng.choice([0, 0, 1, 8]))
    elif op == "append":
        dtype = rng.choice(["bf16", "bf16", "fp16", "e4m3"])
        qtype = dtype if dtype != "e4m3" else rng.choice(["bf16", "bf16", "fp16"])
        kv, group = rng.choice([1, 2, 4, 8, 8]), rng.choice([1, 2, 4, 4, 5, 7, 8])
        n = rng.choice([1, 1, 3, 8, 40, 100])
        top = 1.9e8 / (kv * (group + 2) * dim * 2)
        one = rng.random() < 0.5
        big = _log(rng, 1, max(2, top / n))
        rows = [1 if one else max(1, int(big * rng.uniform(0.1, 1.0))) for _ in range(n)]
        ctx = [rng.choice([0, _log(rng, 1, 2000), _log(rng, 1, 2000)]) for _ in range(n)]
        c = _append("", ctx, rows, kv * group, kv, dim, rotary, neox, rng.choice([8, 16, 16, 32, 64]), dtype, qtype,
                    rng.choice(["nhd", "nhd", "hnd", "pf", "packed"]), rng.choice([0, 0, 100, 100000]), factor, m)
    elif op == "select":
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        beams = rng.choice([1, 2, 3, 4, 4, 5, 8, 16, 32])
        vocab = _log(rng, 100, 262144)
        requests = _log(rng, 1, max(1, min(64, 6.5e7 / (beams * vocab * SIZES[dtype]))))
        c = _select("", requests, beams, vocab, min(rng.choice([beams, 2 * beams, 1, 2 * beams]), 64), dtype,
                    rng.choice([0.0, 0.0, 0.1, 0.4]), rng.choice([0.0, 0.0, 0.2, 1.0]))
    else:
        dtype, kv, page = rng.choice(["bf16", "bf16", "fp16", "e4m3"]), rng.choice([1, 2, 4, 8, 8]), rng.choice([8, 16, 16, 32, 64])
        beams, n = rng.choice([2, 3, 4, 4, 8, 16, 32]), rng.choice([1, 1, 2, 5, 8])
        # a call's last pages, below the largest listed call's
        layers = _log(rng, 1, max(1, min(80, 1.6e8 / (n * beams * page * kv * dim * SIZES[dtype] * 2))))
        tokens = [_log(rng, 1, 8192) for _ in range(n)]
        c = _reorder("", layers, tokens, beams, kv, dim, page, dtype, rng.choice(["nhd", "nhd", "hnd", "pf", "packed"]))
    del c["name"]
    return c


# ------------------------------------------------------------------ inputs
def _page_first(case):
    return case["layout"] in ("pf", "packed")


def _lists(case):
    """Pages of each block list, and how many of them a request's beams share."""
    ps = case["page"]
    if case["op"] == "append":
        return [(-(-(c + r) // ps), 0) for c, r in zip(_ints(case["ctx"]), _ints(case["rows"]))]
    # beams share the prompt, the first half of the tokens
    return [(-(-n // ps), (n // 2) // ps) for n in _ints(case["tokens"])]


def _blocks(case):
    w = case.get("beams", 1)
    return sum(s + (n - s) * w for n, s in _lists(case)) * 9 // 8 + 9


def _cache(case, phys):
    """The cache tensor as vLLM hands it over (head-major pages keep their [2,
    blocks, page, heads, dim] shape and permuted strides)."""
    return phys.permute(0, 1, 3, 2, 4) if case["layout"] == "hnd" else phys


def _kv_rows(case, cache):
    """K and V as [blocks, page, heads, dim] views of the cache tensor."""
    lay, d = case["layout"], case["dim"]
    if lay in ("nhd", "hnd"):
        return cache[0], cache[1]
    if lay == "pf":
        return cache[:, 0], cache[:, 1]
    return cache[..., :d].permute(0, 2, 1, 3), cache[..., d:].permute(0, 2, 1, 3)


def _phys(case, gen):
    """One layer's memory, N(0,1) values."""
    nb, ps, h, d = _blocks(case), case["page"], case["kv"], case["dim"]
    shape = {"nhd": (2, nb, ps, h, d), "hnd": (2, nb, h, ps, d), "pf": (nb, 2, ps, h, d), "packed": (nb, h, ps, 2 * d)}
    x = torch.randn(shape[case["layout"]], generator=gen, device=DEV, dtype=torch.float16 if case["dtype"] == "fp16" else torch.bfloat16)
    return x.to(DTYPES[case["dtype"]])


def _frequencies(case):
    r = case["rotary"]
    f = 500000.0 ** (-torch.arange(0, r, 2, dtype=torch.float64) / r) / case["factor"]
    return f.float().to(DEV)


def _inputs_rows(case, s, gen):
    s["inv_freq"] = _frequencies(case)
    if case["op"] == "rotate":
        T, heads, dim = case["rows"], case["heads"], case["dim"]
        joint = torch.randn(T, heads + case["inside"], dim, generator=gen, device=DEV).to(DTYPES[case["dtype"]])
        s["x"] = joint[:, :heads]
        # a batch's rows: runs of consecutive positions
        start = torch.randint(0, case["far"], (-(-T // 512),), generator=gen, device=DEV)
        s["positions"] = (start.repeat_interleave(512)[:T] + torch.arange(T, device=DEV)) % case["far"]
        return
    ctx, rows = _ints(case["ctx"]), _ints(case["rows"])
    T, heads, kv, dim = sum(rows), case["heads"], case["kv"], case["dim"]
    joint = torch.randn(T, heads + 2 * kv, dim, generator=gen, device=DEV).to(DTYPES[case["qtype"]])
    s["q"], s["k"], s["v"] = joint[:, :heads], joint[:, heads: heads + kv], joint[:, heads + kv:]
    s["layer"] = _cache(case, _phys(case, gen))
    s["k_scale"] = s["v_scale"] = None
    if case["dtype"] == "e4m3":
        s["k_scale"] = torch.rand(kv, generator=gen, device=DEV) * 0.01 + 0.01
        s["v_scale"] = torch.rand(kv, generator=gen, device=DEV) * 0.01 + 0.01
    seqs, at, begin = [], 0, 0
    for c, r, (n, _) in zip(ctx, rows, _lists(case)):
        seqs.append((begin, at, r, c))
        at += r
        begin += n
    s["seqs"] = seqs
    slots = np.concatenate([np.arange(c, c + r) for c, r in zip(ctx, rows)])
    s["positions"] = torch.from_numpy(slots + case["shift"]).to(DEV) if case["shift"] else None
    # pages in the order of the block lists, any of the pool's but the null block
    ids = torch.randperm(_blocks(case) - 1, generator=torch.Generator().manual_seed(s["seed"] + 1))[:begin] + 1
    s["bt"] = ids.to(torch.int32).to(DEV)


def _inputs_beams(case, s, gen):
    rng = np.random.default_rng(s["seed"] + 2)
    W = case["beams"]
    if case["op"] == "select":
        B, V = case["requests"], case["vocab"]
        # logits as a model leaves them: a wide body, some likely tokens in each row, which
        # the beams of a request share in part
        x = torch.randn(B, W, V, generator=gen, device=DEV).mul_(2.0)
        likely = torch.randint(0, V, (B, 1, 24), generator=gen, device=DEV).expand(B, W, 24).contiguous()
        x.scatter_add_(2, likely, 6.0 + 2.0 * torch.randn(B, W, 24, generator=gen, device=DEV))
        s["logits"] = x.to(DTYPES[case["dtype"]])
        scores = -20.0 - 3.0 * rng.random((B, W)).cumsum(1)
        scores[rng.random(B) < case["first"], 1:] = -np.inf
        s["scores"] = torch.from_numpy(scores.astype(np.float32)).to(DEV)
        s["ended"] = torch.from_numpy(rng.random((B, W)) < case["ended"]).to(DEV) if case["ended"] else None
        s["end_token"] = 2
        return
    lists, nb = _lists(case), _blocks(case)
    free = iter((rng.permutation(nb - 1) + 1).tolist())
    table, beams = [], []
    for (n, shared), tokens in zip(lists, _ints(case["tokens"])):
        beams.append((len(table), n, W, tokens))
        prompt = [next(free) for _ in range(shared)]
        for _ in range(W):
            table += prompt + [next(free) for _ in range(n - shared)]
    s["beams"] = beams
    s["bt"] = torch.tensor(table, dtype=torch.int32, device=DEV)
    s["parents"] = torch.from_numpy(rng.integers(0, W, (len(beams), W)).astype(np.int32)).to(DEV)
    L = case["layers"]
    per = -(-L // MAX_ARENAS)
    s["arenas"] = [torch.stack([_phys(case, gen) for _ in range(min(per, L - i))]) for i in range(0, L, per)]
    s["layers"] = [_cache(case, p) for a in s["arenas"] for p in a]


def prepare(case, seed):
    s = dict(case=case, op=case["op"], seed=seed)
    gen = torch.Generator(device=DEV).manual_seed(seed)
    (_inputs_rows if case["op"] in ("rotate", "append") else _inputs_beams)(case, s, gen)
    if "layout" in case:
        s["page_first"] = _page_first(case)
    return s


# ------------------------------------------------------------- plain forms
def _rotated(s, x, positions):
    """Rows [T, heads, dim] rotated to their positions, in 32 bits."""
    r, m = s["case"]["rotary"], s["case"]["m"]
    angle = positions.double()[:, None] * s["inv_freq"].double()
    cos, sin = (angle.cos() * m).float()[:, None], (angle.sin() * m).float()[:, None]
    x = x.float()
    out = x.clone()
    if s["case"]["neox"]:
        a, b = x[..., : r // 2], x[..., r // 2: r]
        out[..., : r // 2] = a * cos - b * sin
        out[..., r // 2: r] = b * cos + a * sin
    else:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        out[..., 0:r:2] = a * cos - b * sin
        out[..., 1:r:2] = b * cos + a * sin
    return out


def _rotate_plain(s):
    return _rotated(s, s["x"], s["positions"]).to(s["x"].dtype)


def _append_plain(s):
    case, ps = s["case"], s["case"]["page"]
    token = torch.cat([torch.arange(c, c + r, device=DEV) for _, _, r, c in s["seqs"]])
    begin = torch.cat([torch.full((r,), b, device=DEV) for b, _, r, _ in s["seqs"]])
    page, slot = s["bt"][begin + token // ps].long(), token % ps
    positions = token if s["positions"] is None else s["positions"]
    new = (_rotated(s, s["k"], positions), s["v"].float())
    for rows, x, scale in zip(_kv_rows(case, s["layer"]), new, (s["k_scale"], s["v_scale"])):
        if scale is not None:
            x = (x / scale[None, :, None]).clamp_(-448, 448)
        rows[page, slot] = x.to(rows.dtype)
    return _rotated(s, s["q"], positions).to(s["q"].dtype), s["layer"]


def _select_plain(s):
    B, W, V = s["logits"].shape
    k = s["case"]["k"]
    x = s["logits"].double()
    top = x.amax(-1, keepdim=True)
    score = s["scores"].double()[..., None] + (x - top - (x - top).exp().sum(-1, keepdim=True).log())
    if s["ended"] is not None:
        only = torch.full((V,), -math.inf, device=DEV, dtype=torch.float64)
        only[s["end_token"]] = 0.0
        score = torch.where(s["ended"][..., None], s["scores"].double()[..., None] + only, score)
    best, at = score.view(B, W * V).sort(dim=-1, descending=True, stable=True)
    best, at = best[:, :k], at[:, :k]
    if best.shape[1] < k:
        best = torch.nn.functional.pad(best, (0, k - best.shape[1]), value=-math.inf)
        at = torch.nn.functional.pad(at, (0, k - at.shape[1]))
    none = best == -math.inf
    return (best.float(), torch.where(none, -1, at // V).to(torch.int32), torch.where(none, -1, at % V).to(torch.int32))


def _reorder_plain(s):
    case, ps = s["case"], s["case"]["page"]
    bt = s["bt"]
    src, dst, slots = [], [], []
    for (b, stride, w, n), parent in zip(s["beams"], s["parents"].long()):
        lists = bt[b: b + stride * w].view(w, stride)
        full = n // ps
        if n % ps:
            own_page = lists[:, full].long()
            slot = torch.arange(n % ps, device=DEV)
            src.append(own_page[parent].repeat_interleave(n % ps))
            dst.append(own_page.repeat_interleave(n % ps))
            slots.append(slot.repeat(w))
        lists[:, :full] = lists[parent, :full]
    if src:
        src, dst, slots = torch.cat(src), torch.cat(dst), torch.cat(slots)
        for layer in s["layers"]:
            for rows in _kv_rows(case, layer):
                rows[dst, slots] = rows[src, slots]
    return bt, s["arenas"]


# ------------------------------------------------------------------ passes
def run(s):
    if not own:
        return {"rotate": _rotate_plain, "append": _append_plain, "select": _select_plain, "reorder": _reorder_plain}[s["op"]](s)
    from daric_amd import cache_ops
    c = s["case"]
    if s["op"] == "rotate":
        return cache_ops.rotate_rows(s["x"], s["positions"], s["inv_freq"], c["rotary"], c["neox"], attention_scale=c["m"])
    if s["op"] == "append":
        q = cache_ops.append_tokens(s["layer"], s["page_first"], s["bt"], s["k"], s["v"], s["seqs"], s["inv_freq"],
                                    c["rotary"], c["neox"], positions=s["positions"], attention_scale=c["m"], q=s["q"],
                                    k_scale=s["k_scale"], v_scale=s["v_scale"])
        return q, s["layer"]
    if s["op"] == "select":
        return cache_ops.select_beams(s["logits"], s["scores"], c["k"], ended=s["ended"], end_token=s["end_token"])
    cache_ops.reorder_beams(s["layers"], s["page_first"], s["bt"], s["parents"], s["beams"])
    return s["bt"], s["arenas"]


def work(case):
    if case["op"] == "rotate":
        values = case["rows"] * case["heads"] * case["dim"]
        return {"bytes": 2 * values * SIZES[case["dtype"]] + 8 * case["rows"],
                "flops": 3 * case["rows"] * case["heads"] * case["rotary"]}
    if case["op"] == "append":
        T, heads, kv, dim = sum(_ints(case["rows"])), case["heads"], case["kv"], case["dim"]
        size, new = SIZES[case["dtype"]], SIZES[case["qtype"]]
        return {"bytes": T * dim * (2 * heads * new + 2 * kv * (new + size)) + (8 * T if case["shift"] else 0),
                "flops": 3 * T * (heads + kv) * case["rotary"]}
    if case["op"] == "select":
        B, W, k = case["requests"], case["beams"], case["k"]
        values = B * W * case["vocab"]
        return {"bytes": values * SIZES[case["dtype"]] + B * (4 * W + 12 * k), "flops": 2 * values}
    W, ps = case["beams"], case["page"]
    tokens = _ints(case["tokens"])
    row = case["layers"] * 2 * case["kv"] * case["dim"] * SIZES[case["dtype"]]
    # parents are any of the beams: how many are read, and how many beams move
    read, moved = W * (1 - (1 - 1 / W) ** W), W - 1
    return {"bytes": int(sum(n % ps for n in tokens) * row * (read + moved) + sum(n // ps for n in tokens) * 4 * (read + moved)),
            "flops": 0}


# --------------------------------------------------------- the definitions
def _exact_turn(case, x, positions):
    """The rows as complex numbers times m exp(i p f), in 64 bits."""
    r, f = case["rotary"], _frequencies(case).double()
    turn = torch.polar(torch.full((), case["m"], dtype=torch.float64, device=DEV), positions.double()[:, None] * f)[:, None]
    x = x.double()
    if case["neox"]:
        z = torch.complex(x[..., : r // 2].contiguous(), x[..., r // 2: r].contiguous()) * turn
        return torch.cat([z.real, z.imag, x[..., r:]], -1)
    z = torch.view_as_complex(x[..., :r].reshape(*x.shape[:-1], r // 2, 2).contiguous()) * turn
    return torch.cat([torch.view_as_real(z).flatten(-2), x[..., r:]], -1)


def _exact_select(s):
    B, W, V = s["logits"].shape
    k = s["case"]["k"]
    score = np.full((B, k), -np.inf)
    parent, token = np.full((B, k), -1, np.int64), np.full((B, k), -1, np.int64)
    for b in range(B):
        found = []
        for w in range(W):
            base = float(s["scores"][b, w])
            if s["ended"] is not None and bool(s["ended"][b, w]):
                found.append((-base, w, s["end_token"]))
                continue
            x = s["logits"][b, w].double().cpu().numpy()
            lse = x.max() + math.log(math.fsum(np.exp(x - x.max())))
            # a beam's k best, and all that are as good as the last of them
            near = np.flatnonzero(x >= np.partition(x, -min(k, V))[-min(k, V)])
            found += [(-(base + (x[v] - lse)), w, int(v)) for v in near]
        for i, (c, w, v) in enumerate(sorted(t for t in found if t[0] != math.inf)[:k]):
            score[b, i], parent[b, i], token[b, i] = -c, w, v
    return tuple(torch.from_numpy(x).to(DEV) for x in (score, parent, token))


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "rotate":
        return _exact_turn(case, s["x"], s["positions"])
    if s["op"] == "select":
        return _exact_select(s)
    if s["op"] == "append":
        layer = s["layer"].double()
        K, V = _kv_rows(case, layer)
        q = torch.empty(s["q"].shape, dtype=torch.float64, device=DEV)
        for b, at, r, c in s["seqs"]:
            rows = slice(at, at + r)
            p = torch.arange(c, c + r, device=DEV)
            where = p.cpu().numpy()
            pages = s["bt"][b:].cpu().numpy()[where // case["page"]]
            p = p + case["shift"]
            q[rows] = _exact_turn(case, s["q"][rows], p)
            for to, x, scale in ((K, _exact_turn(case, s["k"][rows], p), s["k_scale"]), (V, s["v"][rows].double(), s["v_scale"])):
                if scale is not None:
                    x = (x / scale.double()[:, None]).clamp(-448, 448)
                to[torch.from_numpy(pages).long().to(DEV), torch.from_numpy(where % case["page"]).to(DEV)] = x
        return q, layer
    bt = s["bt"].cpu().numpy()
    for (b, stride, w, n), parent in zip(s["beams"], s["parents"].cpu().numpy()):
        lists = bt[b: b + stride * w].reshape(w, stride)
        lists[:, : n // case["page"]] = lists[parent, : n // case["page"]]
    return torch.from_numpy(bt.astype(np.int64)).to(DEV), [None] * len(s["arenas"])
