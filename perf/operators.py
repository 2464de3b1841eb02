"""The serving operators on inputs of real use: what they compute, in plain form, and the calls that a user makes.

Three operators work between the projections of a (pruned) transformer whose
products run as ``SpMMPlan.spmm``:

  append    keys and values of new tokens into a paged cache, with the rotary
            position rotation of keys and queries on the way
  attend    attention of one new token per sequence over that cache
  adapters  low-rank adapters of many requests beside a shared projection

``own`` false: ``run`` computes them in elementary torch operations in 32 bits;
true: through ``sparse_computation_b200``.  ``exact`` gives the same outputs
from the definitions in 64 bits.
"""
import math
import random

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
MAX_POSITION = 16384  # rows of the rotation tables in the append cases


# ------------------------------------------------------------------- cases --

def _append(tokens, seqs, q_heads, kv_heads, head_dim, rotary, pairs, types, page, features, context, name=None):
    """``tokens`` new tokens of ``seqs`` sequences that hold up to ``context`` tokens already."""
    case = dict(op="append", tokens=tokens, seqs=seqs, q_heads=q_heads, kv_heads=kv_heads, head_dim=head_dim,
                rotary=rotary, pairs=pairs, type=types[0], cache=types[1], page=page, features=features,
                context=context)
    return dict(case, name=name) if name else case


def _attend(seqs, shortest, longest, q_heads, kv_heads, head_dim, types, page, window, features, name=None):
    """One new token of ``seqs`` sequences with ``shortest`` to ``longest`` cached tokens each."""
    case = dict(op="attend", seqs=seqs, shortest=shortest, longest=longest, q_heads=q_heads, kv_heads=kv_heads,
                head_dim=head_dim, type=types[0], cache=types[1], page=page, window=window, features=features)
    return dict(case, name=name) if name else case


def _adapters(tokens, adapters, idle, features_in, features_out, rank_min, rank_max, types, runs, features, name=None):
    """``tokens`` columns; ``idle`` of them without an adapter, the others spread over ``adapters`` adapters,
    in runs (prompts) or mixed (one token per request)."""
    case = dict(op="adapters", tokens=tokens, adapters=adapters, idle=idle, features_in=features_in,
                features_out=features_out, rank_min=rank_min, rank_max=rank_max, type=types[0], weights=types[1],
                runs=runs, features=features)
    return dict(case, name=name) if name else case


def listed():
    return [
        # One decoding step of a few requests through the 512-wide transformer-base layers (8 heads of 64), all
        # fp32 and feature-major as the sparse products leave it: latency alone.
        _append(4, 4, 8, 8, 64, 64, False, ("f32", "f32"), 16, True, 512, "append step base 4"),
        # A step of 128 requests (the widest B of the layer stack) with grouped heads, fp32 activations into a
        # 16-bit cache.
        _append(128, 128, 32, 8, 128, 128, False, ("f32", "bf16"), 64, True, 300, "append step 128"),
        # Prompts of seven requests at once: odd token count, head size off the powers of two, a partial rotation in
        # neighbouring pairs, pages that end inside the prompts, 16-bit token-major activations.
        _append(4099, 7, 20, 4, 80, 32, True, ("bf16", "bf16"), 24, False, 100, "append prompts 4099"),
        # The smallest attention: four short requests, fp32 transformer-base heads.
        _attend(4, 1, 200, 8, 8, 64, ("f32", "f32"), 16, 0, True, "attend base 4"),
        # The layer stack's width of requests at the lengths that model translates, fp32 throughout.
        _attend(128, 16, 1024, 8, 8, 64, ("f32", "f32"), 16, 0, True, "attend base 128"),
        # A ragged serving batch with grouped heads, fp32 activations over a 16-bit cache.
        _attend(32, 100, 8192, 32, 8, 128, ("f32", "bf16"), 64, 0, True, "attend batch 32"),
        # Odd sizes: five query heads a group, a head size off the powers of two, a sliding window, pages of 48.
        _attend(61, 0, 6000, 25, 5, 80, ("f16", "f16"), 48, 1000, False, "attend window 61"),
        # One long document: all the parallelism has to come from its length.
        _attend(1, 131071, 131071, 32, 8, 128, ("bf16", "bf16"), 64, 0, False, "attend long 1"),
        # Four requests' adapters beside a 512 x 512 projection, fp32: latency alone.
        _adapters(4, 3, 1, 512, 512, 4, 8, ("f32", "f32"), False, True, "adapters base 4"),
        # 128 requests beside the 2048 x 512 projection, an adapter each but for some without one.
        _adapters(128, 100, 9, 512, 2048, 4, 64, ("f32", "bf16"), False, True, "adapters own 128"),
        # 96 requests that share 40 large adapters of ragged ranks, 16-bit token-major activations.
        _adapters(96, 40, 5, 4096, 4096, 8, 64, ("bf16", "bf16"), False, False, "adapters shared 96"),
        # Prompts of six requests, feature-major fp32 activations, an adapter each.
        _adapters(2049, 6, 100, 2048, 2048, 16, 64, ("f32", "f16"), True, True, "adapters prompts 2049"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attend", "adapters"])
    if op == "append":
        kv = rng.choice([1, 2, 4, 5, 8])
        cache = rng.choice(["f32", "bf16", "f16"])
        kind = "f32" if cache == "f32" else rng.choice(["f32", cache])
        dim = rng.choice([32, 64, 80, 96, 128])
        seqs = _log(rng, 1, 200)
        tokens = seqs if rng.random() < 0.5 else seqs + _log(rng, 8, 3500)
        return _append(tokens, seqs, kv * rng.choice([1, 2, 4, 5, 8]) if kv < 8 else kv * rng.choice([1, 4]), kv, dim,
                       rng.choice([dim, dim, dim // 2]), rng.random() < 0.4, (kind, cache),
                       rng.choice([1, 16, 24, 64, 128]), rng.random() < 0.5, _log(rng, 1, 400))
    if op == "attend":
        kv = rng.choice([1, 2, 5, 8])
        cache = rng.choice(["f32", "bf16", "f16"])
        kind = "f32" if cache == "f32" else rng.choice(["f32", cache])
        dim = rng.choice([32, 64, 80, 96, 128])
        seqs = _log(rng, 1, 128)
        most = max(8, min(65536, int(2.0e8 / (seqs * kv * dim * BYTES[cache]))))
        longest = _log(rng, 4, most)
        return _attend(seqs, rng.choice([0, 1, longest // 4, longest // 2]), longest, kv * rng.choice([1, 2, 4, 5, 8]), kv, dim, (kind, cache),
                       rng.choice([1, 16, 24, 64, 128]), rng.choice([0, 0, max(1, longest // 3)]), rng.random() < 0.5)
    weights = rng.choice(["f32", "bf16", "f16"])
    kind = "f32" if weights == "f32" else rng.choice(["f32", weights])
    runs = rng.random() < 0.4
    tokens = _log(rng, 64, 2048) if runs else _log(rng, 1, 160)
    low = rng.choice([1, 4, 8, 16])
    return _adapters(tokens, _log(rng, 1, 8 if runs else min(100, tokens)), rng.randint(0, tokens // 8),
                     rng.choice([512, 520, 1000, 2048]), rng.choice([512, 904, 2048]), low,
                     rng.choice([low, 16 if low < 16 else 24, 64]), (kind, weights), runs, rng.random() < 0.5)


# -------------------------------------------------- what a case fixes alone --

def _lengths(case):
    """The cached lengths of an attend case: the ends of the range and values between, spread over their logarithm."""
    n, lo, hi = case["seqs"], case["shortest"], case["longest"]
    rng = random.Random(n * 7919 + hi)
    inner = [int(math.exp(rng.uniform(math.log(max(1, lo)), math.log(max(1, hi))))) for _ in range(n)]
    return ([hi, lo] + inner)[:n]


def _spans(case):
    """(cached, new) tokens of each sequence of an append case."""
    rng = random.Random(case["tokens"] * 31 + case["seqs"])
    new = [1] * case["seqs"]
    spare = case["tokens"] - case["seqs"]
    cuts = sorted(rng.randint(0, spare) for _ in range(case["seqs"] - 1))
    for i, (a, b) in enumerate(zip([0] + cuts, cuts + [spare])):
        new[i] += b - a
    return [(rng.randint(0, case["context"]), n) for n in new]


def _ranks(case):
    rng = random.Random(case["adapters"] * 131 + case["rank_max"])
    return [rng.randint(case["rank_min"], case["rank_max"]) for _ in range(case["adapters"])]


def _seen(case):
    """Keys that each sequence of an attend case attends to."""
    w = case["window"]
    return [min(n, w) if w else n for n in _lengths(case)]


def _counts(case):
    """Tokens of each adapter."""
    busy = case["tokens"] - case["idle"]
    return [busy // case["adapters"] + (i < busy % case["adapters"]) for i in range(case["adapters"])]


def work(case):
    if case["op"] == "append":
        e, c, d = BYTES[case["type"]], BYTES[case["cache"]], case["head_dim"]
        row = case["q_heads"] * d * 2 * e + 2 * case["kv_heads"] * d * (e + c)
        return {"bytes": case["tokens"] * (row + case["rotary"] * 4 + 12),
                "flops": case["tokens"] * (case["q_heads"] + case["kv_heads"]) * case["rotary"] * 3}
    if case["op"] == "attend":
        e, c, d = BYTES[case["type"]], BYTES[case["cache"]], case["head_dim"]
        keys = sum(_seen(case))
        pages = sum(-(-n // case["page"]) for n in _seen(case))
        return {"bytes": keys * case["kv_heads"] * d * 2 * c + case["seqs"] * case["q_heads"] * (2 * d * e + 4)
                + 4 * pages + 4 * case["seqs"], "flops": 4 * keys * case["q_heads"] * d}
    e, c = BYTES[case["type"]], BYTES[case["weights"]]
    both = case["features_in"] + case["features_out"]
    used = [(r, n) for r, n in zip(_ranks(case), _counts(case)) if n]
    busy = case["tokens"] - case["idle"]
    return {"bytes": sum(r for r, _ in used) * both * c + busy * case["features_in"] * e
            + 2 * case["tokens"] * case["features_out"] * e + 4 * case["tokens"],
            "flops": sum(2 * r * n * both for r, n in used)}


# ------------------------------------------------------------------ inputs --

def _device():
    return torch.device("cuda" if torch.cuda.is_available() else "cpu")


def _normal(gen, shape, kind, scale=1.0):
    x = torch.randn(shape, generator=gen, device=gen.device, dtype=torch.float32)
    return (x * scale).to(TYPES[kind])


def _rows(gen, tokens, heads, dim, kind, features):
    """[tokens, heads, dim] activations; with ``features`` a view of the feature-major matrix that a product leaves."""
    if features:
        return _normal(gen, (heads * dim, tokens), kind).view(heads, dim, tokens).permute(2, 0, 1)
    return _normal(gen, (tokens, heads, dim), kind)


def _table(gen, case, pages_of):
    """A page table in which the pages of all sequences are scattered over the pool, and the pool's page count."""
    dev = gen.device
    total = sum(pages_of)
    pool = total + 8
    where = torch.randperm(pool, generator=gen, device=dev)[:total].to(torch.int32).cpu().numpy()
    table = np.zeros((len(pages_of), max(1, max(pages_of))), np.int32)
    table[np.arange(table.shape[1])[None, :] < np.array(pages_of)[:, None]] = where
    return torch.from_numpy(table).to(dev), pool


def prepare(case, seed):
    dev = _device()
    gen = torch.Generator(device=dev).manual_seed(seed)
    order = random.Random(seed)
    state = {"case": case}
    if case["op"] == "append":
        spans = _spans(case)
        order.shuffle(spans)
        h, d, page = case["kv_heads"], case["head_dim"], case["page"]
        state["table"], pool = _table(gen, case, [-(-(a + n) // page) for a, n in spans])
        state["k_pages"] = _normal(gen, (pool, h, page, d), case["cache"])
        state["v_pages"] = _normal(gen, (pool, h, page, d), case["cache"])
        state["q"] = _rows(gen, case["tokens"], case["q_heads"], d, case["type"], case["features"])
        state["k"] = _rows(gen, case["tokens"], h, d, case["type"], case["features"])
        state["v"] = _rows(gen, case["tokens"], h, d, case["type"], case["features"])
        ids = np.concatenate([np.full(n, i, np.int32) for i, (_, n) in enumerate(spans)])
        at = np.concatenate([np.arange(a, a + n, dtype=np.int32) for a, n in spans])
        state["ids"] = None if case["tokens"] == case["seqs"] else torch.from_numpy(ids).to(dev)
        state["positions"] = torch.from_numpy(at).to(dev)
        half = case["rotary"] // 2
        freq = 10000.0 ** (-torch.arange(half, device=dev, dtype=torch.float64) / half)
        angle = torch.arange(MAX_POSITION, device=dev, dtype=torch.float64)[:, None] * freq[None, :]
        state["cos"], state["sin"] = angle.cos().float(), angle.sin().float()
        if own:
            import sparse_computation_b200 as sc
            state["pages"] = sc.PagedKVCache(state["k_pages"], state["v_pages"])
            state["rope"] = sc.RotaryTable(state["cos"], state["sin"], interleaved=case["pairs"])
    elif case["op"] == "attend":
        lengths = _lengths(case)
        order.shuffle(lengths)
        h, d, page = case["kv_heads"], case["head_dim"], case["page"]
        state["table"], pool = _table(gen, case, [-(-n // page) for n in lengths])
        state["k_pages"] = _normal(gen, (pool, h, page, d), case["cache"], 1.5)
        state["v_pages"] = _normal(gen, (pool, h, page, d), case["cache"])
        state["q"] = _rows(gen, case["seqs"], case["q_heads"], d, case["type"], case["features"])
        state["lengths"] = torch.tensor(lengths, dtype=torch.int32, device=dev)
        if own:
            import sparse_computation_b200 as sc
            pages = sc.PagedKVCache(state["k_pages"], state["v_pages"])
            state["plan"] = sc.DecodeAttention(pages, case["q_heads"], case["seqs"], window=case["window"])
    else:
        n, k, m = case["tokens"], case["features_in"], case["features_out"]
        ranks = _ranks(case)
        state["down"] = [_normal(gen, (r, k), case["weights"], k ** -0.5) for r in ranks]
        state["up"] = [_normal(gen, (m, r), case["weights"], r ** -0.5) for r in ranks]
        state["scales"] = [order.choice([0.5, 1.0, 2.0]) for _ in ranks]
        ids = [-1] * case["idle"] + [i for i, c in enumerate(_counts(case)) for _ in range(c)]
        if not case["runs"]:
            order.shuffle(ids)
        state["ids"] = torch.tensor(ids, dtype=torch.int32, device=dev)
        shape = (lambda f: (f, n)) if case["features"] else (lambda f: (n, f))
        turn = (lambda x: x) if case["features"] else (lambda x: x.t())
        state["x"] = turn(_normal(gen, shape(k), case["type"]))
        state["base"] = turn(_normal(gen, shape(m), case["type"]))
        state["owner"] = torch.repeat_interleave(torch.arange(len(ranks), device=dev),
                                                 torch.tensor(ranks, device=dev))
        state["scale_of"] = torch.tensor(state["scales"], device=dev)[state["owner"]]
        if own:
            import sparse_computation_b200 as sc
            state["set"] = sc.LowRankAdapters(state["down"], state["up"], state["scales"])
    return state


# --------------------------------------------------------------------- run --

def _rotated(x, cos, sin, rotary, pairs):
    """x [tokens, heads, dim] fp32; cos and sin [tokens, rotary / 2]."""
    c, s = cos[:, None, :], sin[:, None, :]
    y = x.clone()
    if pairs:
        a, b = x[..., 0:rotary:2], x[..., 1:rotary:2]
        y[..., 0:rotary:2], y[..., 1:rotary:2] = a * c - b * s, b * c + a * s
    else:
        a, b = x[..., :rotary // 2], x[..., rotary // 2:rotary]
        y[..., :rotary // 2], y[..., rotary // 2:rotary] = a * c - b * s, b * c + a * s
    return y


def _plain_append(state):
    case, page = state["case"], state["case"]["page"]
    at = state["positions"].long()
    ids = torch.arange(len(at), device=at.device) if state["ids"] is None else state["ids"].long()
    where, slot = state["table"][ids, at // page].long(), at % page
    cos, sin = state["cos"][at], state["sin"][at]
    q = _rotated(state["q"].float(), cos, sin, case["rotary"], case["pairs"])
    k = _rotated(state["k"].float(), cos, sin, case["rotary"], case["pairs"])
    state["k_pages"][where, :, slot] = k.to(state["k_pages"].dtype)
    state["v_pages"][where, :, slot] = state["v"].float().to(state["v_pages"].dtype)
    return {"q": q.to(TYPES[case["type"]]), "k": state["k_pages"], "v": state["v_pages"]}


def _plain_attend(state):
    case = state["case"]
    page, h, d = case["page"], case["kv_heads"], case["head_dim"]
    n = max(1, case["longest"])
    j = torch.arange(n, device=state["q"].device)
    where, slot = state["table"][:, j // page].long(), (j % page)[None, :]
    k = state["k_pages"][where, :, slot].float()  # [seqs, n, kv heads, dim]
    v = state["v_pages"][where, :, slot].float()
    q = state["q"].float().reshape(case["seqs"], h, case["q_heads"] // h, d)
    z = torch.matmul(q, k.permute(0, 2, 3, 1)) * (1.0 / math.sqrt(d))
    length = state["lengths"].long()[:, None]
    seen = j[None, :] < length
    if case["window"]:
        seen = seen & (j[None, :] >= length - case["window"])
    z = torch.where(seen[:, None, None, :], z, float("-inf"))
    top = z.amax(-1, keepdim=True)
    top = torch.where(top == float("-inf"), 0.0, top)
    p = torch.exp(z - top)
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, v.permute(0, 2, 1, 3)) / torch.where(total == 0, 1.0, total)
    lse = (top + torch.log(total)).reshape(case["seqs"], case["q_heads"])
    return {"out": out.reshape(case["seqs"], case["q_heads"], d).to(TYPES[case["type"]]), "lse": lse}


def _plain_adapters(state):
    down = torch.cat(state["down"], 0).float()
    up = torch.cat(state["up"], 1).float()
    v = torch.matmul(down, state["x"].float()) * state["scale_of"][:, None]
    v = torch.where(state["owner"][:, None] == state["ids"][None, :], v, 0.0)
    return {"y": (state["base"].float() + torch.matmul(up, v)).to(TYPES[state["case"]["type"]])}


def run(state):
    case = state["case"]
    if not own:
        return {"append": _plain_append, "attend": _plain_attend, "adapters": _plain_adapters}[case["op"]](state)
    if case["op"] == "append":
        q = state["pages"].append(state["k"], state["v"], state["positions"], state["table"], seq_ids=state["ids"],
                                  rope=state["rope"], q=state["q"])
        return {"q": q, "k": state["k_pages"], "v": state["v_pages"]}
    if case["op"] == "attend":
        out = None
        if case["features"]:  # feature-major, as the next product wants it
            h, d, n = case["q_heads"], case["head_dim"], case["seqs"]
            out = torch.empty((h * d, n), dtype=state["q"].dtype, device=state["q"].device)
            out = out.view(h, d, n).permute(2, 0, 1)
        out, lse = state["plan"].attend(state["q"], state["table"], state["lengths"], out=out, return_lse=True)
        return {"out": out, "lse": lse}
    return {"y": state["set"].apply(state["x"], state["ids"], base=state["base"])}


# ------------------------------------------------------------------- exact --

def exact(case, seed):
    """The definitions in 64 bits, one sequence, token or adapter after the other."""
    state = prepare(case, seed)
    if case["op"] == "append":
        half, pairs = case["rotary"] // 2, case["pairs"]
        first = torch.arange(half, device=state["q"].device) * (2 if pairs else 1)
        second = first + (1 if pairs else half)
        at = state["positions"].long()
        angle = torch.complex(state["cos"].double(), state["sin"].double())[at].unsqueeze(1)

        def turned(x):
            y = x.double().clone(memory_format=torch.contiguous_format)
            z = torch.complex(y[:, :, first], y[:, :, second]) * angle
            y[:, :, first], y[:, :, second] = z.real, z.imag
            return y

        q, k, v = turned(state["q"]), turned(state["k"]), state["v"].double()
        spot = at.cpu().numpy()
        rows = np.arange(len(spot)) if state["ids"] is None else state["ids"].cpu().numpy()
        flat = state["table"].cpu().numpy()[rows, spot // case["page"]].astype(np.int64) * case["page"] + spot % case["page"]
        to = torch.from_numpy(flat).to(k.device)

        def filled(pool, new):
            by_slot = pool.double().transpose(1, 2).clone(memory_format=torch.contiguous_format)
            by_slot.view(-1, case["kv_heads"], case["head_dim"])[to] = new
            return by_slot.transpose(1, 2)

        keys, values = filled(state["k_pages"], k), filled(state["v_pages"], v)
        return {"q": q, "k": keys, "v": values}
    if case["op"] == "attend":
        s, hq, h, d = case["seqs"], case["q_heads"], case["kv_heads"], case["head_dim"]
        out = torch.zeros((s, hq, d), dtype=torch.float64, device=state["q"].device)
        lse = torch.full((s, hq), float("-inf"), dtype=torch.float64, device=state["q"].device)
        for i, n in enumerate(state["lengths"].tolist()):
            start = max(0, n - case["window"]) if case["window"] else 0
            if n == start:
                continue
            of = state["table"][i, :-(-n // case["page"])].long()
            k = state["k_pages"][of].double().transpose(0, 1).reshape(h, -1, d)[:, start:n]
            v = state["v_pages"][of].double().transpose(0, 1).reshape(h, -1, d)[:, start:n]
            q = state["q"][i].double().reshape(h, hq // h, d)
            z = torch.einsum("hgd,hnd->hgn", q, k) / d ** 0.5
            lse[i] = torch.logsumexp(z, -1).reshape(hq)
            out[i] = torch.einsum("hgn,hnd->hgd", torch.softmax(z, -1), v).reshape(hq, d)
        return {"out": out, "lse": lse}
    y = state["base"].double().clone(memory_format=torch.contiguous_format)
    for a, (down, up, scale) in enumerate(zip(state["down"], state["up"], state["scales"])):
        mine = torch.nonzero(state["ids"] == a)[:, 0]
        if len(mine):
            y[:, mine] += scale * (up.double() @ (down.double() @ state["x"][:, mine].double()))
    return {"y": y}
