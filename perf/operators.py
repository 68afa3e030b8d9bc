"""Cases that measure the cache's masked-attention and page operators.

Four operators over the paged key/value pools ``(num_blocks, block_size, kv
heads, head_dim)``:

* ``window``: attention of a step's queries over the last ``window`` keys of
  their sequence and its first ``sinks`` keys (decodes and prefill chunks);
* ``tree``: attention of drafted token trees over the cached context and, in
  the draft, each token's ancestors and itself;
* ``fork``: new slots that continue other slots' sequences: full blocks are
  shared, the partly filled last block is copied, in every layer;
* ``copy``: contents of whole blocks copied to other blocks, in every layer.

``run`` computes them in plain torch operations (``own`` false) or through
``nifre_b200.PagedKVCache`` (``own`` true), on the same inputs.
"""

import math
import random

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
DEV = "cuda"


# ---------------------------------------------------------------- cases
def listed():
    gqa64 = dict(hq=32, hkv=8, d=64, bs=16, dtype="bf16")  # the 1B benchmark shape
    gqa128 = dict(hq=32, hkv=8, d=128, bs=16, dtype="bf16")  # the 8B benchmark shape
    return [
        # one interactive user of a windowed model: the latency of a layer
        dict(name="window decode 1", op="window", seqs=1, qlen=1, ctx_lo=700, ctx_hi=700, window=512, sinks=4, **gqa64),
        # a serving batch of the 1B decode benchmark's context lengths
        dict(name="window decode 64", op="window", seqs=64, qlen=1, ctx_lo=512, ctx_hi=4096, window=1024, sinks=4,
             **gqa64),
        # long-running streams, most of whose cache the window has left behind
        dict(name="window decode long", op="window", seqs=64, qlen=1, ctx_lo=4096, ctx_hi=16384, window=4096, sinks=64,
             **gqa128),
        # float32 decodes of the 124M engine (12 heads, short contexts)
        dict(name="window decode fp32", op="window", seqs=8, qlen=1, ctx_lo=32, ctx_hi=320, window=128, sinks=1, hq=12,
             hkv=12, d=64, bs=16, dtype="fp32"),
        # the mixed benchmark's four prefill chunks over cached prefixes
        dict(name="window chunks", op="window", seqs=4, qlen=512, ctx_lo=512, ctx_hi=2048, window=1024, sinks=4,
             **gqa64),
        # one long prompt, prefilled in large chunks by a windowed half-precision model
        dict(name="window chunk long", op="window", seqs=1, qlen=2048, ctx_lo=8192, ctx_hi=8192, window=4096, sinks=0,
             hq=32, hkv=8, d=128, bs=16, dtype="fp16"),
        # speculative decoding for one user: a small tree
        dict(name="tree 1", op="tree", seqs=1, qlen=16, ctx_lo=700, ctx_hi=700, **gqa64),
        # a batch with short drafts: bound by the cache's bytes
        dict(name="tree batch short", op="tree", seqs=32, qlen=7, ctx_lo=512, ctx_hi=4096, **gqa64),
        # a batch with wide drafts
        dict(name="tree batch wide", op="tree", seqs=16, qlen=32, ctx_lo=512, ctx_hi=4096, **gqa64),
        # few long sequences with large trees
        dict(name="tree long", op="tree", seqs=8, qlen=64, ctx_lo=4096, ctx_hi=32768, **gqa128),
        # four prompts sampled four ways each, 16 layers
        dict(name="fork", op="fork", seqs=4, copies=4, ctx_lo=500, ctx_hi=1500, layers=16, **gqa64),
        # blocks moved together when a pool is compacted, 16 layers
        dict(name="copy blocks", op="copy", blocks=1000, layers=16, **gqa64),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    while True:  # no dearer than the largest listed cases
        case = _draw(rng)
        w = work(case)
        if w["bytes"] <= 1.0e9 and w["flops"] <= 1.3e11:
            return case


def _draw(rng):
    op = rng.choice(["window", "window", "window", "tree", "tree", "tree", "fork", "copy"])
    hkv = rng.choice([1, 2, 4, 8])
    shape = dict(hq=hkv * rng.choice([1, 2, 4, 4, 8]), hkv=hkv, d=rng.choice([64, 128]), bs=rng.choice([16, 16, 32, 64]),
                 dtype=rng.choice(["bf16", "bf16", "fp16"]))
    if rng.random() < 0.15:  # shapes and types outside the tensor cores' layouts
        shape.update(hq=hkv * rng.choice([1, 3]), d=rng.choice([32, 64, 80]), dtype=rng.choice(["fp32", "fp32", "fp16"]))
    if op == "window":
        lo = _log(rng, 16, 4000)
        hi = _log(rng, lo, 8000)
        qlen = rng.choice([1, 1, 1, rng.randint(2, 15), _log(rng, 16, 600)])
        seqs = _log(rng, 1, 64 if qlen == 1 else 6)
        return dict(op=op, seqs=seqs, qlen=qlen, ctx_lo=lo, ctx_hi=hi, window=_log(rng, 1, 4096),
                    sinks=rng.choice([0, 1, 4, rng.randint(2, 130)]), **shape)
    if op == "tree":
        lo = _log(rng, 1, 4000)
        hi = _log(rng, lo, 8000)
        qlen = _log(rng, 1, 64)
        return dict(op=op, seqs=_log(rng, 1, 24), qlen=qlen, ctx_lo=lo, ctx_hi=hi, **shape)
    if op == "fork":
        lo = _log(rng, 1, 1000)
        return dict(op=op, seqs=_log(rng, 1, 8), copies=rng.randint(1, 6), ctx_lo=lo, ctx_hi=_log(rng, lo, 2000),
                    layers=rng.choice([1, 5, 16]), **shape)
    return dict(op=op, blocks=_log(rng, 1, 1000 * 16 // shape["bs"]), layers=rng.choice([1, 4, 12]), **shape)


def _lens(case):
    """Context lengths of the case's sequences: evenly spaced over the range, whatever the seed."""
    n, lo, hi = case["seqs"], case["ctx_lo"], case["ctx_hi"]
    return [lo + (hi - lo) * (2 * i + 1) // (2 * n) for i in range(n)]


def _item(case):
    return 4 if case["dtype"] == "fp32" else 2


def work(case):
    """Bytes and operations of one pass: every visible key and value row, query and output row once."""
    row = case["hkv"] * case["d"] * _item(case)  # one token's keys (or values)
    if case["op"] == "copy":
        return {"bytes": 4 * case["layers"] * case["blocks"] * case["bs"] * row, "flops": 0}
    if case["op"] == "fork":  # the rows of the partly filled blocks: read once per source, written once per copy
        tails = sum(c % case["bs"] for c in _lens(case))
        shared = sum(c // case["bs"] for c in _lens(case)) * case["copies"]  # table entries: 4 bytes each
        return {"bytes": 2 * case["layers"] * tails * row * (1 + case["copies"]) + 4 * shared + 8, "flops": 0}
    n, qrow = case["qlen"], case["hq"] * case["d"] * _item(case)
    keys = pairs = 0
    for c in _lens(case):
        if case["op"] == "tree":
            keys += c + n
            pairs += n * c + sum(_depths(_parents(case, 0)))  # the draft's share is small: one tree stands for all
        else:
            w, s = case["window"], case["sinks"]
            first = max(0, c - w + 1)
            keys += c + n - first + min(s, first)
            for p in range(c, c + n):
                first = max(0, p - w + 1)
                pairs += p + 1 - first + min(s, first)
    return {"bytes": 2 * keys * row + 2 * case["seqs"] * n * qrow, "flops": 4 * pairs * case["hq"] * case["d"]}


def _parents(case, seed):
    """One drafted tree: token i continues token parents[i] < i, or the context (-1).  Drafts branch most near their root."""
    r = random.Random("%d %d" % (seed, case["qlen"]))
    return [-1 if i == 0 else max(-1, i - 1 - int(r.expovariate(0.5))) for i in range(case["qlen"])]


def _depths(parents):
    depth = []
    for p in parents:
        depth.append(1 if p < 0 else depth[p] + 1)
    return depth


# ---------------------------------------------------------------- inputs
def _inputs(case, seed):
    """What the case's program has: lengths, block tables, pools, queries (or block lists), trees."""
    r = random.Random(seed)
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt, bs, hkv, d = _DT[case["dtype"]], case["bs"], case["hkv"], case["d"]
    new = case.get("qlen", 0)
    x = {"new": new}
    if case["op"] == "copy":
        nb = 2 * case["blocks"] + 3
        x["order"] = r.sample(range(nb), nb)
    else:
        x["ctx"] = _lens(case)
        r.shuffle(x["ctx"])
        need = [-(-(c + new) // bs) for c in x["ctx"]]
        extra = sum(case["copies"] for c in x["ctx"] if c % bs) if case["op"] == "fork" else 0
        nb = sum(need) + extra + 2
        x["order"] = r.sample(range(nb), nb)  # the order in which the pool hands its blocks out
        x["tables"], at = [], 0
        for n in need:
            x["tables"].append(x["order"][at:at + n])
            at += n
        x["spare"] = x["order"][at:]
    x["num_blocks"] = nb
    shape = (case.get("layers", 1), nb, bs, hkv, d)
    x["k"] = torch.empty(shape, dtype=dt, device=DEV).normal_(generator=g)
    x["v"] = torch.empty(shape, dtype=dt, device=DEV).normal_(generator=g)
    if new:
        x["q"] = torch.empty(case["seqs"] * new, case["hq"] * d, dtype=dt, device=DEV).normal_(generator=g)
    if case["op"] == "tree":
        x["parents"] = [_parents(case, seed + i) for i in range(case["seqs"])]
    return x


def _visible(parents):
    """(n, n) truth values: token i sees token j when j is i or one of its ancestors."""
    n = len(parents)
    m = torch.eye(n, dtype=torch.bool)
    for i, p in enumerate(parents):
        if p >= 0:
            m[i] |= m[p]
    return m


def _cache(case, x, slots):
    """A nifre_b200 cache that holds the case's sequences in the case's blocks."""
    from nifre_b200 import PagedKVCache
    longest = max(x["ctx"]) + x["new"] if "ctx" in x else case["bs"]
    cache = PagedKVCache(case.get("layers", 1), longest, case["hkv"], case["d"], device=DEV, dtype=_DT[case["dtype"]],
                         block_size=case["bs"], enable_prefix_cache=False, num_blocks=x["num_blocks"])
    cache.init_batch(slots)
    cache.block_allocator.set_free_order(x["order"][::-1])
    return cache


def _append(cache, row, plan, rows):
    blank = torch.zeros(1, row, dtype=cache.dtype, device=DEV).expand(rows, row)
    for layer in range(cache.num_layers):
        cache.append_step(layer, blank, blank, plan)


def prepare(case, seed):
    x = _inputs(case, seed)
    s = {"case": case}
    S, n, bs, row = case.get("seqs", 0), x["new"], case["bs"], case["hkv"] * case["d"]
    if case["op"] == "copy":
        src, dst = x["order"][:case["blocks"]], x["order"][case["blocks"]:2 * case["blocks"]]
        s["src"], s["dst"] = (torch.tensor(b, dtype=torch.int32, device=DEV) for b in (src, dst))
    elif case["op"] == "fork":
        s["from"] = [i for i in range(S) for _ in range(case["copies"])]
        s["to"] = list(range(S, S + len(s["from"])))
    else:
        s["q"] = x["q"]
    if own:
        cache = s["cache"] = _cache(case, x, S * (1 + case.get("copies", 0)) if S else 1)
        if S:
            # the sequences' blocks, in the order of the tables: room for all of a sequence, then its lengths
            starts = [sum(x["ctx"][:i]) for i in range(S)]
            for i in range(S):
                cache.block_tables[i].ensure_capacity(x["ctx"][i] + n)
            _append(cache, row, cache.plan(list(range(S)), x["ctx"], starts, q_heads=case["hq"]), sum(x["ctx"]))
        if n:
            plan = cache.plan(list(range(S)), [n] * S, [n * i for i in range(S)], q_heads=case["hq"])
            _append(cache, row, plan, n * S)
            if case["op"] == "window":
                s["view"] = cache.plan_window(plan, case["window"], case["sinks"], q_heads=case["hq"])
            else:
                s["view"] = cache.plan_tree(plan, x["parents"], q_heads=case["hq"])
            s["out"] = torch.empty_like(x["q"])
        for layer in range(cache.num_layers):
            cache.k[layer].copy_(x["k"][layer])
            cache.v[layer].copy_(x["v"][layer])
        return s
    s["k"], s["v"] = x["k"], x["v"]
    if case["op"] == "copy":
        s["src"], s["dst"] = s["src"].long(), s["dst"].long()
    elif case["op"] == "fork":
        src, dst, spare = [], [], list(x["spare"])
        for i in s["from"]:
            c = x["ctx"][i]
            if c % bs:
                a, b = x["tables"][i][c // bs], spare.pop(0)
                src += [a * bs + t for t in range(c % bs)]
                dst += [b * bs + t for t in range(c % bs)]
        s["src"], s["dst"] = (torch.tensor(b, dtype=torch.long, device=DEV) for b in (src, dst))
    else:
        most = max(len(t) for t in x["tables"])
        s["tables"] = torch.tensor([t + [0] * (most - len(t)) for t in x["tables"]], device=DEV)
        s["ctx"] = torch.tensor(x["ctx"], device=DEV)
        if case["op"] == "window":
            first = [max(0, c - case["window"] + 1) for c in x["ctx"]]
            s["keys"] = max(c + n - f + min(case["sinks"], f) for c, f in zip(x["ctx"], first))
        else:
            s["keys"] = max(x["ctx"]) + n
            s["sees"] = torch.stack([_visible(p) for p in x["parents"]]).to(DEV)
    return s


# ---------------------------------------------------------------- one pass
def run(state):
    op = state["case"]["op"]
    if own:
        cache = state["cache"]
        if op == "window":
            return cache.window_attention_step(0, state["q"], state["view"], state["out"])
        if op == "tree":
            return cache.tree_attention_step(0, state["q"], state["view"], state["out"])
        if op == "fork":
            cache.fork(state["from"], state["to"])
        else:
            cache.copy_blocks(state["src"], state["dst"])
        return list(cache.k) + list(cache.v)
    if op == "window":
        return _window(state)
    if op == "tree":
        return _tree(state)
    k, v = state["k"], state["v"]
    if op == "fork":
        k, v = (t.view(t.shape[0], -1, *t.shape[3:]) for t in (k, v))
    k[:, state["dst"]] = k[:, state["src"]]
    v[:, state["dst"]] = v[:, state["src"]]
    return list(state["k"].unbind(0)) + list(state["v"].unbind(0))


def _window(s):
    case = s["case"]
    n, w, sinks = case["qlen"], case["window"], case["sinks"]
    ctx = s["ctx"][:, None]
    # the keys that some query of the sequence sees: its first ones, then those from the first query's window on
    first = (ctx - w + 1).clamp(min=0)
    kept = first.clamp(max=sinks)
    j = torch.arange(s["keys"], device=DEV)[None]
    pos = torch.where(j < kept, j, j - kept + first)
    at = ctx + torch.arange(n, device=DEV)[None]  # the queries' positions
    p, t = pos[:, None, :], at[:, :, None]
    return _attend(s, pos.clamp(max=ctx + n - 1), (p <= t) & ((p > t - w) | (p < sinks)))


def _tree(s):
    n = s["case"]["qlen"]
    ctx = s["ctx"][:, None]
    pos = torch.arange(s["keys"], device=DEV)[None].expand(len(s["ctx"]), -1)
    draft = (pos - ctx).clamp(0, n - 1)
    sees = torch.gather(s["sees"], 2, draft[:, None, :].expand(-1, n, -1))
    p, c = pos[:, None, :], ctx[:, :, None]
    return _attend(s, pos.clamp(max=ctx + n - 1), (p < c) | ((p < c + n) & sees))


def _attend(s, pos, sees):
    """Softmax attention in 32 bits: queries (S x n rows), keys at pos (S, K), truth values sees (S, n, K)."""
    case = s["case"]
    S, n, hkv, d = case["seqs"], case["qlen"], case["hkv"], case["d"]
    rows = torch.gather(s["tables"], 1, pos // case["bs"]) * case["bs"] + pos % case["bs"]
    k, v = (t.view(-1, hkv, d)[rows].float() for t in (s["k"], s["v"]))  # (S, K, hkv, d)
    q = s["q"].view(S, n, hkv, -1, d).float()
    scores = torch.einsum("snhgd,skhd->shgnk", q, k) / math.sqrt(d)
    scores = scores.masked_fill(~sees[:, None, None], -math.inf)
    e = torch.exp(scores - scores.amax(-1, keepdim=True))
    out = torch.einsum("shgnk,skhd->snhgd", e / e.sum(-1, keepdim=True), v)
    return out.reshape(S * n, -1).to(s["q"].dtype)


# ---------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    """Sequence by sequence and token by token's key list, in 64 bits; None for copies, which compute nothing."""
    if case["op"] in ("fork", "copy"):
        return None
    x = _inputs(case, seed)
    n, bs, hkv, d = case["qlen"], case["bs"], case["hkv"], case["d"]
    group = case["hq"] // hkv
    out = torch.empty(case["seqs"] * n, hkv * group, d, dtype=torch.float64, device=DEV)
    for i, c in enumerate(x["ctx"]):
        table = torch.tensor(x["tables"][i], device=DEV)
        k, v = (t[0][table].reshape(-1, hkv, d)[:c + n].double() for t in (x["k"], x["v"]))
        key = torch.arange(c + n, device=DEV)
        for t0 in range(0, n, 64):
            t = torch.arange(t0, min(n, t0 + 64), device=DEV)
            if case["op"] == "window":
                behind = (c + t)[:, None] - key[None]
                hidden = (behind < 0) | ((behind >= case["window"]) & (key >= case["sinks"])[None])
            else:
                hidden = torch.ones(len(t), c + n, dtype=torch.bool, device=DEV)
                hidden[:, :c] = False
                for a in t.tolist():
                    node = a
                    while node >= 0:
                        hidden[a - t0, c + node] = False
                        node = x["parents"][i][node]
            q = x["q"].view(-1, hkv, group, d)[i * n + t0:i * n + t0 + len(t)].double()
            for h in range(hkv):
                z = (q[:, h].reshape(-1, d) @ k[:, h].T).view(len(t), group, -1) * d ** -0.5
                z[hidden[:, None].expand_as(z)] = -math.inf
                a = torch.softmax(z, -1)
                out[i * n + t0:i * n + t0 + len(t), h * group:(h + 1) * group] = a @ v[:, h]
    return out.view(case["seqs"] * n, -1)
