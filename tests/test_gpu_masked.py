"""Windowed and tree attention over the paged pools against the definition in 64 bits (needs a B200).

Tolerances are oracle.masked.tolerance (derived there from the roundings the
kernels make).  The pools start as NaN everywhere, so that a key row no token
sees (behind the window, past the sequence, never written) shows if it reaches
an output.
"""

import numpy as np
import pytest
import torch

from oracle.masked import attend, tolerance, tree_seen, window_seen

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module", autouse=True)
def _lib_built():
    from nifre_b200 import _lib
    _lib.load()


class Step:
    """A cache with contexts of ``ctx`` tokens and a step of ``n`` new ones (rows ``pad`` apart in q and out)."""

    def __init__(self, ctx, n, hq, hkv, d, bs, dtype, seed=0, layers=1, pad=0, room=16, cls=None):
        from nifre_b200 import PagedKVCache
        g = torch.Generator().manual_seed(seed)
        self.ctx, self.n, self.hq, self.hkv, self.d, self.dtype = list(ctx), list(n), hq, hkv, d, dtype
        S = len(ctx)
        most = max(c + m for c, m in zip(ctx, n)) + room
        if cls is None:
            self.cache = PagedKVCache(layers, most, hkv, d, device=DEV, dtype=dtype, block_size=bs,
                                      enable_prefix_cache=False)
        else:
            self.cache = cls(layers, most, hkv, d, device=DEV, dtype=dtype)
        self.cache.init_batch(S)
        for t in (*self.cache.k, *self.cache.v):
            t.fill_(float("nan"))
        if cls is None:
            self.cache.block_allocator.set_free_order(torch.randperm(self.cache.num_blocks, generator=g).tolist())
        self.g = g
        filled = [i for i in range(S) if ctx[i]]
        # k[s], v[s]: rows of every layer's keys and values of sequence s (layers, tokens, Hkv, D)
        self.k = [torch.empty(layers, 0, hkv, d, dtype=dtype, device=DEV) for _ in range(S)]
        self.v = [t.clone() for t in self.k]
        if filled:
            self._append(filled, [ctx[i] for i in filled])
        self.start, at = [], pad
        for m in self.n:
            self.start.append(at)
            at += m + pad
        self.rows = at
        self.plan = self._append(list(range(S)), self.n, self.start, at, q_heads=hq)
        self.q = self.rand(layers, self.rows, hq * d)

    def rand(self, *shape):
        return torch.randn(*shape, generator=self.g).to(self.dtype).to(DEV)

    def _append(self, slots, lens, starts=None, rows=None, q_heads=None):
        starts = starts or [sum(lens[:i]) for i in range(len(lens))]
        rows = rows or sum(lens)
        plan = self.cache.plan(slots, lens, starts, q_heads=q_heads)
        ks, vs = [], []
        for layer in range(self.cache.num_layers):
            k, v = self.rand(rows, self.hkv * self.d), self.rand(rows, self.hkv * self.d)
            self.cache.append_step(layer, k, v, plan)
            ks.append(k.view(rows, self.hkv, self.d))
            vs.append(v.view(rows, self.hkv, self.d))
        k, v = torch.stack(ks), torch.stack(vs)
        for s, m, st in zip(slots, lens, starts):
            self.k[s] = torch.cat([self.k[s], k[:, st:st + m]], 1)
            self.v[s] = torch.cat([self.v[s], v[:, st:st + m]], 1)
        return plan

    def check(self, out, seen_of, layer=0, scale=None, q=None):
        """out against the definition, every row; rows between the sequences' keep their 7."""
        q = self.q[layer] if q is None else q
        used = torch.zeros(self.rows, dtype=torch.bool)
        scale = self.d ** -0.5 if scale is None else scale
        for s, (c, m, st) in enumerate(zip(self.ctx, self.n, self.start)):
            used[st:st + m] = True
            ref, wabs, most = attend(q[st:st + m].view(m, self.hq, self.d), self.k[s][layer], self.v[s][layer],
                                     seen_of(s), scale)
            tol = tolerance(ref, wabs, most, c + m, self.d, self.dtype)
            got = out[st:st + m].view(m, self.hq, self.d).double()
            err = (got - ref).abs()
            assert torch.isfinite(got).all(), (s, c, m)
            assert (err <= tol).all(), (s, c, m, float((err / tol).max()), float(err.max()))
        assert (out[~used.to(out.device)] == 7).all()
        self.cache.check_status()

    def window(self, window, sinks, layer=0, q=None, **kw):
        view = self.cache.plan_window(self.plan, window, sinks, q_heads=self.hq)
        q = self.q[layer] if q is None else q
        out = torch.full((self.rows, self.hq * self.d), 7, dtype=self.dtype, device=DEV)
        self.cache.window_attention_step(layer, q, view, out, **kw)
        self.check(out, lambda s: window_seen(self.ctx[s], self.n[s], window, sinks), layer, q=q, **kw)
        return out

    def tree(self, masks, layer=0, q=None, parents=None, **kw):
        given = dict(masks=masks) if parents is None else dict(parents=parents)
        view = self.cache.plan_tree(self.plan, q_heads=self.hq, **given)
        q = self.q[layer] if q is None else q
        out = torch.full((self.rows, self.hq * self.d), 7, dtype=self.dtype, device=DEV)
        self.cache.tree_attention_step(layer, q, view, out, **kw)
        self.check(out, lambda s: tree_seen(self.ctx[s], torch.as_tensor(masks[s])), layer, q=q, **kw)
        return out


# query heads, KV heads, head_dim, block size, type
SHAPES = [(32, 8, 64, 16, BF), (8, 8, 64, 32, HF), (8, 1, 128, 16, HF), (16, 4, 128, 64, BF), (4, 2, 64, 16, BF),
          (12, 12, 64, 16, F32), (6, 2, 80, 8, HF), (4, 4, 32, 5, F32), (3, 1, 7, 3, BF), (16, 1, 256, 16, F32),
          (40, 2, 64, 16, BF), (6, 2, 64, 16, HF), (8, 1, 64, 48, BF), (4, 4, 96, 16, BF)]
IDS = [f"{a}q{b}kv{c}d{d}b{str(e)[6:]}" for a, b, c, d, e in SHAPES]


@pytest.mark.parametrize("window,sinks", [(1, 0), (5, 1), (64, 4), (130, 33), (1000, 0), (3, 1 << 30)])
@pytest.mark.parametrize("shape", SHAPES, ids=IDS)
def test_window_attention(shape, window, sinks):
    """Empty and short contexts, block and tile edges, decodes, short chunks and prefill chunks in one step."""
    hq, hkv, d, bs, dtype = shape
    st = Step([0, 1, 15, 16, 300, 777, 0], [1, 5, 1, 40, 2, 1, 70], hq, hkv, d, bs, dtype, seed=window + sinks, pad=2)
    st.window(window, sinks)


def _random_tree(n, g):
    parents = [-1] + [int(torch.randint(-1, i, (1,), generator=g)) for i in range(1, n)]
    return parents


@pytest.mark.parametrize("shape", SHAPES, ids=IDS)
def test_tree_attention(shape):
    from nifre_b200 import tree_visibility
    hq, hkv, d, bs, dtype = shape
    n = [1, 7, 33, 2, 64, 16, 90]
    st = Step([0, 3, 16, 250, 600, 31, 129], n, hq, hkv, d, bs, dtype, seed=3, pad=1)
    parents = [_random_tree(m, st.g) for m in n]
    parents[3] = None  # a chain
    masks = [np.tril(np.ones((m, m), bool)) if p is None else tree_visibility(p) for m, p in zip(n, parents)]
    st.tree(masks, parents=parents)


@pytest.mark.parametrize("shape", [SHAPES[i] for i in (0, 2, 5, 6, 10)], ids=[IDS[i] for i in (0, 2, 5, 6, 10)])
def test_tree_masks_that_leave_rows_empty(shape):
    """Any mask goes, later tokens and empty rows among it; a token that sees nothing gets zeros."""
    hq, hkv, d, bs, dtype = shape
    n = [9, 40, 3, 65]
    st = Step([0, 0, 50, 130], n, hq, hkv, d, bs, dtype, seed=4)
    rng = np.random.default_rng(0)
    masks = [rng.integers(0, 2, size=(m, m)).astype(bool) for m in n]
    masks[0][3] = False
    masks[1][:] = False
    masks[2][:] = False
    out = st.tree(masks)
    assert (out[st.start[0] + 3] == 0).all() and (out[st.start[1]:st.start[1] + 40] == 0).all()


@pytest.mark.parametrize("shape", SHAPES[:7], ids=IDS[:7])
def test_values_of_unseen_keys_do_not_matter(shape):
    """NaN and infinities in keys and values that a token does not see, though others of its group do."""
    hq, hkv, d, bs, dtype = shape
    n = [12, 30]
    st = Step([70, 200], n, hq, hkv, d, bs, dtype, seed=5)
    masks = [np.eye(m, dtype=bool) for m in n]
    for s in range(2):
        masks[s][:, 0] = True
        masks[s][5, 4] = True
    bad = {4: float("nan"), 7: float("inf"), 9: float("-inf")}
    for s in range(2):
        for j, x in bad.items():
            t = st.ctx[s] + j
            block, off = st.cache.block_tables[s].resolve(t)
            st.cache.k[0][block, off] = x
            st.cache.v[0][block, off] = x
            st.k[s][0, t], st.v[s][0, t] = x, x
    view = st.cache.plan_tree(st.plan, masks=masks, q_heads=hq)
    out = torch.full((st.rows, hq * d), 7, dtype=dtype, device=DEV)
    st.cache.tree_attention_step(0, st.q[0], view, out)
    hit = {4, 5, 7, 9}
    for s in range(2):
        for i in range(n[s]):
            row = out[st.start[s] + i]
            if i in hit:
                assert not torch.isfinite(row).any()
                continue
            ref, wabs, most = attend(st.q[0][st.start[s] + i].view(1, hq, d), st.k[s][0], st.v[s][0],
                                     tree_seen(st.ctx[s], torch.as_tensor(masks[s]))[i:i + 1], d ** -0.5)
            tol = tolerance(ref, wabs, most, st.ctx[s] + n[s], d, dtype)
            assert ((row.view(1, hq, d).double() - ref).abs() <= tol).all()
    # a window's chunk: keys behind the later tokens' windows
    st = Step([40], [40], hq, hkv, d, bs, dtype, seed=6)
    for t in (45, 50):
        block, off = st.cache.block_tables[0].resolve(t)
        st.cache.v[0][block, off] = float("nan")
    view = st.cache.plan_window(st.plan, 8, 2, q_heads=hq)
    out = torch.full((st.rows, hq * d), 7, dtype=dtype, device=DEV)
    st.cache.window_attention_step(0, st.q[0], view, out)
    seen = window_seen(40, 40, 8, 2)
    touched = seen[:, 45] | seen[:, 50]
    assert torch.isfinite(out[~touched]).all() and not torch.isfinite(out[touched]).any()
    ref, wabs, most = attend(st.q[0].view(40, hq, d), st.k[0][0], st.v[0][0], seen, d ** -0.5)
    tol = tolerance(ref, wabs, most, 80, d, dtype)
    err = (out.view(40, hq, d).double() - ref).abs()
    assert (err[~touched] <= tol[~touched]).all()


@pytest.mark.parametrize("shape", [SHAPES[i] for i in (0, 2, 3, 5, 8)], ids=[IDS[i] for i in (0, 2, 3, 5, 8)])
def test_keys_split_into_many_parts(shape, monkeypatch):
    from nifre_b200 import masked, tree_visibility
    hq, hkv, d, bs, dtype = shape
    monkeypatch.setattr(masked, "unit_share_for", lambda *a: 64)
    monkeypatch.setattr(masked, "item_share_for", lambda *a: 512)
    n = [1, 3, 48]
    st = Step([1300, 2500, 1500], n, hq, hkv, d, bs, dtype, seed=7, pad=1)
    st.window(700, 20)
    masks = [tree_visibility(_random_tree(m, st.g)) for m in n]
    st.tree(masks)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_strided_unaligned_queries_and_scale(dtype):
    """q as a column slice of a wider projection (rows not 16-byte aligned), out rows with their own stride, a scale
    of the caller's, several layers with windows of their own."""
    st = Step([100, 0, 37], [1, 20, 3], 8, 2, 64, 16, dtype, seed=8, layers=3, pad=1)
    for layer, (w, s) in enumerate([(30, 2), (1 << 20, 0), (9, 0)]):
        wide = st.rand(st.rows, 8 * 64 + 131)
        q = wide[:, 65:65 + 512]
        st.window(w, s, layer=layer, q=q, scale=0.31)
    view = st.cache.plan_window(st.plan, 30, 2, q_heads=8)
    buf = torch.full((st.rows, 530), 7, dtype=dtype, device=DEV)
    st.cache.window_attention_step(1, st.q[1], view, buf[:, 9:521])
    st.check(buf[:, 9:521], lambda s: window_seen(st.ctx[s], st.n[s], 30, 2), 1)
    assert (buf[:, :9] == 7).all() and (buf[:, 521:] == 7).all()


def _split(monkeypatch, keys=16, item_keys=128):
    """Parts of ``keys`` keys, and of ``item_keys`` for the tensor cores' items; the last one as short as it comes."""
    from nifre_b200 import masked
    even = masked.even_shares
    monkeypatch.setattr(masked, "unit_share_for", lambda *a: keys)
    monkeypatch.setattr(masked, "item_share_for", lambda *a: item_keys)
    monkeypatch.setattr(masked, "even_shares", lambda k, share, align, least, each=0: even(k, share, align, 1, 0))


def _tree_out(st, masks, hq):
    view = st.cache.plan_tree(st.plan, masks=masks, q_heads=hq)
    out = torch.full((st.rows, hq * st.d), 7, dtype=st.dtype, device=DEV)
    return st.cache.tree_attention_step(0, st.q[0], view, out).clone()


def _set_key(st, s, t, x, what="k"):
    block, off = st.cache.block_tables[s].resolve(t)
    getattr(st.cache, what)[0][block, off] = x


@pytest.mark.parametrize("split", [False, True])
@pytest.mark.parametrize("shape", SHAPES, ids=IDS)
def test_scores_that_are_not_numbers_reach_the_output(shape, split, monkeypatch):
    """A NaN query row, and a NaN key that a row sees -- as the only seen key of a warp, a part, a step, or of the row
    -- give NaN in all of the row; the other rows keep their bits."""
    hq, hkv, d, bs, dtype = shape
    if split:
        _split(monkeypatch)
    n = [1, 1, 5, 2, 40, 200, 33, 2]
    st = Step([8, 0, 48, 16, 64, 128, 0, 70], n, hq, hkv, d, bs, dtype, seed=21, pad=1)
    masks = [np.eye(m, dtype=bool) for m in n]
    masks[4][7, [0, 20]] = True
    masks[5][::3, :90] = True
    masks[6][20:, 5] = True
    want = _tree_out(st, masks, hq)
    keys = {0: 0, 1: 0, 2: 3, 4: 20, 5: 150, 6: 5}  # the drafted token of each sequence whose key is NaN
    for s, j in keys.items():
        _set_key(st, s, st.ctx[s] + j, float("nan"))
    _set_key(st, 3, 10, float("nan"))  # and a key of a context: every row of its sequence
    st.q[0][st.start[5] + 170] = float("nan")
    st.q[0][st.start[7] + 1] = float("nan")
    st.q[0][st.start[4] + 2, d // 2] = float("nan")  # one element of the first head's query
    out = _tree_out(st, masks, hq)
    for s, m in enumerate(n):
        for i in range(m):
            row, was = out[st.start[s] + i], want[st.start[s] + i]
            if (s in keys and masks[s][i, keys[s]]) or s == 3 or (s, i) in ((5, 170), (7, 1)):
                assert torch.isnan(row).all(), (s, i)
            elif (s, i) == (4, 2):
                assert torch.isnan(row[:d]).all() and torch.equal(row[d:], was[d:])
            else:
                assert torch.equal(row, was), (s, i)
    st.cache.check_status()


@pytest.mark.parametrize("split", [False, True])
@pytest.mark.parametrize("shape", SHAPES, ids=IDS)
def test_scores_of_minus_infinity(shape, split, monkeypatch):
    """Seen keys that score -inf weigh nothing beside others; a row that sees only such keys is 0 / 0."""
    hq, hkv, d, bs, dtype = shape
    if split:
        _split(monkeypatch)
    ctx, n = [0, 0, 48, 0, 128], [2, 5, 6, 40, 180]
    st = Step(ctx, n, hq, hkv, d, bs, dtype, seed=22, pad=1)
    st.q.view(1, st.rows, hq, d)[..., 0] = 1
    masks = [np.eye(m, dtype=bool) for m in n]
    masks[1][:, 4] = True
    masks[3][10:, :4] = True
    masks[3][30] = False
    low = {0: [1], 1: [0, 1, 4], 2: [5], 3: [0, 1, 2, 3, 20], 4: list(range(100, 180))}
    for s, js in low.items():
        for j in js:
            block, off = st.cache.block_tables[s].resolve(ctx[s] + j)
            st.cache.k[0][block, off, :, 0] = float("-inf")
    out = _tree_out(st, masks, hq)
    for s, m in enumerate(n):
        finite = np.asarray(masks[s]).copy()
        finite[:, low[s]] = False
        seen = tree_seen(ctx[s], torch.as_tensor(finite))
        rows = st.start[s] + np.arange(m)
        ref, wabs, most = attend(st.q[0][rows].view(m, hq, d), st.k[s][0], st.v[s][0], seen, d ** -0.5)
        tol = tolerance(ref, wabs, most, ctx[s] + m, d, dtype)
        for i in range(m):
            row = out[rows[i]].view(hq, d).double()
            if not seen[i].any() and masks[s][i].any():
                assert torch.isnan(row).all(), (s, i)
            else:
                assert ((row - ref[i]).abs() <= tol[i]).all(), (s, i)
    st.cache.check_status()


@pytest.mark.parametrize("split", [False, True])
@pytest.mark.parametrize("shape", SHAPES, ids=IDS)
def test_values_of_seen_keys_with_weights_near_zero(shape, split, monkeypatch):
    """A value that is not finite reaches every row that sees its key, also where the key's weight underflows to 0 and
    other rows of its tile do not see it (as 0 * NaN does in the definition's arithmetic)."""
    hq, hkv, d, bs, dtype = shape
    if split:
        _split(monkeypatch)
    ctx, n = [16, 40, 100], [5, 30, 150]
    st = Step(ctx, n, hq, hkv, d, bs, dtype, seed=27, pad=1)
    st.q.view(1, st.rows, hq, d)[..., 0] = 100
    masks = [np.tril(np.ones((m, m), dtype=bool)) for m in n]
    for s in range(3):
        block, off = st.cache.block_tables[s].resolve(ctx[s] + 2)
        st.cache.k[0][block, off, :, 0] = -3e4  # scores of -3e6 / sqrt(d)
        st.cache.v[0][block, off] = float("nan")
    out = _tree_out(st, masks, hq)
    for s, m in enumerate(n):
        for i in range(m):
            row = out[st.start[s] + i]
            assert (torch.isnan(row) if i >= 2 else torch.isfinite(row)).all(), (s, i)
    st.cache.check_status()


def test_large_scores_and_long_window():
    """Scores far from 0 (one key takes all the weight) and a running maximum that moves late."""
    st = Step([3000], [4], 8, 2, 64, 16, BF, seed=9)
    for t in (10, 1500, 2999):
        block, off = st.cache.block_tables[0].resolve(t)
        st.cache.k[0][block, off] *= 8
        st.k[0][0, t] *= 8
    st.window(2500, 16)
    st.window(4000, 0, scale=2.0)


@pytest.mark.parametrize("scale", [0.0, -0.2, 1.0])
def test_scales(scale):
    st = Step([60, 10], [1, 60], 4, 2, 64, 16, BF, seed=11, pad=1)
    st.window(40, 3, scale=scale)
    st.tree([np.tril(np.ones((m, m), bool)) for m in st.n], scale=scale)


@pytest.mark.parametrize("hq,hkv,d", [(16, 8, 128), (8, 8, 96)])
def test_pools_past_32_bit_offsets(hq, hkv, d):
    """Blocks whose elements lie more than 2^31 past the pool's start, decodes, a chunk and a tree."""
    from nifre_b200 import PagedKVCache
    bs, per = 16, 16 * hkv * d
    blocks = (1 << 31) // per + 64
    cache = PagedKVCache(1, 1024, hkv, d, device=DEV, dtype=HF, block_size=bs, enable_prefix_cache=False, num_blocks=blocks)
    cache.init_batch(2)  # blocks are handed out from the last one down
    g = torch.Generator().manual_seed(16)
    st = Step.__new__(Step)
    st.cache, st.g, st.dtype, st.hq, st.hkv, st.d = cache, g, HF, hq, hkv, d
    st.k = [torch.empty(1, 0, hkv, d, dtype=HF, device=DEV) for _ in range(2)]
    st.v = [t.clone() for t in st.k]
    st.ctx, st.n, st.start, st.rows = [300, 200], [1, 40], [0, 1], 41
    st._append([0, 1], st.ctx)
    st.plan = st._append([0, 1], st.n, st.start, 41, q_heads=hq)
    assert min(b for t in cache.block_tables for b in t.physical_blocks()) * per > 1 << 31
    st.q = st.rand(1, 41, hq * d)
    st.window(150, 20)
    st.tree([np.tril(np.ones((m, m), bool)) for m in st.n])
    src = cache.block_tables[0].physical_blocks()[0]
    cache.copy_blocks([src], [3])
    assert torch.equal(cache.k[0][3], cache.k[0][src]) and torch.equal(cache.v[0][3], cache.v[0][src])


def test_plans_are_not_made_inside_a_capture():
    st = Step([20], [1], 4, 2, 64, 16, HF, seed=17)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="capture"):
            st.cache.plan_window(st.plan, 4, q_heads=4)
        st.q.add_(0)


def test_dense_cache_rows():
    from nifre_b200 import KVCache
    for room in (9, 13):  # rows of 128 and of 132 tokens
        st = Step([30, 100], [1, 19], 4, 4, 64, None, HF, seed=10, cls=KVCache, room=room)
        st.window(50, 3)
        st.tree([np.tril(np.ones((m, m), bool)) for m in st.n])


def test_plans_of_other_caches_and_kinds_are_refused():
    a, b = (Step([10], [2], 4, 2, 64, 16, HF, seed=i) for i in range(2))
    out = torch.empty_like(a.q[0])
    w = a.cache.plan_window(a.plan, 4, q_heads=4)
    t = a.cache.plan_tree(a.plan, [None], q_heads=4)
    with pytest.raises(ValueError, match="another cache"):
        b.cache.window_attention_step(0, a.q[0], w, out)
    with pytest.raises(ValueError, match="window's"):
        a.cache.tree_attention_step(0, a.q[0], w, out)
    with pytest.raises(ValueError, match="tree's"):
        a.cache.window_attention_step(0, a.q[0], t, out)
    with pytest.raises(IndexError, match="layer_id"):
        a.cache.window_attention_step(1, a.q[0], w, out)
    for q, o in ((a.q[0][:1], out[:1]), (a.q[0][:, :128], out), (a.q[0].float(), out), (a.q[0], out.float()),
                 (a.q[0], out[:1]), (a.q[0], out[:1].expand(2, -1))):
        with pytest.raises(ValueError):
            a.cache.window_attention_step(0, q, w, o)
    with pytest.raises(ValueError, match="another cache, window"):
        a.cache.plan_window(a.plan, 5, q_heads=4, into=w)
    from nifre_b200 import _lib
    with pytest.raises(_lib.NifreError, match="CUDA tensor"):
        a.cache.window_attention_step(0, a.q[0].cpu(), w, out.cpu())
    a.cache.free()
    a.cache.init_batch(1)
    with pytest.raises(ValueError, match="init_batch"):
        a.cache.window_attention_step(0, a.q[0], w, out)


def test_plans_of_an_earlier_batch_are_refused():
    st = Step([10], [2], 4, 2, 64, 16, HF, seed=3)
    view = st.cache.plan_window(st.plan, 4, q_heads=4)
    out = torch.empty_like(st.q[0])
    st.cache.window_attention_step(0, st.q[0], view, out)
    st.cache.init_batch(1)  # the pools may come back at the same addresses
    with pytest.raises(ValueError, match="init_batch"):
        st.cache.window_attention_step(0, st.q[0], view, out)
    with pytest.raises(ValueError, match="into"):
        st.cache.plan_window(st.cache.plan([0], [2], [0]), 4, q_heads=4, into=view)


def test_step_plans_of_an_earlier_batch_or_length_are_refused():
    st = Step([10, 20], [2, 1], 4, 2, 64, 16, HF, seed=26)
    c = st.cache
    c.truncate(1, 20)
    with pytest.raises(ValueError, match="changed"):
        c.plan_window(st.plan, 4, q_heads=4)
    plan = c.plan([0, 1], [2, 1], [0, 2], q_heads=4)
    c.plan_window(plan, 4)  # of an open step
    kv = torch.zeros(3, 128, dtype=HF, device=DEV)
    c.append_step(0, kv, kv, plan)
    view = c.plan_tree(plan, [[-1, 0], None])  # and of a closed one
    c.keep_tokens(plan, [[1], []])
    with pytest.raises(ValueError, match="changed"):
        c.plan_tree(plan, [[-1, 0], None], into=view)
    other = Step([10, 20], [2, 1], 4, 2, 64, 16, HF, seed=26)
    with pytest.raises(ValueError, match="another cache's"):
        c.plan_window(other.plan, 4, q_heads=4)
    other.cache.init_batch(2)
    other.cache.pos_host[:] = [12, 21]
    with pytest.raises(ValueError, match="init_batch"):
        other.cache.plan_window(other.plan, 4, q_heads=4)


def test_bad_records_are_flagged_not_followed():
    """Work lists and block tables with values out of range: skipped and flagged by the kernels' own checks."""
    from nifre_b200 import _lib
    st = Step([40, 40], [1, 1], 4, 2, 64, 16, F32, seed=12)
    view = st.cache.plan_window(st.plan, 30, 0, q_heads=4)
    at, _ = __import__("nifre_b200.masked", fromlist=["WorkLists"]).WorkLists.offsets(view.room)
    good = view.buf.clone()
    for index, value, bit in ((at[0] + 4, 99, "bad slot=1"), (at[0] + 5, 77, "bad slot=1"), (at[0] + 6, -1, "bad slot=1")):
        view.buf.copy_(good)
        view.buf[index] = value
        out = torch.full((2, 256), 7, dtype=F32, device=DEV)
        st.cache.window_attention_step(0, st.q[0], view, out)
        with pytest.raises(_lib.NifreError, match=bit):
            st.cache.check_status()
        assert (out == 7).all(1).sum() == 1  # the other sequence's row is there
    view.buf.copy_(good)
    st.cache.bt_dev[0, 1] = 10_000
    out = torch.full((2, 256), 7, dtype=F32, device=DEV)
    st.cache.window_attention_step(0, st.q[0], view, out)
    with pytest.raises(_lib.NifreError, match="bad block=1"):
        st.cache.check_status()


@pytest.mark.parametrize("dtype,n", [(F32, 1), (F32, 4), (BF, 1), (BF, 7)])
@pytest.mark.parametrize("field,value", [(0, -16), (0, -(1 << 31)), (0, 8), (6, 40)])
def test_bad_units_are_flagged_not_followed(dtype, n, field, value):
    """A first key below 0 or inside a group of 16, more tokens than the launch is sized for."""
    from nifre_b200 import _lib
    from nifre_b200.masked import WorkLists
    st = Step([40, 40], [n, n], 4, 1, 64, 16, dtype, seed=28, room=64)
    view = st.cache.plan_window(st.plan, 30, 0, q_heads=4)
    at, _ = WorkLists.offsets(view.room)
    wide = torch.zeros(80, 256, dtype=dtype, device=DEV)  # rows enough for the larger group
    wide[:2 * n] = st.q[0]
    row, rows = view.buf[at[0] + 5:at[0] + 7].tolist()  # of the first unit's group
    view.buf[at[0] + field] = value
    out = torch.full((80, 256), 7, dtype=dtype, device=DEV)
    st.cache.window_attention_step(0, wide, view, out)
    with pytest.raises(_lib.NifreError, match="bad slot=1"):
        st.cache.check_status()
    left = torch.ones(80, dtype=torch.bool)
    left[:2 * n] = False
    left[row:row + rows] = True
    assert torch.equal((out == 7).all(1).cpu(), left)


@pytest.mark.parametrize("split", [False, True])
@pytest.mark.parametrize("shape", SHAPES, ids=IDS)
def test_keys_of_missing_blocks_are_left_out(shape, split, monkeypatch):
    """Block ids out of range: flagged, and their keys take no part, whatever the other blocks hold."""
    from nifre_b200 import _lib
    hq, hkv, d, bs, dtype = shape
    if split:
        _split(monkeypatch, item_keys=256)
    ctx, n = [40, 200, 400, 300, 150, 500], [1, 3, 12, 40, 100, 130]
    st = Step(ctx, n, hq, hkv, d, bs, dtype, seed=25, pad=1)
    gone = {0: [0], 1: [2], 2: [1, 4], 3: [3], 4: [0, (150 + 20) // bs]}  # logical blocks; sequence 5 has all of its own
    for s, blocks in gone.items():
        for b in blocks:
            st.cache.bt_dev[s, b] = 1 << 20 if b % 2 else -1
    gone[5] = []
    lost = lambda s: [t for b in gone[s] for t in range(b * bs, min((b + 1) * bs, ctx[s] + n[s]))]  # noqa: E731
    masks = [np.eye(m, dtype=bool) for m in n]

    def check(out, seen_of):
        with pytest.raises(_lib.NifreError, match="bad block=1"):
            st.cache.check_status()
        for s, m in enumerate(n):
            seen = seen_of(s).clone()
            seen[:, lost(s)] = False
            rows = slice(st.start[s], st.start[s] + m)
            ref, wabs, most = attend(st.q[0][rows].view(m, hq, d), st.k[s][0], st.v[s][0], seen, d ** -0.5)
            tol = tolerance(ref, wabs, most, ctx[s] + m, d, dtype)
            err = (out[rows].view(m, hq, d).double() - ref).abs()[seen.any(1)]
            assert (err <= tol[seen.any(1)]).all(), (s, float(err.max()))

    check(_tree_out(st, masks, hq), lambda s: tree_seen(ctx[s], torch.as_tensor(masks[s])))
    view = st.cache.plan_window(st.plan, 170, 70, q_heads=hq)
    out = st.cache.window_attention_step(0, st.q[0], view, torch.full_like(st.q[0], 7))
    check(out, lambda s: window_seen(ctx[s], n[s], 170, 70))


@pytest.mark.parametrize("field,value", [(4, 99), (5, 139), (6, -1), (6, 1000), (0, 8), (0, 4096)])
def test_bad_tensor_core_items_are_flagged_not_followed(field, value):
    from nifre_b200 import _lib
    from nifre_b200.masked import WorkLists
    st = Step([40, 40], [70, 70], 4, 2, 64, 16, BF, seed=16)
    view = st.cache.plan_window(st.plan, 30, 0, q_heads=4)
    at, _ = WorkLists.offsets(view.room)
    assert view.buf[1] == 2 and view.buf[0] == 0  # two items, no units
    view.buf[at[1] + field] = value
    out = torch.full((140, 256), 7, dtype=BF, device=DEV)
    st.cache.window_attention_step(0, st.q[0], view, out)
    with pytest.raises(_lib.NifreError, match="bad slot=1"):
        st.cache.check_status()
    assert int((out == 7).all(1).sum()) == 70  # the other sequence's rows are there


@pytest.mark.parametrize("shape", [SHAPES[i] for i in (0, 3, 5)], ids=[IDS[i] for i in (0, 3, 5)])
def test_captured_decode_steps_with_refilled_plans(shape):
    """A CUDA graph of a layer's append and windowed attention, replayed over the next steps of the batch with
    plan(fixed_layout=True) and plan_window(into=...)."""
    from nifre_b200 import PagedKVCache
    hq, hkv, d, bs, dtype = shape
    S, ctx = 5, [3, 100, 47, 260, 15]
    st = Step(ctx, [1] * S, hq, hkv, d, bs, dtype, seed=13, room=64)
    cache = st.cache
    q, out = torch.empty(S, hq * d, dtype=dtype, device=DEV), torch.empty(S, hq * d, dtype=dtype, device=DEV)
    k, v = (torch.empty(S, hkv * d, dtype=dtype, device=DEV) for _ in range(2))
    graph = view = key = None
    replays = 0
    for step in range(12):
        for t in (q, k, v):
            t.copy_(st.rand(*t.shape))
        plan = cache.plan(range(S), [1] * S, range(S), q_heads=hq, fixed_layout=True)
        fresh = view is None or plan.layout_key != key
        view = cache.plan_window(plan, 40, 4, q_heads=hq, into=None if fresh else view)
        if fresh:
            key = plan.layout_key
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                cache.append_step(0, k, v, plan)
                cache.window_attention_step(0, q, view, out)
        else:
            cache._close(plan)
            replays += 1
        graph.replay()
        for s in range(S):
            st.k[s] = torch.cat([st.k[s], k[s].view(1, 1, hkv, d)], 1)
            st.v[s] = torch.cat([st.v[s], v[s].view(1, 1, hkv, d)], 1)
            c = st.k[s].shape[1] - 1
            ref, wabs, most = attend(q[s].view(1, hq, d), st.k[s][0], st.v[s][0], window_seen(c, 1, 40, 4), d ** -0.5)
            tol = tolerance(ref, wabs, most, c + 1, d, dtype)
            assert ((out[s].view(1, hq, d).double() - ref).abs() <= tol).all(), (step, s)
    assert replays >= 6
    cache.check_status()


def test_refilled_plan_on_another_stream():
    """A call on another stream than the refill's, whose stream is busy, waits for the refill."""
    st = Step([2000, 700], [1, 1], 8, 8, 64, 16, BF, seed=15)
    view = st.cache.plan_window(st.plan, 100, 4, q_heads=8)
    other, out = torch.cuda.Stream(), torch.zeros_like(st.q[0])
    torch.cuda.synchronize()
    with torch.cuda.stream(other):
        st.cache.window_attention_step(0, st.q[0], view, out)
    torch.cuda.synchronize()
    st.ctx = [c + 1 for c in st.ctx]
    st.plan = st._append([0, 1], [1, 1], st.start, st.rows, q_heads=8)
    torch.cuda.synchronize()
    torch.cuda._sleep(20_000_000)
    assert st.cache.plan_window(st.plan, 100, 4, q_heads=8, into=view) is view
    with torch.cuda.stream(other):
        st.cache.window_attention_step(0, st.q[0], view, out)
    torch.cuda.synchronize()
    st.check(out, lambda s: window_seen(st.ctx[s], st.n[s], 100, 4))


def test_refill_and_calls_on_another_stream_than_the_plans():
    """A plan made on a busy stream, refilled and called on another one and dropped at once: the first upload does not
    come after the refill, and the first stream's allocations do not get the plan's memory while the other runs."""
    st = Step([2000, 700], [1, 1], 8, 8, 64, 16, BF, seed=24)
    other = torch.cuda.Stream()
    warm = st.cache.plan_window(st.plan, 100, 4, q_heads=8)
    out = torch.empty_like(st.q[0])
    st.cache.window_attention_step(0, st.q[0], warm, out)
    outs = [torch.zeros_like(out) for _ in range(2)]
    torch.cuda.synchronize()
    torch.cuda._sleep(200_000_000)
    view = st.cache.plan_window(st.plan, 100, 4, q_heads=8)
    sizes = view.buf.numel(), view.ws.numel()
    st.ctx = [c + 1 for c in st.ctx]
    with torch.cuda.stream(other):
        st.plan = st._append([0, 1], [1, 1], st.start, st.rows, q_heads=8)
        assert st.cache.plan_window(st.plan, 100, 4, q_heads=8, into=view) is view
        st.cache.window_attention_step(0, st.q[0], view, outs[0])
        torch.cuda._sleep(200_000_000)
        st.cache.window_attention_step(0, st.q[0], view, outs[1])
    del view
    other_bufs = [torch.zeros(sizes[0], dtype=torch.int32, device=DEV), torch.full((sizes[1],), 5.0, device=DEV)]
    torch.cuda.synchronize()
    assert int(other_bufs[0].count_nonzero()) == 0 and bool((other_bufs[1] == 5).all())
    for o in outs:
        st.check(o, lambda s: window_seen(st.ctx[s], st.n[s], 100, 4))


def test_two_plans_on_two_streams():
    """Plans have work queues and partial rows of their own: different plans' calls may overlap."""
    st = Step([2000, 1500, 900], [1, 8, 20], 32, 8, 64, 16, BF, seed=14)
    views = [st.cache.plan_window(st.plan, 1200, 4, q_heads=32) for _ in range(2)]
    want = torch.empty_like(st.q[0])
    st.cache.window_attention_step(0, st.q[0], views[0], want)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [torch.zeros_like(want) for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for view, stream, out in zip(views, streams, outs):
            with torch.cuda.stream(stream):
                st.cache.window_attention_step(0, st.q[0], view, out)
    torch.cuda.synchronize()
    for out in outs:
        assert torch.equal(out, want)  # and the same bits every time
    st.cache.check_status()


def test_attention_module_with_a_window():
    """Attention(window=...) over padded prefills and decodes, layers with and without windows sharing a step."""
    from nifre_b200 import Attention, PagedKVCache
    g = torch.Generator().manual_seed(15)
    hq, hkv, d, L = 8, 2, 64, 3
    cache = PagedKVCache(L, 256, hkv, d, device=DEV, dtype=BF, block_size=16, enable_prefix_cache=False)
    cache.init_batch(3)
    layers = [Attention(hq, d, window=20, sinks=3), Attention(hq, d), Attention(hq, d, window=5)]
    ks = [[torch.empty(0, hkv, d, dtype=BF, device=DEV) for _ in range(3)] for _ in range(L)]
    vs = [[t.clone() for t in r] for r in ks]
    rand = lambda *s: torch.randn(*s, generator=g).to(BF).to(DEV)  # noqa: E731
    for T, lens in ((50, [50, 17, 33]), (1, None), (1, None), (4, [4, 1, 3])):
        for layer, att in enumerate(layers):
            q, k, v = rand(3, T, hq * d), rand(3, T, hkv * d), rand(3, T, hkv * d)
            out = att(q, k, v, kv_cache=cache, layer_id=layer, input_lens=lens)
            for b in range(3):
                n = lens[b] if lens else T
                assert torch.count_nonzero(out[b, :T - n]) == 0
                c = ks[layer][b].shape[0]
                ks[layer][b] = torch.cat([ks[layer][b], k[b, T - n:].view(n, hkv, d)])
                vs[layer][b] = torch.cat([vs[layer][b], v[b, T - n:].view(n, hkv, d)])
                seen = window_seen(c, n, att.window or 1 << 20, att.sinks)
                ref, wabs, most = attend(q[b, T - n:].view(n, hq, d), ks[layer][b], vs[layer][b], seen, d ** -0.5)
                tol = tolerance(ref, wabs, most, c + n, d, BF)
                assert ((out[b, T - n:].view(n, hq, d).double() - ref).abs() <= tol).all()
    cache.check_status()
