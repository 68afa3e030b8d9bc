"""Copying, forking, compacting and freeing blocks of the cache on the GPU: bit for bit (needs a B200)."""

import pytest
import torch

from oracle.masked import attend, tolerance, tree_seen, window_seen

pytestmark = pytest.mark.gpu

DEV = "cuda"


def _cache(L=2, hkv=2, d=64, bs=16, dtype=torch.bfloat16, slots=6, max_len=256, num_blocks=None, prefix=False):
    from nifre_b200 import PagedKVCache
    c = PagedKVCache(L, max_len, hkv, d, device=DEV, dtype=dtype, block_size=bs, enable_prefix_cache=prefix,
                     num_blocks=num_blocks)
    c.init_batch(slots)
    return c


def _grow(cache, slots, lens, g, model):
    """Append random rows; ``model[slot]``: [layers][2] lists of the rows a slot should hold."""
    w = cache.n_heads * cache.head_dim
    starts = [sum(lens[:i]) for i in range(len(lens))]
    plan = cache.plan(slots, lens, starts, q_heads=cache.n_heads)
    for layer in range(cache.num_layers):
        k, v = (torch.randn(sum(lens), w, generator=g).to(cache.dtype).to(DEV) for _ in range(2))
        cache.append_step(layer, k, v, plan)
        for s, n, st in zip(slots, lens, starts):
            for i, t in enumerate((k, v)):
                model[s][layer][i] = torch.cat([model[s][layer][i], t[st:st + n].view(n, cache.n_heads, -1)])
    return plan


def _model(cache):
    empty = lambda: torch.empty(0, cache.n_heads, cache.head_dim, dtype=cache.dtype, device=DEV)  # noqa: E731
    return {s: [[empty(), empty()] for _ in range(cache.num_layers)] for s in range(cache.batch_size)}


def _copy(model, s):
    return [[t.clone() for t in pair] for pair in model[s]]


def _cut(model, s, n):
    return [[t[:n].clone() for t in pair] for pair in model[s]]


def _same(cache, model):
    for s in range(cache.batch_size):
        assert cache.length(s) == int(cache.pos[s]) == model[s][0][0].shape[0], s
        for layer in range(cache.num_layers):
            k, v = cache.get(s, layer)
            assert torch.equal(k, model[s][layer][0]) and torch.equal(v, model[s][layer][1]), (s, layer)
    live = {b for t in cache.block_tables for b in t.physical_blocks()}
    if cache.prefix_cache is not None:
        live |= set(cache.prefix_cache.entries.values())
    assert cache.block_allocator.allocated_count == len(live)
    cache.check_status()


@pytest.mark.parametrize("dtype,hkv,d,bs", [(torch.bfloat16, 2, 64, 16), (torch.float32, 3, 32, 5),
                                            (torch.float16, 1, 7, 3), (torch.float16, 8, 128, 32)])
@pytest.mark.parametrize("n", [1, 200])
def test_copy_blocks(dtype, hkv, d, bs, n):
    g = torch.Generator().manual_seed(n)
    c = _cache(L=3, hkv=hkv, d=d, bs=bs, dtype=dtype, num_blocks=401)
    for t in (*c.k, *c.v):
        t.copy_(torch.randn(t.shape, generator=g).to(dtype))
    ids = torch.randperm(401, generator=g).tolist()
    src, dst = ids[:n], ids[n:2 * n]
    want = [t.clone() for t in (*c.k, *c.v)]
    for t in want:
        t[dst] = t[src]
    before = [t.clone() for t in (*c.k, *c.v)]
    c.copy_blocks(src, dst)
    assert all(torch.equal(a, b) for a, b in zip((*c.k, *c.v), want))
    for t, b in zip((*c.k, *c.v), before):
        t.copy_(b)
    s = torch.tensor(src, dtype=torch.int32, device=DEV)
    e = torch.tensor(dst, dtype=torch.int32, device=DEV)
    c.copy_blocks(s, e)
    assert all(torch.equal(a, b) for a, b in zip((*c.k, *c.v), want))
    c.copy_blocks([], [])
    c.copy_blocks(s[:0], e[:0])
    c.check_status()
    from nifre_b200 import _lib
    e[0] = 401
    c.copy_blocks(s, e)
    with pytest.raises(_lib.NifreError, match="bad block=1"):
        c.check_status()
    with pytest.raises(ValueError, match="destinations"):
        c.copy_blocks(s, e[:0])


@pytest.mark.parametrize("bs", [16, 5])
def test_fork_shares_full_blocks_and_copies_the_last(bs):
    g = torch.Generator().manual_seed(0)
    c = _cache(bs=bs)
    m = _model(c)
    _grow(c, [0, 1], [37, 2 * bs], g, m)
    used = c.allocated_blocks
    c.fork([0, 0, 1], [2, 3, 4])
    m[2], m[3], m[4] = _copy(m, 0), _copy(m, 0), _copy(m, 1)
    assert c.allocated_blocks == used + 2  # a tail each for slots 2 and 3, none for slot 4
    _same(c, m)
    _grow(c, [0, 2, 3, 4, 1], [1, 20, 2, 7, bs], g, m)  # they part ways
    _same(c, m)
    c.fork([2, 2, 2], [0, 1, 4])  # over what they held
    m[0], m[1], m[4] = _copy(m, 2), _copy(m, 2), _copy(m, 2)
    _same(c, m)
    tables = [t.physical_blocks() for t in c.block_tables]
    _grow(c, [0], [1], g, m)
    c.fork([2, 2, 2], [0, 1, 4])  # again: the slots keep their own last blocks
    m[0] = _copy(m, 2)
    _same(c, m)
    assert [t.physical_blocks()[:len(tables[i])] for i, t in enumerate(c.block_tables)] == tables
    c.fork([5], [0])  # an empty sequence
    m[0] = _copy(m, 5)
    _same(c, m)
    for s in range(6):
        c.reset_slot(s)
    assert c.allocated_blocks == 0


def test_fork_of_many_slots_and_an_exhausted_pool():
    from nifre_b200 import BlockPoolExhaustedError
    g = torch.Generator().manual_seed(1)
    c = _cache(L=1, slots=300, max_len=32, num_blocks=301)
    m = _model(c)
    _grow(c, [0, 1], [17, 3], g, m)
    c.fork([0] * 298, range(2, 300))  # lists of more records than the kernel arguments hold
    for s in range(2, 300):
        m[s] = _copy(m, 0)
    _same(c, m)
    c.reset_slot(7)
    _grow(c, [1], [20], g, m)
    m[7] = _copy({0: [[t[:0] for t in p] for p in m[1]]}, 0)
    with pytest.raises(BlockPoolExhaustedError):
        c.fork([1, 1], [7, 0])
    m[0] = m[7]
    _same(c, m)


def test_truncate_copies_a_shared_last_block():
    g = torch.Generator().manual_seed(2)
    c = _cache()
    m = _model(c)
    _grow(c, [0], [50], g, m)
    c.fork([0], [1])
    m[1] = _copy(m, 0)
    c.truncate(1, 20)  # into a block that slot 0 holds too
    m[1] = _cut(m, 1, 20)
    _same(c, m)
    _grow(c, [1, 0], [15, 3], g, m)
    _same(c, m)
    for n in (32, 31, 16, 0):
        c.truncate(0, n)
        m[0] = _cut(m, 0, n)
        _same(c, m)
    _grow(c, [0], [40], g, m)
    _same(c, m)


@pytest.mark.parametrize("bs", [16, 5])
def test_keep_tokens_moves_the_accepted_path(bs):
    g = torch.Generator().manual_seed(3)
    c = _cache(bs=bs)
    m = _model(c)
    ctx = [0, 13, 16, 31, 40, 2]
    _grow(c, [s for s in range(6) if ctx[s]], [x for x in ctx if x], g, m)
    paths = [[0], [0, 1, 2], [1, 2, 3, 9], [], [2, 5, 6, 7, 8, 9, 19], [0, 3, 4, 5, 11]]
    n = [1, 8, 20, 4, 20, 12]
    for _ in range(3):
        at = [c.length(s) for s in range(6)]
        plan = _grow(c, list(range(6)), n, g, m)
        c.keep_tokens(plan, paths)
        for s in range(6):
            keep = list(range(at[s])) + [at[s] + t for t in paths[s]]
            m[s] = [[t[keep].clone() for t in pair] for pair in m[s]]
        k = [[c.get(s, layer) for layer in range(2)] for s in range(6)]
        for s in range(6):
            assert c.length(s) == int(c.pos[s]) == at[s] + len(paths[s])
            for layer in range(2):
                assert torch.equal(k[s][layer][0], m[s][layer][0]) and torch.equal(k[s][layer][1], m[s][layer][1])
    c.check_status()


def test_keep_tokens_leaves_a_fork_alone():
    """A draft whose blocks were forked before the path was kept: the fork still holds the whole draft."""
    g = torch.Generator().manual_seed(4)
    c = _cache()
    m = _model(c)
    _grow(c, [0], [10], g, m)
    plan = _grow(c, [0], [30], g, m)
    c.fork([0], [1])
    m[1] = _copy(m, 0)
    c.keep_tokens(plan, [[3, 9, 20]])
    m[0] = [[t[[*range(10), 13, 19, 30]].clone() for t in pair] for pair in m[0]]
    for s in (0, 1):
        for layer in range(2):
            k, v = c.get(s, layer)
            assert torch.equal(k, m[s][layer][0]) and torch.equal(v, m[s][layer][1])


def test_compact_moves_live_blocks_and_the_prefix_index():
    g = torch.Generator().manual_seed(5)
    c = _cache(prefix=True, num_blocks=60)
    m = _model(c)
    c.block_allocator.set_free_order(torch.randperm(60, generator=g).tolist())
    ids = list(range(48))
    _grow(c, [0, 1, 2], [48, 30, 70], g, m)
    c.register_prefix(0, ids)
    c.fork([2], [3])
    m[3] = _copy(m, 2)
    c.reset_slot(1)
    m[1] = _cut(m, 1, 0)
    _same(c, m)
    live = c.compact()
    assert live == c.allocated_blocks
    held = {b for t in c.block_tables for b in t.physical_blocks()} | set(c.prefix_cache.entries.values())
    assert held == set(range(live))
    _same(c, m)
    assert c.try_load_prefix(4, ids) == 48
    m[4] = _copy(m, 0)
    _same(c, m)
    _grow(c, [4, 0, 2], [5, 5, 5], g, m)
    _same(c, m)
    assert c.compact() == c.allocated_blocks  # nothing left to move, or blocks at the end
    _same(c, m)


@pytest.mark.parametrize("bs,window,sinks", [(16, 40, 4), (16, 16, 0), (5, 30, 7), (32, 64, 40)])
def test_freed_blocks_behind_a_window(bs, window, sinks):
    """A stream that frees what its window leaves behind: bounded blocks, the same outputs, refusals elsewhere."""
    g = torch.Generator().manual_seed(6)
    hq, hkv, d, dtype = 4, 2, 64, torch.bfloat16
    bound = -(-(window + 16) // bs) + -(-sinks // bs) + 16 // bs + 4
    c = _cache(L=1, bs=bs, slots=2, max_len=2000, num_blocks=bound + 9)
    m = _model(c)
    steps = [9, 1, 1, 17, 1, 3, 16, 1] * 16
    for i, n in enumerate(steps):
        at = c.length(0)
        plan = _grow(c, [0], [n], g, m)
        q = torch.randn(n, hq * d, generator=g).to(dtype).to(DEV)
        view = c.plan_window(plan, window, sinks, q_heads=hq)
        out = torch.zeros_like(q)
        c.window_attention_step(0, q, view, out)
        ref, wabs, most = attend(q.view(n, hq, d), m[0][0][0], m[0][0][1], window_seen(at, n, window, sinks), d ** -0.5)
        assert ((out.view(n, hq, d).double() - ref).abs() <= tolerance(ref, wabs, most, at + n, d, dtype)).all(), i
        c.free_outside_window(0, window, sinks)
        assert c.allocated_blocks <= bound + 9
    c.check_status()
    assert c.length(0) > (bound + 9) * bs  # more tokens went by than the pool holds
    assert c._hole_end[0] > 0
    with pytest.raises(ValueError, match="freed"):
        c.get(0, 0)
    plan = c.plan([0], [1], [0], q_heads=hq)
    one = torch.zeros(1, hq * d, dtype=dtype, device=DEV)
    with pytest.raises(ValueError, match="window_attention_step"):
        c.attention_step(0, one, plan, one.clone())
    with pytest.raises(ValueError, match="freed"):
        c.plan_window(plan, 4 * window + 200, sinks, q_heads=hq)
    with pytest.raises(ValueError, match="freed"):
        c.plan_window(plan, window, sinks + 300, q_heads=hq)
    with pytest.raises(ValueError, match="freed"):
        c.plan_tree(plan, [None], q_heads=hq)
    c.append_step(0, one[:, :hkv * d], one[:, :hkv * d], plan)
    with pytest.raises(ValueError, match="freed"):
        c.truncate(0, int(c._hole_end[0]) - 1)
    # a fork of it shares the holes
    c.fork([0], [1])
    assert c._hole_end[1] == c._hole_end[0]
    c.reset_slot(0)
    c.reset_slot(1)
    assert c.allocated_blocks == 0 and not c._hole_end.any()
    _grow(c, [0], [20], g, {0: _model(c)[0]})
    c.check_status()


def test_speculative_decoding_run():
    """The operators together: a prompt, forks of it, drafted trees verified and kept step after step, beside plain
    decodes, the outputs always those of a sequence written token by token."""
    from nifre_b200 import tree_visibility
    g = torch.Generator().manual_seed(7)
    hq, hkv, d, dtype = 8, 2, 64, torch.bfloat16
    c = _cache(L=2, slots=4)
    m = _model(c)
    _grow(c, [0], [45], g, m)
    c.fork([0, 0], [1, 2])
    m[1], m[2] = _copy(m, 0), _copy(m, 0)
    trees = [[-1, 0, 0, 1, 1, 2], [-1, -1, 0, 1, 3, 4, 2, 5], [-1]]
    paths = [[0, 1, 4], [1, 3, 4, 5, 7], [0]]
    rand = lambda *s: torch.randn(*s, generator=g).to(dtype).to(DEV)  # noqa: E731
    for step in range(5):
        at = [c.length(s) for s in range(3)]
        n = [len(t) for t in trees]
        plan = c.plan([0, 1, 2], n, [0, 6, 14], q_heads=hq)
        view = c.plan_tree(plan, trees, q_heads=hq)
        for layer in range(2):
            q, k, v = rand(15, hq * d), rand(15, hkv * d), rand(15, hkv * d)
            c.append_step(layer, k, v, plan)
            out = c.tree_attention_step(layer, q, view, torch.zeros_like(q))
            for s, st in zip(range(3), (0, 6, 14)):
                for i, t in enumerate((k, v)):
                    m[s][layer][i] = torch.cat([m[s][layer][i], t[st:st + n[s]].view(n[s], hkv, d)])
                seen = tree_seen(at[s], torch.as_tensor(tree_visibility(trees[s])))
                ref, wabs, most = attend(q[st:st + n[s]].view(n[s], hq, d), *m[s][layer], seen, d ** -0.5)
                tol = tolerance(ref, wabs, most, at[s] + n[s], d, dtype)
                assert ((out[st:st + n[s]].view(n[s], hq, d).double() - ref).abs() <= tol).all(), (step, s)
        c.keep_tokens(plan, paths)
        for s in range(3):
            keep = list(range(at[s])) + [at[s] + t for t in paths[s]]
            m[s] = [[t[keep].clone() for t in pair] for pair in m[s]]
            assert c.length(s) == len(keep)
        if step == 2:
            c.truncate(1, 50)
            m[1] = _cut(m, 1, 50)
            c.fork([1], [3])
            m[3] = _copy(m, 1)
            c.reset_slot(3)
            m[3] = _cut(m, 3, 0)
            c.compact()
    for s in range(3):
        c.truncate(s, c.length(s))
    _same(c, m)


@pytest.mark.parametrize("slots", [2, 140])
@pytest.mark.parametrize("how", ["compacted", "reused"])
def test_keep_tokens_moves_paths_longer_than_a_block(slots, how):
    """Paths of 30 rows in a row, in blocks with consecutive ids (after compact(), and in slots that were cleared and
    filled again); lists that travel as arguments and lists in device memory."""
    g = torch.Generator().manual_seed(8)
    c = _cache(L=2, hkv=1, slots=slots, max_len=64, num_blocks=4 * slots)
    m = _model(c)
    every = list(range(slots))
    if how == "reused":
        _grow(c, every, [60] * slots, g, m)
        for s in every:
            c.reset_slot(s)
            m[s] = _cut(m, s, 0)
    else:
        c.block_allocator.set_free_order(torch.randperm(c.num_blocks, generator=g).tolist())
    _grow(c, every, [20] * slots, g, m)
    plan = _grow(c, every, [40] * slots, g, m)
    if how == "compacted":
        c.reset_slot(slots - 1)
        m[slots - 1] = _cut(m, slots - 1, 0)
        c.compact()
        plan = None
        for s in every:
            c.truncate(s, min(c.length(s), 20))
            m[s] = _cut(m, s, 20)
        _grow(c, [slots - 1], [20], g, m)
        c.compact()
        plan = _grow(c, every, [40] * slots, g, m)
    paths = [list(range(1, 31)) for _ in every]
    paths[0] = [0, 2, *range(5, 38)]
    c.keep_tokens(plan, paths)
    for s in every:
        m[s] = [[t[[*range(20), *(20 + j for j in paths[s])]].clone() for t in pair] for pair in m[s]]
        c.truncate(s, c.length(s))
    _same(c, m)
