"""Work lists and host checks of windowed and tree attention and of the page operators (CPU only)."""

import ctypes

import numpy as np
import pytest
import torch

from nifre_b200 import Attention, PagedKVCache, _lib
from nifre_b200.block_allocator import BlockAllocator
from nifre_b200.block_table import BlockTable
from nifre_b200.masked import WorkLists, build_lists, even_shares, mask_words, tree_visibility, virtual_keys
from oracle.masked import window_seen


def _keys_of(pos0, ntok, window, sinks):
    """kept, gap and count of the virtual keys of a group."""
    return [int(x[0]) for x in virtual_keys(np.asarray([pos0]), np.asarray([ntok]), window, sinks)]


@pytest.mark.parametrize("window,sinks", [(1, 0), (7, 1), (16, 16), (100, 4), (1000, 40), (1 << 30, 0), (33, 1 << 30)])
@pytest.mark.parametrize("rows", [(16, 0), (8, 256), (32, 128)])
def test_units_cover_each_tokens_keys_once(window, sinks, rows):
    """Every key a token sees is read exactly once by its group's units, every token is in one group, parts are
    numbered in order, and the merge records cover exactly the rows of groups with several parts."""
    rng = np.random.default_rng(window + sinks)
    S = 9
    n = rng.integers(1, 90, size=S)
    n[:3] = 1
    ctx = rng.integers(0, 700, size=S)
    ctx[0] = 0
    slots = rng.permutation(20)[:S]
    starts = np.cumsum(n) - n + 3
    unit_rows, item_rows = rows
    group = 4
    lists = build_lists(slots, n, starts, ctx, group, unit_rows, item_rows, workers=8, kv_heads=2, window=window,
                        sinks=sinks, unit_share=64, item_share=256)
    units, cover = {}, {}
    for kind, recs in (("unit", lists.units), ("item", lists.items)):
        for k0, k1, pp, zero, *g in recs.tolist():
            assert k0 % (128 if kind == "item" else 16) == 0 and k0 < k1 and zero == 0
            units.setdefault(tuple(g), []).append((pp & 0xffff, k0, k1, pp >> 16, kind))
    merged = {tuple(r) for r in lists.merge.tolist()}
    n_merge = 0
    taken = np.zeros(lists.part_rows, dtype=int)
    for g, us in units.items():
        slot, q0, ntok, pos0, c, nd, _, part0 = g
        s = slots.tolist().index(slot)
        assert c == ctx[s] and nd == n[s] and q0 - starts[s] == pos0 - ctx[s]
        for t in range(ntok):
            assert (s, pos0 + t) not in cover
            cover[(s, pos0 + t)] = g
        us = sorted(us)
        kept, gap, count = _keys_of(pos0, ntok, window, sinks)
        assert [u[0] for u in us] == list(range(len(us))) and {u[3] for u in us} == {len(us)}
        assert us[0][1] == 0 and us[-1][2] == count and all(a[2] == b[1] for a, b in zip(us, us[1:]))
        limit = item_rows if us[0][4] == "item" else max(unit_rows, group)
        assert ntok * group <= limit and len({u[4] for u in us}) == 1
        read = [v if v < kept else v + gap for v in range(count)]
        assert len(set(read)) == len(read)
        seen = window_seen(int(pos0), int(ntok), window, sinks)
        assert set(seen.any(0).nonzero().squeeze(1).tolist()) <= set(read)
        if len(us) > 1:
            taken[part0:part0 + len(us) * ntok] += 1
            for row in range(0, ntok * group, 4):
                assert (len(us), row, int(us[0][4] == "item"), 0, *g) in merged
                n_merge += 1
    for recs, shares in ((lists.units, lists.unit_shares), (lists.items, lists.item_shares)):
        assert not len(recs) or (shares[0] == 0 and shares[-1] == len(recs) and (np.diff(shares) > 0).all())
    assert len(cover) == n.sum()
    assert n_merge == len(merged) == len(lists.merge) and (taken == 1).all()


def test_tree_lists_carry_every_mask_row():
    parents = [[-1, 0, 0, 1], [-1] * 40, [-1]]
    words = [mask_words(tree_visibility(p)) for p in parents]
    lists = build_lists([2, 0, 1], [4, 40, 1], [0, 4, 44], [100, 0, 5], 8, 16, 0, 8, 1, words=words, unit_share=64)
    for _, _, _, _, slot, q0, ntok, pos0, ctx, nd, mask0, _ in lists.units.tolist():
        s = [2, 0, 1].index(slot)
        seen = tree_visibility(parents[s])
        w = (nd + 31) // 32
        for t in range(ntok):
            row = lists.masks[mask0 + t * w: mask0 + (t + 1) * w].astype(np.uint32)
            bits = [(int(row[j // 32]) >> (j % 32)) & 1 for j in range(nd)]
            assert bits == seen[pos0 - ctx + t].astype(int).tolist()


def test_tree_visibility_and_bits():
    assert tree_visibility([-1, 0, 1, 0, -1]).astype(int).tolist() == [
        [1, 0, 0, 0, 0], [1, 1, 0, 0, 0], [1, 1, 1, 0, 0], [1, 0, 0, 1, 0], [0, 0, 0, 0, 1]]
    for bad in ([0], [-1, 1], [-2], [-1, 0, 5]):
        with pytest.raises(ValueError, match="parents"):
            tree_visibility(bad)
    rng = np.random.default_rng(0)
    for n in (1, 31, 32, 33, 64, 65):
        seen = rng.integers(0, 2, size=(n, n)).astype(bool)
        w = mask_words(seen).astype(np.uint32)
        assert w.shape == (n, (n + 31) // 32)
        back = [[(int(w[i, j // 32]) >> (j % 32)) & 1 for j in range(n)] for i in range(n)]
        assert back == seen.astype(int).tolist()


def test_shares_of_the_other_kernels():
    """Groups of more than 8 rows are cut where there are fewer of them than CTAs, by length; never below 64 keys."""
    from nifre_b200.masked import unit_share_for
    rows, cut = np.array([16]), lambda keys, n, d=64: unit_share_for(np.full(n, keys), rows, 148, 12, d, 0)
    assert cut(500, 25) == 0 and cut(100, 1) == 0
    assert cut(3000, 1) == 128 and cut(200, 1) == 64
    assert 1024 >= cut(4000, 25) >= 512
    assert cut(3000, 1, 256) == 2 * cut(3000, 1, 128)
    assert unit_share_for(np.array([3000]), np.array([8]), 148, 12, 64, 0) >= 128


def test_even_shares_cover_every_group_in_order():
    rng = np.random.default_rng(1)
    for n, most, share, align in ((1, 5, 64, 16), (9, 3000, 448, 16), (40, 200, 64, 16), (5, 9000, 256, 128), (64, 1041, 464, 16)):
        keys = rng.integers(1, most, size=n)
        least = 4 * align
        each = int(rng.integers(0, 60))
        g, k0, k1, at = even_shares(keys, share, align, least, each)
        assert (k0 < k1).all() and (k0 % align == 0).all()
        assert (np.diff(g) >= 0).all() and set(g.tolist()) == set(range(n))
        for i in range(n):
            mine = g == i
            assert k0[mine][0] == 0 and k1[mine][-1] == keys[i] and (k1[mine][:-1] == k0[mine][1:]).all()
            if mine.sum() > 1:
                assert (k1[mine] - k0[mine]).min() >= min(least, share - align)
        assert at[0] == 0 and at[-1] == len(g) and (np.diff(at) > 0).all()
        sizes = np.add.reduceat(k1 - k0, at[:-1])
        assert sizes.max() <= share + 2 * (least + align)  # each bound moves by less than least and the rounding


def test_packed_lists_and_room():
    lists = build_lists([0, 1], [1, 40], [0, 1], [500, 20], 4, 16, 0, 4, 1, window=300, sinks=3, unit_share=64)
    room = lists.room(lists.sizes())
    assert all(r >= n and r % 64 == 0 for r, n in zip(room[:5], lists.sizes()[:5]))
    host = lists.pack(room)
    at, total = WorkLists.offsets(room)
    assert len(host) == total and all(a % 4 == 0 for a in at)
    assert host[:8].tolist() == [len(lists.unit_shares) - 1, 0, len(lists.merge), len(lists.units), 0, 0, 0, 0]
    assert host[at[4]:at[4] + len(lists.unit_shares)].tolist() == lists.unit_shares.tolist()
    assert host[at[0]:at[0] + lists.units.size].tolist() == lists.units.reshape(-1).tolist()


def test_too_many_parts_are_refused():
    with pytest.raises(ValueError, match="parts"):
        build_lists([0], [1], [0], [40_000 * 64], 1, 16, 0, 1, 1, window=1 << 30, unit_share=64)


def test_masked_arguments_struct_matches_the_header(tmp_path):
    import shutil
    import subprocess
    from pathlib import Path
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "nifre_b200.h"', 'int main(void) {',
             '  printf("%zu %d\\n", sizeof(NfMaskedArgs), NF_MOVE_LIST);']
    lines += [f'  printf("%zu\\n", offsetof(NfMaskedArgs, {f}));' for f, _ in _lib.NfMaskedArgs._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["  return 0;\n}"]))
    root = Path(__file__).resolve().parent.parent
    subprocess.check_call([cc, "-I", str(root / "include"), str(src), "-o", str(exe)])
    got = [int(x) for x in subprocess.check_output([str(exe)], text=True).split()]
    assert got == [ctypes.sizeof(_lib.NfMaskedArgs), _lib.MOVE_LIST,
                   *(getattr(_lib.NfMaskedArgs, f).offset for f, _ in _lib.NfMaskedArgs._fields_)]


def _args(**kw):
    base = dict(out=256, q=256, k_pool=256, v_pool=256, block_tables=256, units=256, items=256, merge=256,
                unit_shares=256, item_shares=256, counts=256, masks=256, mask_words=4, ws=256, ws_rows=4, queue=256, status=256, dtype=2, num_q_heads=8,
                num_kv_heads=2, head_dim=64, block_size=16, num_blocks=4, num_slots=1, max_blocks_per_seq=4, num_rows=1,
                max_units=1, unit_tokens=1, max_items=0, max_merge=0, window=4, sinks=0, scale=1.0)
    base.update(kw)
    return _lib.NfMaskedArgs(**base)


@pytest.mark.parametrize("change,match", [
    (dict(dtype=7), "dtype"), (dict(num_q_heads=7), "multiple"), (dict(num_kv_heads=0), "multiple"),
    (dict(num_q_heads=1 << 13, num_kv_heads=1), "at most"), (dict(head_dim=257), "head_dim"), (dict(head_dim=0), "head_dim"),
    (dict(block_size=0), "sizes"), (dict(num_rows=0), "sizes"), (dict(max_units=-1), "work list"),
    (dict(max_units=0), "work list"), (dict(unit_tokens=0), "unit_tokens"), (dict(unit_tokens=1 << 20), "unit_tokens"),
    (dict(q=None), "null"), (dict(units=None), "null"), (dict(ws=None), "null"), (dict(status=None), "null"),
    (dict(q_row_stride=-1), "stride"), (dict(units=260), "aligned"), (dict(q=257), "aligned"),
    (dict(window=0), "window"), (dict(sinks=-1), "sinks")])
def test_window_entry_point_refuses(change, match):
    """Host-side checks: nothing is launched."""
    lib = _lib.load()
    a = _args(**change)
    assert lib.nf_window_attention(ctypes.addressof(a), None) in (1, 3)
    assert match in lib.nf_last_error().decode()


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), float("-inf")])
def test_a_scale_that_is_not_finite_is_refused(scale):
    lib = _lib.load()
    for fn in (lib.nf_window_attention, lib.nf_tree_attention):
        a = _args(scale=scale)
        assert fn(ctypes.addressof(a), None) == 1 and b"scale" in lib.nf_last_error()


def test_tree_entry_point_and_limits_refuse():
    lib = _lib.load()
    a = _args(masks=None)
    assert lib.nf_tree_attention(ctypes.addressof(a), None) == 1 and b"mask" in lib.nf_last_error()
    assert lib.nf_tree_attention(None, None) == 1
    x, y = ctypes.c_int32(0), ctypes.c_int32(0)
    assert lib.nf_masked_limits(2, 8, 2, 64, 16, ctypes.byref(x), ctypes.byref(y)) == 0 and x.value >= 4
    assert lib.nf_masked_limits(2, 8, 3, 64, 16, ctypes.byref(x), ctypes.byref(y)) == 1
    assert lib.nf_masked_limits(2, 8, 2, 300, 16, ctypes.byref(x), ctypes.byref(y)) == 3


def test_move_entry_points_refuse():
    lib = _lib.load()

    def move(**kw):
        d = dict(k=256, v=256, ls=0, layers=1, row=16, rows=4, moves=256, n=1, most=1, pos=None, n_pos=0, pos_out=None,
                 slots=0, dev=1, status=256)
        d.update(kw)
        return lib.nf_kv_move(d["k"], d["v"], d["ls"], d["layers"], d["row"], d["rows"], d["moves"], d["n"], d["most"],
                              d["pos"], d["n_pos"], d["pos_out"], d["slots"], d["dev"], d["status"], None)

    for bad in (dict(k=None), dict(row=0), dict(row=3), dict(layers=0), dict(rows=0), dict(n=-1), dict(moves=None),
                dict(n_pos=1), dict(k=257), dict(moves=258), dict(dev=0, n=129), dict(status=None)):
        assert move(**bad) == 1, bad
    assert move(n=0) == 0
    rec = np.asarray([[0, 1, 5, 0]], dtype=np.int32)  # more rows than max_rows
    assert move(dev=0, moves=rec.ctypes.data) == 1 and b"max_rows" in lib.nf_last_error()
    assert lib.nf_copy_blocks(256, 256, 0, 1, 32, 4, None, None, 1, 256, None) == 1
    assert lib.nf_copy_blocks(256, 256, 0, 1, 32, 4, None, None, 0, 256, None) == 0


def test_attention_window_arguments():
    with pytest.raises(ValueError, match="sinks need"):
        Attention(4, 64, sinks=2)
    for w, s in ((0, 0), (-3, 0), (2.5, 0), (4, -1)):
        with pytest.raises(ValueError, match="window"):
            Attention(4, 64, window=w, sinks=s)
    q = torch.zeros(1, 3, 256)
    with pytest.raises(ValueError, match="needs a kv_cache"):
        Attention(4, 64, window=2)(q, q, q)


# ---------------------------------------------------------------- block bookkeeping
def test_allocator_retains_and_releases_many():
    a, b = BlockAllocator(8), BlockAllocator(8)
    x, y = a.allocate_many(5), b.allocate_many(5)
    assert x == y
    a.retain_many([x[1], x[3]])
    for i in (x[1], x[3]):
        b.retain(i)
    a.release_many([x[3], x[0], x[4]])
    for i in (x[3], x[0], x[4]):
        b.release(i)
    assert a.free_ids() == b.free_ids() and a.allocated_count == b.allocated_count == 3
    a.release_many([])
    for bad in ([8], [-1]):
        with pytest.raises(ValueError, match="out of range"):
            a.retain_many(bad)
    with pytest.raises(ValueError, match="not allocated"):
        a.release_many([x[0]])


def test_allocator_compaction():
    a = BlockAllocator(10)
    ids = a.allocate_many(7)  # 9 .. 3
    a.release_many([ids[0], ids[4], ids[5]])  # 9, 5, 4
    a.retain(8)
    src, dst = a.compact()
    assert sorted(src) == [6, 7, 8] and len(set(dst)) == 3 and max(dst) < 4 and 3 not in dst
    assert [a.refcount(i) for i in range(5)].count(1) == 3 and sorted(a.refcount(i) for i in range(4)) == [1, 1, 1, 2]
    assert a.refcount(dst[src.index(8)]) == 2
    assert a.allocate_many(2) == [4, 5] and a.free_count == 4
    full = BlockAllocator(3)
    full.allocate_many(3)
    assert full.compact() == ([], [])
    assert BlockAllocator(3).compact() == ([], [])


def test_table_sharing_shrinking_and_freed_entries():
    a = BlockAllocator(10)
    t, u = BlockTable(a, 4), BlockTable(a, 4)
    t.ensure_capacity(20)
    blocks = t.physical_blocks()
    u.share(blocks[:3])
    assert [a.refcount(b) for b in blocks] == [2, 2, 2, 1, 1]
    with pytest.raises(ValueError, match="non-empty"):
        u.share(blocks[:1])
    e = t.epoch
    assert t.free_blocks(1, 3) == 2 and t.free_blocks(1, 3) == 0
    assert t.physical_blocks() == [blocks[0], -1, -1, *blocks[3:]] and a.refcount(blocks[1]) == 1
    with pytest.raises(IndexError, match="no allocated block"):
        t.resolve(5)
    t.shrink(4)
    assert t.epoch != e and len(t) == 4 and a.refcount(blocks[4]) == 0
    t.rename(np.asarray([*range(10), -1]))
    assert t.physical_blocks() == [blocks[0], -1, -1, blocks[3]]
    t.clear()
    u.clear()
    assert a.free_count == 10


def test_page_and_plan_refusals_before_any_launch():
    """Arguments are checked on the host (no CUDA device needed)."""
    from nifre_b200 import KVCache
    from types import SimpleNamespace
    c = PagedKVCache(1, 64, 2, 64, device="cpu", dtype=torch.float16)
    c.batch_size, c.num_blocks, c._dev_index, c._plan = 4, 8, 0, None
    c.pos_host = np.asarray([20, 0, 0, 0])
    c.block_allocator = BlockAllocator(8)
    c.block_tables = [BlockTable(c.block_allocator, 16) for _ in range(4)]
    c._init_holes(4)
    for src, dst, match in (([0], [1, 2], "source slots"), ([0, 0], [1, 1], "distinct"), ([0], [0], "distinct")):
        with pytest.raises(ValueError, match=match):
            c.fork(src, dst)
    with pytest.raises(IndexError, match="out of range"):
        c.fork([0], [4])
    for src, dst in (([0], [1, 2]), ([0, 1], [2, 2]), ([0, 1], [1, 2]), ([8], [0]), ([-1], [0])):
        with pytest.raises(ValueError):
            c.copy_blocks(src, dst)
    with pytest.raises(ValueError, match="int32"):
        c.copy_blocks(torch.zeros(2), torch.ones(2))
    with pytest.raises(_lib.NifreError, match="CUDA tensor"):
        c.copy_blocks(torch.zeros(2, dtype=torch.int32), torch.ones(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="length"):
        c.truncate(0, 21)
    with pytest.raises(ValueError, match="window"):
        c.free_outside_window(0, 0)
    plan = SimpleNamespace(closed=False, slots=np.asarray([0]), ctx_before=np.asarray([16]), q_lens=np.asarray([4]), n_seqs=1,
                           q_heads=4, rows_needed=4, q_starts=np.asarray([0]))
    with pytest.raises(RuntimeError, match="not finished"):
        c.keep_tokens(plan, [[0]])
    plan.closed = True
    for path in ([1, 1], [2, 1], [-1], [4]):
        with pytest.raises(ValueError, match="ascending"):
            c.keep_tokens(plan, [path])
    with pytest.raises(ValueError, match="paths"):
        c.keep_tokens(plan, [])
    plan.ctx_before = np.asarray([10])
    with pytest.raises(ValueError, match="not the 14"):
        c.keep_tokens(plan, [[0]])
    open_plan = SimpleNamespace(closed=False, slots=np.asarray([2]))
    c._plan = open_plan
    with pytest.raises(RuntimeError, match="not finished"):
        c.fork([0], [2])
    with pytest.raises(RuntimeError, match="not finished"):
        c.compact()
    for w, s in ((0, 0), (1.5, 0), (4, -1)):
        with pytest.raises(ValueError, match="window|sinks"):
            c.plan_window(plan, w, s)
    with pytest.raises(ValueError, match="parents or masks"):
        c.plan_tree(plan)
    with pytest.raises(ValueError, match="trees for"):
        c.plan_tree(plan, [])
    with pytest.raises(ValueError, match="a tree of"):
        c.plan_tree(plan, [[-1]])
    with pytest.raises(ValueError, match="q_heads"):
        c.plan_window(plan, 4, q_heads=3)
    c._hole_first[0], c._hole_end[0] = 0, 16
    with pytest.raises(ValueError, match="freed"):
        c.plan_tree(plan, [[-1, 0, 1, 2]])
    with pytest.raises(ValueError, match="were freed"):
        c.plan_window(plan, 100, 0)
    dense = KVCache(1, 64, 2, 64, device="cpu", dtype=torch.float16)
    for call in (lambda: dense.fork([0], [1]), dense.compact):
        with pytest.raises(ValueError, match="dense"):
            call()


def _host_cache(slots=4, num_blocks=40, bs=16, max_len=512):
    """A cache's host side without a device; ``moved``: what _move_rows was asked for."""
    c = PagedKVCache(1, max_len, 2, 64, device="cpu", dtype=torch.float16, block_size=bs)
    c.batch_size, c.num_blocks, c._dev_index = slots, num_blocks, 0
    c.pos_host = np.zeros(slots, dtype=np.int64)
    c.block_allocator = BlockAllocator(num_blocks)
    c.block_tables = [BlockTable(c.block_allocator, bs) for _ in range(slots)]
    c._init_holes(slots)
    c.moved = []
    c._move_rows = lambda moves, pos, most: c.moved.append((list(moves), list(pos), most))
    return c


@pytest.mark.parametrize("bs", [16, 5])
@pytest.mark.parametrize("ascending", [True, False])
def test_kept_paths_longer_than_a_block(bs, ascending):
    """Records of a kept path have block_size rows at most, also where consecutive blocks have consecutive ids, and
    move every row of the path behind the context in order."""
    from types import SimpleNamespace
    c = _host_cache(slots=3, bs=bs, num_blocks=60)
    if ascending:  # ids are handed out from the end of the free list
        c.block_allocator.set_free_order(range(59, -1, -1))
    ctx, n = [20, 0, 7], [40, 40, 3]
    paths = [list(range(1, 31)), [0, *range(2, 40)], [2]]
    for s in range(3):
        c.block_tables[s].ensure_capacity(ctx[s] + n[s])
        c.pos_host[s] = ctx[s] + n[s]
    row = lambda s, t: c.block_tables[s].resolve(t)[0] * bs + t % bs  # noqa: E731
    rows = np.arange(60 * bs)
    want = [[row(s, t) for t in [*range(ctx[s]), *(ctx[s] + j for j in paths[s])]] for s in range(3)]
    plan = SimpleNamespace(closed=True, slots=np.arange(3), ctx_before=np.asarray(ctx), q_lens=np.asarray(n), n_seqs=3)
    c.keep_tokens(plan, paths)
    ((moves, pos, most),) = c.moved
    assert most == bs
    for a, b, count, _ in np.asarray(moves).reshape(-1, 4).tolist():
        assert 0 < count <= most
        for i in range(count):
            rows[b + i] = rows[a + i]
    for s in range(3):
        kept = ctx[s] + len(paths[s])
        assert [rows[row(s, t)] for t in range(kept)] == want[s]
        assert pos[2 * s:2 * s + 2] == [s, kept] and c.length(s) == kept


def test_a_refused_move_leaves_the_positions():
    from types import SimpleNamespace
    c = _host_cache()
    c.block_tables[0].ensure_capacity(30)
    c.pos_host[0] = 30

    def refuse(*a):
        raise _lib.NifreError("nf_kv_move")

    c._move_rows = refuse
    plan = SimpleNamespace(closed=True, slots=np.asarray([0]), ctx_before=np.asarray([20]), q_lens=np.asarray([10]), n_seqs=1)
    with pytest.raises(_lib.NifreError):
        c.keep_tokens(plan, [[1, 3]])
    assert c.length(0) == 30


def test_a_refill_on_another_stream_is_ordered_and_kept(monkeypatch):
    """The refill's copy waits for the last upload, and the buffers are recorded for the stream it runs on."""
    from types import SimpleNamespace
    from nifre_b200.masked import MaskedPlan
    log = []
    now = SimpleNamespace(name="B", wait_event=lambda e: log.append("B waits for the upload"))
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: now)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(torch.Tensor, "pin_memory", lambda t: t)
    c = _host_cache()
    c._sm_count, c._stream = 148, lambda: now.name
    c.pos_host[:] = [20, 0, 0, 0]
    plan = SimpleNamespace(slots=np.asarray([0]), q_lens=np.asarray([2]), q_starts=np.asarray([0]), generation=c._generation,
                           ctx_before=np.asarray([18]), n_seqs=1, q_heads=4, rows_needed=2, closed=True)
    view = MaskedPlan("window", 8, 0, 4, 2)
    view.owner, view.generation, view.room, view.streams = c, c._generation, (64,) * 5 + (8, 4), {"A"}
    view.buf = SimpleNamespace(device="cuda", copy_=lambda *a, **k: log.append("copy"),
                               record_stream=lambda s: log.append("buf kept for " + s.name))
    view.ws = SimpleNamespace(numel=lambda: 8, record_stream=lambda s: log.append("ws kept for " + s.name))
    view.ready = SimpleNamespace(record=lambda s: log.append("upload on " + s.name))
    assert c.plan_window(plan, 8, q_heads=4, into=view) is view
    assert log == ["B waits for the upload", "buf kept for B", "ws kept for B", "copy", "upload on B"]
    assert view.streams == {"B"}
    del log[:]
    c.plan_window(plan, 8, q_heads=4, into=view)  # again on the same stream
    assert log == ["copy", "upload on B"]


def test_plans_of_another_batch_or_of_changed_slots_are_refused():
    from types import SimpleNamespace
    a, b = _host_cache(), _host_cache()
    assert a._generation != b._generation
    a.pos_host[:2] = [12, 9]
    plan = SimpleNamespace(slots=np.asarray([0, 1]), q_lens=np.asarray([2, 3]), q_starts=np.asarray([0, 2]), closed=True,
                           ctx_before=np.asarray([10, 6]), n_seqs=2, q_heads=4, rows_needed=5, generation=b._generation)
    for call in (lambda: a.plan_window(plan, 8), lambda: a.plan_tree(plan, [None, None])):
        plan.generation = b._generation
        with pytest.raises(ValueError, match="another cache's"):
            call()
        plan.generation = a._generation
        for closed, pos in ((True, [11, 9]), (True, [12, 0]), (False, [12, 9])):
            plan.closed, a.pos_host[:2] = closed, pos
            with pytest.raises(ValueError, match="changed"):
                call()


def test_a_fork_that_the_pool_cannot_hold_leaves_every_destination_empty():
    """Also those that an earlier fork had given the right blocks."""
    from nifre_b200 import BlockPoolExhaustedError
    c = _host_cache(num_blocks=5)
    c.block_tables[0].ensure_capacity(40)
    c.pos_host[0] = 40
    c.fork([0], [1])
    assert c.length(1) == 40 and c.block_allocator.free_count == 1
    c.block_tables[3].ensure_capacity(16)
    c.pos_host[3] = 16
    with pytest.raises(BlockPoolExhaustedError, match="need 1 blocks, only 0 free"):
        c.fork([0, 0], [1, 2])
    assert [c.length(s) for s in range(4)] == [40, 0, 0, 16]
    assert len(c.block_tables[1]) == len(c.block_tables[2]) == 0
    assert c.moved[-1][:2] == ([], [1, 0, 2, 0])
    assert c.block_allocator.free_count == 1  # slot 1's own last block
