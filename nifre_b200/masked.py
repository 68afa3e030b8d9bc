"""Work lists of attention over part of a sequence's keys (windows with sinks, drafted token trees).

No counterpart in the reference, whose attention is causal over the whole
sequence (``src/inference/attention.py:144-152``).  The lists are built on the
host once per step (numpy) and uploaded in one copy; every layer of the step
uses them.  ``include/nifre_b200.h`` defines the records (``NfMaskedArgs``).
"""

from __future__ import annotations

import ctypes

import numpy as np
import torch

from nifre_b200 import _lib

MAX_PARTS = 32767  # parts of one group (a unit record's 15 bits)
HEAD = 8  # counts (4) and the kernels' work queues (4, zero) at the start of the buffer


def tree_visibility(parents) -> np.ndarray:
    """(n, n) truth values of one drafted tree: token i sees its ancestors and itself.

    ``parents[i] < i`` is the token that token i continues, -1 the context.
    """
    parents = np.asarray(parents, dtype=np.int64).reshape(-1)
    n = len(parents)
    if (parents < -1).any() or (parents >= np.arange(n)).any():
        raise ValueError("parents[i] must be -1 (the context) or the index of an earlier drafted token")
    seen = np.eye(n, dtype=bool)
    for i in np.flatnonzero(parents >= 0).tolist():
        seen[i] |= seen[parents[i]]
    return seen


def mask_words(seen: np.ndarray) -> np.ndarray:
    """Truth values (n, n) as bit rows: (n, ceil(n / 32)) int32, bit j % 32 of word j // 32 for key j."""
    n = seen.shape[1]
    words = (n + 31) // 32
    padded = np.zeros((seen.shape[0], words * 32), dtype=np.uint8)
    padded[:, :n] = seen
    return np.packbits(padded, axis=1, bitorder="little").view(np.int32)


def virtual_keys(pos0, ntok, window: int, sinks: int):
    """Keys of a group whose tokens stand at pos0 .. pos0 + ntok - 1, without the blocks of 16 between the sinks
    and the first token's window: (kept, gap, count); key v is key v for v < kept, else v + gap."""
    lo = np.maximum(0, pos0 - window + 1) // 16 * 16
    kept = np.minimum((sinks + 15) // 16 * 16, lo)
    gap = lo - kept
    return kept, gap, pos0 + ntok - gap


def even_shares(keys, share: int, align: int, least: int, each: int = 0):
    """Cut groups of ``keys`` keys into shares of about ``share`` keys by laying them end to end (then every worker has
    the same to do whatever the groups' lengths, and no group has more parts than that needs).

    A share is a run of units: the end of one group, whole groups, the start of
    another.  A group counts ``each`` keys more than it has (what a unit costs
    besides its keys).  Cuts sit at multiples of ``align`` of their group and
    at least ``least`` keys from its ends, else at its nearer end.  Returns per
    unit (group, first key, end), in order, and the shares' first units (and
    the number of units).
    """
    keys = np.asarray(keys, dtype=np.int64)
    end = np.cumsum(keys)
    start = end - keys
    cost = np.cumsum(keys + each)
    cuts = np.arange(share, int(cost[-1]), share)
    g = np.searchsorted(cost, cuts, side="right")
    at = cuts - (cost[g] - keys[g])  # below 0: among what the group costs besides
    at = (np.maximum(at, 0) + align // 2) // align * align
    low, high = at < least, keys[g] - at < least
    at = np.where(low & (~high | (2 * at <= keys[g])), 0, np.where(high, keys[g], at))
    where = np.unique(np.concatenate([[0], start[g] + at, [int(end[-1])]]))  # the shares' bounds
    bounds = np.unique(np.concatenate([start, where]))  # every unit's start (and the end)
    first, stop = bounds[:-1], bounds[1:]
    group = np.searchsorted(end, first, side="right")
    return group, first - start[group], stop - start[group], np.searchsorted(bounds, where)


class WorkLists:
    """Units, tensor-core items and merge records of one step (each record with its group's fields), the shares of
    units and items that workers take, the mask words, and their place in one int32 buffer."""

    def __init__(self, units, items, merge, masks, unit_shares, item_shares, part_rows: int, unit_tokens: int,
                 max_parts: int):
        self.units, self.items, self.merge, self.masks = units, items, merge, masks
        self.unit_shares, self.item_shares = unit_shares, item_shares
        self.part_rows, self.unit_tokens, self.max_parts = part_rows, unit_tokens, max_parts

    def sizes(self):
        """Entries of each list, the partial rows, the tokens of the largest unit's group and the most parts."""
        return (len(self.units), len(self.items), len(self.merge), len(self.masks), self.part_rows, self.unit_tokens,
                self.max_parts)

    @staticmethod
    def room(sizes):
        """Capacities for lists of these sizes: whole multiples of 64 entries, so that the next steps' lists of the
        same batch fit as well (the launches are sized by the capacities)."""
        return (*(-(-n // 64) * 64 for n in sizes[:5]), sizes[5], -(-sizes[6] // 4) * 4)

    @staticmethod
    def offsets(room):
        """Start of units, items, merge records, masks and the units' and items' shares (there are at most as many
        shares as units), and the length."""
        at = [HEAD]
        for n in (12 * room[0], 12 * room[1], 12 * room[2], room[3], room[0] + 1, room[1] + 1):
            at.append(at[-1] + -(-n // 4) * 4)
        return at[:6], at[6]

    def pack(self, room) -> np.ndarray:
        at, total = self.offsets(room)
        host = np.zeros(total, dtype=np.int32)
        host[:4] = (max(0, len(self.unit_shares) - 1), max(0, len(self.item_shares) - 1), len(self.merge),
                    len(self.units))
        for start, part in zip(at, (self.units, self.items, self.merge, self.masks, self.unit_shares,
                                    self.item_shares)):
            host[start:start + part.size] = part.reshape(-1)
        return host


def build_lists(slots, q_lens, q_starts, ctx, group: int, unit_rows: int, item_rows: int, workers: int, kv_heads: int,
                head_dim: int = 64, window=None, sinks: int = 0, words=None, unit_share=None, item_share=None) -> WorkLists:
    """Work lists of a step whose sequences get ``q_lens`` new tokens behind ``ctx`` cached ones.

    ``window``/``sinks``, or ``words``: each sequence's mask rows (``mask_words``).
    ``group``: query heads per KV head.  Groups of units hold up to
    ``unit_rows`` query rows; sequences with more tokens than that go to the
    tensor cores' items (``item_rows`` rows) where there are any.
    """
    slots, q_lens, q_starts, ctx = (np.asarray(a, dtype=np.int64) for a in (slots, q_lens, q_starts, ctx))
    t_unit, t_item = max(1, unit_rows // group), item_rows // group
    span = q_lens + (ctx if words is not None else np.minimum(ctx, window + sinks))
    if not item_rows and int((-(-q_lens // t_unit) * span).sum()) * kv_heads < 100 * workers:
        # few groups of few keys: smaller ones, for the kernel of few columns, fill the GPU (float32, 12 heads: a tree of
        # 16 tokens on 500 keys 17.7 us, 19.6 in tiles; on 3000 keys 30.9 and 20.9)
        t_unit = max(1, 8 // group)
    routed = (q_lens > t_unit) & (t_item > 0)
    per = np.where(routed, max(1, t_item), t_unit)
    n_groups = -(-q_lens // per)
    seq = np.repeat(np.arange(len(slots)), n_groups)
    first = np.cumsum(n_groups) - n_groups
    tok0 = (np.arange(len(seq)) - first[seq]) * per[seq]
    ntok = np.minimum(per[seq], q_lens[seq] - tok0)
    pos0 = ctx[seq] + tok0
    if words is None:
        keys = virtual_keys(pos0, ntok, window, sinks)[2]
        mask0 = np.zeros(len(seq), dtype=np.int64)
        masks = np.zeros(0, dtype=np.int32)
    else:
        keys = ctx[seq] + q_lens[seq]
        start = np.cumsum([0] + [w.size for w in words])
        mask0 = start[:-1][seq] + tok0 * np.asarray([w.shape[1] for w in words], dtype=np.int64)[seq]
        masks = np.concatenate([w.reshape(-1) for w in words])
    on_items = routed[seq]
    cuts = []  # (group, first key, end) of every unit and of every item, and the shares of them
    for on, share, align, least, each, share_for in ((~on_items, unit_share, 16, 64, 48, unit_share_for),
                                                     (on_items, item_share, 128, 128, 256, item_share_for)):
        mine = np.flatnonzero(on)
        if not len(mine):
            cuts.append((mine, mine, mine, mine))
            continue
        k = keys[mine]
        share = share or share_for(k, ntok[mine] * group, workers, kv_heads, head_dim, item_rows)
        if share:
            g, k0, k1, at = even_shares(k, share, align, least, each)
        else:  # whole groups, the longest first
            g = np.argsort(-k, kind="stable")
            k0, k1, at = 0 * k, k[g], np.arange(len(k) + 1)
        cuts.append((mine[g], k0, k1, at))
    parts = np.zeros(len(seq), dtype=np.int64)
    for g, *_ in cuts:
        parts += np.bincount(g, minlength=len(seq))
    if parts.max() > MAX_PARTS:
        raise ValueError(f"a sequence's keys are cut into {int(parts.max())} parts, at most {MAX_PARTS}")
    rows = np.where(parts > 1, parts * ntok, 0)
    part0 = np.cumsum(rows) - rows
    groups = np.stack([slots[seq], q_starts[seq] + tok0, ntok, pos0, ctx[seq], q_lens[seq], mask0, part0], axis=1)
    if groups.max() >= 1 << 31:
        raise ValueError("the step's work lists exceed 32-bit indices")

    def listed(g, k0, k1, _):
        """Unit records, a group's parts numbered in the order of their keys."""
        j = np.arange(len(g)) - np.searchsorted(g, g) if len(g) and (np.diff(g) >= 0).all() else 0 * g
        return np.concatenate([np.stack([k0, k1, j | parts[g] << 16, 0 * g], axis=1), groups[g]], axis=1).astype(np.int32)

    split_groups = np.flatnonzero(parts > 1)
    fours = -(-ntok[split_groups] * group // 4)  # a merge record covers four rows
    m = np.repeat(split_groups, fours)
    t = np.arange(len(m)) - np.repeat(np.cumsum(fours) - fours, fours)
    merge = np.concatenate([np.stack([parts[m], 4 * t, on_items[m], 0 * t], axis=1), groups[m]], axis=1).astype(np.int32)
    return WorkLists(listed(*cuts[0]), listed(*cuts[1]), merge, masks, cuts[0][3], cuts[1][3], int(rows.sum()),
                     int(ntok[~on_items].max()) if (~on_items).any() else 0, int(parts.max()))


def unit_share_for(keys, rows, workers: int, kv_heads: int, head_dim: int, item_rows: int) -> int:
    """Keys per share of units: one a worker, and 64 at least.  (Finer shares and a queue over them cost more in
    partial results than they even out: 64 windows of 4096 keys, 296 CTAs, 165 us in 127 shares, 175 in 444, 178 in
    592.)  Without ``item_rows`` the kernels of other types and shapes: of few rows, a CTA a (unit, KV head, four
    rows), eight an SM, which is quick on 256 keys and would rather not merge; of more, a CTA a (unit, KV head), two an
    SM with heads of up to 128, and no cuts (0) where there are CTAs enough or keys few (a float32 chunk of 200 tokens,
    12 heads, window 256: 31 us, 39 uncut; 8 of them 128 uncut, 141 cut); with long shares several a CTA, which
    even out (16 trees of 16 tokens on up to 4000 keys: 204 us, 244 in one turn)."""
    if not item_rows:
        if rows.max() > 8:
            ctas, total = workers * (2 if head_dim <= 128 else 1), int(keys.sum()) * kv_heads
            while total >= 1024 * ctas:
                ctas *= 2
            if len(keys) * kv_heads >= ctas or keys.max() <= 128:
                return 0
            return max(64, -(-total // (ctas * 32)) * 32)
        each = kv_heads * max(1, -(-int(rows.max()) // 4))  # CTAs a unit
        return max(256 if len(keys) * each >= 48 else 128,
                   -(-int(keys.sum()) * each // (workers * 8 * 16)) * 16)
    workers = max(1, workers * 8 // kv_heads)  # eight KV heads at a time an SM
    return max(64, -(-int(keys.sum() + 48 * len(keys)) // (workers * 16)) * 16)


def item_share_for(keys, rows, workers: int, kv_heads: int, head_dim: int, item_rows: int) -> int:
    """Keys per share of tensor-core items, 0 for whole groups.

    Whole groups need no merge, but the workers end unevenly; equal shares cost
    partial results (written and read: 4 (head_dim + 4) bytes a row and part)
    and the merge's launch.  Both are estimated in microseconds from a tile's
    time (256 rows x 128 keys 1.8 at head_dim 64, 2.0 at 128; 128 rows 1.2), 4
    an item, 4 a merge, 0.3 a part of the longest group and 3 TB/s, which fit the
    measured cases within a fifth.
    """
    tiles = -(-keys // 128)
    cost = np.where(rows <= 128, 1.2, 1.8 if head_dim == 64 else 2.0)
    each = tiles * cost + 4.0
    best, share = max(float(each.max()), -(-len(keys) * kv_heads // workers) * float(each.mean())), 0
    total, work = int(keys.sum()) + 256 * len(keys), float((tiles * cost).sum())
    even = max(256, -(-total // (max(1, workers // kv_heads) * 128)) * 128)
    for s in (even, 2 * even, 4 * even):
        shares = -(-total // s)
        cuts = max(0, shares - 1)
        parts = cuts + min(cuts, len(keys))  # partial results: two at a group's first cut, one more at each further
        cut = work / shares * -(-shares * kv_heads // workers) + 8.0 + 0.3 * float(keys.max()) / s + \
            parts * float(rows.mean()) * kv_heads * 4 * (head_dim + 4) * 2 / 3e6
        if cut < best:
            best, share = cut, s
    return share


class MaskedPlan:
    """Device work lists of one step for one window, or one set of drafted trees (``PagedKVCache.plan_window`` and
    ``plan_tree``); valid for every layer of the step, as long as the sequences' blocks stay theirs."""

    def __init__(self, kind: str, window: int, sinks: int, q_heads: int, rows_needed: int):
        self.kind, self.window, self.sinks, self.q_heads, self.rows_needed = kind, window, sinks, q_heads, rows_needed
        self.room = None
        self.buf = self.ws = None  # the uploaded lists; partial rows of the split keys
        self.args = None  # NfMaskedArgs of the step; a layer's call sets its pointers
        self.args_ptr = 0
        self.fn = None
        self.owner = None
        self.generation = 0  # of the cache's pools
        self.streams = set()  # streams that the buffers are known to
        self.ready = None
        self.upload_bytes = 0


class MaskedAttentionOps:
    """Windowed and tree attention of ``PagedKVCache`` (and the dense ``KVCache``)."""

    def plan_window(self, plan, window: int, sinks: int = 0, q_heads: int | None = None,
                    into: MaskedPlan | None = None) -> MaskedPlan:
        """Work lists of ``plan``'s step for layers whose queries see the last ``window`` keys (their own position
        included) and the first ``sinks`` keys of their sequence.

        ``plan`` is the step's ``plan(...)``; layers with different windows, or
        with none, share it: each window has a ``MaskedPlan`` of its own.
        ``q_heads``: query heads of the attention calls (default: those of
        ``plan``).  ``into``: a plan of the same window from an earlier step of
        the batch, whose device buffers are filled again, so that a CUDA graph
        captured with it reads the new step (refill on the stream that
        replays it, or once its calls are done); ValueError where the new lists do not fit them (then
        capture again with a new plan).
        """
        if int(window) != window or window <= 0:
            raise ValueError(f"window must be a positive whole number, got {window}")
        if int(sinks) != sinks or sinks < 0:
            raise ValueError(f"sinks must be a whole number of at least 0, got {sinks}")
        window, sinks = min(int(window), 1 << 30), min(int(sinks), 1 << 30)
        self._check_window_holes(plan.slots, plan.ctx_before, window, sinks)
        return self._plan_masked("window", plan, q_heads, into, window, sinks, None)

    def plan_tree(self, plan, parents=None, masks=None, q_heads: int | None = None,
                  into: MaskedPlan | None = None) -> MaskedPlan:
        """Work lists of ``plan``'s step where each sequence's new tokens are a drafted tree.

        The new tokens of sequence i see its whole cached context and, among
        themselves, what ``parents[i]`` or ``masks[i]`` says: ``parents[i][j]``
        is the earlier drafted token that token j continues (-1: the context),
        and token j sees its ancestors and itself; ``masks[i]`` is an (n, n)
        array of truth values, row j for what token j sees (a row with nothing
        to see, before an empty context, gives zeros).  Exactly one of the two;
        ``None`` for a sequence: its tokens are a chain.  ``q_heads`` and
        ``into`` as for ``plan_window``.
        """
        if (parents is None) == (masks is None):
            raise ValueError("plan_tree takes parents or masks")
        given = parents if masks is None else masks
        if len(given) != plan.n_seqs:
            raise ValueError(f"{len(given)} trees for {plan.n_seqs} sequences")
        if self._holes_of(plan.slots):
            raise ValueError("a sequence whose blocks were freed behind its window cannot be attended as a whole")
        words = []
        for n, t in zip(plan.q_lens.tolist(), given):
            if t is None:
                seen = np.tril(np.ones((n, n), dtype=bool))
            elif masks is None:
                seen = tree_visibility(t)
            else:
                seen = np.asarray(t.cpu() if torch.is_tensor(t) else t).astype(bool)
            if seen.shape != (n, n):
                raise ValueError(f"a tree of {seen.shape} for {n} new tokens")
            words.append(mask_words(seen))
        return self._plan_masked("tree", plan, q_heads, into, 0, 0, words)

    def masked_limits(self, q_heads: int) -> tuple[int, int]:
        """Query rows of the largest unit's and the largest tensor-core item's group (``nf_masked_limits``)."""
        memo = self.__dict__.setdefault("_masked_limit_memo", {})
        if q_heads not in memo:
            a, b = ctypes.c_int32(0), ctypes.c_int32(0)
            _lib.check(_lib.load().nf_masked_limits(_lib.dtype_code(self.dtype), q_heads, self.n_heads, self.head_dim,
                                                    self.block_size, ctypes.byref(a), ctypes.byref(b)),
                       "nf_masked_limits")
            memo[q_heads] = (a.value, b.value)
        return memo[q_heads]

    def _plan_masked(self, kind, plan, q_heads, into, window, sinks, words) -> MaskedPlan:
        q_heads = plan.q_heads if q_heads is None else int(q_heads)
        if q_heads is None or q_heads <= 0 or q_heads % self.n_heads:
            raise ValueError(f"q_heads must be a positive multiple of the cache's {self.n_heads} heads, got {q_heads}")
        if int(plan.slots.max()) >= self.batch_size:
            raise IndexError(f"cache slot out of range [0, {self.batch_size})")
        if plan.generation != self._generation:
            raise ValueError("the step's plan is another cache's, or was made before the cache's last init_batch")
        if (self.pos_host[plan.slots] != plan.ctx_before + (plan.q_lens if plan.closed else 0)).any():
            raise ValueError("a slot's length has changed since the step was planned")
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("plans are made outside a CUDA graph capture (and refilled with into=)")
        unit_rows, item_rows = self.masked_limits(q_heads)
        lists = build_lists(plan.slots, plan.q_lens, plan.q_starts, plan.ctx_before, q_heads // self.n_heads, unit_rows,
                            item_rows, self.sm_count, self.n_heads, self.head_dim, window,
                            sinks, words)
        sizes = lists.sizes()
        if into is None:
            view = MaskedPlan(kind, window, sinks, q_heads, plan.rows_needed)
            view.room = lists.room(sizes)
        else:
            view = into
            if (view.kind, view.window, view.sinks, view.q_heads) != (kind, window, sinks, q_heads) \
                    or view.owner is not self or view.generation != self._generation:
                raise ValueError("into is the plan of another cache, window or set of heads")
            if any(n > r for n, r in zip(sizes, view.room)):
                raise ValueError(f"the step's lists {sizes} do not fit the plan's room {view.room}")
            view.rows_needed = plan.rows_needed
        host = torch.from_numpy(lists.pack(view.room)).pin_memory()
        view.upload_bytes = host.numel() * 4
        if into is not None:
            if self._stream() not in view.streams:
                self._adopt_stream(view, self._stream())
            view.buf.copy_(host, non_blocking=True)
            view.ready.record(torch.cuda.current_stream(self.device))
            view.streams = {self._stream()}  # the others wait for this upload
            return view
        view.buf = host.to(self.device, non_blocking=True)
        D, room = self.head_dim, view.room
        view.ws = torch.empty(room[4] * q_heads * (-(-D // 4) * 4 + 4), dtype=torch.float32, device=self.device)
        at, _ = lists.offsets(room)
        base = view.buf.data_ptr()
        ptr = lambda i: base + 4 * at[i] if room[i] else None  # noqa: E731
        view.args = _lib.NfMaskedArgs(
            block_tables=self._bt_ptr, units=ptr(0), items=ptr(1), merge=ptr(2), counts=base, masks=ptr(3),
            unit_shares=base + 4 * at[4], item_shares=base + 4 * at[5],
            mask_words=room[3], ws=view.ws.data_ptr() if room[4] else None, ws_rows=room[4], queue=base + 16,
            status=self._status_ptr, dtype=self._dt_code, num_q_heads=q_heads, num_kv_heads=self.n_heads, head_dim=D,
            block_size=self.block_size, num_blocks=self.num_blocks, num_slots=self.batch_size,
            max_blocks_per_seq=self.max_blocks_per_seq, max_units=room[0], unit_tokens=room[5], max_items=room[1],
            max_merge=room[2], max_parts=room[6], window=window, sinks=sinks)
        view.args_ptr = ctypes.addressof(view.args)
        lib = _lib.load()
        view.fn = lib.nf_tree_attention if kind == "tree" else lib.nf_window_attention
        view.owner, view.generation = self, self._generation
        view.ready = torch.cuda.Event()
        view.ready.record(torch.cuda.current_stream(self.device))
        view.streams = {self._stream()}
        return view

    def window_attention_step(self, layer_id: int, q: torch.Tensor, view: MaskedPlan, out: torch.Tensor,
                              scale: float | None = None) -> torch.Tensor:
        """out[row] = attention of q[row] over the keys of its sequence in ``view``'s window and sinks, for the step's
        rows; the other rows of ``out`` are left untouched.

        ``q``/``out``: (rows, Hq*D) in the pool dtype with unit column stride
        (``out`` must not overlap ``q``).  ``scale`` defaults to 1 / sqrt(D).
        Keys that a query does not see contribute nothing, whatever their rows
        hold.  Calls with the same plan must not overlap on the GPU (its work
        queue and partial rows are shared); a CUDA graph that captured one needs
        the plan kept alive.
        """
        if view.kind != "window":
            raise ValueError("the plan is a tree's: use tree_attention_step")
        return self._masked_step(layer_id, q, view, out, scale)

    def tree_attention_step(self, layer_id: int, q: torch.Tensor, view: MaskedPlan, out: torch.Tensor,
                            scale: float | None = None) -> torch.Tensor:
        """out[row] = attention of the drafted token q[row] over its sequence's context and the drafted tokens that it
        sees (``plan_tree``).  Arguments as for ``window_attention_step``."""
        if view.kind != "tree":
            raise ValueError("the plan is a window's: use window_attention_step")
        return self._masked_step(layer_id, q, view, out, scale)

    def _masked_step(self, layer_id, q, view, out, scale):
        if not q.is_cuda or q.device != out.device:
            _lib.require_cuda(q, "q")
            raise ValueError("q and out must be on the same device")
        if view.owner is not self:
            raise ValueError("the plan belongs to another cache")
        if view.generation != self._generation:
            raise ValueError("the plan was made before the cache's last init_batch")
        width = view.q_heads * self.head_dim
        shape = q.shape
        if len(shape) != 2 or shape[1] != width or q.stride(1) != 1:
            raise ValueError(f"q must be (rows, {width}) with unit column stride")
        if out.shape != shape or out.stride(1) != 1 or (shape[0] > 1 and out.stride(0) < width):
            raise ValueError("out must have q's shape, unit column stride and rows of their own")
        if q.dtype != self.dtype or out.dtype != self.dtype:
            raise ValueError(f"q/out dtype must be the cache dtype {self.dtype}")
        if shape[0] < view.rows_needed:
            raise ValueError(f"q has {shape[0]} rows, the step uses rows up to {view.rows_needed}")
        if not 0 <= layer_id < self.num_layers:
            raise IndexError(f"layer_id {layer_id} out of range [0, {self.num_layers})")
        if q.device.index != self._dev_index:
            raise ValueError(f"q is on {q.device}, the cache on {self.device}")
        if torch.cuda.current_device() != self._dev_index:
            with torch.cuda.device(self._dev_index):
                return self._masked_step(layer_id, q, view, out, scale)
        stream = self._stream()
        if stream not in view.streams:
            self._adopt_stream(view, stream)
        a = view.args
        a.out, a.q, a.k_pool, a.v_pool = out.data_ptr(), q.data_ptr(), self._k_ptr[layer_id], self._v_ptr[layer_id]
        a.out_row_stride, a.q_row_stride, a.num_rows = out.stride(0), q.stride(0), shape[0]
        a.scale = self.head_dim ** -0.5 if scale is None else scale
        rc = view.fn(view.args_ptr, stream)
        if rc:
            _lib.check(rc, "nf_%s_attention" % view.kind)
        return out

    @staticmethod
    def _adopt_stream(view, stream) -> None:
        """First call or refill of a plan on another stream than its last upload's: that upload comes first, and the
        buffers stay until this stream is done with them.  (A capturing stream orders and keeps nothing: its graph's
        user does.)"""
        if torch.cuda.is_current_stream_capturing():
            return
        cur = torch.cuda.current_stream(view.buf.device)
        cur.wait_event(view.ready)
        view.buf.record_stream(cur)
        if view.ws.numel():
            view.ws.record_stream(cur)
        view.streams.add(stream)
