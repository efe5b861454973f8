"""Lowering of rotary positions to one launch.

A KTIR program turns pairs of a tile by two stores, x cos - y sin and y cos + x sin, where x and y are tiles of the same
tensor and cos, sin come from tables through an index tensor (the position of a token) and are spread over the heads
(notebooks/demo_gen_mlir.py:471-569 of the reference has such a kernel).  Backwards x and y change places.  Neighbouring
pairs of stores that read the same rows of the tables (queries and keys) and the copies of what lies behind the pairs join
the launch.
"""
from __future__ import annotations

import ctypes as C
from typing import List, Optional, Tuple

import numpy as np

from . import runtime as R
from .dtypes import bytes_per_elem
from .lower import ArenaMap, Footprint, Statement, _access_offsets, _points, _runs_meet, _runs_overlap, strip_views
from .lower_scatter import row_form
from .trace import Access, IndirectAccess, Node, Store, Unsupported

MOST_TOKENS = 2 ** 31 - 1                # of an item, whose tokens 32 bits count


def _term(n: Node) -> Optional[Tuple[Access, IndirectAccess]]:
    """x * (a table row spread over the heads) -> (tile of x, table access)."""
    n = strip_views(n)
    if n.kind != "ew" or n.attrs.get("op") != "arith.mulf" or n.dtype != "f32" or len(n.args) != 2:
        return None
    for x, t in (n.args, n.args[::-1]):
        x, t = strip_views(x), strip_views(t)
        if x.kind == "cast" and x.dtype == "f32":
            x = strip_views(x.args[0])
        if x.kind != "load" or x.dtype not in ("f16", "f32") or t.kind != "bcast" or list(t.attrs.get("dims", [])) != [1] or len(t.shape) != 3:
            continue
        t = strip_views(t.args[0])
        if t.kind == "iload" and t.dtype == "f32":
            return x.attrs["access"], t.attrs["access"]
    return None


def _turned(st: Store):
    """(op, [(tile, table), (tile, table)]) of a store of the sum or difference of two such products, rounded once."""
    if not isinstance(st.target, Access):
        return None
    root = strip_views(st.value)
    if root.dtype == "f16" and root.kind == "cast" and root.args[0].dtype == "f32":
        root = strip_views(root.args[0])
    if root.kind != "ew" or root.attrs.get("op") not in ("arith.subf", "arith.addf") or root.dtype != "f32":
        return None
    terms = [_term(a) for a in root.args]
    return None if None in terms else (root.attrs["op"], terms)


def _tile3(acc: Access) -> Tuple[Tuple[int, int, int], Tuple[int, int, int]]:
    """(tokens, heads, pairs) and their element strides."""
    shape, strides = tuple(acc.shape), tuple(acc.strides)
    if len(shape) == 4 and shape[3] == 1:
        shape, strides = shape[:3], strides[:3]
    if acc.coords is not None or len(shape) != 3 or np.asarray(acc.view.base).size != 1:
        raise Unsupported("rotary tile must be [tokens, heads, pairs]")
    return shape, strides


class _At:
    """A direct tile at the points of a store."""

    def __init__(self, acc: Access, st: Store, sel: np.ndarray):
        self.shape, self.strides = _tile3(acc)
        self.off, self.dtype = _access_offsets(acc, st, sel), acc.view.dtype

    def same(self, o: "_At") -> bool:
        return (self.shape, self.strides, self.dtype) == (o.shape, o.strides, o.dtype) and np.array_equal(self.off, o.off)

    def behind(self, o: "_At") -> int:
        """Elements from ``o`` to here, the same at every point; only the extent of the last dimension may differ."""
        d = self.off - o.off
        if self.shape[:2] != o.shape[:2] or self.strides[:2] != o.strides[:2] or self.dtype != o.dtype or not len(d) or (d != d[0]).any():
            raise Unsupported("rotary tiles that do not lie at a fixed distance")
        return int(d[0])


class _Pairs:
    """One tensor's pair of stores: the lower and the upper element of every pair, in and out."""

    def __init__(self, first: Store, second: Store, arena: ArenaMap):
        a, b = _turned(first), _turned(second)
        if a is None or b is None or {a[0], b[0]} != {"arith.subf", "arith.addf"} or first.axes != second.axes:
            raise Unsupported("not a turned pair")
        (sel, self.cores), (sel2, _) = _points(first), _points(second)
        if not len(sel) or not np.array_equal(sel, sel2):
            raise Unsupported("a pair stored at different points")
        self.sel, self.axes = sel, first.axes
        (dif, s_dif), (_, s_add) = ((a[1], first), (b[1], second)) if a[0] == "arith.subf" else ((b[1], second), (a[1], first))
        total = b[1] if a[0] == "arith.subf" else a[1]
        x, y = (_At(t[0], first, sel) for t in dif)
        cos, sin = (self._table(t[1]) for t in dif)
        for u, v in (total, total[::-1]):                     # y cos + x sin
            if _At(u[0], first, sel).same(y) and _At(v[0], first, sel).same(x) and \
                    self._key(self._table(u[1])) == self._key(cos) and self._key(self._table(v[1])) == self._key(sin):
                break
        else:
            raise Unsupported("the sum does not turn the pair of the difference")
        ox, oy = _At(s_dif.target, first, sel), _At(s_add.target, first, sel)
        if len({t.shape for t in (x, y, ox, oy)}) != 1 or len({t.dtype for t in (x, y, ox, oy)}) != 1 or x.dtype not in ("f16", "f32"):
            raise Unsupported("rotary tiles of different shapes or types")
        d_in, d_out = y.behind(x), oy.behind(ox)
        if d_in == 0 or d_out == 0 or (d_in > 0) != (d_out > 0) or x.strides[2] != y.strides[2] or ox.strides[2] != oy.strides[2]:
            raise Unsupported("rotary halves that change places")
        self.inverse = d_in < 0
        self.i, self.o = (y, oy) if self.inverse else (x, ox)
        self.partner = abs(d_in), abs(d_out)
        self.tokens, self.heads, self.pairs = x.shape
        self.pair_stride = x.strides[2] if self.pairs > 1 else 1
        if self.pairs > 1 and ox.strides[2] != self.pair_stride:
            raise Unsupported("rotary pairs laid out differently in and out")
        if self.pair_stride != 1 and (self.pair_stride, self.partner) != (2, (1, 1)):
            raise Unsupported("rotary pairs that are neither halves nor neighbours")
        self.cos, self.sin = cos, sin
        if (cos.rows, cos.cols, sin.rows, sin.cols) != (self.tokens, self.pairs) * 2:
            raise Unsupported("rotary tables must give one row of angles per token")
        if self._lookup(cos) != self._lookup(sin):
            raise Unsupported("cos and sin rows of different positions")
        self.rest, self.rest_at = 0, (0, 0)

    def _table(self, acc: IndirectAccess):
        f = row_form(acc, self.axes, self.sel)
        if f.idx2_off is not None or (f.rows > 1 and f.pos_stride) or (f.base != f.base[0]).any() or f.idx_dtype not in ("i32", "i64"):
            raise Unsupported("rotary table addressed in another way than by position")
        return f

    @staticmethod
    def _lookup(f):
        return f.idx_off.tobytes(), f.idx_stride if f.rows > 1 else 0, f.idx_mult, f.idx_dtype

    def _key(self, f):
        return self._lookup(f) + (int(f.base[0]), f.rows, f.cols)

    def joins(self, o: "_Pairs") -> bool:
        return (self.axes, self.tokens, self.pairs, self.pair_stride, self.inverse, self.i.dtype) == \
            (o.axes, o.tokens, o.pairs, o.pair_stride, o.inverse, o.i.dtype) and np.array_equal(self.sel, o.sel) and \
            self._key(self.cos) == self._key(o.cos) and self._key(self.sin) == self._key(o.sin)

    def take_rest(self, st: Store) -> bool:
        """``st`` copies what lies behind the pairs."""
        src = strip_views(st.value)
        if self.rest or src.kind != "load" or not isinstance(st.target, Access) or st.axes != self.axes:
            return False
        try:
            if not np.array_equal(_points(st)[0], self.sel):
                return False
            i, o = _At(src.attrs["access"], st, self.sel), _At(st.target, st, self.sel)
            if i.shape != o.shape or i.strides[2] != 1 or o.strides[2] != 1:
                return False
            at = i.behind(self.i), o.behind(self.o)
        except Unsupported:
            return False
        ends = [p + self.pairs for p in self.partner] if self.pair_stride == 1 else [2 * self.pairs] * 2
        if at[0] < ends[0] or at[1] < ends[1]:
            return False
        self.rest, self.rest_at = i.shape[2], at
        return True

    def runs(self, which: int) -> Tuple[np.ndarray, np.ndarray, int]:
        """(starts, ends, runs per point) in bytes of what is read (0) or written (1)."""
        t = (self.i, self.o)[which]
        if self.pair_stride == 1:
            pieces = [(0, self.pairs), (self.partner[which], self.partner[which] + self.pairs)]
        else:
            pieces = [(0, 2 * self.pairs)]
        if self.rest:
            pieces.append((self.rest_at[which], self.rest_at[which] + self.rest))
        whole = [list(pieces[0])]
        for lo, hi in pieces[1:]:
            if lo < whole[-1][1]:
                raise Unsupported("rotary halves that overlap")
            if lo == whole[-1][1]:
                whole[-1][1] = hi
            else:
                whole.append([lo, hi])
        starts, n = t.off[:, None] + np.array([w[0] for w in whole])[None, :], np.array([w[1] - w[0] for w in whole])
        for count, stride in ((self.heads, t.strides[1]), (self.tokens, t.strides[0])):
            if count == 1:
                continue
            if len(n) == 1 and stride == n[0]:
                n = n * count                                  # one behind the other: a longer run
            else:
                starts = (starts[:, None, :] + (np.arange(count, dtype=np.int64) * stride)[None, :, None]).reshape(len(t.off), -1)
                n = np.tile(n, count)
        bpe = bytes_per_elem(t.dtype)
        starts = starts * bpe
        return starts.reshape(-1), (starts + (n * bpe)[None, :]).reshape(-1), starts.shape[1]


class RotaryStatement(Statement):
    kind = "rotary"

    def __init__(self, dev: R.Device, pairs: List[_Pairs], arena: ArenaMap, stmt_id: int):
        p0 = pairs[0]
        table = [p0.cos.idx_off]
        for p in pairs:
            table += [p.i.off, p.o.off]
        table = np.ascontiguousarray(np.stack(table, axis=1))
        self.args = a = R.RotaryArgs()
        steps = [p0.cos.idx_stride] + [s for p in pairs for s in (p.i.strides[0], p.o.strides[0])]
        tokens = p0.tokens
        if tokens == 1 and len(table) > 1:         # (a tile of one token does not say how far the next one is)
            steps = [int(s) for s in table[1] - table[0]]
        if 1 < len(table) <= MOST_TOKENS // tokens and (np.diff(table, axis=0) == np.array(steps)[None, :] * tokens).all():
            tokens, table = tokens * len(table), table[:1]     # the tiles follow one another: one run of tokens
        a.n_items, a.tokens, a.pairs = len(table), tokens, p0.pairs
        a.dtype, a.idx_dtype = R.DTYPE_CODE[p0.i.dtype], R.DTYPE_CODE[p0.cos.idx_dtype]
        a.n_tensors, a.inverse, a.pos_stride, a.pair_stride = len(pairs), int(p0.inverse), steps[0], p0.pair_stride
        a.table_stride, a.cos_off, a.sin_off = p0.cos.idx_mult, int(p0.cos.base[0]), int(p0.sin.base[0])
        self.fps: List[Footprint] = []
        neg = np.array([-1])

        def whole(al):
            self.fps.append(Footprint(np.array([al.byte_lo]), np.array([al.byte_hi]), neg, neg, False, stmt_id))
            return al
        a.cos_end = whole(arena.check_range(a.cos_off, a.cos_off + p0.pairs, "f32", "Read from")).byte_hi // 4
        a.sin_end = whole(arena.check_range(a.sin_off, a.sin_off + p0.pairs, "f32", "Read from")).byte_hi // 4
        idx = p0.cos.idx_off
        last = idx + (p0.tokens - 1) * p0.cos.idx_stride
        if p0.cos.idx_stride < 0 or a.table_stride < 0:
            raise Unsupported("rotary positions or tables walked backwards")
        whole(arena.check_range(int(idx.min()), int(last.max()) + 1, p0.cos.idx_dtype, "Read from"))
        align = 8
        self._bytes = 0
        for k, p in enumerate(pairs):
            t = a.t[k]
            t.heads, t.rest = p.heads, p.rest
            (t.in_token, t.in_head), (t.out_token, t.out_head) = p.i.strides[:2], p.o.strides[:2]
            if len(table) == 1 and tokens > p0.tokens:
                t.in_token, t.out_token = steps[1 + 2 * k], steps[2 + 2 * k]
            (t.in_partner, t.out_partner), (t.in_rest, t.out_rest) = p.partner, p.rest_at
            for w in (0, 1):
                starts, ends, per = p.runs(w)
                bpe = bytes_per_elem(p.i.dtype)
                arena.check_range(int(starts.min()) // bpe, int(ends.max()) // bpe, p.i.dtype, "Scatter to" if w else "Read from")
                self.fps.append(Footprint(starts, ends, np.repeat(p.sel, per), np.repeat(p.cores, per), bool(w), stmt_id))
                self._bytes += int((ends - starts).sum())
        while (table[:, 1:] % align).any():
            align //= 2
        a.align = align
        # Everything is read before anything is stored: nothing that is written may be read by another part of the launch.
        writes = [f for f in self.fps if f.write]
        for k, w in enumerate(writes):
            if _runs_meet(w.starts, w.ends):
                raise Unsupported("a rotary launch that stores an element twice")
            for f in self.fps:
                if f is not w and _runs_overlap(w.starts, w.ends, f.starts, f.ends):
                    raise Unsupported("a rotary launch that reads what it writes")
        self.table = table
        for n, v in enumerate(table[0]):
            a.first[n] = int(v)
        a.dev_item_offsets = self.dev_table = dev.upload(table)
        self.device_arrays = [self.dev_table]

    def launch(self, dev, arena_ptr):
        self.args.arena = arena_ptr
        dev.check(dev.lib.ktb_launch_rotary(dev.h, C.byref(self.args)))

    def footprints(self):
        return self.fps

    def bytes_moved(self):
        return self._bytes


def try_lower_rotary(dev, stores: List[Store], arena: ArenaMap, stmt_id: int):
    """(statement, how many of the first ``stores`` it runs), or None."""
    if len(stores) < 2 or _turned(stores[0]) is None or _turned(stores[1]) is None:
        return None
    try:
        pairs, used = [_Pairs(stores[0], stores[1], arena)], 2
        while True:
            if used < len(stores) and pairs[-1].take_rest(stores[used]):
                used += 1
            if len(pairs) == R.ROTARY_TENSORS or used + 2 > len(stores):
                break
            try:
                nxt = _Pairs(stores[used], stores[used + 1], arena)
            except Unsupported:
                break
            if not nxt.joins(pairs[0]):
                break
            pairs.append(nxt)
            used += 2
        return RotaryStatement(dev, pairs, arena, stmt_id), used
    except Unsupported:
        return None
