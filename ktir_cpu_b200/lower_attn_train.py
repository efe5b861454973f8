"""Lowering of attention over whole sequences: the forward pass that keeps the log-sum-exp of its rows, and the gradients.

The matchers accept what ``kernels.attention_forward`` and ``kernels.attention_backward`` say and what computes the same: per
pair of a tile of query rows (position-major, the query heads of one key head) and a tile of keys, scores
scale * (Q @ K^T) and a mask that compares a key position with a query position or a length;

* forward: the online-softmax loop that ``lower_attn`` describes with finite initial maximum and zero initial sum, O = acc /
  max(L, tiny), and M + log(L) stored behind it;
* backward: P = exp(S - lse), 0 where masked, dS = P * (dO @ V^T - rowsum(dO * O)); dQ = scale * sum over key tiles of
  dS @ K; dK = scale * sum over query tiles of dS^T @ Q and dV = sum of P^T @ dO.

Tiles of all cores are regrouped per head, so the kernels use their own tiles whatever sizes the text used.  Tiles may run
past the end of their tensor, where a read gives zero and a store is dropped (ktir_cpu/memory.py:217-306), as long as the
mask hides such keys.
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass
from typing import List, Optional, Tuple

import numpy as np

from . import runtime as R
from .dtypes import bytes_per_elem
from .lower import ArenaMap, Footprint, Statement, _points, _row_broadcast, _row_reduce, _runs_meet, _runs_overlap, _skip, strip_views
from .lower_attn import _const_value, _ew, _int_affine
from .lower_mm import _is_zero_const, _unext
from .trace import Access, LoopInfo, Node, Store, Unsupported, iv_full


SMS, TILE, STEP = 148, 128, 64           # SMs; rows that a CTA owns, rows that it streams at a time
# What scores may be at most, by the scale: the forward kernel starts from a maximum of -10^30, the backward one multiplies by 1 / ln 2.
FORWARD_SCORES, BACKWARD_SCORES = 1.0e30, 1.0e38


def _scores_below(scale: float, head_dim: int, bound: float) -> bool:
    """Whether all scores that f16 operands can have are below ``bound`` in magnitude."""
    return abs(float(np.float32(scale))) * head_dim * 65504.0 ** 2 <= bound       # (false for a NaN)


# ---- pieces of the expressions ------------------------------------------------------------------------------------
def _load(n: Node, dtype: str = "f16") -> Optional[Access]:
    """The direct f16 tile behind views and an extension to f32 (or a tile of another type as it is)."""
    n = _unext(n) if dtype == "f16" else strip_views(n)
    return n.attrs["access"] if n.kind == "load" and n.dtype == dtype else None


def _load_t(n: Node) -> Optional[Access]:
    """The tile behind a transposition."""
    n = _unext(n)
    return _load(n.args[0]) if n.kind == "transpose" and tuple(n.attrs["perm"]) == (1, 0) else None


def _by_const(n: Node) -> Tuple[Optional[float], Node]:
    """n = c * x -> (c, x); (None, n) where it is no such product."""
    m = _ew(n, "arith.mulf")
    if m is not None:
        for c, x in (m.args, m.args[::-1]):
            v = _const_value(c)
            if v is not None:
                return v, strip_views(x)
    return None, strip_views(n)


def _product(n: Node, right_t) -> Optional[Tuple[Access, Access]]:
    """A plain product of two tiles, the right one transposed: (left, right)."""
    n = strip_views(n)
    if n.kind != "matmul" or n.attrs.get("batched") or n.dtype != "f32" or not _is_zero_const(n.args[2] if len(n.args) > 2 else None):
        return None
    a, b = _load(n.args[0]), right_t(n.args[1])
    return None if a is None or b is None else (a, b)


def _scores(n: Node):
    """scale * (Q @ K^T) -> dict(q, k, scale)."""
    scale, qk = _by_const(n)
    ab = _product(qk, _load_t)
    return None if ab is None else dict(q=ab[0], k=ab[1], scale=1.0 if scale is None else scale)


def _probability(n: Node):
    """exp(scores - lse), 0 where a mask hides the key -> dict(q, k, scale, lse, cond)."""
    p = strip_views(n)
    cond = None
    sel = _ew(p, "arith.select")
    if sel is not None:
        if _const_value(sel.args[2]) != 0.0:
            return None
        cond, p = strip_views(sel.args[0]), strip_views(sel.args[1])
    e = _ew(p, "math.exp")
    sub = _ew(e.args[0], "arith.subf") if e is not None else None
    if sub is None or p.dtype != "f32":
        return None
    m = _scores(sub.args[0])
    lse = _row_broadcast(sub.args[1], p.shape)
    lse = _load(lse, "f32") if lse is not None else None
    if m is None or lse is None:
        return None
    return dict(m, lse=lse, cond=cond, tile=tuple(p.shape))


def _score_gradient(n: Node):
    """P * (dO @ V^T - rowsum(dO * O)) -> the probability's dict with do, v, o."""
    mul = _ew(n, "arith.mulf")
    if mul is None:
        return None
    for a, b in (mul.args, mul.args[::-1]):
        sub = _ew(b, "arith.subf")
        m = _probability(a) if sub is not None else None
        if m is None:
            continue
        dov = _product(sub.args[0], _load_t)
        d = _row_broadcast(sub.args[1], m["tile"])
        rr = _row_reduce(d, ("arith.addf",)) if d is not None else None
        both = _ew(rr[0], "arith.mulf") if rr is not None else None
        if dov is None or both is None or rr[2] not in (None, 0.0) or both.dtype != "f32":
            continue
        x, y = _load(both.args[0]), _load(both.args[1])
        if x is None or y is None:
            continue
        do, v = dov
        o = y if _same(x, do) else x if _same(y, do) else None
        if o is not None:
            return dict(m, do=do, v=v, o=o)
    return None


def _same(a: Access, b: Access) -> bool:
    """The same elements at every point."""
    if a is b:
        return True
    if (a.view.dtype, tuple(a.shape), tuple(a.strides)) != (b.view.dtype, tuple(b.shape), tuple(b.strides)) or a.coords is not None or b.coords is not None:
        return False
    x, y = np.asarray(a.off), np.asarray(b.off)
    n = max(x.ndim, y.ndim)
    grow = lambda v: v.reshape(v.shape + (1,) * (n - v.ndim))   # noqa: E731
    x, y = grow(x), grow(y)
    if any(p != q and 1 not in (p, q) for p, q in zip(x.shape, y.shape)):
        return False
    return bool((x == y).all())


def _iter_of(n: Node, loop: LoopInfo, k: int) -> bool:
    n = strip_views(n)
    return n.kind == "iter" and n.attrs.get("loop") is loop and n.attrs["index"] == k


def _transposed(n: Node) -> Optional[Node]:
    n = strip_views(n)
    return strip_views(n.args[0]) if n.kind == "transpose" and tuple(n.attrs["perm"]) == (1, 0) else None


def match_gradient(value: Node):
    """("dq" | "dk" | "dv", dict) of a stored gradient, or None."""
    root = strip_views(value)
    if not (root.kind == "cast" and root.dtype == "f16" and root.args[0].dtype == "f32"):
        return None
    factor, fin = _by_const(root.args[0])
    if fin.kind != "loopres":
        return None
    loop, k = fin.attrs["loop"], fin.attrs["index"]
    y = strip_views(loop.yields[k])
    if y.kind != "matmul" or y.attrs.get("batched") or len(y.args) != 3 or not _iter_of(y.args[2], loop, k) or \
            not _is_zero_const(loop.inits[k]):
        return None
    right = _load(y.args[1])
    if right is None:
        return None
    m = _score_gradient(y.args[0])
    if m is not None:
        ok = _same(right, m["k"]) and factor == m["scale"]
        return ("dq", dict(m, loop=loop)) if ok else None
    left = _transposed(y.args[0])
    if left is None:
        return None
    m = _score_gradient(left)
    if m is not None:
        return ("dk", dict(m, loop=loop)) if _same(right, m["q"]) and factor == m["scale"] else None
    m = _probability(left)
    if m is not None and factor is None:
        return "dv", dict(m, loop=loop, do=right)
    return None


def match_forward(value: Node):
    """The online-softmax loop of ``kernels.attention_forward``: dict(q, k, v, scale, cond, loop, indices), or None."""
    root = strip_views(value)
    if not (root.kind == "cast" and root.dtype == "f16" and root.args[0].dtype == "f32"):
        return None
    div = _ew(root.args[0], "arith.divf")
    if div is None:
        return None
    acc_fin = strip_views(div.args[0])
    if acc_fin.kind != "loopres" or len(acc_fin.shape) != 2:
        return None
    safe = _row_broadcast(div.args[1], acc_fin.shape)
    mx = _ew(safe, "arith.maximumf") if safe is not None else None
    if mx is None:
        return None
    loop: LoopInfo = acc_fin.attrs["loop"]
    l_fin, tiny = (strip_views(x) for x in mx.args)
    if l_fin.kind != "loopres":
        l_fin, tiny = tiny, l_fin
    floor = _const_value(tiny)
    # (a row that sees a key has a sum of 1 at least, up to rounding: the floor only catches sums of 0)
    if l_fin.kind != "loopres" or l_fin.attrs["loop"] is not loop or len(loop.yields) != 3 or floor is None or not 0.0 < floor <= 0.5:
        return None
    ia, il = acc_fin.attrs["index"], l_fin.attrs["index"]
    im = ({0, 1, 2} - {ia, il}).pop()
    m_new, l_new, acc_new = (strip_views(loop.yields[k]) for k in (im, il, ia))
    big = _ew(m_new, "arith.maximumf")
    if big is None or acc_new.kind != "matmul" or acc_new.attrs.get("batched") or len(acc_new.args) != 3:
        return None
    rmax = big.args[1] if _iter_of(big.args[0], loop, im) else big.args[0] if _iter_of(big.args[1], loop, im) else None
    rr = _row_reduce(rmax, ("arith.maximumf",)) if rmax is not None else None
    if rr is None or rr[2] not in (None, float("-inf")):
        return None
    masked = sc = strip_views(rr[0])
    cond = None
    sel = _ew(masked, "arith.select")
    if sel is not None:
        if _const_value(sel.args[2]) != float("-inf"):
            return None
        cond, sc = strip_views(sel.args[0]), strip_views(sel.args[1])
    m = _scores(sc)
    p = _ew(acc_new.args[0], "math.exp")
    sub = _ew(p.args[0], "arith.subf") if p is not None else None
    v = _load(acc_new.args[1])
    if m is None or sub is None or v is None or strip_views(sub.args[0]) is not masked or \
            _row_broadcast(sub.args[1], masked.shape) is not m_new:
        return None

    def is_alpha(n):
        e = _ew(n, "math.exp")
        d = _ew(e.args[0], "arith.subf") if e is not None else None
        return d is not None and _iter_of(d.args[0], loop, im) and strip_views(d.args[1]) is m_new

    scaled = _ew(acc_new.args[2], "arith.mulf")
    alpha = _row_broadcast(scaled.args[1], acc_new.shape) if scaled is not None else None
    if alpha is None or not _iter_of(scaled.args[0], loop, ia) or not is_alpha(alpha):
        return None
    ladd = _ew(l_new, "arith.addf")
    lmul = _ew(ladd.args[0], "arith.mulf") if ladd is not None else None
    lr = _row_reduce(ladd.args[1], ("arith.addf",)) if ladd is not None else None
    if lmul is None or lr is None or lr[2] not in (None, 0.0) or strip_views(lr[0]) is not p or \
            not _iter_of(lmul.args[0], loop, il) or not is_alpha(lmul.args[1]):
        return None
    m_init, l_init, acc_init = (_const_value(loop.inits[i]) for i in (im, il, ia))
    # (the initial maximum has to be below every score, so that its value does not matter, and finite, for rows that see nothing)
    if m_init is None or not -3.0e38 < m_init <= -1.0e20 or l_init != 0.0 or acc_init != 0.0 or not m["scale"] > 0.0:
        return None
    return dict(m, v=v, cond=cond, loop=loop, im=im, il=il, m_init=m_init, tile=tuple(masked.shape))


def _is_lse(value: Node, m: dict) -> bool:
    """M + log(L) of the loop."""
    add = _ew(_skip(value), "arith.addf")
    if add is None or add.dtype != "f32":
        return False

    def fin(n, k):
        n = strip_views(n)
        return n.kind == "loopres" and n.attrs["loop"] is m["loop"] and n.attrs["index"] == k
    for a, b in (add.args, add.args[::-1]):
        log = _ew(b, "math.log")
        if log is not None and fin(a, m["im"]) and fin(log.args[0], m["il"]):
            return True
    return False


# ---- where the tiles lie ------------------------------------------------------------------------------------------
@dataclass
class _Walk:
    """Tiles [rows, heads(, head_dim)] of one tensor [positions, heads(, head_dim)] at the points of a store and the trips of
    a loop: element offset of position 0 of head 0, strides, extents, and first position and head [points, trips]."""
    base: int
    row: int
    head: int
    rows: int
    heads: int
    dtype: str
    count: Tuple[int, int]
    row0: np.ndarray
    head0: np.ndarray

    def tensor(self):
        return self.base, self.row, self.head, self.rows, self.heads, self.dtype


def _walk(acc: Access, axes, sel: np.ndarray, trips: Optional[int], hd: Optional[int], arena: ArenaMap, what: str) -> _Walk:
    nd = 2 if hd is None else 3
    if acc.coords is not None or len(acc.shape) != nd or len(acc.view.shape) != nd or np.asarray(acc.view.base).size != 1:
        raise Unsupported("attention tile must be a box of a [positions, heads, head_dim] tensor")
    if hd is not None and (acc.shape[2] != hd or acc.view.shape[2] != hd or acc.strides[2] != 1):
        raise Unsupported("attention tile must hold whole heads")
    ext = tuple(axes) + ((trips,) if trips is not None else ())
    off = iv_full(acc.off, ext).reshape(-1, trips if trips is not None else 1)[sel]
    base = int(np.asarray(acc.view.base).reshape(-1)[0])
    sr, sh = int(acc.strides[0]), int(acc.strides[1])
    rows, heads = int(acc.view.shape[0]), int(acc.view.shape[1])
    if sr <= 0 or sh <= 0:
        raise Unsupported("attention tensor with a stride that is not positive")
    rel = off - base
    if sr >= sh:
        r, rem = np.divmod(rel, sr)
        h, rem = np.divmod(rem, sh)
    else:
        h, rem = np.divmod(rel, sh)
        r, rem = np.divmod(rem, sr)
    if not r.size or rem.any() or (r < 0).any() or (r >= rows).any() or (h < 0).any() or (h + acc.shape[1] > heads).any():
        raise Unsupported("attention tile not aligned to positions and heads")
    last = base + (rows - 1) * sr + (heads - 1) * sh + (hd or 1)
    al = arena.check_range(base, last, acc.view.dtype, what)
    if (r + acc.shape[0] > rows).any() and (sr < sh or (base + rows * sr) * bytes_per_elem(acc.view.dtype) < al.byte_hi):
        raise Unsupported("attention tile that runs from one tensor into other memory")
    return _Walk(base, sr, sh, rows, heads, acc.view.dtype, (int(acc.shape[0]), int(acc.shape[1])), r, h)


def _rectangle(w: _Walk) -> Tuple[int, int, int, int]:
    """(first row, rows, first head, heads) that the tiles of a store cover, each once."""
    r, h = w.row0[:, 0], w.head0[:, 0]
    b, g = w.count
    r0, h0 = int(r.min()), int(h.min())
    i, j = (r - r0) // b, (h - h0) // g
    ni, nj = int(i.max()) + 1, int(j.max()) + 1
    if ((r - r0) % b).any() or ((h - h0) % g).any() or len(r) != ni * nj or len(np.unique(i * nj + j)) != ni * nj:
        raise Unsupported("attention tiles do not cover [rows x heads] exactly once")
    return r0, min(ni * b, w.rows - r0), h0, nj * g


def _streams_all(w: _Walk):
    """The loop walks the whole tensor from its start, tile after tile, the same at every point."""
    if (w.row0 != np.arange(w.row0.shape[1])[None, :] * w.count[0]).any() or w.row0.shape[1] * w.count[0] < w.rows or \
            (w.head0 != w.head0[:, :1]).any():
        raise Unsupported("attention loop must walk a whole tensor")


def _mask(m: dict, q: _Walk, k: _Walk, ext, sel, trips: int):
    """(causal, delta): key j is visible to query i iff j <= i + delta, all keys if not causal."""
    grp, over = q.count[1], bool((k.row0 + k.count[0] > k.rows).any())
    cond = m["cond"]
    if cond is None:
        if over:
            raise Unsupported("attention tiles past the last key need a mask")
        return 0, 0
    if cond.kind != "ew" or cond.attrs.get("op") != "arith.cmpi" or cond.attrs.get("pred") not in ("ule", "sle", "ult", "slt"):
        raise Unsupported("attention mask must be a comparison of a key position with a query position or a length")
    strict = cond.attrs["pred"].endswith("lt")
    kr, kc, kconst, _ = _int_affine(cond.args[0])
    qr, qc, qconst, qdiv = _int_affine(cond.args[1])
    if (kr, kc) != (0, 1) or qc != 0 or qr not in (0, 1) or (qr == 1 and qdiv != grp):
        raise Unsupported("attention mask must be a comparison of a key position with a query position or a length")
    kfull, qfull = (iv_full(v, ext).reshape(-1, trips)[sel] for v in (kconst, qconst))
    if cond.attrs["pred"].startswith("u") and ((kfull < 0).any() or (qfull < 0).any()):
        raise Unsupported("attention mask compares negative positions as unsigned ones")
    kfull = kfull - k.row0
    if qr == 0:                                  # key position < length
        bound = qfull - kfull + (0 if strict else 1)
        if (bound < k.rows).any():
            raise Unsupported("attention mask hides keys of the tensor")
        if over and (bound > k.rows).any():
            raise Unsupported("attention mask shows keys past the tensor")
        return 0, 0
    d = qfull - q.row0 - kfull - (1 if strict else 0)
    if (d != d.flat[0]).any():
        raise Unsupported("attention mask offset differs between cores or tiles")
    delta = int(d.flat[0])
    if over and q.rows - 1 + delta >= k.rows:
        raise Unsupported("attention mask shows keys past the tensor")
    if abs(delta) > 1 << 30:
        raise Unsupported("attention mask offset")
    return 1, delta


def _aligned(*walks: _Walk):
    for w in walks:
        if w.base % 8 or w.row % 8 or w.head % 8:
            raise Unsupported("attention tensors must lie on boundaries of 8 elements")
        if w.rows > 1 << 30 or w.heads > 1 << 20:
            raise Unsupported("attention tensor too long")


def _written(w: _Walk, rect, hd: int) -> Tuple[np.ndarray, np.ndarray]:
    """Byte runs of rows and heads of a stored tensor."""
    r0, nr, h0, nh = rect
    bpe = bytes_per_elem(w.dtype)
    start = w.base + r0 * w.row + h0 * w.head
    if w.head == hd or nh == 1:
        length = nh * hd if w.head == hd else hd
        if w.row == length or nr == 1:
            starts, length = np.array([start]), length if nr == 1 else nr * length
        else:
            starts = start + np.arange(nr, dtype=np.int64) * w.row
    else:
        length = hd
        starts = (start + np.arange(nr, dtype=np.int64)[:, None] * w.row + np.arange(nh, dtype=np.int64)[None, :] * w.head).reshape(-1)
    return starts * bpe, (starts + length) * bpe


def _footprints(arena: ArenaMap, reads, writes, stmt_id: int) -> List[Footprint]:
    """Whole tensors read, the given runs written; both sets apart from each other and among themselves."""
    fps = []
    for w in reads:
        al = arena.find(w.base * bytes_per_elem(w.dtype))
        fps.append(Footprint(np.array([al.byte_lo]), np.array([al.byte_hi]), np.array([-1]), np.array([-1]), False, stmt_id))
    for s, e in writes:
        neg = np.full(len(s), -1)
        fps.append(Footprint(s, e, neg, neg, True, stmt_id))
    return fps


def _disjoint(arena: ArenaMap, reads, writes) -> bool:
    """No written run overlaps a tensor that is read, or another written run, of its own tensor either."""
    if any(_runs_meet(*w) for w in writes):
        return False
    spans = [(f.starts, f.ends) for f in _footprints(arena, reads, [], 0)]
    return not any(_runs_overlap(*a, *b) for i, a in enumerate(writes) for b in list(writes[i + 1:]) + spans)


def dense_plan(q_len: int, kv_len: int, heads: int, head_dim: int, causal: int, delta: int, twice: bool) -> Tuple[int, int]:
    """How the forward pass deals out its work: (whether a CTA takes single pairs of 128-row tiles, parts that the keys are cut into).

    Either an item is a late pair of tiles of a head and an early one, so that all items cost the same and neighbours read the same
    keys, or a single pair, late ones first and dealt out to and fro, which is half as coarse.  Keys cut into parts make more items
    of few.  The way that an estimate in microseconds of the busiest CTA finds best is taken: 1.73 a page of 128 keys (1.55, 64
    wide; 1.27 for one tile alone), 3 to start and end a pair, 2 more and a share of joining for a part.  It is within 6 % of what 21
    shapes took as pairs, single or not, within 15 in parts.  Measured, items of two pairs / single ones / the best parts: 842
    positions of 8 heads 31.0 / 18.6 / 16.8; 1531 queries of 32 heads over 4603 keys 117.0 / 107.4 / 113.9; 1024 over 16384 keys 442.6
    / 226.6 / 249.8; one query over 8192 keys 88.3 / 88.3 / 32.9; 2048 positions of 128 heads 148.9 / 134.9, of 256 heads, whose keys
    L2 does not hold, 254.8 / 268.1."""
    q0 = np.arange(0, q_len, 256, dtype=np.int64)
    two = q0 + 128 < q_len
    seen = np.clip(np.where(two, q0 + 256, q0 + 128) + delta, 0, kv_len) if causal else np.full(len(q0), kv_len)
    pages, page = -(-seen // 128), np.where(two, 1.73 if head_dim == 128 else 1.55, 1.27) * (2 if twice else 1)
    n, best = len(pages), (0, 1)
    if n * heads > 16 * SMS:                     # (many items: no order of them is far from the others)
        return best

    def busiest(single, parts):
        own = 3.0 + (2.0 if parts > 1 else 0.0) + -(-pages // parts) * page
        if single:
            cost = np.repeat(own[::-1], heads * parts)
        else:
            pairs = own[::-1][:(n + 1) // 2].copy()
            pairs[:n // 2] += own[:n // 2]
            cost = np.tile(np.repeat(pairs, parts), heads)
        rounds = -(-len(cost) // SMS)
        cost = np.pad(cost, (0, rounds * SMS - len(cost))).reshape(rounds, SMS)
        if single:
            cost[1::2] = cost[1::2, ::-1]
        return cost.sum(0).max() + (5.0 if parts == 1 else 8.0 + 8.0 * parts * q_len * heads * head_dim / 8e6)
    least = busiest(0, 1)
    for parts in (1, 2, 3, 4, 5, 6, 8, 12, 16):
        if parts > 1 and (n * heads * parts > 4 * SMS or parts * 192 > kv_len):
            break
        for single in (0, 1):
            t = busiest(single, parts)
            if t < 0.97 * least:
                best, least = (single, parts), t
    return best


# (An output's error stays below 1.5 of its rounding from some 20 rows on, a gradient's, three sums of which each may be off, from 200.)
FEW_ROWS_FORWARD, FEW_ROWS_BACKWARD = 24, 256


def few_rows(q_len: int, heads: int, causal: int, delta: int, most: int) -> bool:
    """Whether at most ``most`` rows see a key.

    P and dS are rounded to f16 before they are multiplied.  Every result is a sum of many products, so that over many rows these
    roundings come to as much as the result's own and together to 1.41 of it.  Over a few rows they are a matter of luck: of sixty
    draws of one query over 700 keys the error of an output was 1.42 of the rounding on average and 1.76 at most, of a gradient
    over 2 x 2 positions 1.4 and 2.1.  There the kernels multiply what the rounding left out too."""
    return (q_len + min(delta, 0) if causal else q_len) * heads <= most


class AttentionDenseStatement(Statement):
    """The forward pass; the store of the rows' log-sum-exp behind it joins."""
    kind = "attention_dense"

    def __init__(self, dev: R.Device, stores: List[Store], m: dict, arena: ArenaMap, stmt_id: int):
        store, self.used = stores[0], 1
        if not isinstance(store.target, Access):
            raise Unsupported("attention output through an indirect tile")
        sel, _ = _points(store)
        if not len(sel):
            raise Unsupported("a store that no core executes")
        T = m["loop"].trips
        ext = tuple(store.axes) + (T,)
        hd = int(m["q"].shape[-1])
        if hd not in (64, 128):
            raise Unsupported("attention over whole sequences supports head_dim 64 and 128")
        if not np.float32(m["scale"]) > 0.0 or not _scores_below(m["scale"], hd, min(-m["m_init"], FORWARD_SCORES)):
            raise Unsupported("a score scale that is not positive, or scores that may reach the initial maximum")
        q = _walk(m["q"], store.axes, sel, None, hd, arena, "Read from")
        o = _walk(store.target, store.axes, sel, None, hd, arena, "Scatter to")
        k, v = (_walk(m[x], store.axes, sel, T, hd, arena, "Read from") for x in ("k", "v"))
        grp = q.count[1]
        for a, b in ((o, q), (v, k)):
            if a.count != b.count or (a.rows, a.heads) != (b.rows, b.heads) or (a.row0 != b.row0).any() or (a.head0 != b.head0).any():
                raise Unsupported("attention tensors differ in tiles or shape")
        _streams_all(k)
        if k.count[1] != 1 or q.heads != k.heads * grp or (q.head0 % grp).any() or (k.head0[:, :1] != q.head0 // grp).any() or \
                m["tile"] != (q.count[0] * grp, k.count[0]) or {w.dtype for w in (q, k, v, o)} != {"f16"}:
            raise Unsupported("key heads do not follow the query heads")
        causal, delta = _mask(m, q, k, ext, sel, T)
        _aligned(q, k, v, o)
        rect = r0, nr, h0, nh = _rectangle(o)
        self.args = a = R.AttnDenseArgs()
        # the launch covers the rectangle that the cores at hand store, from its own first row and head on
        for n, w, r, h in (("q", q, r0, h0), ("o", o, r0, h0), ("k", k, 0, h0 // grp), ("v", v, 0, h0 // grp)):
            setattr(a, f"{n}_off", w.base + r * w.row + h * w.head)
            setattr(a, f"{n}_row", w.row)
            setattr(a, f"{n}_head", w.head)
        a.q_len, a.kv_len, a.heads, a.kv_group, a.head_dim = nr, k.rows, nh, grp, hd
        a.causal, a.causal_delta = causal, delta + r0 if causal else 0
        a.scale = float(np.float32(m["scale"]))
        a.lse_off = -1
        writes = [_written(o, rect, hd)]
        if len(stores) > 1 and isinstance(stores[1].target, Access) and stores[1].axes == store.axes and \
                np.array_equal(_points(stores[1])[0], sel) and _is_lse(stores[1].value, m):
            lse = _walk(stores[1].target, store.axes, sel, None, None, arena, "Scatter to")
            if lse.count == q.count and (lse.rows, lse.heads) == (q.rows, q.heads) and (lse.row0 == q.row0).all() and \
                    (lse.head0 == q.head0).all() and lse.dtype == "f32":
                a.lse_off, a.lse_row, a.lse_head = lse.base + r0 * lse.row + h0 * lse.head, lse.row, lse.head
                writes.append(_written(lse, rect, 1))
                self.used = 2
        if not _disjoint(arena, (q, k, v), writes):
            raise Unsupported("attention stored over a tensor that it reads")
        seen = np.full(nr, k.rows) if not causal else np.clip(np.arange(nr) + 1 + a.causal_delta, 0, k.rows)
        self.flops = int(4 * nh * hd * seen.sum())
        self._bytes = 2 * hd * (2 * nr * nh + 2 * k.rows * (nh // grp)) + (4 * nr * nh if self.used == 2 else 0)
        # (by the whole tensors: a rank that has some of the heads sums in the same parts; one that has some of the rows cuts
        # them at other keys, and may differ in the last bit)
        a.twice = few_rows(q.rows, q.heads, causal, delta, FEW_ROWS_FORWARD)
        a.single, a.parts = dense_plan(q.rows, k.rows, q.heads, hd, causal, delta, bool(a.twice))
        self.device_arrays = []
        if a.parts > 1:
            a.scratch_bytes = 4 * a.parts * (-(-nr // 32) * 32) * nh * (hd + 1)
            a.dev_scratch = dev.alloc(a.scratch_bytes)
            self.device_arrays = [a.dev_scratch]
            self.launches = 2
        self.fps = _footprints(arena, (q, k, v), writes, stmt_id)

    def launch(self, dev, arena_ptr):
        self.args.arena = arena_ptr
        dev.check(dev.lib.ktb_launch_attention_dense(dev.h, C.byref(self.args)))

    def footprints(self):
        return self.fps

    def bytes_moved(self):
        return self._bytes


def grad_parts(q_len: int, kv_len: int, heads: int, kv_heads: int, causal: int, delta: int) -> Tuple[int, int]:
    """Parts that the walks of the key tiles and of the query tiles are cut into.

    CTAs take tiles as they come free, longest first, so that a walk matters only where it is not well below an SM's share of
    all steps: one key head of eight over 1000 positions is 8 walks of 128 steps of 0.8 us, and 64 of 16 for the queries (64
    wide 92 us whole, 31 in eight parts; over 8192 positions, 128 wide 846 whole, 459 in two, 395 in four).  Such walks are cut to
    three quarters of the share, or to nine steps where that is more (a part costs two microseconds to start and end, joining three)."""
    def steps(rows, first, last, copies):
        """Of every tile: streamed tiles from that of position ``first`` to that of ``last`` (arrays over the tiles)."""
        return np.maximum(last // STEP + 1 - first // STEP, 0) * copies
    k0, q0 = np.arange(0, kv_len, TILE, dtype=np.int64), np.arange(0, q_len, TILE, dtype=np.int64)
    k_first = np.clip(k0 - delta, 0, None) if causal else np.zeros_like(k0)
    of_keys = np.where(k_first < q_len, steps(kv_len, k_first, q_len - 1, heads // kv_heads), 0)
    q_last = np.minimum(np.minimum(q0 + TILE, q_len) - 1 + delta, kv_len - 1) if causal else np.full_like(q0, kv_len - 1)
    of_queries = np.where(q_last >= 0, steps(q_len, 0, np.maximum(q_last, 0), 1), 0)
    most = max(0.75 * (int(of_keys.sum()) * kv_heads * 1.3 + int(of_queries.sum()) * heads) / SMS, 9)
    return tuple(min(16, max(1, round(int(n.max()) / most))) for n in (of_keys, of_queries))


def grad_scratch_bytes(a: "R.AttnBwdArgs") -> int:
    """``ktb_attention_bwd_scratch_bytes``: a counter, three floats per query (in tiles of 64) and head, one per key and key head,
    two per block of queries and head and one per block of keys and key head, where a block is 64 or 256 rows of a head or as many of up to eight heads; and the
    f32 sums of the parts of cut walks."""
    def up(n):
        return -(-n // 256) * 256

    def blocks(rows, n):
        return -(-rows // (block >> min(3, n.bit_length() - 1)))
    padded, kv_heads = -(-a.q_len // 64) * 64, a.heads // a.kv_group
    block = 64 if a.q_len * a.heads + a.kv_len * kv_heads <= 16384 else 256
    total = up(256 + 4 * a.heads * (3 * padded + 2 * blocks(padded, a.heads)) + 4 * kv_heads * (blocks(a.kv_len, kv_heads) + a.kv_len))
    if a.want & R.ATTN_DQ and a.query_parts > 1:
        total += up(4 * a.query_parts * a.head_dim * a.dq_rows * a.dq_heads)
    if a.want & (R.ATTN_DK | R.ATTN_DV) and a.key_parts > 1:
        total += 2 * up(4 * a.key_parts * a.head_dim * a.dk_rows * a.dk_heads)
    return total


class AttentionGradStatement(Statement):
    """dQ, dK and dV, or some of them, of one attention: stores join as long as they are of the same tensors and mask."""
    kind = "attention_bwd"
    launches = 2                                  # what the rows bring, the gradients

    def __init__(self, dev: R.Device, store: Store, arena: ArenaMap, stmt_id: int):
        self.dev, self.arena, self.id = dev, arena, stmt_id
        self.parts = {}
        name, part = self._part(store)
        self.parts[name] = part
        self.device_arrays = []
        self._bind()

    def _part(self, store: Store):
        found = match_gradient(store.value)
        if found is None or not isinstance(store.target, Access):
            raise Unsupported("not a gradient of attention")
        name, m = found
        sel, _ = _points(store)
        if not len(sel):
            raise Unsupported("a store that no core executes")
        T = m["loop"].trips
        ext = tuple(store.axes) + (T,)
        hd = int(m["q"].shape[-1])
        if hd not in (64, 128):
            raise Unsupported("attention gradient supports head_dim 64 and 128")
        if not _scores_below(m["scale"], hd, BACKWARD_SCORES):
            raise Unsupported("a score scale that is not finite, or scores that may not be")
        over_keys = name == "dq"

        def own(acc, what="Read from"):
            return _walk(acc, store.axes, sel, None, hd, self.arena, what)

        def streamed(acc, h=hd):
            w = _walk(acc, store.axes, sel, T, h, self.arena, "Read from")
            _streams_all(w)
            return w
        q_side, k_side = (own, streamed) if over_keys else (streamed, own)
        t = {"q": q_side(m["q"]), "k": k_side(m["k"]), "do": q_side(m["do"])}
        t["lse"] = _walk(m["lse"], store.axes, sel, None, None, self.arena, "Read from") if over_keys else streamed(m["lse"], None)
        if name != "dv":
            t["v"], t["o"] = k_side(m["v"]), q_side(m["o"])
        q, k = t["q"], t["k"]
        out = own(store.target, "Scatter to")
        grp = q.count[1]
        mirror = q if over_keys else k
        for w in (t["do"], t["lse"]) + ((t["o"],) if "o" in t else ()):
            if w.count != q.count or (w.rows, w.heads) != (q.rows, q.heads) or (w.row0 != q.row0).any() or (w.head0 != q.head0).any():
                raise Unsupported("attention tensors of the queries differ in tiles or shape")
        if "v" in t and (t["v"].count != k.count or (t["v"].rows, t["v"].heads) != (k.rows, k.heads) or (t["v"].row0 != k.row0).any() or (t["v"].head0 != k.head0).any()):
            raise Unsupported("keys and values differ in tiles or shape")
        if out.count != mirror.count or (out.rows, out.heads) != (mirror.rows, mirror.heads) or (out.row0 != mirror.row0).any() or (out.head0 != mirror.head0).any():
            raise Unsupported("a gradient stored elsewhere than its tensor lies")
        if k.count[1] != 1 or q.heads != k.heads * grp or (q.head0 % grp).any() or (k.head0[:, :1] != q.head0[:, :1] // grp).any() or \
                m["tile"] != (q.count[0] * grp, k.count[0]):
            raise Unsupported("key heads do not follow the query heads")
        if {w.dtype for w in (q, k, t["do"], out)} != {"f16"}:
            raise Unsupported("attention operands must be f16")
        mask = _mask(m, q, k, ext, sel, T)
        _aligned(*[w for n, w in t.items() if n != "lse"], out)
        common = {n: w.tensor() for n, w in t.items()}
        common.update(mask=mask, scale=float(np.float32(m["scale"])), grp=grp, hd=hd)
        return name, dict(common=common, walks=t, out=out, rect=_rectangle(out))

    def try_absorb(self, store: Store) -> bool:
        try:
            name, part = self._part(store)
        except Unsupported:
            return False
        if name in self.parts:
            return False
        for p in self.parts.values():
            both = p["common"].keys() & part["common"].keys()
            if any(p["common"][n] != part["common"][n] for n in both):
                return False
        other = {"dk": "dv", "dv": "dk"}.get(name)
        if other in self.parts and self.parts[other]["rect"] != part["rect"]:
            return False
        trial = dict(self.parts, **{name: part})
        if not self._apart(trial):
            return False
        self.parts = trial
        self._bind()
        return True

    def _apart(self, parts) -> bool:
        hd = next(iter(parts.values()))["common"]["hd"]
        return _disjoint(self.arena, [w for p in parts.values() for w in p["walks"].values()],
                         [_written(p["out"], p["rect"], hd) for p in parts.values()])

    def _bind(self):
        if not self._apart(self.parts):
            raise Unsupported("a gradient stored over a tensor that it is made from")
        walks, common = {}, {}
        for p in self.parts.values():
            walks.update(p["walks"])
            common.update(p["common"])
        hd = common["hd"]
        if "v" not in walks:                      # dV alone: the kernel wants all operands, and does nothing with these
            walks["v"], walks["o"] = walks["k"], walks["do"]
        self.args = a = R.AttnBwdArgs()
        for n, w in walks.items():
            setattr(a, f"{n}_off", w.base)
            setattr(a, f"{n}_row", w.row)
            setattr(a, f"{n}_head", w.head)
        q, k = walks["q"], walks["k"]
        a.q_len, a.kv_len, a.heads, a.kv_group, a.head_dim = q.rows, k.rows, q.heads, common["grp"], hd
        a.causal, a.causal_delta = common["mask"]
        a.scale = common["scale"]
        writes = []
        seen = np.full(q.rows, k.rows) if not a.causal else np.clip(np.arange(q.rows) + 1 + a.causal_delta, 0, k.rows)
        self._bytes = 2 * hd * (3 * q.rows * q.heads + 2 * k.rows * k.heads)
        for name, p in self.parts.items():
            w = p["out"]
            setattr(a, f"{name}_off", w.base)
            setattr(a, f"{name}_row", w.row)
            setattr(a, f"{name}_head", w.head)
            a.want |= {"dq": R.ATTN_DQ, "dk": R.ATTN_DK, "dv": R.ATTN_DV}[name]
            pre = "dq" if name == "dq" else "dk"
            for n, v in zip(("row0", "rows", "head0", "heads"), p["rect"]):
                setattr(a, f"{pre}_{n}", v)
            writes.append(_written(w, p["rect"], hd))
            self._bytes += 2 * hd * p["rect"][1] * p["rect"][3]
        self.flops = int(10 * q.heads * hd * seen.sum())
        for ptr in self.device_arrays:
            self.dev.free(ptr)
        self.device_arrays = []
        # (of a single key, that same kernel keeps what two orders of a sum differ by from passing for a gradient)
        a.twice = a.kv_len == 1 or few_rows(a.q_len, a.heads, a.causal, a.causal_delta, FEW_ROWS_BACKWARD)
        self._cut(self.dev, *grad_parts(a.q_len, a.kv_len, a.heads, k.heads, a.causal, a.causal_delta))
        self.fps = _footprints(self.arena, walks.values(), writes, self.id)

    def _cut(self, dev, key_parts: int, query_parts: int):
        """The parts of the walks, and scratch for them.  (They follow from the whole tensors: a rank that has some of the heads
        sums in the same parts; one that has some of the rows cuts them elsewhere, and may differ in the last bit.)"""
        a = self.args
        for ptr in self.device_arrays:
            dev.free(ptr)
        a.key_parts, a.query_parts = key_parts, query_parts
        a.scratch_bytes = grad_scratch_bytes(a)
        a.dev_scratch = dev.alloc(a.scratch_bytes)
        self.device_arrays = [a.dev_scratch]
        self.launches = 3 if max(key_parts, query_parts) > 1 else 2

    def launch(self, dev, arena_ptr):
        self.args.arena = arena_ptr
        dev.check(dev.lib.ktb_launch_attention_bwd(dev.h, C.byref(self.args)))

    def footprints(self):
        return self.fps

    def bytes_moved(self):
        return self._bytes


def try_lower_attention_train(dev, stores: List[Store], arena: ArenaMap, stmt_id: int):
    """(statement, how many of the first ``stores`` it runs), or None."""
    m = match_forward(stores[0].value)
    if m is not None:
        try:
            stmt = AttentionDenseStatement(dev, stores, m, arena, stmt_id)
        except Unsupported:
            return None
        return stmt, stmt.used
    if match_gradient(stores[0].value) is None:
        return None
    try:
        stmt = AttentionGradStatement(dev, stores[0], arena, stmt_id)
    except Unsupported:
        return None
    used = 1
    while used < len(stores) and stmt.try_absorb(stores[used]):
        used += 1
    return stmt, used
