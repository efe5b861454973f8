"""Attention over whole sequences and its gradients: the KTIR text against the formulas in 64 bits and the formulas' gradient
against differences, what plans as one launch and what does not, and (on the GPU) the kernels against the formulas.

The bars are sums of the roundings that the kernels make.  P and dS are rounded to f16 before they are multiplied: half a step,
2^-11 of the value, or 2^-25 below the normal numbers after the kernel's shift (2^14 for P <= 1, 2^14 / B for dS, where B is at most
four times |dO| |V| in 2-norms).  Results are rounded to f16: 2^-11 (and 2^-25).  Scores, exp, sums and statistics are f32: F32 =
2^-16 of the sums of absolute values leaves 2^7 roundings of 2^-24 and a 2^-22 exp on scores of a few units each.
"""
import ctypes as C
import math

import numpy as np
import pytest

from ktir_cpu_b200 import HardwareConfig, KTIRInterpreter, kernels as K, runtime as R
from ktir_cpu_b200.interpreter import Session
from ktir_cpu_b200.lower_attn_train import FEW_ROWS_BACKWARD, FEW_ROWS_FORWARD, dense_plan, few_rows, grad_parts, grad_scratch_bytes
from ktir_cpu_b200.parser import KTIRParser
from oracle.numpy_interp import OracleInterpreter

HALF, F32 = 2.0 ** -11, 2.0 ** -16
FWD, BWD = "attention_forward_kernel", "attention_backward_kernel"


def _inputs(q_len, kv_len, heads, kv_heads, hd, seed=0, grad=1.0):
    rng = np.random.default_rng(seed)
    f = lambda *s: rng.standard_normal(s, dtype=np.float32).astype(np.float16)     # noqa: E731
    kw = dict(query_ptr=f(q_len, heads, hd), key_ptr=f(kv_len, kv_heads, hd), value_ptr=f(kv_len, kv_heads, hd))
    return kw, (rng.standard_normal((q_len, heads, hd)) * grad).astype(np.float16)


def _scale(hd):
    return np.float32(1.0 / math.sqrt(hd))


def _seen(q_len, kv_len, causal):
    i, j = np.arange(q_len)[:, None], np.arange(kv_len)[None, :]
    return j <= i + kv_len - q_len if causal else np.ones((q_len, kv_len), bool)


def formulas(kw, do, causal, o=None, lse=None, scale=None, half=HALF):
    """Outputs in 64 bits and, for each, a bound on what the kernels' roundings move: name -> (value, bound).  ``half``: of P and dS."""
    q, k, v = (kw[n].astype(np.float64).transpose(1, 0, 2) for n in ("query_ptr", "key_ptr", "value_ptr"))
    grp, (q_len, kv_len) = len(q) // len(k), (q.shape[1], k.shape[1])
    k, v = np.repeat(k, grp, 0), np.repeat(v, grp, 0)
    scale = float(_scale(q.shape[2])) if scale is None else float(scale)
    seen = _seen(q_len, kv_len, causal)
    with np.errstate(all="ignore"):
        s = np.where(seen, scale * (q @ k.transpose(0, 2, 1)), -np.inf)
        m = np.maximum(s.max(-1, keepdims=True), -1e30)
        e = np.exp(s - m)
        total = e.sum(-1, keepdims=True)
        p = e / np.maximum(total, 1e-30)
        out = {}
        if do is None:
            res, spread = p @ v, p @ np.abs(v)
            out["output_ptr"] = (res, (half + F32) * spread + HALF * np.abs(res) + 2.0 ** -25)
            l64 = (m + np.log(total))[..., 0]
            out["lse_ptr"] = (l64[..., None], 2.0 ** -19 * (1 + np.abs(np.where(np.isfinite(l64), l64, 0)))[..., None])
        else:
            do, o, lse = do.astype(np.float64).transpose(1, 0, 2), o.astype(np.float64).transpose(1, 0, 2), lse.astype(np.float64).T[..., None]
            p = np.where(seen, np.exp(s - lse), 0.0)
            dp, d = do @ v.transpose(0, 2, 1), (do * o).sum(-1, keepdims=True)
            ds = p * (dp - d)
            norm = lambda x: np.sqrt((x * x).sum(-1))     # noqa: E731
            shared = lambda x: x.reshape((-1, grp) + x.shape[1:]).sum(1)     # noqa: E731
            big = norm(do).reshape(-1, grp * q_len).max(-1) * norm(v)[::grp].max(-1) + np.abs(d).reshape(-1, grp * q_len).max(-1)
            floor = np.repeat(2.0 * big, grp)[:, None, None] * 2.0 ** -39      # half of f16's smallest step, shifted back
            # what f32 moves in dS: P from the scores, dO V^T and D from their own sums
            size = p * (np.abs(do) @ np.abs(v).transpose(0, 2, 1) + (np.abs(do) * np.abs(o)).sum(-1, keepdims=True))
            eds = half * np.abs(ds) + F32 * size + np.where(seen, floor, 0)
            ep = (half + F32) * p + np.where(seen, 2.0 ** -39, 0)
            for name, val, err in (("query_grad_ptr", scale * (ds @ k), scale * (eds @ np.abs(k) + F32 * (np.abs(ds) @ np.abs(k)))),
                                   ("key_grad_ptr", scale * shared(ds.transpose(0, 2, 1) @ q), scale * shared(eds.transpose(0, 2, 1) @ np.abs(q) + F32 * (np.abs(ds).transpose(0, 2, 1) @ np.abs(q)))),
                                   ("value_grad_ptr", shared(p.transpose(0, 2, 1) @ do), shared(ep.transpose(0, 2, 1) @ np.abs(do)))):
                out[name] = (val, err + HALF * np.abs(val) + 2.0 ** -25)
    back = lambda x: x.transpose(1, 0, 2)     # noqa: E731
    return {n: ((back(v)[..., 0], back(b)[..., 0]) if n == "lse_ptr" else (back(v), back(b))) for n, (v, b) in out.items()}


def _check(got, want):
    for n, (val, bound) in want.items():
        x = got[n].astype(np.float64)
        fin = np.isfinite(val)
        np.testing.assert_array_equal(x[~fin], val[~fin], err_msg=n)
        off = np.abs(x[fin] - val[fin]) / bound[fin]
        assert np.isfinite(x[fin]).all() and (off <= 1).all(), (n, int((off > 1).sum()), float(off.max()))


def _kwargs(fn, kw, q_len, heads, hd, do=None, o=None, lse=None, scale=None):
    scale = _scale(hd) if scale is None else scale
    if fn == FWD:
        return dict(output_ptr=np.full((q_len, heads, hd), np.nan, np.float16), lse_ptr=np.full((q_len, heads), np.nan, np.float32), **kw, scale=scale)
    nan = lambda a: np.full_like(a, np.nan)     # noqa: E731
    return dict(query_grad_ptr=nan(kw["query_ptr"]), key_grad_ptr=nan(kw["key_ptr"]), value_grad_ptr=nan(kw["value_ptr"]), **kw,
                output_ptr=o, lse_ptr=lse, output_grad_ptr=do, scale=scale)


def _forward_results(kw, causal, scale=None):
    """What a forward pass leaves: O as f16 and lse as f32."""
    want = formulas(kw, None, causal, scale=scale)
    return want["output_ptr"][0].astype(np.float16), want["lse_ptr"][0].astype(np.float32)


def _oracle(src, fn, kw):
    ora = OracleInterpreter()
    ora.load(src)
    with np.errstate(all="ignore"):
        return ora.execute_function(fn, **kw)


def _session(src, fn, kw, **more):
    t = [(k, v.shape, v.dtype) for k, v in kw.items() if isinstance(v, np.ndarray)]
    return Session(R.PlanOnlyDevice(), KTIRParser().parse_module(src).get_function(fn), t, dict(scale=kw["scale"]), arena_ptr=0, **more)


# (queries, keys, heads, key heads, head size, causal): even tiles; odd lengths; more keys; more queries (rows that see nothing);
# one of each; groups that divide no tile
TEXT = [(32, 32, 2, 2, 16, True), (19, 19, 4, 2, 8, False), (13, 29, 3, 1, 8, True), (21, 9, 2, 2, 8, True), (1, 1, 1, 1, 8, True),
        (1, 17, 6, 2, 8, False), (9, 1, 2, 1, 8, True)]


@pytest.mark.parametrize("blocks", [(None, None), (4, 8)])
@pytest.mark.parametrize("q_len,kv_len,heads,kv_heads,hd,causal", TEXT)
def test_text_says_the_formulas(q_len, kv_len, heads, kv_heads, hd, causal, blocks):
    blocks = [b if b is None else min(b, n) for b, n in zip(blocks, (q_len, kv_len))]
    kw, do = _inputs(q_len, kv_len, heads, kv_heads, hd)
    got = _oracle(K.attention_forward(q_len, kv_len, heads, kv_heads, hd, causal, *blocks), FWD, _kwargs(FWD, kw, q_len, heads, hd))
    _check(got, formulas(kw, None, causal))
    o, lse = _forward_results(kw, causal)
    got = _oracle(K.attention_backward(q_len, kv_len, heads, kv_heads, hd, causal, *blocks), BWD, _kwargs(BWD, kw, q_len, heads, hd, do, o, lse))
    _check(got, formulas(kw, do, causal, o, lse))


@pytest.mark.parametrize("q_len,kv_len,causal", [(5, 5, True), (4, 7, False), (6, 4, True)])
def test_gradient_formulas_against_differences(q_len, kv_len, causal):
    """<dO, O(x + h u) - O(x - h u)> / 2h = <gradient, u>, in 64 bits: h = 2^-14 leaves h^2 of the third derivative (order 10)
    and 2^-52 / h of rounding, both below 1e-7."""
    kw, do = _inputs(q_len, kv_len, 4, 2, 8, seed=5)
    kw = {n: x.astype(np.float64) for n, x in kw.items()}
    fwd = formulas(kw, None, causal)
    grads = formulas(kw, do, causal, fwd["output_ptr"][0], fwd["lse_ptr"][0])
    rng, h = np.random.default_rng(1), 2.0 ** -14
    for x, g in (("query_ptr", "query_grad_ptr"), ("key_ptr", "key_grad_ptr"), ("value_ptr", "value_grad_ptr")):
        u = rng.standard_normal(kw[x].shape)
        up, down = (formulas({**kw, x: kw[x] + t * u}, None, causal)["output_ptr"][0] for t in (h, -h))
        np.testing.assert_allclose((do * (up - down)).sum() / (2 * h), (grads[g][0] * u).sum(), rtol=1e-6, atol=1e-6)


# ---- plans ---------------------------------------------------------------------------------------------------------
PLANS = [(256, 256, 8, 2, 128, True, None, None), (197, 197, 12, 12, 64, False, None, None), (100, 333, 6, 2, 64, True, 16, 64),
         (333, 100, 5, 1, 128, True, 10, 32), (1, 1, 7, 7, 128, True, None, None), (1, 500, 12, 4, 64, False, None, 100),
         (37, 37, 4, 4, 128, True, 37, 1)]


@pytest.mark.parametrize("q_len,kv_len,heads,kv_heads,hd,causal,bq,bn", PLANS)
def test_each_direction_plans_as_one_statement(q_len, kv_len, heads, kv_heads, hd, causal, bq, bn):
    kw, do = _inputs(q_len, kv_len, heads, kv_heads, hd)
    full = _kwargs(FWD, kw, q_len, heads, hd)
    sess = _session(K.attention_forward(q_len, kv_len, heads, kv_heads, hd, causal, bq, bn), FWD, full)
    st, = sess.plan.statements
    a = st.args
    assert st.kind == "attention_dense" and (a.q_len, a.kv_len, a.heads, a.kv_group, a.head_dim) == (q_len, kv_len, heads, heads // kv_heads, hd)
    assert (a.causal, a.causal_delta) == ((1, kv_len - q_len) if causal else (0, 0)) and a.lse_off >= 0
    assert sess.plan.fully_overwritten == {"output_ptr", "lse_ptr"}
    full = _kwargs(BWD, kw, q_len, heads, hd, do, do, full["lse_ptr"])
    sess = _session(K.attention_backward(q_len, kv_len, heads, kv_heads, hd, causal, bq, bn), BWD, full)
    st, = sess.plan.statements
    a = st.args
    assert st.kind == "attention_bwd" and a.want == 7 and (a.q_len, a.kv_len, a.heads, a.kv_group, a.head_dim) == (q_len, kv_len, heads, heads // kv_heads, hd)
    assert (a.causal, a.causal_delta) == ((1, kv_len - q_len) if causal else (0, 0)) and a.scale == _scale(hd)
    assert (a.dq_row0, a.dq_rows, a.dq_head0, a.dq_heads, a.dk_row0, a.dk_rows, a.dk_head0, a.dk_heads) == (0, q_len, 0, heads, 0, kv_len, 0, kv_heads)
    assert sess.plan.fully_overwritten == {"query_grad_ptr", "key_grad_ptr", "value_grad_ptr"}


def _kinds(src, fn, kw):
    try:
        return [s.kind for s in _session(src, fn, kw).plan.statements]
    except NotImplementedError:
        return []


@pytest.mark.parametrize("old,new", [
    ("%masked_o : f32):", "%masked_o : f32):\n          %never = arith.constant 0.0 : f32"),       # (an unused value changes nothing)
    ("arith.cmpi sle, %k_pos, %q_pos", "arith.cmpi sge, %k_pos, %q_pos"), ("arith.cmpi sle, %k_pos, %q_pos", "arith.cmpi ule, %k_pos, %q_pos"),
    ("%low = arith.constant -1.0e30", "%low = arith.constant -10.0"), ("%tiny = arith.constant 1.0e-30", "%tiny = arith.constant 2.0"),
    ("arith.maximumf %m_run, %rmax", "arith.minimumf %m_run, %rmax"), ("arith.addf %m_fin, %l_log", "arith.subf %m_fin, %l_log"),
    ("%l_init = tensor.splat %zero", "%l_init = tensor.splat %tiny"), ("arith.divui %r, %c_grp", "arith.divui %r, %c_bn")])
def test_other_forward_texts_are_not_taken_for_it(old, new):
    kw, _ = _inputs(64, 40, 4, 2, 64)
    src = K.attention_forward(64, 40, 4, 2, 64, True, 16, 8)
    assert old in src
    full = _kwargs(FWD, kw, 64, 4, 64)
    assert _kinds(src, FWD, full) == ["attention_dense"]
    changed = _kinds(src.replace(old, new), FWD, full)
    if "never" in new:
        assert changed == ["attention_dense"]
    elif "l_log" in old:
        assert changed == ["attention_dense", "generic"]            # O as before, the other store on its own
    else:
        assert "attention_dense" not in changed


@pytest.mark.parametrize("old,new,left", [
    ("%dq_sc = tensor.splat %scale", "%dq_sc = tensor.splat %zero", ["generic", "attention_bwd"]),
    ("%dk_sc = tensor.splat %scale", "%dk_sc = tensor.splat %zero", ["attention_bwd", "generic", "attention_bwd"]),
    ("%a_dpd = arith.subf", "%a_dpd = arith.addf", ["generic", "attention_bwd"]),
    # (another tensor in dO's or O's place is a gradient of its own, not one of the same attention)
    ("ins(%dv_t, %b_do", "ins(%dv_t, %b_q", ["attention_bwd", "attention_bwd"]),
    ("%b_doo = arith.mulf %b_do, %b_o", "%b_doo = arith.mulf %b_do, %b_do", ["attention_bwd", "attention_bwd"]),
    ("%a_k0 = arith.muli %j, %c_bn", "%a_k0 = arith.muli %c0, %c_bn", ["generic", "attention_bwd"])])
def test_other_gradient_texts_are_not_taken_for_it(old, new, left):
    kw, do = _inputs(64, 64, 4, 2, 64)
    src = K.attention_backward(64, 64, 4, 2, 64, True, 16, 32)
    assert old in src
    full = _kwargs(BWD, kw, 64, 4, 64, do, do, np.zeros((64, 4), np.float32))
    assert _kinds(src, BWD, full) == ["attention_bwd"]
    assert _kinds(src.replace(old, new), BWD, full) == left


def test_some_of_the_gradients():
    kw, do = _inputs(64, 64, 4, 2, 64)
    src = K.attention_backward(64, 64, 4, 2, 64, True)
    full = _kwargs(BWD, kw, 64, 4, 64, do, do, np.zeros((64, 4), np.float32))
    lines = src.split("\n")
    for drop, want in ((("dq",), 6), (("dk",), 5), (("dv",), 3), (("dq", "dk"), 4), (("dk", "dv"), 1)):
        text = "\n".join(ln for ln in lines if not any(f"ktdp.store %{d}_3" in ln for d in drop))
        st, = _session(text, BWD, full).plan.statements
        assert st.kind == "attention_bwd" and st.args.want == want


@pytest.mark.parametrize("grad,over,never", [("query_grad", "output_grad", 1), ("key_grad", "value", 2), ("value_grad", "key_grad", 6)])
def test_a_gradient_over_what_is_read_or_stored_does_not_join(grad, over, never):
    kw, do = _inputs(64, 64, 2, 2, 64)
    src = K.attention_backward(64, 64, 2, 2, 64, False).replace(f"construct_memory_view %{grad}_ptr", f"construct_memory_view %{over}_ptr")
    try:
        plan = _session(src, BWD, _kwargs(BWD, kw, 64, 2, 64, do, do, np.zeros((64, 2), np.float32))).plan
    except NotImplementedError:
        return
    for st in plan.statements:
        assert st.kind != "attention_bwd" or st.args.want & never != never


@pytest.mark.parametrize("world", [2, 3])
def test_ranks_take_their_heads(world):
    kw, do = _inputs(64, 96, 12, 6, 64)
    full = _kwargs(BWD, kw, 64, 12, 64, do, do, np.zeros((64, 12), np.float32))
    src = K.attention_backward(64, 96, 12, 6, 64, True, 16, 32)
    covered = []
    for r in range(world):
        a = _session(src, BWD, full, shard=(r, world)).plan.statements[0].args
        covered.append((a.dq_head0, a.dq_heads, a.dk_head0, a.dk_heads, a.want))
    per = 6 // world
    assert covered == [(r * per * 2, per * 2, r * per, per, 7) for r in range(world)]


@pytest.mark.parametrize("scale,fwd,bwd", [(0.0, 0, 1), (-0.5, 0, 1), (float("nan"), 0, 0), (float("inf"), 0, 0), (1e-30, 1, 1)])
def test_scales_that_the_kernels_do_not_take_run_step_by_step(scale, fwd, bwd):
    kw, do = _inputs(64, 64, 4, 2, 64)
    o, lse = _forward_results(kw, True)
    for fn, make, kind, fused in ((FWD, K.attention_forward, "attention_dense", fwd), (BWD, K.attention_backward, "attention_bwd", bwd)):
        sess = _session(make(64, 64, 4, 2, 64, True), fn, _kwargs(fn, kw, 64, 4, 64, do, o, lse, np.float32(scale)))
        kinds = {s.kind for s in sess.plan.statements}
        assert kinds == ({kind} if fused else {"generic"})


@pytest.mark.parametrize("q_len,kv_len,heads,kv_heads,causal,parts", [
    (2048, 2048, 256, 256, True, (1, 1)), (197, 197, 12, 12, False, (1, 1)), (8192, 8192, 16, 4, True, (1, 1)),   # enough tiles
    (1000, 1000, 8, 1, False, (11, 1)), (1, 8192, 32, 8, True, (1, 4)), (4096, 4096, 1, 1, False, (3, 3)), (1, 1, 1, 1, True, (1, 1)),
    (100, 20, 2, 2, True, (1, 1)), (4096, 64, 8, 1, False, (16, 1))])
def test_long_walks_are_cut_where_there_are_few(q_len, kv_len, heads, kv_heads, causal, parts):
    assert grad_parts(q_len, kv_len, heads, kv_heads, int(causal), kv_len - q_len if causal else 0) == parts


@pytest.mark.parametrize("q_len,kv_len,heads,hd,causal,plan", [
    (2048, 2048, 256, 128, 1, (0, 1)), (197, 197, 12, 64, 0, (0, 1)), (1, 1, 1, 128, 1, (0, 1)), (842, 842, 8, 64, 0, (1, 4)), (1024, 1024, 8, 128, 1, (1, 4)),
    (1531, 4603, 32, 128, 1, (1, 1)), (1, 8192, 32, 128, 1, (0, 4)), (1024, 65536, 37, 128, 0, (1, 1)), (8192, 8192, 512, 64, 1, (0, 1)), (100, 7, 3, 64, 1, (0, 1)),
    (4096, 4096, 16, 128, 1, (1, 1)), (1, 65536, 4, 64, 0, (0, 16))])
def test_few_items_are_single_or_in_parts(q_len, kv_len, heads, hd, causal, plan):
    assert dense_plan(q_len, kv_len, heads, hd, causal, kv_len - q_len if causal else 0, False) == plan


def test_few_rows_are_those_that_see_a_key():
    assert few_rows(1, 256, 0, 0, 256) and not few_rows(1, 257, 0, 0, 256) and not few_rows(300, 1, 0, -299, 256)
    assert few_rows(8000, 8, 1, 32 - 8000, 256) and not few_rows(33, 8, 1, 50, 256)


@pytest.mark.parametrize("parts", [(1, 1), (3, 1), (1, 5), (8, 8), (0, 0)])
@pytest.mark.parametrize("want", [7, 1, 2, 6])
def test_scratch_is_what_the_library_asks_for(parts, want, build_lib):
    a = R.AttnBwdArgs()
    for heads, group, q_len, kv_len, hd in ((1, 1, 1, 1, 64), (14, 2, 333, 1, 128), (256, 1, 2048, 2048, 128), (40, 8, 65, 8191, 64)):
        a.q_len, a.kv_len, a.heads, a.kv_group, a.head_dim, a.want = q_len, kv_len, heads, group, hd, want
        a.dq_rows, a.dq_heads, a.dk_rows, a.dk_heads = q_len, heads, kv_len, heads // group
        a.key_parts, a.query_parts = parts
        assert grad_scratch_bytes(a) == R.lib().ktb_attention_bwd_scratch_bytes(C.byref(a))


# ---- kernels -------------------------------------------------------------------------------------------------------
# (queries, keys, heads, key heads, head size, causal): one token; keys and queries around tiles of 64 and 128; odd lengths;
# groups; more queries than keys by more and by less than a tile; a context before a few queries; no mask
CASES = [(1, 1, 1, 1, 128, True), (1, 1, 2, 1, 64, False), (1, 300, 6, 2, 128, True), (64, 64, 2, 2, 64, True), (65, 65, 2, 2, 128, True),
         (127, 129, 3, 3, 64, True), (128, 128, 4, 1, 128, True), (129, 127, 4, 2, 128, True), (197, 197, 5, 5, 64, False), (300, 111, 3, 1, 64, True),
         (513, 100, 2, 2, 128, True), (70, 500, 14, 2, 128, False), (257, 771, 3, 3, 128, True), (640, 640, 2, 1, 64, True), (191, 64, 2, 2, 64, False),
         (1000, 3, 2, 2, 128, False), (3, 1000, 10, 2, 64, True), (385, 449, 7, 1, 128, True),
         # few tiles with long walks: in parts
         (1000, 1000, 8, 1, 64, True), (1, 3000, 4, 2, 128, True), (130, 4000, 2, 2, 64, False), (2000, 70, 5, 1, 128, False)]


def _run(src, fn, full, kind, times=1):
    gpu = KTIRInterpreter()
    gpu.load(src)
    outs = [gpu.execute_function(fn, **full) for _ in range(times)]
    kinds = [s.kind for sess in gpu._sessions.values() for s in sess.plan.statements]
    gpu.close()
    assert kinds == [kind]
    for other in outs[1:]:
        for n, x in outs[0].items():
            np.testing.assert_array_equal(np.ascontiguousarray(x).view(np.uint8), np.ascontiguousarray(other[n]).view(np.uint8))
    return outs[0]


@pytest.mark.gpu
@pytest.mark.parametrize("q_len,kv_len,heads,kv_heads,hd,causal", CASES)
def test_forward(q_len, kv_len, heads, kv_heads, hd, causal, build_lib):
    kw, _ = _inputs(q_len, kv_len, heads, kv_heads, hd, seed=q_len)
    src = K.attention_forward(q_len, kv_len, heads, kv_heads, hd, causal)
    got = _run(src, FWD, _kwargs(FWD, kw, q_len, heads, hd), "attention_dense", times=3)
    _check(got, formulas(kw, None, causal))


@pytest.mark.gpu
@pytest.mark.parametrize("plan", [(0, 1), (1, 1), (0, 3), (1, 2), (1, 7)])
@pytest.mark.parametrize("c", [(2500, 1540, 2, 1, 128, True), (257, 2200, 3, 3, 64, True), (1, 4400, 1, 1, 128, True), (300, 2000, 30, 2, 64, False), (700, 1601, 4, 4, 128, True),
                               (513, 70, 120, 4, 64, False), (90, 33, 5, 1, 128, True), (1100, 1100, 70, 7, 64, True)])
def test_forward_however_it_is_dealt_out(c, plan, build_lib, monkeypatch):
    """Parts that rows see nothing of, rows that see nothing at all, a last part that fills no step, more parts than pages, more items
    than SMs."""
    from ktir_cpu_b200 import lower_attn_train
    monkeypatch.setattr(lower_attn_train, "dense_plan", lambda *a: plan)
    kw, _ = _inputs(*c[:5], seed=c[1])
    got = _run(K.attention_forward(*c), FWD, _kwargs(FWD, kw, c[0], c[2], c[4]), "attention_dense", times=3)
    _check(got, formulas(kw, None, c[5]))


FEW = [(2, 2, 4, 4, 128, True), (1, 1, 8, 8, 64, False), (6, 14, 8, 4, 64, False), (1, 700, 8, 8, 128, True), (20, 100, 2, 2, 64, False), (3, 5000, 8, 1, 64, True),
       (7, 7, 4, 1, 128, True), (130, 65, 1, 1, 128, False), (100, 8, 4, 4, 64, True), (2, 129, 3, 1, 128, False)]


@pytest.mark.gpu
@pytest.mark.parametrize("c", FEW)
def test_few_rows_lose_nothing_to_f16_operands(c, build_lib):
    """Where few rows see a key, what f16 leaves out of P and dS is multiplied too: 2^-11 of 2^-11 is all that stays out."""
    kw, do = _inputs(*c[:5], seed=c[1])
    got = _run(K.attention_forward(*c), FWD, _kwargs(FWD, kw, c[0], c[2], c[4]), "attention_dense", times=3)
    delta = c[1] - c[0] if c[5] else 0
    _check(got, formulas(kw, None, c[5], half=HALF * HALF if few_rows(c[0], c[2], c[5], delta, FEW_ROWS_FORWARD) else HALF))
    o, lse = _forward_results(kw, c[5])
    got = _run(K.attention_backward(*c), BWD, _kwargs(BWD, kw, c[0], c[2], c[4], do, o, lse), "attention_bwd", times=3)
    assert few_rows(c[0], c[2], c[5], delta, FEW_ROWS_BACKWARD)
    _check(got, formulas(kw, do, c[5], o, lse, half=HALF * HALF))


@pytest.mark.gpu
@pytest.mark.parametrize("q_len,heads,kv_heads,hd,causal", [(1, 4, 4, 64, False), (1, 8, 2, 128, True), (60, 8, 8, 128, False), (60, 4, 1, 64, True)])
def test_one_key_has_no_gradient_of_its_scores(q_len, heads, kv_heads, hd, causal, build_lib):
    """P is 1 whatever the scores are, and O is V: dQ and dK are nothing, not what two orders of a sum differ by."""
    kw, do = _inputs(q_len, 1, heads, kv_heads, hd, seed=hd)
    o, lse = _forward_results(kw, causal)
    got = _run(K.attention_backward(q_len, 1, heads, kv_heads, hd, causal), BWD, _kwargs(BWD, kw, q_len, heads, hd, do, o, lse), "attention_bwd")
    assert not got["query_grad_ptr"].any() and not got["key_grad_ptr"].any() and got["value_grad_ptr"].any()


@pytest.mark.gpu
@pytest.mark.parametrize("q_len,kv_len,heads,kv_heads,hd,causal", CASES)
def test_backward(q_len, kv_len, heads, kv_heads, hd, causal, build_lib):
    kw, do = _inputs(q_len, kv_len, heads, kv_heads, hd, seed=kv_len)
    o, lse = _forward_results(kw, causal)
    src = K.attention_backward(q_len, kv_len, heads, kv_heads, hd, causal)
    got = _run(src, BWD, _kwargs(BWD, kw, q_len, heads, hd, do, o, lse), "attention_bwd", times=3)
    _check(got, formulas(kw, do, causal, o, lse))


@pytest.mark.gpu
@pytest.mark.parametrize("grad", [2.0 ** -10, 1e-6, 100.0])
def test_gradients_of_any_size(grad, build_lib):
    """dS is shifted into the range of f16 and back: small gradients keep their precision, large ones do not overflow."""
    kw, do = _inputs(300, 300, 2, 2, 128, grad=grad)
    o, lse = _forward_results(kw, True)
    got = _run(K.attention_backward(300, 300, 2, 2, 128, True), BWD, _kwargs(BWD, kw, 300, 2, 128, do, o, lse), "attention_bwd")
    _check(got, formulas(kw, do, True, o, lse))


@pytest.mark.gpu
def test_one_loud_row_and_a_silent_one(build_lib):
    """A row of dO 10^5 times the others', one of zeros, and values of a wide range."""
    kw, do = _inputs(200, 333, 4, 2, 64, grad=0.01)
    do[17, 1] *= 1000
    do[30] = 0
    kw["value_ptr"][100] *= 50
    o, lse = _forward_results(kw, False)
    got = _run(K.attention_backward(200, 333, 4, 2, 64, False), BWD, _kwargs(BWD, kw, 200, 4, 64, do, o, lse), "attention_bwd")
    want = formulas(kw, do, False, o, lse)
    _check(got, want)
    # dQ is shifted row by row: the quiet rows keep f16's precision next to the loud one
    quiet = np.abs(got["query_grad_ptr"].astype(np.float64) - want["query_grad_ptr"][0])[31:]
    assert np.linalg.norm(quiet) <= 2 ** -10.5 * np.linalg.norm(want["query_grad_ptr"][0][31:])
    assert (got["query_grad_ptr"][30] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [0.01, 1.0, 3.0])
def test_other_scales(scale, build_lib):
    """Flat probabilities (1 / keys each, below the normal numbers of f16 without the shift) and peaked ones."""
    kw, do = _inputs(500, 2000, 1, 1, 64)
    s = np.float32(scale)
    fw = _run(K.attention_forward(500, 2000, 1, 1, 64, False), FWD, _kwargs(FWD, kw, 500, 1, 64, scale=s), "attention_dense")
    if scale < 2:          # (at 3 the scores reach 100: the f32 bar of a few units does not hold)
        _check(fw, formulas(kw, None, False, scale=s))
    o, lse = fw["output_ptr"], fw["lse_ptr"]
    got = _run(K.attention_backward(500, 2000, 1, 1, 64, False), BWD, _kwargs(BWD, kw, 500, 1, 64, do, o, lse, s), "attention_bwd")
    want = formulas(kw, do, False, o, lse, scale=s)
    for n, (val, bound) in want.items():
        assert np.linalg.norm(got[n] - val) <= 2 ** -10.5 * np.linalg.norm(val) + np.linalg.norm(bound) * (scale > 2), n


@pytest.mark.gpu
def test_infinite_and_nan_gradients_stay_in_their_rows(build_lib):
    kw, do = _inputs(150, 150, 2, 2, 64)
    o, lse = _forward_results(kw, True)
    do[40, 0, 3], do[140, 1, 0] = np.nan, np.inf
    got = _run(K.attention_backward(150, 150, 2, 2, 64, True), BWD, _kwargs(BWD, kw, 150, 2, 64, do, o, lse), "attention_bwd")
    bad = ~np.isfinite(got["query_grad_ptr"].astype(np.float64)).all(-1)
    assert bad[40, 0] and bad[140, 1] and bad.sum() == 2
    # (a hidden pair is 0 * NaN in the formula, so dK and dV of the keys behind are not defined; head 1's first tile is clean)
    assert not np.isfinite(got["key_grad_ptr"][:41, 0].astype(np.float64)).any()
    clean = do.copy()
    clean[40, 0], clean[140, 1] = 0, 0
    want = formulas(kw, clean, True, o, lse)["query_grad_ptr"]
    ok = ~bad
    assert (np.abs(got["query_grad_ptr"].astype(np.float64) - want[0])[ok] <= want[1][ok]).all()


@pytest.mark.gpu
def test_sessions_side_by_side_and_new_inputs(build_lib):
    """Two plans with scratch of their own run in turn, their launches replayed from graphs, on inputs that change."""
    cases = [(200, 200, 2, 2, 64, True), (130, 260, 4, 2, 128, False)]
    interps, sessions, data = [], [], []
    for c in cases:
        q_len, kv_len, heads, kv_heads, hd, causal = c
        gpu = KTIRInterpreter()
        gpu.load(K.attention_backward(*c))
        kw, do = _inputs(*c[:5])
        o, lse = _forward_results(kw, causal)
        sess, _ = gpu.session(BWD, **_kwargs(BWD, kw, q_len, heads, hd, do, o, lse))
        interps.append(gpu)
        sessions.append(sess)
    for turn in range(4):
        for c, sess in zip(cases, sessions):
            q_len, kv_len, heads, kv_heads, hd, causal = c
            kw, do = _inputs(*c[:5], seed=10 + turn)
            o, lse = _forward_results(kw, causal)
            full = _kwargs(BWD, kw, q_len, heads, hd, do, o, lse)
            held = [sess.upload(n, x) for n, x in full.items() if isinstance(x, np.ndarray)]
            data.append((c, kw, do, o, lse, held))
        for sess in sessions:
            sess.run()
        for (c, kw, do, o, lse, _), sess in zip(data[-2:], sessions):
            got = {n: sess.download(n) for n in ("query_grad_ptr", "key_grad_ptr", "value_grad_ptr")}
            sess.dev.sync()
            _check(got, formulas(kw, do, c[5], o, lse))
    for gpu in interps:
        gpu.close()


@pytest.mark.gpu
def test_many_calls_in_flight(build_lib):
    """Candidates of one text on inputs of their own, several under way at a time: one plan's scratch and parts serve them all."""
    from ktir_cpu_b200.batch import Candidate, evaluate_many
    cands = []
    for seed in range(4):
        for c in ((40, 1700, 8, 2, 64, False), (300, 300, 2, 1, 128, True)):
            kw, do = _inputs(*c[:5], seed=seed)
            o, lse = _forward_results(kw, c[5])
            cands.append(Candidate(K.attention_forward(*c), FWD, _kwargs(FWD, kw, c[0], c[2], c[4])))
            cands.append(Candidate(K.attention_backward(*c), BWD, _kwargs(BWD, kw, c[0], c[2], c[4], do, o, lse)))
        x = _inputs(70, 70, 4, 2, 64, seed=seed)[0]
        cos, sin = K.rotary_tables(200, 64)
        at = np.random.default_rng(seed).integers(0, 200, 70).astype(np.int32)
        cands.append(Candidate(K.rotary(70, 4, 2, 64, table_rows=200), "rotary_kernel", dict(
            query_out_ptr=np.zeros((70, 4, 64), np.float16), key_out_ptr=np.zeros((70, 2, 64), np.float16), query_ptr=x["query_ptr"],
            key_ptr=x["key_ptr"], positions_ptr=at, cos_ptr=cos, sin_ptr=sin)))
    res = evaluate_many(cands)
    assert not res.errors
    for i, c in enumerate(cands):
        gpu = KTIRInterpreter()
        gpu.load(c.source)
        want = gpu.execute_function(c.function, **c.kwargs)
        gpu.close()
        assert res.outputs[i].keys() and all(v.tobytes() == want[n].tobytes() for n, v in res.outputs[i].items()), (i, c.function)


@pytest.mark.gpu
def test_a_training_step_of_an_attention_layer(build_lib):
    """Queries and keys turned, attention forward and backward, gradients turned back: every stage against its formula on what
    the stage before it gave."""
    S, H, G, hd, part = 333, 6, 2, 128, 96
    kw, do = _inputs(S, S, H, G, hd, seed=3)
    cos, sin = K.rotary_tables(1024, part)
    pos = ((np.arange(S) + 200) % 333).astype(np.int32)

    def turn(q, k, inverse):
        gpu = KTIRInterpreter()
        gpu.load(K.rotary(S, H, G, hd, part, 1024, "half", inverse))
        r = gpu.execute_function("rotary_kernel", query_out_ptr=np.zeros_like(q), key_out_ptr=np.zeros_like(k), query_ptr=q, key_ptr=k,
                                 positions_ptr=pos, cos_ptr=cos, sin_ptr=sin)
        assert [s.kind for sess in gpu._sessions.values() for s in sess.plan.statements] == ["rotary"]
        gpu.close()
        c, s = cos[pos].astype(np.float64)[:, None], sin[pos].astype(np.float64)[:, None] * (-1 if inverse else 1)
        for x, y in ((q, r["query_out_ptr"]), (k, r["key_out_ptr"])):
            n, x = part // 2, x.astype(np.float64)
            want = np.concatenate([x[..., :n] * c - x[..., n:part] * s, x[..., n:part] * c + x[..., :n] * s, x[..., part:]], -1)
            np.testing.assert_allclose(y.astype(np.float64), want, rtol=HALF, atol=2.0 ** -20)
        return r["query_out_ptr"], r["key_out_ptr"]

    q, k = turn(kw["query_ptr"], kw["key_ptr"], False)
    turned = dict(query_ptr=q, key_ptr=k, value_ptr=kw["value_ptr"])
    fw = _run(K.attention_forward(S, S, H, G, hd, True), FWD, _kwargs(FWD, turned, S, H, hd), "attention_dense")
    _check(fw, formulas(turned, None, True))
    bw = _run(K.attention_backward(S, S, H, G, hd, True), BWD, _kwargs(BWD, turned, S, H, hd, do, fw["output_ptr"], fw["lse_ptr"]), "attention_bwd")
    _check(bw, formulas(turned, do, True, fw["output_ptr"], fw["lse_ptr"]))
    turn(bw["query_grad_ptr"], bw["key_grad_ptr"], True)


@pytest.mark.gpu
@pytest.mark.parametrize("c", [(100, 200, 8, 4, 64, True), (400, 300, 8, 2, 128, False), (48, 1600, 8, 2, 64, True)])   # (gradients, outputs in parts)
def test_shards_add_up_to_the_whole(c, build_lib):
    kw, do = _inputs(*c[:5])
    o, lse = _forward_results(kw, c[5])
    for fn, make, full, kind in ((FWD, K.attention_forward, _kwargs(FWD, kw, c[0], 8, c[4]), "attention_dense"),
                                 (BWD, K.attention_backward, _kwargs(BWD, kw, c[0], 8, c[4], do, o, lse), "attention_bwd")):
        src = make(*c, 16, 64)
        whole = _run(src, fn, full, kind)
        gpu = KTIRInterpreter()
        gpu.load(src)
        for name in [n for n, x in full.items() if isinstance(x, np.ndarray) and np.isnan(x).all()]:
            got = np.zeros(whole[name].shape, whole[name].dtype)
            for r in range(2):
                part = gpu.execute_shard(fn, r, 2, **full)[name]
                per = part.shape[1] // 2
                got[:, r * per:(r + 1) * per] = part[:, r * per:(r + 1) * per]
            np.testing.assert_array_equal(got, whole[name], err_msg=name)
        gpu.close()


def _device_case(gpu, arrays):
    """Arrays behind one another in device memory: (arena, name -> byte offset)."""
    dev, at, offs = gpu.device, 0, {}
    for n, x in arrays.items():
        offs[n] = at
        at = (at + x.nbytes + 255) // 256 * 256
    arena = dev.alloc(at)
    for n, x in arrays.items():
        dev.h2d(arena + offs[n], x)
        dev.sync()
    return arena, offs


@pytest.mark.gpu
def test_heads_before_positions_and_rows_left_alone(build_lib):
    """Tensors laid out [heads][positions][head_dim] and with gaps between rows; dQ of some rows and heads only: the rest of the
    buffer stays as it was, in front of, between and behind."""
    gpu = KTIRInterpreter()
    dev = gpu.device
    S, T, H, G, hd = 150, 210, 4, 2, 64
    kw, do = _inputs(S, T, H, G, hd)
    o, lse = _forward_results(kw, True)
    wide = lambda x, n: np.concatenate([x, np.full(x.shape[:-1] + (n,), np.nan, x.dtype)], -1)     # noqa: E731
    arrays = dict(q=np.ascontiguousarray(kw["query_ptr"].transpose(1, 0, 2)), k=wide(kw["key_ptr"], 8), v=np.ascontiguousarray(kw["value_ptr"].transpose(1, 0, 2)),
                  o=wide(o, 24), do=do, lse=np.ascontiguousarray(lse.T), dq=np.full((S, H, hd + 8), 7, np.float16), dk=np.full((G, T, hd), 7, np.float16),
                  dv=np.full((T, G, hd), 7, np.float16))
    arena, offs = _device_case(gpu, arrays)
    a = R.AttnBwdArgs()
    a.arena = arena
    for n in arrays:
        setattr(a, n + "_off", offs[n] // (4 if n == "lse" else 2))
    for n, row, head in (("q", hd, S * hd), ("k", G * (hd + 8), hd + 8), ("v", hd, T * hd), ("o", H * (hd + 24), hd + 24), ("do", H * hd, hd), ("lse", 1, S),
                         ("dq", H * (hd + 8), hd + 8), ("dk", hd, T * hd), ("dv", G * hd, hd)):
        setattr(a, n + "_row", row)
        setattr(a, n + "_head", head)
    a.q_len, a.kv_len, a.heads, a.kv_group, a.head_dim, a.causal, a.causal_delta, a.scale, a.want = S, T, H, H // G, hd, 1, T - S, _scale(hd), 7
    a.dq_row0, a.dq_rows, a.dq_head0, a.dq_heads, a.dk_row0, a.dk_rows, a.dk_head0, a.dk_heads = 13, 130, 1, 2, 70, 140, 1, 1
    a.scratch_bytes = dev.lib.ktb_attention_bwd_scratch_bytes(C.byref(a))
    a.dev_scratch = dev.alloc(a.scratch_bytes)
    dev.check(dev.lib.ktb_launch_attention_bwd(dev.h, C.byref(a)))
    got = {n: np.empty_like(arrays[n]) for n in ("dq", "dk", "dv")}
    for n, x in got.items():
        dev.d2h(x, arena + offs[n])
    dev.sync()
    want = formulas(kw, do, True, o, lse)
    dq = got["dq"]
    for name, x, sel in (("query_grad_ptr", dq[..., :hd], (slice(13, 143), slice(1, 3))), ("key_grad_ptr", got["dk"].transpose(1, 0, 2), (slice(70, 210), slice(1, 2))),
                         ("value_grad_ptr", got["dv"], (slice(70, 210), slice(1, 2)))):
        _check({name: x[sel]}, {name: (want[name][0][sel], want[name][1][sel])})
        rest = np.ones(x.shape, bool)
        rest[sel] = False
        assert (x[rest] == 7).all()
    assert (dq[..., hd:] == 7).all()
    # the forward pass on the same layouts
    arrays2 = dict(q=arrays["q"], k=arrays["k"], v=arrays["v"], o=np.full((H, S, hd + 8), 7, np.float16), lse=np.full((H, S + 5), 7, np.float32))
    arena2, offs2 = _device_case(gpu, arrays2)
    b = R.AttnDenseArgs()
    b.arena = arena2
    for n in arrays2:
        setattr(b, n + "_off", offs2[n] // (4 if n == "lse" else 2))
    for n, row, head in (("q", hd, S * hd), ("k", G * (hd + 8), hd + 8), ("v", hd, T * hd), ("o", hd + 8, S * (hd + 8)), ("lse", 1, S + 5)):
        setattr(b, n + "_row", row)
        setattr(b, n + "_head", head)
    b.q_len, b.kv_len, b.heads, b.kv_group, b.head_dim, b.causal, b.causal_delta, b.scale = S, T, H, H // G, hd, 1, T - S, _scale(hd)
    dev.check(dev.lib.ktb_launch_attention_dense(dev.h, C.byref(b)))
    go, gl = np.empty_like(arrays2["o"]), np.empty_like(arrays2["lse"])
    dev.d2h(go, arena2 + offs2["o"])
    dev.d2h(gl, arena2 + offs2["lse"])
    dev.sync()
    _check(dict(output_ptr=go[..., :hd].transpose(1, 0, 2), lse_ptr=gl[:, :S].T), formulas(kw, None, True))
    assert (go[..., hd:] == 7).all() and (gl[:, S:] == 7).all()
    for p in (arena, arena2, a.dev_scratch):
        dev.free(p)
    gpu.close()


@pytest.mark.gpu
def test_launchers_refuse(build_lib):
    kw, do = _inputs(64, 64, 4, 2, 64)
    o, lse = _forward_results(kw, True)
    gpu = KTIRInterpreter()
    gpu.load(K.attention_backward(64, 64, 4, 2, 64, True))
    sess, _ = gpu.session(BWD, **_kwargs(BWD, kw, 64, 4, 64, do, o, lse))
    dev, (st,) = gpu.device, sess.plan.statements

    def refused(launch, args, field, value, code, word):
        a = type(args).from_buffer_copy(args)
        a.arena = sess.arena
        setattr(a, field, value)
        before = dev.launch_count()
        assert getattr(dev.lib, launch)(dev.h, C.byref(a)) == code, field
        assert word in dev.lib.ktb_last_error(dev.h).decode() and dev.launch_count() == before, field
    for field, value, code in (("head_dim", 32, -3), ("head_dim", 256, -3), ("kv_group", 0, -2), ("kv_group", 3, -2), ("heads", -4, -2), ("q_len", -1, -2),
                               ("q_len", 0, -3), ("kv_len", 0, -3), ("want", 0, -2), ("want", 8, -2), ("scale", float("nan"), -2), ("scale", float("inf"), -2),
                               ("dq_row0", -1, -2), ("dq_rows", 65, -2), ("dq_heads", 5, -2), ("dq_head0", 1, -2), ("dk_rows", 65, -2), ("dk_head0", 1, -2),
                               ("dk_row0", 64, -2), ("k_row", 12, -3), ("q_off", st.args.q_off + 4, -3), ("dv_head", 2, -3), ("dev_scratch", None, -2),
                               ("dev_scratch", st.args.dev_scratch + 16, -2), ("scratch_bytes", st.args.scratch_bytes - 1, -2),
                               ("key_parts", -1, -2), ("query_parts", 65, -2), ("key_parts", 2, -2), ("query_parts", 2, -2), ("twice", 2, -2), ("twice", -1, -2)):
        refused("ktb_launch_attention_bwd", st.args, field, value, code, "attention_bwd")
    assert dev.lib.ktb_attention_bwd_scratch_bytes(C.byref(st.args)) == st.args.scratch_bytes
    fwd = KTIRInterpreter()
    fwd.load(K.attention_forward(64, 64, 4, 2, 64, True))
    fs, _ = fwd.session(FWD, **_kwargs(FWD, kw, 64, 4, 64))
    for field, value, code in (("head_dim", 96, -3), ("kv_group", 0, -2), ("kv_group", 3, -2), ("q_len", -1, -2), ("kv_len", 0, -3), ("scale", 0.0, -3),
                               ("scale", -1.0, -3), ("scale", float("nan"), -3), ("v_row", 12, -3), ("o_off", 4, -3), ("parts", -1, -2), ("parts", 65, -2), ("twice", 2, -2), ("twice", -1, -2), ("single", 2, -2),
                               ("parts", 2, -2)):
        refused("ktb_launch_attention_dense", fs.plan.statements[0].args, field, value, code, "attention_dense")
    fwd.close()
    gpu.close()


@pytest.mark.gpu
@pytest.mark.parametrize("case", [(40, 40, 4, 2, 32, True), (50, 30, 2, 2, 96, True), (33, 70, 2, 1, 16, False)])
def test_other_head_sizes_run_step_by_step(case, build_lib):
    """Head sizes without a kernel give the oracle's results all the same."""
    q_len, kv_len, heads, kv_heads, hd, causal = case
    kw, do = _inputs(q_len, kv_len, heads, kv_heads, hd)
    o, lse = _forward_results(kw, causal)
    for fn, make, full in ((FWD, K.attention_forward, _kwargs(FWD, kw, q_len, heads, hd)), (BWD, K.attention_backward, _kwargs(BWD, kw, q_len, heads, hd, do, o, lse))):
        gpu = KTIRInterpreter(latency_config=HardwareConfig(lx_size_mb=8))
        gpu.load(make(q_len, kv_len, heads, kv_heads, hd, causal, min(q_len, 16), min(kv_len, 16)))
        got = gpu.execute_function(fn, **full)
        assert {s.kind for sess in gpu._sessions.values() for s in sess.plan.statements} == {"generic"}
        gpu.close()
        _check(got, formulas(kw, None, causal) if fn == FWD else formulas(kw, do, causal, o, lse))


# ---- ranges of the inputs ------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("scale", [-0.25, -0.5, 0.0, -0.0])
@pytest.mark.parametrize("c", [(150, 150, 2, 2, 128, True), (100, 197, 6, 2, 64, False), (70, 90, 3, 1, 128, False), (300, 111, 8, 4, 64, True), (9, 30, 2, 1, 64, True)])
def test_gradients_with_a_score_scale_of_zero_or_below(c, scale, build_lib):
    """A hidden key has no probability whatever sign the scale has.  (scale Q) K^T = |scale| Q (-K)^T, so that the formulas with -K
    give dQ, dV and -dK.)"""
    kw, do = _inputs(*c[:5], seed=c[1])
    mirrored = dict(kw, key_ptr=-kw["key_ptr"])
    o, lse = _forward_results(mirrored, c[5], scale=abs(scale))
    got = _run(K.attention_backward(*c), BWD, _kwargs(BWD, kw, c[0], c[2], c[4], do, o, lse, np.float32(scale)), "attention_bwd")
    got["key_grad_ptr"] = -got["key_grad_ptr"]
    _check(got, formulas(mirrored, do, c[5], o, lse, scale=abs(scale)))


@pytest.mark.parametrize("scale,low,fwd,bwd", [(1e15, "-1.0e30", 1, 1), (1e22, "-1.0e30", 0, 1), (1e10, "-1.0e20", 0, 1), (1e6, "-1.0e20", 1, 1),
                                               (3e27, "-1.0e30", 0, 0), (-3e27, "-1.0e30", 0, 0), (3e38, "-2.0e38", 0, 0)])
def test_scores_that_may_reach_the_initial_maximum_or_infinity_run_step_by_step(scale, low, fwd, bwd):
    """64 products of f16 are up to 2.7e11: times the scale, they stay above the initial maximum, or their row would not get its
    own, and times 1 / ln 2 they are finite."""
    kw, do = _inputs(64, 64, 4, 2, 64)
    lse = np.zeros((64, 4), np.float32)
    for fn, make, kind, fused in ((FWD, K.attention_forward, "attention_dense", fwd), (BWD, K.attention_backward, "attention_bwd", bwd)):
        src = make(64, 64, 4, 2, 64, True).replace("%low = arith.constant -1.0e30", f"%low = arith.constant {low}")
        assert set(_kinds(src, fn, _kwargs(fn, kw, 64, 4, 64, do, do, lse, np.float32(scale)))) == ({kind} if fused else {"generic"})


@pytest.mark.gpu
def test_launchers_refuse_scores_without_bounds(build_lib):
    kw, do = _inputs(64, 64, 4, 2, 64)
    for fn, make, launch, bad, good, code in ((FWD, K.attention_forward, "ktb_launch_attention_dense", (4e18, 3e38, float("inf")), 3e18, -3),
                                              (BWD, K.attention_backward, "ktb_launch_attention_bwd", (4e26, -4e26, 3e38, float("-inf")), -3e26, -2)):
        gpu = KTIRInterpreter()
        gpu.load(make(64, 64, 4, 2, 64, True))
        sess, _ = gpu.session(fn, **_kwargs(fn, kw, 64, 4, 64, do, do, np.zeros((64, 4), np.float32)))
        a = sess.plan.statements[0].args
        a.arena = sess.arena
        for scale in bad + (good,):
            a.scale = scale
            before = gpu.device.launch_count()
            rc = getattr(gpu.device.lib, launch)(gpu.device.h, C.byref(a))
            assert rc == (0 if scale == good else code) and (gpu.device.launch_count() == before) == (scale != good), scale
        gpu.device.sync()
        gpu.close()


def _close(got, want, what):
    """Rounding errors, in 2-norms: of P or dS and of the result, each 2^-11 of a value at most and less than two thirds of that on
    average, are together below 2^-10.5."""
    off = np.linalg.norm(got.astype(np.float64) - want) / np.linalg.norm(want)
    assert off <= 2 ** -10.5, (what, float(off))


LOUD = [(700, 700, 2, 2, 128, True), (700, 700, 8, 1, 64, True), (500, 700, 1, 1, 128, True), (600, 430, 12, 4, 64, True), (300, 2000, 2, 1, 128, True)]


@pytest.mark.gpu
@pytest.mark.parametrize("loud", [1e5, 1e6])
@pytest.mark.parametrize("c", LOUD)
def test_a_loud_query_costs_keys_that_it_does_not_see_nothing(c, loud, build_lib):
    q_len, kv_len, heads, _, hd, _ = c
    kw, do = _inputs(*c[:5], seed=q_len, grad=0.01)
    quiet = do.copy()
    at = max(20, q_len - kv_len + 20)
    do[at] = np.clip(do[at].astype(np.float32) * loud, -6e4, 6e4).astype(np.float16)
    o, lse = _forward_results(kw, True)
    got = _run(K.attention_backward(*c), BWD, _kwargs(BWD, kw, q_len, heads, hd, do, o, lse), "attention_bwd")
    quiet[at] = 0
    want = formulas(kw, quiet, True, o, lse)
    behind = at + kv_len - q_len + 1                             # the first key that the loud query does not see
    _close(got["key_grad_ptr"][behind:], want["key_grad_ptr"][0][behind:], "dK")
    _close(got["key_grad_ptr"][behind:behind + 20], want["key_grad_ptr"][0][behind:behind + 20], "dK right behind")
    _close(got["value_grad_ptr"][behind:], want["value_grad_ptr"][0][behind:], "dV")
    rest = np.arange(q_len) != at
    _close(got["query_grad_ptr"][rest], want["query_grad_ptr"][0][rest], "dQ")


@pytest.mark.gpu
@pytest.mark.parametrize("loud", [1e5, 1e6])
@pytest.mark.parametrize("c", LOUD)
def test_a_loud_value_costs_queries_that_do_not_see_it_nothing(c, loud, build_lib):
    q_len, kv_len, heads, _, hd, _ = c
    kw, do = _inputs(*c[:5], seed=q_len)
    kw["value_ptr"] = (kw["value_ptr"] * np.float16(0.01)).astype(np.float16)
    at = kv_len - 30
    kw["value_ptr"][at] = np.clip(kw["value_ptr"][at].astype(np.float32) * loud, -6e4, 6e4).astype(np.float16)
    o, lse = _forward_results(kw, True)
    got = _run(K.attention_backward(*c), BWD, _kwargs(BWD, kw, q_len, heads, hd, do, o, lse), "attention_bwd")
    want = formulas(kw, do, True, o, lse)
    before = q_len - 30                                          # the first query that sees the loud value
    _close(got["query_grad_ptr"][:before], want["query_grad_ptr"][0][:before], "dQ")
    _close(got["query_grad_ptr"][before - 20:before], want["query_grad_ptr"][0][before - 20:before], "dQ right before")
    _check(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("hidden", [True, False])
@pytest.mark.parametrize("c", [(16, 16, 2, 2, 64, True), (12, 40, 4, 2, 128, True), (20, 20, 3, 3, 64, False)])
def test_few_keys_of_very_different_values(c, hidden, build_lib):
    """A small difference of dO V^T and D is a gradient unless it is small next to that key's own value.  The large value is seen by
    the last query only, or has next to no probability: a score of -16 and less next to the others'."""
    kw, do = _inputs(*c[:5], seed=c[1])
    at = -1 if hidden else 0
    kw["value_ptr"][at] = np.clip(kw["value_ptr"][at].astype(np.float32) * 1e4, -6e4, 6e4).astype(np.float16)
    if not hidden:
        kw["query_ptr"][..., 0], kw["key_ptr"][..., 0], kw["key_ptr"][0] = 8, 2, 0
        kw["key_ptr"][0, :, 0] = 2 - 2 * math.sqrt(c[4])
    o, lse = _forward_results(kw, c[5])
    got = _run(K.attention_backward(*c), BWD, _kwargs(BWD, kw, c[0], c[2], c[4], do, o, lse), "attention_bwd")
    _check(got, formulas(kw, do, c[5], o, lse, half=HALF * HALF))


@pytest.mark.gpu
@pytest.mark.parametrize("c", [(200, 4000, 2, 2, 64, False), (600, 3000, 1, 1, 128, False), (30, 5000, 8, 1, 128, False), (3000, 3000, 1, 1, 64, True)])
def test_keys_far_below_the_largest_score_keep_their_precision(c, build_lib):
    """The first key has 13 more than the others, and a value of 0: what is left are probabilities of 2 * 10^-6, below the normal numbers of f16."""
    q_len, kv_len, heads, _, hd, causal = c
    kw, _ = _inputs(*c[:5], seed=hd)
    kw["query_ptr"][..., 0], kw["key_ptr"][..., 0], kw["value_ptr"][0] = 8, 0, 0
    kw["key_ptr"][0] = 0
    kw["key_ptr"][0, :, 0] = 13 / 8 * math.sqrt(hd)
    got = _run(K.attention_forward(*c), FWD, _kwargs(FWD, kw, q_len, heads, hd), "attention_dense")
    want = formulas(kw, None, causal)
    _check(got, want)
    far = 500 if causal else 0
    _close(got["output_ptr"][far:], want["output_ptr"][0][far:], "O")


@pytest.mark.gpu
@pytest.mark.parametrize("c", [(150, 150, 2, 2, 128, True), (300, 333, 2, 1, 64, False), (90, 90, 40, 40, 64, True), (3, 2000, 2, 2, 128, False)])
@pytest.mark.parametrize("what", [np.nan, np.inf, -np.inf])
def test_special_values_in_keys(c, what, build_lib):
    """A NaN score, or one of infinity, makes its row NaN; one of -infinity has no probability; a hidden one does nothing."""
    kw, _ = _inputs(*c[:5])
    n = c[1] - c[0] if c[5] else 0
    for j in range(8):
        x = {k: v.copy() for k, v in kw.items()}
        x["key_ptr"][c[1] // 2 + j, 0, 5] = what
        x["query_ptr"][:, 0, 5] = np.abs(x["query_ptr"][:, 0, 5])
        got = _run(K.attention_forward(*c), FWD, _kwargs(FWD, x, c[0], c[2], c[4]), "attention_dense")
        _check(got, formulas(x, None, c[5]))


@pytest.mark.gpu
@pytest.mark.parametrize("c", [(150, 150, 2, 2, 128, True), (1, 1, 2, 2, 64, False), (40, 2000, 2, 2, 128, True)])
def test_a_row_whose_scores_are_all_minus_infinity(c, build_lib):
    kw, _ = _inputs(*c[:5])
    first = c[1] - c[0]
    kw["key_ptr"][:first + 1, :, 3] = -np.inf
    kw["query_ptr"][..., 3] = 1
    got = _run(K.attention_forward(*c), FWD, _kwargs(FWD, kw, c[0], c[2], c[4]), "attention_dense")
    assert (got["output_ptr"][0] == 0).all() and (got["lse_ptr"][0] == -np.inf).all()
    _check(got, formulas(kw, None, c[5]))


@pytest.mark.parametrize("block", [16, 64])
@pytest.mark.parametrize("strides", ["[64, 64, 1]", "[8, 256, 1]", "[256, 8, 1]", "[64, 8, 1]", "[256, 56, 1]"])
def test_an_element_stored_twice_is_not_one_launch(strides, block):
    """Rows or heads of a tile's result over one another: the last one stays, which CTAs in no order do not promise."""
    kw, do = _inputs(64, 64, 4, 1, 64)
    rows = strides.split(",")[0] + ", 64, 1]"
    for fn, make, ptr, bit, old, new in ((FWD, K.attention_forward, "output", 0, "[256, 64, 1]", strides), (BWD, K.attention_backward, "query_grad", R.ATTN_DQ, "[256, 64, 1]", strides),
                                         (BWD, K.attention_backward, "key_grad", R.ATTN_DK, "[64, 64, 1]", rows), (BWD, K.attention_backward, "value_grad", R.ATTN_DV, "[64, 64, 1]", rows)):
        src = make(64, 64, 4, 1, 64, True, block, block)
        full = _kwargs(fn, kw, 64, 4, 64, do, do, np.zeros((64, 4), np.float32))
        i = src.index(f"construct_memory_view %{ptr}_ptr")
        assert "strides: " + old in src[i:]
        try:
            plan = _session(src[:i] + src[i:].replace("strides: " + old, "strides: " + new, 1), fn, full).plan.statements
        except NotImplementedError:
            continue
        if ptr in ("output", "query_grad") or new.startswith("[8,"):
            assert not any(s.kind == "attention_dense" or s.kind == "attention_bwd" and s.args.want & bit for s in plan), ptr


@pytest.mark.gpu
def test_launcher_refuses_more_steps_than_it_counts(build_lib):
    """Heads may lie over one another in what is read, so that few bytes are many steps."""
    gpu = KTIRInterpreter()
    kw, do = _inputs(64, 64, 4, 2, 64)
    gpu.load(K.attention_backward(64, 64, 4, 2, 64, True))
    sess, _ = gpu.session(BWD, **_kwargs(BWD, kw, 64, 4, 64, do, do, np.zeros((64, 4), np.float32)))
    a = sess.plan.statements[0].args
    a.arena, a.q_len, a.heads, a.kv_group, a.scratch_bytes = sess.arena, 1 << 20, 1 << 15, 1 << 15, 1 << 60
    before = gpu.device.launch_count()
    assert gpu.device.lib.ktb_launch_attention_bwd(gpu.device.h, C.byref(a)) == -3 and gpu.device.launch_count() == before
    assert b"steps" in gpu.device.lib.ktb_last_error(gpu.device.h)
    gpu.close()


# More items than SMs, so that a CTA takes one after the other: walks of keys, of queries, and empty ones (queries that see nothing) in
# every order; the last two with more than sixteen items an SM, which are handed out head by head.
MANY = [(300, 300, 60, 60, 128, True), (500, 500, 48, 48, 64, True), (700, 300, 40, 40, 128, True), (300, 700, 48, 12, 128, False), (257, 197, 64, 64, 64, False),
        (450, 130, 60, 30, 64, True), (130, 130, 620, 620, 64, True), (200, 150, 640, 640, 128, False)]


@pytest.mark.gpu
@pytest.mark.parametrize("c", MANY)
def test_ctas_that_take_many_items(c, build_lib):
    kw, do = _inputs(*c[:5], seed=c[1])
    items = -(-c[1] // 128) * c[3] + -(-c[0] // 128) * c[2]
    assert items > 148 and (c[2] < 600 or items > 16 * 148)
    assert grad_parts(*c[:4], int(c[5]), c[1] - c[0] if c[5] else 0) == (1, 1) and not few_rows(c[0], c[2], c[5], c[1] - c[0], FEW_ROWS_BACKWARD)
    o, lse = _forward_results(kw, c[5])
    got = _run(K.attention_backward(*c), BWD, _kwargs(BWD, kw, c[0], c[2], c[4], do, o, lse), "attention_bwd", times=3)
    _check(got, formulas(kw, do, c[5], o, lse))
    got = _run(K.attention_forward(*c), FWD, _kwargs(FWD, kw, c[0], c[2], c[4]), "attention_dense", times=3)
    _check(got, formulas(kw, None, c[5]))


@pytest.mark.gpu
@pytest.mark.parametrize("parts", [(2, 3), (5, 1)])
@pytest.mark.parametrize("c", [(300, 300, 40, 40, 128, True), (450, 430, 30, 10, 128, False), (500, 130, 40, 20, 64, True)])
def test_ctas_that_take_many_parts(c, parts, build_lib, monkeypatch):
    from ktir_cpu_b200 import lower_attn_train
    monkeypatch.setattr(lower_attn_train, "grad_parts", lambda *a: parts)
    kw, do = _inputs(*c[:5], seed=c[1])
    o, lse = _forward_results(kw, c[5])
    got = _run(K.attention_backward(*c), BWD, _kwargs(BWD, kw, c[0], c[2], c[4], do, o, lse), "attention_bwd", times=3)
    _check(got, formulas(kw, do, c[5], o, lse))
