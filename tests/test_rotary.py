"""Rotary positions: the KTIR text against the formula in 64 bits, which plans run as one launch and which do not, and (on
the GPU) the kernel against the oracle, bit for bit: products and sums are f32 operations of their own on both sides."""
import ctypes as C

import numpy as np
import pytest

from ktir_cpu_b200 import KTIRInterpreter, kernels as K, runtime as R
from ktir_cpu_b200.interpreter import Session
from ktir_cpu_b200.parser import KTIRParser
from oracle.numpy_interp import OracleInterpreter

# (tokens, heads, key heads, head size, turned part, layout, backwards, type, tokens per core): one token; a part whose
# halves start off every boundary; odd counts; one pair; several tokens per core; heads that fill no vector of heads
CASES = [(1, 32, 8, 128, 128, "half", False, "f16", None), (1, 4, 1, 64, 64, "interleaved", True, "f16", None),
         (7, 5, 3, 80, 26, "half", False, "f16", None), (7, 5, 3, 80, 26, "interleaved", False, "f16", None),
         (12, 6, 2, 96, 48, "half", True, "f32", 4), (12, 3, 3, 96, 50, "interleaved", True, "f32", 3),
         (33, 9, 1, 256, 110, "half", False, "f16", 11), (5, 2, 0, 16, 2, "half", False, "f16", 1),
         (64, 8, 2, 128, 64, "interleaved", False, "f16", 16), (3, 1, 1, 30, 30, "half", True, "f32", 1)]


def _case(tokens, heads, kv_heads, dim, part, layout, inverse, dtype, block, rows=300, seed=0):
    rng = np.random.default_rng(seed)
    dt = np.dtype({"f16": np.float16, "f32": np.float32}[dtype])
    cos, sin = K.rotary_tables(rows, part)
    kw = dict(query_out_ptr=np.zeros((tokens, heads, dim), dt))
    if kv_heads:
        kw["key_out_ptr"] = np.zeros((tokens, kv_heads, dim), dt)
    kw["query_ptr"] = rng.standard_normal((tokens, heads, dim)).astype(dt)
    if kv_heads:
        kw["key_ptr"] = rng.standard_normal((tokens, kv_heads, dim)).astype(dt)
    kw.update(positions_ptr=rng.integers(0, rows, tokens).astype(np.int32), cos_ptr=cos, sin_ptr=sin)
    return K.rotary(tokens, heads, kv_heads, dim, part, rows, layout, inverse, dtype, block), kw


def _formula(x, kw, part, layout, inverse):
    n = part // 2
    turn = kw["cos_ptr"].astype(np.float64) + 1j * kw["sin_ptr"].astype(np.float64) * (-1 if inverse else 1)
    turn = turn[kw["positions_ptr"]][:, None, :]
    j = np.arange(n)
    a, b = (j, j + n) if layout == "half" else (2 * j, 2 * j + 1)
    y = x.astype(np.float64)
    z = (y[..., a] + 1j * y[..., b]) * turn
    y[..., a], y[..., b] = z.real, z.imag
    return y


def _oracle(src, kw):
    ora = OracleInterpreter()
    ora.load(src)
    return ora.execute_function("rotary_kernel", **kw)


def _session(src, kw):
    t = [(k, v.shape, v.dtype) for k, v in kw.items()]
    return Session(R.PlanOnlyDevice(), KTIRParser().parse_module(src).get_function("rotary_kernel"), t, {}, arena_ptr=0)


@pytest.mark.parametrize("case", CASES)
def test_text_turns_pairs_by_the_angle_of_the_position(case):
    src, kw = _case(*case)
    got = _oracle(src, kw)
    for name in ("query", "key") if case[2] else ("query",):
        want = _formula(kw[name + "_ptr"], kw, case[4], case[5], case[6])
        # |x cos|, |y sin| <= 6: two products and a sum, half a step of f32 each, and the rounding of the result
        step = 2.0 ** -11 if case[7] == "f16" else 2.0 ** -24
        np.testing.assert_allclose(got[name + "_out_ptr"].astype(np.float64), want, rtol=step, atol=3 * 12 * 2.0 ** -24)


@pytest.mark.parametrize("case", CASES)
def test_turning_back_gives_the_inputs(case):
    """Forward, then backwards: the gradient of the rotation is its inverse (tables of unit length up to f32)."""
    if case[7] == "f16":
        case = case[:7] + ("f32",) + case[8:]
    src, kw = _case(*case)
    got = _oracle(src, kw)
    back = K.rotary(*case[:5], 300, case[5], not case[6], case[7], case[8])
    again = _oracle(back, {**kw, "query_ptr": got["query_out_ptr"], **({"key_ptr": got["key_out_ptr"]} if case[2] else {})})
    np.testing.assert_allclose(again["query_out_ptr"], kw["query_ptr"], rtol=0, atol=12 * 8 * 2.0 ** -24)


@pytest.mark.parametrize("case", [c for c in CASES if c[4] > 2])
def test_plans_as_one_launch(case):
    src, kw = _case(*case)
    sess = _session(src, kw)
    st, = sess.plan.statements
    assert st.kind == "rotary" and st.args.n_tensors == (2 if case[2] else 1) and bool(st.args.inverse) == case[6]
    assert (st.args.n_items, st.args.tokens) == (1, case[0]) and st.args.pairs == case[4] // 2
    assert sess.plan.fully_overwritten == {k for k in kw if "_out" in k}


@pytest.mark.parametrize("change", [("arith.subf %query_ac", "arith.addf %query_ac"), ("%query_a, %query_sin", "%query_b, %query_sin"),
                                    ("%query_b, %query_cos", "%query_b, %query_sin"), ("arith.mulf %query_a, %query_cos", "arith.addf %query_a, %query_cos")])
def test_other_sums_are_not_taken_for_a_turn(change):
    src, kw = _case(4, 2, 0, 16, 16, "half", False, "f16", 2)
    assert change[0] in src
    sess = _session(src.replace(*change), kw)
    assert "rotary" not in [s.kind for s in sess.plan.statements]


def test_in_place_runs_step_by_step():
    src, kw = _case(4, 2, 0, 16, 16, "half", False, "f16", 2)
    src = src.replace("construct_memory_view %query_out_ptr", "construct_memory_view %query_ptr")
    try:
        kinds = [s.kind for s in _session(src, kw).plan.statements]
    except NotImplementedError:
        kinds = []
    assert "rotary" not in kinds


def test_tables_are_those_of_64_bits():
    cos, sin = K.rotary_tables(1 << 20, 4, base=10000.0, stretch=2.0)
    p = (1 << 20) - 1
    assert cos.dtype == np.float32 and cos.shape == (1 << 20, 2)
    want = np.array([p / 2.0, p / 2.0 * 10000.0 ** -0.5])
    np.testing.assert_array_equal(cos[p], np.cos(want).astype(np.float32))
    np.testing.assert_array_equal(sin[p], np.sin(want).astype(np.float32))
    slow = K.rotary_tables(64, 8, stretch=4.0, rescale_base=True)
    first = K.rotary_tables(64, 8)
    np.testing.assert_array_equal(slow[0][:, 0], first[0][:, 0])                 # the fastest pair as before
    np.testing.assert_allclose(slow[1][:, 3], np.sin(np.arange(64) / 4.0 * 10000.0 ** -0.75), rtol=0, atol=2.0 ** -24)


@pytest.mark.parametrize("tokens,heads,kv_heads,dim,part,layout", [
    (944, 8, 0, 104, 4, "half"), (266, 9, 2, 256, 8, "half"), (816, 10, 0, 64, 4, "half"), (442, 11, 1, 256, 8, "interleaved"), (4096, 64, 8, 256, 6, "half")])
def test_small_parts_of_long_heads_fit_the_scratchpad(tokens, heads, kv_heads, dim, part, layout):
    """A core's tokens are as many as fit with what is behind the pairs, too."""
    src, kw = _case(tokens, heads, kv_heads, dim, part, layout, False, "f32", None)
    assert [s.kind for s in _session(src, kw).plan.statements] == ["rotary"]


@pytest.mark.gpu
@pytest.mark.parametrize("case", CASES)
def test_kernel_has_the_oracles_bits(case, build_lib):
    src, kw = _case(*case)
    gpu = KTIRInterpreter()
    gpu.load(src)
    got = gpu.execute_function("rotary_kernel", **kw)
    again = gpu.execute_function("rotary_kernel", **kw)
    kinds = [s.kind for sess in gpu._sessions.values() for s in sess.plan.statements]
    gpu.close()
    assert case[4] == 2 or kinds == ["rotary"]
    want = _oracle(src, kw)
    for k in want:
        np.testing.assert_array_equal(got[k], want[k], err_msg=k)
        np.testing.assert_array_equal(again[k], want[k], err_msg=k)


@pytest.mark.gpu
def test_every_vector_length(build_lib):
    """Lengths whose halves start at 2, 4, 8 and 16 bytes, rests likewise."""
    for dtype in ("f16", "f32"):
        for layout in ("half", "interleaved"):
            for dim, part in ((64, 32), (64, 24), (64, 20), (62, 22), (61, 18), (64, 62), (72, 50), (16, 14), (16, 6), (8, 6)):
                case = (9, 13, 2, dim, part, layout, False, dtype, 3)
                src, kw = _case(*case)
                gpu = KTIRInterpreter()
                gpu.load(src)
                got = gpu.execute_function("rotary_kernel", **kw)
                assert [s.kind for sess in gpu._sessions.values() for s in sess.plan.statements] == ["rotary"]
                gpu.close()
                want = _oracle(src, kw)
                for k in want:
                    np.testing.assert_array_equal(got[k], want[k], err_msg=f"{k} {case}")


@pytest.mark.gpu
def test_special_values_and_positions(build_lib):
    """Infinities and NaN stay in their pair; a position past the tables reads zeros; a negative one is reported."""
    src, kw = _case(8, 4, 2, 64, 48, "half", False, "f16", 4)
    kw["query_ptr"][0, 0, 3] = np.inf
    kw["query_ptr"][1, 2, 47] = np.nan
    kw["query_ptr"][2, 1, :] = 65504
    kw["query_ptr"][3, 1, 60] = np.nan
    kw["positions_ptr"][5] = 300
    kw["positions_ptr"][6] = 2 ** 31 - 1
    gpu = KTIRInterpreter()
    gpu.load(src)
    with np.errstate(all="ignore"):
        want = _oracle(src, kw)
    got = gpu.execute_function("rotary_kernel", **kw)
    for k in want:
        np.testing.assert_array_equal(got[k], want[k], err_msg=k)
    kw["positions_ptr"][4] = -3
    with pytest.raises(IndexError, match="-3 is negative"):
        gpu.execute_function("rotary_kernel", **kw)
    kw["positions_ptr"][4] = 0
    gpu.execute_function("rotary_kernel", **kw)
    gpu.close()


@pytest.mark.gpu
def test_cores_in_any_order_and_parts_of_the_grid(build_lib):
    """Tokens that the cores take from the back: no single run of tokens; a rank's cores only."""
    case = (24, 4, 2, 64, 64, "half", False, "f16", 4)
    src, kw = _case(*case)
    back = src.replace("    %t0 = arith.muli %pid, %c_bt : index\n",
                       "    %c_last = arith.constant 5 : index\n    %rev = arith.subi %c_last, %pid : index\n"
                       "    %t0 = arith.muli %rev, %c_bt : index\n")
    want = _oracle(src, kw)
    gpu = KTIRInterpreter()
    gpu.load(back)
    got = gpu.execute_function("rotary_kernel", **kw)
    st, = [s for sess in gpu._sessions.values() for s in sess.plan.statements]
    assert st.kind == "rotary" and st.args.n_items == 6
    parts = [gpu.execute_shard("rotary_kernel", r, 3, **kw) for r in range(3)]
    gpu.close()
    for k in want:
        np.testing.assert_array_equal(got[k], want[k], err_msg=k)
        if "_out" in k:
            np.testing.assert_array_equal(sum(p[k].astype(np.float32) for p in parts), want[k].astype(np.float32))


@pytest.mark.gpu
def test_launcher_refuses(build_lib):
    src, kw = _case(8, 4, 2, 64, 48, "half", False, "f16", 4)
    gpu = KTIRInterpreter()
    gpu.load(src)
    sess, _ = gpu.session("rotary_kernel", **kw)
    st, = sess.plan.statements
    dev = gpu.device
    for field, value, code in (("n_tensors", 0, -2), ("n_tensors", 5, -2), ("dtype", 2, -3), ("idx_dtype", 1, -3), ("pairs", 0, -2),
                               ("pair_stride", 0, -2), ("tokens", -1, -2), ("align", 3, -2), ("align", 0, -2), ("table_stride", -1, -2),
                               ("dev_item_offsets", None, -2)):
        a = R.RotaryArgs.from_buffer_copy(st.args)
        a.arena = sess.arena
        setattr(a, field, value)
        before = dev.launch_count()
        assert dev.lib.ktb_launch_rotary(dev.h, C.byref(a)) == code, field
        assert b"rotary" in dev.lib.ktb_last_error(dev.h) and dev.launch_count() == before
    for field, value in (("heads", -1), ("rest", -1), ("in_partner", 0), ("out_partner", -24)):
        a = R.RotaryArgs.from_buffer_copy(st.args)
        a.arena = sess.arena
        setattr(a.t[1], field, value)
        assert dev.lib.ktb_launch_rotary(dev.h, C.byref(a)) == -2, field
    a = R.RotaryArgs.from_buffer_copy(st.args)
    a.arena, a.n_items = sess.arena, 0
    assert dev.lib.ktb_launch_rotary(dev.h, C.byref(a)) == 0
    gpu.close()


@pytest.mark.gpu
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("case", [(33, 9, 2, 64, 64, "half", False, "f16", 11), (33, 9, 2, 64, 64, "interleaved", False, "f16", 11), (16, 4, 4, 96, 48, "half", True, "f32", 4),
                                  (21, 5, 1, 72, 50, "half", False, "f16", 3)])
def test_arena_on_any_boundary_of_its_types(case, wide, build_lib):
    """All tensors moved by 4, 8, ... bytes: vectors are as long as the addresses allow, those of the tables too."""
    src, kw = _case(*case)
    if wide:                                        # positions of 64 bits
        src = src.replace(f"memref<{case[0]}xi32>", f"memref<{case[0]}xi64>")
        kw["positions_ptr"] = kw["positions_ptr"].astype(np.int64)
    want = _oracle(src, kw)
    gpu = KTIRInterpreter()
    gpu.load(src)
    sess, _ = gpu.session("rotary_kernel", **kw)
    st, = sess.plan.statements
    assert st.kind == "rotary" and st.args.idx_dtype == R.DTYPE_CODE["i64" if wide else "i32"]
    dev = gpu.device
    offs = {n: sess.device_ptr(n) - sess.arena for n in kw}
    room = dev.alloc(max(o + kw[n].nbytes for n, o in offs.items()) + 64)
    for shift in (4, 8, 12, 16, 24, 2, 1):
        a = R.RotaryArgs.from_buffer_copy(st.args)
        a.arena = room + shift
        refused = shift % (8 if wide else 4) != 0
        if not refused:
            for n, x in kw.items():
                dev.h2d(room + shift + offs[n], x)
            dev.sync()
        assert dev.lib.ktb_launch_rotary(dev.h, C.byref(a)) == (-2 if refused else 0), shift
        if refused:
            assert b"arena" in dev.lib.ktb_last_error(dev.h)
            continue
        for n, x in want.items():
            got = np.empty_like(x)
            dev.d2h(got, room + shift + offs[n])
            dev.sync()
            np.testing.assert_array_equal(got, x, err_msg=f"{n} {shift}")
    dev.free(room)
    gpu.close()


@pytest.mark.parametrize("tokens,block", [(8, 2), (2, 2)])
@pytest.mark.parametrize("strides", ["[64, 0, 1]", "[0, 16, 1]", "[64, 8, 1]", "[16, 16, 1]"])
def test_an_element_stored_twice_is_not_one_launch(strides, tokens, block):
    """Heads or tokens over one another: the last one stays, which threads in no order do not promise."""
    src, kw = _case(tokens, 4, 0, 16, 16, "half", False, "f16", block)
    i = src.index("construct_memory_view %query_out_ptr")
    assert "strides: [64, 16, 1]" in src[i:]
    assert [s.kind for s in _session(src, kw).plan.statements] == ["rotary"]
    src = src[:i] + src[i:].replace("strides: [64, 16, 1]", "strides: " + strides, 1)
    assert "rotary" not in [s.kind for s in _session(src, kw).plan.statements]


@pytest.mark.parametrize("most,items", [(2 ** 31 - 1, 1), (12, 1), (11, 3), (1, 3)])
def test_tokens_that_an_item_cannot_count_stay_items(most, items, monkeypatch):
    from ktir_cpu_b200 import lower_rotary
    monkeypatch.setattr(lower_rotary, "MOST_TOKENS", most)
    st, = _session(*_case(12, 2, 0, 16, 16, "half", False, "f16", 4)).plan.statements
    assert st.kind == "rotary" and (st.args.n_items, st.args.tokens) == (items, 12 // items)


# (tokens, heads, key heads, head size, turned part, layout, backwards, type, tokens per core, cores in reverse): where four heads go to
# a thread (148 x 4096 of its vectors and more; half as many for rows of 16 bytes), head counts that are no multiple of four, heads of one
# thread in both tensors, rests, several items
LARGE = [(27000, 9, 1, 128, 128, "half", False, "f16", None, False), (27000, 9, 1, 128, 128, "interleaved", True, "f16", None, False),
         (9000, 13, 2, 128, 64, "half", False, "f32", 36, True), (16000, 10, 3, 96, 48, "interleaved", True, "f32", None, False),
         (40000, 5, 2, 96, 64, "half", True, "f16", 100, True), (60000, 3, 2, 64, 32, "interleaved", False, "f16", None, False),
         (16384, 9, 1, 128, 54, "half", False, "f16", None, False), (16384, 9, 1, 128, 54, "interleaved", True, "f16", 64, True),
         (9000, 13, 2, 96, 50, "half", True, "f32", 45, True), (9000, 6, 5, 96, 26, "interleaved", False, "f32", None, False),
         (30000, 2, 1, 62, 22, "half", False, "f16", None, False), (8000, 6, 1, 61, 18, "interleaved", True, "f16", None, False)]


def _restated(x, kw, part, layout, inverse):
    """In f32, products and sums rounded one by one."""
    n = part // 2
    cos, sin = kw["cos_ptr"][kw["positions_ptr"]][:, None], kw["sin_ptr"][kw["positions_ptr"]][:, None]
    j = np.arange(n)
    a, b = (j, j + n) if layout == "half" else (2 * j, 2 * j + 1)
    y, u, v = x.copy(), x[..., a].astype(np.float32), x[..., b].astype(np.float32)
    sin = -sin if inverse else sin
    y[..., a], y[..., b] = u * cos - v * sin, v * cos + u * sin
    return y


@pytest.mark.gpu
@pytest.mark.parametrize("case", LARGE)
def test_four_heads_to_a_thread(case, build_lib):
    src, kw = _case(*case[:9])
    if case[9]:
        cores = case[0] // case[8]
        src = src.replace("    %t0 = arith.muli %pid, %c_bt : index\n", f"    %c_last = arith.constant {cores - 1} : index\n    %rev = arith.subi %c_last, %pid : index\n"
                                                                         f"    %t0 = arith.muli %rev, %c_bt : index\n")
    gpu = KTIRInterpreter()
    gpu.load(src)
    got = gpu.execute_function("rotary_kernel", **kw)
    st, = [s for sess in gpu._sessions.values() for s in sess.plan.statements]
    assert st.kind == "rotary" and st.args.n_items == (case[0] // case[8] if case[9] else 1)
    gpu.close()
    for name in ("query", "key"):
        np.testing.assert_array_equal(got[name + "_out_ptr"], _restated(kw[name + "_ptr"], kw, *case[4:7]), err_msg=name)


@pytest.mark.parametrize("case", CASES)
def test_restatement_has_the_oracles_bits(case):
    src, kw = _case(*case)
    want = _oracle(src, kw)
    for name in ("query", "key") if case[2] else ("query",):
        np.testing.assert_array_equal(want[name + "_out_ptr"], _restated(kw[name + "_ptr"], kw, *case[4:7]))
