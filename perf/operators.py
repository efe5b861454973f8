"""The measured operators of attention layers in training and serving: rotary positions, attention that keeps the
log-sum-exp of its rows, and its gradient.

A program of this framework plans a KTIR function once with ``session`` and runs it with ``Session.run`` on tensors that
stay in device memory; that is the form measured where ``own`` is true.  Where it is false the same operators are
computed in elementary torch operations, in 32 bits, rounded once at the end.

Queries, keys and values are ``[positions, heads, head_dim]``; a batch folds into the heads.  ``heads / kv_heads`` query
heads share a key head.  Under the causal mask query i of n sees the keys up to i + (keys - n), so with fewer keys than
queries the first rows see nothing: their output is 0, their log-sum-exp -inf, and no gradient flows through them.
"""
import math

import numpy as np
import torch

own = False

NP = {"f16": np.float16, "f32": np.float32}
TORCH = {"f16": torch.float16, "f32": torch.float32}
KINDS = {"rotary": "rotary_kernel", "forward": "attention_forward_kernel", "backward": "attention_backward_kernel"}


def listed():
    return [
        # one new token of one sequence: rotated queries and keys, where latency counts
        dict(name="rotary_token", kind="rotary", tokens=1, heads=32, kv_heads=8, dim=128, part=128, layout="half",
             table=4096, base=10000.0, stretch=1.0, inverse=False, dtype="f16"),
        # a decode batch: every sequence at a position of its own in a long stretched context
        dict(name="rotary_batch_interleaved", kind="rotary", tokens=64, heads=64, kv_heads=8, dim=128, part=128,
             layout="interleaved", table=131072, base=500000.0, stretch=8.0, inverse=False, dtype="f16"),
        # prefill of packed sequences
        dict(name="rotary_prefill", kind="rotary", tokens=8192, heads=64, kv_heads=8, dim=128, part=128, layout="half",
             table=8192, base=500000.0, stretch=1.0, inverse=False, dtype="f16"),
        # the gradient in a model that rotates half of a head, in f32, an odd number of tokens
        dict(name="rotary_gradient_part_f32", kind="rotary", tokens=4001, heads=20, kv_heads=20, dim=96, part=48,
             layout="interleaved", table=8192, base=10000.0, stretch=1.0, inverse=True, dtype="f32"),
        # a small encoder: odd length, nothing masked, small heads
        dict(name="forward_197", kind="forward", queries=197, keys=197, heads=12, kv_heads=12, dim=64, causal=False),
        # training batch of 8 with 32 heads
        dict(name="forward_2048", kind="forward", queries=2048, keys=2048, heads=256, kv_heads=256, dim=128, causal=True),
        # a chunk of 1531 positions after an earlier context, grouped heads
        dict(name="forward_chunk", kind="forward", queries=1531, keys=4603, heads=32, kv_heads=8, dim=128, causal=True),
        # the gradients of the same layers
        dict(name="backward_197", kind="backward", queries=197, keys=197, heads=12, kv_heads=12, dim=64, causal=False),
        dict(name="backward_2048", kind="backward", queries=2048, keys=2048, heads=256, kv_heads=256, dim=128, causal=True),
        # long sequence, few key heads: little to spread over the machine but the sequence
        dict(name="backward_8192_grouped", kind="backward", queries=8192, keys=8192, heads=16, kv_heads=4, dim=128, causal=True),
        # cross attention: lengths that differ and fill no tile
        dict(name="backward_cross", kind="backward", queries=1000, keys=2777, heads=32, kv_heads=8, dim=64, causal=False),
        # more queries than keys: the first 233 rows see nothing
        dict(name="backward_empty_rows", kind="backward", queries=777, keys=544, heads=48, kv_heads=48, dim=128, causal=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rotary", "rotary", "forward", "forward", "backward", "backward", "backward"])
    group, kv = rng.choice([1, 1, 2, 4, 5, 8]), rng.choice([1, 2, 4, 8, 12, 16])
    if kind == "rotary":
        dim = rng.choice([64, 80, 96, 128, 128, 192, 256])
        part = dim if rng.random() < 0.5 else 2 * rng.randint(4, dim // 2)
        dtype = rng.choice(["f16", "f16", "f32"])
        tokens = _log(rng, 1, max(1, min(16384, (8192 * 72 * 128) // (group * kv * dim + kv * dim))))
        return dict(kind=kind, tokens=tokens, heads=group * kv, kv_heads=kv, dim=dim, part=part,
                    layout=rng.choice(["half", "interleaved"]), table=max(tokens, _log(rng, 512, 131072)),
                    base=rng.choice([10000.0, 500000.0]), stretch=rng.choice([1.0, 4.0]), inverse=rng.random() < 0.4,
                    dtype=dtype)
    batch = rng.choice([1, 2, 4])
    heads, kv, dim = batch * group * kv, batch * kv, rng.choice([64, 128, 128])
    most = (2048 * 2048 * 256 * 128) // (heads * dim)
    queries = _log(rng, 1, 8192)
    keys = queries if rng.random() < 0.6 else _log(rng, 1, 8192)
    if queries * keys > most:
        shrink = math.sqrt(most / (queries * keys))
        queries, keys = max(1, int(queries * shrink)), max(1, int(keys * shrink))
    return dict(kind=kind, queries=queries, keys=keys, heads=heads, kv_heads=kv, dim=dim, causal=rng.random() < 0.7)


# ---- tensors of a case, in the order of the function's arguments: name -> (shape, type) --------------------------
def _tensors(c):
    if c["kind"] == "rotary":
        q, k = (c["tokens"], c["heads"], c["dim"]), (c["tokens"], c["kv_heads"], c["dim"])
        t = (c["table"], c["part"] // 2)
        return dict(query_out_ptr=(q, c["dtype"]), key_out_ptr=(k, c["dtype"]), query_ptr=(q, c["dtype"]),
                    key_ptr=(k, c["dtype"]), positions_ptr=((c["tokens"],), "i32"), cos_ptr=(t, "f32"), sin_ptr=(t, "f32"))
    q, k = (c["queries"], c["heads"], c["dim"]), (c["keys"], c["kv_heads"], c["dim"])
    rows = (c["queries"], c["heads"])
    if c["kind"] == "forward":
        return dict(output_ptr=(q, "f16"), lse_ptr=(rows, "f32"), query_ptr=(q, "f16"), key_ptr=(k, "f16"), value_ptr=(k, "f16"))
    return dict(query_grad_ptr=(q, "f16"), key_grad_ptr=(k, "f16"), value_grad_ptr=(k, "f16"), query_ptr=(q, "f16"),
                key_ptr=(k, "f16"), value_ptr=(k, "f16"), output_ptr=(q, "f16"), lse_ptr=(rows, "f32"),
                output_grad_ptr=(q, "f16"))


def _outputs(c):
    return {"rotary": ["query_out_ptr", "key_out_ptr"], "forward": ["output_ptr", "lse_ptr"],
            "backward": ["query_grad_ptr", "key_grad_ptr", "value_grad_ptr"]}[c["kind"]]


def _scale(c):
    return float(np.float32(1.0 / math.sqrt(c["dim"])))


def _inputs(c, seed):
    """name -> device tensor for everything that the call reads, from the seed alone."""
    gen = torch.Generator("cuda").manual_seed(seed)

    def normal(shape, dtype, scale=1.0):
        return (torch.randn(shape, generator=gen, device="cuda") * scale).to(TORCH[dtype])

    t = _tensors(c)
    if c["kind"] == "rotary":
        # packed sequences: runs of positions that start over; a decode batch has one position per sequence
        if c["tokens"] <= 256:
            pos = torch.randint(0, c["table"], (c["tokens"],), generator=gen, device="cuda")
        else:
            pos = (torch.arange(c["tokens"], device="cuda") + torch.randint(0, c["table"], (1,), generator=gen, device="cuda")) % c["table"]
        angle = torch.arange(c["table"], dtype=torch.float64, device="cuda")[:, None] / c["stretch"] * \
            c["base"] ** (-torch.arange(0, c["part"], 2, dtype=torch.float64, device="cuda") / c["part"])
        return dict(query_ptr=normal(*t["query_ptr"]), key_ptr=normal(*t["key_ptr"]), positions_ptr=pos.int(),
                    cos_ptr=angle.cos().float(), sin_ptr=angle.sin().float())
    data = {k: normal(*t[k]) for k in ("query_ptr", "key_ptr", "value_ptr")}
    if c["kind"] == "backward":      # what the forward pass left, and the gradient that arrives
        o, lse = _forward(c, data)
        data.update(output_ptr=o, lse_ptr=lse, output_grad_ptr=normal(*t["output_grad_ptr"], 0.05))
    return data


class _DeviceTensor:
    """Lets torch see a session's tensor, which lies in the backend's own device memory.  Holds the interpreter: it
    frees its sessions' memory when it goes, and an output may outlive the state that it came from."""

    def __init__(self, interp, session, name, shape, dtype):
        self.interp = interp
        self.__cuda_array_interface__ = dict(shape=shape, typestr=dtype.str, data=(session.device_ptr(name), False), version=3)


def _session(c, data):
    """The planned function, its tensors filled with the inputs."""
    from ktir_cpu_b200 import KTIRInterpreter, kernels
    if c["kind"] == "rotary":
        source, scalars = kernels.rotary(c["tokens"], c["heads"], c["kv_heads"], c["dim"], c["part"], c["table"], c["layout"],
                                         inverse=c["inverse"], dtype=c["dtype"]), {}
    else:
        make = kernels.attention_forward if c["kind"] == "forward" else kernels.attention_backward
        source = make(c["queries"], c["keys"], c["heads"], c["kv_heads"], c["dim"], causal=c["causal"])
        scalars = dict(scale=np.float32(_scale(c)))
    interp = KTIRInterpreter()
    interp.load(source)
    types = {"i32": np.int32, **NP}
    tensors = {k: (s, np.dtype(types[d])) for k, (s, d) in _tensors(c).items()}
    shapes = {k: np.empty(*v) for k, v in tensors.items()}           # never touched: a session is planned from shapes
    session, _ = interp.session(KINDS[c["kind"]], **shapes, **scalars)
    views = {k: torch.as_tensor(_DeviceTensor(interp, session, k, *v), device="cuda") for k, v in tensors.items()}
    for k, v in views.items():
        if k in data:
            v.copy_(data[k])
    torch.cuda.synchronize()
    return dict(interp=interp, session=session, outputs={k: views[k] for k in _outputs(c)})


def prepare(case, seed):
    data = _inputs(case, seed)
    return _session(case, data) if own else dict(case=case, data=data)


def run(state):
    if own:
        state["session"].run()
        return state["outputs"]
    case, data = state["case"], state["data"]
    if case["kind"] == "rotary":
        return _rotary(case, data)
    return dict(zip(_outputs(case), (_forward if case["kind"] == "forward" else _backward)(case, data)))


# ---- plain forms --------------------------------------------------------------------------------------------------
def _turn(c, x, cos, sin):
    """x [tokens, heads, dim] with its first ``part`` elements per head turned, the rest as it is."""
    n, y = c["part"] // 2, x.float()
    half = c["layout"] == "half"
    a, b = (y[..., :n], y[..., n:2 * n]) if half else (y[..., 0:2 * n:2], y[..., 1:2 * n:2])
    sin = -sin if c["inverse"] else sin
    turned = (a * cos - b * sin, b * cos + a * sin)
    turned = torch.cat(turned, -1) if half else torch.stack(turned, -1).flatten(-2)
    return torch.cat((turned, y[..., 2 * n:]), -1).to(x.dtype)


def _rotary(c, d):
    pos = d["positions_ptr"].long()
    cos, sin = d["cos_ptr"][pos][:, None], d["sin_ptr"][pos][:, None]
    return dict(query_out_ptr=_turn(c, d["query_ptr"], cos, sin), key_out_ptr=_turn(c, d["key_ptr"], cos, sin))


def _heads_first(x, copies=1):
    return x.float().permute(1, 0, 2).repeat_interleave(copies, 0)


def _hidden(c, device="cuda"):
    """[queries, keys]: which keys a query does not see."""
    i, j = torch.arange(c["queries"], device=device), torch.arange(c["keys"], device=device)
    return j > i[:, None] + (c["keys"] - c["queries"]) if c["causal"] else torch.zeros((1, 1), dtype=torch.bool, device=device)


def _scores(c, d):
    """[heads, queries, keys] scaled scores, -inf where hidden."""
    group = c["heads"] // c["kv_heads"]
    s = _heads_first(d["query_ptr"]) @ _heads_first(d["key_ptr"], group).transpose(1, 2) * _scale(c)
    return s.masked_fill(_hidden(c), -math.inf)


def _forward(c, d):
    s = _scores(c, d)
    m = s.amax(-1, keepdim=True).clamp(min=-1e30)
    p = torch.exp(s - m)
    total = p.sum(-1, keepdim=True)
    o = p @ _heads_first(d["value_ptr"], c["heads"] // c["kv_heads"]) / total.clamp(min=1e-30)
    return o.permute(1, 0, 2).to(torch.float16).contiguous(), (m + total.log())[..., 0].T.contiguous()


def _backward(c, d):
    group = c["heads"] // c["kv_heads"]
    q, k, v = _heads_first(d["query_ptr"]), _heads_first(d["key_ptr"], group), _heads_first(d["value_ptr"], group)
    do, o = _heads_first(d["output_grad_ptr"]), _heads_first(d["output_ptr"])
    p = torch.exp(_scores(c, d) - d["lse_ptr"].T[..., None]).masked_fill(_hidden(c), 0.0)
    ds = p * (do @ v.transpose(1, 2) - (do * o).sum(-1, keepdim=True))
    shared = lambda x: x.unflatten(0, (-1, group)).sum(1)      # noqa: E731  (the query heads of a key head add up)
    grads = ds @ k * _scale(c), shared(ds.transpose(1, 2) @ q) * _scale(c), shared(p.transpose(1, 2) @ do)
    return [g.permute(1, 0, 2).to(torch.float16).contiguous() for g in grads]


# ---- what a pass cannot do without ---------------------------------------------------------------------------------
def _visible(c):
    """Pairs of a query and a key that it sees, in one head."""
    if not c["causal"]:
        return c["queries"] * c["keys"]
    seen = np.arange(c["queries"]) + 1 + c["keys"] - c["queries"]
    return int(np.clip(seen, 0, None).sum())


def work(case):
    size = {"f16": 2, "f32": 4, "i32": 4}
    if case["kind"] == "rotary":
        rows = case["tokens"] * (case["heads"] + case["kv_heads"])
        used = 2 * 4 * case["part"] // 2 * min(case["tokens"], case["table"]) + 4 * case["tokens"]
        return dict(bytes=2 * rows * case["dim"] * size[case["dtype"]] + used, flops=3 * rows * case["part"])
    total = sum(math.prod(s) * size[d] for s, d in _tensors(case).values())
    return dict(bytes=total, flops=(4 if case["kind"] == "forward" else 10) * case["heads"] * case["dim"] * _visible(case))


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------
def _exact_rotary(c, d):
    out = {}
    n = c["part"] // 2
    angle_rows = d["positions_ptr"].long()
    turn = torch.complex(d["cos_ptr"].double()[angle_rows], d["sin_ptr"].double()[angle_rows])
    turn = turn.conj() if c["inverse"] else turn
    for name in ("query", "key"):
        x = d[name + "_ptr"].double()
        y = x.clone()
        first = torch.arange(n, device=x.device) * (1 if c["layout"] == "half" else 2)
        second = first + (n if c["layout"] == "half" else 1)
        z = torch.complex(x[..., first], x[..., second]) * turn[:, None]
        y[..., first], y[..., second] = z.real, z.imag
        out[name + "_out_ptr"] = y
    return out


def exact(case, seed):
    d = _inputs(case, seed)
    if case["kind"] == "rotary":
        return _exact_rotary(case, d)
    group, scale, gone = case["heads"] // case["kv_heads"], _scale(case), _hidden(case)
    out = {k: torch.zeros(s, dtype=torch.float64, device="cuda") for k, (s, _) in _tensors(case).items() if k in _outputs(case)}
    for h in range(case["heads"]):
        q, k, v = (d[n][:, h // g].double() for n, g in (("query_ptr", 1), ("key_ptr", group), ("value_ptr", group)))
        s = (scale * (q @ k.T)).masked_fill(gone, -math.inf)
        if case["kind"] == "forward":
            out["lse_ptr"][:, h] = torch.logsumexp(s, 1)
            out["output_ptr"][:, h] = torch.softmax(s, 1).nan_to_num(0.0) @ v      # (rows that see nothing)
            continue
        lse, o, do = d["lse_ptr"][:, h].double(), d["output_ptr"][:, h].double(), d["output_grad_ptr"][:, h].double()
        p = torch.where(gone, 0.0, torch.exp(s - lse[:, None]))
        ds = p * (do @ v.T - (do * o).sum(1, keepdim=True))
        out["query_grad_ptr"][:, h] = scale * (ds @ k)
        out["key_grad_ptr"][:, h // group] += scale * (ds.T @ q)
        out["value_grad_ptr"][:, h // group] += p.T @ do
    return out
