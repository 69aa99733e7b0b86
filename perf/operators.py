"""The operators of linear layers in 8 bits, as cases that can be timed and compared.

A case is one pass through one operator:
  norm     the residual's addition, the root-mean-square norm, and its output as rows of 8 bits (e4m3) with a scale a row;
  rows     rows of any other activation (an attention's output, a gated activation) to 8 bits with a scale a row;
  product  the matrix product of 8-bit rows and 8-bit weights with bias, activation (plain or gated) and residual in its epilogue.
Sizes are those of the layers this repository benchmarks (hidden 4096 and 5120, feed-forward 12288 and 17408, 32 query and 8 KV heads
of 128) and odd ones of no model.  Streams and activations have a few channels that are much larger than the others, as
those of trained models do; weights are normal with the benchmark's deviation, in 8 bits with a scale an output row, which a program lays
out once when it loads a model.
"""
import math

import torch

own = False
DEVICE = "cuda:0"
EPS = 1e-6
TOP = 448.0                                   # the largest number e4m3 holds


# ---------------------------------------------------------------------------------------------- the cases
def _norm(name, rows, hidden, delta="bfloat16", pick=0):
    return dict(name=name, op="norm", rows=rows, hidden=hidden, delta=delta, pick=pick)


def _rows(name, rows, cols, dtype="bfloat16"):
    return dict(name=name, op="rows", rows=rows, cols=cols, dtype=dtype)


def _product(name, m, n, k, out="bfloat16", bias=False, act="none", gated=False, residual=False):
    return dict(name=name, op="product", m=m, n=n, k=k, out=out, bias=bias, act=act, gated=gated, residual=residual)


def listed():
    return [
        # one user's chat, one token: the norm before a projection; latency is all
        _norm("norm-token", 1, 4096),
        # a prompt's full step through a wide model
        _norm("norm-prompt", 4096, 5120),
        # the last norm on the rows whose logits are wanted, from a float32 result, at an odd width
        _norm("norm-picked", 700, 1001, delta="float32", pick=333),
        # eight requests decoding: the attention's output before its projection
        _rows("rows-decode", 8, 4096),
        # a prompt's step: the gated activation before the down projection
        _rows("rows-prompt", 4096, 12288),
        # one token's queries, keys and values
        _product("qkv-token", 1, 6144, 4096),
        # the benchmark's headline, eight requests decoding: gate and up with the gated activation
        _product("gate-up-decode", 8, 24576, 4096, act="silu", gated=True),
        # a loaded server: the down projection added to the float32 stream
        _product("down-64", 64, 4096, 12288, out="float32", residual=True),
        # a short prompt through a feed-forward of odd sizes with biases
        _product("odd-gelu", 173, 1003, 1000, bias=True, act="gelu", residual=True),
        # a portion of a prompt (the scheduler's default 512): queries, keys and values with a bias
        _product("qkv-portion", 512, 6144, 4096, bias=True),
        # time to the first token of a long prompt: gate and up
        _product("gate-up-prompt", 2048, 24576, 4096, act="silu", gated=True),
        # the scheduler's largest step: the down projection added to the stream
        _product("down-prompt", 4096, 4096, 12288, out="float32", residual=True),
    ]


def draw(rng):
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    def size(lo, hi):
        n = log_int(lo, hi)
        return n if rng.random() < 0.4 else max(1, -(-n // 64) * 64)          # odd ones, and such as layers have

    op = rng.choice(["norm", "rows", "product", "product"])
    if op == "norm":
        rows = log_int(1, 4096)
        case = _norm("", rows, size(96, 5120), rng.choice(["bfloat16", "bfloat16", "float32", "none"]),
                     rng.randint(1, rows) if rng.random() < 0.2 else 0)
    elif op == "rows":
        case = _rows("", log_int(1, 4096), size(96, 12288), rng.choice(["bfloat16", "bfloat16", "float32"]))
    else:
        gated = rng.random() < 0.3
        n = size(96, 24576)
        case = _product("", log_int(1, 4096), -(-n // 16) * 16 if gated else n, size(96, 12288), rng.choice(["bfloat16", "bfloat16", "float32"]),
                        rng.random() < 0.4, rng.choice(["silu", "relu"] if gated else ["none", "none", "none", "silu", "gelu", "relu2"]), gated,
                        rng.random() < 0.5)
        most = 4096 * 4096 * 12288
        while case["m"] * case["n"] * case["k"] > most:
            case["m"] = max(1, case["m"] // 2)
    del case["name"]
    return case


# ---------------------------------------------------------------------------------------------- inputs
def _columns(k):
    """Columns of an 8-bit row: zeros follow the data up to a multiple of 128."""
    return -(-k // 128) * 128


def _to_8_bits(x):
    """[r, k] float32 -> (e4m3 [r, columns], scale [r]): what quantised weights and activations are."""
    top = x.abs().amax(dim=1, keepdim=True)
    inv = torch.where(top > 0, TOP / top, torch.zeros_like(top))
    q = torch.zeros((x.shape[0], _columns(x.shape[1])), dtype=torch.float32, device=x.device)
    q[:, :x.shape[1]] = x * inv
    return q.to(torch.float8_e4m3fn), (top / TOP).squeeze(1)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)

    def normal(*shape, std=1.0):
        return torch.randn(shape, generator=g, device=DEVICE) * std

    def channels(k):                          # a channel in two hundred is some ten times the others
        return 1 + 10 * (torch.rand(k, generator=g, device=DEVICE) < 0.005) * torch.rand(k, generator=g, device=DEVICE)

    s = dict(case=dict(case))
    if case["op"] == "norm":
        t, h = case["rows"], case["hidden"]
        s["x"] = normal(t, h, std=2.0) * channels(h)
        s["delta"] = None if case["delta"] == "none" else normal(t, h, std=0.3).to(getattr(torch, case["delta"]))
        s["weight"] = 1 + normal(h, std=0.2)
        s["pick"] = None
        if case["pick"]:
            s["pick"] = torch.randint(0, t, (case["pick"],), generator=g, device=DEVICE, dtype=torch.int32)
        r = case["pick"] or t
        s["new_x"] = torch.empty_like(s["x"])
        s["out"] = torch.empty((r, _columns(h)), dtype=torch.float8_e4m3fn, device=DEVICE)
        s["scale"] = torch.empty(r, device=DEVICE)
    elif case["op"] == "rows":
        x = normal(case["rows"], case["cols"], std=0.5) * torch.nn.functional.silu(normal(case["rows"], case["cols"])) * channels(case["cols"])
        s["x"] = x.to(getattr(torch, case["dtype"]))
        s["out"] = torch.empty((case["rows"], _columns(case["cols"])), dtype=torch.float8_e4m3fn, device=DEVICE)
        s["scale"] = torch.empty(case["rows"], device=DEVICE)
    else:
        m, n, k = case["m"], case["n"], case["k"]
        s["a"], s["a_scale"] = _to_8_bits(normal(m, k) * channels(k))
        w, s["w_scale"] = _to_8_bits(normal(n, k, std=0.02))
        s["w"] = w
        s["bias"] = normal(n, std=0.1) if case["bias"] else None
        width, dtype = n // 2 if case["gated"] else n, getattr(torch, case["out"])
        s["residual"] = normal(m, width).to(dtype) if case["residual"] else None
        s["out"] = torch.empty((m, width), dtype=dtype, device=DEVICE)
        if own:                               # a program lays its weights out once, when it loads them
            from vllm_lite_b200.csrc import ops
            s["w"] = ops.pack_8bit(w)
    return s


# ---------------------------------------------------------------------------------------------- one pass
def _plain_8_bits(h, out, scale):
    top = h.abs().amax(dim=1, keepdim=True)
    inv = torch.where(top > 0, TOP / top, torch.zeros_like(top))
    out.zero_()
    out[:, :h.shape[1]] = (h * inv).to(torch.float8_e4m3fn)
    scale.copy_((top / TOP).squeeze(1))


def _plain_act(v, name):
    if name == "silu":
        return v / (1 + torch.exp(-v))
    if name == "relu":
        return v * (v > 0)
    if name == "relu2":
        return (v * (v > 0)).square()
    if name == "gelu":
        return 0.5 * v * (1 + torch.erf(v * 0.5 ** 0.5))
    return v


def _plain(s):
    case = s["case"]
    if case["op"] == "norm":
        x = s["x"] if s["pick"] is None else s["x"][s["pick"].long()]
        if s["delta"] is not None:
            x = x + (s["delta"] if s["pick"] is None else s["delta"][s["pick"].long()]).float()
        if s["pick"] is None and s["delta"] is not None:
            s["new_x"].copy_(x)
        _plain_8_bits(x / torch.sqrt(x.square().mean(dim=1, keepdim=True) + EPS) * s["weight"], s["out"], s["scale"])
        return
    if case["op"] == "rows":
        _plain_8_bits(s["x"].float(), s["out"], s["scale"])
        return
    y = (s["a"].float() @ s["w"].float().t()) * s["a_scale"][:, None] * s["w_scale"]
    if s["bias"] is not None:
        y = y + s["bias"]
    if case["gated"]:                         # eight gate rows of the weight, their eight up rows, and so on
        y = y.view(y.shape[0], -1, 2, 8)
        y = (_plain_act(y[:, :, 0], case["act"]) * y[:, :, 1]).reshape(y.shape[0], -1)
    else:
        y = _plain_act(y, case["act"])
    s["out"].copy_(y if s["residual"] is None else y + s["residual"].float())


def _own(s):
    from vllm_lite_b200.csrc import ops
    case = s["case"]
    if case["op"] == "norm":
        ops.add_rmsnorm_8bit(s["x"], s["delta"], s["weight"], EPS, s["out"], s["scale"], rows=s["pick"], into=s["new_x"])
    elif case["op"] == "rows":
        ops.rows_8bit(s["x"], s["out"], s["scale"])
    else:
        ops.gemm_8bit(s["a"], s["a_scale"], s["w"], s["w_scale"], s["out"], bias=s["bias"], act=None if case["act"] == "none" else case["act"],
                      gated=case["gated"], residual=s["residual"])


def run(state):
    (_own if own else _plain)(state)
    case = state["case"]
    if case["op"] == "product":
        return state["out"]
    got = dict(values=state["out"], scale=state["scale"])
    if case["op"] == "norm" and state["pick"] is None and state["delta"] is not None:
        got["stream"] = state["new_x"]
    return got


# ---------------------------------------------------------------------------------------------- what a pass cannot do without
_SIZE = {"bfloat16": 2, "float32": 4, "none": 0}


def work(case):
    if case["op"] == "norm":
        h, r = case["hidden"], case["pick"] or case["rows"]
        stream = 4 if not case["pick"] and case["delta"] != "none" else 0
        return {"bytes": r * h * (4 + _SIZE[case["delta"]] + stream + 1) + 4 * h + 4 * r, "flops": 6 * r * h}
    if case["op"] == "rows":
        return {"bytes": case["rows"] * (case["cols"] * (_SIZE[case["dtype"]] + 1) + 4), "flops": 3 * case["rows"] * case["cols"]}
    m, n, k = case["m"], case["n"], case["k"]
    width = n // 2 if case["gated"] else n
    moved = m * k + n * k + 4 * (m + n) + 4 * n * case["bias"] + m * width * _SIZE[case["out"]] * (2 if case["residual"] else 1)
    return {"bytes": moved, "flops": 2 * m * n * k}


# ---------------------------------------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    """The numbers that 8-bit values are rounded from stand in the place of those values."""
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    d = torch.float64
    if case["op"] == "product":
        y = torch.einsum("mk,nk->mn", s["a"].to(d) * s["a_scale"].to(d)[:, None], s["w"].to(d) * s["w_scale"].to(d)[:, None])
        if s["bias"] is not None:
            y += s["bias"].to(d)
        f = {"none": lambda v: v, "silu": lambda v: v * torch.sigmoid(v), "relu": lambda v: v.clamp(min=0), "relu2": lambda v: v.clamp(min=0) ** 2,
             "gelu": lambda v: v * torch.special.ndtr(v)}[case["act"]]
        if case["gated"]:
            at = torch.arange(y.shape[1], device=y.device)
            y = f(y[:, at % 16 < 8]) * y[:, at % 16 >= 8]
        else:
            y = f(y)
        return y if s["residual"] is None else y + s["residual"].to(d)
    x, got = s["x"].to(d), {}
    if case["op"] == "norm":
        if s["delta"] is not None:
            x = x + s["delta"].to(d)
            if s["pick"] is None:
                got["stream"] = x
        if s["pick"] is not None:
            x = x.index_select(0, s["pick"].long())
        x = x * s["weight"].to(d) * (torch.linalg.vector_norm(x, dim=1, keepdim=True) ** 2 / x.shape[1] + EPS) ** -0.5
    top = torch.linalg.vector_norm(x, ord=float("inf"), dim=1)
    got["scale"] = top / TOP
    got["values"] = torch.nn.functional.pad(x * (TOP / top)[:, None], (0, s["out"].shape[1] - x.shape[1]))
    return got
