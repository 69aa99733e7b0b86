"""The operators of a serving step over a cache in 8 bits, and of its draw, as cases that can be timed and compared.

A case is one pass through one operator:
  write   head norm and rotation of new queries and keys, and the write of keys and values into pages of 8 bits (e4m3) with a scale, a
          power of two, for each page and head;
  decode  attention of single tokens over such pages;
  prompt  attention of portions of prompts over such pages;
  sample  one token per row of logits: temperature, top-k, top-p, min-p, drawn at given random numbers.
Sizes are those of the layers this repository benchmarks (32 query and 8 KV heads of 128, pages of 64, a vocabulary of 151,936) and odd ones of
no model.  Keys have a few channels that are much larger than the others, as those of trained models do; pages lie anywhere in the pool.
"""
import math

import torch

own = False
DEVICE = "cuda:0"
EPS = 1e-6
THETA = 1000000.0
FIX = float(1 << 40)                          # probabilities are summed as whole multiples of 2^-40 of the largest


# ---------------------------------------------------------------------------------------------- the cases
def _write(name, requests, tokens, before, nq=32, nkv=8, hd=128, page=64):
    return dict(name=name, op="write", requests=requests, tokens=tokens, before=before, nq=nq, nkv=nkv, hd=hd, page=page)


def _decode(name, requests, shortest, longest, nq=32, nkv=8, hd=128, page=64, window=0):
    return dict(name=name, op="decode", requests=requests, shortest=shortest, longest=longest, nq=nq, nkv=nkv, hd=hd, page=page, window=window)


def _prompt(name, requests, tokens, before, nq=32, nkv=8, hd=128, page=64, window=0):
    return dict(name=name, op="prompt", requests=requests, tokens=tokens, before=before, nq=nq, nkv=nkv, hd=hd, page=page, window=window)


def _sample(name, rows, vocab, top_k=0, top_p=1.0, min_p=0.0):
    return dict(name=name, op="sample", rows=rows, vocab=vocab, top_k=top_k, top_p=top_p, min_p=min_p)


def listed():
    return [
        # the benchmark's batch decoding: a token a request, most of them into pages that hold rows already
        _write("write-decode", 64, 1, 1500),
        # a long prompt's full step, which begins inside a page
        _write("write-prompt", 1, 4096, 700),
        # short prompts through heads and pages of other sizes
        _write("write-odd", 5, 77, 13, nq=6, nkv=2, hd=80, page=16),
        # one user's chat: latency is all
        _decode("decode-token", 1, 2800, 2800),
        # the benchmark's headline: eight requests at about 4,096 keys
        _decode("decode-8", 8, 3500, 4096),
        # a loaded server, requests of very different lengths
        _decode("decode-64", 64, 400, 4096),
        # two long documents, 16 query heads on a KV head
        _decode("decode-long", 2, 50000, 65536, nq=64, nkv=4),
        # time to the first token of a prompt of 2,048
        _prompt("prompt-first", 1, 2048, 0),
        # portions (the scheduler's 512) of three prompts that are well under way
        _prompt("prompt-portions", 3, 512, 2500),
        # heads of 80, three query heads a KV head, a window, pages of 16
        _prompt("prompt-odd", 4, 150, 100, nq=6, nkv=2, hd=80, page=16, window=90),
        # one user's chat: the draw behind the logits
        _sample("sample-token", 1, 151936, top_k=20, top_p=0.95, min_p=0.02),
        # a loaded server, every row with options of its own (up to these)
        _sample("sample-64", 64, 151936, top_k=200, top_p=0.9, min_p=0.1),
    ]


def draw(rng):
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    def heads():
        nkv = rng.choice([1, 2, 4, 8])
        return dict(nq=nkv * rng.choice([1, 2, 3, 4, 8]), nkv=nkv, hd=rng.choice([128, 128, 128, 64, 64, 32, 80, 96, 192, 256]),
                    page=rng.choice([64, 64, 64, 128, 32, 16, 8, 40]))

    op = rng.choice(["write", "decode", "decode", "prompt", "prompt", "sample"])
    if op == "write":
        n = log_int(1, 64)
        case = _write("", n, 1 if rng.random() < 0.4 else log_int(1, 4096 // n), log_int(1, 100000) - 1, **heads())
        while case["requests"] * case["tokens"] * (case["nq"] + 2 * case["nkv"]) * case["hd"] > 4096 * 48 * 128:
            case["tokens"] = max(1, case["tokens"] // 2)
    elif op == "decode":
        n, longest = log_int(1, 64), log_int(1, 16384)
        case = _decode("", n, max(1, longest // rng.choice([1, 2, 8])), longest, window=log_int(1, 4096) if rng.random() < 0.2 else 0, **heads())
        while case["requests"] * case["longest"] * case["nkv"] * case["hd"] > 64 * 4096 * 8 * 128:
            case["requests"] = max(1, case["requests"] // 2)
    elif op == "prompt":
        n = log_int(1, 6)
        case = _prompt("", n, log_int(2, 2048 // n), log_int(1, 4096) - 1, window=log_int(1, 4096) if rng.random() < 0.2 else 0, **heads())
        while case["requests"] * case["tokens"] * (case["tokens"] + 2 * case["before"]) * case["nq"] * case["hd"] > 2048 * 2048 * 32 * 128:
            case["before"], case["tokens"] = case["before"] // 2, max(2, case["tokens"] * 3 // 4)
    else:
        case = _sample("", log_int(1, 64), log_int(1000, 151936), rng.choice([0, 0, log_int(1, 1000)]), rng.choice([1.0, 0.5, 0.9, 0.95, 0.99]),
                       rng.choice([0.0, 0.0, 0.01, 0.05, 0.2]))
    del case["name"]
    return case


# ---------------------------------------------------------------------------------------------- inputs
def _scales(top):
    """The least power of two s with top <= 448 * s, which is 0.875 * 2^9 * s; 2^-100 at least."""
    m, e = torch.frexp(top)
    e = torch.where(top > 0, e - 9 + (m > 0.875), -100).clamp(min=-100)
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _pool(normal, pages, nkv, page, hd, channels):
    """Pages of a cache in 8 bits: (e4m3 [pages, nkv, page, hd], float32 [pages, nkv])."""
    x = normal(pages, nkv, page, hd) * channels
    scale = _scales(x.abs().amax(dim=(2, 3)))
    return (x / scale[:, :, None, None]).to(torch.float8_e4m3fn), scale


def _lengths(case):
    """Cached tokens before the step, of each request, and new ones."""
    n = case["requests"]
    if case["op"] == "decode":
        span = case["longest"] - case["shortest"]
        return [case["shortest"] - 1 + (span * i // max(1, n - 1) if n > 1 else span) for i in range(n)], [1] * n
    # requests that go on from other places, and bring a little fewer tokens one by one
    return [case["before"] + (37 * i if case["before"] else 0) for i in range(n)], [max(1, case["tokens"] - (i * case["tokens"]) // (4 * n)) for i in range(n)]


def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)

    def normal(*shape, std=1.0):
        return torch.randn(shape, generator=g, device=DEVICE) * std

    def channels(k):                          # a channel in fifty is some times the others
        return 1 + 6 * (torch.rand(k, generator=g, device=DEVICE) < 0.02) * torch.rand(k, generator=g, device=DEVICE)

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device=DEVICE)

    s = dict(case=dict(case))
    if case["op"] == "sample":
        r, v = case["rows"], case["vocab"]
        # a few tokens that stand out over a broad rest
        s["logits"] = normal(r, v, std=2.0) + 9 * torch.rand((r, v), generator=g, device=DEVICE) ** 64
        s["temperature"] = 0.5 + torch.rand(r, generator=g, device=DEVICE)
        if r > 4:
            s["temperature"][::5] = 0.0       # some requests decode greedily
        mine = torch.rand((3, r), generator=g, device=DEVICE) if r > 1 else torch.zeros(3, 1, device=DEVICE)
        s["top_k"] = (case["top_k"] * (1 - mine[0] * 0.9)).ceil().to(torch.int32)
        s["top_p"] = 1 - (1 - case["top_p"]) * (1 - mine[1] * 0.9)
        s["min_p"] = case["min_p"] * (1 - mine[2] * 0.9)
        s["uniform"] = torch.rand(r, generator=g, device=DEVICE)
        s["token"] = torch.empty(r, dtype=torch.int32, device=DEVICE)
        return s

    n, nq, nkv, hd, page = case["requests"], case["nq"], case["nkv"], case["hd"], case["page"]
    before, new = _lengths(case)
    blocks = [-(-(b + k) // page) for b, k in zip(before, new)]
    first = (lambda b: b // page) if case["op"] == "write" else (lambda b: 0)        # a write touches a request's last pages only
    used = [m - first(b) for b, m in zip(before, blocks)]
    pages = sum(used) + 3
    where = torch.randperm(pages, generator=g, device=DEVICE).to(torch.int32)
    table = torch.full((n, max(blocks)), -1, dtype=torch.int32, device=DEVICE)
    at = 0
    for i in range(n):
        table[i, first(before[i]):blocks[i]] = where[at:at + used[i]]
        at += used[i]
    kc, vc = channels(hd), channels(hd)
    s["k"], s["k_scale"] = _pool(normal, pages, nkv, page, hd, kc)
    s["v"], s["v_scale"] = _pool(normal, pages, nkv, page, hd, 0.5 * vc)
    s["table"], s["err"] = table, torch.zeros(1, dtype=torch.int32, device=DEVICE)
    total = sum(new)
    s["req"] = torch.repeat_interleave(torch.arange(n, device=DEVICE), torch.tensor(new, device=DEVICE)).to(torch.int32)
    s["cu"] = ints([sum(new[:i]) for i in range(n + 1)])
    s["pos"] = torch.arange(total, device=DEVICE, dtype=torch.int32) - s["cu"][s["req"].long()] + ints(before)[s["req"].long()]
    if case["op"] == "write":
        s["slots"] = table[s["req"].long(), (s["pos"] // page).long()] * page + s["pos"] % page
        s["qkv"] = torch.cat([normal(total, nq * hd, std=2.0), normal(total, nkv * hd, std=2.0) * kc.repeat(nkv),
                              normal(total, nkv * hd, std=0.5) * vc.repeat(nkv)], dim=1).to(torch.bfloat16)
        s["qw"], s["kw"] = 1 + normal(hd, std=0.2), 1 + normal(hd, std=0.2)
        s["freq"] = (1.0 / THETA ** (torch.arange(0, hd, 2, device=DEVICE, dtype=torch.float64) / hd)).float()
        s["q"] = torch.empty((total, nq * hd), dtype=torch.bfloat16, device=DEVICE)
        pages, s["visit"] = torch.unique(s["slots"].long() // page, return_inverse=True)       # the pages that the step reaches
        s["pages"] = pages
        return s
    s["q"] = normal(total, nq * hd, std=1.5).to(torch.bfloat16)
    s["out"] = torch.empty_like(s["q"])
    s["longest"] = max(b + k for b, k in zip(before, new))
    if case["op"] == "decode":                # the workspace that a program keeps: partial results, and counters that are left zero
        pieces = 2 + -(-600 // (total * nkv))
        s["scratch"] = torch.empty(total * nq * pieces * (hd + 2), device=DEVICE)
        s["arrivals"] = torch.zeros(total * nq, dtype=torch.int32, device=DEVICE)
    else:                                     # stretches of up to 128 tokens: row of the table, first token, tokens, first position
        start = [sum(new[:i]) for i in range(n)]
        s["tiles"] = ints([(i, start[i] + lo, min(128, new[i] - lo), before[i] + lo) for i in range(n) for lo in range(0, new[i], 128)])
    return s


# ---------------------------------------------------------------------------------------------- one pass
def _plain_write(s):
    case = s["case"]
    nq, nkv, hd, page = case["nq"], case["nkv"], case["hd"], case["page"]
    x = s["qkv"].float().view(-1, nq + 2 * nkv, hd)
    angle = s["pos"].double()[:, None] * s["freq"].double()
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]

    def head(h, w):
        h = h / torch.sqrt(h.square().mean(dim=2, keepdim=True) + EPS) * w
        a, b = h[..., :hd // 2], h[..., hd // 2:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=2)

    s["q"].copy_(head(x[:, :nq], s["qw"]).flatten(1))
    row = s["slots"].long() % page
    _plain_rows(s["k"], s["k_scale"], head(x[:, nq:nq + nkv], s["kw"]), s["pages"], s["visit"], row)
    _plain_rows(s["v"], s["v_scale"], x[:, nq + nkv:], s["pages"], s["visit"], row)


def _plain_rows(cache, scale, x, pages, inverse, row):
    """New rows x [T, nkv, hd] into rows `row` of pages[inverse], and those pages' earlier rows under the scale that both share."""
    size = cache.shape[2]
    lowest = torch.full_like(pages, size).scatter_reduce(0, inverse, row, "amin")                # rows below it were there before
    top = torch.zeros((pages.numel(), x.shape[1]), device=DEVICE).scatter_reduce(0, inverse[:, None].expand(-1, x.shape[1]), x.abs().amax(dim=2), "amax")
    need = _scales(top)
    old = torch.where((lowest > 0)[:, None], scale[pages], torch.zeros_like(need))
    now = torch.maximum(old, need)
    kept = (torch.arange(size, device=DEVICE) < lowest[:, None])[:, None, :, None]
    there = cache[pages].float()
    cache[pages] = torch.where(kept, there * (old / now)[:, :, None, None], there).to(torch.float8_e4m3fn)
    cache.view(torch.uint8)[pages[inverse], :, row] = (x / now[inverse][:, :, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    scale[pages] = now


def _plain_attention(s):
    """All requests side by side, padded to the longest: queries [n, most, heads], keys [n, longest]."""
    case = s["case"]
    n, nq, nkv, hd, page = case["requests"], case["nq"], case["nkv"], case["hd"], case["page"]
    req, pos = s["req"].long(), s["pos"].long()
    table = s["table"].long().clamp(min=0)
    place = torch.arange(pos.numel(), device=DEVICE) - s["cu"].long()[req]                       # a token's place within its request
    most = case["tokens"] if case["op"] == "prompt" else 1
    q = torch.zeros((n, most, nq, hd), device=DEVICE)
    q[req, place] = s["q"].float().view(-1, nq, hd)
    at = torch.full((n, most), -1, device=DEVICE, dtype=torch.long)
    at[req, place] = pos

    def rows(cache, scale):                   # [n, nkv, keys, hd]
        return (cache[table].float() * scale[table][..., None, None]).transpose(1, 2).reshape(n, nkv, -1, hd)

    k, v = rows(s["k"], s["k_scale"]), rows(s["v"], s["v_scale"])
    key = torch.arange(k.shape[2], device=DEVICE)
    seen = key <= at[:, :, None]
    if case["window"]:
        seen &= key > at[:, :, None] - case["window"]
    q = q.view(n, most, nkv, nq // nkv, hd).permute(0, 2, 3, 1, 4).reshape(n, nkv, -1, hd)
    score = (q @ k.transpose(2, 3)).mul_(hd ** -0.5).view(n, nkv, nq // nkv, most, -1)
    score.masked_fill_(~seen[:, None, None], float("-inf"))
    top = score.amax(dim=4, keepdim=True).clamp(min=-1e30)
    score.sub_(top).exp_()
    total = score.sum(dim=4, keepdim=True)
    out = (score.flatten(2, 3) @ v).view(n, nkv, nq // nkv, most, hd) / total.clamp(min=1e-30)
    s["out"].copy_(out.permute(0, 3, 1, 2, 4).reshape(n, most, nq * hd)[req, place])


def _plain_sample(s):
    logits, t = s["logits"], s["temperature"]
    vocab = logits.shape[1]
    greedy = t <= 0
    x = logits * (1 / torch.where(greedy, torch.ones_like(t), t))[:, None]
    top = x.amax(dim=1, keepdim=True)
    mass = (torch.exp(x - top) * FIX).long()
    order = torch.sort(x, dim=1, descending=True)
    k = s["top_k"].long()
    kth = order.values.gather(1, (torch.where((k > 0) & (k < vocab), k, torch.full_like(k, vocab)) - 1)[:, None])
    mass = mass * (x >= kth)
    summed = mass.gather(1, order.indices).cumsum(dim=1)
    goal = (s["top_p"].double() * summed[:, -1].double()).long()[:, None]
    nucleus = order.values.gather(1, (summed <= goal).sum(dim=1, keepdim=True).clamp(max=vocab - 1))
    mass = mass * ((x >= nucleus) | (s["top_p"] >= 1)[:, None])
    mass = mass * (mass >= (s["min_p"].double() * FIX).long()[:, None])
    summed = mass.cumsum(dim=1)
    goal = torch.minimum((s["uniform"].double() * summed[:, -1].double()).long(), summed[:, -1] - 1)[:, None]
    first = torch.where(logits == logits.amax(dim=1, keepdim=True), torch.arange(vocab, device=DEVICE), vocab).amin(dim=1)
    s["token"].copy_(torch.where(greedy, first, (summed <= goal).sum(dim=1)))


def _own(s):
    from vllm_lite_b200.csrc import ops
    case = s["case"]
    if case["op"] == "sample":
        ops.sample(s["logits"], s["temperature"], s["top_k"], s["top_p"], s["uniform"], s["token"], min_p=s["min_p"])
        return
    nq, nkv, hd = case["nq"], case["nkv"], case["hd"]
    cache = (s["k"], s["v"], s["k_scale"], s["v_scale"])
    if case["op"] == "write":
        ops.qk_norm_rope_write_8bit(s["qkv"], s["pos"], s["slots"], s["cu"], s["qw"], s["kw"], EPS, s["freq"], hd, *cache, nq, nkv, hd, s["err"],
                                    q_out=s["q"])
    elif case["op"] == "decode":
        ops.flash_decode_8bit(s["q"], s["out"], *cache, s["table"], s["req"], s["pos"], nq, nkv, hd, hd ** -0.5, case["window"], s["longest"], s["err"],
                              scratch=s["scratch"], arrivals=s["arrivals"])
    else:
        ops.flash_prefill_8bit(s["q"], s["out"], *cache, s["table"], s["tiles"], nq, nkv, hd, hd ** -0.5, case["window"], s["err"])


def run(state):
    op = state["case"]["op"]
    if own:
        _own(state)
    elif op == "write":
        _plain_write(state)
    elif op == "sample":
        _plain_sample(state)
    else:
        _plain_attention(state)
    if op == "write":
        return {name: state[name] for name in ("q", "k", "v", "k_scale", "v_scale")}
    return state["token" if op == "sample" else "out"]


# ---------------------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    if case["op"] == "sample":
        return {"bytes": 4 * case["rows"] * case["vocab"] + 24 * case["rows"], "flops": 4 * case["rows"] * case["vocab"]}
    nq, nkv, hd, page = case["nq"], case["nkv"], case["hd"], case["page"]
    before, new = _lengths(case)
    total = sum(new)
    if case["op"] == "write":
        return {"bytes": total * hd * (2 * (nq + 2 * nkv) + 2 * nq + 2 * nkv) + 12 * total, "flops": total * hd * (7 * (nq + nkv) + 3 * nkv)}
    reach = case["window"] or 1 << 40
    pairs = sum(sum(min(reach, b + i + 1) for i in range(k)) for b, k in zip(before, new))
    keys = sum(min(b + k, reach + k - 1) for b, k in zip(before, new))
    return {"bytes": 2 * keys * nkv * (hd + 4 / page) + 4 * total * nq * hd, "flops": 4 * pairs * nq * hd}


# ---------------------------------------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    """The numbers that 8-bit values are rounded from stand in the place of those values."""
    s, d = prepare(case, seed), torch.float64
    if case["op"] == "sample":
        return None                           # token ids alone, and those are whole numbers
    nq, nkv, hd, page = case["nq"], case["nkv"], case["hd"], case["page"]
    if case["op"] == "write":
        x = s["qkv"].to(d).unflatten(1, (nq + 2 * nkv, hd))
        turn = torch.polar(torch.ones((), dtype=d, device=DEVICE), torch.outer(s["pos"].to(d), s["freq"].to(d)))[:, None]

        def head(h, w):
            h = h * w.to(d) * (torch.linalg.vector_norm(h, dim=2, keepdim=True) ** 2 / hd + EPS) ** -0.5
            z = torch.complex(*h.split(hd // 2, dim=2)) * turn
            return torch.cat([z.real, z.imag], dim=2)

        got = dict(q=head(x[:, :nq], s["qw"]).flatten(1))
        for name, new in (("k", head(x[:, nq:nq + nkv], s["kw"])), ("v", x[:, nq + nkv:])):
            cache, scale = s[name].to(d), s[name + "_scale"].to(d)
            start = 0
            slots = s["slots"].tolist()
            while start < len(slots):         # a stretch of tokens that share a page
                p, low = divmod(slots[start], page)
                end = start
                while end < len(slots) and slots[end] // page == p:
                    end += 1
                rows = new[start:end]
                least = torch.exp2(torch.ceil(torch.log2(rows.abs().amax(dim=(0, 2)) / 448)))
                both = torch.maximum(least, scale[p]) if low else least
                if low:
                    cache[p, :, :low] *= (scale[p] / both)[:, None, None]
                cache[p, :, low:low + end - start] = rows.transpose(0, 1) / both[:, None, None]
                scale[p] = both
                start = end
            got[name], got[name + "_scale"] = cache, scale
        return got
    out = torch.empty((s["q"].shape[0], nq, hd), dtype=d, device=DEVICE)
    cu, pos, group = s["cu"].tolist(), s["pos"].to(torch.int64), nq // nkv
    for i in range(case["requests"]):
        mine = slice(cu[i], cu[i + 1])
        p = pos[mine]
        pages = s["table"][i, :int(p[-1]) // page + 1].long()
        for h in range(nkv):
            k, v = ((c[pages, h].to(d) * sc[pages, h].to(d)[:, None, None]).flatten(0, 1)[:int(p[-1]) + 1]
                    for c, sc in ((s["k"], s["k_scale"]), (s["v"], s["v_scale"])))
            j = torch.arange(k.shape[0], device=DEVICE)
            ahead = j[None] > p[:, None]
            if case["window"]:
                ahead |= j[None] <= p[:, None] - case["window"]
            q = s["q"][mine].to(d).unflatten(1, (nq, hd))[:, h * group:(h + 1) * group]
            score = torch.einsum("tgd,jd->gtj", q, k) / math.sqrt(hd)
            out[mine, h * group:(h + 1) * group] = torch.einsum("gtj,jd->tgd", torch.softmax(score.masked_fill(ahead, float("-inf")), dim=2), v)
    return out.flatten(1)
