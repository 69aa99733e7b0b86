"""A cache in 8 bits: its write, and the attention of single tokens and of prompt portions over it, against their definitions in 64 bits.

Tolerances.  A rounding to e4m3 is off by half a step: 2^-4 of a value, or 2^-10 of the scale where it is subnormal; to bfloat16 by 2^-8 of a value.

The write's numbers before they are rounded: a mean of up to 256 squares, a root, a quotient and the rotation's two products and sum in float32, each off by
2^-24 of a number that is at most the head's largest times 16: 2^-18 of the head's largest covers them.  Where such a number decides whether a
page's scale is one power of two or the next, either is right.

Attention, with W = sum_j p_j |v_j| and A the largest sum_d |q_d k_jd| scale of the keys read: float32 sums of up to 256 products, cut by the tensor
cores instead of rounded, are off by 2^-20 of the sum of their absolute values, so a weight by 2^-20 A of itself, numerator and denominator together twice that; the
base-2 exponential and its argument's rounding add 2^-20 (1 + A); a weight is rounded to a half, 2^-11 of it; weights below 2^-31 of the largest
may vanish: fewer than 2^17 keys, 2^-14 of the largest value at worst, and 2^-20 of it with the keys of these tests (fewer than 2^11)."""
import math

import pytest
import torch

from vllm_lite_b200.csrc import ops

gpu = pytest.mark.gpu
DEV = "cuda:0"
EPS = 1e-6
D = torch.float64


# ---------------------------------------------------------------------------------------------- what a cache holds
def least_scale(top):
    """The least power of two s, 2^-100 at least, with top <= 448 s."""
    if top == 0:
        return 2.0 ** -100
    m, e = math.frexp(top)
    return 2.0 ** max(-100, e - 9 + (m > 0.875))


class Cache:
    """Pools of pages that nobody owns yet: bytes of NaN under scales that are none, so that whatever reads one shows it."""

    def __init__(self, requests, longest, nkv, ps, hd, seed=0, spare=3):
        g = torch.Generator().manual_seed(seed)
        self.nkv, self.ps, self.hd = nkv, ps, hd
        per = -(-longest // ps)
        n = requests * per + spare
        self.k, self.v = (torch.full((n, nkv, ps, hd), 0x7f, dtype=torch.uint8, device=DEV).view(ops.E4M3) for _ in range(2))
        self.k_scale, self.v_scale = (torch.full((n, nkv), float("nan"), device=DEV) for _ in range(2))
        self.table = torch.randperm(n, generator=g)[:requests * per].view(requests, per).to(torch.int32).to(DEV)
        self.err = torch.zeros(1, dtype=torch.int32, device=DEV)

    @property
    def tensors(self):
        return self.k, self.v, self.k_scale, self.v_scale

    def fill(self, lengths, seed=0, spread=3):
        """Random keys and values of the requests' first tokens, pages' scales 2^-spread to 2^spread around 2^-6."""
        g = torch.Generator(device=DEV).manual_seed(seed)
        for cache, scale in ((self.k, self.k_scale), (self.v, self.v_scale)):
            for r, n in enumerate(lengths):
                for b in range(-(-n // self.ps)):
                    page, rows = int(self.table[r, b]), min(self.ps, n - b * self.ps)
                    x = torch.randn(self.nkv, rows, self.hd, generator=g, device=DEV) * 60
                    cache.view(torch.uint8)[page, :, :rows] = x.clamp(-448, 448).to(ops.E4M3).view(torch.uint8)
                    scale[page] = torch.exp2(torch.randint(-6 - spread, -5 + spread, (self.nkv,), generator=g, device=DEV).float())
            self.table_lengths = lengths
        for r, n in enumerate(lengths):                       # what lies behind a request's last page is nobody's
            self.table[r, -(-n // self.ps):] = -1
        return self

    def rows(self, r, n):
        """Keys and values of request r's first n tokens, [n, nkv, hd] in 64 bits."""
        pages = self.table[r, :-(-n // self.ps)].long()
        return tuple((c[pages].to(D) * s[pages].to(D)[..., None, None]).transpose(1, 2).reshape(-1, self.nkv, self.hd)[:n]
                     for c, s in ((self.k, self.k_scale), (self.v, self.v_scale)))


def batch(cache, before, new):
    """positions, request numbers, cu_seqlens, slots of requests that hold `before` tokens and bring `new`."""
    pos = torch.cat([torch.arange(b, b + n) for b, n in zip(before, new)]).to(torch.int32).to(DEV)
    req = torch.cat([torch.full((n,), r) for r, n in enumerate(new)]).to(torch.int32).to(DEV)
    cu = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32, device=DEV)
    slots = cache.table[req.long(), (pos // cache.ps).long()] * cache.ps + pos % cache.ps
    return pos, req, cu, slots


# ---------------------------------------------------------------------------------------------- the write
def turned_heads(x, weight, pos, inv_freq, rot):
    """x [T, heads, hd] in 64 bits: norm, then the rotation of the first rot features."""
    x = x.to(D)
    if weight is not None:
        x = x / torch.sqrt(x.square().mean(dim=2, keepdim=True) + EPS) * weight.to(D)
    if rot:
        angle = pos.to(D)[:, None, None] * inv_freq.to(D)
        a, b, c, s = x[..., :rot // 2], x[..., rot // 2:rot], torch.cos(angle), torch.sin(angle)
        x = torch.cat([a * c - b * s, b * c + a * s, x[..., rot:]], dim=2)
    return x


def check_write(cache, was, qkv, q, pos, req, slots, nq, qw, kw, inv_freq, rot):
    """`was`: (k, v, k_scale, v_scale) before the write."""
    nkv, hd, ps = cache.nkv, cache.hd, cache.ps
    T = qkv.shape[0]
    x = qkv.view(T, nq + 2 * nkv, hd)
    want = turned_heads(x[:, :nq], qw, pos, inv_freq, rot)
    slack = 2.0 ** -18 * want.abs().amax(dim=2, keepdim=True)
    assert ((q.to(D).view(T, nq, hd) - want).abs() <= 2.0 ** -8 * want.abs() + slack).all()
    keys, values = turned_heads(x[:, nq:nq + nkv], kw, pos, inv_freq, rot), x[:, nq + nkv:].to(D)
    at = slots.long()
    for new, now, before, scale, scale_before in ((keys, cache.k, was[0], cache.k_scale, was[2]), (values, cache.v, was[1], cache.v_scale, was[3])):
        touched = torch.zeros(now.shape[0], dtype=torch.bool, device=DEV)
        for page in at[at >= 0].div(ps, rounding_mode="floor").unique().tolist():
            touched[page] = True
            mine = ((at >= 0) & (at.div(ps, rounding_mode="floor") == page)).nonzero()[:, 0]
            row0, n = int(at[mine[0]]) % ps, mine.numel()
            rows = new[mine].transpose(0, 1)                                       # [nkv, n, hd]
            slack = 2.0 ** -18 * rows.abs().amax(dim=(1, 2))
            for h in range(nkv):
                top, old, s = float(rows[h].abs().max()), float(scale_before[page, h]) if row0 else 0.0, float(scale[page, h])
                assert max(old, least_scale(top - float(slack[h]))) <= s <= max(old, least_scale(top + float(slack[h])))
                got = now[page, h].to(D) * s
                off = (got[row0:row0 + n] - rows[h]).abs()
                assert (off <= torch.maximum(2.0 ** -4 * rows[h].abs(), torch.tensor(2.0 ** -10 * s, dtype=D, device=DEV)) * (1 + 2.0 ** -10) + slack[h]).all()
                if row0:                                                           # earlier rows: as they were, but for what became subnormal
                    there = before[page, h, :row0].to(D) * old
                    assert ((got[:row0] - there).abs() <= (2.0 ** -10 * s if s > old else 0.0)).all()
            assert torch.equal(now.view(torch.uint8)[page, :, row0 + n:], before.view(torch.uint8)[page, :, row0 + n:])
        assert torch.equal(now.view(torch.uint8)[~touched], before.view(torch.uint8)[~touched])
        assert torch.equal(scale.view(torch.int32)[~touched], scale_before.view(torch.int32)[~touched])


def copies(cache):
    return tuple(t.view(torch.uint8).clone().view(t.dtype) if t.dtype == ops.E4M3 else t.clone() for t in cache.tensors)


WRITES = [
    # nq, nkv, hd, ps, rot, requests' tokens before and new
    (2, 1, 16, 16, 16, [0], [1]),
    (32, 8, 128, 64, 128, [0, 63, 64, 130], [1, 1, 1, 1]),
    (32, 8, 128, 64, 128, [0, 60, 200], [300, 70, 1]),
    (6, 2, 80, 16, 80, [3, 0, 15, 16, 31], [40, 1, 2, 33, 1]),
    (4, 2, 64, 1, 64, [0, 5], [9, 3]),
    (3, 3, 48, 7, 24, [2, 7], [30, 6]),
    (4, 1, 256, 256, 256, [100], [600]),
    (4, 2, 192, 40, 0, [39, 0], [100, 41]),
    (1, 1, 112, 128, 100, [70, 3], [150, 1]),
]


@gpu
@pytest.mark.parametrize("nq,nkv,hd,ps,rot,before,new", WRITES)
@pytest.mark.parametrize("normed", [True, False])
def test_write(nq, nkv, hd, ps, rot, before, new, normed):
    g = torch.Generator(device=DEV).manual_seed(hd + ps)
    normal = lambda *s: torch.randn(*s, generator=g, device=DEV)
    cache = Cache(len(new), max(b + n for b, n in zip(before, new)), nkv, ps, hd).fill(before)
    cache.table = Cache(len(new), max(b + n for b, n in zip(before, new)), nkv, ps, hd).table      # (the same pages, none given back)
    pos, req, cu, slots = batch(cache, before, new)
    T = sum(new)
    qkv = (normal(T, (nq + 2 * nkv) * hd) * torch.exp2(3 * normal(T, 1))).to(torch.bfloat16)       # tokens of very different sizes
    inv_freq = (1e6 ** (-torch.arange(0, rot, 2, dtype=D, device=DEV) / max(rot, 1))).float() if rot else None
    qw, kw = (1 + 0.2 * normal(hd), 1 + 0.2 * normal(hd)) if normed else (None, None)
    was, rows = copies(cache), qkv.clone()
    for out in (torch.full((T, nq * hd), 3.0, dtype=torch.bfloat16, device=DEV), None):
        fresh = qkv.clone()
        for t, w in zip(cache.tensors, was):
            t.view(torch.uint8 if t.dtype == ops.E4M3 else t.dtype).copy_(w.view(torch.uint8 if w.dtype == ops.E4M3 else w.dtype))
        got = ops.qk_norm_rope_write_8bit(fresh, pos, slots, cu, qw, kw, EPS, inv_freq, rot, *cache.tensors, nq, nkv, hd, cache.err, q_out=out)
        q = got[:, :nq * hd] if out is None else got
        assert int(cache.err) == 0
        assert torch.equal(fresh[:, nq * hd:], rows[:, nq * hd:]) and (out is None or torch.equal(fresh, rows))
        check_write(cache, was, rows, q, pos, req, slots, nq, qw, kw, inv_freq, rot)


@gpu
@pytest.mark.parametrize("nkv,hd,ps", [(5, 128, 16), (6, 64, 32), (3, 32, 64), (7, 256, 16), (5, 128, 17), (9, 128, 64)])
def test_write_of_several_heads_at_a_time(nkv, hd, ps):
    """Pages that a few warps hold, and more pages than a launch needs to share angles: heads beside one another, their number no multiple of a block's."""
    test_write(nkv * 2, nkv, hd, ps, hd, [0, 5, ps - 1, 3 * ps, 7], [40, 1, 30, 2 * ps + 3, 60], True)
    test_write(nkv, nkv, hd, ps, 0, [11, 0], [700, 350], False)


@gpu
@pytest.mark.parametrize("nkv,hd,ps", [(3, 128, 64), (5, 64, 100), (2, 256, 48), (4, 32, 256), (2, 112, 100)])
def test_write_of_one_long_portion_among_short_ones(nkv, hd, ps):
    """Far more rows for some pages than portions have on average."""
    test_write(nkv * 3, nkv, hd, ps, hd, [7] + [(11 * i) % ps for i in range(9)], [2 * ps + 30] + [1] * 4 + [2] * 5, True)


@gpu
@pytest.mark.parametrize("hd,rot,ps", [(128, 128, 16), (80, 80, 8), (256, 0, 64)])
@pytest.mark.parametrize("new", [[0, 2], [2, 0], [0, 0, 3], [3, 0, 1, 0], [1, 0, 0, 30, 1, 0] + [0] * 26, [7, 0, 0, 0, 0, 0, 0]])
def test_write_of_as_many_tokens_as_requests_but_not_one_each(hd, rot, ps, new):
    assert sum(new) == len(new)
    test_write(4, 2, hd, ps, rot, [(5 * i) % (ps + 3) for i in range(len(new))], new, True)


@gpu
def test_far_positions():
    """Angles of positions that float32 holds, whose products with a frequency it does not: off by the rounding of the sine's own arithmetic only."""
    nq, nkv, hd, ps = 2, 1, 128, 64
    before = [100000, 1000000]
    cache = Cache(2, 64 * 2, nkv, ps, hd)
    pos = torch.tensor(before, dtype=torch.int32, device=DEV)
    slots = cache.table[:, 0].contiguous() * ps + pos % ps
    cu = torch.tensor([0, 1, 2], dtype=torch.int32, device=DEV)
    qkv = torch.randn(2, 4 * hd, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV).to(torch.bfloat16)
    inv_freq = (1e6 ** (-torch.arange(0, hd, 2, dtype=D, device=DEV) / hd)).float()
    q = torch.empty(2, nq * hd, dtype=torch.bfloat16, device=DEV)
    cache.k_scale.zero_(), cache.v_scale.zero_()                                   # earlier rows of zeros
    cache.k.view(torch.uint8).zero_(), cache.v.view(torch.uint8).zero_()
    ops.qk_norm_rope_write_8bit(qkv, pos, slots, cu, None, None, EPS, inv_freq, hd, *cache.tensors, nq, nkv, hd, cache.err, q_out=q)
    want = turned_heads(qkv.view(2, 4, hd)[:, :nq], None, pos, inv_freq, hd)
    # the product's error, up to 2^-24 of 10^6, is added to first order: its square, half of it, is left
    assert ((q.to(D).view(2, nq, hd) - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -18 + (1e6 * 2.0 ** -24) ** 2 / 2) * want.abs().amax()).all()


def write_values(cache, x, before, new):
    """Keys and values x [T, nkv, hd] into the cache, no norm, no rotation."""
    nkv, hd = cache.nkv, cache.hd
    T = x.shape[0]
    pos, req, cu, slots = batch(cache, before, new)
    qkv = torch.cat([torch.zeros(T, nkv * hd, device=DEV), x.reshape(T, -1), x.reshape(T, -1)], dim=1).to(torch.bfloat16)
    ops.qk_norm_rope_write_8bit(qkv, pos, slots, cu, None, None, EPS, None, 0, *cache.tensors, nkv, nkv, hd, cache.err)


@gpu
@pytest.mark.parametrize("ps", [16, 64, 100])
def test_token_by_token_or_at_once(ps):
    """Tokens that come one by one, in portions, or all at once leave the same page, to the bit: scales are powers of two, so rows that move to a larger
    one keep their bits while none is subnormal (here: multiples of 1 / 8 from 1 to 2 times 2^0 to 2^9)."""
    nkv, hd, n = 2, 32, 90
    g = torch.Generator(device=DEV).manual_seed(5)
    x = (1 + torch.randint(0, 8, (n, nkv, hd), generator=g, device=DEV) / 8) * torch.exp2((torch.arange(n, device=DEV) // 10).float())[:, None, None]
    x *= torch.randint(0, 2, x.shape, generator=g, device=DEV) * 2 - 1
    got = []
    for cuts in ([n], [1] * n, [7, 1, 30, 2, 50]):
        cache, at = Cache(1, n, nkv, ps, hd, seed=2), 0
        for c in cuts:
            write_values(cache, x[at:at + c], [at], [c])
            at += c
        assert int(cache.err) == 0
        k, v = cache.rows(0, n)
        assert torch.equal(k, x.to(D)) and torch.equal(v, x.to(D))                 # (every number is an e4m3 value times the scale)
        got.append((k, cache.k_scale[cache.table[0].long()]))
    assert all(torch.equal(a, b) for other in got[1:] for a, b in zip(got[0], other))


@gpu
def test_scales_at_their_borders():
    """A page's largest number on both sides of 448 times a power of two, the smallest and largest that bfloat16 holds, and none."""
    tops = [448.0, 450.0, 224.0, 225.0, 1.0, 0.0, 2.0 ** -92, 448 * 2.0 ** -100, 2.0 ** -126, 2.0 ** -133, 3.3895e38, 3.0e38, 2.0 ** 127]
    tops = [float(torch.tensor(t).to(torch.bfloat16)) for t in tops]
    cache = Cache(len(tops), 4, 1, 4, 16)
    x = torch.zeros(len(tops), 1, 16, device=DEV)
    x[:, 0, 3] = torch.tensor(tops, device=DEV)
    x[:, 0, 7] = -x[:, 0, 3] / 2
    write_values(cache, x, [0] * len(tops), [1] * len(tops))
    for r, top in enumerate(tops):
        page = int(cache.table[r, 0])
        s = least_scale(top)
        assert float(cache.k_scale[page, 0]) == s == float(cache.v_scale[page, 0]), top
        got = cache.k[page, 0, 0].to(D) * s
        assert float(got[3]) == pytest.approx(top, rel=2.0 ** -4, abs=2.0 ** -10 * s) and float(got[7]) == pytest.approx(-top / 2, rel=2.0 ** -4, abs=2.0 ** -10 * s)


@gpu
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_numbers_that_are_none(bad):
    """The page and head they come to, and no other; the page's next life begins anew."""
    nkv, hd, ps = 2, 32, 8
    cache = Cache(2, 24, nkv, ps, hd)
    x = torch.randn(35, nkv, hd, generator=torch.Generator(device=DEV).manual_seed(3), device=DEV)
    x[9, 1, 4] = bad                                                                # request 0's token 9: page 1, head 1
    write_values(cache, x[:35], [0, 0], [23, 12])
    t = cache.table.long()
    lost = torch.isnan(cache.k_scale)
    assert lost[t[0, 1], 1] and not lost[t[0, 1], 0] and not lost[t[0, 0]].any() and not lost[t[0, 2]].any() and not lost[t[1, :2]].any()
    write_values(cache, x[:1], [23], [1])                                           # another page of the request
    assert torch.isnan(cache.v_scale[t[0, 1], 1]) and not torch.isnan(cache.v_scale[t[0, 2]]).any()
    write_values(cache, x[:1], [0], [1])                                            # page 0 again, from its first row
    write_values(cache, x[:8], [8], [8])                                            # and page 1
    assert not torch.isnan(cache.k_scale[t[0, :2]]).any() and not torch.isnan(cache.v_scale[t[0, :2]]).any()
    k, _ = cache.rows(0, 16)
    assert ((k[8:] - x[:8].to(torch.bfloat16).to(D)).abs() <= 2.0 ** -4 * x[:8].to(torch.bfloat16).to(D).abs() + 2.0 ** -10).all()


@gpu
def test_tokens_that_are_not_written():
    """Padded tokens (position -1, in no request), tokens without a slot, slots beyond the pool and out of order: nothing else moves; what names no place is flagged."""
    nq, nkv, hd, ps = 2, 1, 32, 8
    cache = Cache(2, 16, nkv, ps, hd).fill([8, 8])
    was = copies(cache)
    qkv = torch.randn(6, 4 * hd, generator=torch.Generator(device=DEV).manual_seed(4), device=DEV).to(torch.bfloat16)
    same = lambda: all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(cache.tensors, was))
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)

    def go(pos, slots, cu):
        cache.err.zero_()
        ops.qk_norm_rope_write_8bit(qkv, i32(pos), i32(slots) if slots is not None else None, i32(cu), None, None, EPS, None, 0, *cache.tensors, nq, nkv, hd,
                                    cache.err, q_out=torch.empty(6, nq * hd, dtype=torch.bfloat16, device=DEV))
        return int(cache.err)

    assert go([-1] * 6, [-1] * 6, [0, 0, 0]) == 0 and same()
    assert go([8, 9, 10, 11, 12, 13], [-1] * 6, [0, 6]) == 0 and same()
    assert go([8, 9, 10, 11, 12, 13], None, [0, 6]) == 0 and same()
    assert go([8, 9, 10, 11, 12, 13], [8 * cache.k.shape[0] + i for i in range(6)], [0, 6]) == 2 and same()
    page = int(cache.table[0, 0])                                                   # a first slot that is not its position's row
    assert go([8, 9, 10, 11, 12, 13], [page * 8 + 1 + i for i in range(6)], [0, 6]) == 2 and same()
    assert go([8, 9, 10, 11, 12, 13], [page * 8 + i for i in (0, 1, 5, 3, 4, 5)], [0, 6]) == 2                # one row elsewhere: skipped, the others written
    now = cache.k.view(torch.uint8)[page, 0]
    assert torch.equal(now[2], was[0].view(torch.uint8)[page, 0, 2]) and not torch.equal(now[3], was[0].view(torch.uint8)[page, 0, 3])
    assert go([8, 9, 10, 11, 12, 13], [-1] * 6, [0, 9]) == 0                       # bounds beyond the tokens: no request


# ---------------------------------------------------------------------------------------------- attention
def check_attention(cache, q, out, pos, req, nq, window, scale, only=None):
    nkv, hd = cache.nkv, cache.hd
    group = nq // nkv
    for t in range(q.shape[0]) if only is None else only:
        p = int(pos[t])
        lo = max(0, p - window + 1) if window else 0
        k, v = (x[lo:] for x in cache.rows(int(req[t]), p + 1))
        mine = q[t, :nq * hd].to(D).view(nkv, group, hd)
        score = torch.einsum("hgd,jhd->hgj", mine, k) * scale
        w = torch.softmax(score, dim=2)
        want, W = torch.einsum("hgj,jhd->hgd", w, v), torch.einsum("hgj,jhd->hgd", w, v.abs())
        A = (torch.einsum("hgd,jhd->hgj", mine.abs(), k.abs()) * scale).amax(dim=2, keepdim=True)
        tol = 2.0 ** -8 * want.abs() + (2.0 ** -11 + 2.0 ** -19 * A + 2.0 ** -20 * (1 + A)) * W + 2.0 ** -20 * v.abs().amax()
        got = out[t].to(D).view(nkv, group, hd)
        assert torch.isfinite(got).all() and ((got - want).abs() <= tol).all(), (t, p, float(((got - want).abs() / tol).max()))


def queries(T, nq, hd, seed, extra=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(T, nq * hd + extra, generator=g, device=DEV) * torch.exp2(torch.randint(-3, 2, (T, 1), generator=g, device=DEV).float())).to(torch.bfloat16)


ATTENTION = [
    # nq, nkv, hd, ps, window
    (1, 1, 16, 16, None), (2, 1, 32, 64, None), (32, 8, 128, 64, None), (16, 8, 64, 16, 5), (6, 2, 80, 8, 20), (40, 2, 64, 40, None), (9, 1, 128, 128, 64),
    (16, 1, 256, 64, None), (4, 2, 192, 7, 100), (3, 3, 48, 1, None), (5, 1, 112, 256, 1), (34, 2, 96, 64, None), (12, 4, 144, 16, None), (8, 1, 240, 32, 33),
    (200, 1, 32, 64, None),
]


@gpu
@pytest.mark.parametrize("nq,nkv,hd,ps,window", ATTENTION)
def test_single_tokens(nq, nkv, hd, ps, window):
    lengths = [1, 2, 15, 16, 17, 63, 64, 65, 200, 777]
    cache = Cache(len(lengths), max(lengths), nkv, ps, hd, seed=1).fill(lengths, seed=hd)
    pos, req = (torch.tensor(v, dtype=torch.int32, device=DEV) for v in ([n - 1 for n in lengths], list(range(len(lengths)))))
    q = queries(len(lengths), nq, hd, 7, extra=2 * nkv * hd)                       # (rows that hold keys and values too)
    out = torch.full((len(lengths), nq * hd), 3.0, dtype=torch.bfloat16, device=DEV)
    ops.flash_decode_8bit(q, out, *cache.tensors, cache.table, req, pos, nq, nkv, hd, hd ** -0.5, window, max(lengths), cache.err)
    assert int(cache.err) == 0
    check_attention(cache, q, out, pos, req, nq, window, hd ** -0.5)
    # one request alone: many blocks share its keys
    for r in (0, 4, 9):
        alone = torch.full((1, nq * hd), 3.0, dtype=torch.bfloat16, device=DEV)
        ops.flash_decode_8bit(q[r:r + 1], alone, *cache.tensors, cache.table, req[r:r + 1], pos[r:r + 1], nq, nkv, hd, hd ** -0.5, window, lengths[r], cache.err)
        check_attention(cache, q[r:r + 1], alone, pos[r:r + 1], req[r:r + 1], nq, window, hd ** -0.5)
    assert int(cache.err) == 0


def tiles_of(before, new, most=128):
    start = [sum(new[:i]) for i in range(len(new))]
    return torch.tensor([(r, start[r] + lo, min(most, n - lo), before[r] + lo) for r, n in enumerate(new) for lo in range(0, n, most)],
                        dtype=torch.int32, device=DEV).view(-1, 4)


@gpu
@pytest.mark.parametrize("nq,nkv,hd,ps,window", ATTENTION)
def test_prompt_portions(nq, nkv, hd, ps, window):
    before, new = [0, 0, 300, 63, 129, 5], [1, 130, 33, 2, 64, 300]
    longest = max(b + n for b, n in zip(before, new))
    cache = Cache(len(new), longest, nkv, ps, hd, seed=1).fill([b + n for b, n in zip(before, new)], seed=hd)
    pos, req, _, _ = batch(cache, before, new)
    q = queries(sum(new), nq, hd, 8, extra=2 * nkv * hd)
    out = torch.full((sum(new), nq * hd), 3.0, dtype=torch.bfloat16, device=DEV)
    only = [0, 1, 2, 31, 32, 64, 100, 130, 131, 140, 163, 164, 165, 166, 200, 229, 230, 262, 300, 400, 528, 529]
    for most in (128, 50):
        ops.flash_prefill_8bit(q, out.fill_(3.0), *cache.tensors, cache.table, tiles_of(before, new, most), nq, nkv, hd, hd ** -0.5, window, cache.err)
        assert int(cache.err) == 0
        check_attention(cache, q, out, pos, req, nq, window, hd ** -0.5, only)
    assert torch.isfinite(out).all()


@gpu
@pytest.mark.parametrize("nq,nkv,hd,ps,window", [(8, 2, 128, 64, None), (4, 1, 64, 16, None), (6, 2, 80, 40, 900), (4, 1, 256, 64, None), (32, 1, 128, 128, 1500)])
@pytest.mark.parametrize("own", [True, False])
def test_few_tokens_with_many_keys(nq, nkv, hd, ps, window, own):
    """Keys shared out among blocks and joined (a weight, a product and a sum a share in float32: 2^-20 of the sums as they are allowed anyway holds 16 of them)."""
    before, new = [1900, 0, 700, 1337, 511], [3, 1, 40, 64, 1]
    cache = Cache(len(new), 1984, nkv, ps, hd, seed=4).fill([b + n for b, n in zip(before, new)], seed=hd + 1)
    pos, req, _, _ = batch(cache, before, new)
    q = queries(sum(new), nq, hd, 9, extra=16)
    out = torch.full((sum(new) + 1, nq * hd), 3.0, dtype=torch.bfloat16, device=DEV)
    floats = ops.flash_prefill_8bit_scratch(hd, DEV)
    scratch = torch.full((floats + 64,), float("nan"), device=DEV) if own else None
    for _ in range(2):
        ops.flash_prefill_8bit(q, out[:-1], *cache.tensors, cache.table, tiles_of(before, new), nq, nkv, hd, hd ** -0.5, window, cache.err,
                               scratch=scratch[:floats] if own else None)
    assert int(cache.err) == 0 and (out[-1] == 3.0).all()
    assert not own or torch.isnan(scratch[floats:]).all()
    check_attention(cache, q, out[:-1], pos, req, nq, window, hd ** -0.5, [0, 1, 2, 3, 4, 20, 43, 44, 60, 107, 108])


@gpu
@pytest.mark.parametrize("nq,nkv,hd,ps,window,tokens", [(32, 8, 128, 64, None, 1260), (64, 8, 64, 16, None, 640), (128, 16, 32, 64, 1200, 700), (40, 8, 256, 64, None, 600)])
def test_last_round_of_few_blocks(nq, nkv, hd, ps, window, tokens):
    """More blocks than SMs and few of them in the last round, whose keys are shared out; prompts of several lengths, so that some have too few keys for it."""
    before, new = [700, 0, 900], [tokens - 300, 200, 100]
    cache = Cache(len(new), max(b + n for b, n in zip(before, new)), nkv, ps, hd, seed=4).fill([b + n for b, n in zip(before, new)], seed=hd + 1)
    pos, req, _, _ = batch(cache, before, new)
    q = queries(tokens, nq, hd, 9)
    out = torch.full((tokens, nq * hd), 3.0, dtype=torch.bfloat16, device=DEV)
    whole = torch.full_like(out, 3.0)
    tiles = tiles_of(before, new)
    for o, scratch in ((out, None), (whole, torch.empty(ops.flash_prefill_8bit_scratch(hd, DEV), device=DEV))):
        ops.flash_prefill_8bit(q, o, *cache.tensors, cache.table, tiles, nq, nkv, hd, hd ** -0.5, window, cache.err, scratch=scratch)
    assert int(cache.err) == 0 and torch.equal(out, whole)
    g = torch.Generator().manual_seed(1)
    check_attention(cache, q, out, pos, req, nq, window, hd ** -0.5, sorted({0, 1, 63, 64, tokens - 301, tokens - 300, tokens - 101, tokens - 100, tokens - 1}
                                                                            | set(torch.randint(0, tokens, (12,), generator=g).tolist())))


@gpu
@pytest.mark.parametrize("which", ["k_scale", "v_scale"])
def test_a_lost_page_among_shared_keys(which):
    """One share of the keys is none: so is the result of those who read it, whatever share it is, and nobody else's."""
    nq, nkv, hd, ps, n = 4, 2, 64, 64, 1600
    cache = Cache(1, n, nkv, ps, hd).fill([n])
    q = queries(4, nq, hd, 5)
    for lost in (0, 12, 24):
        scale = getattr(cache, which)
        page, kept = int(cache.table[0, lost]), scale.clone()
        scale[page, 1] = float("nan")
        out = ops.flash_prefill_8bit(q, torch.empty_like(q), *cache.tensors, cache.table, tiles_of([n - 4], [4]), nq, nkv, hd, hd ** -0.5, None, cache.err).view(4, nq, hd)
        assert torch.isfinite(out[:, :2]).all() and torch.isnan(out[:, 2:]).all()
        out = ops.flash_prefill_8bit(q, torch.empty_like(q), *cache.tensors, cache.table, tiles_of([n - 4], [4]), nq, nkv, hd, hd ** -0.5, 700, cache.err).view(4, nq, hd)
        assert torch.isfinite(out[:, :2]).all() and torch.isnan(out[:, 2:]).all() == (lost == 24) and torch.isfinite(out[:, 2:]).all() == (lost != 24)
        scale.copy_(kept)
    assert int(cache.err) == 0


@gpu
def test_pages_of_very_different_scales():
    """Values of a page 2^14 below the largest page's, which alone is looked at (its key is the only one near the query), keep their bits."""
    nq, nkv, hd, ps = 4, 1, 64, 64
    cache = Cache(1, 256, nkv, ps, hd).fill([256], spread=0)
    pages = cache.table[0].long()
    cache.v_scale[pages] *= torch.tensor([[1.0], [2.0 ** 14], [1.0], [2.0 ** 3]], device=DEV)
    cache.k.view(torch.uint8)[pages[0], 0, 10] = torch.full((hd,), 448.0, device=DEV).to(ops.E4M3).view(torch.uint8)
    q = torch.full((256, nq * hd), 4.0, dtype=torch.bfloat16, device=DEV)
    pos, req = torch.arange(256, dtype=torch.int32, device=DEV), torch.zeros(256, dtype=torch.int32, device=DEV)
    k, v = cache.rows(0, 256)
    assert float((q[0, :hd].to(D) * k[10, 0]).sum() - (q[0, :hd].to(D) * k[:, 0]).sum(dim=1).topk(2).values[1]) * hd ** -0.5 > 60
    out = torch.empty_like(q)
    ops.flash_prefill_8bit(q, out, *cache.tensors, cache.table, tiles_of([0], [256]), nq, nkv, hd, hd ** -0.5, None, cache.err)
    assert ((out[255].to(D).view(nq, hd) - v[10]).abs() <= (2.0 ** -8 + 2.0 ** -10) * v[10].abs()).all()
    ops.flash_decode_8bit(q[255:], out[255:].fill_(0), *cache.tensors, cache.table, req[255:], pos[255:], nq, nkv, hd, hd ** -0.5, None, 256, cache.err)
    assert ((out[255].to(D).view(nq, hd) - v[10]).abs() <= (2.0 ** -8 + 2.0 ** -10) * v[10].abs()).all()


@gpu
@pytest.mark.parametrize("which", ["k_scale", "v_scale"])
@pytest.mark.parametrize("ps", [16, 64])
def test_a_page_that_is_lost_shows_where_it_is_read(which, ps):
    nq, nkv, hd = 4, 2, 64
    n = 256
    cache = Cache(1, n, nkv, ps, hd).fill([n])
    lost = 96 // ps                                                                 # the page of position 96, head 1
    getattr(cache, which)[int(cache.table[0, lost]), 1] = float("nan")
    pos, req = torch.arange(n, dtype=torch.int32, device=DEV), torch.zeros(n, dtype=torch.int32, device=DEV)
    q, first, last = queries(n, nq, hd, 3), lost * ps, lost * ps + ps
    for window in (None, 40):
        for kind in ("prompt", "single"):
            out = torch.full((n, nq * hd), 3.0, dtype=torch.bfloat16, device=DEV)
            if kind == "prompt":
                ops.flash_prefill_8bit(q, out, *cache.tensors, cache.table, tiles_of([0], [n]), nq, nkv, hd, hd ** -0.5, window, cache.err)
            else:
                ops.flash_decode_8bit(q, out, *cache.tensors, cache.table, req, pos, nq, nkv, hd, hd ** -0.5, window, n, cache.err)
            nan = torch.isnan(out.view(n, nkv, -1))
            reads = (pos >= first) & ((pos - window + 1 < last) if window else torch.ones_like(pos, dtype=torch.bool))
            assert not nan[:, 0].any() and torch.equal(nan[:, 1].all(dim=1), reads) and torch.equal(nan[:, 1].any(dim=1), reads), (kind, window)
    assert int(cache.err) == 0


@gpu
def test_rows_that_a_launch_does_not_serve_stay():
    nq, nkv, hd, ps = 4, 2, 64, 16
    lengths = [40, 50, 60]
    cache = Cache(3, 64, nkv, ps, hd).fill(lengths)
    q = queries(3, nq, hd, 3)
    pos, req = (torch.tensor(v, dtype=torch.int32, device=DEV) for v in ([39, 49, 59], [0, 1, 2]))
    args = (*cache.tensors, cache.table, req, pos, nq, nkv, hd, hd ** -0.5, None)
    out = torch.full((3, nq * hd), 3.0, dtype=torch.bfloat16, device=DEV)
    ops.flash_decode_8bit(q, out, *args, 64, cache.err, token_index=torch.tensor([2, 0], dtype=torch.int32, device=DEV))
    assert (out[1] == 3).all()
    check_attention(cache, q, out, pos, req, nq, None, hd ** -0.5, only=[0, 2])
    ops.flash_decode_8bit(q, out.fill_(3), *args, 64, cache.err, token_index=torch.tensor([], dtype=torch.int32, device=DEV))
    ops.flash_prefill_8bit(q, out, *cache.tensors, cache.table, tiles_of([], []), nq, nkv, hd, hd ** -0.5, None, cache.err)
    assert (out == 3).all()
    # padded places: rows of zeros; positions beyond the bound: the same, flagged
    pos2 = torch.tensor([-1, 49, 59], dtype=torch.int32, device=DEV)
    ops.flash_decode_8bit(q, out, *cache.tensors, cache.table, req, pos2, nq, nkv, hd, hd ** -0.5, None, 50, cache.err)
    assert (out[0] == 0).all() and (out[2] == 0).all() and int(cache.err) == 0x10
    cache.err.zero_()
    check_attention(cache, q, out, pos, req, nq, None, hd ** -0.5, only=[1])
    # all padded
    ops.flash_decode_8bit(q, out.fill_(3), *cache.tensors, cache.table, req, torch.full_like(pos, -1), nq, nkv, hd, hd ** -0.5, None, 50, cache.err)
    assert (out == 0).all() and int(cache.err) == 0


@gpu
def test_pages_that_are_none():
    """A missing page, one beyond the pool, a table that ends early: flagged, never followed; what is there is read."""
    nq, nkv, hd, ps = 4, 2, 64, 16
    cache = Cache(1, 64, nkv, ps, hd).fill([64])
    q = queries(64, nq, hd, 3)
    pos, req = torch.arange(64, dtype=torch.int32, device=DEV), torch.zeros(64, dtype=torch.int32, device=DEV)
    good = cache.table.clone()
    for bad in (-1, cache.k.shape[0], 1 << 30, "short"):
        table = good.clone()
        if bad == "short":
            table = table[:, :2].contiguous()
        else:
            table[0, 1] = bad
        out = torch.empty(64, nq * hd, dtype=torch.bfloat16, device=DEV)
        for kind in ("single", "prompt"):
            cache.err.zero_()
            if kind == "single":
                ops.flash_decode_8bit(q[63:], out[63:], *cache.tensors, table, req[63:], pos[63:], nq, nkv, hd, hd ** -0.5, None, 64, cache.err)
            else:
                ops.flash_prefill_8bit(q, out, *cache.tensors, table, tiles_of([0], [64]), nq, nkv, hd, hd ** -0.5, None, cache.err)
            assert int(cache.err) == 4 and torch.isfinite(out[63]).all(), (kind, bad)
    cache.err.zero_()
    # a window that leaves the missing page out reads it nowhere
    table = good.clone()
    table[0, 0] = -1
    ops.flash_decode_8bit(q[63:], out[63:], *cache.tensors, table, req[63:], pos[63:], nq, nkv, hd, hd ** -0.5, 48, 64, cache.err)
    check_attention(cache, q, out, pos, req, nq, 48, hd ** -0.5, only=[63])
    ops.flash_prefill_8bit(q, out, *cache.tensors, table, torch.tensor([[0, 63, 1, 63]], dtype=torch.int32, device=DEV), nq, nkv, hd, hd ** -0.5, 48, cache.err)
    check_attention(cache, q, out, pos, req, nq, 48, hd ** -0.5, only=[63])
    assert int(cache.err) == 0


@gpu
def test_a_pool_of_more_than_four_gigabytes():
    nq, nkv, hd, ps, pages = 8, 8, 128, 64, 66000                                   # 2^32 bytes are 65,536 pages
    k, v = (torch.empty(pages, nkv, ps, hd, dtype=torch.uint8, device=DEV).view(ops.E4M3) for _ in range(2))
    ks, vs = (torch.zeros(pages, nkv, device=DEV) for _ in range(2))
    cache = Cache(2, 192, nkv, ps, hd)
    cache.k, cache.v, cache.k_scale, cache.v_scale = k, v, ks, vs
    cache.table = torch.tensor([[pages - 1, 40000, 65535], [65537, 3, 33000]], dtype=torch.int32, device=DEV)
    x = torch.randn(2 * 150, nkv, hd, generator=torch.Generator(device=DEV).manual_seed(6), device=DEV)
    write_values(cache, x, [0, 0], [150, 150])
    for r in range(2):
        got, want = cache.rows(r, 150)[0], x[r * 150:r * 150 + 150].to(torch.bfloat16).to(D)
        assert ((got - want).abs() <= 2.0 ** -4 * want.abs() + 2.0 ** -10).all()
    q = queries(300, nq, hd, 3)
    pos, req, _, _ = batch(cache, [0, 0], [150, 150])
    out = torch.empty(300, nq * hd, dtype=torch.bfloat16, device=DEV)
    ops.flash_prefill_8bit(q, out, *cache.tensors, cache.table, tiles_of([0, 0], [150, 150]), nq, nkv, hd, hd ** -0.5, None, cache.err)
    check_attention(cache, q, out, pos, req, nq, None, hd ** -0.5, only=[0, 149, 150, 299])
    ops.flash_decode_8bit(q, out.fill_(3), *cache.tensors, cache.table, req, pos, nq, nkv, hd, hd ** -0.5, None, 150, cache.err)
    check_attention(cache, q, out, pos, req, nq, None, hd ** -0.5, only=[0, 149, 150, 299])
    assert int(cache.err) == 0


@gpu
def test_write_and_attention_together():
    """Prompts in portions beside requests that decode, as an engine's steps are: every attention against the cache as it is then, and what the cache holds in
    the end against the keys and values that came."""
    nq, nkv, hd, ps = 8, 2, 64, 16
    g = torch.Generator(device=DEV).manual_seed(9)
    cache = Cache(3, 200, nkv, ps, hd)
    inv_freq = (1e4 ** (-torch.arange(0, hd, 2, dtype=D, device=DEV) / hd)).float()
    qw, kw = (1 + 0.2 * torch.randn(hd, generator=g, device=DEV) for _ in range(2))
    have, came = [0, 0, 0], [[], [], []]
    for new in ([50, 0, 0], [1, 70, 0], [1, 33, 40], [1, 1, 60], [1, 1, 1], [1, 1, 1], [60, 1, 2], [1, 1, 1]):
        pos, req, cu, slots = batch(cache, have, new)
        qkv = torch.randn(sum(new), (nq + 2 * nkv) * hd, generator=g, device=DEV).to(torch.bfloat16)
        rows = qkv.clone().view(-1, nq + 2 * nkv, hd)
        ops.qk_norm_rope_write_8bit(qkv, pos, slots, cu, qw, kw, EPS, inv_freq, hd, *cache.tensors, nq, nkv, hd, cache.err)
        keys = turned_heads(rows[:, nq:nq + nkv], kw, pos, inv_freq, hd)
        for r in range(3):
            came[r].append(torch.stack([keys[req == r], rows[:, nq + nkv:].to(D)[req == r]]))
        out = torch.full((sum(new), nq * hd), 3.0, dtype=torch.bfloat16, device=DEV)
        many = [n if n > 1 else 0 for n in new]
        tiles = torch.tensor([(r, int(cu[r]) + lo, min(128, n - lo), have[r] + lo) for r, n in enumerate(many) for lo in range(0, n, 128)], dtype=torch.int32, device=DEV)
        common, sizes = (qkv, out, *cache.tensors, cache.table), (nq, nkv, hd, hd ** -0.5, None)
        if tiles.numel():
            ops.flash_prefill_8bit(*common, tiles, *sizes, cache.err)
        single = torch.tensor([int(cu[r]) for r, n in enumerate(new) if n == 1], dtype=torch.int32, device=DEV)
        if single.numel():
            ops.flash_decode_8bit(*common, req, pos, *sizes, 200, cache.err, token_index=single)
        have = [a + b for a, b in zip(have, new)]
        check_attention(cache, qkv, out, pos, req, nq, None, hd ** -0.5)
    assert int(cache.err) == 0
    for r in range(3):
        for got, want, scale in zip(cache.rows(r, have[r]), torch.cat(came[r], dim=1), (cache.k_scale, cache.v_scale)):
            s = scale[cache.table[r].long()].to(D).repeat_interleave(ps, dim=0)[:have[r], :, None]
            # rounded to e4m3 once, and once more where a later scale made it subnormal
            assert ((got - want).abs() <= 2.0 ** -4 * want.abs() * (1 + 2.0 ** -10) + 2.0 ** -9 * s + 2.0 ** -18 * want.abs().amax()).all()


@gpu
def test_captured_and_replayed():
    """Two graphs that share a workspace, replayed in turn with other lengths and other queries."""
    nq, nkv, hd, ps = 8, 2, 128, 64
    cache = Cache(4, 1100, nkv, ps, hd).fill([1100, 900, 1000, 700])
    floats, counters = ops.flash_decode_8bit_scratch(4, nq, nkv, hd)
    scratch, arrivals = torch.empty(floats, device=DEV), torch.zeros(counters, dtype=torch.int32, device=DEV)
    stream, sets = torch.cuda.Stream(), []
    for B in (4, 2):
        pos, req = torch.zeros(B, dtype=torch.int32, device=DEV), torch.arange(B, dtype=torch.int32, device=DEV)
        q, out = queries(B, nq, hd, B), torch.empty(B, nq * hd, dtype=torch.bfloat16, device=DEV)
        call = lambda q=q, out=out, req=req, pos=pos: ops.flash_decode_8bit(q, out, *cache.tensors, cache.table, req, pos, nq, nkv, hd, hd ** -0.5, None, 1100,
                                                                            cache.err, scratch=scratch, arrivals=arrivals)
        call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(stream), torch.cuda.graph(graph, stream=stream):
            call()
        sets.append((graph, pos, req, q, out))
    for turn in range(4):
        for graph, pos, req, q, out in sets:
            B = pos.numel()
            pos.copy_(torch.tensor([1099, 899, 999, 699][:B], device=DEV) // (1, 3, 2, 900)[turn])
            q.copy_(queries(B, nq, hd, 10 + turn))
            graph.replay()
            torch.cuda.synchronize()
            check_attention(cache, q, out, pos, req, nq, None, hd ** -0.5)
    assert int(cache.err) == 0 and not arrivals.any()


@gpu
def test_on_another_stream():
    nq, nkv, hd, ps = 4, 2, 64, 64
    cache = Cache(2, 300, nkv, ps, hd)
    x = torch.randn(300 + 250, nkv, hd, generator=torch.Generator(device=DEV).manual_seed(2), device=DEV)
    q = queries(550, nq, hd, 3)
    pos, req, _, _ = batch(cache, [0, 0], [300, 250])
    tiles = tiles_of([0, 0], [300, 250])
    out = torch.empty(550, nq * hd, dtype=torch.bfloat16, device=DEV)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        write_values(cache, x, [0, 0], [300, 250])
        ops.flash_prefill_8bit(q, out, *cache.tensors, cache.table, tiles, nq, nkv, hd, hd ** -0.5, None, cache.err)
        ops.flash_decode_8bit(q, out, *cache.tensors, cache.table, req, pos, nq, nkv, hd, hd ** -0.5, None, 300, cache.err,
                              token_index=torch.tensor([299, 549], dtype=torch.int32, device=DEV))
    side.synchronize()
    check_attention(cache, q, out, pos, req, nq, None, hd ** -0.5, only=[0, 100, 298, 299, 300, 548, 549])


# ---------------------------------------------------------------------------------------------- refusals
def entry_args():
    host = torch.zeros(64)                                   # never read or written
    return host, -host.data_ptr() % 16 + host.data_ptr()


@pytest.mark.parametrize("change,code", [
    (dict(hd=24), -2), (dict(hd=272), -2), (dict(rot=6), -2), (dict(rot=144), -2), (dict(stride=100), -3), (dict(q_stride=100), -3), (dict(ps=0), -3), (dict(pages=0), -3),
    (dict(qkv=2), -3), (dict(q=2), -3), (dict(k=8), -3), (dict(v=8), -3), (dict(pages=1 << 30), -2), (dict(nkv=0), -3), (dict(T=0), 0), (dict(cu=None), -3)])
def test_the_write_refuses_before_any_launch(change, code):
    host, at = entry_args()
    c = dict(qkv=0, q=0, k=0, v=0, cu=at, B=1, rot=128, T=1, nq=2, nkv=1, hd=128, ps=64, pages=4, stride=512, q_stride=256)
    c.update(change)
    got = ops._fn("cache_8bit", "vl_qk_norm_rope_write_8bit")(at + c["qkv"], c["stride"], at + c["q"], c["q_stride"], at, at, c["cu"], c["B"], None, None, 1e-6, at, c["rot"],
                                                              at + c["k"], at + c["v"], at, at, c["T"], c["nq"], c["nkv"], c["hd"], c["ps"], c["pages"], None, 0)
    assert got == code


@pytest.mark.parametrize("change,code", [
    (dict(hd=64), -2), (dict(nq=3), -3), (dict(nkv=0), -3), (dict(ps=0), -3), (dict(pages=0), -3), (dict(blocks=0), -3), (dict(stride=250), -3), (dict(stride=258), -3),
    (dict(bound=0), -3), (dict(floats=700), -3), (dict(q=4), -3), (dict(k=8), -3), (dict(v=8), -3), (dict(part=None), -3), (dict(part=8), -3), (dict(arrivals=None), -3), (dict(pages=1 << 30), -2),
    (dict(T=1 << 30), -2), (dict(T=0), 0)])
def test_single_tokens_are_refused_before_any_launch(change, code):
    host, at = entry_args()
    c = dict(q=0, k=0, v=0, stride=256, blocks=2, T=1, nq=2, nkv=1, hd=128, ps=64, pages=4, bound=100, floats=780, part=at, arrivals=at)
    c.update(change)
    got = ops._fn("flash_decode_8bit", "vl_flash_decode_8bit", {"FA_HD": 128})(
        at + c["q"], c["stride"], at + c["k"], at + c["v"], at, at, at, c["blocks"], at, at, c["T"], c["nq"], c["nkv"], c["hd"], c["ps"], c["pages"], 0.1, 0, c["bound"],
        c["part"], c["floats"], None, None, at, c["arrivals"], 0, 0)
    assert got == code


@pytest.mark.parametrize("change,code", [
    (dict(hd=64), -2), (dict(nq=3), -3), (dict(nkv=0), -3), (dict(ps=0), -3), (dict(pages=0), -3), (dict(blocks=0), -3), (dict(stride=250), -3), (dict(stride=260), -3),
    (dict(window=-1), -3), (dict(scratch=4), -3), (dict(floats=10), -3), (dict(q=8), -3), (dict(out=8), -3), (dict(k=8), -3), (dict(tiles=4), -3), (dict(pages=1 << 30), -2), (dict(n=1 << 16), -2), (dict(n=0), 0)])
def test_prompt_portions_are_refused_before_any_launch(change, code):
    host, at = entry_args()
    c = dict(q=0, out=0, k=0, v=0, tiles=0, stride=256, blocks=2, n=1, nq=2, nkv=1, hd=128, ps=64, pages=4, window=0, scratch=0, floats=1 << 30)
    c.update(change)
    got = ops._fn("flash_tc5_8bit", "vl_flash_prefill_8bit", {"FA_HD": 128})(
        at + c["q"], c["stride"], at + c["out"], at + c["k"], at + c["v"], at, at, at, c["blocks"], at + c["tiles"], c["n"], c["nq"], c["nkv"], c["hd"], c["ps"], c["pages"], 0.1,
        c["window"], at + c["scratch"], c["floats"], None, 0)
    assert got == code


def test_tensors_on_the_cpu_are_refused():
    t = torch.zeros(4, 4)
    with pytest.raises(ops.KernelError):
        ops.qk_norm_rope_write_8bit(t.bfloat16(), t, None, None, None, None, 0.0, None, 0, None, None, None, None, 1, 1, 16, None)
    with pytest.raises(ops.KernelError):
        ops.flash_decode_8bit(t.bfloat16(), t, *[t] * 4, t, t, t, 1, 1, 16, 1.0, None, 4, None)
    with pytest.raises(ops.KernelError):
        ops.flash_prefill_8bit(t.bfloat16(), t, *[t] * 4, t, t, 1, 1, 16, 1.0, None, None)


@gpu
def test_another_device_than_the_current_one(monkeypatch):
    cache = Cache(1, 64, 2, 16, 64).fill([64])
    pos, req, cu, slots = batch(cache, [0], [4])
    qkv = queries(4, 4, 64, 1, extra=2 * 2 * 64)
    out = torch.empty(4, 256, dtype=torch.bfloat16, device=DEV)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 1)
    for call in (lambda: ops.qk_norm_rope_write_8bit(qkv, pos, slots, cu, None, None, EPS, None, 0, *cache.tensors, 4, 2, 64, cache.err),
                 lambda: ops.flash_decode_8bit(qkv, out, *cache.tensors, cache.table, req, pos, 4, 2, 64, 0.1, None, 64, cache.err),
                 lambda: ops.flash_prefill_8bit(qkv, out, *cache.tensors, cache.table, tiles_of([0], [4]), 4, 2, 64, 0.1, None, cache.err)):
        with pytest.raises(ops.KernelError, match="current device"):
            call()


@gpu
def test_refusals():
    nq, nkv, hd, ps = 4, 2, 64, 16
    cache = Cache(1, 64, nkv, ps, hd).fill([64])
    pos, req, cu, slots = batch(cache, [0], [4])
    qkv, out = queries(4, nq, hd, 1, extra=2 * nkv * hd), torch.full((4, nq * hd), 3.0, dtype=torch.bfloat16, device=DEV)
    inv = torch.ones(hd // 2, device=DEV)
    was = copies(cache)
    good = dict(qkv=qkv, positions=pos, slots=slots, cu_seqlens=cu, q_weight=None, k_weight=None, eps=EPS, inv_freq=inv, rotary_dim=hd, k_cache=cache.k, v_cache=cache.v,
                k_scale=cache.k_scale, v_scale=cache.v_scale, num_heads=nq, num_kv_heads=nkv, head_dim=hd, err=cache.err)
    for bad in (dict(qkv=qkv.float()), dict(qkv=qkv[:, :-16]), dict(positions=pos.long()), dict(positions=pos[:3]), dict(slots=slots[:3]), dict(cu_seqlens=None),
                dict(cu_seqlens=cu.long()), dict(q_weight=torch.ones(hd - 1, device=DEV)), dict(k_weight=torch.ones(hd, device=DEV).bfloat16()), dict(inv_freq=inv[:5]),
                dict(inv_freq=inv[:3], rotary_dim=6), dict(k_cache=cache.k.view(torch.uint8)), dict(k_cache=cache.k[1:]), dict(k_scale=cache.k_scale[1:]),
                dict(v_scale=cache.v_scale.double()), dict(v_cache=cache.v[:, :, :8]), dict(num_kv_heads=3), dict(head_dim=24, num_heads=4), dict(q_out=out[:, 1:]),
                dict(q_out=out.float())):
        with pytest.raises(ops.KernelError):
            ops.qk_norm_rope_write_8bit(**{**good, **bad})
    good = dict(q=qkv, out=out, k_cache=cache.k, v_cache=cache.v, k_scale=cache.k_scale, v_scale=cache.v_scale, block_table=cache.table, num_heads=nq, num_kv_heads=nkv,
                head_dim=hd, scale=0.1, window=None, err=cache.err)
    common = [dict(q=qkv.float()), dict(q=qkv[:, :nq * hd - 16].contiguous()), dict(out=out[:3]), dict(out=out.float()), dict(k_cache=cache.k.view(torch.uint8)), dict(k_scale=cache.k_scale[:, :1]),
              dict(block_table=cache.table.long()), dict(block_table=cache.table[0]), dict(num_heads=3), dict(num_kv_heads=1), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")),
              dict(window=-3), dict(q=qkv[:, ::2])]
    single = dict(req_index=torch.zeros(4, dtype=torch.int32, device=DEV), positions=pos, max_context=64)
    for bad in common + [dict(req_index=pos[:2]), dict(positions=pos.long()), dict(max_context=0), dict(token_index=pos.long()), dict(scratch=torch.empty(8, device=DEV)),
                         dict(arrivals=torch.zeros(2, dtype=torch.int32, device=DEV)), dict(arrivals=torch.zeros(999, device=DEV))]:
        with pytest.raises(ops.KernelError):
            ops.flash_decode_8bit(**{**good, **single, **bad})
    tiles = tiles_of([0], [4])
    for bad in common + [dict(tiles=tiles[:, :3].contiguous()), dict(tiles=tiles.long()), dict(tiles=tiles[0]), dict(scratch=torch.empty(8, device=DEV)),
                         dict(scratch=torch.empty(1 << 24, device=DEV)[1:]), dict(scratch=torch.empty(1 << 24, device=DEV).double())]:
        with pytest.raises(ops.KernelError):
            ops.flash_prefill_8bit(**{**good, "tiles": tiles, **bad})
    off = torch.empty(4 * (nq + 2 * nkv) * hd + 1, dtype=torch.bfloat16, device=DEV)[1:].view(4, -1)     # rows that begin on two bytes
    for call in (lambda: ops.qk_norm_rope_write_8bit(off, pos, slots, cu, None, None, EPS, None, 0, *cache.tensors, nq, nkv, hd, cache.err),
                 lambda: ops.flash_decode_8bit(**{**good, **single, "q": off}), lambda: ops.flash_prefill_8bit(**{**good, "tiles": tiles, "q": off})):
        with pytest.raises(ops.KernelError):
            call()
    assert (out == 3).all() and int(cache.err) == 0
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(cache.tensors, was))
