"""Sampling with min-p, and rows that a cluster of blocks shares.

A token's mass is floor(exp(s - max) 2^40), a whole number, so what is kept and what is drawn is checked exactly wherever no threshold lies nearer to a token than the
exponential's own rounding: the reference works in 64 bits, and rows in which one comes nearer than 2^-20 of itself are not looked at."""
import itertools

import pytest
import torch

from vllm_lite_b200.csrc import ops
from vllm_lite_b200.sampling import SamplingParams

gpu = pytest.mark.gpu
DEV = "cuda:0"
D = torch.float64
NEAR = 2.0 ** -20


def reference(row, t, k, tp, mp, u):
    """The token drawn from one row, in 64 bits; None where a threshold or the draw comes too near to another token."""
    x = torch.nan_to_num(row.to(torch.float32) * (1 / torch.tensor(t, dtype=torch.float32)), nan=-float("inf"), posinf=float("inf"), neginf=-float("inf"))
    x = x.to(D)
    w = torch.exp(x - x.max())
    w = torch.where(w >= 2.0 ** -40, w, torch.zeros_like(w))
    V = x.numel()
    if 0 < k < V:
        w = torch.where(x >= x.topk(k).values[-1], w, torch.zeros_like(w))
    if tp < 1:
        order = torch.argsort(x, descending=True, stable=True)
        cum = w[order].cumsum(0) / w.sum()
        at = int((cum <= tp).sum())
        ties = (x[order] == x[order[min(at, V - 1)]]).nonzero()[:, 0]
        edges = torch.cat([cum[:1] * 0, cum])[[int(ties[0]), int(ties[-1]) + 1]]      # any of the values that tie brings them all
        if ((edges - tp).abs() < NEAR).any():
            return None
        w = torch.where(x >= x[order[min(at, V - 1)]], w, torch.zeros_like(w))
    if mp > 0:
        if ((w - mp).abs() < NEAR * mp).any() and mp < 1:
            return None
        w = torch.where(w >= mp, w, torch.zeros_like(w))
    cum = w.cumsum(0) / w.sum()
    token = int((cum <= u).sum())
    lo = float(cum[token - 1]) if token else 0.0
    if token >= V or (lo > 0 and abs(u - lo) < NEAR) or abs(u - float(cum[token])) < NEAR:
        return None
    return token


def draw(logits, t, k, tp, mp, u, logprob=False):
    R = logits.shape[0]
    f = lambda v, dt=torch.float32: torch.as_tensor(v, dtype=dt, device=DEV).expand(R).contiguous()
    token = torch.full((R + 1,), -7, dtype=torch.int32, device=DEV)
    lp = torch.empty(R, device=DEV) if logprob else None
    ops.sample(logits, f(t), f(k, torch.int32), f(tp), f(u), token, lp, min_p=f(mp))
    assert int(token[R]) == -7
    return (token[:R], lp) if logprob else token[:R]


@gpu
@pytest.mark.parametrize("V", [1, 2, 31, 1000, 1025, 2049, 5003, 16385, 151936, 420001])
@pytest.mark.parametrize("kind", ["normal", "ties", "peaked"])
def test_draws(V, kind):
    """420,001 numbers are more than the shared memory of eight blocks holds."""
    R = 5
    g = torch.Generator(device=DEV).manual_seed(V)
    logits = torch.randn(R, V, generator=g, device=DEV) * 3
    if kind == "ties":
        logits = (logits * 2).round() / 2
    if kind == "peaked":
        logits[:, :: max(1, V // 7)] += 9
    seen = 0
    for k, tp, mp in itertools.product((0, 1, 40, 3000), (1.0, 0.9, 0.2), (0.0, 0.01, 0.3, 1.0)):
        u = torch.rand(R, generator=g, device=DEV)
        got, lp = draw(logits, 0.8, k, tp, mp, u, logprob=True)
        assert (lp <= 0).all()
        for r in range(R):
            want = reference(logits[r], 0.8, k, tp, mp, float(u[r]))
            seen += want is not None
            assert want is None or int(got[r]) == want, (k, tp, mp, r)
    assert seen > 3 * 48 or V < 3


@gpu
@pytest.mark.parametrize("V", [342880, 342881, 343001, 420001, 1000003])
def test_rows_that_shared_memory_does_not_hold(V):
    """Slices longer than what a block holds, all logits far below zero, behind a launch that leaves large numbers in every block's shared memory: a number that is
    none of the row's would stand above its maximum."""
    R = 3
    g = torch.Generator(device=DEV).manual_seed(V)
    logits = torch.randn(R, V, generator=g, device=DEV) * 3 - 60
    big = torch.full((4096, 4096), 1e4, dtype=torch.bfloat16, device=DEV)
    seen = 0
    for k, tp, mp in itertools.product((0, 1, 40, 5000), (1.0, 0.9), (0.0, 0.05, 1.0)):
        u = torch.rand(R, generator=g, device=DEV)
        big @ big
        got, lp = draw(logits, 0.9, k, tp, mp, u, logprob=True)
        assert (lp <= 0).all() and (got >= 0).all() and (got < V).all()
        for r in range(R):
            want = reference(logits[r], 0.9, k, tp, mp, float(u[r]))
            seen += want is not None
            assert want is None or int(got[r]) == want, (k, tp, mp, r)
    assert seen > 24
    big @ big
    got, lp = draw(logits, 0.0, 0, 1.0, 0.0, 0.5, logprob=True)
    # masses are whole multiples of 2^-40 of the largest, rounded down, of exponentials that are off by 2^-22 of themselves
    want = torch.log_softmax(logits.to(D), dim=1).amax(dim=1)
    assert torch.equal(got.long(), logits.argmax(dim=1)) and ((lp.to(D) - want).abs() <= 2.0 ** -22 + V * 2.0 ** -40 + 2.0 ** -23 * want.abs()).all()


@gpu
def test_min_p_keeps_the_probable_ones():
    """Tokens at known probabilities relative to the first: kept up to the bound and at it, in every order with the other options; each can be drawn."""
    rel = torch.tensor([1.0, 0.5, 0.25, 0.125, 0.0625, 0.03125])
    logits = torch.full((1, 4000), -50.0)
    at = torch.tensor([3500, 17, 999, 2048, 2047, 3])
    logits[0, at] = torch.log(rel)
    logits = logits.to(DEV)
    for mp, n in ((0.0, 6), (0.03, 6), (0.04, 5), (0.06, 5), (0.2, 3), (0.3, 2), (0.51, 1), (1.0, 1)):
        seen = {int(draw(logits, 1.0, 0, 1.0, mp, u / 512)) for u in range(512)}
        assert seen == set(at[:n].tolist()), mp
        assert {int(draw(logits, 1.0, 2, 1.0, mp, u / 64)) for u in range(64)} == set(at[:min(n, 2)].tolist())
        assert {int(draw(logits, 1.0, 0, 0.85, mp, u / 512)) for u in range(512)} == set(at[:min(n, 3)].tolist())     # 0.51, 0.76, 0.89 of the mass
        assert {int(draw(logits, 0.5, 0, 1.0, mp ** 2, u / 2048)) for u in range(0, 2048)} == set(at[:n].tolist())    # probabilities squared
        assert int(draw(logits, 0.0, 0, 1.0, mp, 0.99)) == 3500


@gpu
@pytest.mark.parametrize("V", [5, 3000, 40000])
def test_rows_of_strange_numbers(V):
    inf, nan = float("inf"), float("nan")
    rows = torch.zeros(8, V, device=DEV)
    rows[1] = -inf
    rows[2], rows[2, 3] = -inf, 1.0
    rows[3, 4] = inf
    rows[4] = nan
    rows[5, 1:] = nan
    rows[6, ::2] = -0.0
    rows[7] = -inf
    rows[7, V // 2:] = 2.0
    for k, tp, mp in ((0, 1.0, 0.0), (2, 0.5, 0.1), (V - 1, 0.9, 1.0), (0, 0.3, 0.0)):
        for t in (0.0, 0.7):
            for u in (0.0, 0.5, 0.9999999):
                got = draw(rows, t, k, tp, mp, u).tolist()
                assert got[1] == 0 and got[2] == 3 and got[3] == 4 and got[4] == 0 and got[5] == 0, (k, tp, mp, t, u)
                assert V // 2 <= got[7] < V and all(0 <= x < V for x in got)
                if t == 0:
                    assert got[0] == 0 and got[6] == 0 and got[7] == V // 2
    # values that tie are kept together: every token of a flat row can be drawn, 0 and -0 alike
    assert {int(draw(rows[6:7, :5], 1.0, 2, 0.3, 1.0, u / 50)) for u in range(50)} == set(range(5))


@gpu
def test_a_row_alone_and_among_others():
    """Draws do not depend on who shares the launch, on the row's place in memory, or on how many blocks hold it."""
    R, V = 70, 30011
    g = torch.Generator(device=DEV).manual_seed(1)
    logits = torch.randn(R, V, generator=g, device=DEV) * 3
    t, u = 0.3 + torch.rand(R, generator=g, device=DEV), torch.rand(R, generator=g, device=DEV)
    t[::9] = 0
    k, tp, mp = torch.randint(0, 50, (R,), generator=g, device=DEV, dtype=torch.int32), 1 - 0.5 * torch.rand(R, generator=g, device=DEV), 0.2 * torch.rand(R, generator=g, device=DEV)
    together = torch.empty(R, dtype=torch.int32, device=DEV)
    ops.sample(logits, t, k, tp, u, together, min_p=mp)
    for r in range(0, R, 3):
        for pad in (0, 1, 2):                                # rows that begin on 16 bytes, 4 and 8
            buf = torch.empty(V + pad, device=DEV)
            buf[pad:] = logits[r]
            one = torch.empty(1, dtype=torch.int32, device=DEV)
            ops.sample(buf[pad:].view(1, V), t[r:r + 1], k[r:r + 1], tp[r:r + 1], u[r:r + 1], one, min_p=mp[r:r + 1])
            assert int(one) == int(together[r])
    # the same distribution in a longer row, whose other tokens have no mass
    longer = torch.full((R, 6 * V), -float("inf"), device=DEV)
    longer[:, :V] = logits
    again = torch.empty_like(together)
    ops.sample(longer, t, k, tp, u, again, min_p=mp)
    assert torch.equal(together, again)


@gpu
def test_captured_draws_follow_their_inputs():
    R, V = 3, 151936
    g = torch.Generator(device=DEV).manual_seed(2)
    logits, u = torch.randn(R, V, generator=g, device=DEV) * 3, torch.zeros(R, device=DEV)
    t, k, tp, mp = (torch.full((R,), x, device=DEV) for x in (0.9, 20, 0.9, 0.05))
    token = torch.empty(R, dtype=torch.int32, device=DEV)
    call = lambda: ops.sample(logits, t, k.int(), tp, u, token, min_p=mp)
    call()
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    k = k.int()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream), torch.cuda.graph(graph, stream=stream):
        ops.sample(logits, t, k, tp, u, token, min_p=mp)
    for x in (0.1, 0.6, 0.95):
        u.fill_(x)
        graph.replay()
        torch.cuda.synchronize()
        for r in range(R):
            want = reference(logits[r], 0.9, 20, 0.9, 0.05, float(u[r]))
            assert want is None or int(token[r]) == want


@gpu
def test_refusals():
    logits, R = torch.zeros(4, 10, device=DEV), 4
    token = torch.full((4,), 9, dtype=torch.int32, device=DEV)
    ones = torch.ones(4, device=DEV)
    for bad in (dict(min_p=ones.double()), dict(min_p=ones[:3]), dict(min_p=ones.cpu()), dict(top_p=ones[:2]), dict(out_token=token[:3]), dict(logits=logits[:, ::2]),
                dict(logits=logits.half()), dict(logits=logits[:, :0].contiguous())):
        with pytest.raises(ops.KernelError):
            ops.sample(**{**dict(logits=logits, temperature=ones, top_k=None, top_p=None, uniform=ones * 0.5, out_token=token, min_p=None), **bad})
    assert (token == 9).all()


def test_parameters():
    assert SamplingParams(min_p=0.3).validate().min_p == 0.3 and SamplingParams().min_p == 0.0 and SamplingParams(min_p=1).validate()
    for bad in (-0.1, 1.1, float("nan")):
        with pytest.raises(ValueError):
            SamplingParams(min_p=bad).validate()
