"""A cache in 8 bits at its edges: who may write what a launch reads, and when; tokens between others that are not written; pages whose sizes lie far apart;
numbers that are none.  Checks and tolerances are those of tests/test_8bit_cache.py."""
from types import SimpleNamespace

import pytest
import torch

from test_8bit_cache import Cache, D, DEV, batch, check_attention, copies, least_scale, queries, tiles_of, turned_heads
from vllm_lite_b200.csrc import ops

gpu = pytest.mark.gpu


# ---------------------------------------------------------------------------------------------- who brings the step's description
@pytest.fixture
def dependent_launches():
    was = ops._pdl
    ops.set_pdl(True)
    yield
    ops.set_pdl(was)


@gpu
@pytest.mark.parametrize("before,new", [([300, 40], [100, 200]), ([1900, 700], [3, 40]), ([0, 20], [1500, 1000])])
def test_tiles_and_table_that_a_kernel_writes(dependent_launches, before, new):
    """Behind a kernel of this library, itself behind a long one, both of which let the next one start at once: the attention waits for what they write (the pages of
    another request stand in the table until then)."""
    nq, nkv, hd, ps = 8, 2, 64, 64
    lengths = [b + n for b, n in zip(before, new)]
    cache = Cache(2, max(lengths), nkv, ps, hd, seed=1).fill([max(lengths)] * 2, seed=3)
    pos, req, _, _ = batch(cache, before, new)
    q, tiles = queries(sum(new), nq, hd, 8), tiles_of(before, new)
    out = torch.full((sum(new), nq * hd), 3.0, dtype=torch.bfloat16, device=DEV)
    late_table, late_tiles = cache.table.flip(0).contiguous(), torch.zeros_like(tiles)
    ids = lambda n: torch.arange(n, dtype=torch.int32, device=DEV)
    first, rows, items = torch.zeros(1, dtype=torch.int32, device=DEV), ids(2), ids(tiles.shape[0])
    wide = torch.ones(1, (1 << 22) + 1, device=DEV)                                # (a row of such a width is one block's)
    long_out = torch.empty_like(wide)
    as_floats = lambda t: t.view(torch.float32)                                    # (rows of numbers times one keep their bits)
    scratch = torch.empty(ops.flash_prefill_8bit_scratch(hd, DEV), device=DEV)
    torch.cuda.synchronize()
    ops.embed(first, wide, long_out, cache.err)
    ops.embed(rows, as_floats(cache.table), as_floats(late_table), cache.err)
    ops.embed(items, as_floats(tiles), as_floats(late_tiles), cache.err)
    ops.flash_prefill_8bit(q, out, *cache.tensors, late_table, late_tiles, nq, nkv, hd, hd ** -0.5, None, cache.err, scratch=scratch)
    assert torch.equal(late_table, cache.table) and torch.equal(late_tiles, tiles) and int(cache.err) == 0
    only = sorted({0, 1, new[0] - 1, new[0], sum(new) // 2, sum(new) - 1})
    check_attention(cache, q, out, pos, req, nq, None, hd ** -0.5, only)
    again = torch.full_like(out, 3.0)                                              # what is there already: the same results, to the bit
    torch.cuda.synchronize()
    ops.flash_prefill_8bit(q, again, *cache.tensors, late_table, late_tiles, nq, nkv, hd, hd ** -0.5, None, cache.err, scratch=scratch, settled=True)
    assert torch.equal(again, out)


@pytest.mark.parametrize("settled", [True, False, None])
def test_a_step_says_who_brought_its_description(monkeypatch, settled):
    from vllm_lite_b200.parts import attention_dispatch
    from vllm_lite_b200.parts.base import StepBatch
    said = []
    monkeypatch.setattr(ops, "flash_prefill_8bit_scratch", lambda *a: 8)
    monkeypatch.setattr(ops, "flash_prefill_8bit", lambda *a, **k: said.append(k["settled"]))
    monkeypatch.setattr(ops, "flash_decode_8bit", lambda *a, **k: said.append(k["settled"]))
    workspace = SimpleNamespace(get=lambda name, shape, dtype: torch.empty(shape, dtype=dtype), zeros=lambda name, n, dtype: torch.zeros(n, dtype=dtype))
    step = SimpleNamespace(workspace=workspace, tag="", err=None, query_tiles=None, max_query_len=7, single_tokens=torch.zeros(2, dtype=torch.int32), single_context=9,
                           req_index=None, positions=None)
    if settled is not None:
        step.settled = settled
    spec = SimpleNamespace(num_heads=4, num_kv_heads=2, head_dim=64, window=None)
    cache = SimpleNamespace(k=None, v=None, k_scale=None, v_scale=None)
    attention_dispatch.run_8bit(torch.zeros(9, 512), None, cache, SimpleNamespace(block_table=None, max_context=9), step, spec, 0.1)
    assert said == [bool(settled)] * 2 and "settled" in StepBatch.__dataclass_fields__


# ---------------------------------------------------------------------------------------------- tokens that are not written, among others that are
def check_rows(cache, was, x, slots, req, pos, which):
    """Keys or values x [T, nkv, hd], in 64 bits and off by `slack` of a head's largest, against what the cache holds: a row that is written, under the least power
    of two for the rows written and, unless row 0 is among them, the one the page had; other rows of a page up to its request's last token
    as they were, unless the page begins anew."""
    ps, slots = cache.ps, slots.tolist()
    now, before, scale, scale_before = (cache.k, was[0], cache.k_scale, was[2]) if which == "k" else (cache.v, was[1], cache.v_scale, was[3])
    pages = {}
    for t, s in enumerate(slots):                                                  # (a page that no token of its request goes to is not touched)
        if s >= 0:
            pages.setdefault(s // ps, {})[s % ps] = t
    reach = {}
    for t in range(len(slots)):
        page = int(cache.table[int(req[t]), int(pos[t]) // ps])
        reach[page] = max(reach.get(page, 0), int(pos[t]) % ps + 1)
    for page in range(now.shape[0]):
        rows = pages.get(page, {})
        same = lambda a, b: torch.equal(a.view(torch.uint8), b.view(torch.uint8))
        if not rows:
            assert same(now[page], before[page]) and torch.equal(scale.view(torch.int32)[page], scale_before.view(torch.int32)[page])
            continue
        for h in range(cache.nkv):
            new = torch.stack([x[t, h] for t in rows.values()])
            old = 0.0 if 0 in rows else float(scale_before[page, h])
            s, top = float(scale[page, h]), float(new.abs().max())
            assert max(old, least_scale(top * (1 - 2.0 ** -18))) <= s <= max(old, least_scale(top * (1 + 2.0 ** -18)))
            for r in range(ps):
                got = now[page, h, r].to(D) * s
                if r in rows:
                    want = x[rows[r], h]
                    assert ((got - want).abs() <= torch.maximum(2.0 ** -4 * want.abs(), torch.tensor(2.0 ** -10 * s, dtype=D, device=DEV)) * (1 + 2.0 ** -10)
                            + 2.0 ** -18 * top).all(), (page, h, r)
                elif 0 in rows or r >= reach[page]:
                    assert same(now[page, h, r], before[page, h, r]), (page, h, r)
                else:
                    assert ((got - before[page, h, r].to(D) * old).abs() <= (2.0 ** -10 * s if s > old else 0.0)).all(), (page, h, r)


@gpu
@pytest.mark.parametrize("hd,ps,rot,before,new", [
    (128, 64, 128, [30, 0, 64, 10], [200, 70, 10, 1]), (128, 16, 0, [5, 0, 16], [40, 33, 3]), (256, 100, 256, [20], [300]), (32, 256, 32, [100, 0], [300, 20]),
    (80, 16, 80, [3, 0], [40, 20]), (128, 64, 64, [10, 64], [150, 30]), (144, 200, 0, [30], [100]),
    (64, 16, 64, [9, 0, 20], [3, 0, 0]), (80, 8, 80, [3, 0, 5, 16, 0, 0], [1, 1, 4, 0, 0, 0]), (256, 16, 0, [7] + [0] * 39, [40] + [0] * 39), (128, 64, 128, [5, 64, 0, 9], [1] * 4)])
@pytest.mark.parametrize("pattern", ["first", "last alone", "every third", "half", "all but one page"])
def test_some_tokens_are_not_written(hd, ps, rot, before, new, pattern):
    nq, nkv = 4, 2
    longest = max(b + n for b, n in zip(before, new))
    cache = Cache(len(new), longest, nkv, ps, hd, seed=2)
    whole = cache.table.clone()
    cache.fill([longest] * len(new), seed=hd, spread=6).table = whole              # pages that hold rows of older tokens all over
    pos, req, cu, slots = batch(cache, before, new)
    T = sum(new)
    g = torch.Generator(device=DEV).manual_seed(hd + ps)
    at = torch.arange(T, device=DEV) - cu[req.long()]
    count = (cu[1:] - cu[:-1])[req.long()]
    drop = {"first": at == 0, "last alone": at < count - 1, "every third": (at + req) % 3 == 0, "half": torch.rand(T, generator=g, device=DEV) < 0.5,
            "all but one page": pos // ps != before[0] // ps}[pattern]
    slots = torch.where(drop, torch.full_like(slots, -1), slots)
    qkv = (torch.randn(T, (nq + 2 * nkv) * hd, generator=g, device=DEV) * torch.exp2(4 * torch.randn(T, 1, generator=g, device=DEV))).to(torch.bfloat16)
    inv_freq = (1e6 ** (-torch.arange(0, rot, 2, dtype=D, device=DEV) / max(rot, 1))).float() if rot else None
    was, rows = copies(cache), qkv.view(T, nq + 2 * nkv, hd)
    q = torch.full((T, nq * hd), 3.0, dtype=torch.bfloat16, device=DEV)
    ops.qk_norm_rope_write_8bit(qkv, pos, slots, cu, None, None, 1e-6, inv_freq, rot, *cache.tensors, nq, nkv, hd, cache.err, q_out=q)
    assert int(cache.err) == 0
    turned = turned_heads(rows[:, :nq + nkv], None, pos, inv_freq, rot)
    want = turned[:, :nq]
    assert ((q.to(D).view(T, nq, hd) - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -18 * want.abs().amax(dim=2, keepdim=True)).all()
    check_rows(cache, was, turned[:, nq:], slots, req, pos, "k")
    check_rows(cache, was, rows[:, nq + nkv:].to(D), slots, req, pos, "v")


@gpu
@pytest.mark.parametrize("hd,ps", [(128, 64), (80, 16)])
@pytest.mark.parametrize("new", [[20], [5, 0, 0, 0, 0]])
def test_slots_of_another_row_behind_tokens_that_are_not_written(hd, ps, new):
    """The first slot of a page that is one says where the page is: flagged where it is another row's, below the pool's first or beyond its last."""
    nkv = 2
    cache = Cache(len(new), 32, nkv, ps, hd).fill([32] * len(new))
    pos, req, cu, slots = batch(cache, [3] * len(new), new)
    was = copies(cache)
    qkv = torch.ones(sum(new), 3 * nkv * hd, dtype=torch.bfloat16, device=DEV)
    for third in (1, 2, int(slots[2]) + 1, cache.k.shape[0] * ps + 5, (1 << 31) - 1):
        cache.err.zero_()
        bad = slots.clone()
        bad[:2], bad[2], bad[3:] = -1, third, -5
        ops.qk_norm_rope_write_8bit(qkv, pos, bad, cu, None, None, 1e-6, None, 0, *cache.tensors, nkv, nkv, hd, cache.err)
        assert int(cache.err) == 2 and all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(cache.tensors, was)), third


# ---------------------------------------------------------------------------------------------- pages whose sizes lie far apart
def far_apart(cache, lengths, small, bits, which):
    """Makes the pages `small` (numbers within a request) of every request 2^bits smaller."""
    for name in which:
        scale = getattr(cache, name)
        for r, n in enumerate(lengths):
            for b in range(-(-n // cache.ps)):
                if b in small:
                    scale[int(cache.table[r, b])] *= 2.0 ** -bits


@gpu
@pytest.mark.parametrize("nq,nkv,hd", [(8, 2, 128), (4, 4, 16), (6, 1, 48), (5, 1, 256), (2, 1, 80), (130, 1, 32)])
@pytest.mark.parametrize("bits", [22, 23, 33, 45, 80])
@pytest.mark.parametrize("which", [("k_scale",), ("v_scale",), ("k_scale", "v_scale")])
def test_rows_that_read_small_pages_alone(nq, nkv, hd, bits, which):
    """A prompt whose first two pages are far smaller than its later ones: the tokens of the first two read no other, and get what single tokens get.  (Their
    queries are as much larger as their keys are smaller, so that their scores are ordinary ones.)"""
    ps, n = 32, 128
    cache = Cache(2, n, nkv, ps, hd, seed=1).fill([n, n], seed=hd, spread=1)
    far_apart(cache, [n, n], (0, 1), bits, which)
    pos, req, _, _ = batch(cache, [0, 0], [n, n])
    q = queries(2 * n, nq, hd, 8)
    if "k_scale" in which:
        q = torch.where((pos < 2 * ps)[:, None], q * 2.0 ** bits, q)
    out = torch.full((2 * n, nq * hd), 3.0, dtype=torch.bfloat16, device=DEV)
    sizes = (nq, nkv, hd, hd ** -0.5, None)
    early = [0, 1, 2, 30, 31, 32, 33, 63, 128, 150, 191]
    ops.flash_prefill_8bit(q, out, *cache.tensors, cache.table, tiles_of([0, 0], [n, n]), *sizes, cache.err)
    assert int(cache.err) == 0
    check_attention(cache, q, out, pos, req, nq, None, hd ** -0.5, early)
    if "k_scale" not in which:                                                     # (else the larger keys' scores leave a later row nothing to be off by)
        check_attention(cache, q, out, pos, req, nq, None, hd ** -0.5, [64, 65, 127, 192, 255])
    assert torch.isfinite(out).all()
    alone = torch.full_like(out, 3.0)
    ops.flash_decode_8bit(q, alone, *cache.tensors, cache.table, req, pos, *sizes, n, cache.err)
    check_attention(cache, q, alone, pos, req, nq, None, hd ** -0.5, early)


@gpu
@pytest.mark.parametrize("nq,nkv,hd,ps", [(4, 2, 64, 64), (3, 1, 144, 16), (4, 1, 128, 40), (2, 2, 32, 7)])
@pytest.mark.parametrize("before,new", [([1500, 300], [90, 20]), ([0, 900], [700, 256])])
@pytest.mark.parametrize("bits", [25, 50])
def test_windows_that_leave_large_pages_behind(nq, nkv, hd, ps, before, new, bits):
    """Every fourth stretch of 256 tokens is large, and a window of 150 reads it from some tokens alone; keys shared out among blocks and whole."""
    lengths, window = [b + n for b, n in zip(before, new)], 150
    cache = Cache(2, max(lengths), nkv, ps, hd, seed=1).fill(lengths, seed=hd, spread=1)
    small = [b for b in range(-(-max(lengths) // ps)) if b * ps // 256 % 4 != 1]
    far_apart(cache, lengths, small, bits, ("v_scale",))
    pos, req, _, _ = batch(cache, before, new)
    q, out = queries(sum(new), nq, hd, 8), torch.full((sum(new), nq * hd), 3.0, dtype=torch.bfloat16, device=DEV)
    ops.flash_prefill_8bit(q, out, *cache.tensors, cache.table, tiles_of(before, new), nq, nkv, hd, hd ** -0.5, window, cache.err)
    assert int(cache.err) == 0
    check_attention(cache, q, out, pos, req, nq, window, hd ** -0.5, sorted(set(range(0, sum(new), 13)) | {new[0] - 1, new[0], sum(new) - 1}))


@gpu
def test_few_tokens_behind_pages_far_apart():
    """Shares of one item's keys, some of which hold pages far apart and some not."""
    nq, nkv, hd, ps, before, new = 8, 2, 128, 64, [1900, 700], [5, 3]
    lengths = [b + n for b, n in zip(before, new)]
    cache = Cache(2, max(lengths), nkv, ps, hd, seed=1).fill(lengths, seed=3, spread=1)
    far_apart(cache, lengths, (3, 9, 10, 29), 40, ("v_scale",))
    far_apart(cache, lengths, (5, 10, 28), 40, ("k_scale",))
    pos, req, _, _ = batch(cache, before, new)
    q, out = queries(8, nq, hd, 8), torch.full((8, nq * hd), 3.0, dtype=torch.bfloat16, device=DEV)
    ops.flash_prefill_8bit(q, out, *cache.tensors, cache.table, tiles_of(before, new), nq, nkv, hd, hd ** -0.5, None, cache.err)
    assert int(cache.err) == 0
    check_attention(cache, q, out, pos, req, nq, None, hd ** -0.5)


@gpu
def test_lost_and_missing_pages_among_pages_far_apart():
    """What a page's scale that is none, and a page that the table does not hold, do elsewhere, they do here."""
    nq, nkv, hd, ps, n = 4, 2, 64, 32, 256
    cache = Cache(1, n, nkv, ps, hd).fill([n], spread=1)
    far_apart(cache, [n], (0, 1), 40, ("v_scale",))
    pos, req = torch.arange(n, dtype=torch.int32, device=DEV), torch.zeros(n, dtype=torch.int32, device=DEV)
    q = queries(n, nq, hd, 3)
    for which in ("k_scale", "v_scale"):
        scale = getattr(cache, which)
        kept = scale.clone()
        scale[int(cache.table[0, 1]), 1] = float("nan")
        for window in (None, 40):
            out = ops.flash_prefill_8bit(q, torch.full_like(q, 3.0), *cache.tensors, cache.table, tiles_of([0], [n]), nq, nkv, hd, hd ** -0.5, window, cache.err)
            nan = torch.isnan(out.view(n, nkv, -1))
            reads = (pos >= ps) & ((pos - window + 1 < 2 * ps) if window else torch.ones_like(pos, dtype=torch.bool))
            assert not nan[:, 0].any() and torch.equal(nan[:, 1].all(dim=1), reads) and torch.equal(nan[:, 1].any(dim=1), reads)
        scale.copy_(kept)
    assert int(cache.err) == 0
    for bad in (-1, cache.k.shape[0]):
        table = cache.table.clone()
        table[0, 2] = bad
        cache.err.zero_()
        out = ops.flash_prefill_8bit(q, torch.full_like(q, 3.0), *cache.tensors, table, tiles_of([0], [n]), nq, nkv, hd, hd ** -0.5, None, cache.err)
        assert int(cache.err) == 4 and torch.isfinite(out).all()
        check_attention(cache, q, out, pos, req, nq, None, hd ** -0.5, [0, 31, 63])


# ---------------------------------------------------------------------------------------------- the largest sizes
@pytest.mark.parametrize("T,bound,code", [(1, (1 << 31) - 1, -2), (1, (1 << 31) - 128, -2), (1, (1 << 30) + 1, -2), (64, (1 << 31) - 1, -2), (200, 1 << 30, -2)])
def test_bounds_beyond_the_largest_are_refused_before_any_launch(T, bound, code):
    host = torch.zeros(64)                                   # never read or written
    at = -host.data_ptr() % 16 + host.data_ptr()
    got = ops._fn("flash_decode_8bit", "vl_flash_decode_8bit", {"FA_HD": 128})(
        at, 256, at, at, at, at, at, 2, at, at, T, 2, 1, 128, 64, 4, 0.1, 0, bound, at, 3 * T * 2 * 130, None, None, at, at, 0, 0)
    assert got == code


@gpu
def test_windows_wider_than_any_context():
    """The widest window that is a number, and no window, are one thing: the same results, to the bit, however keys are shared out."""
    nq, nkv, hd, ps, n = 8, 2, 128, 64, 3000
    cache = Cache(2, n, nkv, ps, hd, seed=1).fill([n, 1000], seed=3)
    q = queries(5, nq, hd, 8)
    pos, req, _, _ = batch(cache, [n - 4, 999], [4, 1])
    results = {}
    for window in (None, (1 << 31) - 1, (1 << 31) - 100, 1 << 30):
        prompt, single = torch.full_like(q, 3.0), torch.full_like(q, 3.0)
        ops.flash_prefill_8bit(q, prompt, *cache.tensors, cache.table, tiles_of([n - 4, 999], [4, 1]), nq, nkv, hd, hd ** -0.5, window, cache.err)
        ops.flash_decode_8bit(q, single, *cache.tensors, cache.table, req, pos, nq, nkv, hd, hd ** -0.5, window, n, cache.err)
        results[window] = (prompt, single)
    assert int(cache.err) == 0
    check_attention(cache, q, results[None][0], pos, req, nq, None, hd ** -0.5)
    assert all(torch.equal(a, b) for r in results.values() for a, b in zip(r, results[None]))


@gpu
def test_a_bound_as_large_as_it_may_be():
    nq, nkv, hd, ps = 8, 2, 128, 64
    cache = Cache(2, 500, nkv, ps, hd, seed=1).fill([500, 40], seed=3)
    q, out = queries(2, nq, hd, 8), torch.full((2, nq * hd), 3.0, dtype=torch.bfloat16, device=DEV)
    pos, req, _, _ = batch(cache, [499, 39], [1, 1])
    ops.flash_decode_8bit(q, out, *cache.tensors, cache.table, req, pos, nq, nkv, hd, hd ** -0.5, None, 1 << 30, cache.err)
    check_attention(cache, q, out, pos, req, nq, None, hd ** -0.5)
    with pytest.raises(ops.KernelError):
        ops.flash_decode_8bit(q, out, *cache.tensors, cache.table, req, pos, nq, nkv, hd, hd ** -0.5, None, (1 << 30) + 1, cache.err)
    assert int(cache.err) == 0


# ---------------------------------------------------------------------------------------------- queries that are no numbers
@gpu
@pytest.mark.parametrize("nq,nkv,hd", [(4, 2, 64), (8, 1, 128), (3, 3, 48), (2, 1, 256)])
@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), float("nan")])
@pytest.mark.parametrize("before,window,far", [(0, None, False), (0, 20, False), (1500, None, False), (0, None, True)])
def test_a_query_that_holds_an_infinity(nq, nkv, hd, bad, before, window, far):
    """All scores of such a head are infinite or none, and a softmax of them is none, also where every one of them is minus infinity (keys of positive numbers alone);
    nobody else's result changes."""
    ps, n = 32, 70
    cache = Cache(1, before + n, nkv, ps, hd).fill([before + n], spread=1)
    cache.k.view(torch.uint8).bitwise_and_(0x7f)
    if far:
        far_apart(cache, [before + n], (0,), 40, ("v_scale",))
    pos, req, _, _ = batch(cache, [before], [n])
    q = queries(n, nq, hd, 3)
    q.view(n, nq, hd)[33, nq - 1, 7] = bad
    q.view(n, nq, hd)[0, 0, 9] = bad
    want = torch.zeros(n, nq, dtype=torch.bool, device=DEV)
    want[33, nq - 1] = want[0, 0] = True
    prompt, single = torch.full_like(q, 3.0), torch.full_like(q, 3.0)
    ops.flash_prefill_8bit(q, prompt, *cache.tensors, cache.table, tiles_of([before], [n]), nq, nkv, hd, hd ** -0.5, window, cache.err)
    ops.flash_decode_8bit(q, single, *cache.tensors, cache.table, req, pos, nq, nkv, hd, hd ** -0.5, window, before + n, cache.err)
    assert int(cache.err) == 0
    for out in (prompt, single):
        nan = torch.isnan(out.view(n, nq, hd))
        assert torch.equal(nan.all(dim=2), want) and torch.equal(nan.any(dim=2), want)
    check_attention(cache, q, prompt, pos, req, nq, window, hd ** -0.5, [1, 2, 31, 32, 34, 69])
