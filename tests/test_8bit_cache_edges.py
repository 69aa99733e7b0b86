"""A cache in 8 bits at its edges: who may write what a launch reads, and when; tokens between others that are not written; pages whose sizes lie far apart;
numbers that are none.  Checks and tolerances are those of tests/test_8bit_cache.py."""
from types import SimpleNamespace

import pytest
import torch

from test_8bit_cache import Cache, D, DEV, batch, check_attention, queries, tiles_of
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
