"""Linear layers in 8 bits: rows too long for a block's registers, operands off the 16-byte boundaries, a layer with a bias, and steps of a model
whose products run on pairs of SMs or whose weights are stored in float32.  Tolerances as in test_8bit.py; the sum of squares of a long row has up to 33 terms a thread and 10 steps of
joining, 1.3e-6 of the norm at worst, within the 2e-6 that a scale is given there."""
from types import SimpleNamespace

import pytest
import torch

from test_8bit import (DEV, JOINED, LOW, PAIRED, check_product, check_rows, columns, dependent, empty_rows, norm_of, normal,  # noqa: F401
                       operands, run_product)
from vllm_lite_b200.csrc import ops

gpu = pytest.mark.gpu

# 16,390 columns are no multiple of eight (registers hold 16,384 of such rows), 33,000 are (32,768)
LONG = [(2, 16390), (3, 33000)]


@gpu
@pytest.mark.parametrize("elsewhere", [False, True])
@pytest.mark.parametrize("delta", [None, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("r,h", LONG)
def test_norms_of_long_rows(r, h, delta, elsewhere):
    x, w = normal(1, r, h, std=2.0), 1 + normal(2, h, std=0.3)
    x[:, :h // 100] *= 20
    d = None if delta is None else normal(3, r, h).to(delta)
    xg, out, scale = x.to(DEV), *empty_rows(r, h)
    into = torch.full_like(xg, 7.0) if elsewhere else None
    ops.add_rmsnorm_8bit(xg, None if d is None else d.to(DEV), w.to(DEV), 1e-6, out, scale, into=into)
    new = x if d is None else x + d.float()
    assert torch.equal(xg.cpu(), x if elsewhere else new)
    if elsewhere:
        assert torch.equal(into.cpu(), torch.full_like(x, 7.0) if d is None else new)
    check_rows(norm_of(new, w, 1e-6), out, scale, columns(h))


@gpu
@pytest.mark.parametrize("with_delta", [False, True])
@pytest.mark.parametrize("r,h", LONG)
def test_norms_of_picked_long_rows(r, h, with_delta):
    x, w, d = normal(4, r, h), 1 + normal(5, h, std=0.3), normal(6, r, h).bfloat16()
    pick = torch.tensor([r - 1, 0, 1, 1], dtype=torch.int32)
    xg, out, scale = x.to(DEV), *empty_rows(4, h)
    into = torch.full_like(xg, 7.0)
    ops.add_rmsnorm_8bit(xg, d.to(DEV) if with_delta else None, w.to(DEV), 1e-5, out, scale, rows=pick.to(DEV), into=into)
    assert torch.equal(xg.cpu(), x) and (into == 7).all()
    check_rows(norm_of((x + d.float() if with_delta else x)[pick.long()], w, 1e-5), out, scale, columns(h))


@gpu
@pytest.mark.parametrize("dtype,k,shift", [(torch.bfloat16, 16390, 0), (torch.bfloat16, 16400, 1), (torch.float32, 16390, 0), (torch.float32, 33000, 0),
                                           (torch.bfloat16, 33000, 0), (torch.bfloat16, 65537, 0)])
def test_long_rows(dtype, k, shift):
    x = normal(9, 2, k, std=0.02).to(dtype)
    flat = torch.zeros(2 * k + shift, dtype=dtype, device=DEV)
    xg = flat[shift:].view(2, k)
    xg.copy_(x)
    out, scale = empty_rows(2, k)
    ops.rows_8bit(xg, out, scale)
    check_rows(x.double(), out, scale, columns(k))


def shifted(t):
    """The same values in a contiguous tensor that begins one element behind a 16-byte boundary."""
    flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
    view = flat[1:].view(t.shape)
    view.copy_(t)
    assert view.data_ptr() % 16 == t.element_size()
    return view


@gpu
@pytest.mark.parametrize("which", ["a_scale", "w_scale", "bias", "residual", "out"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("m,n,k", [(5, 528, 1000), (16, 528, 1000), (40, 528, 256), JOINED[0], PAIRED[0]])
def test_a_product_of_operands_off_sixteen_bytes(m, n, k, gated, dtype, which):
    """Everything but the rows and the weights may begin anywhere."""
    a, sa, w, sw = operands(47, m, n, k)
    width = n // 2 if gated else n
    t = dict(a_scale=sa, w_scale=sw, bias=normal(48, n).to(DEV), residual=normal(49, m, width).to(DEV, dtype), out=torch.empty(m, width, device=DEV, dtype=dtype))
    p, how = ops.pack_8bit(w), dict(act="silu", gated=gated)
    want = ops.gemm_8bit(a, w=p, **t, **how).clone()
    t[which] = shifted(t[which])
    t["out"].fill_(float("nan"))
    assert torch.equal(ops.gemm_8bit(a, w=p, **t, **how), want)


@gpu
@pytest.mark.parametrize("m", [3, 20, 130])
def test_a_layer_with_a_bias(m):
    from vllm_lite_b200.parts.base import BuildContext, Workspace
    from vllm_lite_b200.parts.eight_bit import Linear8
    from vllm_lite_b200.parts.linear import Linear
    weight, bias = normal(50, 200, 300, std=0.1).to(DEV, torch.bfloat16), normal(51, 200).to(DEV, torch.bfloat16)
    layer = Linear8(Linear(weight, bias), BuildContext(torch.device(DEV), torch.bfloat16))
    step = SimpleNamespace(workspace=Workspace(torch.device(DEV)), tag="", err=None)
    x = normal(52, m, 300).to(DEV, torch.bfloat16)
    (a, sa), (w, sw) = empty_rows(m, 300), empty_rows(200, 300)
    ops.rows_8bit(x, a, sa)
    ops.rows_8bit(weight, w, sw)
    check_product(layer(x, step, "y"), a, sa, w, sw, bias.float())
    stream = normal(53, m, 200).to(DEV)
    got = stream.clone()
    layer.into_stream(x, got, step, "z")
    check_product(got, a, sa, w, sw, bias.float(), residual=stream)


WIDE = dict(architectures=["Qwen3ForCausalLM"], model_type="qwen3", hidden_size=512, num_hidden_layers=2, num_attention_heads=8,
            num_key_value_heads=4, head_dim=64, intermediate_size=2048, vocab_size=200, rope_theta=10000.0, rms_norm_eps=1e-6,
            tie_word_embeddings=False, max_position_embeddings=2048)


def wide_runner(**kw):
    from vllm_lite_b200.engine import ModelRunner, plan_in_8_bits, random_model
    _, plan, weights = random_model(WIDE, seed=5, dtype="bfloat16", device=DEV, std=0.04)
    gate, up = (weights[f"model.layers.1.mlp.{n}_proj.weight"].clone() for n in ("gate", "up"))
    runner = ModelRunner(plan_in_8_bits(plan, "bfloat16"), weights, dtype=torch.bfloat16, device=DEV, page_size=64, max_context=2048, **kw)
    order = torch.arange(4096, device=DEV).view(2, 256, 8).transpose(0, 1).reshape(-1)      # eight gates, their eight ups
    w, sw = empty_rows(4096, 512)
    ops.rows_8bit(torch.cat([gate, up])[order].contiguous(), w, sw)
    return runner, w, sw


def check_gate_up(runner, w, sw, tag, m):
    """The last layer's product of pairs of SMs, from the values that the engine left in its buffers."""
    left = {key[0]: b for key, b in runner.workspace._buffers.items()}
    a, sa = left[tag + "norm2.8"][:m * 512].view(m, 512), left[tag + "norm2.scale"][:m]
    check_product(left[tag + "mlp.gate_up.act"][:m * 2048].view(m, 2048), a, sa, w, sw, act="silu", gated=True)


@gpu
def test_a_prompt_whose_products_run_on_pairs_of_sms():
    from vllm_lite_b200.engine import StepEntry
    runner, w, sw = wide_runner(num_pages=40, max_requests=4)
    assert runner.model.clusters(1500) and ops.gemm_8bit_plan(1500, 4096, 512)[1]
    tokens = [(7 * i + 3) % 200 for i in range(1500)]
    runner.step([StepEntry("a", tokens, [1499])])
    runner.check_device_errors()
    assert not ops._pdl
    check_gate_up(runner, w, sw, "", 1500)


@gpu
def test_a_recorded_step_whose_products_run_on_pairs_of_sms():
    """1,200 requests of one token: a bucket of 2,048, recorded and then replayed with the same tokens."""
    from vllm_lite_b200.engine import StepEntry
    runner, w, sw = wide_runner(num_pages=1300, max_requests=1200)
    assert runner.model.clusters(2048)
    entries = [StepEntry(i, [i % 200], [0]) for i in range(1200)]
    first = runner.step(entries).clone()
    runner.check_device_errors()
    assert not ops._pdl and runner.graph_replays == 0
    for e in entries:
        runner.release(e.request_id)
    again = runner.step(entries)
    runner.check_device_errors()
    assert runner.graph_replays == 1 and torch.equal(again, first)
    check_gate_up(runner, w, sw, "g2048.1024.", 2048)


MIDDLE = [(64, 30000, 2048), (40, 29001, 2100)]              # tiles of 112 rows of w


def test_the_sizes_reach_low_tiles():
    for sizes, height in ((LOW, 96), (MIDDLE, 112), (PAIRED, 256), (JOINED, 128), ([(16, 20000, 2048)], 0)):
        for m, n, k in sizes:
            assert [ops.gemm_8bit_tile(m, n, columns(k), overlapped) for overlapped in (False, True)] == [height, height]
    with pytest.raises(ops.KernelError):
        ops.gemm_8bit_tile(64, 4096, 100)


@gpu
@pytest.mark.parametrize("m,n,k", MIDDLE)
def test_tiles_of_112_rows(m, n, k, dependent):
    run_product(m, n, k, dict(bias=True, act="silu", residual=True))
    run_product(m, n, k, dict(bias=True), torch.bfloat16)
    if n % 16 == 0:
        run_product(m, n, k, dict(gated=True, act="silu", residual=True, bias=True))
        run_product(m, n, k, dict(gated=True, act="silu"), torch.bfloat16)


@gpu
def test_a_model_stored_in_float32():
    """Its weights reach 8 bits from float32 rows; error bound of whole rows as in test_8bit_model.py."""
    import helpers as H
    from test_8bit_model import TOL_RMS
    from vllm_lite_b200.engine import ModelRunner, StepEntry, load_model_dir
    _, plan, weights = load_model_dir(H.model_dir("B", "float32"), "bfloat16", DEV, eight_bit=True)
    assert weights["model.layers.0.mlp.down_proj.weight"].dtype == torch.float32
    runner = ModelRunner(plan, weights, dtype=torch.bfloat16, device=DEV, page_size=8, num_pages=32, max_requests=4)
    tokens = H.tokens_for("B", 40, 9)
    rows = [runner.step([StepEntry("a", tokens[:30], [0, 29])]).float().cpu(), runner.step([StepEntry("a", tokens[30:], [9])]).float().cpu()]
    runner.check_device_errors()
    want = H.plain_logits("B", tokens, "float32")[[0, 29, 39]]
    got = torch.cat(rows)
    assert ((got - want).norm(dim=1) <= TOL_RMS * want.norm(dim=1)).all()
