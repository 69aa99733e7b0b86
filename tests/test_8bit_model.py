"""A model whose linear layers run in 8 bits.

Stage by stage, from the values that the engine itself left in its buffers: each product, norm and rounding to 8 bits of a one-layer model against
its definition in 64 bits, with the tolerances of tests/test_8bit.py.

As a whole, against the plain implementation without any rounding: the error of all logits of a row, as a root of mean squares, over the logits'
own.  A rounding to 8 bits is off by up to 2^-4 of a value, uniformly, which is 2.6e-2 as a root of mean squares; weights and inputs, 3.7e-2 a product; four
products in a row in each of three layers, if nothing of the stream but their results were left: 12.8e-2, and the bfloat16 engine's
error beside it.  (Values cannot be compared one by one with a reference that rounds in the same places: a difference of e in front of a rounding with steps
of d comes out of it as sqrt(e d), so the smallest one grows to the size of the roundings within a layer.)"""
import dataclasses

import pytest
import torch

import helpers as H
import plain_qwen3 as plain
from test_8bit import check_product, check_rows, norm_of

TOL_RMS = 12.8e-2 + 2.8e-2


def make_runner(which, **kw):
    from vllm_lite_b200.engine import ModelRunner, load_model_dir
    _, plan, weights = load_model_dir(H.model_dir(which), "bfloat16", "cuda:0", eight_bit=True)
    return ModelRunner(plan, weights, dtype=torch.bfloat16, device="cuda:0", page_size=H.TINY[which]["page_size"], num_pages=64, max_requests=32, **kw)


def compare(rows, requests, which):
    assert rows
    for (rid, pos), row in rows.items():
        ref = H.plain_logits(which, requests[rid])[pos]
        err = float((row - ref).norm() / ref.norm())
        assert err <= TOL_RMS, f"{which}: request {rid} position {pos}: {err:.3e}"


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["A", "B", "C"])
@pytest.mark.parametrize("length", [1, 9, 40, 150])
def test_every_stage_of_a_layer(which, length):
    from vllm_lite_b200.csrc import ops
    from vllm_lite_b200.engine import ModelRunner, StepEntry, load_model_dir
    _, plan, weights = load_model_dir(H.model_dir(which), "bfloat16", "cuda:0", eight_bit=True)
    plan = dataclasses.replace(plan, layers=plan.layers[:1], order=plan.order[:1])
    w = {k: v.clone() for k, v in weights.items()}
    runner = ModelRunner(plan, weights, dtype=torch.bfloat16, device="cuda:0", page_size=16, num_pages=32, decode_graphs=False)
    tokens = H.tokens_for(which, length, 5)
    runner.step([StepEntry("a", tokens, [length - 1])])
    runner.check_device_errors()
    cfg = H.TINY[which]["config"]
    hidden, inter, eps = cfg["hidden_size"], cfg["intermediate_size"], cfg["rms_norm_eps"]
    width = cfg["num_attention_heads"] * cfg["head_dim"]
    left = {k[0].split("/")[-1]: v for k, v in runner.workspace._buffers.items()}

    def buffer(tag, *shape):
        n = 1
        for size in shape:
            n *= size
        return left[tag][:n].view(*shape)

    def rows(tag, k):
        return buffer(tag + ".8", length, ops.eight_bit_columns(k)), buffer(tag + ".scale", length)

    def to_8_bits(*names):
        t = torch.cat([w[f"model.layers.0.{n}.weight"] for n in names])
        values, scale = (torch.empty(t.shape[0], ops.eight_bit_columns(t.shape[1]), device="cuda:0").to(ops.E4M3), torch.empty(t.shape[0], device="cuda:0"))
        ops.rows_8bit(t.contiguous(), values, scale)
        return values, scale

    def norm(name):
        return w[f"model.layers.0.{name}.weight"].float().cpu()

    embedded = w["model.embed_tokens.weight"][torch.tensor(tokens, device="cuda:0")].float()
    stream = buffer("residual", length, hidden)
    check_rows(norm_of(embedded.cpu(), norm("input_layernorm"), eps), *rows("norm1", hidden), ops.eight_bit_columns(hidden))
    kv = cfg["num_key_value_heads"] * cfg["head_dim"]            # (queries and keys are normed and turned in place: the values are as they were)
    check_product(buffer("attn.qkv", length, width + 2 * kv)[:, width + kv:], *rows("norm1", hidden), *to_8_bits("self_attn.v_proj"))
    attended = buffer("attn.out", length, width)
    check_rows(attended.double().cpu(), *rows("attn.o.in", width), ops.eight_bit_columns(width))
    check_product(stream, *rows("attn.o.in", width), *to_8_bits("self_attn.o_proj"), residual=embedded)
    check_rows(norm_of(stream.cpu(), norm("post_attention_layernorm"), eps), *rows("norm2", hidden), ops.eight_bit_columns(hidden))
    order = torch.arange(2 * inter).view(2, inter // 8, 8).transpose(0, 1).reshape(-1)      # eight gates, their eight ups
    gate_up, scale = to_8_bits("mlp.gate_proj", "mlp.up_proj")
    order = order.to("cuda:0")
    gate_up = gate_up.view(torch.uint8)[order].view(ops.E4M3)
    activated = buffer("mlp.gate_up.act", length, inter)
    check_product(activated, *rows("norm2", hidden), gate_up, scale[order], act="silu", gated=True)
    check_rows(activated.double().cpu(), *rows("mlp.down.in", inter), ops.eight_bit_columns(inter))
    check_product(buffer("mlp.down", length, hidden), *rows("mlp.down.in", inter), *to_8_bits("mlp.down_proj"))


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["A", "B", "C"])
def test_prompts_and_single_tokens(which):
    """A prompt whole, another in portions, then tokens one by one, alone and beside each other."""
    runner = make_runner(which)
    a, b = H.tokens_for(which, 60, 1), H.tokens_for(which, 45, 2)
    steps = [([("a", a[:50], [0, 17, 49])], []), ([("b", b[:7], [6]), ("a", a[50:51], [0])], []), ([("b", b[7:40], [0, 32])], [])]
    for i in range(5):
        steps.append(([("a", a[51 + i:52 + i], [0]), ("b", b[40 + i:41 + i], [0])], []))
    steps.append(([("a", a[56:57], [0])], ["b"]))
    compare(H.run_schedule(runner, steps), {"a": a[:57], "b": b}, which)


@pytest.mark.gpu
def test_many_requests_side_by_side():
    """Twenty requests decoding: a recorded step beyond the kernel of few rows."""
    runner = make_runner("B")
    requests = {i: H.tokens_for("B", 6 + i % 5, 30 + i) for i in range(20)}
    steps = [([(i, t[:-3], [len(t) - 4]) for i, t in requests.items()], [])]
    for k in (3, 2, 1):
        steps.append(([(i, [t[-k]], [0]) for i, t in requests.items()], []))
    compare(H.run_schedule(runner, steps), requests, "B")
    assert runner.graph_replays >= 2


@pytest.mark.gpu
def test_the_engine_generates_with_it():
    from vllm_lite_b200 import LLMEngine, SamplingParams
    prompts = [H.tokens_for("B", n, n) for n in (5, 33, 70)]
    got = []
    for lookahead in (True, False):
        engine = LLMEngine(H.model_dir("B"), kv_blocks=64, block_size=8, max_batch_size=4, eight_bit=True, lookahead=lookahead)
        got.append(engine.generate(prompts, max_tokens=12, sampling_params=SamplingParams()))
        engine.runner.check_device_errors()
    assert got[0] == got[1] and all(len(t) == 12 for t in got[0])


def test_the_plan_in_8_bits_binds_the_same_tensors():
    from vllm_lite_b200.config import plan_from_config_json
    from vllm_lite_b200.parts import cache_needs, declare_model, in_8_bits
    for config in (H.TINY_A, H.TINY_B, H.TINY_C):
        _, plan = plan_from_config_json(config)
        eight = in_8_bits(plan)
        assert declare_model(eight) == declare_model(plan) and cache_needs(eight) == cache_needs(plan)
        assert {b.kind for b in eight.layers} == {"pre_norm_8bit"} and {b.kind for b in plan.layers} == {"pre_norm"}


def test_refusals():
    import dataclasses
    from vllm_lite_b200.config import plan_from_config_json
    from vllm_lite_b200.engine import plan_in_8_bits
    _, plan = plan_from_config_json(H.TINY_A)
    with pytest.raises(ValueError, match="bfloat16"):
        plan_in_8_bits(plan, "float32")
    with pytest.raises(ValueError, match="layer 1"):
        plan_in_8_bits(dataclasses.replace(plan, layers=(plan.layers[0], dataclasses.replace(plan.layers[1], kind="sandwich"))), "bfloat16")
    with pytest.raises(ValueError, match="layer 0"):
        plan_in_8_bits(plan_in_8_bits(plan, "bfloat16"), "bfloat16")


def test_steps_of_clusters_are_launched_the_plain_way(monkeypatch):
    from types import SimpleNamespace
    from vllm_lite_b200.engine.runner import ModelRunner
    model = SimpleNamespace(may_pair=lambda tokens: False, clusters=lambda tokens: tokens > 40)
    runner = SimpleNamespace(model=model)
    asked = [ModelRunner._launches_dependent(runner, t, recorded) for t in (1, 40, 41, 64, 100) for recorded in (False, True)]
    assert asked == [True, True, True, True, False, False, False, False, False, False]
    del model.clusters
    assert ModelRunner._launches_dependent(runner, 64, False) and ModelRunner._launches_dependent(runner, 100, True)
