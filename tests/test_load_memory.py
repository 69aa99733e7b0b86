"""What a model needs while it is built: an engine that owns its weights gives a layer's tensors up as the layer has been built."""
import pytest
import torch

import helpers as H
from vllm_lite_b200.engine import load_model_dir
from vllm_lite_b200.parts import BLOCKS, CausalLM, declare_model
from vllm_lite_b200.parts.base import BuildContext, prefixed

DEEP = dict(architectures=["Qwen3ForCausalLM"], model_type="qwen3", hidden_size=512, num_hidden_layers=8, num_attention_heads=8,
            num_key_value_heads=4, head_dim=64, intermediate_size=2048, vocab_size=64, rope_theta=10000.0, rms_norm_eps=1e-6,
            tie_word_embeddings=False, max_position_embeddings=256)


def layer_names(plan):
    return [set(prefixed(BLOCKS.get(b.kind).declare(b), plan.layer_prefix.format(i))) for i, b in enumerate(plan.layers)]


def test_a_layers_tensors_leave_the_dict_when_it_is_built(monkeypatch):
    _, plan, weights = load_model_dir(H.model_dir("B"), "bfloat16", "cpu")
    names, every, seen = layer_names(plan), set(weights), []
    block = BLOCKS.get("pre_norm")
    init = block.__init__

    def noted(self, spec, w, ctx):
        seen.append(set(weights))
        init(self, spec, w, ctx)

    monkeypatch.setattr(block, "__init__", noted)
    ctx = BuildContext(torch.device("cpu"), torch.bfloat16)
    CausalLM(plan, weights, ctx)
    assert set(weights) == every and len(seen) == len(names)
    del seen[:]
    CausalLM(plan, weights, ctx, own_weights=True)
    left = set(every)
    for before, own in zip(seen, names):
        assert own <= before == left
        left -= own
    assert set(weights) == left and left == every - set().union(*names)


def test_no_tensor_belongs_to_two_parts():
    """What a layer gives up is nobody else's: every declared name has one part."""
    from vllm_lite_b200.config import plan_from_config_json
    for config in (H.TINY_A, H.TINY_B, H.TINY_C, DEEP):
        _, plan = plan_from_config_json(config)
        names = layer_names(plan)
        assert sum(map(len, names)) == len(set().union(*names)) < len(declare_model(plan))


@pytest.mark.gpu
@pytest.mark.parametrize("eight_bit", [False, True])
def test_a_model_is_built_beside_one_layer_of_copies(eight_bit):
    from vllm_lite_b200.csrc import ops
    from vllm_lite_b200.engine import ModelRunner, plan_in_8_bits, random_model
    # the kernels of a first build are loaded before memory is looked at
    ops.pack_8bit(ops.rows_8bit(torch.ones(16, 128, device="cuda:0"), torch.empty(16, 128, dtype=ops.E4M3, device="cuda:0"), torch.empty(16, device="cuda:0")))
    _, plan, weights = random_model(DEEP, seed=3, dtype="bfloat16", device="cuda:0", std=0.02)
    total = sum(w.numel() * w.element_size() for w in weights.values())
    layer = total / 8
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    runner = ModelRunner(plan_in_8_bits(plan, "bfloat16") if eight_bit else plan, weights, dtype=torch.bfloat16, device="cuda:0", page_size=16,
                         num_pages=4, max_requests=2, own_weights=True)
    peak, after = torch.cuda.max_memory_allocated() - before, torch.cuda.memory_allocated() - before
    assert not weights and len(runner.model.layers) == 8
    # stacked matrices and their 8-bit forms of the layer in work (no more than two copies of it), and the small cache
    assert peak <= 2.2 * layer
    assert after <= (-0.45 if eight_bit else 0.05) * total
