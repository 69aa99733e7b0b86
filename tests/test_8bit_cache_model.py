"""Models whose keys and values are kept in 8 bits.

Stage by stage, from what the engine itself left in its buffers: the cache's pages and the attention of a one-layer model against their definitions in 64 bits,
with the tolerances of tests/test_8bit_cache.py.

As a whole, against the plain implementation without any rounding: the error of all logits of a row, as a root of mean squares, over the logits' own.  A
rounding to e4m3 is off by up to 2^-4 of a value, uniformly, which is 2.6e-2 as a root of mean squares (once more as much at most where a page's scale grows).  A value's
error is an output's; a key's is a score's, whose own size is about one in these models, and with it a weight's: 3.7e-2 an attention, 11.1e-2 in three layers
in a row if nothing of the stream but their results were left; the bfloat16 engine's error beside it."""
import dataclasses

import pytest
import torch

import helpers as H
from test_8bit_cache import check_attention

gpu = pytest.mark.gpu
TOL_RMS = 11.1e-2 + 2.8e-2


def make_runner(which, page_size=None, eight_bit=False, **kw):
    from vllm_lite_b200.engine import ModelRunner, load_model_dir
    _, plan, weights = load_model_dir(H.model_dir(which), "bfloat16", "cuda:0", eight_bit=eight_bit, eight_bit_cache=True)
    return ModelRunner(plan, weights, dtype=torch.bfloat16, device="cuda:0", page_size=page_size or H.TINY[which]["page_size"], num_pages=64, max_requests=32, **kw)


def compare(rows, requests, which, tol=TOL_RMS):
    assert rows
    for (rid, pos), row in rows.items():
        ref = H.plain_logits(which, requests[rid])[pos]
        err = float((row - ref).norm() / ref.norm())
        assert err <= tol, f"{which}: request {rid} position {pos}: {err:.3e}"


@gpu
@pytest.mark.parametrize("which", ["A", "B", "C"])
@pytest.mark.parametrize("ps", [8, 64])
def test_every_stage_of_a_layer(which, ps):
    """A prompt in portions, then single tokens: what each step left in its buffers and in the cache."""
    from vllm_lite_b200.engine import ModelRunner, StepEntry, load_model_dir
    _, plan, weights = load_model_dir(H.model_dir(which), "bfloat16", "cuda:0", eight_bit_cache=True)
    plan = dataclasses.replace(plan, layers=plan.layers[:1], order=plan.order[:1])
    runner = ModelRunner(plan, weights, dtype=torch.bfloat16, device="cuda:0", page_size=ps, num_pages=32, decode_graphs=False)
    mixer = runner.model.layers[0].mixer
    s, cache = mixer.spec, runner.storage.call_caches[0]
    tokens, at = H.tokens_for(which, 60, 5), 0

    class View:                                              # the cache as the checks of the operators see it
        nkv, hd = s.num_kv_heads, s.head_dim
        k, v, k_scale, v_scale = cache.k, cache.v, cache.k_scale, cache.v_scale

        def rows(self, r, n):
            pages = torch.tensor(runner.cache.requests["a"].block_tables[0][:-(-n // ps)], device="cuda:0")
            return tuple((c[pages].double() * x[pages].double()[..., None, None]).transpose(1, 2).reshape(-1, self.nkv, self.hd)[:n]
                         for c, x in ((self.k, self.k_scale), (self.v, self.v_scale)))
    for n in (1, 37, 1, 1, 20):
        runner.step([StepEntry("a", tokens[at:at + n], [n - 1])])
        runner.check_device_errors()
        left = {k[0].split("/")[-1]: v for k, v in runner.workspace._buffers.items()}
        width = (s.num_heads + 2 * s.num_kv_heads) * s.head_dim
        qkv, out = left["attn.qkv"][:n * width].view(n, width), left["attn.out"][:n * s.num_heads * s.head_dim].view(n, -1)
        pos = torch.arange(at, at + n)
        check_attention(View(), qkv, out, pos, torch.zeros(n, dtype=torch.long), s.num_heads, s.window, mixer.scale)
        at += n
    k, v = View().rows(0, at)
    assert torch.isfinite(k).all() and float(k.abs().amax()) > 0 and torch.isfinite(v).all()


@gpu
@pytest.mark.parametrize("which", ["A", "B", "C", "L"])
@pytest.mark.parametrize("eight_bit", [False, True])
def test_logits_of_prompts_cut_anywhere_beside_requests_that_decode(which, eight_bit):
    requests = {r: H.tokens_for(which, n, 40 + r) for r, n in enumerate((50, 33, 70))}
    runner = make_runner(which, eight_bit=eight_bit)
    schedule = [[(0, 20)], [(0, 1), (1, 30)], [(0, 13), (1, 1), (2, 65)], [(0, 1), (1, 1), (2, 1)], [(0, 1), (1, 1), (2, 1)], [(0, 14), (2, 3)]]
    rows = {}
    from vllm_lite_b200.engine import StepEntry
    have = dict.fromkeys(requests, 0)
    for step in schedule:
        entries = [StepEntry(r, requests[r][have[r]:have[r] + n], list(range(n))) for r, n in step]
        logits = runner.step(entries).cpu()
        i = 0
        for r, n in step:
            for j in range(n):
                rows[r, have[r] + j] = logits[i]
                i += 1
            have[r] += n
    runner.check_device_errors()
    compare(rows, requests, which, TOL_RMS + (12.8e-2 if eight_bit else 0))


@gpu
def test_decode_steps_from_graphs():
    """Recorded and replayed steps, many requests, pages that change hands."""
    from vllm_lite_b200.engine import StepEntry
    which, rows = "B", {}
    runner = make_runner(which, page_size=8)
    requests = {r: H.tokens_for(which, 24 + r, 70 + r) for r in range(7)}
    for wave in (range(4), range(4, 7)):
        for r in wave:
            logits = runner.step([StepEntry(r, requests[r][:16 + r], [15 + r])])
            rows[r, 15 + r] = logits[0].cpu()
        for i in range(8):
            logits = runner.step([StepEntry(r, [requests[r][16 + r + i]], [0]) for r in wave]).cpu()
            for j, r in enumerate(wave):
                rows[r, 16 + r + i] = logits[j]
        for r in wave:
            runner.release(r)
    runner.check_device_errors()
    assert runner.graph_replays > 0
    compare(rows, requests, which)


@gpu
def test_generation_with_min_p():
    from vllm_lite_b200 import LLMEngine, SamplingParams
    prompts = [H.tokens_for("B", n, n) for n in (5, 33, 70)]
    got = []
    for lookahead in (True, False):
        engine = LLMEngine(H.model_dir("B"), kv_blocks=64, block_size=8, max_batch_size=4, eight_bit_cache=True, lookahead=lookahead)
        got.append(engine.generate(prompts, max_tokens=12, sampling_params=SamplingParams(temperature=0.9, top_k=30, top_p=0.95, min_p=0.02, seed=3)))
        engine.runner.check_device_errors()
    assert got[0] == got[1] and all(len(t) == 12 for t in got[0])
    # min_p = 1 leaves the most probable token alone: what greedy decoding gives
    engine = LLMEngine(H.model_dir("B"), kv_blocks=64, block_size=8, max_batch_size=4, eight_bit_cache=True)
    first = engine.generate(prompts, max_tokens=12, sampling_params=SamplingParams(temperature=0.9, min_p=1.0, seed=3))
    engine = LLMEngine(H.model_dir("B"), kv_blocks=64, block_size=8, max_batch_size=4, eight_bit_cache=True)
    assert first == engine.generate(prompts, max_tokens=12, sampling_params=SamplingParams())


@gpu
def test_a_cache_too_small_for_all_requests():
    """Requests that are pre-empted and computed again: the run ends, nothing is flagged."""
    from vllm_lite_b200 import LLMEngine, SamplingParams
    engine = LLMEngine(H.model_dir("A"), kv_blocks=14, block_size=8, max_batch_size=4, eight_bit_cache=True, max_model_len=100)
    out = engine.generate([H.tokens_for("A", 20, i) for i in range(4)], max_tokens=30, sampling_params=SamplingParams())
    engine.runner.check_device_errors()
    assert [len(o) for o in out] == [30] * 4


@gpu
def test_calls_that_share_a_cache_and_layers_that_run_twice():
    """A call that reads an earlier call's pages writes none of its own."""
    from vllm_lite_b200.engine import ModelRunner, StepEntry, load_model_dir
    _, plan, weights = load_model_dir(H.model_dir("A"), "bfloat16", "cuda:0", eight_bit_cache=True)
    plan = dataclasses.replace(plan, order=(plan.order[0], dataclasses.replace(plan.order[1], cache_of=0)))
    runner = ModelRunner(plan, weights, dtype=torch.bfloat16, device="cuda:0", page_size=16, num_pages=32)
    tokens = H.tokens_for("A", 40, 1)
    runner.step([StepEntry("a", tokens[:30], [29])])
    before = runner.storage.scales[0].clone()
    for t in tokens[30:]:
        assert torch.isfinite(runner.step([StepEntry("a", [t], [0])])).all()
    runner.check_device_errors()
    assert len(runner.storage.paged) == 1 and runner.storage.paged[0].shape[0] == 1 and not torch.equal(before, runner.storage.scales[0])


@gpu
def test_pages_take_half_the_memory():
    from vllm_lite_b200.engine import ModelRunner, load_model_dir
    size = []
    for eight in (False, True):
        _, plan, weights = load_model_dir(H.model_dir("A"), "bfloat16", "cuda:0", eight_bit_cache=eight)
        size.append(ModelRunner(plan, weights, dtype=torch.bfloat16, device="cuda:0", page_size=64, num_pages=32).storage.bytes())
    scales = 2 * 32 * 4 * H.TINY_A["num_key_value_heads"] * H.TINY_A["num_hidden_layers"]
    assert size[1] == size[0] // 2 + scales


def test_sizes_of_pages():
    from vllm_lite_b200.cache import CacheLayout, PagedKV
    from vllm_lite_b200.cache.sizing import page_bytes
    need = PagedKV(8, 128, eight_bit=True)
    assert page_bytes(CacheLayout.from_needs([need] * 36, [None] * 36), 64, 2) == [36 * 2 * 8 * (64 * 128 + 4)]
    both = CacheLayout.from_needs([need, PagedKV(8, 128)], [None, None])
    assert len(both.paged_groups) == 2 and page_bytes(both, 64, 2) == [2 * 8 * (64 * 128 + 4), 2 * 8 * 64 * 128 * 2]


def test_the_plan_binds_the_same_tensors():
    from vllm_lite_b200.config import plan_from_config_json
    from vllm_lite_b200.engine.loading import plan_in_8_bits, plan_with_8_bit_cache
    from vllm_lite_b200.parts import cache_needs, declare_model
    for config in (H.TINY_A, H.TINY_B, H.TINY_C):
        _, plan = plan_from_config_json(config)
        eight = plan_with_8_bit_cache(plan, "bfloat16")
        assert declare_model(eight) == declare_model(plan)
        assert [dataclasses.replace(n, eight_bit=False) for n in cache_needs(eight)] == cache_needs(plan) and all(n.eight_bit for n in cache_needs(eight))
        both = plan_with_8_bit_cache(plan_in_8_bits(plan, "bfloat16"), "bfloat16")
        assert cache_needs(both) == cache_needs(eight) == cache_needs(plan_in_8_bits(eight, "bfloat16"))
        assert {b.mixer.kind for b in both.layers} == {"gqa_attention_8bit"}


def test_refusals():
    from vllm_lite_b200.config import plan_from_config_json
    from vllm_lite_b200.engine.loading import plan_with_8_bit_cache
    _, plan = plan_from_config_json(H.TINY_A)
    with pytest.raises(ValueError, match="bfloat16"):
        plan_with_8_bit_cache(plan, "float32")
    block = plan.layers[1]
    for change in (dict(softcap=5.0), dict(unit_sink=True), dict(window=8, keep_first=2), dict(gate="g"), dict(kind="other"),
                   dict(position=dataclasses.replace(block.mixer.position, rotary_dim=6))):
        with pytest.raises(ValueError, match="layer 1"):
            plan_with_8_bit_cache(dataclasses.replace(plan, layers=(plan.layers[0], dataclasses.replace(block, mixer=dataclasses.replace(block.mixer, **change)))), "bfloat16")
    with pytest.raises(ValueError, match="layer 0"):
        plan_with_8_bit_cache(dataclasses.replace(plan, layers=(dataclasses.replace(block, mixer=None),) + tuple(plan.layers[1:])), "bfloat16")


@pytest.mark.parametrize("head_dim", [8, 24, 100, 272, 512])
def test_heads_that_have_no_form(head_dim):
    from vllm_lite_b200.engine import load_model_dir
    from vllm_lite_b200.parts.eight_bit import cache_in_8_bits
    _, plan, _ = load_model_dir(H.model_dir("A"), "bfloat16", "cpu")
    layers = list(plan.layers)
    layers[-1] = dataclasses.replace(layers[-1], mixer=dataclasses.replace(layers[-1].mixer, head_dim=head_dim))
    with pytest.raises(ValueError, match=f"layer {len(layers) - 1}: .*{head_dim}"):
        cache_in_8_bits(dataclasses.replace(plan, layers=tuple(layers)))


def test_one_cache_has_one_type():
    from vllm_lite_b200.cache import PagedKV
    from vllm_lite_b200.cache.spec import widened
    with pytest.raises(ValueError):
        widened(PagedKV(2, 16, eight_bit=True), PagedKV(2, 16))
    assert widened(PagedKV(2, 16, 8, eight_bit=True), PagedKV(2, 16, 12, eight_bit=True)) == PagedKV(2, 16, 12, eight_bit=True)


def test_command_line(capsys, monkeypatch):
    from vllm_lite_b200 import cli
    monkeypatch.delenv("VLLM_MODEL", raising=False)
    args = cli.build_parser().parse_args(["-m", "/x", "--eight-bit-cache", "--min-p", "0.1"])
    assert args.eight_bit_cache and args.min_p == 0.1 and not cli.build_parser().parse_args(["-m", "/x"]).eight_bit_cache
    with pytest.raises(SystemExit):
        cli.main(["--model", ".", "--eight-bit-cache", "--dtype", "float32", "--prompt-ids", "1"])
    assert "--dtype bfloat16" in capsys.readouterr().err
