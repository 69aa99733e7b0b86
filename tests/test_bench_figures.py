"""The denominators of bench.py's roofline figures, from the sizes alone (no GPU)."""
import json
import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent
sys.path.insert(0, str(ROOT))
import bench  # noqa: E402


@pytest.mark.parametrize("size,weights_gb,kv_per_token,prefill_flops", [
    ("8b", 15.137, 147456, 2.97e13), ("14b", 27.98, 163840, 5.584e13), ("32b", 63.97, 262144, 1.322e14)])
def test_bytes_a_decode_step_reads_and_flops_of_the_prefill(size, weights_gb, kv_per_token, prefill_flops):
    """Every matrix of the layers and the vocabulary head once, in bfloat16 (the embedding is a row
    gather); keys and values of all layers per cached token; 2 flops per matrix element and token plus
    the causal half of the attention products."""
    layers, hidden, heads, inter = bench.SIZES[size]
    cfg = dict(bench.QWEN3_8B, num_hidden_layers=layers, hidden_size=hidden, num_attention_heads=heads,
               intermediate_size=inter)
    w, kv, flops = bench.model_bytes_and_flops(cfg, layers)
    assert abs(w / 1e9 - weights_gb) < 0.01
    assert kv == kv_per_token
    assert abs(flops / prefill_flops - 1) < 0.005
    half, _, _ = bench.model_bytes_and_flops(cfg, layers // 2)
    vocab_head = 2 * cfg["vocab_size"] * hidden
    assert abs((w - vocab_head) / (half - vocab_head) - 2) < 1e-3        # fewer layers: the layers' share shrinks, the head stays


def test_contract_edges_need_no_gpu():
    two = subprocess.run([sys.executable, str(ROOT / "bench.py"), "--gpus", "2"], capture_output=True, text=True)
    assert two.returncode == 2 and len(two.stdout.strip().splitlines()) == 1
    ref = subprocess.run([sys.executable, str(ROOT / "bench.py"), "--impl", "reference"], capture_output=True, text=True)
    line = json.loads(ref.stdout)
    assert ref.returncode == 0 and line["impl"] == "reference" and "unavailable" in line


def test_a_timed_step_records_every_dense_product(monkeypatch):
    """The per-kernel tables divide by what these products took: each one that the dispatcher can choose is recorded, the library's too."""
    import re
    from types import SimpleNamespace
    import torch
    from vllm_lite_b200.csrc import ops
    from vllm_lite_b200.parts import linear, matmul
    entries = {bench.OP_OF.get(n, n) for n in bench.DENSE_PRODUCTS}
    chosen = {m for module in (matmul, linear) for m in re.findall(r"\bops\.(gemm_\w+|mm)\(", Path(module.__file__).read_text())}
    assert {m for m in chosen if not m.endswith("_ok")} == entries and set(bench.DENSE_PRODUCTS) <= set(bench.TIMED_OPS)
    assert set(bench.PROMPT_PRODUCTS) <= set(bench.DENSE_PRODUCTS) and all(hasattr(ops, bench.OP_OF.get(n, n)) for n in bench.TIMED_OPS)

    class Event:
        def __init__(self, enable_timing):
            pass

        def record(self):
            pass

        def elapsed_time(self, other):
            return 1.0

    for name, stub in (("Event", Event), ("synchronize", lambda: None), ("_sleep", lambda n: None)):
        monkeypatch.setattr(torch.cuda, name, stub)
    for name in entries - {"mm"}:
        monkeypatch.setattr(ops, name, lambda *a, **k: None)
    monkeypatch.setattr(ops, "sm_pairs", lambda: 74)
    before = {n: getattr(ops, bench.OP_OF.get(n, n)) for n in bench.TIMED_OPS}

    def step(entries):
        for M, N in ((1, 64), (12, 64), (300, 64), (2048, 64), (2048, 40960)):
            matmul.gemm_bf16(torch.zeros(M, 64, dtype=torch.bfloat16), torch.zeros(N, 64, dtype=torch.bfloat16),
                             torch.zeros(M, N, dtype=torch.bfloat16) if M == 300 else None)

    got = bench.timed_step(SimpleNamespace(step=step, decode_graphs=True), [])
    assert {k: v[0] for k, v in got.items()} == {n: 1 for n in bench.DENSE_PRODUCTS if n != "gemm_f32"}
    assert before == {n: getattr(ops, bench.OP_OF.get(n, n)) for n in bench.TIMED_OPS}


def test_a_prompts_floor_with_products_in_8_bits():
    """Half the layers' products' time goes; attention and the head stay at the bfloat16 rate.  8B sizes: 28.5 of the prompt's 29.7 TFLOP are products
    of the layers (36 of 192.9 million elements, 2,048 tokens), 139,000 tokens/s are 0.61 of the floor's rate, not 1.18 of it."""
    cfg = dict(bench.QWEN3_8B)
    flops = bench.model_bytes_and_flops(cfg, 36)[2]
    elements = (32 + 16) * 128 * 4096 + 4096 * 4096 + 3 * 4096 * 12288
    assert bench.layer_elements(cfg) == elements
    rate = 1702.9
    assert abs(bench.prefill_floor_ms(cfg, 36, rate) / (flops / (rate * 1e9)) - 1) < 1e-9
    floor = bench.prefill_floor_ms(cfg, 36, rate, eight_bit=True)
    products = 2 * 2048 * 36 * elements
    assert abs(floor / ((flops - products) / (rate * 1e9) + products / (2 * rate * 1e9)) - 1) < 1e-9
    assert abs(floor / (2048 / 139000 * 1e3) - 0.615) < 0.01
    # what stands in the output is this floor over the time, wherever a prompt is timed
    code = Path(bench.__file__).read_text()
    main = code[code.index("def main("):]
    assert "prefill_flops" not in main and main.count("prefill_floor_ms(") == 3


def test_bytes_a_decode_step_reads_with_products_in_8_bits():
    """A byte an element of the layers' matrices and four a row of them; the head stays bfloat16, norms and cache as they were."""
    cfg = dict(bench.QWEN3_8B)
    wide, kv, flops = bench.model_bytes_and_flops(cfg, 36)
    narrow, kv8, flops8 = bench.model_bytes_and_flops(cfg, 36, True)
    rows = (32 + 2 * 8) * 128 + 4096 + 2 * 12288 + 4096
    assert (kv8, flops8) == (kv, flops) and wide - narrow == 36 * (bench.layer_elements(cfg) - 4 * rows)
    assert abs(narrow / 1e9 - 8.198) < 0.02
