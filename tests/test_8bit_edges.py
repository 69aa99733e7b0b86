"""Linear layers in 8 bits at the ends of what they take; tolerances as in test_8bit.py where none is named."""
import pytest
import torch

from test_8bit import DEV, JOINED, PAIRED, operands
from vllm_lite_b200.csrc import ops

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("m,n,k", [(3, 528, 1000), (16, 528, 1000), (16, 5120, 512), (24, 528, 1000), JOINED[0], PAIRED[0]])
def test_scales_whose_product_or_whose_sum_leaves_the_range_of_float32(m, n, k):
    """Scales times powers of two give the result times their product, to the bit: rows of up to 2^118 times common values, whose sums times
    the row's scale alone would overflow, and rows and weights so small that the two scales' product alone is not a normal number.  (A result below
    2^-126 is rounded once more: 2^-149 of it.)"""
    a, sa, w, sw = operands(45, m, n, k, std_w=0.2)
    p, plain, got = ops.pack_8bit(w), torch.empty(m, n, device=DEV), torch.empty(m, n, device=DEV)
    ops.gemm_8bit(a, sa, p, sw, plain)
    ops.gemm_8bit(a, sa * 2.0 ** 118, p, sw, got)
    assert torch.isfinite(got).all() and torch.equal(got, plain * 2.0 ** 118)
    ops.gemm_8bit(a, sa * 2.0 ** -100, p, sw * 2.0 ** -17, got)
    assert ((got.double() - plain.double() * 2.0 ** -117).abs() <= 2.0 ** -149).all()


@gpu
@pytest.mark.parametrize("m,n,k", [(3, 528, 1000), (16, 528, 1000), (24, 528, 1000), JOINED[0], PAIRED[0]])
def test_gates_and_ups_of_small_rows(m, n, k):
    """The same with a gate: its weights' scale takes the row's power of two back, the up's makes it smaller still."""
    a, sa, w, sw = operands(46, m, n, k, std_w=0.2)
    p, plain, got = ops.pack_8bit(w), torch.empty(m, n // 2, device=DEV), torch.empty(m, n // 2, device=DEV)
    ops.gemm_8bit(a, sa, p, sw, plain, act="relu", gated=True)
    gate = torch.arange(n, device=DEV) % 16 < 8
    ops.gemm_8bit(a, sa * 2.0 ** -100, p, torch.where(gate, sw * 2.0 ** 100, sw * 2.0 ** -17), got, act="relu", gated=True)
    # an up below 2^-126 is off by 2^-150, the product by as much times its gate; where either is below, the last bits of both results count too
    every = torch.empty(m, n, device=DEV)
    ops.gemm_8bit(a, sa, p, sw, every, act="relu")
    assert ((got.double() - plain.double() * 2.0 ** -117).abs() <= 2.0 ** -149 * (1 + every[:, gate].amax().double())).all()


def test_scratch_off_sixteen_bytes_is_refused_before_any_launch():
    """The entry point itself, which asks before it calls CUDA: the second launch reads the scratch memory 16 bytes at a time."""
    m, n, k = JOINED[0]
    columns = ops.eight_bit_columns(k)
    floats = ops.gemm_8bit_plan(m, n, columns, False)[0]
    assert floats
    host = torch.zeros(floats + 8)                            # never read or written
    at = -host.data_ptr() % 16 + host.data_ptr()
    for off in (4, 8, 12):
        code = ops._fn("gemm_8bit", "vl_gemm_8bit")(at, at, at, at, at, ops.F32, None, None, -1, 0, m, n, columns, at + off, floats, 0, None, 0)
        assert code == -2


@gpu
def test_scratch_of_the_callers_off_sixteen_bytes():
    m, n, k = JOINED[0]
    a, sa, w, sw = operands(49, m, n, k)
    p, floats = ops.pack_8bit(w), ops.gemm_8bit_plan(m, n, ops.eight_bit_columns(k))[0]
    buf, out = torch.zeros(floats + 8, device=DEV), torch.full((m, n), 3.0, device=DEV)
    for off in (1, 2, 3):
        with pytest.raises(ops.KernelError):
            ops.gemm_8bit(a, sa, p, sw, out, scratch=buf[off:])
    assert (out == 3).all() and not buf.any()
    want = ops.gemm_8bit(a, sa, p, sw, torch.empty_like(out))
    assert torch.equal(ops.gemm_8bit(a, sa, p, sw, out, scratch=buf[4:]), want)
