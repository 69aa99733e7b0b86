"""Rows in 8 bits and the products that read them, against the definitions in 64 bits.

Tolerances.  A scale is a float32 number behind a norm (a sum of squares, a root, a quotient, three products: a few units in the last
place of 2^-24 each): 2e-6 of itself.  A value q of a row is the e4m3 number nearest to h / scale: half a step away at most, which is
2^-4 of the value where e4m3 is normal (2^-6 and more) and 2^-10 below, plus what h / scale itself is off (1e-5 of it).
A product's sum is exact but for the float32 additions: each tensor-core step adds 32 products to the running sum and may be off
by 2^-23 of what it has added so far, K / 32 steps and 32 more for the joining of partial sums.  Behind it follow an activation (slope `L`, and
1e-5 of its value for the fast exponential), and one rounding to the output's type (half a unit in the last of its 8 or 24 bits: 2^-8 bfloat16, 2^-24 float32)."""
import pytest
import torch

from vllm_lite_b200.csrc import ops

DEV = "cuda:0"
gpu = pytest.mark.gpu
F8 = torch.float8_e4m3fn


def columns(k):
    return -(-k // 128) * 128


def normal(seed, *shape, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, generator=g) * std


def check_rows(h, out, scale, width):
    """out * scale stands for h (float64, on the CPU)."""
    out, scale = out.float().double().cpu(), scale.double().cpu()
    k = h.shape[1]
    assert out.shape == (h.shape[0], width) and not out[:, k:].any()
    top = h.abs().amax(dim=1)
    assert ((scale - top / 448).abs() <= 2e-6 * top / 448).all()
    v = torch.where(top[:, None] > 0, h * 448 / top[:, None], torch.zeros_like(h))
    off = (out[:, :k] - v).abs()
    assert (off <= (v.abs() * 2.0 ** -4).clamp(min=2.0 ** -10) + 1e-5 * v.abs()).all()


def norm_of(x, weight, eps):
    x = x.double()
    return x / torch.sqrt((x * x).mean(dim=1, keepdim=True) + eps) * weight.double()


def empty_rows(r, k):
    return torch.full((r, columns(k)), 1.5, device=DEV).to(F8), torch.full((r,), -1.0, device=DEV)


NORM_SIZES = [(1, 4096), (3, 96), (2, 1), (5, 130), (7, 1001), (150, 512), (2, 5120), (9, 2050), (3, 8192), (2, 20000), (700, 128), (1200, 1000)]


@gpu
@pytest.mark.parametrize("delta", [None, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("r,h", NORM_SIZES)
def test_norm_rows(r, h, delta):
    x, w = normal(1, r, h, std=2.0), 1 + normal(2, h, std=0.3)
    x[:, : max(1, h // 100)] *= 20
    d = None if delta is None else normal(3, r, h).to(delta)
    xg, out, scale = x.to(DEV), *empty_rows(r, h)
    assert ops.add_rmsnorm_8bit(xg, None if d is None else d.to(DEV), w.to(DEV), 1e-6, out, scale) is out
    new = x if d is None else x + d.float()                           # one float32 addition: equal to the bit
    assert torch.equal(xg.cpu(), new)
    check_rows(norm_of(new, w, 1e-6), out, scale, columns(h))


@gpu
@pytest.mark.parametrize("h", [64, 1001, 4096])
@pytest.mark.parametrize("with_delta", [False, True])
def test_norm_of_picked_rows_leaves_the_stream(h, with_delta):
    x, w, d = normal(4, 40, h), 1 + normal(5, h, std=0.3), normal(6, 40, h).bfloat16()
    pick = torch.tensor([39, 0, 17, 17, 3], dtype=torch.int32)
    xg, out, scale = x.to(DEV), *empty_rows(5, h)
    into = torch.full_like(xg, 7.0)
    ops.add_rmsnorm_8bit(xg, d.to(DEV) if with_delta else None, w.to(DEV), 1e-5, out, scale, rows=pick.to(DEV), into=into)
    assert torch.equal(xg.cpu(), x) and (into == 7).all()
    new = x + d.float() if with_delta else x
    check_rows(norm_of(new[pick.long()], w, 1e-5), out, scale, columns(h))


@gpu
@pytest.mark.parametrize("h", [96, 2048, 3000, 4096, 5120, 8192, 1001])
def test_a_norm_does_not_see_how_many_rows_there_are(h):
    x, w = normal(8, 2500, h).to(DEV), normal(9, h).to(DEV)
    d = normal(10, 2500, h).to(DEV, torch.bfloat16)
    many = empty_rows(2500, h)
    ops.add_rmsnorm_8bit(x, d, w, 1e-6, *many, into=torch.empty_like(x))
    for r in (0, 1234, 2499):
        few = empty_rows(1, h)
        ops.add_rmsnorm_8bit(x[r:r + 1].clone(), d[r:r + 1].clone(), w, 1e-6, *few)
        assert torch.equal(few[0][0].view(torch.uint8), many[0][r].view(torch.uint8)) and torch.equal(few[1][0], many[1][r])


@gpu
@pytest.mark.parametrize("h", [100, 4096])
def test_norm_into_other_memory(h):
    x, d, w = normal(7, 6, h), normal(8, 6, h).bfloat16(), torch.ones(h)
    xg, out, scale = x.to(DEV), *empty_rows(6, h)
    into = torch.empty_like(xg)
    ops.add_rmsnorm_8bit(xg, d.to(DEV), w.to(DEV), 1e-6, out, scale, into=into)
    assert torch.equal(xg.cpu(), x) and torch.equal(into.cpu(), x + d.float())
    again, scale2 = empty_rows(6, h)
    ops.add_rmsnorm_8bit(into, None, w.to(DEV), 1e-6, again, scale2)
    assert torch.equal(again.view(torch.uint8), out.view(torch.uint8)) and torch.equal(scale, scale2)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("r,k", NORM_SIZES + [(2, 12288), (1, 33000)])
def test_rows(r, k, dtype):
    x = normal(9, r, k, std=0.02).to(dtype)
    out, scale = empty_rows(r, k)
    assert ops.rows_8bit(x.to(DEV), out, scale) is out
    check_rows(x.double(), out, scale, columns(k))


@gpu
@pytest.mark.parametrize("k", [200, 4096])
def test_rows_that_are_zeros_tiny_huge_or_not_finite(k):
    x = normal(10, 8, k)
    x[0] = 0
    x[1] *= 1e-38                                        # below 2^-100: counts as zeros
    x[2] *= 2e-29                                        # small, but not below
    x[3] *= 1e37
    x[4, 5] = float("nan")
    x[5, 7] = float("inf")
    x[6, -1] = -float("inf")
    out, scale = empty_rows(8, k)
    ops.rows_8bit(x.to(DEV), out, scale)
    q, s = out.float().cpu(), scale.cpu()
    assert s[0] == 0 and not q[0].any() and not q[1].any() and s[1] >= 0
    check_rows(x[[2, 3, 7]].double(), out[[2, 3, 7]], scale[[2, 3, 7]], columns(k))
    assert torch.isnan(s[4]) and torch.isnan(q[4, 5])
    assert not torch.isfinite(s[5:7]).any() and torch.isnan(q[5, 7]) and torch.isnan(q[6, k - 1])


@gpu
def test_rows_off_the_sixteen_byte_boundary():
    """Contiguous views that begin anywhere: the rows are the same."""
    base = normal(11, 1 + 6 * 512).to(DEV)
    for dtype in (torch.float32, torch.bfloat16):
        flat = base.to(dtype)
        view, whole = flat[1:].view(6, 512), flat[1:].clone().view(6, 512)
        a, sa = empty_rows(6, 512)
        b, sb = empty_rows(6, 512)
        ops.rows_8bit(view, a, sa)
        ops.rows_8bit(whole, b, sb)
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)) and torch.equal(sa, sb)
        x = base[1:].view(6, 512)
        d = flat[1:].view(6, 512)
        a, sa = empty_rows(6, 512)
        ops.add_rmsnorm_8bit(x, d, torch.ones(513, device=DEV)[1:], 1e-6, a, sa, into=torch.empty(6 * 512 + 1, device=DEV)[1:].view(6, 512))
        check_rows(norm_of(x.cpu() + d.float().cpu(), torch.ones(512), 1e-6), a, sa, 512)


@gpu
def test_nothing_to_do():
    out, scale = empty_rows(0, 64)
    ops.rows_8bit(torch.empty(0, 64, device=DEV), out, scale)
    ops.add_rmsnorm_8bit(torch.empty(0, 64, device=DEV), None, torch.ones(64, device=DEV), 1e-6, out, scale)
    w = ops.pack_8bit(torch.zeros(32, 128, device=DEV).to(F8))
    y = torch.empty(0, 32, device=DEV)
    ops.gemm_8bit(out, scale, w, torch.ones(32, device=DEV), y)


# ---------------------------------------------------------------------------------------------- products
def unpacked(p, n):
    """The layout's definition, written out: strips of 16 rows, blocks of 128 columns, pieces of 16 exchanged by xor."""
    p = p.view(torch.uint8).cpu()
    strips, blocks = p.shape[:2]
    p = p.view(strips, blocks, 16, 8, 16)
    w = torch.empty(strips, 16, blocks, 8, 16, dtype=torch.uint8)
    for row in range(16):
        for piece in range(8):
            w[:, row, :, piece] = p[:, :, row, piece ^ (row & 7)]
    w = w.reshape(strips * 16, blocks * 128)
    assert not w[n:].any()
    return w[:n]


@gpu
@pytest.mark.parametrize("n,k", [(16, 128), (1, 128), (33, 384), (250, 1024)])
def test_packing(n, k):
    w = normal(12, n, k).to(F8)
    p = ops.pack_8bit(w.to(DEV))
    assert p.shape == (-(-n // 16), k // 128, 16, 128) and torch.equal(unpacked(p, n), w.view(torch.uint8))


def operands(seed, m, n, k, std_w=0.05):
    a, sa = empty_rows(m, k)
    w, sw = empty_rows(n, k)
    ops.rows_8bit(normal(seed, m, k).to(DEV), a, sa)
    ops.rows_8bit(normal(seed + 1, n, k, std=std_w).to(DEV), w, sw)
    return a, sa, w, sw


FUNCTIONS = {None: (lambda v: v, lambda v: torch.ones_like(v)), "silu": (lambda v: v * torch.sigmoid(v), lambda v: torch.full_like(v, 1.1)),
             "relu": (lambda v: v.clamp(min=0), lambda v: torch.ones_like(v)), "relu2": (lambda v: v.clamp(min=0) ** 2, lambda v: 2 * v.abs() + 1e-3),
             "tanh": (torch.tanh, lambda v: torch.ones_like(v)), "gelu": (lambda v: v * torch.special.ndtr(v), lambda v: torch.full_like(v, 1.13))}


def check_product(got, a, sa, w, sw, bias=None, act=None, gated=False, residual=None):
    k = a.shape[1]
    av, wv = a.float().double() * sa.double()[:, None], w.float().double() * sw.double()[:, None]
    y, mass = av @ wv.t(), av.abs() @ wv.abs().t()
    if bias is not None:
        y, mass = y + bias.double(), mass + bias.double().abs()
    off = (k / 32 + 32 + 4) * 2.0 ** -23 * mass
    f, slope = FUNCTIONS[act]
    if gated:
        pick = torch.arange(y.shape[1], device=y.device) % 16 < 8
        g, u, og, ou = y[:, pick], y[:, ~pick], off[:, pick], off[:, ~pick]
        off = (slope(g) * og + 1e-5 * f(g).abs()) * (u.abs() + ou) + f(g).abs() * ou
        y = f(g) * u
    else:
        off = slope(y) * off + 1e-5 * f(y).abs()
        y = f(y)
    if residual is not None:
        y = y + residual.double()
    off = off + 2.0 ** (-24 if got.dtype == torch.float32 else -8) * 1.01 * (y.abs() + off) + 1e-30
    assert got.shape == y.shape and torch.isfinite(got).all()
    worst = ((got.double() - y).abs() / off).max().item() if got.numel() else 0.0
    assert worst <= 1, f"{worst} times the tolerance"


SIZES = [(1, 16, 128), (1, 1, 1), (1, 4096, 4096), (2, 130, 100), (3, 48, 4224), (5, 1003, 1000), (8, 6144, 512), (8, 64, 12288), (9, 17, 300),
         (15, 272, 640), (16, 512, 2048), (17, 512, 2048), (24, 100, 700), (31, 640, 1152), (32, 2048, 256), (33, 257, 129), (48, 96, 5120),
         (63, 1000, 512), (64, 4096, 1024), (65, 384, 384), (100, 130, 2000), (128, 1024, 768), (129, 129, 129), (173, 1003, 1000), (200, 2304, 512),
         (255, 512, 640), (256, 256, 4096), (257, 513, 257), (300, 4096, 256), (512, 640, 384), (700, 1111, 200), (1024, 2048, 512), (1500, 520, 130),
         (2048, 384, 256), (2049, 255, 640), (4097, 128, 128)]


@gpu
@pytest.mark.parametrize("m,n,k", SIZES)
def test_products(m, n, k):
    a, sa, w, sw = operands(20, m, n, k)
    p = ops.pack_8bit(w)
    for dtype in (torch.bfloat16, torch.float32):
        out = torch.full((m, n), float("nan"), device=DEV, dtype=dtype)
        assert ops.gemm_8bit(a, sa, p, sw, out) is out
        check_product(out, a, sa, w, sw)


EPILOGUES = [dict(bias=True), dict(act="silu"), dict(act="gelu", bias=True), dict(act="relu2", residual=True), dict(act="tanh"), dict(residual=True),
             dict(act="relu", bias=True, residual=True), dict(gated=True, act="silu"), dict(gated=True, act="relu", bias=True),
             dict(gated=True, act="silu", residual=True, bias=True)]
EPILOGUE_SIZES = [(1, 32, 256), (7, 1008, 300), (16, 176, 512), (40, 1008, 512), (130, 272, 640), (320, 528, 256), (1030, 2064, 384)]


@gpu
@pytest.mark.parametrize("m,n,k", [(2100, 2600, 256), (1000, 10000, 128), (700, 14000, 300), (3000, 5000, 128), (4500, 4100, 384), (257, 40000, 128)])
def test_products_of_several_rounds(m, n, k):
    """More tiles than pairs of SMs: both accumulators in turn, whole tiles and halves of tiles in the last round."""
    a, sa, w, sw = operands(25, m, n, k)
    p, bias = ops.pack_8bit(w), normal(26, n).to(DEV)
    res = normal(27, m, n).to(DEV)
    out = torch.full((m, n), float("nan"), device=DEV)
    ops.gemm_8bit(a, sa, p, sw, out, bias=bias, residual=res)
    check_product(out, a, sa, w, sw, bias, residual=res)
    if n % 16 == 0:
        half = torch.full((m, n // 2), float("nan"), device=DEV, dtype=torch.bfloat16)
        ops.gemm_8bit(a, sa, p, sw, half, act="silu", gated=True)
        check_product(half, a, sa, w, sw, act="silu", gated=True)


@gpu
@pytest.mark.parametrize("how", EPILOGUES, ids=lambda d: "-".join(f"{k}={v}" for k, v in d.items()))
@pytest.mark.parametrize("m,n,k", EPILOGUE_SIZES)
def test_epilogues(m, n, k, how):
    a, sa, w, sw = operands(30, m, n, k, std_w=0.2)
    p = ops.pack_8bit(w)
    gated = how.get("gated", False)
    width = n // 2 if gated else n
    bias = normal(31, n).to(DEV) if how.get("bias") else None
    for dtype in (torch.bfloat16, torch.float32):
        res = normal(32, m, width).to(DEV, dtype) if how.get("residual") else None
        out = torch.full((m, width), float("nan"), device=DEV, dtype=dtype)
        ops.gemm_8bit(a, sa, p, sw, out, bias=bias, act=how.get("act"), gated=gated, residual=res)
        check_product(out, a, sa, w, sw, bias, how.get("act"), gated, res)
        if res is not None:                                   # the sum may go where the residual stands
            same = res.clone()
            ops.gemm_8bit(a, sa, p, sw, same, bias=bias, act=how.get("act"), gated=gated, residual=same)
            assert torch.equal(same, out)


# sizes that the plan gives to pairs of SMs, and such whose K is shared out among blocks and joined by a second launch
PAIRED, JOINED = [(1030, 8208, 384), (999, 12001, 200)], [(130, 144, 6000), (50, 99, 5100)]
LOW = [(64, 20000, 2048), (40, 19001, 2100)]                  # tiles of fewer than 128 rows of w


@pytest.fixture(params=[False, True], ids=["", "dependent"])
def dependent(request):
    ops.set_pdl(request.param)
    yield request.param
    ops.set_pdl(False)


def run_product(m, n, k, how, dtype=torch.float32):
    a, sa, w, sw = operands(35, m, n, k, std_w=0.2)
    gated = how.get("gated", False)
    width = n // 2 if gated else n
    bias = normal(36, n).to(DEV) if how.get("bias") else None
    res = normal(37, m, width).to(DEV, dtype) if how.get("residual") else None
    out = torch.full((m, width), float("nan"), device=DEV, dtype=dtype)
    p = ops.pack_8bit(w)
    torch.cuda.synchronize()                                  # with dependent launches W counts as a constant
    ops.gemm_8bit(a, sa, p, sw, out, bias=bias, act=how.get("act"), gated=gated, residual=res)
    check_product(out, a, sa, w, sw, bias, how.get("act"), gated, res)


@gpu
@pytest.mark.parametrize("how", EPILOGUES, ids=lambda d: "-".join(f"{k}={v}" for k, v in d.items()))
@pytest.mark.parametrize("m,n,k", [PAIRED[0], JOINED[0], LOW[0]])
def test_epilogues_of_pairs_and_of_the_join(m, n, k, how, dependent):
    run_product(m, n, k, how)
    run_product(m, n, k, how, torch.bfloat16)


@gpu
@pytest.mark.parametrize("m,n,k", [PAIRED[1], JOINED[1], LOW[1], (24, 2048, 2048), (64, 4096, 1024)])
def test_odd_sizes_of_pairs_and_of_the_join(m, n, k, dependent):
    run_product(m, n, k, dict(bias=True, act="silu", residual=True))
    run_product(m, n, k, dict(bias=True), torch.bfloat16)


def test_the_sizes_above_reach_those_kernels():
    for m, n, k in PAIRED + JOINED:
        for overlapped in (False, True):
            floats, clusters = ops.gemm_8bit_plan(m, n, ops.eight_bit_columns(k), overlapped)
            assert clusters == ((m, n, k) in PAIRED) and (floats > 0) == ((m, n, k) in JOINED)


@gpu
@pytest.mark.parametrize("m,n,k", PAIRED + JOINED + LOW)
def test_pairs_and_the_join_repeat_to_the_bit_and_rows_stay_apart(m, n, k):
    a, sa, w, sw = operands(41, m, n, k)
    p = ops.pack_8bit(w)
    first, second = torch.empty(m, n, device=DEV), torch.empty(m, n, device=DEV)
    ops.gemm_8bit(a, sa, p, sw, first)
    ops.gemm_8bit(a, sa, p, sw, second)
    assert torch.equal(first, second)
    changed, sb = a.clone(), sa.clone()
    changed.view(torch.uint8)[m // 2].fill_(0x7F)            # NaN
    sb[m // 2] = float("nan")
    sb[3] = 0
    changed.view(torch.uint8)[3] = 0
    bias = normal(42, n).to(DEV)
    ops.gemm_8bit(a, sa, p, sw, first, bias=bias)
    ops.gemm_8bit(changed, sb, p, sw, second, bias=bias)
    keep = [i for i in range(m) if i not in (3, m // 2)]
    assert torch.isnan(second[m // 2]).all() and torch.equal(second[3], bias) and torch.equal(second[keep], first[keep])


@gpu
@pytest.mark.parametrize("m", [1, 8, 20, 100, 300, 1100])
def test_a_product_repeats_to_the_bit_and_a_row_does_not_see_the_others(m):
    a, sa, w, sw = operands(40, m, 528, 1000)
    p = ops.pack_8bit(w)
    first, second = torch.empty(m, 528, device=DEV), torch.empty(m, 528, device=DEV)
    ops.gemm_8bit(a, sa, p, sw, first)
    ops.gemm_8bit(a, sa, p, sw, second)
    assert torch.equal(first, second)
    changed, sb = a.clone(), sa.clone()
    changed.view(torch.uint8)[0].fill_(0x7F)                 # NaN
    sb[0] = float("nan")
    ops.gemm_8bit(changed, sb, p, sw, second)
    assert torch.isnan(second[0]).all() and torch.equal(second[1:], first[1:])


@gpu
@pytest.mark.parametrize("m", [1, 8, 40, 300])
def test_zero_rows_and_not_finite_ones(m):
    a, sa, w, sw = operands(50, m, 100, 256)
    sa[m // 2] = 0
    a.view(torch.uint8)[m // 2] = 0
    bias = normal(51, 100).to(DEV)
    out = torch.empty(m, 100, device=DEV)
    ops.gemm_8bit(a, sa, ops.pack_8bit(w), sw, out, bias=bias)
    assert torch.equal(out[m // 2], bias)
    sa[0] = float("inf")
    ops.gemm_8bit(a, sa, ops.pack_8bit(w), sw, out, bias=bias)
    assert not torch.isfinite(out[0]).any()


@gpu
@pytest.mark.parametrize("m", [4, 50, 600])
def test_another_stream(m):
    """Launches go to the current stream, behind what made their inputs there."""
    a, sa, w, sw = operands(60, m, 256, 512)
    p = ops.pack_8bit(w)
    want = torch.empty(m, 256, device=DEV)
    ops.gemm_8bit(a, sa, p, sw, want)
    x = normal(60, m, 512).to(DEV)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        b, sb = empty_rows(m, 512)
        out = torch.empty(m, 256, device=DEV)
        ops.rows_8bit(x, b, sb)
        ops.gemm_8bit(b, sb, p, sw, out)
    side.synchronize()
    assert torch.equal(out, want)


@gpu
@pytest.mark.parametrize("m", [4, 50, 600])
def test_another_thread(m):
    """A thread whose first call this is."""
    import threading
    a, sa, w, sw = operands(65, m, 256, 512)
    p, got = ops.pack_8bit(w), []
    want, out = torch.empty(m, 256, device=DEV), torch.empty(m, 256, device=DEV)
    ops.gemm_8bit(a, sa, p, sw, want)
    torch.cuda.synchronize()

    def work():
        try:
            got.append(ops.gemm_8bit(a, sa, p, sw, out))
        except Exception as e:
            got.append(e)

    t = threading.Thread(target=work)
    t.start()
    t.join()
    torch.cuda.synchronize()
    assert got[0] is out and torch.equal(out, want)


@gpu
def test_products_in_a_graph():
    a, sa, w, sw = operands(70, 8, 256, 512)
    p = ops.pack_8bit(w)
    x, out, want = normal(70, 8, 512).to(DEV), torch.zeros(8, 256, device=DEV), torch.empty(8, 256, device=DEV)
    ops.gemm_8bit(a, sa, p, sw, want)
    ops.rows_8bit(x, a, sa)                                   # everything is loaded
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.rows_8bit(x, a, sa)
        ops.gemm_8bit(a, sa, p, sw, out)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


@gpu
def test_refusals():
    d = dict(device=DEV)
    x, w, out, scale = torch.zeros(4, 100, **d), torch.ones(100, **d), *empty_rows(4, 100)
    bad = [lambda: ops.rows_8bit(x.cpu(), out, scale), lambda: ops.rows_8bit(x.half(), out, scale), lambda: ops.rows_8bit(x, out[:, :100], scale),
           lambda: ops.rows_8bit(x, out.float(), scale), lambda: ops.rows_8bit(x, out, scale[:3]), lambda: ops.rows_8bit(x.t(), out, scale),
           lambda: ops.rows_8bit(x[0], out, scale), lambda: ops.rows_8bit(x[:3], out, scale),
           lambda: ops.rows_8bit(torch.zeros(4, 0, **d), torch.zeros(4, 0, **d).to(F8), scale),
           lambda: ops.add_rmsnorm_8bit(x, None, w[:99], 1e-6, out, scale), lambda: ops.add_rmsnorm_8bit(x.bfloat16(), None, w, 1e-6, out, scale),
           lambda: ops.add_rmsnorm_8bit(x, x[:3], w, 1e-6, out, scale), lambda: ops.add_rmsnorm_8bit(x, x.half(), w, 1e-6, out, scale),
           lambda: ops.add_rmsnorm_8bit(x, x, w, 1e-6, out, scale, rows=torch.zeros(4, dtype=torch.int64, **d)),
           lambda: ops.add_rmsnorm_8bit(x, x, w, 1e-6, out, scale, rows=torch.zeros(3, dtype=torch.int32, **d)),
           lambda: ops.add_rmsnorm_8bit(x, x, w, 1e-6, out, scale, into=x[:2]),
           lambda: ops.pack_8bit(torch.zeros(4, 100, **d).to(F8)), lambda: ops.pack_8bit(torch.zeros(4, 128, **d)),
           lambda: ops.pack_8bit(torch.zeros(0, 128, **d).to(F8))]
    for f in bad:
        with pytest.raises(ops.KernelError):
            f()
    a, sa, wv, sw = operands(80, 4, 32, 100)
    p, y = ops.pack_8bit(wv), torch.zeros(4, 32, **d)
    good = dict(a=a, a_scale=sa, w=p, w_scale=sw, out=y)
    ops.gemm_8bit(**good)
    half = torch.zeros(4, 16, **d)
    for change in (dict(a=a[:3]), dict(a=a.float()), dict(a_scale=sa[:3]), dict(w=p[:1]), dict(w=wv), dict(w_scale=sw[:16]), dict(out=y.half()),
                   dict(out=y.t()), dict(out=half), dict(bias=sw[:31]), dict(bias=sw.bfloat16()), dict(act="softmax"), dict(act="capped_swish"),
                   dict(residual=y.bfloat16()), dict(residual=half), dict(gated=True), dict(gated=True, out=half), dict(gated=True, act="gelu", out=half),
                   dict(a=a.cpu()), dict(a=torch.zeros(4, 256, **d).to(F8))):
        with pytest.raises(ops.KernelError):
            ops.gemm_8bit(**{**good, **change})
    shifted = torch.zeros(4 * 128 + 8, **d).to(F8)[8:].view(4, 128)
    with pytest.raises(ops.KernelError):                     # rows begin on 16-byte boundaries
        ops.gemm_8bit(**{**good, "a": shifted})
    with pytest.raises(ops.KernelError):
        ops.gemm_8bit(a, sa, ops.pack_8bit(torch.zeros(40, 128, **d).to(F8)), torch.zeros(40, **d), torch.zeros(4, 20, **d), act="silu", gated=True)


def test_what_a_product_wants():
    """Scratch memory holds every part of a shared K; few rows want neither scratch nor clusters, many rows clusters."""
    for n, columns in ((16, 128), (4096, 12288), (24576, 4096), (1003, 1024)):
        for m in (1, 8, 16):
            assert ops.gemm_8bit_plan(m, n, columns) == (0, False)
        for m in (17, 24, 64, 128, 300, 512):
            floats, clusters = ops.gemm_8bit_plan(m, n, columns)
            parts, rest = divmod(floats, m * -(-n // 128) * 128)
            assert rest == 0 and parts in (0, 2, 3, 4, 5, 6, 7, 8) and not (parts and clusters) and parts <= max(1, columns // 128)
    assert ops.gemm_8bit_plan(64, 4096, 12288)[0] and ops.gemm_8bit_plan(4096, 4096, 12288) == (0, True)
    with pytest.raises(ops.KernelError):
        ops.gemm_8bit_plan(64, 4096, 100)


@gpu
def test_scratch_of_the_callers():
    a, sa, w, sw = operands(90, 64, 4096, 12288)
    p, floats = ops.pack_8bit(w), ops.gemm_8bit_plan(64, 4096, 12288)[0]
    assert floats
    want, out = torch.empty(64, 4096, device=DEV), torch.empty(64, 4096, device=DEV)
    ops.gemm_8bit(a, sa, p, sw, want)
    ops.gemm_8bit(a, sa, p, sw, out, scratch=torch.full((floats + 5,), float("nan"), device=DEV))
    assert torch.equal(out, want)
    for bad in (torch.empty(floats - 1, device=DEV), torch.empty(floats, device=DEV, dtype=torch.float64), torch.empty(floats)):
        with pytest.raises(ops.KernelError):
            ops.gemm_8bit(a, sa, p, sw, out, scratch=bad)


def test_columns_of_a_row():
    assert [ops.eight_bit_columns(k) for k in (1, 128, 129, 4096, 4097)] == [128, 128, 256, 4096, 4224]


def test_tensors_on_the_cpu_are_refused():
    x = torch.zeros(2, 128)
    with pytest.raises(ops.KernelError):
        ops._say_what_is_wrong(x, torch.float32, "x", 2)
