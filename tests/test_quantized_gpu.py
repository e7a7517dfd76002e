"""The operators of quantised linear layers on the device against plain restatements in 64 bits: rows to e4m3 with and without the
residual sum and the norm, the product of 8-bit rows with 8-bit weights, the product with 4-bit weights.

Tolerances.  A rounding is off by at most half a step: 2^-8 of the value for bfloat16.  A float32 sum of k terms, in whatever
order, is off by at most k 2^-23 of the sum of the terms' magnitudes (2^-24 a rounding; the tensor cores may cut instead of
round, which is at most twice that).  Whole numbers whose sums stay below 2^24 are exact, and then so is the result."""
import pytest
import torch

from fms_b200.kernels.build import load_library

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
HALF_STEP = 2.0 ** -8  # of bfloat16, relative
E4M3 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def ops():
    from fms_b200.kernels import ops as o

    yield o
    o.check_error_flag("cuda")


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def normal(g, *shape, std=1.0):
    return torch.empty(shape, dtype=F32, device="cuda").normal_(0.0, std, generator=g)


def whole(g, lo, hi, *shape):
    return torch.randint(lo, hi + 1, shape, generator=g, device="cuda")


def nearest_e4m3(v):
    """float64 -> (nearest e4m3 value, ties to even; how far from a tie, in steps)."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    n = v / step
    return (torch.round(n) * step).clamp(-448, 448), ((n - torch.floor(n)) - 0.5).abs()


# ---- rows to e4m3 ----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,dim", [(1, 1), (3, 7), (5, 16), (2, 17), (9, 240), (300, 129), (7, 4096), (4, 5001), (300, 14336), (3, 33000)])
def test_quantize_rows(ops, dtype, rows, dim):
    x = (normal(gen(rows + dim), rows, dim) * 3).to(dtype)
    y = ops.quantize_rows(x)
    most = x.double().abs().amax(1, keepdim=True)
    scale = (most[:, 0] / 448).float()
    want, _ = nearest_e4m3(x.double() * 448 / most)
    assert y.values.dtype == E4M3 and y.shape == (rows, dim) and y.values.shape[1] % 16 == 0
    assert torch.equal(y.scales, scale)
    assert torch.equal(y.values[:, :dim].double(), want)
    assert int(y.values[:, dim:].view(torch.uint8).sum()) == 0
    # what they stand for is within half a step of a value's own binade (1/16 relative), or of the smallest (2^-10 of a scale)
    back = y.dequantize()
    assert bool(((back - x.float()).abs() <= x.float().abs() * 2.0 ** -4 * (1 + 2.0 ** -20) + scale[:, None] * 2.0 ** -10).all())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("off", [1, 2, 3, 5])
@pytest.mark.parametrize("rows,dim", [(3, 64), (4, 517), (300, 1000), (5, 8193), (2, 33001)])
def test_rows_that_begin_anywhere(ops, dtype, rows, dim, off):
    g = gen(off + dim)
    moved = lambda t: torch.cat((t.new_zeros(off), t.reshape(-1)))[off:].view(t.shape)  # noqa: E731
    x, res, gain = normal(g, rows, dim).to(dtype), normal(g, rows, dim), (1 + normal(g, dim, std=0.1)).to(dtype)
    a, b = ops.quantize_rows(x), ops.quantize_rows(moved(x))
    assert torch.equal(a.values.view(torch.uint8), b.values.view(torch.uint8)) and torch.equal(a.scales, b.scales)
    first, other = res.clone(), moved(res)
    a = ops.add_rmsnorm_quantized(first, x, gain, 1e-5)
    for b in (ops.add_rmsnorm_quantized(other, x, gain, 1e-5), ops.add_rmsnorm_quantized(res.clone(), moved(x), moved(gain), 1e-5)):
        assert torch.equal(a.values.view(torch.uint8), b.values.view(torch.uint8))
        # the same squares in another order: as far apart as either may be from the exact scale
        torch.testing.assert_close(a.scales, b.scales, atol=0, rtol=2 * 2.0 ** -24 * (max(34, dim / 256) / 2 + 10))
    assert torch.equal(first, other)


def test_quantize_rows_of_zeros_tiny_and_not_finite(ops):
    x = normal(gen(1), 8, 70)
    x[1] = 0.0
    x[2] = -0.0
    x[3] = 3e-32  # a scale below 2^-110
    x[4, 5] = float("nan")
    x[5, 0] = float("inf")
    x[6] *= 1e30
    y = ops.quantize_rows(x)
    alone = ops.quantize_rows(x[[0, 7]].contiguous())
    assert torch.equal(y.values[[0, 7]].view(torch.uint8), alone.values.view(torch.uint8)) and torch.equal(y.scales[[0, 7]], alone.scales)
    for r in (1, 2, 3):
        assert float(y.scales[r]) == 0.0 and float(y.values[r].float().abs().max()) == 0.0
    assert not torch.isfinite(y.scales[4]) and not torch.isfinite(y.scales[5])
    assert int(y.values[:, 70:].view(torch.uint8).sum()) == 0
    assert bool(torch.isfinite(y.scales[6])) and float(y.values[6].float().abs().max()) == 448.0


@pytest.mark.parametrize("dtype", [BF16, F32, None])
@pytest.mark.parametrize("gain_dtype", [BF16, F32])
@pytest.mark.parametrize("rows,dim,eps", [(1, 1, 1e-5), (5, 240, 1e-5), (3, 17, 1e-6), (2, 5001, 1e-3), (300, 4096, 1e-5), (4, 8192, 1e-5), (300, 16384, 1e-5), (3, 20000, 1e-5)])
def test_add_rmsnorm_quantized(ops, dtype, gain_dtype, rows, dim, eps):
    g = gen(rows * dim)
    res = normal(g, rows, dim) * 3
    delta = None if dtype is None else normal(g, rows, dim).to(dtype)
    gain = (1 + normal(g, dim, std=0.1)).to(gain_dtype)
    total = res.clone() if delta is None else res + delta.float()
    y = ops.add_rmsnorm_quantized(res, delta, gain, eps)
    assert torch.equal(res, total)
    t = total.double() * gain.double()
    norm = t / (total.double().square().mean(1, keepdim=True) + eps).sqrt()
    # the sum of squares: up to 24 terms a thread and 10 levels, halved by the root, rsqrtf's 2 units, six further roundings
    torch.testing.assert_close(y.scales.double(), norm.abs().amax(1) / 448, atol=0, rtol=2.0 ** -24 * (34 / 2 + 4 + 6))
    # t has at most 48 bits and t * 448 at most 51: the quotient is exact but for float64's last place, and exactly a tie where it is one
    want, _ = nearest_e4m3(t * 448 / t.abs().amax(1, keepdim=True))
    assert torch.equal(y.values[:, :dim].double(), want)
    assert int(y.values[:, dim:].view(torch.uint8).sum()) == 0


def test_add_rmsnorm_quantized_gathers_rows_and_leaves_the_stream(ops):
    g = gen(3)
    res, delta, gain = normal(g, 9, 112), normal(g, 9, 112).to(BF16), 1 + normal(g, 112, std=0.1)
    before = res.clone()
    rows = torch.tensor([7, 0, 7, 8], dtype=torch.int32, device="cuda")
    y = ops.add_rmsnorm_quantized(res, delta, gain, 1e-5, rows)
    assert torch.equal(res, before)
    whole_ = ops.add_rmsnorm_quantized(res, delta, gain, 1e-5)
    assert torch.equal(y.values.view(torch.uint8), whole_.values.view(torch.uint8)[rows.long()]) and torch.equal(y.scales, whole_.scales[rows.long()])
    none = ops.add_rmsnorm_quantized(res, None, gain, 1e-5, rows[:0])
    assert none.shape == (0, 112)


def test_add_rmsnorm_quantized_rows_of_zeros_and_not_finite(ops):
    g = gen(4)
    res, gain = normal(g, 5, 100), 1 + normal(g, 100, std=0.1)
    res[1] = 0.0
    res[2, 99] = float("nan")
    res[3, 0] = float("-inf")
    alone = ops.add_rmsnorm_quantized(res[[0, 4]].contiguous(), None, gain, 1e-5)
    y = ops.add_rmsnorm_quantized(res, None, gain, 1e-5)
    assert torch.equal(y.values[[0, 4]].view(torch.uint8), alone.values.view(torch.uint8)) and torch.equal(y.scales[[0, 4]], alone.scales)
    assert float(y.scales[1]) == 0.0 and float(y.values[1].float().abs().max()) == 0.0
    assert bool(torch.isnan(y.scales[2:4]).all())
    assert int(y.values[:, 100:].view(torch.uint8).sum()) == 0


@pytest.mark.parametrize("rows,dim", [(40, 1000), (2, 40)])
def test_ties_go_to_the_even_value(ops, rows, dim):
    """Whole numbers under a largest value of 7 * 2^n: x * 448 / max is a whole number of 64ths, so that many quotients lie exactly between
    two e4m3 values, normal and subnormal ones."""
    g = gen(rows)
    x = whole(g, -(7 << 13), 7 << 13, rows, dim).float()
    x[:, ::3] = whole(g, -40, 40, rows, x[:, ::3].shape[1]).float() * 7  # quotients of odd multiples of 2^-10 * 7 and the like
    x[:, 0] = 7 << 13
    want, border = nearest_e4m3(x.double() * 448 / (7 << 13))
    assert int((border == 0).sum()) > 0
    assert torch.equal(ops.quantize_rows(x).values[:, :dim].double(), want)
    y = ops.add_rmsnorm_quantized(x.clone(), None, torch.ones(dim, device="cuda"), 1e-5)
    assert torch.equal(y.values[:, :dim].double(), want)


# ---- products of 8-bit rows and weights --------------------------------------------------------------------------------
SHAPES = [(1, 1, 1), (1, 16, 16), (3, 37, 75), (8, 300, 128), (16, 129, 400), (17, 128, 256), (64, 200, 4096), (100, 72, 1000), (128, 130, 640),
          (129, 65, 136), (200, 1000, 272), (256, 256, 2048), (257, 100, 96), (300, 520, 1040), (513, 264, 640), (1100, 1536, 512),
          # equal runs of a multiprocessor's steps, joined by a second kernel; more tiles than multiprocessors
          (5, 72, 2600), (130, 1000, 2500), (256, 2100, 4100), (33, 20000, 96), (200, 38000, 64)]


def e4m3_case(m, n, k, seed, big=8):
    """Whole numbers of up to ``big`` (e4m3 holds those up to 16) and scales that are powers of two."""
    g = gen(seed)
    x, w = whole(g, -big, big, m, k).float(), whole(g, -big, big, n, k).float()
    sx, sw = 2.0 ** whole(g, -3, 3, m).float(), 2.0 ** whole(g, -3, 3, n).float()
    return x, w, sx, sw, normal(g, n)


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_linear_e4m3_whole_numbers_are_exact(ops, m, n, k):
    x, w, sx, sw, _ = e4m3_case(m, n, k, m + n + k)
    y = ops.linear_e4m3(ops.QuantizedRows.of(x.to(E4M3), sx), ops.e4m3_weight(w.to(E4M3), sw), None, F32)
    want = (x.double() @ w.double().t()) * sx.double()[:, None] * sw.double()[None, :]
    assert torch.equal(y.double(), want)


@pytest.mark.parametrize("out_dtype", [BF16, F32])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("m,n,k", SHAPES[2:])
def test_linear_e4m3(ops, m, n, k, out_dtype, biased):
    g = gen(m * n + k)
    x, w = ops.quantize_rows(normal(g, m, k).to(BF16)), ops.quantize_e4m3(normal(g, n, k, std=0.02))
    bias = normal(g, n).to(BF16) if biased else None
    y = ops.linear_e4m3(x, w, bias, out_dtype)
    xd, wd = x.values[:, :k].double() * x.scales.double()[:, None], w.rows.values[:, :k].double() * w.rows.scales.double()[:, None]
    want = xd @ wd.t() + (0 if bias is None else bias.double())
    # the sum, the scales' product and its product with the sum, the bias; then the rounding to the result's type
    bound = (k + 4) * 2.0 ** -23 * (xd.abs() @ wd.abs().t()) + 2.0 ** -24 * want.abs() + (HALF_STEP * want.abs() if out_dtype == BF16 else 0) + 1e-30
    assert y.dtype == out_dtype and bool(((y.double() - want).abs() <= bound).all())
    assert torch.equal(ops.linear(x, w, bias, out_dtype), y)


@pytest.mark.parametrize("k", [1040, 2576])
@pytest.mark.parametrize("m", [1, 7, 40, 256, 300])
def test_a_row_of_linear_e4m3_does_not_depend_on_the_others(ops, m, k):
    g = gen(m)
    x, w = ops.quantize_rows(normal(g, m, k)), ops.quantize_e4m3(normal(g, 520, k, std=0.02))
    y = ops.linear_e4m3(x, w, None, F32)
    x.values.view(torch.uint8)[: m - 1] = 0x7F  # NaN
    x.scales[: m - 1] = float("nan")
    z = ops.linear_e4m3(x, w, None, F32)
    assert torch.equal(z[m - 1], y[m - 1]) and bool(torch.isnan(z[: m - 1]).all())
    if m <= 256:  # the same kernel for fewer rows
        few = ops.linear_e4m3(ops.QuantizedRows(x.values[m - 1:], x.scales[m - 1:], x.dim), w, None, F32)
        assert torch.equal(few[0], y[m - 1])


@pytest.mark.parametrize("act", [0, 1, 2, 3])
@pytest.mark.parametrize("m,hidden,k", [(1, 5, 40), (8, 200, 256), (33, 100, 512), (250, 72, 144), (300, 300, 512), (1100, 264, 256),
                                        (7, 300, 2600), (256, 1000, 4100), (33, 9600, 144), (130, 19000, 64)])
def test_gated_linear_e4m3(ops, act, m, hidden, k):
    g = gen(act + m)
    x, w = ops.quantize_rows(normal(g, m, k)), ops.quantize_e4m3(normal(g, 2 * hidden, k, std=k ** -0.5))
    bias = normal(g, 2 * hidden, std=0.1).to(BF16)
    y = ops.gated_linear_e4m3(x, w, bias, act)
    xd, wd = x.values[:, :k].double() * x.scales.double()[:, None], w.rows.values[:, :k].double() * w.rows.scales.double()[:, None]
    z = xd @ wd.t() + bias.double()
    off = (k + 4) * 2.0 ** -23 * (xd.abs() @ wd.abs().t()) + 2.0 ** -22 * z.abs()
    gate, up = z[:, :hidden], z[:, hidden:]
    f = torch.nn.functional
    a = [f.silu, f.gelu, lambda t: f.gelu(t, approximate="tanh"), torch.relu][act](gate)
    # slopes of these activations stay below 1.2; expf, erff and tanhf are good to a few units of float32 in 1
    a_off = 1.2 * off[:, :hidden] + 2.0 ** -20 * (a.abs() + gate.abs())
    bound = a_off * up.abs() + (a.abs() + a_off) * off[:, hidden:] + (HALF_STEP + 2.0 ** -23) * ((a * up).abs() + a_off * up.abs()) + 1e-30
    assert bool(((y.double() - a * up).abs() <= bound).all())
    assert torch.equal(ops.gated_linear(x, w, bias, act), y)


# ---- products with 4-bit weights ---------------------------------------------------------------------------------------
INT4_SHAPES = [(1, 1, 8, 32), (1, 40, 32, 32), (3, 37, 72, 64), (8, 300, 128, 128), (8, 129, 1000, 32), (9, 200, 640, 128), (16, 10000, 256, 64), (16, 72, 4096, 4096),
               (5, 9600, 384, 128), (17, 128, 256, 128), (33, 130, 640, 64), (64, 264, 4096, 128), (100, 72, 1000, 32), (112, 4096, 512, 96), (128, 2100, 384, 256),
               (129, 65, 136, 1000), (256, 256, 2048, 128), (257, 100, 96, 32), (600, 264, 1160, 160),
               # runs of a warp that reach into the next tile, with odd ends; more tiles than a thread block has warps
               (2, 4720, 1288, 128), (7, 7120, 648, 64), (3, 2400, 2056, 32), (4, 90000, 136, 128), (1, 80000, 32, 32)]


def int4_case(m, n, k, group, zeros, seed):
    g = gen(seed)
    groups = -(-k // min(group, (k + 31) // 32 * 32))
    q = whole(g, 0, 15, n, k).to(torch.uint8)
    z = whole(g, 0, 15, n, groups).to(torch.uint8) if zeros else None
    at = torch.arange(k, device="cuda") // group
    centred = q.double() - (z.double()[:, at] if zeros else 8.0)
    return g, q, z, centred, groups, at


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("m,n,k,group", INT4_SHAPES)
def test_linear_int4_whole_numbers_are_exact(ops, m, n, k, group, zeros):
    g, q, z, centred, groups, at = int4_case(m, n, k, group, zeros, m + n + k)
    scales = 2.0 ** whole(g, -2, 2, n, groups).float()
    x = whole(g, -1, 1, m, k).float() * 2.0 ** whole(g, 0, 1, m, 1).float()
    w = ops.pack_int4(q, scales, z, group)
    assert torch.equal(w.dequantize().double(), centred * scales.double()[:, at])
    want = x.double() @ (centred * scales.double()[:, at]).t()
    assert torch.equal(ops.linear_int4(x.to(BF16), w), want.float().to(BF16))  # exact in float32, rounded once


# with the rows of x that a pair's tile has on 148 multiprocessors
PAIR_TILES = [(270, 616, 136, 128, 96), (300, 6144, 136, 64, 128), (307, 4840, 392, 32, 128), (520, 4840, 136, 128, 192), (307, 6248, 136, 128, 160),
              (407, 6248, 264, 64, 224), (700, 6144, 136, 128, 256), (720, 4840, 264, 256, 256)]


@pytest.mark.parametrize("m,n,k,group,tile", PAIR_TILES)
def test_linear_int4_of_tiles_of_every_width(ops, m, n, k, group, tile):
    if torch.cuda.get_device_properties(0).multi_processor_count == 148:
        assert load_library("gemm_int4").fms_linear_int4_tile(m, n) == tile
    g, q, z, centred, groups, at = int4_case(m, n, k, group, True, m + n + k)
    scales = 2.0 ** whole(g, -2, 2, n, groups).float()
    x = whole(g, -1, 1, m, k).float() * 2.0 ** whole(g, 0, 1, m, 1).float()
    want = x.double() @ (centred * scales.double()[:, at]).t()
    assert torch.equal(ops.linear_int4(x.to(BF16), ops.pack_int4(q, scales, z, group)), want.float().to(BF16))


@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("m,n,k,group", INT4_SHAPES)
def test_linear_int4(ops, m, n, k, group, biased):
    g, q, z, centred, groups, at = int4_case(m, n, k, group, biased, m * n + k)
    scales = (0.002 + 0.01 * normal(g, n, groups).abs()).to(BF16)
    x, bias = normal(g, m, k).to(BF16), normal(g, n).to(BF16) if biased else None
    y = ops.linear_int4(x, ops.pack_int4(q, scales, z, group), bias)
    w = centred * scales.double()[:, at]
    if m > 8:
        w = w.float().to(BF16).double()  # q - z times s is exact in float32: rounded once, to what the tensor cores multiply
    want = x.double() @ w.t() + (0 if bias is None else bias.double())
    bound = (k + 4) * 2.0 ** -23 * (x.double().abs() @ w.abs().t()) + (HALF_STEP + 2.0 ** -24) * want.abs() + 1e-30
    assert y.dtype == BF16 and bool(((y.double() - want).abs() <= bound).all())
    assert torch.equal(ops.linear(x, ops.pack_int4(q, scales, z, group), bias), y)


@pytest.mark.parametrize("m", [1, 8, 16, 17, 40, 300])
def test_a_row_of_linear_int4_does_not_depend_on_the_others(ops, m):
    g = gen(m)
    w = ops.quantize_int4(normal(g, 520, 1040, std=0.02), 128)
    x = normal(g, m, 1040).to(BF16)
    y = ops.linear_int4(x, w)
    x[: m - 1] = float("nan")
    z = ops.linear_int4(x, w)
    assert torch.equal(z[m - 1], y[m - 1]) and bool(torch.isnan(z[: m - 1].float()).all())


@pytest.mark.parametrize("act", [0, 1, 2, 3])
@pytest.mark.parametrize("m,hidden,k,group", [(1, 5, 40, 32), (1, 16, 136, 32), (8, 208, 256, 128), (8, 4992, 256, 64), (16, 4800, 384, 32), (9, 80, 1040, 1040), (16, 72, 144, 144), (17, 200, 256, 128),
                                              (3, 4720, 1288, 128), (6, 2400, 648, 64), (2, 40000, 136, 128), (5, 39984, 72, 32)])
def test_gated_linear_int4(ops, act, m, hidden, k, group):
    g = gen(act + m)
    w = ops.quantize_int4(normal(g, 2 * hidden, k, std=k ** -0.5), group)
    x, bias = normal(g, m, k).to(BF16), normal(g, 2 * hidden, std=0.1).to(BF16)
    y = ops.gated_linear_int4(x, w, bias, act)
    wd = w.dequantize().double()
    if m > 8 or hidden % 16:
        two = ops.gated_activation(ops.linear_int4(x, w, bias), act)
        assert torch.equal(y, two)
        return
    z = x.double() @ wd.t() + bias.double()
    off = (k + 4) * 2.0 ** -23 * (x.double().abs() @ wd.abs().t()) + 2.0 ** -22 * z.abs()
    gate, up = z[:, :hidden], z[:, hidden:]
    f = torch.nn.functional
    a = [f.silu, f.gelu, lambda t: f.gelu(t, approximate="tanh"), torch.relu][act](gate)
    a_off = 1.2 * off[:, :hidden] + 2.0 ** -20 * (a.abs() + gate.abs())
    bound = a_off * up.abs() + (a.abs() + a_off) * off[:, hidden:] + (HALF_STEP + 2.0 ** -23) * ((a * up).abs() + a_off * up.abs()) + 1e-30
    assert bool(((y.double() - a * up).abs() <= bound).all())


# ---- together, and as they are called ----------------------------------------------------------------------------------
def test_none_of_no_rows(ops):
    w8, w4 = ops.quantize_e4m3(torch.ones(32, 64, device="cuda")), ops.quantize_int4(torch.ones(32, 64, device="cuda"), 32)
    x = torch.empty(0, 64, dtype=BF16, device="cuda")
    assert ops.quantize_rows(x).shape == (0, 64)
    assert ops.linear_e4m3(ops.quantize_rows(x), w8).shape == (0, 32) and ops.linear_int4(x, w4).shape == (0, 32)
    assert ops.gated_linear_e4m3(x, w8, None, 0).shape == (0, 16) and ops.gated_linear_int4(x, w4, None, 0).shape == (0, 16)
    assert ops.add_rmsnorm_quantized(torch.empty(0, 64, device="cuda"), None, torch.ones(64, device="cuda"), 1e-5).shape == (0, 64)


def run_of_them(ops, res, delta, gain, w8, w4):
    h = ops.add_rmsnorm_quantized(res, delta, gain, 1e-5)
    a = ops.linear_e4m3(h, w8)
    return ops.linear_int4(ops.linear_e4m3(ops.quantize_rows(ops.linear_int4(a, w4)), w8), w4)


@pytest.mark.parametrize("rows", [3, 20, 300])
def test_a_run_of_them_captured_replayed_and_on_another_stream(ops, rows):
    g = gen(rows)
    w8, w4 = ops.quantize_e4m3(normal(g, 512, 512, std=0.05)), ops.quantize_int4(normal(g, 512, 512, std=0.05), 64)
    res, delta, gain = normal(g, rows, 512), normal(g, rows, 512).to(BF16), 1 + normal(g, 512, std=0.1)
    start = res.clone()
    want = run_of_them(ops, res, delta, gain, w8, w4)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for s in streams:  # two at once
        with torch.cuda.stream(s):
            mine = start.clone()
            for _ in range(3):
                mine.copy_(start)
                y = run_of_them(ops, mine, delta, gain, w8, w4)
            got.append(y)
    torch.cuda.synchronize()
    assert all(torch.equal(y, want) for y in got)
    graphs, held = [], start.clone()
    for _ in range(2):  # two captured graphs share nothing but the inputs
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held.copy_(start)
            y = run_of_them(ops, held, delta, gain, w8, w4)
        graphs.append((graph, y))
    for _ in range(3):
        for graph, y in graphs:
            y.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, want)


def test_tensor_memory_is_given_back(ops):
    """Blocks that share a multiprocessor's tensor memory, many times over, and then kernels that want all of it."""
    g = gen(5)
    many, few = ops.quantize_e4m3(normal(g, 28672, 512, std=0.04)), ops.quantize_e4m3(normal(g, 512, 2576, std=0.02))
    int4, bf16 = ops.quantize_int4(normal(g, 512, 512, std=0.04)), normal(g, 512, 512).to(BF16)
    x, long, wide = ops.quantize_rows(normal(g, 32, 512)), ops.quantize_rows(normal(g, 32, 2576)), ops.quantize_rows(normal(g, 600, 512))
    xb, wideb = normal(g, 32, 512).to(BF16), normal(g, 600, 512).to(BF16)

    def run():
        return [ops.gated_linear_e4m3(x, many, None, 0), ops.linear_e4m3(x, many), ops.linear_e4m3(long, few), ops.linear_int4(xb, int4), ops.linear(xb, bf16)]

    def whole():
        return [ops.linear_e4m3(wide, many), ops.linear_int4(wideb, int4), ops.linear(wideb, bf16)]

    first, all_of_it = run(), whole()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        captured = [y for _ in range(8) for y in run()]
    for _ in range(25):
        graph.replay()
        again = whole()
    for y, want in zip(captured + again, 8 * first + all_of_it):
        assert torch.equal(y, want)


@pytest.mark.parametrize("kind", ["e4m3", "int4"])
def test_layers_of_long_prompts_back_to_back(ops, kind):
    """Many layers' launches in the queue at once, those of the pairs of thread blocks among kernels of thousands of blocks."""
    g = gen(6)
    make = ops.quantize_e4m3 if kind == "e4m3" else ops.quantize_int4
    qkv, dense = make(normal(g, 1536, 1024, std=0.03)), make(normal(g, 1024, 1024, std=0.03))
    wide, down = make(normal(g, 4096, 1024, std=0.03)), make(normal(g, 1024, 2048, std=0.03))
    head, gain = normal(g, 4000, 1024).to(BF16), torch.ones(1024, device="cuda", dtype=BF16)
    start = normal(g, 8192, 1024)

    def norm(residual, delta, rows=None):
        if kind == "e4m3":
            return ops.add_rmsnorm_quantized(residual, delta, gain, 1e-5, rows)
        return ops.add_rmsnorm(residual, delta, gain, 1e-5, BF16, rows)

    def run():
        residual, delta = start.clone(), None
        for _ in range(12):
            a = ops.linear(norm(residual, delta), qkv)
            delta = ops.linear(a[:, :1024].contiguous(), dense)
            delta = ops.linear(ops.gated_linear(norm(residual, delta), wide, None, 0), down)
        rows = torch.arange(31, 8192, 256, device="cuda", dtype=torch.int32)
        last = ops.add_rmsnorm(residual, delta, gain, 1e-5, BF16, rows)
        return ops.linear(last, head)

    first = run()
    for _ in range(6):
        again = run()
    assert bool(torch.isfinite(first).all()) and torch.equal(again, first)


def test_calls_on_two_streams_at_once(ops):
    g = gen(8)
    e4m3, int4 = ops.quantize_e4m3(normal(g, 6144, 2576, std=0.02)), ops.quantize_int4(normal(g, 6144, 2576, std=0.02))
    xs = [normal(g, rows, 2576).to(BF16) for rows in (1, 8, 40, 200, 700)]

    def run():
        return [f for x in xs for f in (ops.linear_e4m3(x, e4m3), ops.gated_linear_e4m3(x, e4m3, None, 1), ops.linear_int4(x, int4),
                                        ops.gated_linear_int4(x, int4, None, 1))]

    want = run()
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [None, None]
    for _ in range(10):
        for i, stream in enumerate(streams):  # the one's launches run beside the other's
            with torch.cuda.stream(stream):
                got[i] = run()
    torch.cuda.synchronize()
    for ys in got:
        for y, w in zip(ys, want):
            assert torch.equal(y, w)


def test_weights_straight_after_what_makes_them(ops):
    """A product asks for its weights before the kernel in front of it is done; the weight's constructor has waited for them."""
    g = gen(9)
    for _ in range(5):
        raw, x = normal(g, 4096, 2048, std=0.02), normal(g, 8, 2048).to(BF16)
        y8 = ops.linear_e4m3(x, ops.quantize_e4m3(raw))
        y4 = ops.linear_int4(x, ops.quantize_int4(raw))
        torch.cuda.synchronize()
        assert torch.equal(ops.linear_e4m3(x, ops.quantize_e4m3(raw)), y8) and torch.equal(ops.linear_int4(x, ops.quantize_int4(raw)), y4)


def test_refusals_on_the_device(ops):
    E = ops.KernelError
    x, w = torch.ones(4, 64, dtype=BF16, device="cuda"), torch.ones(32, 64, device="cuda")
    w8, w4 = ops.quantize_e4m3(w), ops.quantize_int4(w, 32)
    for call in (
        lambda: ops.quantize_rows(x.t()),                                                          # not contiguous
        lambda: ops.quantize_rows(x.half()),
        lambda: ops.quantize_rows(x[0]),
        lambda: ops.add_rmsnorm_quantized(x, None, x[0], 1e-5),                                    # a bfloat16 stream
        lambda: ops.add_rmsnorm_quantized(x.float(), x[:2], x[0], 1e-5),
        lambda: ops.add_rmsnorm_quantized(x.float(), x, x[0, :8].contiguous(), 1e-5),
        lambda: ops.add_rmsnorm_quantized(x.float(), x, x[0], 1e-5, torch.zeros(1, dtype=torch.int64, device="cuda")),
        lambda: ops.linear_e4m3(x[:, :32].contiguous(), w8),
        lambda: ops.linear_e4m3(x, w8, None, torch.float16),
        lambda: ops.linear_e4m3(x, w8, torch.ones(31, device="cuda")),
        lambda: ops.linear_e4m3(x, w4),
        lambda: ops.linear_int4(x.float(), w4),
        lambda: ops.linear_int4(x[:, :32].contiguous(), w4),
        lambda: ops.linear_int4(ops.quantize_rows(x), w4),
        lambda: ops.linear_int4(x, w8),
        lambda: ops.linear_int4(torch.ones(1 + 4 * 64, dtype=BF16, device="cuda")[1:].view(4, 64), w4),  # not 16-byte aligned
        lambda: ops.linear(x, w4, None, F32),
        lambda: ops.gated_linear_e4m3(x, ops.quantize_e4m3(w[:31]), None, 0),
        lambda: ops.gated_linear_e4m3(x, w8, None, 7),
        lambda: ops.gated_linear_int4(x, w4, None, 7),
        lambda: ops.linear_int4(x.cpu(), w4),
    ):
        with pytest.raises(E):
            call()
    with pytest.raises(E):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops.quantize_e4m3(w)
    torch.cuda.synchronize()
    assert ops.linear_int4(x, w4).shape == (4, 32)


# ---- behind a kernel that is still running -------------------------------------------------------------------------------
def behind(make, use, inputs):
    """``use(make(x))`` captured as one graph and replayed with other inputs in the same buffers, against the same kernels one at a time."""
    held = inputs[0].clone()
    use(make(held))  # libraries are loaded
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = use(make(held))
    got = []
    for x in inputs:
        held.copy_(x)
        graph.replay()
        got.append(y.clone())
    for x, y in zip(inputs, got):
        made = make(x)
        torch.cuda.synchronize()
        want = use(made)
        torch.cuda.synchronize()
        assert torch.equal(y, want)


@pytest.mark.parametrize("m", [1, 8, 40, 200, 700])
@pytest.mark.parametrize("kind", ["e4m3", "int4", "gated e4m3", "gated int4"])
def test_a_bias_that_the_kernel_before_writes(ops, kind, m):
    """A matrix-vector product of some 20 us writes the bias, and the product behind it starts while it runs."""
    n, k = 1024, 4096
    g = gen(m)
    wide, raw, x = normal(g, n, 16384, std=0.01).to(BF16), normal(g, n, k, std=0.02), normal(g, m, k).to(BF16)
    w = ops.quantize_e4m3(raw) if "e4m3" in kind else ops.quantize_int4(raw)
    rows = ops.quantize_rows(x) if "e4m3" in kind else x
    inputs = [normal(g, 1, 16384, std=2.0 ** i).to(BF16) for i in range(4)]
    torch.cuda.synchronize()

    def use(bias):
        return ops.gated_linear(rows, w, bias[0], 0) if "gated" in kind else ops.linear(rows, w, bias[0], BF16)

    behind(lambda held: ops.linear(held, wide), use, inputs)


@pytest.mark.parametrize("rows,dim", [(8, 4096), (300, 4096), (5, 1001)])
def test_a_gain_that_the_kernel_before_writes(ops, rows, dim):
    g = gen(rows)
    wide, res, delta = normal(g, dim, 16384, std=0.01).to(BF16), normal(g, rows, dim), normal(g, rows, dim).to(BF16)
    inputs = [normal(g, 1, 16384, std=2.0 ** i).to(BF16) for i in range(4)]
    picked = torch.arange(rows, dtype=torch.int32, device="cuda")

    def use(gain):
        y = ops.add_rmsnorm_quantized(res, delta, gain[0], 1e-5, picked)  # of gathered rows: the stream stays as it is
        return torch.cat((y.values.view(torch.uint8).flatten(), y.scales.view(torch.uint8)))

    behind(lambda held: ops.linear(held, wide), use, inputs)


@pytest.mark.parametrize("rows", [1, 3, 8, 20, 300])
@pytest.mark.parametrize("dim", [512, 520])
def test_a_run_of_them_replayed_with_other_inputs(ops, rows, dim):
    """Every buffer between the operators holds other values with every replay: none may be those of the replay before."""
    g = gen(rows + dim)
    w8, w4 = ops.quantize_e4m3(normal(g, dim, dim, std=0.05)), ops.quantize_int4(normal(g, dim, dim, std=0.05), 64)
    b8, b4 = ops.quantize_e4m3(normal(g, 2 * dim, dim, std=0.05)), ops.quantize_int4(normal(g, 2 * dim, dim, std=0.05))
    res, gain = normal(g, rows, dim), 1 + normal(g, dim, std=0.1)
    inputs = [normal(g, rows, dim, std=2.0 ** (i % 3)).to(BF16) for i in range(6)]

    def run(delta):
        stream = res.clone()
        a = ops.linear_int4(ops.linear_e4m3(ops.add_rmsnorm_quantized(stream, delta, gain, 1e-5), w8), w4)
        b = ops.linear_e4m3(ops.quantize_rows(ops.gated_linear_int4(a, b4, None, 0)), w8)
        c = ops.gated_linear_e4m3(ops.add_rmsnorm_quantized(stream, b, gain, 1e-5), b8, None, 0)
        return torch.cat((ops.linear_int4(c, w4).float(), stream))

    behind(lambda held: held * 1, run, inputs)


# ---- biases ----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, BF16, torch.float16])
@pytest.mark.parametrize("m,n,k", [(1, 40, 72), (8, 320, 128), (9, 200, 640), (40, 72, 2600), (100, 1000, 272), (200, 20000, 96), (300, 520, 1040)])
def test_a_bias_of_more_bits_keeps_them(ops, m, n, k, dtype):
    """Whole numbers below 2^12 and a bias of 16 bits behind the point: their sum in float32 is exact up to its one rounding."""
    g = gen(m + n + k)
    x, w = whole(g, -1, 1, m, k).float(), whole(g, -1, 1, n, k).float()
    bias = ((whole(g, -2 ** 20, 2 ** 20, n).double() + 0.5) * 2.0 ** -16).to(dtype)
    want = (x.double() @ w.double().t() + bias.double()).float()
    one = lambda r: torch.ones(r, device="cuda")  # noqa: E731
    rows, w8 = ops.QuantizedRows.of(x.to(E4M3), one(m)), ops.e4m3_weight(w.to(E4M3), one(n))
    assert torch.equal(ops.linear_e4m3(rows, w8, bias, F32), want)
    assert torch.equal(ops.linear_e4m3(rows, w8, bias), want.to(BF16))
    w4 = ops.pack_int4((w + 8).to(torch.uint8), torch.ones(n, -(-k // 128), device="cuda"))
    assert torch.equal(ops.linear_int4(x.to(BF16), w4, bias), want.to(BF16))
    relu = torch.relu(want[:, : n // 2].double()) * want[:, n // 2:].double()  # at most 12 + 16 bits each: rounded once to float32, once to bfloat16
    assert torch.equal(ops.gated_linear_e4m3(rows, w8, bias, 3), relu.float().to(BF16))
    if m <= 8 and n % 32 == 0:
        assert torch.equal(ops.gated_linear_int4(x.to(BF16), w4, bias, 3), relu.float().to(BF16))


# ---- rows whose squares overflow float32 -------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, None])
@pytest.mark.parametrize("rows,dim", [(5, 240), (3, 17), (2, 5001), (300, 4096), (300, 16384), (6, 8192), (4, 1000), (3, 20000), (2, 33001)])
def test_the_norm_of_rows_with_large_values(ops, dtype, rows, dim):
    g = gen(rows + dim)
    res = normal(g, rows, dim)
    res[0] *= 1e25
    res[1, 0] = 3e38  # one value alone
    if rows > 2:
        res[2] = 3.4e38 * torch.sign(res[2])  # every value
    delta = None if dtype is None else normal(g, rows, dim, std=1e24).to(dtype)
    if delta is not None:
        delta[1:] = 0
    gain = 1 + normal(g, dim, std=0.1)
    total = res.clone() if delta is None else res + delta.float()
    y = ops.add_rmsnorm_quantized(res, delta, gain, 1e-5)
    assert torch.equal(res, total)
    t = total.double() * gain.double()
    norm = t / (total.double().square().mean(1, keepdim=True) + 1e-5).sqrt()
    # the sum of squares: a thread's runs of 8 values, 4 of them or one for every 4,096 values of the row, and 10 levels; the rest as above
    terms = 8 * max(4, -(-(dim + 16) // 4096)) + 10
    torch.testing.assert_close(y.scales.double(), norm.abs().amax(1) / 448, atol=0, rtol=2.0 ** -24 * (terms / 2 + 4 + 6))
    want, _ = nearest_e4m3(t * 448 / t.abs().amax(1, keepdim=True))
    assert torch.equal(y.values[:, :dim].double(), want)
    if rows > 3:  # the others' rows do not see it
        alone = ops.add_rmsnorm_quantized(total[3:].contiguous(), None, gain, 1e-5)
        assert torch.equal(alone.values.view(torch.uint8), y.values[3:].view(torch.uint8))


# ---- the gated product of more rows, and the sizes of calls on two streams, against 64 bits ------------------------------------
def activated(gate, act):
    f = torch.nn.functional
    return [f.silu, f.gelu, lambda t: f.gelu(t, approximate="tanh"), torch.relu][act](gate)


@pytest.mark.parametrize("act", [0, 1, 2, 3])
@pytest.mark.parametrize("m,hidden,k,group", [(1, 5, 40, 32), (9, 80, 1040, 1040), (16, 4800, 384, 32), (17, 200, 256, 128), (64, 1000, 648, 64), (112, 9600, 136, 128),
                                              (130, 2000, 264, 32), (300, 520, 1160, 160), (700, 3000, 136, 128)])
def test_gated_linear_int4_of_more_rows(ops, act, m, hidden, k, group):
    """The product in bfloat16, its weights rounded beyond 8 rows, then the activation of that: every rounding is counted."""
    g = gen(act + m)
    w = ops.quantize_int4(normal(g, 2 * hidden, k, std=k ** -0.5), group)
    x, bias = normal(g, m, k).to(BF16), normal(g, 2 * hidden, std=0.1).to(BF16)
    y = ops.gated_linear_int4(x, w, bias, act)
    wd = w.dequantize().double() if m <= 8 else w.dequantize().to(BF16).double()
    z = x.double() @ wd.t() + bias.double()
    off = (k + 4) * 2.0 ** -23 * (x.double().abs() @ wd.abs().t()) + (HALF_STEP + 2.0 ** -22) * z.abs()
    gate, up = z[:, :hidden], z[:, hidden:]
    a = activated(gate, act)
    # slopes of these activations stay below 1.2; expf, erff and tanhf are good to a few units of float32 in 1
    a_off = 1.2 * off[:, :hidden] + 2.0 ** -20 * (a.abs() + gate.abs())
    u_off = off[:, hidden:]
    bound = a_off * up.abs() + (a.abs() + a_off) * u_off + (HALF_STEP + 2.0 ** -23) * (a.abs() + a_off) * (up.abs() + u_off) + 1e-30
    assert y.shape == (m, hidden) and bool(((y.double() - a * up).abs() <= bound).all())


@pytest.mark.parametrize("m", [1, 8, 40, 200, 700])
def test_products_of_a_wide_matrix(ops, m):
    n, k = 6144, 2576
    g = gen(m)
    x, raw = normal(g, m, k).to(BF16), normal(g, n, k, std=0.02)
    e4m3, int4 = ops.quantize_e4m3(raw), ops.quantize_int4(raw)
    rows = ops.quantize_rows(x)
    for xd, wd, linear, gated in ((rows.dequantize().double(), e4m3.dequantize().double(), lambda: ops.linear_e4m3(rows, e4m3), lambda: ops.gated_linear_e4m3(rows, e4m3, None, 1)),
                                  (x.double(), int4.dequantize().double() if m <= 8 else int4.dequantize().to(BF16).double(),
                                   lambda: ops.linear_int4(x, int4), lambda: ops.gated_linear_int4(x, int4, None, 1))):
        z = xd @ wd.t()
        off = (k + 6) * 2.0 ** -23 * (xd.abs() @ wd.abs().t()) + 2.0 ** -22 * z.abs()  # dequantize() rounds a value times its scale
        assert bool(((linear().double() - z).abs() <= off + HALF_STEP * (z.abs() + off)).all())
        gate, up = z[:, : n // 2], z[:, n // 2:]
        off = off + HALF_STEP * z.abs()  # a product of its own in front of the activation
        a, a_off, u_off = activated(gate, 1), 1.2 * off[:, : n // 2] + 2.0 ** -20 * gate.abs(), off[:, n // 2:]
        a_off = a_off + 2.0 ** -20 * a.abs()
        bound = a_off * up.abs() + (a.abs() + a_off) * u_off + (HALF_STEP + 2.0 ** -23) * (a.abs() + a_off) * (up.abs() + u_off)
        assert bool(((gated().double() - a * up).abs() <= bound).all())


@pytest.mark.parametrize("m", [1, 16, 100])
@pytest.mark.parametrize("n,k", [(100, 2176), (1000, 2176), (100, 2064), (128, 2048)])
def test_linear_e4m3_at_the_fewest_steps_that_are_cut(ops, m, n, k):
    """17 steps of 128 a tile and few tiles: equal runs, joined; 16: whole tiles."""
    x, w, sx, sw, bias = e4m3_case(m, n, k, m + n + k)
    y = ops.linear_e4m3(ops.QuantizedRows.of(x.to(E4M3), sx), ops.e4m3_weight(w.to(E4M3), sw), None, F32)
    assert torch.equal(y.double(), (x.double() @ w.double().t()) * sx.double()[:, None] * sw.double()[None, :])
    half = n // 2
    relu = ops.gated_linear_e4m3(ops.QuantizedRows.of(x.to(E4M3), sx), ops.e4m3_weight(w.to(E4M3), sw), None, 3)
    want = (torch.relu(y[:, :half].double()) * y[:, half:].double()).float().to(BF16)
    assert torch.equal(relu, want)


# with the accumulator's columns of a pair's tile on 148 multiprocessors
E4M3_TILES = [(257, 264, 64), (257, 2376, 80), (257, 3056, 96), (257, 3600, 112), (257, 4280, 128), (257, 4824, 144), (257, 5368, 160), (257, 6048, 176),
              (517, 4280, 192), (517, 4688, 208), (517, 5096, 224), (517, 5504, 240), (517, 5776, 256)]


@pytest.mark.parametrize("m,n,tile", E4M3_TILES)
def test_linear_e4m3_of_tiles_of_every_width(ops, m, n, tile):
    if torch.cuda.get_device_properties(0).multi_processor_count == 148:
        assert load_library("gemm_e4m3").fms_e4m3_tile(m, n, 0) == tile
    x, w, sx, sw, _ = e4m3_case(m, n, 272, m + n)
    y = ops.linear_e4m3(ops.QuantizedRows.of(x.to(E4M3), sx), ops.e4m3_weight(w.to(E4M3), sw), None, F32)
    assert torch.equal(y.double(), (x.double() @ w.double().t()) * sx.double()[:, None] * sw.double()[None, :])
