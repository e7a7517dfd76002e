"""Quantised weights without a device: the packed layout and what it stands for, rounding to 4 bits, and what is refused."""
import pytest
import torch

from fms_b200.kernels import ops

BF16 = torch.bfloat16


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("out,dim,group", [(1, 8, 32), (16, 128, 128), (37, 328, 64), (40, 1000, 32), (17, 136, 136), (5, 1160, 160), (33, 256, 1024)])
def test_packed_weights_stand_for_what_was_given(out, dim, group, zeros):
    g = gen(out + dim)
    groups = -(-dim // min(group, (dim + 31) // 32 * 32))
    q = torch.randint(0, 16, (out, dim), generator=g, dtype=torch.uint8)
    s = (torch.rand(out, groups, generator=g) + 0.1).to(BF16)
    z = torch.randint(0, 16, (out, groups), generator=g, dtype=torch.uint8) if zeros else None
    w = ops.pack_int4(q, s, z, group)
    at = torch.arange(dim) // group
    want = (q.float() - (z.float()[:, at] if zeros else 8.0)) * s.float()[:, at]
    assert w.shape == (out, dim) and torch.equal(w.dequantize(), want)


def test_the_layout_of_a_block():
    """Value k of row r: word 16 r + 4 place + k // 32 of its block, place = (k // 8 % 4) ^ (r // 2 % 4), bits 4 (k % 8 // 2) + 16 (k % 2);
    behind the 256 words a block's scales and zero points, 16 rows at a time."""
    q = torch.randint(0, 16, (32, 256), generator=gen(0), dtype=torch.uint8)
    scales = torch.arange(1, 129).view(32, 4).float()
    w = ops.pack_int4(q, scales, None, 64)
    assert w.per == 2 and w.blocks.shape == (2, 2, 256 + 32)
    for r, k in ((0, 0), (0, 1), (3, 13), (17, 200), (31, 255), (9, 127), (14, 64)):
        word = int(w.blocks[r // 16, k // 128, r % 16 * 16 + ((k // 8 % 4) ^ (r // 2 % 4)) * 4 + k % 128 // 32])
        assert (word >> (4 * (k % 8 // 2) + 16 * (k % 2))) & 15 == int(q[r, k])
        group = int(w.blocks[r // 16, k // 128, 256 + k % 128 // 64 * 16 + r % 16])
        assert (group >> 16) & 0xFFFF == 0x4308  # bfloat16 136
        assert torch.tensor([group << 16], dtype=torch.int64).to(torch.int32).view(torch.float32).item() == float(scales[r, k // 64])


@pytest.mark.parametrize("dtype", [torch.float32, BF16])
@pytest.mark.parametrize("out,dim,group", [(5, 64, 32), (33, 200, 64), (4, 72, 72), (4100, 32, 32)])
def test_rounding_to_four_bits(out, dim, group, dtype):
    w = (torch.randn(out, dim, generator=gen(out)) * 0.02).to(dtype)
    w[0] = 0.0
    w[1] = w[1].abs() + 1.0  # one sign: the steps reach down to zero all the same
    got = ops.quantize_int4(w, group)
    groups = -(-dim // group)
    wide = torch.zeros(out, groups * group)
    wide[:, :dim] = w.float()
    wide = wide.view(out, groups, group)
    # half a step for the value and half a step for the zero point that moved it; the scale's rounding moves the ends by up to 15 steps' 2^-8
    step = ((wide.amax(2).clamp(min=0) - wide.amin(2).clamp(max=0)) / 15)[:, torch.arange(dim) // group]
    assert bool(((got.dequantize() - w.float()).abs() <= step * (1.0 + 15 * 2.0 ** -8 + 2.0 ** -6) + 1e-30).all())
    assert float(got.dequantize()[0].abs().max()) == 0.0


def test_rows_that_need_a_copy_get_one():
    v = torch.randn(3, 32, generator=gen(1)).to(torch.float8_e4m3fn)
    s = torch.ones(3)
    assert ops.QuantizedRows.of(v, s).values.data_ptr() == v.data_ptr()
    odd = ops.QuantizedRows.of(v[:, :21], s)
    assert odd.shape == (3, 21) and odd.values.shape == (3, 32)
    assert torch.equal(odd.dequantize(), v[:, :21].float()) and float(odd.values[:, 21:].float().abs().max()) == 0.0


def test_refusals():
    E = ops.KernelError
    q, s = torch.zeros(4, 64, dtype=torch.uint8), torch.ones(4, 2)
    v = torch.zeros(4, 32).to(torch.float8_e4m3fn)
    for call in (
        lambda: ops.pack_int4(q.float(), s, None, 32),
        lambda: ops.pack_int4(q[0], s, None, 32),
        lambda: ops.pack_int4(q[:, :60], s, None, 32),                      # no multiple of 8
        lambda: ops.pack_int4(q, s, None, 48),                              # no multiple of 32
        lambda: ops.pack_int4(q, s, None, 0),
        lambda: ops.pack_int4(q, s, None, 64),                              # one group, two scales
        lambda: ops.pack_int4(q, s.long(), None, 32),
        lambda: ops.pack_int4(q, s, s, 32),                                 # zero points are whole numbers
        lambda: ops.pack_int4(q + 16, s, None, 32),
        lambda: ops.pack_int4(q, s, torch.full((4, 2), 16), 32),
        lambda: ops.pack_int4(q, s, torch.full((4, 2), -1), 32),
        lambda: ops.quantize_int4(q, 32),
        lambda: ops.quantize_int4(torch.ones(4, 64), 40),
        lambda: ops.QuantizedRows.of(torch.zeros(4, 32), torch.ones(4)),
        lambda: ops.QuantizedRows.of(v, torch.ones(3)),
        lambda: ops.QuantizedRows.of(v, torch.ones(4, dtype=BF16)),
        lambda: ops.QuantizedRows(v, torch.ones(4), 40),
        lambda: ops.quantize_rows(torch.ones(4, 32)),                       # on the CPU
        lambda: ops.quantize_e4m3(torch.ones(4, 32)),
        lambda: ops.add_rmsnorm_quantized(torch.ones(4, 32), None, torch.ones(32), 1e-5),
        lambda: ops.linear_e4m3(ops.QuantizedRows.of(v, torch.ones(4)), ops.e4m3_weight(v, torch.ones(4))),
        lambda: ops.linear_int4(torch.ones(2, 64, dtype=BF16), ops.pack_int4(q, s, None, 32)),
    ):
        with pytest.raises(E):
            call()


# ---- a model's configuration -------------------------------------------------------------------------------------------
def test_linear_config_of_a_model():
    from fms_b200.models import get_model
    from fms_b200.models.llama import LLaMA, LLaMAConfig
    from fms_b200.parts.linear import Linear, linear_options

    assert linear_options(None) == linear_options({"linear_type": "torch_linear"}) == ()
    assert LLaMA(LLaMAConfig(nlayers=1)).decoder_spec().layers[0].mixer.options == ()
    spec = LLaMA(LLaMAConfig(nlayers=1), linear_config={"linear_type": "int4", "group_size": 64}).decoder_spec()
    assert dict(spec.layers[0].mixer.options) == dict(spec.layers[0].feed_forward.options) == {"linear_type": "int4", "group_size": 64}
    for bad in ({"linear_type": "gptq"}, {"linear_type": "int4", "group_size": 48}, {"linear_type": "fp8", "group_size": 64}, {"linear_type": "int4", "bits": 3}):
        with pytest.raises(ValueError):
            LLaMAConfig(linear_config=bad)
        with pytest.raises(ValueError):
            get_model("llama", "micro", device_type="cpu", linear_config=bad)
    with pytest.raises(ValueError, match="bfloat16"):
        get_model("llama", "tiny-a", device_type="cpu", data_type="fp32", linear_config={"linear_type": "int4"})
    with pytest.raises(ValueError, match="no quantised"):
        get_model("goletar", "tiny", device_type="cpu", linear_config={"linear_type": "fp8"})
    with pytest.raises(ValueError, match="multiple of 8"):
        Linear(12, 8, options=(("linear_type", "int4"),))
    with pytest.raises(ValueError):
        Linear(16, 8, options=(("linear_type", "int3"),))


def test_a_layer_quantises_what_it_is_given():
    from fms_b200.parts.base import Part
    from fms_b200.parts.linear import Linear

    layer = Linear(72, 40, bias=True, options=(("linear_type", "int4"), ("group_size", 32)))
    w = torch.randn(40, 72, generator=gen(3)).to(BF16)
    layer.set_tensor("weight", w)
    layer.set_tensor("bias", torch.zeros(40, dtype=BF16))
    want = ops.quantize_int4(w, 32)
    assert isinstance(layer.tensor("weight"), ops.Int4Weight) and torch.equal(layer.tensor("weight").blocks, want.blocks)
    assert layer.kernel_libraries(BF16) == ["gemm_int4"] and not layer.by_sequence() and not layer.takes_quantized_rows
    root = Part()
    root.add("layer", layer)
    assert sorted(root.state_dict()) == ["layer.bias", "layer.weight.blocks"]
    with pytest.raises(ValueError, match="bfloat16"):
        layer.finalize("cpu", torch.float32)
    with pytest.raises(ValueError):
        layer.set_tensor("weight", w[:, :64])


def test_the_plain_rounding_to_four_bits_is_the_same():
    import plain_quantized as pq

    w = (torch.randn(37, 200, generator=gen(4)) * 0.02).to(BF16)
    for group in (32, 64, 128, 256):
        assert torch.equal(ops.quantize_int4(w, group).dequantize().double(), pq.int4_of(w, group))


# ---- how a product is cut ------------------------------------------------------------------------------------------------
PAIR_SHAPES = [(300, 6144), (512, 6144), (512, 28672), (700, 6144), (1024, 28672), (2048, 4096), (2048, 6144), (4096, 4096), (257, 264), (113, 40000), (8192, 128256)]


@pytest.mark.parametrize("m,n", PAIR_SHAPES)
def test_pairs_of_blocks_take_rows_by_32(m, n):
    """The instruction of a pair of thread blocks whose weights lie in tensor memory exists for 32, 64, ... 256 columns."""
    from fms_b200.kernels.build import load_library

    tile = load_library("gemm_int4").fms_linear_int4_tile
    assert tile(m, n) in range(32, 257, 32)
    assert tile(8, n) == tile(112, n) == 0


@pytest.mark.parametrize("file,kernel", [("gemm_e4m3.cu", "e4m3_join_kernel"), ("gemm_int4.cu", "int4_join_kernel"), ("gemm_int4.cu", "int4_few_rows_kernel"),
                                         ("quantize_rows.cu", "quantize_rows_kernel"), ("quantize_rows.cu", "add_rmsnorm_quantized_kernel")])
def test_only_weights_are_read_before_the_kernel_in_front_is_done(file, kernel):
    """A kernel starts while the one in front of it still runs, and may read a bias, scales or rows behind griddepcontrol.wait only."""
    import os
    import re

    from fms_b200.kernels.build import CSRC

    with open(os.path.join(CSRC, file)) as f:
        text = re.sub(r"//[^\n]*", "", f.read())
    body = text[re.search(rf"{kernel}\(", text).start():]
    ahead = body[: body.index("pdl_wait();")]
    assert not re.search(r"bias\[|sx\[|slots\[|rows\[|__ldg|load_gain\(\)|load_run<", ahead), ahead[-600:]


def test_rows_come_through_the_coherent_path():
    """A kernel that starts while the one in front still writes its rows must not read them as data that nobody writes meanwhile."""
    import os
    import re

    from fms_b200.kernels.build import CSRC

    with open(os.path.join(CSRC, "quantize_rows.cu")) as f:
        text = re.sub(r"//[^\n]*", "", f.read())
    assert "__restrict__" not in text and "__ldg" not in text and "ld.global.nc" not in text
    with open(os.path.join(CSRC, "gemm_int4.cu")) as f:
        assert "__ldg" not in f.read()


def test_a_bias_is_added_as_it_is():
    from fms_b200.kernels import quantized

    b = 1 + torch.arange(16) * 2.0 ** -20
    for kept in (b, b.to(BF16)):
        got, code = quantized._bias("linear", kept, 16)
        assert got is kept and code == (ops.F32 if kept.dtype == torch.float32 else ops.BF16)
    got, code = quantized._bias("linear", b.half(), 16)
    assert code == ops.F32 and torch.equal(got, b.half().float())
    with pytest.raises(ops.KernelError):
        quantized._bias("linear", b, 15)


def test_the_checked_build_checks_what_the_kernels_index():
    """FMS_IN stands at what is computed per value: runs of a row, stores of bytes, the residual, sums in scratch memory, packed blocks."""
    import os
    import re

    from fms_b200.kernels.build import CSRC

    text = {}
    for name in ("quantize_rows.cu", "gemm_e4m3.cu", "gemm_int4.cu"):
        with open(os.path.join(CSRC, name)) as f:
            text[name] = re.sub(r"//[^\n]*", "", f.read())
    rows = text["quantize_rows.cu"]
    for function in ("load_run", "store_run"):
        body = rows[rows.index(f" {function}("):]
        body = body[: body.index("\n}")]
        for line in body.splitlines():
            if re.search(r"row\[|run\.load|reinterpret_cast", line) and "FMS_IN" not in line:
                before = body[: body.index(line)].rstrip().splitlines()[-1]
                assert "FMS_IN" in before or re.match(r"\s*(static|template)", line), line
    assert "FMS_IN(blockIdx" not in rows  # the grid's own size
    for name in ("gemm_e4m3.cu", "gemm_int4.cu"):
        lines = text[name].splitlines()
        for i, line in enumerate(lines):
            if re.search(r"\bslot\[\(size_t|__ldcg\(", line):
                assert "FMS_IN" in line, line
    few = text["gemm_int4.cu"]
    few = few[few.index("int4_few_rows_kernel("):]
    few = few[: few.index("\n}")]
    assert few.count("FMS_IN(") >= 5


def test_a_cut_has_more_blocks_than_tiles():
    """Equal runs of an 8-bit product's steps: a run reaches into two tiles at most only where there are no fewer blocks than tiles, and a
    block's sums have two places."""
    import ctypes

    from fms_b200.kernels.build import load_library

    floats = load_library("gemm_e4m3").fms_e4m3_scratch
    floats.restype, floats.argtypes = ctypes.c_long, [ctypes.c_long] * 4
    cut = set()
    for glu in (0, 1):
        for steps in (1, 15, 16, 17, 18, 19, 24, 33, 64, 112, 400):
            for tiles in range(1, 110):
                columns = tiles * (64 if glu else 128)
                got = floats(16, columns * (2 if glu else 1), steps * 128, glu)
                if got:
                    blocks = got // (2 * 16 * 128)
                    assert got == blocks * 2 * 16 * 128 and tiles < blocks <= 148 and blocks * 4 <= tiles * steps
                    cut.add(steps)
    assert min(cut) == 17
