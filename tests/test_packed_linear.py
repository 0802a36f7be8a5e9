"""packed_linear against a 64-bit product with the unpacked weight.

Tolerance.  One rounding to the output's type is half a step: eps / 2 of the value.  The sum
is held in fp32: a product passes at most 32 additions inside its matrix instruction (or the
fold over a wavefront), one for each of the k / 32 that follow, and at most 32 more for group
scale, joins and bias, each off by 2^-24 of what has been summed, which stays below the sum of
magnitudes |x| (code + zero) scale.  So |error| <= eps / 2 |y| + (k / 32 + 64) 2^-24 magnitude.
"""
import pytest
import torch

from gpu_util import announce
from oracle import serving as osv


def make(m, n, k, groups, dtype, scale_dtype=None, asym=False, bias=False, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(m, k, generator=g).to(dtype)
    codes = torch.randint(0, 16, (n, k), generator=g)
    scale = ((0.5 + torch.rand(n, groups, generator=g)) * 0.02).to(scale_dtype or dtype)
    zero = osv.pack4(torch.randint(0, 16, (n, groups), generator=g), dim=0) if asym else None
    b = torch.randn(n, generator=g).to(dtype) if bias else None
    return x, osv.pack4(codes), scale, zero, b


def check(got, x, packed, scale, zero, bias):
    want, mag = osv.packed_linear(x, packed, scale, zero, bias)
    eps = torch.finfo(got.dtype).eps
    off = (got.cpu().double() - want).abs()
    bound = eps / 2 * want.abs() + (x.shape[1] / 32 + 64) * 2.0 ** -24 * mag + torch.finfo(got.dtype).smallest_normal * eps
    assert got.dtype is x.dtype and got.shape == want.shape
    worst = (off / bound).max().item() if off.numel() else 0.0
    assert (off <= bound).all(), f"{worst:.3g} times the bound"


def on(dev, *tensors):
    return [None if t is None else t.to(dev) for t in tensors]


SHAPES = [  # m, n, k, groups
    (1, 1, 8, 1), (1, 16, 32, 1), (1, 17, 128, 1), (1, 64, 4096, 32), (2, 33, 96, 3), (3, 100, 352, 11),
    (5, 1001, 1056, 33), (7, 15, 2048, 16), (8, 256, 512, 4), (15, 48, 1024, 8), (16, 130, 640, 5),
    (17, 96, 256, 2), (31, 65, 512, 16), (33, 40, 384, 3), (64, 272, 896, 7), (65, 129, 256, 4), (130, 31, 192, 6),
    (1, 7, 1, 1), (3, 20, 13, 1), (20, 9, 100, 1), (4, 30, 1000, 1), (64, 64, 8, 1), (1, 2048, 64, 2),
    (1, 40, 16384, 128), (16, 16, 14336, 112), (300, 70, 160, 5), (2, 5000, 128, 1),
]


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k,groups", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_shapes(gpu, m, n, k, groups, dtype):
    from compressed_tensors_amd.linear import packed_linear

    for asym, bias, scale_dtype in ((False, False, None), (True, True, None), (True, False, torch.float32),
                                    (False, True, torch.float16 if dtype is torch.bfloat16 else torch.bfloat16)):
        announce("packed_linear", m, n, k, groups, dtype, asym, bias, scale_dtype)
        data = make(m, n, k, groups, dtype, scale_dtype, asym, bias, seed=m + n + k)
        check(packed_linear(*on(gpu, *data)), *data)


@pytest.mark.gpu
def test_strided_shaped_and_offset_inputs(gpu):
    from compressed_tensors_amd.linear import packed_linear

    x, packed, scale, zero, bias = make(12, 80, 256, 2, torch.bfloat16, asym=True, bias=True, seed=3)
    dev = on(gpu, x, packed, scale, zero, bias)
    want = packed_linear(*dev)
    check(want, x, packed, scale, zero, bias)
    wide = torch.full((12, 512), 99.0, dtype=x.dtype, device=gpu)
    wide[:, 128:384] = dev[0]
    assert torch.equal(packed_linear(wide[:, 128:384], *dev[1:]), want)  # rows of a wider tensor
    wide[:, 131:387] = dev[0]
    assert torch.equal(packed_linear(wide[:, 131:387], *dev[1:]), want)  # off a 16-byte boundary
    assert torch.equal(packed_linear(dev[0].t().contiguous().t(), *dev[1:]), want)  # columns outermost
    assert torch.equal(packed_linear(dev[0].view(3, 4, 256), *dev[1:]), want.view(3, 4, 80))
    assert torch.equal(packed_linear(dev[0][0], *dev[1:]), packed_linear(dev[0][:1], *dev[1:])[0])
    assert torch.equal(packed_linear(dev[0][:1].expand(12, 256), *dev[1:]), packed_linear(dev[0][:1].repeat(12, 1), *dev[1:]))
    words = torch.zeros(80, 33, dtype=torch.int32, device=gpu)
    words[:, 1:] = dev[1]
    assert torch.equal(packed_linear(dev[0], words[:, 1:], *dev[2:]), want)
    flat = torch.zeros(80 * 32 + 1, dtype=torch.int32, device=gpu)
    flat[1:] = dev[1].flatten()
    assert torch.equal(packed_linear(dev[0], flat[1:].view(80, 32), *dev[2:]), want)  # words off a 16-byte boundary
    assert packed_linear(dev[0][:0], *dev[1:]).shape == (0, 80)


@pytest.mark.gpu
def test_a_row_of_a_batch_does_not_see_the_others(gpu):
    from compressed_tensors_amd.linear import packed_linear

    x, packed, scale, zero, bias = make(16, 64, 512, 4, torch.bfloat16, asym=True, seed=5)
    x[3, 17], x[4, 200], x[5, 0] = float("inf"), float("nan"), float("-inf")
    got = packed_linear(*on(gpu, x, packed, scale, zero)).cpu()
    want, _ = osv.packed_linear(x, packed, scale, zero)
    for row in (3, 4, 5):  # inf * 0 where a code equals its zero point is NaN, elsewhere the infinity stays
        assert torch.equal(got[row].isnan(), want[row].isnan())
        fine = ~want[row].isnan()
        assert torch.equal(got[row][fine].double(), want[row][fine])
    clean = [i for i in range(16) if i not in (3, 4, 5)]
    check(got[clean], x[clean], packed, scale, zero, None)


@pytest.mark.gpu
def test_extreme_codes_and_scales(gpu):
    from compressed_tensors_amd.linear import packed_linear

    for code in (0, 8, 15):
        x, packed, scale, zero, _ = make(4, 32, 256, 2, torch.float16, asym=True, seed=code)
        packed = osv.pack4(torch.full((32, 256), code))
        scale[0], scale[1], scale[2] = 0.0, -0.01, torch.finfo(torch.float16).tiny
        check(packed_linear(*on(gpu, x, packed, scale, zero)), x, packed, scale, zero, None)
    x, packed, scale, _, _ = make(3, 16, 128, 1, torch.bfloat16, torch.float32, seed=9)
    scale[:] = 1e-30
    check(packed_linear(*on(gpu, x, packed, scale)), x, packed, scale, None, None)


@pytest.mark.gpu
def test_large_weight_offsets(gpu):
    """more than 2^31 codes and 2^32 bytes of output behind them: the last columns are right"""
    from compressed_tensors_amd.linear import packed_linear

    n, k = 600_000, 4096
    words = torch.randint(-2**31, 2**31, (n, k // 8), dtype=torch.int32, device=gpu)
    scale = (torch.rand(n, k // 128, device=gpu) * 0.01).bfloat16()
    x = torch.randn(4096, k, device=gpu).bfloat16()
    got = packed_linear(x[:2], words, scale)
    for at in (0, n // 2, n - 32):
        check(got[:, at:at + 32].contiguous(), x[:2].cpu(), words[at:at + 32].cpu(), scale[at:at + 32].cpu(), None, None)
    got = packed_linear(x, words, scale)
    check(got[-2:, -32:].contiguous(), x[-2:].cpu(), words[-32:].cpu(), scale[-32:].cpu(), None, None)


@pytest.mark.gpu
def test_captured_graph_and_streams(gpu):
    from compressed_tensors_amd.linear import packed_linear

    first = on(gpu, *make(3, 96, 512, 4, torch.bfloat16, asym=True, bias=True, seed=1))
    second = on(gpu, *make(40, 96, 512, 4, torch.bfloat16, asym=True, bias=True, seed=2))
    eager = [packed_linear(*first), packed_linear(*second)]
    graphs, outs = [], []
    for data in (first, second):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(packed_linear(*data))
        graphs.append(g)
    for i in range(3):  # two graphs alive at once, eager work between the replays
        graphs[0].replay()
        graphs[1].replay()
        assert torch.equal(packed_linear(*first), eager[0])
        torch.cuda.synchronize()
        assert torch.equal(outs[0], eager[0]) and torch.equal(outs[1], eager[1])
        outs[0].zero_(), outs[1].zero_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = [packed_linear(*second) for _ in range(4)]
    here = [packed_linear(*second) for _ in range(4)]
    torch.cuda.synchronize()
    assert all(torch.equal(t, eager[1]) for t in on_side + here)


def packed_module(dev, dtype, symmetric, strategy, bias=True, n=96, k=256, seed=0):
    """a CompressedLinear that keeps its weight packed, filled with random codes"""
    from compressed_tensors_amd import CompressedLinear
    from compressed_tensors_amd.quantization import QuantizationArgs, QuantizationScheme

    spec = dict(num_bits=4, type="int", symmetric=symmetric, strategy=strategy)
    if strategy == "group":
        spec["group_size"] = 64
    layer = torch.nn.Linear(k, n, bias=bias).to(dtype).to(dev)
    module = CompressedLinear.from_linear(layer, QuantizationScheme(targets=["Linear"], weights=QuantizationArgs(**spec)),
                                          "pack-quantized", keep_packed=True)
    _, packed, scale, zero, b = make(1, n, k, k // 64 if strategy == "group" else 1, dtype, asym=not symmetric, bias=bias, seed=seed)
    module.weight_packed.data.copy_(packed)
    module.weight_scale.data.copy_(scale)
    module.weight_shape.data.copy_(torch.tensor([n, k]))
    if zero is not None:
        module.weight_zero_point.data.copy_(zero)
    if bias:
        module.bias.data.copy_(b)
    return module, packed, scale, zero, b


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("symmetric,strategy,bias", [(True, "group", True), (False, "group", False), (False, "channel", True)])
def test_compressed_linear_that_keeps_its_weight_packed(gpu, dtype, symmetric, strategy, bias):
    from compressed_tensors_amd.config import QuantizationStatus

    announce("keep_packed", dtype, symmetric, strategy, bias)
    module, packed, scale, zero, b = packed_module(gpu, dtype, symmetric, strategy, bias)
    for m in (1, 5, 40, 192):
        x = torch.randn(m, 256).to(dtype)
        with torch.no_grad():
            check(module(x.to(gpu)), x, packed, scale, zero, b)
    # many rows, and calls that are differentiated, go through the decompressed weight
    dense = module.compressor.decompress_module(module)
    x = torch.randn(193, 256).to(dtype).to(gpu)
    with torch.no_grad():
        assert torch.equal(module(x), torch.nn.functional.linear(x, dense, module.bias))
    x = torch.randn(3, 256).to(dtype).to(gpu).requires_grad_()
    y = module(x)
    y.float().square().sum().backward()
    other = x.detach().clone().requires_grad_()
    torch.nn.functional.linear(other, dense, module.bias).float().square().sum().backward()
    assert torch.equal(x.grad, other.grad)
    assert module.quantization_status == QuantizationStatus.COMPRESSED and not hasattr(module, "weight")


@pytest.mark.gpu
def test_keep_packed_with_other_types_of_scales_and_inputs(gpu):
    """any number of rows takes what few rows take; inputs of 32 bits go through the decompressed weight"""
    announce("keep_packed, other types")
    module, packed, scale, zero, b = packed_module(gpu, torch.bfloat16, True, "group", bias=False)
    module.weight_scale.data = module.weight_scale.data.float()
    dense = module.compressor.decompress_module(module)
    with torch.no_grad():
        x = torch.randn(193, 256).to(torch.bfloat16)
        check(module(x[:7].to(gpu)), x[:7], packed, scale, zero, b)
        assert torch.equal(module(x.to(gpu)), torch.nn.functional.linear(x.to(gpu), dense.to(x.dtype)))
        x = torch.randn(3, 256).to(gpu)
        assert torch.equal(module(x), torch.nn.functional.linear(x, dense.float()))


def test_keep_packed_refusals():
    from compressed_tensors_amd import CompressedLinear
    from compressed_tensors_amd.quantization import QuantizationArgs, QuantizationScheme

    def convert(fmt="pack-quantized", k=256, **spec):
        args = QuantizationArgs(**{**dict(num_bits=4, type="int", symmetric=True, strategy="group", group_size=64), **spec})
        return CompressedLinear.from_linear(torch.nn.Linear(k, 32), QuantizationScheme(targets=["Linear"], weights=args), fmt,
                                            keep_packed=True)

    for bad in (dict(num_bits=8), dict(group_size=16), dict(group_size=64, k=96), dict(actorder="group"),
                dict(fmt="int-quantized", num_bits=8, strategy="channel", group_size=None)):
        with pytest.raises(NotImplementedError, match="keep_packed"):
            convert(**bad)
    assert convert().keep_packed and convert(actorder="weight").keep_packed


def test_refusals():
    from compressed_tensors_amd.linear import packed_linear

    x, packed, scale, zero, bias = make(2, 16, 128, 2, torch.bfloat16, asym=True, bias=True)
    for bad in ((x[:, :120], packed, scale), (x, packed.long(), scale), (x, packed, scale[:8]), (x, packed, scale[:, 0]),
                (x, packed, scale, zero.long()), (x, packed, scale, zero[:1]), (x, packed, scale, None, bias[:3]),
                (x, packed, scale, None, bias.float()), (x, packed, scale[:, :1].repeat(1, 3)), (x[:, :0], packed[:, :0], scale)):
        with pytest.raises(ValueError):
            packed_linear(*bad)
    for bad in ((x.float(), packed, scale), (x, packed, scale.double()), (x.clone().requires_grad_(), packed, scale),
                (x, packed, scale, None, bias.clone().requires_grad_())):
        with pytest.raises(NotImplementedError):
            packed_linear(*bad)
    with pytest.raises(RuntimeError, match="GPU only"):
        packed_linear(x, packed, scale, zero, bias)


def test_abi_refusals(ctmi):
    def call(m=1, n=16, k=128, group=128, x=1, dtype=2, scale_dtype=2, stride=128):
        return ctmi.ctmi_packed_linear(x and 16, dtype, stride, 16, 16, scale_dtype, None, None, 16, m, n, k, group, None, 0, None)

    assert call(dtype=0) == -2 and call(scale_dtype=3) == -2
    assert call(group=16) == -2 and call(group=96) == -2 and call(k=0) == -1
    assert call(m=-1) == -1 and call(n=1 << 31) == -2 and call(x=0) == -1
    assert call(m=2, stride=100) == -1
    assert call(m=0) == 0 and call(n=0) == 0
