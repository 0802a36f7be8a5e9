"""CompressedLinear with keep_packed where autograd looks on: what it does not need differentiated
takes the packed product, the rest the decompressed weight, nothing is dropped"""
import pytest
import torch

from gpu_util import announce
from test_packed_linear import check, make, packed_module


def never(*args, **kwargs):
    raise AssertionError("the weight was decompressed")


@pytest.mark.gpu
@pytest.mark.parametrize("symmetric,strategy", [(True, "group"), (False, "channel")])
def test_scales_that_require_grad(gpu, symmetric, strategy, monkeypatch):
    """parameters that a checkpoint's loading made: the scale of a module that stays packed is a constant,
    as it is in a module that does not"""
    announce("keep_packed, scale requires grad", symmetric, strategy)
    module, packed, scale, zero, _ = packed_module(gpu, torch.bfloat16, symmetric, strategy, bias=False)
    module.weight_scale = torch.nn.Parameter(module.weight_scale.data)
    assert module.weight_scale.requires_grad
    x = torch.randn(5, 256).bfloat16()
    with torch.no_grad():
        want = module(x.to(gpu))
    monkeypatch.setattr(module.compressor, "decompress_weight", never)
    got = module(x.to(gpu))
    assert torch.equal(got, want) and not got.requires_grad
    check(got, x, packed, scale, zero, None)


@pytest.mark.gpu
def test_scales_that_require_grad_beside_a_differentiated_input(gpu):
    module, *_ = packed_module(gpu, torch.bfloat16, True, "group", bias=False)
    dense = module.compressor.decompress_module(module)
    module.weight_scale = torch.nn.Parameter(module.weight_scale.data)
    x = torch.randn(3, 256).bfloat16().to(gpu).requires_grad_()
    module(x).float().square().sum().backward()
    other = x.detach().clone().requires_grad_()
    torch.nn.functional.linear(other, dense).float().square().sum().backward()
    assert torch.equal(x.grad, other.grad) and module.weight_scale.grad is None


def test_scales_that_require_grad_are_not_refused():
    """on the CPU the call gets as far as the kernel, which is on the GPU only"""
    module, *_ = packed_module("cpu", torch.bfloat16, True, "group", bias=False)
    module.weight_scale = torch.nn.Parameter(module.weight_scale.data)
    with pytest.raises(RuntimeError, match="GPU only"):
        module(torch.randn(2, 256).bfloat16())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(256,), (1, 256), (40, 256), (2, 3, 256), (0, 256)])
def test_a_bias_that_requires_grad_keeps_the_packed_product(gpu, dtype, shape, monkeypatch):
    announce("keep_packed, bias requires grad", dtype, shape)
    module, *_ = packed_module(gpu, dtype, False, "group")
    assert module.bias.requires_grad  # as from_linear leaves it
    x = torch.randn(shape).to(dtype).to(gpu)
    with torch.no_grad():
        want = module(x)
    monkeypatch.setattr(module.compressor, "decompress_weight", never)
    y = module(x)
    assert torch.equal(y, want) and y.requires_grad
    weight = torch.randn(y.shape).to(dtype).to(gpu)
    for _ in range(2):  # gradients add up
        (module(x) * weight).sum().backward()
    # a sum of m numbers in fp32, rounded once, twice over: half a step each, and of their sum
    exact = 2 * weight.double().reshape(-1, 96).sum(0)
    spread = weight.double().reshape(-1, 96).abs().sum(0)
    bound = torch.finfo(dtype).eps * 1.5 * exact.abs() + 2 * 40 * 2.0 ** -24 * spread
    assert module.bias.grad.dtype is dtype and ((module.bias.grad.double() - exact).abs() <= bound).all()
    # ... and its own gradient: the sum is linear
    v = torch.ones(96, dtype=dtype, device=gpu, requires_grad=True)
    grad, = torch.autograd.grad(module(x), module.bias, v.expand(y.shape), create_graph=True)
    again, = torch.autograd.grad(grad.sum(), v)
    assert (again == weight.reshape(-1, 96).shape[0]).all()


def test_dual_tensors_are_refused():
    """forward-mode derivatives: a call that would drop a tangent raises, with and without no_grad"""
    from torch.autograd import forward_ad

    from compressed_tensors_amd.linear import packed_linear

    x, packed, scale, _, bias = make(2, 16, 128, 2, torch.bfloat16, bias=True)
    with forward_ad.dual_level():
        for i in range(3):
            args = [x, scale, bias]
            args[i] = forward_ad.make_dual(args[i], torch.ones_like(args[i]))
            for mode in (torch.enable_grad(), torch.no_grad()):
                with mode, pytest.raises(NotImplementedError, match="forward-mode"):
                    packed_linear(args[0], packed, args[1], None, args[2])
        with pytest.raises(RuntimeError, match="GPU only"):  # plain tensors inside a level
            packed_linear(x, packed, scale, None, bias)


@pytest.mark.gpu
@pytest.mark.parametrize("grad", [True, False])
def test_dual_tensors_go_through_the_decompressed_weight(gpu, grad):
    from torch.autograd import forward_ad

    module, *_ = packed_module(gpu, torch.bfloat16, True, "group")
    dense = module.compressor.decompress_module(module)
    x, t = torch.randn(3, 256).bfloat16().to(gpu), torch.randn(3, 256).bfloat16().to(gpu)
    bias, bt = module.bias.detach(), torch.randn(96).bfloat16().to(gpu)
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        got = forward_ad.unpack_dual(module(forward_ad.make_dual(x, t)))
        want = forward_ad.unpack_dual(torch.nn.functional.linear(forward_ad.make_dual(x, t), dense, bias))
        assert torch.equal(got.primal, want.primal) and torch.equal(got.tangent, want.tangent)
        del module.bias
        module.bias = forward_ad.make_dual(bias, bt)
        got = forward_ad.unpack_dual(module(x))
        assert torch.equal(got.tangent, bt.expand(3, 96))


@pytest.mark.gpu
@pytest.mark.parametrize("given", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("cast", [torch.bfloat16, torch.float16])
def test_autocast(gpu, given, cast, monkeypatch):
    """inside autocast the product is one in autocast's type, whatever input and bias are, as that
    of a module that does not stay packed"""
    module, packed, scale, zero, _ = packed_module(gpu, torch.bfloat16, True, "group")
    module.bias.data = module.bias.data.float()
    dense = module.compressor.decompress_module(module)
    x = torch.randn(6, 256)
    x = x.to(given)
    with torch.autocast("cuda", dtype=cast):
        ordinary = torch.nn.functional.linear(x.to(gpu), dense, module.bias)
        monkeypatch.setattr(module.compressor, "decompress_weight", never)
        with torch.no_grad():
            got = module(x.to(gpu))
        y = module(x.to(gpu))
    assert got.dtype is ordinary.dtype is cast and torch.equal(y, got)
    check(got, x.to(cast), packed, scale, zero, module.bias.detach().cpu().to(cast))
    y.sum().backward()
    assert module.bias.grad.dtype is torch.float32 and (module.bias.grad == 6).all()
