"""append_kv_blocks on every 16-bit value there is: codes are round(x / scale) with the correctly
rounded quotient, bit for bit, the sign of a zero among them."""
import pytest
import torch

from gpu_util import announce, assert_bit_equal
from oracle import serving as osv
from test_kv_blocks import FP8, pool


def every_value(dtype, order):
    """[1024, 1, 64] all 65536 patterns: next to each other in value, or mixed"""
    bits = torch.arange(65536, dtype=torch.int32)
    if order == "mixed":
        bits = bits[torch.randperm(65536, generator=torch.Generator().manual_seed(0))]
    bits = torch.where(bits >= 32768, bits - 65536, bits).to(torch.int16)
    return bits.view(dtype).view(1024, 1, 64)


@pytest.mark.gpu
@pytest.mark.parametrize("order", ["in order", "mixed"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("codes", [FP8, torch.int8])
@pytest.mark.parametrize("dynamic", [True, False])
def test_every_value(gpu, order, dtype, codes, dynamic):
    from compressed_tensors_amd.modeling import KVBlocks, append_kv_blocks

    announce("append every value", order, dtype, codes, dynamic)
    x = every_value(dtype, order)
    cache = pool(64, 1, 16, 64, codes, seed=4)
    on = KVBlocks(*(t.to(gpu) for t in cache))
    slots = torch.arange(1024)
    append_kv_blocks(x.to(gpu), x.to(gpu), on, slots.to(gpu), dynamic=dynamic)
    osv.kv_append(x, x, cache, slots, dynamic)
    for name, got, want in zip(KVBlocks._fields, on, cache):
        if got.dtype is FP8:  # a NaN's sign is nobody's
            got, want = (torch.where(t.float().isnan(), 0x7F, t.view(torch.uint8)) for t in (got.cpu(), want))
        elif got.dtype is torch.int8:
            got, want = got.view(torch.uint8), want.view(torch.uint8)
        assert_bit_equal(got, want, name)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rest", [1.0, float("inf"), 0.0])
def test_the_sign_of_zero(gpu, dtype, rest):
    """the code of -0.0 is that of -0.0, whatever stands beside it"""
    from compressed_tensors_amd.modeling import KVBlocks, append_kv_blocks

    x = torch.full((20, 2, 64), -0.0).to(dtype)
    x[:, 0, ::3], x[3, 0, 0] = 0.0, rest
    cache = pool(2, 2, 16, 64, FP8)
    on = KVBlocks(*(t.to(gpu) for t in cache))
    append_kv_blocks(x.to(gpu), x.to(gpu), on, torch.arange(20).to(gpu))
    osv.kv_append(x, x, cache, torch.arange(20))
    assert (cache[0].view(torch.uint8)[0, 1] == 0x80).all()
    for name, got, want in zip(KVBlocks._fields[:2], on, cache):
        assert_bit_equal(got.view(torch.uint8), want.view(torch.uint8), name)
