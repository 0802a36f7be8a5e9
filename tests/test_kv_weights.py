"""What attend_kv_blocks keeps of a softmax weight on its way into the second product.

Tolerance: a score's sum, the exponential and the additions as in test_kv_blocks (relative to
sum p |v|), and the weights.  With at most 64 rows a kv head these are three bf16 numbers, which
hold all 24 bits (each leaves at most 2^-8 of what it rounds): 2^-24.  For float16 outputs of more
rows two: 2^-16.  For bf16 outputs of more rows one f16 number for weight times
scale, the largest being 2^7 or more: half a step, eps / 2 = 2^-11, and where f16 has no finer
steps half its smallest, 2^-25, which is 2^-32 of the largest weight times scale, for each key and
as many times as its code says.  Where the sum below is of the same numbers their scale is no less
than 2^-8 of the largest one: off by 2^-24 of the largest weight for a key.
"""
import pytest
import torch

from gpu_util import announce
from oracle import serving as osv
from test_kv_blocks import FP8, attention_case, run_attention


def check(got, q, cache, table, lens, starts, rows, many, keys, steepest):
    """many: more than 64 rows a kv head; keys: how many of them have a value, steepest: by how much
    a value may exceed the sum of p |v| that it is part of"""
    single = many and got.dtype is torch.bfloat16
    want, mag, reach = (t[rows] for t in osv.kv_attend(q, cache, table, lens, starts))
    n, eps = int(max(lens)), torch.finfo(got.dtype).eps
    weight = 2.0 ** -11 + n * 2.0 ** -24 if single else 2.0 ** -16 if many else 2.0 ** -24
    rel = weight + 2.0 ** -20 + 2 * (q.shape[2] / 32 + 40) * 2.0 ** -24 * reach + (n / 32 + 96) * 2.0 ** -24
    low = keys * 2.0 ** -32 * steepest if single else 0.0
    bound = (eps / 2 + 1.004 * weight) * want.abs() + rel * mag + low * mag.amax(dim=2, keepdim=True)
    bound = bound + torch.finfo(got.dtype).smallest_normal * eps
    off = (got.cpu().double()[rows] - want).abs()
    assert (off <= bound).all(), f"{(off / bound).max().item():.3g} times the bound"


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("codes", [FP8, torch.int8])
@pytest.mark.parametrize("news,size", [(1, 16), (1, 64), (65, 16), (65, 64), (200, 48)])
def test_weights_of_values_that_cancel(gpu, dtype, codes, news, size):
    """two values whose sum p v is 0 but for the rounding of their scale: what comes out is the
    kernel's error alone"""
    announce("cancelling values", news, size, codes, dtype)
    for seed in range(4):
        data = attention_case([4 * size + 1], [news if news == 1 else 65], 8, 8, 64, size, codes, dtype, seed=seed)
        q, cache, table, lens, starts = data
        if news == 200:  # several heads a kv head: rows of a tile are heads, too
            q, cache, table, lens, starts = data = attention_case([4 * size + 1], [50], 32, 8, 64, size, codes, dtype, seed=seed)
        first, last = int(table[0, 0]), int(table[0, 4])
        share = q.shape[1] // 8
        values = cache[1].float()
        values[:] = 0
        values[first, :, :, 0] = 96.0
        values[last, :, :, 0] = -112.0
        cache[1].copy_(values.to(codes))
        cache[3][:] = 0.03125
        # scores of the last token's queries in 64 bits; the second value's scale makes up for its weight
        keys = cache[0].float().double() * cache[2].double()[..., None, None]
        for h in range(8):
            k = torch.cat([keys[int(b), h] for b in table[0]])[:lens[0]]
            p = torch.softmax((k @ q[-1, h * share].double()) * 0.125, 0)
            cache[3][last, h] = float(p[0] * 96.0 * 0.03125 / (p[-1] * 112.0))
        got = run_attention(gpu, *data, max_query=q.shape[0])
        check(got, *data, slice(-1, None), q.shape[0] * share > 64, 2, 1)


SPREADS = {"rising": lambda i: 2.0 ** (i * 3 - 30), "falling": lambda i: 2.0 ** (25 - 3 * i), "one huge": lambda i: 1e6 if i == 2 else 0.01,
           "one tiny": lambda i: 1e-12 if i == 1 else 0.5, "beyond": lambda i: (1e-20, 1.0, 1e20, 0.0, -0.25, 1e-38)[i % 6]}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("codes", [FP8, torch.int8])
@pytest.mark.parametrize("spread", list(SPREADS))
@pytest.mark.parametrize("news,size", [(1, 16), (70, 16), (70, 64), (150, 64)])
def test_scales_of_values_far_apart(gpu, dtype, codes, spread, news, size):
    """what a block adds is as right as its own weight is, whatever the other blocks' scales"""
    announce("spread", spread, news, size, codes, dtype)
    data = attention_case([300], [news], 4, 2, 64, size, codes, dtype, seed=news)
    q, cache, table, lens, starts = data
    cache[2][:] *= 6  # some weights far below others
    for i, b in enumerate(table[0].tolist()):
        cache[3][b] *= SPREADS[spread](i)
    if dtype is torch.float16:  # an output that the type holds
        cache[3].clamp_(-1.0, 1.0)
    got = run_attention(gpu, *data, max_query=news)
    # the key with the largest weight times scale has a code of more than 90 among its 64
    check(got, *data, slice(None), news * 2 > 64, 300, 448 / 90)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("codes", [FP8, torch.int8])
@pytest.mark.parametrize("news,size", [(1, 16), (1, 64), (70, 16), (70, 64)])
def test_values_that_are_not_finite_and_seen(gpu, dtype, codes, news, size):
    """NaN codes and infinite scales of keys that every query sees, in steps without a mask"""
    announce("not finite", news, size, codes, dtype)
    data = attention_case([400], [news], 4, 2, 64, size, codes, dtype, seed=3)
    q, cache, table, lens, starts = data
    where = []
    if codes is FP8:
        cache[1].view(torch.uint8)[int(table[0, 1]), 0, 7, 3] = 0x7F
        cache[1].view(torch.uint8)[int(table[0, 0]), 1, 9, 15] = 0xFF
        where = [(slice(0, 2), 7), (slice(2, 4), 9)]
    got = run_attention(gpu, *data, max_query=news).cpu()
    want = torch.zeros_like(got, dtype=torch.bool)
    for heads, d in where:
        want[:, heads, d] = True
    assert torch.equal(got.isnan(), want)
    # an infinite scale: infinities of either sign meet in one sum, unless all codes have one
    cache[1].copy_(torch.where(cache[1].float().isnan() | (cache[1].float() == 0), 1.0, cache[1].float()).to(codes))
    block = int(table[0, 2])
    cache[1][block, 0, 5] = torch.full((size,), 2.0).to(codes)
    cache[1][block, 0, 6] = torch.full((size,), -3.0).to(codes)
    cache[3][block, 0] = float("inf")
    cache[3][int(table[0, 3]), 1] = float("nan")
    got = run_attention(gpu, *data, max_query=news).cpu()
    want, _, _ = osv.kv_attend(*data)
    assert torch.equal(got.isnan(), want.isnan())
    infinite = want.isinf()
    assert infinite[:, :2, 5].all() and torch.equal(got.double()[infinite], want[infinite])
    # in a block that some queries see whole, some in part and some not at all
    cache[1][int(table[0, 3]), 1], cache[3][int(table[0, 3]), 1], cache[3][block, 0] = cache[1][block, 0], 0.5, 0.5
    last = int(table[0, (400 - 1) // size])
    cache[1][last] = torch.full((2, 64, size), 3.0).to(codes)
    cache[3][last] = float("inf")
    got = run_attention(gpu, *data, max_query=news).cpu()
    want, _, _ = osv.kv_attend(*data)
    infinite = want.isinf()
    assert not got.isnan().any() and torch.equal(got.isinf(), infinite) and (got[infinite] > 0).all()
    assert infinite[-1].all() and (news == 1 or not infinite[0].any())
