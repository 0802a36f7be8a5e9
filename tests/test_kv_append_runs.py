"""append_kv_blocks where a block's tokens are not consecutive: slots left out, tokens skipped.  The
runs of a block are written one after the other, by whoever has the first: codes and scales are the
definition's, bit for bit."""
import random

import pytest
import torch

from gpu_util import announce, assert_bit_equal
from oracle import serving as osv
from test_kv_blocks import FP8, pool


def runs_one_call_each(key, value, cache, slots, dynamic):
    """the definition: a call for each run of consecutive slots"""
    t, size = 0, cache[0].shape[2]
    while t < len(slots):
        n = 1
        while slots[t] >= 0 and t + n < len(slots) and slots[t + n] == slots[t] + n and int(slots[t + n]) % size:
            n += 1
        osv.kv_append(key[t:t + n], value[t:t + n], cache, slots[t:t + n], dynamic)
        t += n


def scattered(blocks, size, tokens, rng):
    """slots of at least `tokens` tokens: blocks in any order, in each rising positions with holes,
    skipped tokens anywhere"""
    order, slots = list(range(blocks)), []
    rng.shuffle(order)
    for block in order:
        if len(slots) >= tokens:
            break
        at = rng.choice([0, 0, rng.randrange(size)])
        while at < size:
            run = rng.randint(1, rng.choice([1, 3, size]))
            slots += [block * size + at + i for i in range(min(run, size - at))]
            at += run + rng.choice([0, 0, 1, 2, rng.randrange(1, size)])
            slots += [-1] * rng.choice([0, 0, 1, 1, 2, 70, rng.choice([1, 130, 700])])
    return slots


CASES = {"a hole": [0, 2], "a skipped token": [3, -1, 4], "both, twice": [17, -1, -1, 19, 20, 25, -1, 31, 32, 40],
         "far apart": [5] + [-1] * 61 + [6] + [-1] * 62 + [8, 9] + [-1] * 63 + [10] + [-1] * 64 + [12] + [-1] * 600 + [14, 15],
         "first of a block last": [16, 3, -1, 7, 47], "padded": [-1] * 300 + [33, 35] + [-1] * 500}


def run(gpu, slots, heads, dim, size, codes, dtype, dynamic, blocks, seed=0):
    from compressed_tensors_amd.modeling import KVBlocks, append_kv_blocks

    g = torch.Generator().manual_seed(seed)
    slots = torch.tensor(slots)
    # later tokens are larger: each run's scale grows over the one before
    grow = 2.0 ** (6 * torch.rand(len(slots), 1, 1, generator=g) - 3)
    k, v = ((torch.randn(len(slots), heads, dim, generator=g) * grow).to(dtype) for _ in range(2))
    cache = pool(blocks, heads, size, dim, codes, seed=seed)
    on = KVBlocks(*(t.to(gpu) for t in cache))
    append_kv_blocks(k.to(gpu), v.to(gpu), on, slots.to(gpu), dynamic=dynamic)
    runs_one_call_each(k, v, cache, slots, dynamic)
    for name, got, want in zip(KVBlocks._fields, on, cache):
        view = torch.uint8 if got.element_size() == 1 else torch.float32
        assert_bit_equal(got.view(view), want.view(view), name)


@pytest.mark.gpu
@pytest.mark.parametrize("case", list(CASES))
@pytest.mark.parametrize("codes,dtype", [(FP8, torch.bfloat16), (torch.int8, torch.float16)])
@pytest.mark.parametrize("dynamic", [True, False])
def test_blocks_with_holes(gpu, case, codes, dtype, dynamic):
    announce("append with holes", case, codes, dtype, dynamic)
    run(gpu, CASES[case], 2, 64, 16, codes, dtype, dynamic, 3)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [1000, 2500, 8000, 12000])  # a workgroup looks at 1, some and 32 tokens
@pytest.mark.parametrize("size", [16, 48, 256])
@pytest.mark.parametrize("codes", [FP8, torch.int8])
def test_batches_with_holes(gpu, tokens, size, codes):
    announce("append with holes", tokens, size, codes)
    rng = random.Random(tokens + size)
    blocks = 4 * tokens // size + 8
    run(gpu, scattered(blocks, size, tokens, rng), 1, 64, size, codes, torch.bfloat16, True, blocks, seed=size)


def test_definition_of_runs():
    """a call over tokens with holes and the calls over its runs are the same in the plain statement"""
    for codes in (FP8, torch.int8):
        for slots in CASES.values():
            k, v = torch.randn(len(slots), 2, 64).bfloat16(), torch.randn(len(slots), 2, 64).bfloat16()
            one, other = pool(3, 2, 16, 64, codes), pool(3, 2, 16, 64, codes)
            osv.kv_append(k, v, one, torch.tensor(slots))
            runs_one_call_each(k, v, other, torch.tensor(slots), True)
            assert all(torch.equal(a.float(), b.float()) for a, b in zip(one, other))
