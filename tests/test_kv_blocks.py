"""The 8-bit block cache: planning and append exactly as their definitions, attention against
64 bits.

Tolerance of the attention.  A score's fp32 sum is off by at most (dim / 32 + 40) 2^-24 of
reach = sum |q||k| scale (32 additions inside an instruction, one per instruction, the scales),
its weight p = exp(score - top) by that (twice: its own and the top's share in the sum) and
2^-20 for the exponential and the argument's rounding; weights enter the second product as a
sum of two bf16 numbers (off by 2^-16 of themselves) or, for bf16 outputs, one (eps / 2 =
2^-8: bf16 has 8 significant bits, its neighbours in [1, 2) are 2^-7 apart); sums
over n keys pass n / 32 + 96 additions.  All of it scales with sum p |v|.  Where the weights
are divided by the sum of the rounded weights, w' = w (1 + d) with |d| <= e, the quotient is
sum p (1 + d) v / sum p (1 + d): off by at most e sum p |v| above and, through the sum below,
by e / (1 - e) |o| once more.  The output's rounding is eps / 2 of the value.
"""
import ctypes

import pytest
import torch

from gpu_util import announce, assert_bit_equal
from oracle import serving as osv

FP8 = torch.float8_e4m3fn


def pool(blocks, heads, size, dim, codes, seed=0):
    g = torch.Generator().manual_seed(seed)
    out = []
    for shape in ((blocks, heads, size, dim), (blocks, heads, dim, size)):
        x = torch.randn(*shape, generator=g) * 60
        out.append(x.to(FP8) if codes is FP8 else x.round().clamp(-128, 127).to(torch.int8))
    return out + [0.01 + 0.05 * torch.rand(blocks, heads, generator=g) for _ in range(2)]


def tables(lens, size, seed=0, spare=2, width=None):
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // size) for n in lens]
    order = torch.randperm(sum(need) + spare, generator=g).to(torch.int32)
    table = torch.full((len(lens), width or max(max(need), 1)), -1, dtype=torch.int32)
    at = 0
    for r, n in enumerate(need):
        table[r, :n] = order[at:at + n]
        at += n
    return table, sum(need) + spare


def check_attention(got, q, blocks, table, lens, starts, scale=None, out=None):
    want, mag, reach = osv.kv_attend(q, blocks, table, lens, starts, scale, out)
    eps, n = torch.finfo(got.dtype).eps, max(int(max(lens)) if len(lens) else 0, 1)
    weight = 2.0 ** -8 if got.dtype is torch.bfloat16 else 2.0 ** -16
    rel = weight + 2.0 ** -20 + 2 * (q.shape[2] / 32 + 40) * 2.0 ** -24 * reach + (n / 32 + 96) * 2.0 ** -24
    bound = (eps / 2 + 1.004 * weight) * want.abs() + rel * mag + torch.finfo(got.dtype).smallest_normal * eps
    off = (got.cpu().double() - want).abs()
    assert (off <= bound).all(), f"{(off / bound).max().item():.3g} times the bound"


# ------------------------------------------------------------------------------- attention
def attention_case(lens, news, heads, kv_heads, dim, size, codes, dtype, seed=0, pad=0):
    table, blocks = tables(lens, size, seed)
    cache = pool(blocks, kv_heads, size, dim, codes, seed)
    starts = torch.tensor([0] + list(torch.tensor(news).cumsum(0)), dtype=torch.int32)
    g = torch.Generator().manual_seed(seed + 1)
    q = torch.randn(sum(news) + pad, heads, dim, generator=g).to(dtype)
    return q, cache, table, torch.tensor(lens, dtype=torch.int32), starts


def run_attention(gpu, q, cache, table, lens, starts, **more):
    from compressed_tensors_amd.modeling import KVBlocks, attend_kv_blocks

    return attend_kv_blocks(q.to(gpu), KVBlocks(*(t.to(gpu) for t in cache)), table.to(gpu), lens.to(gpu),
                            None if starts is None else starts.to(gpu), **more)


CASES = [  # lens, new tokens, heads, kv heads, head dim, block size
    ([1], [1], 1, 1, 64, 16),
    ([1, 2, 15, 16, 17, 31, 33], [1] * 7, 8, 2, 128, 16),
    ([0, 5, 0, 64, 65], [1, 1, 1, 1, 1], 4, 4, 64, 64),
    ([300, 63, 64, 65, 128, 1], [1] * 6, 32, 8, 128, 32),
    ([700], [1], 7, 1, 128, 64),
    ([130, 257], [1, 1], 16, 1, 256, 128),
    ([100, 40, 9], [5, 3, 9], 8, 2, 64, 16),
    ([77, 200], [13, 0], 8, 8, 128, 64),
    ([3, 2, 1], [5, 2, 4], 4, 2, 64, 16),  # more queries than keys: the first see nothing
    ([150, 33], [150, 20], 8, 2, 128, 32),
    ([90], [90], 12, 4, 64, 48),
    ([260, 31, 140], [64, 31, 129], 16, 2, 128, 256),
    ([500, 1000], [17, 2], 20, 1, 64, 64),
    ([66], [66], 3, 3, 256, 16),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", range(len(CASES)))
@pytest.mark.parametrize("codes,dtype", [(FP8, torch.bfloat16), (torch.int8, torch.float16),
                                         (torch.int8, torch.bfloat16), (FP8, torch.float16)])
def test_attention(gpu, case, codes, dtype):
    lens, news, heads, kv_heads, dim, size = CASES[case]
    announce("attend", CASES[case], codes, dtype)
    data = attention_case(lens, news, heads, kv_heads, dim, size, codes, dtype, seed=case)
    q, cache, table, lens, starts = data
    hints = {"max_query": max(max(news), 1), "max_seq": max(int(lens.max()), 1)}
    got = run_attention(gpu, *data, **hints)
    check_attention(got, *data)
    # the launch follows the hints, the result does not depend on their being right
    for other in ({}, {"max_query": 1, "max_seq": 1}, {"max_query": 4096, "max_seq": 100000}, {"max_query": 3}):
        check_attention(run_attention(gpu, *data, **other), *data)
    if all(n == 1 for n in news):
        assert torch.equal(run_attention(gpu, q, cache, table, lens, None, max_seq=hints["max_seq"]), got)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_long_sequences_are_split_and_joined(gpu, dtype):
    for lens, news, kv in (([9000, 4097, 3], [1, 1, 1], 1), ([5000], [3], 2), ([6000, 100], [70, 40], 1)):
        announce("attend long", lens, news, dtype)
        data = attention_case(lens, news, 4 * kv, kv, 64, 64, FP8, dtype, seed=7)
        check_attention(run_attention(gpu, *data, max_query=max(news), max_seq=max(lens)), *data)
        again = run_attention(gpu, *data, max_query=max(news), max_seq=max(lens))
        assert torch.equal(again, run_attention(gpu, *data, max_query=max(news), max_seq=max(lens)))


@pytest.mark.gpu
def test_padded_rows_and_strided_queries(gpu):
    q, cache, table, lens, starts = attention_case([40, 70], [2, 6], 8, 2, 64, 16, FP8, torch.bfloat16, pad=5)
    mark = torch.full_like(q, 7.0)
    got = run_attention(gpu, q, cache, table, lens, starts, out=mark.to(gpu))
    check_attention(got, q, cache, table, lens, starts, out=mark)
    assert (got[8:] == 7).all()
    # queries inside a fused projection's rows, a table cut from a wider one
    fused = torch.zeros(13, 12, 64, dtype=q.dtype)
    fused[:, 2:10] = q
    wide = torch.full((2, 9), 3, dtype=torch.int32)
    wide[:, :table.shape[1]] = table
    from compressed_tensors_amd.modeling import KVBlocks, attend_kv_blocks

    on = [t.to(gpu) for t in cache]
    same = attend_kv_blocks(fused.to(gpu)[:, 2:10], KVBlocks(*on), wide.to(gpu)[:, :table.shape[1]], lens.to(gpu),
                            starts.to(gpu), out=mark.to(gpu))
    assert torch.equal(same, got)
    odd = torch.zeros(q.numel() + 3, dtype=q.dtype)
    odd[3:] = q.flatten()
    same = attend_kv_blocks(odd.to(gpu)[3:].view(q.shape), KVBlocks(*on), table.to(gpu), lens.to(gpu), starts.to(gpu),
                            out=mark.to(gpu))
    assert torch.equal(same, got)
    empty = attend_kv_blocks(q.to(gpu)[:0], KVBlocks(*on), table.to(gpu)[:0], lens.to(gpu)[:0])
    assert empty.shape == (0, 8, 64)


@pytest.mark.gpu
@pytest.mark.parametrize("codes", [FP8, torch.int8])
@pytest.mark.parametrize("news", [[1, 1], [7, 40], [90, 33]])
def test_nothing_leaks_from_positions_that_are_hidden(gpu, codes, news):
    """NaN codes behind the last token and at keys a query may not see, infinite scales of
    blocks a request does not name"""
    lens = [90, 33]
    data = attention_case(lens, news, 8, 2, 64, 32, codes, torch.bfloat16, seed=3)
    q, cache, table, lens_t, starts = data
    for r, n in enumerate(lens):
        block, at = int(table[r, (n - 1) // 32]), (n - 1) % 32 + 1
        if codes is FP8:
            cache[0].view(torch.uint8)[block, :, at:] = 0x7F
            cache[1].view(torch.uint8)[block, :, :, at:] = 0xFF
    used = set(table[table >= 0].tolist())
    for b in range(cache[0].shape[0]):
        if b not in used:
            cache[2][b], cache[3][b] = float("inf"), float("nan")
    check_attention(run_attention(gpu, *data, max_query=max(news)), *data)
    if codes is FP8 and news[0] > 1:
        # a NaN at the last key: only the last query of that request sees it
        block, at = int(table[0, 89 // 32]), 89 % 32
        cache[1].view(torch.uint8)[block, 0, 5, at] = 0x7F
        cache[0].view(torch.uint8)[block, 1, at, 3] = 0xFF
        got = run_attention(gpu, *data, max_query=max(news)).cpu()
        last = news[0] - 1
        nan = got.isnan()
        assert nan[last, :4, 5].all() and nan[last, 4:].all()
        nan[last, :4, 5] = False
        nan[last, 4:] = False
        assert not nan.any()
        clean = [t for t in range(q.shape[0]) if t != last]
        want, mag, _ = osv.kv_attend(q, [c.nan_to_num() if c.dtype is torch.float32 else c for c in
                                         (torch.where(cache[0].float().isnan(), 0.0, cache[0].float()),
                                          torch.where(cache[1].float().isnan(), 0.0, cache[1].float()),
                                          cache[2], cache[3])], table, lens_t, starts)
        off = (got.double() - want).abs()[clean]
        assert (off <= 2.0 ** -7 * mag[clean] + 1e-6).all()


@pytest.mark.gpu
@pytest.mark.parametrize("max_query,max_seq", [(1, 1), (7, 1 << 20), (1 << 40, 4097), (1000, 1 << 40)])
def test_any_launch_hint_has_room_in_the_scratch_it_is_given(gpu, ctmi, max_query, max_seq):
    """hints beyond the tokens and the table are cut to them by the call, which may then split
    the keys otherwise than the hints alone would"""
    from compressed_tensors_amd import _lib
    from compressed_tensors_amd.modeling import KVBlocks
    from compressed_tensors_amd.modeling.kv_blocks import _describe

    announce("hints", max_query, max_seq)
    q, cache, table, lens, starts = attention_case([1500, 2049], [5, 2], 8, 2, 64, 64, FP8, torch.bfloat16)
    on = KVBlocks(*(t.to(gpu) for t in cache))
    c, qd, td, ld, sd = _describe(on), q.to(gpu), table.to(gpu), lens.to(gpu), starts.to(gpu)
    out = torch.full_like(qd, 7.0)
    size = ctmi.ctmi_kv_attend_tmp_bytes(7, 2, 8, 2, 64, max_query, max_seq)
    tmp = torch.empty(size + 16, dtype=torch.uint8, device=gpu)
    _lib.check(ctmi.ctmi_kv_attend(
        qd.data_ptr(), _lib.dtype_code(q.dtype), 512, 64, out.data_ptr(), 7, 8, ctypes.byref(c), td.data_ptr(),
        td.shape[1], td.shape[1], ld.data_ptr(), sd.data_ptr(), 2, 0.125, max_query, max_seq, tmp.data_ptr(), size,
        _lib.stream_of(qd.device)))
    check_attention(out, q, cache, table, lens, starts)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_scales_far_apart_and_large_scores(gpu, dtype):
    """a block with tiny values and nearly all of the weight beside one with huge values, scores
    that overflow an exponential taken without the maximum"""
    data = attention_case([200, 64], [1, 1], 4, 1, 64, 16, FP8, dtype, seed=11)
    q, cache, table, lens, starts = data
    cache[2][:] *= 30
    first = int(table[0, 0])
    cache[3][first] = 1e-4
    cache[3][int(table[0, 5])] = 40.0 if dtype is torch.float16 else 1e6
    check_attention(run_attention(gpu, *data), *data)


@pytest.mark.gpu
def test_bad_pages_hide_their_positions(gpu):
    q, cache, table, lens, starts = data = attention_case([100, 60], [1, 9], 8, 2, 64, 16, FP8, torch.bfloat16, seed=5)
    table[0, 2], table[1, 0], table[1, 3] = 1 << 30, -7, cache[0].shape[0]
    check_attention(run_attention(gpu, *data), *data)
    table[0] = -1  # nothing left to see
    got = run_attention(gpu, *data)
    assert (got[0] == 0).all()
    check_attention(got, *data)
    lens[1] = 1000  # beyond the table's width
    check_attention(run_attention(gpu, *data), *data)


@pytest.mark.gpu
def test_offsets_beyond_32_bits(gpu):
    """a pool of more than 4 GiB of codes: blocks at its very end"""
    from compressed_tensors_amd.modeling import KVBlocks, attend_kv_blocks, append_kv_blocks

    blocks, heads, size, dim = 70_000, 4, 128, 128
    key = torch.zeros(blocks, heads, size, dim, dtype=torch.uint8, device=gpu)
    value = torch.zeros(blocks, heads, dim, size, dtype=torch.uint8, device=gpu)
    cache = KVBlocks(key.view(FP8), value.view(FP8), torch.ones(blocks, heads, device=gpu), torch.ones(blocks, heads, device=gpu))
    g = torch.Generator().manual_seed(0)
    k, v = torch.randn(150, heads, dim, generator=g).bfloat16(), torch.randn(150, heads, dim, generator=g).bfloat16()
    table = torch.tensor([[blocks - 1, blocks - 2]], dtype=torch.int32)
    place = torch.arange(150)
    slots = table[0, place // size].long() * size + place % size
    append_kv_blocks(k.to(gpu), v.to(gpu), cache, slots.to(gpu))
    small = [torch.zeros(2, heads, size, dim).to(FP8), torch.zeros(2, heads, dim, size).to(FP8), torch.ones(2, heads), torch.ones(2, heads)]
    osv.kv_append(k, v, small, torch.tensor([1, 0])[place // size] * size + place % size)
    assert_bit_equal(cache.key[-2:].view(torch.uint8), small[0].view(torch.uint8), "keys")
    assert_bit_equal(cache.value[-2:].view(torch.uint8), small[1].view(torch.uint8), "values")
    q = torch.randn(1, 8, dim, generator=g).bfloat16()
    lens = torch.tensor([150], dtype=torch.int32)
    got = attend_kv_blocks(q.to(gpu), cache, table.to(gpu), lens.to(gpu))
    check_attention(got, q, small, torch.tensor([[1, 0]], dtype=torch.int32), lens, None)


# ---------------------------------------------------------------------------------- append
APPENDS = [  # (tokens before, new tokens) of each request, heads, head dim, block size
    ([(0, 1)], 1, 64, 16), ([(15, 1), (16, 1), (17, 1), (0, 1)], 2, 128, 16), ([(5, 40), (0, 33), (31, 2)], 2, 64, 32),
    ([(0, 64), (63, 66)], 3, 128, 64), ([(100, 300)], 1, 256, 128), ([(250, 20), (0, 256)], 2, 64, 256), ([(7, 50)], 1, 64, 48),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", range(len(APPENDS)))
@pytest.mark.parametrize("codes", [FP8, torch.int8])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dynamic", [True, False])
def test_append(gpu, case, codes, dtype, dynamic):
    from compressed_tensors_amd.modeling import KVBlocks, append_kv_blocks

    counts, heads, dim, size = APPENDS[case]
    announce("append", APPENDS[case], codes, dtype, dynamic)
    table, blocks = tables([b + n for b, n in counts], size, seed=case)
    slots = torch.cat([table[r, torch.arange(b, b + n) // size].long() * size + torch.arange(b, b + n) % size
                       for r, (b, n) in enumerate(counts)])
    slots = torch.cat([torch.tensor([-1]), slots, torch.tensor([-1, blocks * size, 1 << 40])])  # a padded batch
    g = torch.Generator().manual_seed(case)
    for size_of_values in (0.3, 20.0):  # below and above what the scales cover
        cache = pool(blocks, heads, size, dim, codes, seed=case)
        k = (torch.randn(len(slots), heads, dim, generator=g) * size_of_values).to(dtype)
        v = (torch.randn(len(slots), heads, dim, generator=g) * size_of_values).to(dtype)
        on = KVBlocks(*(t.to(gpu) for t in cache))
        for again in range(2):  # a second call with the same tokens changes nothing
            append_kv_blocks(k.to(gpu), v.to(gpu), on, slots.to(gpu), dynamic=dynamic)
            osv.kv_append(k, v, cache, slots, dynamic)
            for name, got, want in zip(KVBlocks._fields, on, cache):
                view = torch.uint8 if got.element_size() == 1 else torch.float32
                assert_bit_equal(got.view(view), want.view(view), name)


@pytest.mark.gpu
@pytest.mark.parametrize("codes", [FP8, torch.int8])
def test_append_of_zeros_infinities_and_nan(gpu, codes):
    from compressed_tensors_amd.modeling import KVBlocks, append_kv_blocks

    cache = pool(4, 2, 16, 64, codes, seed=1)
    k, v = torch.randn(6, 2, 64).bfloat16(), torch.randn(6, 2, 64).bfloat16()
    k[0], v[0] = 0, 0  # a block of zeros: the scale is the floor
    k[1, 0, 3], k[2, 1, 5], v[3, 0, 1], v[4, 1, 0] = float("inf"), float("nan"), float("-inf"), float("nan")
    v[5, 0] = float("nan")
    slots = torch.tensor([0, 16, 17, 37, 38, 63])
    on = KVBlocks(*(t.to(gpu) for t in cache))
    append_kv_blocks(k.to(gpu), v.to(gpu), on, slots.to(gpu))
    osv.kv_append(k, v, cache, slots)
    assert float(on.key_scale[0, 0]) == osv.EPS
    for name, got, want in zip(KVBlocks._fields, on, cache):
        # a NaN's sign is nobody's
        assert torch.equal(got.cpu().float().nan_to_num(nan=1e9), want.float().nan_to_num(nan=1e9)), name


@pytest.mark.gpu
def test_append_from_strided_tensors(gpu):
    from compressed_tensors_amd.modeling import KVBlocks, append_kv_blocks

    fused = torch.randn(20, 10, 64).half().to(gpu)  # queries, keys and values of one projection
    slots = torch.arange(20).to(gpu) + 6
    results = []
    odd = torch.zeros(fused.numel() + 1, dtype=fused.dtype, device=gpu)[1:].view(fused.shape).copy_(fused)
    for k, v in ((fused[:, 6:8], fused[:, 8:]), (fused[:, 6:8].contiguous(), fused[:, 8:].contiguous()),
                 (odd[:, 6:8], odd[:, 8:]), (fused[:, 6:8].transpose(1, 2).contiguous().transpose(1, 2), fused[:, 8:])):
        on = KVBlocks(*(t.to(gpu) for t in pool(2, 2, 16, 64, FP8)))
        append_kv_blocks(k, v, on, slots)
        results.append(on)
    for other in results[1:]:
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(results[0], other))


# -------------------------------------------------------------------------------- planning
def run_plan(gpu, lens, new, table, free, num_free, size, total):
    from compressed_tensors_amd.modeling import plan_kv_blocks

    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=gpu)  # noqa: E731
    args = (ints(lens), ints(new), ints(table).view(len(lens), -1), ints(free), ints([num_free]))
    keep = [a.clone() for a in args]
    plan = plan_kv_blocks(*args, block_size=size, total_tokens=total)
    want = osv.kv_plan(lens, new, table, free, num_free, size, total)
    for name, got, w in zip(plan._fields, plan, want):
        assert got.cpu().tolist() == (w if isinstance(w, list) else [w]), name
    assert all(torch.equal(a, k) for a, k in zip(args, keep))
    return plan


@pytest.mark.gpu
@pytest.mark.parametrize("requests", [1, 2, 63, 64, 65, 256, 257, 1000, 4096])
def test_plan(gpu, requests):
    import random

    rng = random.Random(requests)
    for size in (16, 1, 48):
        width = rng.randint(3, 12)
        cap = width * size
        lens = [rng.randint(0, cap - 1) for _ in range(requests)]
        new = [rng.choice([-1, 0, 1, 1, 1, rng.randint(0, cap - n), -9]) for n in lens]
        held = [-(-n // size) for n in lens]
        pool_size = sum(-(-(n + max(a, 0)) // size) for n, a in zip(lens, new)) + 5
        order = list(range(pool_size))
        rng.shuffle(order)
        table, at = [], 0
        for h in held:
            table.append(order[at:at + h] + [-1] * (width - h))
            at += h
        free = order[at:] + [-1] * at
        total = sum(a for a in new if a > 0)
        announce("plan", requests, size, total)
        run_plan(gpu, lens, new, table, free, pool_size - at, size, total)
        run_plan(gpu, lens, new, table, free, pool_size - at, size, total + 37)  # a padded batch
        if total:
            run_plan(gpu, lens, new, table, free, pool_size - at, size, total - 1)
        run_plan(gpu, lens, new, table, free, 0, size, total)  # short of blocks unless ended requests give enough
        run_plan(gpu, lens, new, table, free[:at], pool_size - at, size, total)


@pytest.mark.gpu
def test_plan_of_steps_that_do_not_fit(gpu):
    table = [[0, 1], [2, -1]]
    run_plan(gpu, [20, 3], [13, 1], table, [3, 4], 2, 16, 14)  # request 0 needs a third column
    run_plan(gpu, [-1, 3], [1, 1], table, [3, 4], 2, 16, 14)
    run_plan(gpu, [20, 3], [2**31 - 1, 2**31 - 1], table, [3, 4], 2, 16, 14)
    run_plan(gpu, [20, 3], [1, 1], table, [3, 4], 3, 16, 14)  # num_free beyond the list
    run_plan(gpu, [20, 3], [1, 1], table, [3, 4], -1, 16, 14)
    run_plan(gpu, [20, 3], [-1, 1], table, [3, 4], 2, 16, 14)  # more come back than the list holds
    run_plan(gpu, [0, 3], [16, 1], [[7, 7], [2, -1]], [5, 4], 0, 16, 17)
    run_plan(gpu, [20, 3], [0, 0], table, [3, 4], 2, 16, 0)
    run_plan(gpu, [0, 0], [0, -1], table, [], 0, 16, 0)
    run_plan(gpu, [32, 3], [-1, 20], table, [3, 4, 9, 9], 0, 16, 20)  # blocks of the ended request are used again
    from compressed_tensors_amd.modeling import plan_kv_blocks

    none = torch.zeros(0, dtype=torch.int32, device=gpu)
    plan = plan_kv_blocks(none, none, none.view(0, 2), none + 1, torch.zeros(1, dtype=torch.int32, device=gpu),
                          block_size=16, total_tokens=3)
    assert plan.query_start.tolist() == [0] and plan.slots.tolist() == [-1] * 3 and plan.status.tolist() == [0]


# ---------------------------------------------------------------------------- the run of all
@pytest.mark.gpu
@pytest.mark.parametrize("codes", [FP8, torch.int8])
def test_serving_steps_with_packed_projections(gpu, codes):
    """prompts, decoding, an ended request and a new one in its place: plan, packed projections,
    append, attend, output projection, each step against the plain implementations"""
    from compressed_tensors_amd.linear import packed_linear
    from compressed_tensors_amd.modeling import BlockKVCache

    heads, kv, dim, hidden, size = 4, 2, 64, 256, 16
    g = torch.Generator().manual_seed(0)

    def weight(n, k):
        return (osv.pack4(torch.randint(0, 16, (n, k), generator=g)),
                ((0.5 + torch.rand(n, k // 32, generator=g)) * 0.01).bfloat16())

    qkv, proj = weight((heads + 2 * kv) * dim, hidden), weight(hidden, heads * dim)
    cache = BlockKVCache(2, 12, 3, 6, kv, dim, size, codes, device=gpu)
    plain = [[t.cpu().clone() for t in layer] for layer in cache.layers]
    lens, table, free, num_free = [0] * 3, [[-1] * 6 for _ in range(3)], list(range(11, -1, -1)), 12
    for step, new in enumerate(([20, 33, 0], [1, 1, 17], [1, 1, 1], [-1, 1, 1], [40, 1, 1], [1, 4, 1])):
        total = sum(a for a in new if a > 0)
        cache.plan(torch.tensor(new, dtype=torch.int32, device=gpu), total, max_query=max(new))
        cache.check()
        lens, starts, slots, table, free, num_free, status = osv.kv_plan(lens, new, table, free, num_free, size, total)
        assert status == 0 and cache.block_table.tolist() == table and cache.num_free.tolist() == [num_free]
        x = torch.randn(total, hidden, generator=g).bfloat16()
        for layer in range(2):
            announce("serving step", step, layer, codes)
            mixed = packed_linear(x.to(gpu), *(t.to(gpu) for t in qkv)).view(total, heads + 2 * kv, dim)
            q, k, v = mixed.split([heads, kv, kv], dim=1)
            cache.update(layer, k, v)
            osv.kv_append(k.cpu(), v.cpu(), plain[layer], torch.tensor(slots))
            for got, want in zip(cache.layers[layer][2:], plain[layer][2:]):
                used = sorted({b for row in table for b in row if b >= 0})
                assert torch.equal(got.cpu()[used], want[used])
            o = cache.attend(layer, q)
            check_attention(o, q.cpu(), plain[layer], torch.tensor(table, dtype=torch.int32),
                            torch.tensor(lens, dtype=torch.int32), torch.tensor(starts, dtype=torch.int32))
            x = packed_linear(o.flatten(1), *(t.to(gpu) for t in proj)).cpu()


@pytest.mark.gpu
@pytest.mark.parametrize("codes,kind", [(FP8, "float"), (torch.int8, "int")])
def test_cache_with_the_scales_of_a_calibrated_module(gpu, codes, kind):
    """k_scale / v_scale of an attention module under a kv_cache_scheme: the codes are those
    `quantize` gives with them"""
    from compressed_tensors_amd.modeling import BlockKVCache
    from compressed_tensors_amd.quantization import QuantizationArgs, quantize

    cache = BlockKVCache(1, 4, 1, 4, 2, 64, 16, codes, device=gpu)
    k_scale, v_scale = torch.tensor([0.011]).to(gpu), torch.tensor([0.02, 0.003]).view(2, 1, 1).to(gpu)
    cache.set_scales(0, k_scale, v_scale)
    with pytest.raises(ValueError):
        cache.set_scales(0, torch.ones(3).to(gpu), v_scale)
    k, v = torch.randn(20, 2, 64).bfloat16().to(gpu), torch.randn(20, 2, 64).bfloat16().to(gpu)
    cache.plan(torch.tensor([20], dtype=torch.int32, device=gpu), 20)
    cache.check()
    cache.update(0, k, v)
    args = QuantizationArgs(num_bits=8, type=kind, symmetric=True, strategy="tensor")
    pool = cache.layers[0]
    assert (pool.key_scale == 0.011).all() and (pool.value_scale[:, 1] == v_scale[1, 0, 0]).all()
    for h in range(2):
        for x, scale, got in ((k, k_scale, pool.key), (v, v_scale[h, 0], pool.value.transpose(2, 3))):
            want = quantize(x[:, h].float(), scale, torch.zeros_like(scale), args, dtype=codes)
            assert_bit_equal(got[:2, h].reshape(32, 64)[:20].contiguous().view(torch.uint8), want.cpu().view(torch.uint8), "codes")


@pytest.mark.gpu
def test_step_that_does_not_fit_changes_nothing(gpu):
    from compressed_tensors_amd.modeling import BlockKVCache

    cache = BlockKVCache(1, 2, 2, 4, 1, 64, 16, device=gpu)
    with pytest.raises(ValueError, match="plan"):
        cache.check()
    cache.plan(torch.tensor([20, 0], dtype=torch.int32, device=gpu), 20)
    cache.check()
    before = [t.clone() for t in (cache.seq_lens, cache.block_table, cache.free_blocks, cache.num_free)]
    cache.plan(torch.tensor([0, 17], dtype=torch.int32, device=gpu), 17)
    with pytest.raises(RuntimeError, match="short of 2 blocks"):
        cache.check()
    codes = [t.view(torch.uint8).clone() for t in cache.layers[0]]
    x = torch.randn(17, 1, 64).bfloat16().to(gpu)
    cache.update(0, x, x)
    out = torch.full_like(x, 3.0)
    assert cache.attend(0, x, out=out) is out and (out == 3).all()
    assert all(torch.equal(t.view(torch.uint8), c) for t, c in zip(cache.layers[0], codes))
    assert all(torch.equal(a, b) for a, b in zip(before, (cache.seq_lens, cache.block_table, cache.free_blocks, cache.num_free)))
    cache.plan(torch.tensor([0, 100], dtype=torch.int32, device=gpu), 100)
    with pytest.raises(ValueError, match="longer than its row"):
        cache.check()


@pytest.mark.gpu
def test_captured_decode_step(gpu):
    """a decode step in a graph, replayed over changed lengths, beside a second graph that shares
    the pool, with eager calls between the replays"""
    from compressed_tensors_amd.modeling import KVBlocks, append_kv_blocks, attend_kv_blocks

    lens = [2000, 130, 1]
    q, cache, table, lens_t, _ = attention_case(lens, [1, 1, 1], 8, 2, 64, 64, FP8, torch.bfloat16, seed=2)
    on, table_d, lens_d, q_d = KVBlocks(*(t.to(gpu) for t in cache)), table.to(gpu), lens_t.to(gpu), q.to(gpu)
    k, v = torch.randn(3, 2, 64).bfloat16(), torch.randn(3, 2, 64).bfloat16()
    k_d, v_d, slots = k.to(gpu), v.to(gpu), torch.zeros(3, dtype=torch.int64, device=gpu)
    graphs, outs = [], []
    slots.fill_(-1)
    for max_seq in (4096, 64):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            append_kv_blocks(k_d, v_d, on, slots)
            outs.append(attend_kv_blocks(q_d, on, table_d, lens_d, max_seq=max_seq))
        graphs.append(graph)
    for new_lens in ([2000, 130, 1], [1500, 64, 1], [7, 129, 0]):
        lens_t = torch.tensor(new_lens, dtype=torch.int32)
        lens_d.copy_(lens_t)
        at = [max(n - 1, 0) for n in new_lens]
        slot = torch.tensor([int(table[r, p // 64]) * 64 + p % 64 for r, p in enumerate(at)])
        slots.copy_(slot)
        for graph in graphs:
            graph.replay()
        eager = attend_kv_blocks(q_d, on, table_d, lens_d, max_seq=4096)
        torch.cuda.synchronize()
        osv.kv_append(k, v, cache, slot)
        osv.kv_append(k, v, cache, slot)
        assert torch.equal(outs[0], eager)
        for out in outs:
            check_attention(out, q, cache, table, lens_t, None)


# -------------------------------------------------------------------------------- refusals
def test_refusals():
    from compressed_tensors_amd.modeling import KVBlocks, append_kv_blocks, attend_kv_blocks, plan_kv_blocks

    q, cache, table, lens, starts = attention_case([20, 5], [1, 1], 4, 2, 64, 16, FP8, torch.bfloat16)
    blocks = KVBlocks(*cache)
    k = torch.zeros(2, 2, 64).bfloat16()
    slots = torch.zeros(2, dtype=torch.int64)
    bad_pools = [blocks._replace(value=blocks.value.transpose(2, 3)), blocks._replace(key_scale=blocks.key_scale.half()),
                 blocks._replace(value_scale=blocks.value_scale[:1]), blocks._replace(key=blocks.key[0])]
    for bad in bad_pools:
        with pytest.raises(ValueError):
            append_kv_blocks(k, k, bad, slots)
        with pytest.raises(ValueError):
            attend_kv_blocks(q, bad, table, lens)
    for size, dim, dtype in ((20, 64, FP8), (512, 64, FP8), (16, 80, FP8), (16, 64, torch.uint8)):
        with pytest.raises(NotImplementedError):
            KVBlocks.allocate(2, 2, dim, size, dtype, device="cpu")
    for args in ((k[:, :1], k[:, :1], blocks, slots), (k, k[:1], blocks, slots), (k, k, blocks, slots[:1]),
                 (k, k, blocks, slots.int())):
        with pytest.raises(ValueError):
            append_kv_blocks(*args)
    with pytest.raises(NotImplementedError):
        append_kv_blocks(k.float(), k.float(), blocks, slots)
    with pytest.raises(NotImplementedError):
        append_kv_blocks(k.clone().requires_grad_(), k, blocks, slots)
    for args in ((q[:, :3], blocks, table, lens), (q[..., :32], blocks, table, lens), (q, blocks, table.long(), lens),
                 (q, blocks, table[:1], lens), (q, blocks, table, lens.long()), (q, blocks, table, lens, starts[:2]),
                 (q[:1], blocks, table, lens)):
        with pytest.raises(ValueError):
            attend_kv_blocks(*args)
    for out in (q.float(), q[:, :2], q.transpose(0, 1)):
        with pytest.raises(ValueError):
            attend_kv_blocks(q, blocks, table, lens, out=out)
    with pytest.raises(NotImplementedError):
        attend_kv_blocks(q.float(), blocks, table, lens)
    with pytest.raises(NotImplementedError):
        attend_kv_blocks(q.clone().requires_grad_(), blocks, table, lens)
    one, free = torch.zeros(1, dtype=torch.int32), torch.zeros(4, dtype=torch.int32)
    for args in ((lens.long(), lens, table, free, one), (lens, lens[:1], table, free, one), (lens, lens, table[0], free, one),
                 (lens, lens, table, free, free)):
        with pytest.raises(ValueError):
            plan_kv_blocks(*args, block_size=16, total_tokens=1)
    with pytest.raises(ValueError):
        plan_kv_blocks(lens, lens, table, free, one, block_size=0, total_tokens=1)
    for call in (lambda: append_kv_blocks(k, k, blocks, slots), lambda: attend_kv_blocks(q, blocks, table, lens),
                 lambda: plan_kv_blocks(lens, lens, table, free, one, block_size=16, total_tokens=1)):
        with pytest.raises(RuntimeError, match="GPU only"):
            call()


def test_abi_refusals(ctmi):
    from ctypes import byref

    from compressed_tensors_amd._lib import KVBlocksC

    def blocks(num=4, heads=2, dim=64, size=16, code=3, at=16):
        return KVBlocksC(at, at, at, at, num, heads, dim, size, code)

    def append(b, dtype=2, tokens=2, at=16, stride=128):
        return ctmi.ctmi_kv_append(at, at, dtype, stride, 64, 128, 64, at, tokens, byref(b), 1, None)

    for bad, code in ((blocks(dim=80), -2), (blocks(size=24), -2), (blocks(size=272), -2), (blocks(code=8), -2),
                      (blocks(heads=0), -1), (blocks(num=-1), -1), (blocks(at=0), -1), (blocks(at=8), -1)):
        assert append(bad) == code
    assert append(blocks(), dtype=0) == -2 and append(blocks(), tokens=-1) == -1 and append(blocks(), at=0) == -1
    assert append(blocks(), tokens=0) == 0 and append(blocks(), stride=100) == -1 and append(blocks(), at=24) == -1

    def attend(b=None, dtype=2, tokens=2, heads=4, stride=128, width=3, table_stride=3, requests=2, start=16, at=16,
               max_query=1, max_seq=48, tmp=0):
        b = b or blocks()
        return ctmi.ctmi_kv_attend(at, dtype, stride, 64, at, tokens, heads, byref(b), at, table_stride, width, at, start,
                                   requests, 0.1, max_query, max_seq, None, tmp, None)

    assert attend(blocks(dim=96)) == -2 and attend(dtype=0) == -2 and attend(heads=3) == -1 and attend(heads=0) == -1
    assert attend(table_stride=2) == -1 and attend(start=None, tokens=3) == -1 and attend(at=0) == -1
    assert attend(stride=100) == -1 and attend(at=24) == -1 and attend(max_query=0) == -1 and attend(max_seq=0) == -1
    assert attend(tokens=0) == 0 and attend(requests=0) == 0 and attend(width=1 << 30, table_stride=1 << 30) == -2

    def plan(requests=2, width=3, capacity=4, slots=5, size=16, at=16):
        return ctmi.ctmi_kv_plan(at, at, at, at, at, requests, width, capacity, slots, size, at, at, at, at, at, at, at, None)

    assert plan(requests=4097) == -2 and plan(requests=-1) == -1 and plan(width=0) == -1 and plan(size=0) == -1
    assert plan(at=0) == -1 and plan(capacity=-1) == -1 and plan(slots=1 << 31) == -2


@pytest.mark.parametrize("codes", [FP8, torch.int8])
def test_plain_append_keeps_what_it_is_given(codes):
    """the oracle's own ground: what comes back is within half a step of what went in, older
    codes within half a step more for each time their scale grew"""
    cache = pool(3, 2, 16, 64, codes)
    xs = [torch.randn(1, 2, 64) * 2 ** i for i in range(5)]
    for i, x in enumerate(xs):
        osv.kv_append(x.bfloat16(), x.bfloat16(), cache, torch.tensor([16 + i]))
    for side, transposed in ((0, False), (1, True)):
        codes_of = cache[side].transpose(2, 3) if transposed else cache[side]
        for i, x in enumerate(xs):
            back = codes_of[1, :, i].float() * cache[2 + side][1].view(-1, 1)
            step = cache[2 + side][1].view(-1, 1) * (1.0 if codes is torch.int8 else 2.0 ** -9)
            rel = 0.0 if codes is torch.int8 else 2.0 ** -4
            hops = len(xs) - i
            assert ((back - x[0].bfloat16().float()).abs() <= hops * (step * 0.51 + rel * x[0].abs() * 1.07) ).all()
