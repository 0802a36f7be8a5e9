"""attend_kv_blocks without hints, as BlockKVCache calls it: the launch fits what the batch looks
like, finds its requests by itself and is never refused for their number"""
import pytest
import torch

from gpu_util import announce
from test_kv_blocks import FP8, attention_case, check_attention, run_attention
from test_kv_weights import check


@pytest.mark.gpu
@pytest.mark.parametrize("codes,dtype", [(FP8, torch.bfloat16), (torch.int8, torch.float16)])
@pytest.mark.parametrize("news,heads,kv,dim,size", [
    ([1] * 70, 8, 2, 64, 16), ([0, 3, 0, 0, 1] * 30, 4, 4, 64, 32), ([40] + [1] * 20 + [0] * 60, 8, 2, 128, 16),
    ([0] * 200 + [9], 8, 1, 64, 16), ([0] * 3, 8, 2, 64, 16), ([33, 1, 0, 64, 129, 2], 8, 2, 64, 64), ([5], 66, 1, 64, 16),
    ([1] * 65, 66, 1, 64, 16), ([2, 0] * 130 + [17], 2, 2, 256, 16), ([1, 0, 1] * 1500, 1, 1, 64, 16),
])
def test_any_batch(gpu, codes, dtype, news, heads, kv, dim, size):
    announce("no hints", len(news), sum(news), heads, kv, dim, size, codes)
    g = torch.Generator().manual_seed(len(news))
    lens = [n + int(torch.randint(0, 40, (1,), generator=g)) for n in news]
    for pad in (0, 5):
        data = attention_case(lens, news, heads, kv, dim, size, codes, dtype, seed=2, pad=pad)
        check_attention(run_attention(gpu, *data), *data)


@pytest.mark.gpu
def test_a_decode_step_takes_the_kernel_of_one(gpu):
    """a batch of one token a request through the class, which has no hints: the bits of the call
    that has them, with weights of 24 bits"""
    from compressed_tensors_amd.modeling import BlockKVCache, attend_kv_blocks

    g = torch.Generator().manual_seed(0)
    cache = BlockKVCache(1, 60, 24, 4, 2, 64, 64, device=gpu)
    lens = torch.randint(1, 200, (24,), generator=g, dtype=torch.int32)
    for new in (lens, torch.ones_like(lens)):
        n = int(new.sum())
        cache.plan(new.to(gpu), n)
        cache.check()
        k, v = (torch.randn(n, 2, 64, generator=g).bfloat16().to(gpu) for _ in range(2))
        cache.update(0, k, v)
    q = torch.randn(24, 8, 64, generator=g).bfloat16().to(gpu)
    got = cache.attend(0, q)
    same = attend_kv_blocks(q, cache.layers[0], cache.block_table, cache.seq_lens, cache._current().query_start, max_query=1)
    assert torch.equal(got, same)
    check(got, q.cpu(), [t.cpu() for t in cache.layers[0]], cache.block_table.cpu(), cache.seq_lens.cpu(),
          cache._current().query_start.cpu(), slice(None), False, 0, 0)


@pytest.mark.gpu
def test_many_requests_of_many_heads_are_not_refused(gpu):
    """8192 requests x 64 kv heads x tiles for all 70000 tokens would be more workgroups than a launch has"""
    from compressed_tensors_amd.modeling import KVBlocks, attend_kv_blocks
    from oracle import serving as osv

    announce("many requests and heads")
    requests, kv, heads = 8192, 64, 512
    g = torch.Generator().manual_seed(0)
    news = torch.randint(0, 18, (requests,), generator=g)
    starts = torch.zeros(requests + 1, dtype=torch.int32)
    starts[1:] = news.cumsum(0)
    tokens = int(starts[-1])
    pool = KVBlocks(*(torch.randint(-90, 90, (40, kv, *s), dtype=torch.int8, device=gpu) for s in ((16, 64), (64, 16))),
                    *(torch.rand(40, kv, device=gpu) * 0.02 for _ in range(2)))
    table = torch.randint(0, 40, (requests, 2), generator=g, dtype=torch.int32)
    lens = (news + torch.randint(0, 14, (requests,), generator=g)).to(torch.int32)
    q = torch.randn(tokens, heads, 64, device=gpu, dtype=torch.bfloat16)
    args = (pool, table.to(gpu), lens.to(gpu), starts.to(gpu))
    got = attend_kv_blocks(q, *args)
    for hint in (17, tokens):
        other = attend_kv_blocks(q, *args, max_query=hint, max_seq=32)
        assert (other - got).abs().max() <= 2.0 ** -6 * got.abs().max()
    plain = [t.cpu() for t in pool]
    for r in (0, 1, 4095, 4096, 8190, 8191):
        a, b = int(starts[r]), int(starts[r + 1])
        if a < b:
            check_attention(got[a:b], q[a:b].cpu(), plain, table[r:r + 1], lens[r:r + 1], torch.tensor([0, b - a]))
