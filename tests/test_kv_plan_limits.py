"""plan_kv_blocks at the end of what a length holds"""
import pytest
import torch

from gpu_util import announce


@pytest.mark.gpu
@pytest.mark.parametrize("length,new,status", [(2**31 - 3, 2, 0), (2**31 - 3, 3, -1), (2**31 - 1, 1, -1), (2**31 - 1, 2**31 - 1, -1)])
def test_lengths_of_31_bits(gpu, length, new, status):
    """a request whose length 32 bits would not hold does not fit, whatever its table row does"""
    from compressed_tensors_amd.modeling import plan_kv_blocks

    announce("plan", length, new)
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device=gpu)  # noqa: E731
    size, width = 1 << 20, 5000
    table = torch.arange(width, dtype=torch.int32, device=gpu).view(1, width)
    table[0, 2048:] = -1
    plan = plan_kv_blocks(ints(length), ints(new), table, ints(7000, 7001, 7002), ints(3), block_size=size, total_tokens=4)
    assert plan.status.tolist() == [status]
    assert plan.seq_lens.tolist() == [length + new if status == 0 else length]
    if status == 0:
        last = 2047 * size + length % size
        assert plan.slots.tolist() == [last, last + 1, -1, -1] and plan.num_free.tolist() == [3]
    else:
        assert plan.slots.tolist() == [-1] * 4 and torch.equal(plan.block_table, table) and plan.query_start.tolist() == [0, 0]
