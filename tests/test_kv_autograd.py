"""the block cache's calls refuse what forward-mode differentiation would follow"""
import pytest
import torch
from torch.autograd import forward_ad

from test_kv_blocks import FP8, attention_case


def test_dual_tensors_are_refused():
    from compressed_tensors_amd.modeling import KVBlocks, append_kv_blocks, attend_kv_blocks

    q, cache, table, lens, _ = attention_case([20, 5], [1, 1], 4, 2, 64, 16, FP8, torch.bfloat16)
    blocks, k, slots = KVBlocks(*cache), torch.zeros(2, 2, 64).bfloat16(), torch.zeros(2, dtype=torch.int64)
    with forward_ad.dual_level():
        for mode in (torch.enable_grad(), torch.no_grad()):
            with mode:
                dual = forward_ad.make_dual(k, torch.ones_like(k))
                for args in ((dual, k), (k, dual)):
                    with pytest.raises(NotImplementedError, match="forward-mode"):
                        append_kv_blocks(*args, blocks, slots)
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    attend_kv_blocks(forward_ad.make_dual(q, torch.ones_like(q)), blocks, table, lens)
        with pytest.raises(RuntimeError, match="GPU only"):
            attend_kv_blocks(q, blocks, table, lens)
