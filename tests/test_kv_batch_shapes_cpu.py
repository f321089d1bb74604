"""Tensors of a batch that have the right first size only are refused."""
import pytest
import torch

from gofann import kv_cache as KV


def ints(*n):
    return torch.zeros(*n, dtype=torch.int32)


@pytest.mark.parametrize("table,lens,offset", [((2, 4), (2, 2), (3,)), ((2, 4), (2, 1), (3,)), ((2, 4), (), (3,)),
                                               ((2, 4, 1), (2,), (3,)), ((2, 4), (2,), (3, 1)), ((2, 4), (2,), (2,))])
def test_shapes(table, lens, offset):
    with pytest.raises(ValueError, match="disagree"):
        KV.KVBatch(ints(*table), ints(*lens) if lens else torch.tensor(0, dtype=torch.int32), ints(*offset), 2, 1)
    KV.KVBatch(ints(2, 4), ints(2), ints(3), 2, 1)
