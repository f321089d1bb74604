"""A mask of no words hides every token."""
import math

import pytest
import torch

import kv_reference as R

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [1, 200])
def test_no_words_hide_every_token(rows):
    from gofann.kv_cache import KVCache
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    case = R.Case([300], [rows], 4, 2, 64, torch.bfloat16)
    out, lse = KVCache(64, pages=case.random_pages()).attend(
        case.batch(), case.normal(rows, 4, 64), key_bits=torch.zeros(1, 0, dtype=torch.int32, device="cuda"))
    assert out.eq(0).all() and lse.eq(-math.inf).all()
