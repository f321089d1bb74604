"""A query that is not a number gives an output that is none, not the zeros of a row without keys."""
import math

import pytest
import torch

import kv_reference as R

pytestmark = pytest.mark.gpu


# one row and few, in one thread block and shared; a tile of many columns, whole and shared
@pytest.mark.parametrize("tokens,rows,heads,kv", [(100, 1, 4, 2), (9000, 2, 4, 2), (700, 9, 8, 1), (300, 200, 4, 2),
                                                  (6000, 150, 4, 1), (300, 700, 16, 4)])
@pytest.mark.parametrize("d,dtype", [(64, torch.float16), (128, torch.bfloat16)])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("selected", [False, True])
def test_a_bad_query_shows(tokens, rows, heads, kv, d, dtype, bad, selected):
    from gofann.kv_cache import KVCache
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    case = R.Case([tokens], [rows], heads, kv, d, dtype, spare=60)
    cache, q = KVCache(d, pages=case.random_pages()), case.normal(rows, heads, d)
    ids = None
    if selected:
        ids = torch.full((rows, kv, 40), -1, dtype=torch.int32, device="cuda")
        ids[:, :, 7] = 0
    q[rows - 1, 1, 5] = bad
    q[0, heads - 1, d - 1] = bad
    out, lse = cache.attend(case.batch(), q, selected=ids)
    hit = torch.zeros(rows, heads, dtype=torch.bool, device="cuda")
    hit[rows - 1, 1] = hit[0, heads - 1] = True
    before = torch.tensor(case.row_pos, device="cuda") < 0  # rows before the first token see no key
    assert out[before].eq(0).all() and lse[before].eq(-math.inf).all()
    hit &= ~before[:, None]
    assert out[hit].isnan().all() and lse[hit].isnan().all()
    fine = ~hit & ~before[:, None]
    assert torch.isfinite(out[fine]).all() and torch.isfinite(lse[fine]).all()
    # where nothing is seen it is a row without keys all the same
    out, lse = cache.attend(case.batch(), q, selected=ids, key_bits=torch.zeros(1, 4, dtype=torch.int32, device="cuda"))
    assert out.eq(0).all() and lse.eq(-math.inf).all()
