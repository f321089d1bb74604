"""Queries near either end of bf16, whose scaled products are ordinary logits."""
import pytest
import torch

import kv_reference as R
from test_kv_cache_gpu import run_attend

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [2, 300])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("size,scale", [(1e34, 1e-35), (1e36, 1e-37), (6e37, 2e-38), (1e-35, 1e34), (1e-28, 1e27)])
def test_attend_at_the_ends_of_bf16(rows, d, size, scale):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    case = R.Case([300], [rows], 4, 1, d, torch.bfloat16)
    q = (case.normal(rows, 4, d).float().clamp(-5, 5) * size).to(torch.bfloat16)
    run_attend(case, q=q, scale=scale)
