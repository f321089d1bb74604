"""Queries so large that scores overflow: an infinite score is a score, and blocks that are always kept are kept."""
import math

import pytest
import torch

import kv_reference as R

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("blocks,rows", [(9, 1), (150, 3), (150, 700), (2100, 1)])
@pytest.mark.parametrize("group", [1, 4, 20])
def test_infinite_scores(blocks, rows, group):
    from gofann.kv_cache import KVCache
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    d, want, first, recent = 64, 6, 2, 2
    case = R.Case([64 * blocks], [rows], group, 1, d, torch.bfloat16)
    bounds = torch.randint(-127, 128, (case.n_pages, 1, 2, d), device="cuda", generator=case.g, dtype=torch.int8)
    sign = torch.randint(0, 4, (case.n_pages, 1, 1, 1), device="cuda", generator=case.g)
    # a quarter of the blocks has products of either sign, the others -inf
    bounds = torch.where(sign == 0, bounds, bounds.abs().clamp(min=1))
    unit = torch.rand(case.n_pages, 1, device="cuda", generator=case.g) * 0.01 + 0.01
    q = -(case.normal(rows, group, d).float().abs() + 1).mul(1e37).to(torch.bfloat16)
    batch = case.batch()
    ids, scores = KVCache(d, bounds=bounds, bound_scale=unit).select(batch, q, want, first=first, recent=recent)
    batch.check()
    b = bounds[case.table[0].long(), 0].float()
    seen = set()
    for r in range(0, rows, max(1, rows // 3)):
        n = case.row_pos[r] // 64 + 1
        best = torch.full((n,), -math.inf, device="cuda")
        for h in range(group):
            x = q[r, h].float()
            qs = x.abs().max() / torch.tensor(127.0, device="cuda")
            q8 = (x / qs).round().clamp(-127, 127)
            dot = (q8.clamp(min=0) * b[:n, 0] + q8.clamp(max=0) * b[:n, 1]).sum(-1)  # integers below 2^24
            best = torch.maximum(best, dot * qs)
        score = (best * unit[case.table[0, :n].long(), 0]).cpu()
        kept = lambda i: i < first or i >= n - recent  # noqa: E731
        order = sorted(range(n), key=lambda i: (not kept(i), -float(score[i]), i))[:want]
        assert ids[r, 0].tolist() == sorted(order)
        assert torch.equal(scores[r, 0].cpu(), score[sorted(order)])
        seen |= {float(x) for x in score if math.isinf(x)}
    assert -math.inf in seen
