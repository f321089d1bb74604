"""What follows attention in its stream reads the whole result, where none of its items is shared between blocks too."""
import pytest
import torch

import kv_reference as R

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _device():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


# A table far longer than the sequences: the work is a few units, all of one thread block, and the joining kernel that
# is launched beside it has nothing to do.  rows 1: few query columns, rows 100: many.
CASES = [([60], 1, 8, 8), ([100, 33], 1, 4, 2), ([100], 100, 4, 1), ([64 * 7], 64, 16, 2)]


def setting(lens, rows, heads, kv):
    from gofann.kv_cache import KVCache
    case = R.Case(lens, [min(n, rows) for n in lens], heads, kv, 128, torch.bfloat16, spare=1200)
    q = case.normal(case.n_rows, heads, 128)
    out, lse = torch.empty_like(q), torch.empty(case.n_rows, heads, device="cuda")
    return KVCache(128, pages=case.random_pages()), case.batch(), q, out, lse


@pytest.mark.parametrize("lens,rows,heads,kv", CASES)
def test_the_next_call_reads_the_whole_result(lens, rows, heads, kv):
    cache, batch, q, out, lse = setting(lens, rows, heads, kv)
    cache.attend(batch, q, out=out, lse=lse)
    torch.cuda.synchronize()
    want, want_lse = out.clone(), lse.clone()
    for _ in range(50):
        out.fill_(7.0), lse.fill_(7.0)
        cache.attend(batch, q, out=out, lse=lse)
        got, got_lse = out * 1, lse * 1
        assert torch.equal(got, want) and torch.equal(got_lse, want_lse)


@pytest.mark.parametrize("lens,rows,heads,kv", CASES)
def test_the_next_node_of_a_graph_reads_the_whole_result(lens, rows, heads, kv):
    cache, batch, q, out, lse = setting(lens, rows, heads, kv)
    cache.attend(batch, q, out=out, lse=lse)
    torch.cuda.synchronize()
    want, want_lse = out.clone(), lse.clone()
    got, got_lse = torch.empty_like(out), torch.empty_like(lse)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out.fill_(7.0), lse.fill_(7.0)
        cache.attend(batch, q, out=out, lse=lse)
        got.copy_(out), got_lse.copy_(lse)
    for _ in range(50):
        graph.replay()
        assert torch.equal(got, want) and torch.equal(got_lse, want_lse)


@pytest.mark.parametrize("heads", [32, 9])
def test_long_rows_of_many_heads_are_picked_from_whole_scores(heads):
    """More than 8 query heads: the scoring kernel reads its scores back, whose lines neighbouring rows share; more than
    2048 blocks: the picking kernel reads them from memory."""
    from test_kv_cache_gpu import check_select
    check_select(R.Case([64 * 2300 - 5, 64 * 2101], [3, 2], heads, 1, 64, torch.float16), 40)
