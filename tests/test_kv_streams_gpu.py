"""Calls on a stream that is not the current one, while that stream is busy and the current one takes memory."""
import pytest
import torch

import kv_reference as R

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _device():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def fill_freed_memory():
    """Overwrites what the current stream's allocator has to give at once."""
    torch.cuda.current_stream().synchronize()
    return [torch.full((size,), 0x55, dtype=torch.uint8, device="cuda")
            for size in (512, 512, 512, 2048, 1 << 14, 1 << 17, 1 << 19, 1 << 21, 3 << 20, 5 << 20, 9 << 20) for _ in range(4)]


@pytest.mark.parametrize("rows", [1, 150])
def test_arguments_scratch_and_outputs_outlive_their_names(rows):
    from gofann.kv_cache import KVCache, rope_tables
    case = R.Case([5000, 300], [rows, 1], 8, 2, 128, torch.bfloat16)
    n = case.n_rows
    cos, sin = rope_tables(5000, 128)
    q, k, v = case.normal(n, 8, 128), case.normal(n, 2, 128), case.normal(n, 2, 128)
    pages = case.random_pages()

    def fresh():
        return KVCache(128, pages=pages.clone(), bounds=torch.zeros(case.n_pages, 2, 2, 128, dtype=torch.int8, device="cuda"),
                       bound_scale=torch.zeros(case.n_pages, 2, device="cuda"))

    cache = fresh()
    rq, *_ = cache.append(case.batch(), q, k, v, cos=cos, sin=sin, rotary_dim=128)
    ids, scores = cache.select(case.batch(), rq, 20)
    out, lse = cache.attend(case.batch(), rq)
    want = [x.clone() for x in (rq, ids, scores, out, lse)]
    cache = fresh()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)  # some 0.1 s: the calls below are queued behind it
    # batches, scratch and copies of the arguments are dropped at once
    got_q, *_ = cache.append(case.batch(), q.clone(), k.clone(), v.clone(), cos=cos, sin=sin, rotary_dim=128, stream=side)
    junk = fill_freed_memory()
    got_ids, got_scores = cache.select(case.batch(), got_q, 20, stream=side)
    junk += fill_freed_memory()
    got_out, got_lse = cache.attend(case.batch(), got_q, stream=side)
    junk += fill_freed_memory()
    torch.cuda.synchronize()
    for a, b in zip((got_q, got_ids, got_scores, got_out, got_lse), want):
        assert torch.equal(a, b)


def test_a_graph_outlives_a_larger_call_of_its_batch():
    """The scratch that a captured call uses stays its own when a later call of the batch needs more."""
    from gofann.kv_cache import KVCache
    case = R.Case([3000] * 6, [1] * 6, 4, 2, 64, torch.float16)
    bounds = torch.randint(-100, 100, (case.n_pages, 2, 2, 64), device="cuda", generator=case.g, dtype=torch.int8)
    cache = KVCache(64, pages=case.random_pages(), bounds=bounds, bound_scale=torch.ones(case.n_pages, 2, device="cuda"))
    batch, q = case.batch(), case.normal(6, 4, 64)
    want, _ = cache.select(batch, q, 9)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ids, _ = cache.select(batch, q, 9)
    cache.attend(batch, q)
    junk = fill_freed_memory()
    for _ in range(3):
        ids.fill_(-5)
        graph.replay()
        assert torch.equal(ids, want)
    assert all(bool((x == 0x55).all()) for x in junk)
