"""What the device finds out of range is skipped: nothing is written for it, nothing is read, the status word is set."""
import math

import pytest
import torch

import kv_reference as R

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def _device():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def expect_invalid(batch):
    from gofann import _abi as A
    with pytest.raises(A.GofannError) as e:
        batch.check()
    assert e.value.status == A.ERR_INVALID


def filled(case):
    """A cache whose pages and bounds hold something everywhere."""
    from gofann.kv_cache import KVCache
    pages = torch.randint(0, 256, (case.n_pages, case.kv, R.chunk_size(case.d)), device="cuda", generator=case.g,
                          dtype=torch.uint8) & 0x3b
    bounds = torch.randint(-127, 128, (case.n_pages, case.kv, 2, case.d), device="cuda", generator=case.g, dtype=torch.int8)
    return KVCache(case.d, pages=pages, bounds=bounds, bound_scale=torch.rand(case.n_pages, case.kv, device="cuda",
                                                                            generator=case.g))


def append(case, cache, q, k, v, cos, sin, rotary, interleaved, **kw):
    n = case.n_rows
    outs = [torch.full((n, h, case.d), 9.0, dtype=case.dtype, device="cuda") for h in (case.heads, case.kv, case.kv)]
    batch = case.batch()
    cache.append(batch, q, k, v, cos=cos, sin=sin, rotary_dim=rotary, interleaved=interleaved, q_out=outs[0], k_out=outs[1],
                 v_out=outs[2], **kw)
    return batch, outs


@pytest.mark.parametrize("fault", ["length", "offset above", "offsets descend"])
@pytest.mark.parametrize("d,rows", [(64, 2), (128, 70)])
def test_append_leaves_the_pages_of_a_skipped_sequence(fault, d, rows):
    """The second of three sequences: the others get what they get without it."""
    from gofann.kv_cache import rope_tables
    case = R.Case([200, 64 * 5 - 3, 130], [3, rows, 2], 4, 2, d, BF16)
    q, k, v = case.normal(case.n_rows, 4, d), case.normal(case.n_rows, 2, d), case.normal(case.n_rows, 2, d)
    cos, sin = rope_tables(64 * 8, d)
    right, wrong = filled(case), None
    before = right.pages.clone(), right.bounds.clone(), right.bound_scale.clone()
    wrong = type(right)(d, pages=before[0].clone(), bounds=before[1].clone(), bound_scale=before[2].clone())
    _, want = append(case, right, q, k, v, cos, sin, d, False)
    gone = [1]
    if fault == "length":
        case.seq_len[1] = 64 * case.max_pages + 1
    elif fault == "offset above":
        case.row_offset[2] = case.n_rows + 1  # the third sequence's offsets descend then
        gone = [1, 2]
    else:
        case.row_offset[1] = case.row_offset[2] + 1  # the first sequence has more rows than its own: they are its newest
        gone = [1]
    batch, got = append(case, wrong, q, k, v, cos, sin, d, False)
    expect_invalid(batch)
    for s in gone:
        pages = case.table[s].long()
        for now, then in zip((wrong.pages, wrong.bounds, wrong.bound_scale), before):
            assert torch.equal(now[pages], then[pages])
    if fault != "offsets descend":
        first = case.table[0].long()
        assert torch.equal(wrong.pages[first], right.pages[first]) and torch.equal(wrong.bounds[first], right.bounds[first])
        for a, b in zip(got, want):
            assert torch.equal(a[:3], b[:3]) and a[3 : 3 + rows].eq(9.0).all()


@pytest.mark.parametrize("d,rotary,interleaved", [(64, 64, False), (128, 128, True), (128, 34, False), (64, 2, True)])
@pytest.mark.parametrize("rows", [5, 90])
@pytest.mark.parametrize("explicit", [False, True])
def test_append_does_not_write_rows_without_a_position(d, rotary, interleaved, rows, explicit):
    from gofann.kv_cache import rope_tables
    case = R.Case([201, 130], [rows, 4], 6, 2, d, F16)
    n = case.n_rows
    q, k, v = case.normal(n, 6, d), case.normal(n, 2, d), case.normal(n, 2, d)
    at = torch.tensor(case.row_pos, device="cuda")
    bad = torch.zeros(n, dtype=torch.bool, device="cuda")
    if explicit:
        positions = torch.randint(0, 500, (n,), device="cuda", generator=case.g, dtype=torch.int32)
        bad[[1, 3, rows, n - 1]] = True
        positions[1], positions[3], positions[rows], positions[n - 1] = -1, 500, 1 << 30, -(1 << 31)
        cos, sin = rope_tables(500, rotary)
    else:
        positions = None
        bad = at >= 198  # the newest three of the first sequence
        cos, sin = rope_tables(198, rotary)
    cache = filled(case)
    before = cache.pages.clone()
    batch, (q_out, k_out, v_out) = append(case, cache, q, k, v, cos, sin, rotary, interleaved, positions=positions)
    expect_invalid(batch)
    for x in (q_out, k_out, v_out):
        assert x[bad].eq(9.0).all()
    # the others, by the formula; the skipped rows' places as before
    use = at if positions is None else positions.long()
    use = torch.where(bad, 0, use)
    rq, rk = (R.rotate(x, cos[use], sin[use], rotary, interleaved, torch.float32) for x in (q, k))
    assert torch.equal(q_out[~bad], rq.to(F16)[~bad])
    state = R.decode(before, d)
    for new, old in zip((R.quantise(rk), R.quantise(v.float())), state):
        for r, (s, p) in enumerate(zip(case.row_seq, case.row_pos)):
            if not bad[r]:
                for x, y in zip(old, new):
                    x[int(case.table[s, p // 64]), :, p % 64] = y[r].to(x.dtype)
    for got, want in zip(R.decode(cache.pages, d), state):
        for x, y in zip(got, want):
            assert torch.equal(x, y)
    # the bounds are those of all that the pages hold
    from test_kv_cache_gpu import expect_bounds
    for s, b in {(s, p // 64) for s, p in zip(case.row_seq, case.row_pos)}:
        page = int(case.table[s, b])
        bounds, unit = expect_bounds(case, state, page, min(64, case.lens[s] - 64 * b))
        assert torch.equal(cache.bounds[page], bounds) and torch.equal(cache.bound_scale[page], unit)


@pytest.mark.parametrize("blocks", [5, 300, 2100])
def test_select_gives_a_skipped_sequence_no_blocks(blocks):
    case = R.Case([64 * blocks, 64 * blocks - 9], [2, 3], 4, 2, 64, BF16)
    cache, q = filled(case), case.normal(5, 4, 64)
    want, want_scores = cache.select(case.batch(), q, 4)
    case.seq_len[0] = 64 * case.max_pages + 1
    batch = case.batch()
    ids, scores = cache.select(batch, q, 4)
    expect_invalid(batch)
    assert ids[:2].eq(-1).all() and scores[:2].eq(-math.inf).all()
    assert torch.equal(ids[2:], want[2:]) and torch.equal(scores[2:], want_scores[2:])


@pytest.mark.parametrize("rows,selected", [(1, False), (1, True), (200, False)])
def test_attention_gives_a_skipped_sequence_no_keys(rows, selected):
    case = R.Case([700, 650], [rows, rows], 4, 2, 64, BF16, spare=80)
    from gofann.kv_cache import KVCache
    cache, q = KVCache(64, pages=case.random_pages()), case.normal(2 * rows, 4, 64)
    ids = torch.arange(5, device="cuda").int().expand(2 * rows, 2, 5).contiguous() if selected else None
    want, want_lse = cache.attend(case.batch(), q, selected=ids)
    case.seq_len[0] = 64 * case.max_pages + 1
    batch = case.batch()
    out, lse = cache.attend(batch, q, selected=ids)
    expect_invalid(batch)
    assert out[:rows].eq(0).all() and lse[:rows].eq(-math.inf).all()
    # (other shares of the work: sums in another order)
    assert torch.allclose(out[rows:].float(), want[rows:].float(), atol=2e-2) and torch.allclose(lse[rows:], want_lse[rows:])
    case.seq_len[0] = 700
    case.row_offset[1] = 2 * rows + 1  # no sequence has rows
    batch = case.batch()
    cache.attend(batch, q, selected=ids)
    expect_invalid(batch)
