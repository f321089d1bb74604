"""The cache operators on a GPU against plain 64-bit forms (kv_reference.py).

append and select are integers and single rounded products: codes, params,
bounds, ids and scores have to be equal to the last bit.  attend is held to a
bound from its number formats (kv_reference.attention)."""
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


# ------------------------------------------------------------------- append
def expect_append(case, before, q, k, v, cos, sin, rotary, interleaved, positions=None):
    """Pages' codes and params, bounds, rotated queries and held values after an append, from 32-bit steps."""
    d = case.d
    at = torch.tensor(case.row_pos, device="cuda") if positions is None else positions.long()
    rq = rk = None
    if rotary:
        rq = R.rotate(q, cos[at], sin[at], rotary, interleaved, torch.float32)
        rk = R.rotate(k, cos[at], sin[at], rotary, interleaved, torch.float32)
    else:
        rq, rk = q.float(), k.float()
    new = [R.quantise(rk), R.quantise(v.float())]
    state = R.decode(before, d)
    for r, (s, p) in enumerate(zip(case.row_seq, case.row_pos)):
        if p < 0:
            continue
        page = int(case.table[s, p // R.PAGE])
        for old, add in zip(state, new):
            for x, y in zip(old, add):
                x[page, :, p % R.PAGE] = y[r].to(x.dtype)
    held = []
    for code, scale, low in new:
        c = code.float().unflatten(-1, (-1, R.GROUP))
        held.append(((c * scale.float()[..., None]) + low.float()[..., None]).flatten(-2).to(case.dtype))
    return rq.to(case.dtype), held, state


def expect_bounds(case, state, page, count):
    code, scale, low = (x[page, :, :count] for x in state[0])
    x = (code.float().unflatten(-1, (-1, R.GROUP)) * scale.float()[..., None] + low.float()[..., None]).flatten(-2)
    high, low = x.max(1).values, x.min(1).values
    top = torch.maximum(high.abs(), low.abs()).max(-1).values
    unit = top / torch.full_like(top, 127)
    u = unit[:, None]
    high = torch.where(u > 0, (high / u).ceil().clamp(-127, 127), torch.zeros_like(high))
    low = torch.where(u > 0, (low / u).floor().clamp(-127, 127), torch.zeros_like(low))
    return torch.stack((high, low), 1).to(torch.int8), unit


def run_append(case, q, k, v, rotary, interleaved, positions=None, pages=None, n_positions=None):
    from gofann.kv_cache import KVCache, rope_tables
    cache = KVCache.empty(case.n_pages, case.kv, case.d)
    if pages is not None:
        cache.pages.copy_(pages)
    before = cache.pages.clone()
    cos, sin = rope_tables(n_positions or max(case.lens), rotary)
    batch = case.batch()
    q_out, k_out, v_out = cache.append(batch, q, k, v, cos=cos, sin=sin, rotary_dim=rotary, interleaved=interleaved,
                                       positions=positions, held=True)
    batch.check()
    return cache, before, cos, sin, q_out, k_out, v_out


def check_append(case, rotary, interleaved, positions=None, q=None, k=None, v=None, n_positions=None):
    n = case.n_rows
    q = case.normal(n, case.heads, case.d) if q is None else q
    k = case.normal(n, case.kv, case.d) if k is None else k
    v = case.normal(n, case.kv, case.d) if v is None else v
    pages = torch.randint(0, 256, (case.n_pages, case.kv, R.chunk_size(case.d)), device="cuda", generator=case.g,
                          dtype=torch.uint8) & 0x3b  # finite params in every slot
    cache, before, cos, sin, q_out, k_out, v_out = run_append(case, q, k, v, rotary, interleaved, positions, pages,
                                                              n_positions)
    want_q, held, state = expect_append(case, before, q, k, v, cos, sin, rotary, interleaved, positions)
    assert torch.equal(q_out, want_q)
    assert torch.equal(k_out, held[0]) and torch.equal(v_out, held[1])
    for got, want in zip(R.decode(cache.pages, case.d), state):
        for x, y in zip(got, want):
            assert torch.equal(x, y)
    touched = set()
    for s, p in zip(case.row_seq, case.row_pos):
        if p >= 0:
            touched.add((s, p // R.PAGE))
    for s, b in touched:
        page = int(case.table[s, b])
        bounds, unit = expect_bounds(case, state, page, min(R.PAGE, case.lens[s] - b * R.PAGE))
        assert torch.equal(cache.bounds[page], bounds)
        assert torch.equal(cache.bound_scale[page], unit)
    others = [p for p in range(case.n_pages) if p not in {int(case.table[s, b]) for s, b in touched}]
    assert torch.equal(cache.pages[others], before[others])
    assert not cache.bounds[others].any()
    return cache


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("lens,rows", [([1], [1]), ([64], [1]), ([65], [1]), ([200], [200]), ([63, 130, 1, 129], [1, 70, 1, 2]),
                                       ([40, 0, 64], [0, 0, 3])])
def test_append_equals_the_formula(d, dtype, lens, rows):
    check_append(R.Case(lens, rows, 6, 3, d, dtype), d, False)


@pytest.mark.parametrize("rotary,interleaved", [(0, False), (2, False), (2, True), (34, False), (34, True), (128, True), (126, False)])
def test_append_rotary_forms(rotary, interleaved):
    check_append(R.Case([130, 77], [5, 9], 4, 1, 128, BF16), rotary, interleaved)


def test_append_explicit_positions():
    case = R.Case([90], [40], 2, 2, 64, F16)
    pos = torch.randint(0, 5000, (40,), device="cuda", generator=case.g, dtype=torch.int32)
    check_append(case, 64, False, positions=pos, n_positions=5000)


def test_append_many_sequences():
    lens = [(37 * i) % 150 + 1 for i in range(101)]
    check_append(R.Case(lens, [min(n, 1 + i % 3) for i, n in enumerate(lens)], 8, 2, 64, BF16), 32, True)


def test_append_strided_and_unaligned_rows():
    case = R.Case([100, 70], [30, 70], 4, 2, 64, BF16)
    flat = case.normal(100 * (8 * 64 + 3) + 1)
    fused = flat[1:].view(100, 8 * 64 + 3)
    q, k, v = (fused[:, a * 64 : b * 64].unflatten(1, (-1, 64)) for a, b in ((0, 4), (4, 6), (6, 8)))
    check_append(case, 64, False, q=q, k=k, v=v)


def test_append_extreme_values():
    case = R.Case([64], [64], 1, 1, 128, BF16)
    k, v = case.normal(64, 1, 128), case.normal(64, 1, 128)
    k[0] = 3.0                         # a constant group: scale 0
    k[1] = 0.0
    k[2, 0, 5], k[3, 0, 7], k[4, 0, 9] = float("nan"), float("inf"), -float("inf")
    v[5] = 1e-8                        # below f16's smallest step
    v[6] = 3e38
    v[7, 0, ::2], v[7, 0, 1::2] = 3e38, -3e38
    cache = check_append(case, 0, False, k=k, v=v)
    for _, scale, low in R.decode(cache.pages, 128):
        assert torch.isfinite(scale[case.table[0].long()]).all() and torch.isfinite(low[case.table[0].long()]).all()


@pytest.mark.parametrize("d,dtype", [(64, F16), (128, BF16)])
def test_append_keeps_values_within_half_a_step(d, dtype):
    """Against 64 bits: a held value is within half a scale of the rotated one (and the params' f16 roundings)."""
    case = R.Case([150], [150], 2, 2, d, dtype)
    k, v, q = case.normal(150, 2, d), case.normal(150, 2, d, scale=3.0), case.normal(150, 2, d)
    cache, _, cos, sin, *_ = run_append(case, q, k, v, d, False)
    gk, gv, _, _ = case.sequence(cache.pages, 0)
    (_, ks, _), (_, vs, _) = R.decode(cache.pages[case.table[0].long()], d)
    at = torch.tensor(case.row_pos, device="cuda")
    for got, want, scale in ((gk, R.rotate(k, cos[at], sin[at], d, False), ks), (gv, v.double(), vs)):
        step = scale.transpose(1, 2).flatten(0, 1)[:150].double().repeat_interleave(R.GROUP, -1)
        top = want.abs().unflatten(-1, (-1, R.GROUP)).amax(-1).repeat_interleave(R.GROUP, -1)
        # the minimum moves by 2^-11 of itself, the top of the grid by 15 steps' rounding of 2^-11
        assert bool(((got - want).abs() <= step * (0.5 + 15 * 2.0 ** -11) + 2.0 ** -10 * top).all())


def test_append_one_by_one_is_append_at_once():
    from gofann.kv_cache import KVBatch, KVCache
    n, d = 131, 128
    case = R.Case([n], [n], 2, 2, d, F16)
    q, k, v = case.normal(n, 2, d), case.normal(n, 2, d), case.normal(n, 2, d)
    whole, *_ = run_append(case, q, k, v, d, False)
    from gofann.kv_cache import rope_tables
    cos, sin = rope_tables(n, d)
    steps = KVCache.empty(case.n_pages, 2, d)
    seq_len = torch.zeros(1, dtype=torch.int32, device="cuda")
    batch = KVBatch(case.table, seq_len, torch.tensor([0, 1], dtype=torch.int32, device="cuda"), 1, 1)
    for i in range(n):
        seq_len.fill_(i + 1)
        steps.append(batch, q[i : i + 1], k[i : i + 1], v[i : i + 1], cos=cos, sin=sin, rotary_dim=d)
    assert torch.equal(steps.pages, whole.pages)
    assert torch.equal(steps.bounds, whole.bounds) and torch.equal(steps.bound_scale, whole.bound_scale)


def test_append_in_place_queries_and_no_queries():
    from gofann.kv_cache import KVCache, rope_tables
    case = R.Case([50], [50], 4, 2, 64, BF16)
    q, k, v = case.normal(50, 4, 64), case.normal(50, 2, 64), case.normal(50, 2, 64)
    cos, sin = rope_tables(50, 64)
    a, b = KVCache.empty(case.n_pages, 2, 64), KVCache.empty(case.n_pages, 2, 64)
    want, _, _ = a.append(case.batch(), q, k, v, cos=cos, sin=sin, rotary_dim=64)
    none, _, _ = b.append(case.batch(), None, k, v, cos=cos, sin=sin, rotary_dim=64)
    assert none is None and torch.equal(a.pages, b.pages)
    got, _, _ = a.append(case.batch(), q, k, v, cos=cos, sin=sin, rotary_dim=64, q_out=q)
    assert got is q and torch.equal(q, want)


def test_append_reports_what_is_out_of_range():
    from gofann import _abi as A
    from gofann.kv_cache import KVCache, rope_tables
    for fault in ("page", "position", "rows", "length"):
        case = R.Case([40, 30], [2, 2], 2, 2, 64, BF16)
        cache = KVCache.empty(case.n_pages, 2, 64)
        q, k = case.normal(4, 2, 64), case.normal(4, 2, 64)
        n_positions = 40
        if fault == "page":
            case.table[1, 0] = case.n_pages
        elif fault == "position":
            n_positions = 39
        elif fault == "rows":
            case.seq_len[1] = 1
        else:
            case.seq_len[1] = case.max_pages * 64 + 1
        cos, sin = rope_tables(n_positions, 64)
        batch = case.batch()
        cache.append(batch, q, k, k, cos=cos, sin=sin, rotary_dim=64)
        with pytest.raises(A.GofannError) as e:
            batch.check()
        assert e.value.status == A.ERR_INVALID
        batch.check()  # reported once


# ------------------------------------------------------------------- select
def expect_select(case, q, bounds, bound_scale, want, first, recent):
    group = case.heads // case.kv
    ids = torch.full((case.n_rows, case.kv, want), -1, dtype=torch.int32)
    scores = torch.full((case.n_rows, case.kv, want), -math.inf)
    q, bounds, bound_scale = q.float().cpu(), bounds.cpu().long(), bound_scale.cpu()
    for r, (s, p) in enumerate(zip(case.row_seq, case.row_pos)):
        n = p // R.PAGE + 1 if p >= 0 else 0
        pages = case.table[s, :n].long().cpu()
        for kv in range(case.kv):
            best = torch.full((n,), -math.inf)
            for h in range(kv * group, (kv + 1) * group):
                x = q[r, h]
                top = x.abs().max()
                fine = bool(torch.isfinite(x).all()) and float(top) > 0
                qs = top / torch.tensor(127.0) if fine else torch.tensor(0.0)
                q8 = (x / qs).round().clamp(-127, 127).long() if fine else torch.zeros(case.d, dtype=torch.long)
                dot = (q8.clamp(min=0) * bounds[pages, kv, 0] + q8.clamp(max=0) * bounds[pages, kv, 1]).sum(-1)
                best = torch.maximum(best, dot.float() * qs)
            score = best * bound_scale[pages, kv]
            rank = score.clone()
            at = torch.arange(n)
            rank[(at < first) | (at >= n - recent)] = math.inf
            order = sorted(range(n), key=lambda b: (-float(rank[b]), b))[:want]
            for i, b in enumerate(sorted(order)):
                ids[r, kv, i] = b
                scores[r, kv, i] = score[b]
    return ids, scores


def random_bounds(case, levels=127):
    shape = (case.n_pages, case.kv, 1, case.d)
    a = torch.randint(-levels, levels + 1, shape, device="cuda", generator=case.g)
    b = torch.randint(-levels, levels + 1, shape, device="cuda", generator=case.g)
    bounds = torch.cat((torch.maximum(a, b), torch.minimum(a, b)), 2).to(torch.int8)
    return bounds, torch.rand(case.n_pages, case.kv, device="cuda", generator=case.g) * 0.05


def check_select(case, want, first=1, recent=1, q=None, bounds=None, unit=None):
    from gofann.kv_cache import KVCache
    if bounds is None:
        bounds, unit = random_bounds(case)
    q = case.normal(case.n_rows, case.heads, case.d) if q is None else q
    cache = KVCache(case.d, bounds=bounds, bound_scale=unit)
    batch = case.batch()
    ids, scores = cache.select(batch, q, want, first=first, recent=recent)
    batch.check()
    want_ids, want_scores = expect_select(case, q, bounds, unit, want, first, recent)
    assert torch.equal(ids.cpu(), want_ids)
    assert torch.equal(scores.cpu(), want_scores)
    again, _ = cache.select(batch, q, want, first=first, recent=recent)
    assert torch.equal(ids, again)


@pytest.mark.parametrize("heads,kv", [(1, 1), (2, 1), (3, 1), (4, 2), (8, 1), (9, 1), (24, 2), (5, 5)])
def test_select_head_layouts(heads, kv):
    check_select(R.Case([64 * 21 + 5, 64 * 3], [3, 2], heads, kv, 128, BF16), 7)


@pytest.mark.parametrize("d,dtype", [(64, BF16), (64, F16), (128, F16)])
@pytest.mark.parametrize("lens,rows", [([1], [1]), ([64 * 8], [1]), ([64 * 150 + 1], [1]), ([64 * 40 + 9], [75]),
                                       ([700, 0, 64 * 33, 65], [2, 0, 1, 65])])
def test_select_lengths(d, dtype, lens, rows):
    check_select(R.Case(lens, rows, 4, 2, d, dtype), 8, first=1, recent=2)


@pytest.mark.parametrize("want,first,recent", [(1, 0, 0), (1, 1, 0), (1, 0, 1), (2, 2, 0), (129, 1, 1), (130, 0, 0), (300, 5, 20),
                                               (1024, 0, 1)])
def test_select_widths(want, first, recent):
    check_select(R.Case([64 * 130], [2], 2, 1, 64, BF16), want, first, recent)


def test_select_long_sequence():
    check_select(R.Case([64 * 5003 - 11], [1], 2, 1, 64, BF16), 64)


def test_select_longest_rows():
    """More blocks than a thread block's registers hold."""
    check_select(R.Case([64 * 16390 + 1, 200], [1, 2], 2, 1, 64, F16), 100)


def test_select_many_rows():
    """Rows for every SM: a warp a row."""
    check_select(R.Case([64 * 30 + 7, 700], [610, 20], 2, 2, 64, BF16), 9)
    case = R.Case([64 * 19], [600], 2, 2, 64, BF16)
    bounds, unit = random_bounds(case, levels=1)
    unit[:] = 1.0
    check_select(case, 6, 0, 0, q=torch.ones(600, 2, 64, dtype=BF16, device="cuda"), bounds=bounds, unit=unit)


@pytest.mark.parametrize("blocks", [256, 257, 640, 641, 1024, 1025, 2048, 2049])
@pytest.mark.parametrize("rows", [1, 620])
def test_select_blocks_around_the_kernels_limits(blocks, rows):
    """Where a row's scores change from a warp's registers to a block's, and to memory."""
    check_select(R.Case([64 * blocks - 5], [rows], 2, 2, 64, BF16), 33, first=1, recent=1)


def test_select_ties_go_to_the_lowest_block():
    case = R.Case([64 * 300], [2], 4, 2, 64, F16)
    bounds, unit = random_bounds(case, levels=1)
    bounds[:] = bounds[:4].repeat(case.n_pages // 4 + 1, 1, 1, 1)[: case.n_pages]
    unit[:] = 0.25
    check_select(case, 9, 0, 0, bounds=bounds, unit=unit)
    check_select(case, 9, 1, 1, q=torch.zeros(2, 4, 64, dtype=F16, device="cuda"), bounds=bounds, unit=unit)


def test_select_queries_that_are_not_finite():
    case = R.Case([64 * 20], [4], 4, 2, 128, BF16)
    q = case.normal(4, 4, 128)
    q[0, 0, 3], q[1, 1, 5], q[2] = float("nan"), float("inf"), 0.0
    check_select(case, 5, q=q)


def test_select_unaligned_queries():
    case = R.Case([64 * 20], [3], 4, 2, 64, BF16)
    flat = case.normal(3 * 261 + 1)
    check_select(case, 5, q=flat[1:].view(3, 261)[:, :256].unflatten(1, (4, 64)))


def test_select_rows_before_the_sequence():
    from gofann.kv_cache import KVCache
    case = R.Case([2], [5], 2, 1, 64, BF16)  # three rows have no position
    bounds, unit = random_bounds(case)
    ids, scores = KVCache(64, bounds=bounds, bound_scale=unit).select(case.batch(), case.normal(5, 2, 64), 3)
    assert ids[:3].eq(-1).all() and ids[3:, :, 0].eq(0).all() and ids[3:, :, 1:].eq(-1).all()
    assert scores[:3].eq(-math.inf).all()


def test_select_skips_missing_pages():
    from gofann import _abi as A
    from gofann.kv_cache import KVCache
    case = R.Case([64 * 6], [1], 1, 1, 64, BF16)
    bounds, unit = random_bounds(case)
    case.table[0, 2] = -1
    batch = case.batch()
    ids, _ = KVCache(64, bounds=bounds, bound_scale=unit).select(batch, case.normal(1, 1, 64), 8)
    assert ids[0, 0].tolist() == [0, 1, 3, 4, 5, -1, -1, -1]
    with pytest.raises(A.GofannError):
        batch.check()


def test_select_bounds_cover_every_key():
    """The score is an upper bound of the 8-bit query's product with every key of the block."""
    from gofann.kv_cache import KVCache
    case = R.Case([64 * 9 + 17], [64 * 9 + 17], 1, 1, 128, F16)
    n = case.n_rows
    cache = KVCache.empty(case.n_pages, 1, 128)
    batch = case.batch()
    cache.append(batch, None, case.normal(n, 1, 128), case.normal(n, 1, 128))
    q = case.normal(n, 1, 128)
    ids, scores = cache.select(batch, q, 10)
    k = case.sequence(cache.pages, 0)[0][:, 0]
    x = q[-1, 0].double()
    s = float(q[-1, 0].float().abs().max()) / 127
    dots = (x / s).round() * s @ k.T
    for b in range(10):
        assert ids[-1, 0, b] == b
        assert float(dots[64 * b : 64 * b + 64].max()) <= float(scores[-1, 0, b]) * (1 + 1e-5) + 1e-4


# ------------------------------------------------------------------- attend
def run_attend(case, q=None, pages=None, scale=None, value_scale=0.2, **kw):
    from gofann.kv_cache import KVCache
    pages = case.random_pages(value_scale) if pages is None else pages
    q = case.normal(case.n_rows, case.heads, case.d, scale=2.0) if q is None else q
    scale = case.d ** -0.5 if scale is None else scale
    batch = case.batch()
    out, lse = KVCache(case.d, pages=pages).attend(batch, q, scale=scale, **kw)
    batch.check()
    bits = kw.pop("key_bits", None)
    R.check_attention(out, lse, *R.attention(case, pages, q, scale, bits=bits, **kw))
    return out, lse


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("heads,kv", [(1, 1), (8, 2), (12, 2), (10, 1), (17, 1), (32, 1)])
def test_attend_head_layouts(d, dtype, heads, kv):
    run_attend(R.Case([200, 65], [1, 1], heads, kv, d, dtype))


@pytest.mark.parametrize("lens,rows", [([1], [1]), ([63], [1]), ([64], [1]), ([65], [2]), ([1000, 1, 64, 129], [1, 1, 1, 1]),
                                       ([5000], [1]), ([300], [300]), ([700, 130], [129, 130]), ([513, 0, 90], [3, 0, 90]),
                                       ([1500], [257])])
@pytest.mark.parametrize("causal", [True, False])
def test_attend_lengths(lens, rows, causal):
    run_attend(R.Case(lens, rows, 4, 2, 128, BF16), causal=causal)


@pytest.mark.parametrize("rows", [1, 5, 100, 400])
@pytest.mark.parametrize("window", [1, 64, 100])
@pytest.mark.parametrize("d,causal", [(64, True), (128, False)])
def test_attend_windows(rows, window, d, causal):
    run_attend(R.Case([401, 450], [rows, 1], 4, 1, d, F16), window=window, causal=causal)


@pytest.mark.parametrize("rows", [1, 150])
@pytest.mark.parametrize("d", [64, 128])
def test_attend_hidden_tokens(rows, d):
    case = R.Case([333, 150, 900], [rows] * 3, 4, 2, d, BF16)
    bits = torch.randint(-2 ** 31, 2 ** 31, (3, 2 * case.max_pages), device="cuda", generator=case.g).int()
    bits[1] = 0                 # nothing is shown: empty rows
    bits[2, :20] = 0            # whole blocks hidden
    run_attend(case, key_bits=bits)
    run_attend(case, key_bits=bits[:, :7].contiguous())  # tokens beyond the words are hidden


def test_attend_hides_values_that_are_not_finite():
    case = R.Case([130, 90], [1, 60], 2, 1, 128, BF16)
    pages = case.random_pages()
    clean = pages.clone()
    for s, token in ((0, 70), (1, 3)):
        page, slot = int(case.table[s, token // 64]), token % 64
        for value in (False, True):
            for grp in range(2):
                at = R.param_place(slot, grp, 128, value)
                pages[page, :, at : at + 4] = torch.tensor([0, 0x7E, 0, 0x7C], dtype=torch.uint8, device="cuda")
    bits = torch.full((2, 2 * case.max_pages), -1, dtype=torch.int32, device="cuda")
    bits[0, 2] &= ~(1 << 6)
    bits[1, 0] &= ~(1 << 3)
    q = case.normal(case.n_rows, 2, 128)
    got, _ = run_attend(case, q=q, pages=clean, key_bits=bits)
    from gofann.kv_cache import KVCache
    out, _ = KVCache(128, pages=pages).attend(case.batch(), q, key_bits=bits)
    assert torch.equal(out, got)


@pytest.mark.parametrize("rows", [1, 3, 70])
@pytest.mark.parametrize("d,dtype,heads", [(64, F16, 8), (128, BF16, 4), (128, F16, 20)])
def test_attend_selected_blocks(rows, d, dtype, heads):
    case = R.Case([64 * 20 + 3, 64 * 7], [rows, 1], heads, 2 if heads < 20 else 1, d, dtype)
    sel = torch.rand(case.n_rows, case.kv, 22, device="cuda", generator=case.g).argsort(-1)[..., :9].int()
    sel[..., 4] = -1
    sel[0, 0] = -1                    # a row that reads nothing
    sel[-1, 0, :3] = torch.tensor([21, 1 << 30, -7], dtype=torch.int32)  # no such blocks
    sel = torch.where(sel == 21, torch.full_like(sel, 1 << 29), sel)
    run_attend(case, selected=sel)
    bits = torch.randint(-2 ** 31, 2 ** 31, (2, 2 * case.max_pages), device="cuda", generator=case.g).int()
    run_attend(case, selected=sel, key_bits=bits, window=500)
    run_attend(case, selected=sel, causal=False)


def test_attend_long_gaps_of_nothing_to_read():
    """Runs of hundreds of -1 between the selected blocks, and rows whose causal ends are 100 blocks apart."""
    case = R.Case([64 * 30], [3], 4, 2, 64, BF16)
    sel = torch.full((3, 2, 700), -1, dtype=torch.int32, device="cuda")
    sel[:, :, 3], sel[:, 0, 250], sel[0, 1, 251], sel[:, :, 699] = 4, 7, 9, 20
    run_attend(case, selected=sel)
    run_attend(R.Case([6500, 70], [6500, 2], 1, 1, 64, F16), window=200)
    run_attend(R.Case([6500], [6400], 1, 1, 64, F16))


def test_attend_selected_is_attend_where_all_is_selected():
    case = R.Case([64 * 9 + 1], [4], 8, 2, 128, BF16)
    pages, q = case.random_pages(), case.normal(4, 8, 128)
    sel = torch.arange(10, device="cuda").int().expand(4, 2, 10).contiguous()
    a, la = run_attend(case, q=q, pages=pages)
    b, lb = run_attend(case, q=q, pages=pages, selected=sel)
    assert torch.allclose(a.float(), b.float(), atol=2e-2) and torch.allclose(la, lb, atol=1e-5)


@pytest.mark.parametrize("rows", [1, 200])
@pytest.mark.parametrize("value_scale", [2e-6, 1e-3, 30.0])
def test_attend_value_magnitudes(rows, value_scale):
    case = R.Case([640], [rows], 4, 1, 64, BF16)
    run_attend(case, value_scale=value_scale, scale=0.3 / (value_scale * 8))


@pytest.mark.parametrize("rows", [1, 140])
def test_attend_peaked_and_flat_rows(rows):
    case = R.Case([900], [rows], 4, 2, 128, F16)
    pages = case.random_pages()
    run_attend(case, pages=pages, scale=5.0)     # a handful of keys carry the row
    run_attend(case, pages=pages, scale=0.0)     # every key alike
    run_attend(case, pages=pages, scale=-0.5)
    q = case.normal(rows, 4, 128)
    q[0, 0] = 0.0
    q[0, 1] = 60000.0
    q[-1, 2] = 1e-7
    run_attend(case, q=q, pages=pages, scale=1e-3)


def test_attend_large_bf16_queries():
    case = R.Case([300], [2], 2, 1, 64, BF16)
    run_attend(case, q=case.normal(2, 2, 64, scale=1e30), scale=1e-31)
    run_attend(case, q=case.normal(2, 2, 64, scale=1e-30), scale=1e30)


@pytest.mark.parametrize("rows", [2, 150])
def test_attend_rows_of_bad_queries_stay_alone(rows):
    from gofann.kv_cache import KVCache
    case = R.Case([300], [rows], 4, 2, 64, BF16)
    pages, q = case.random_pages(), case.normal(rows, 4, 64)
    want, _ = KVCache(64, pages=pages).attend(case.batch(), q)
    bad = q.clone()
    bad[1, 2] = float("nan")
    got, _ = KVCache(64, pages=pages).attend(case.batch(), bad)
    keep = torch.ones(rows, 4, dtype=torch.bool, device="cuda")
    keep[1, 2] = False
    assert torch.equal(got[keep], want[keep])


def test_attend_long_sums_do_not_drift():
    """One row over 64k equal weights: the sum of 65536 products keeps its small mean."""
    case = R.Case([65536], [1], 4, 1, 64, F16)
    run_attend(case, scale=0.02)


def test_attend_ragged_batch():
    lens = [(977 * i) % 3000 + 1 for i in range(40)]
    run_attend(R.Case(lens, [1] * 40, 8, 2, 64, BF16))
    rows = [min(n, 1 + 37 * (i % 5)) for i, n in enumerate(lens)]
    run_attend(R.Case(lens, rows, 8, 2, 128, BF16))


def test_attend_strided_unaligned_queries():
    for rows in (3, 150):
        case = R.Case([200], [rows], 4, 2, 64, F16)
        flat = case.normal(rows * 261 + 1)
        run_attend(case, q=flat[1:].view(rows, 261)[:, :256].unflatten(1, (4, 64)))


def test_attend_rows_before_the_sequence():
    for rows in (5, 200):
        case = R.Case([2], [rows], 2, 1, 128, BF16)
        out, lse = run_attend(case)
        assert lse[: rows - 2].eq(-math.inf).all()


def test_attend_pages_beyond_4_gb():
    """Page offsets pass 2^32 bytes."""
    from gofann.kv_cache import chunk_bytes
    n_pages = (1 << 32) // (8 * chunk_bytes(128)) + 200
    for rows in (1, 100):
        case = R.Case([500], [rows], 8, 8, 128, BF16, n_pages=8)
        pages = case.random_pages()
        big = torch.empty((n_pages, 8, chunk_bytes(128)), dtype=torch.uint8, device="cuda")
        big[-8:] = pages
        q = case.normal(rows, 8, 128)
        a, _ = run_attend(case, q=q, pages=pages)
        case.table += n_pages - 8
        from gofann.kv_cache import KVCache
        b, _ = KVCache(128, pages=big).attend(case.batch(), q)
        assert torch.equal(a, b)


def test_attend_reports_missing_pages():
    from gofann import _abi as A
    from gofann.kv_cache import KVCache
    for rows in (1, 130):
        case = R.Case([200], [rows], 2, 1, 64, BF16)
        pages, q = case.random_pages(), case.normal(rows, 2, 64)
        bits = torch.full((1, 8), -1, dtype=torch.int32, device="cuda")
        bits[0, 2:4] = 0
        want, _ = KVCache(64, pages=pages).attend(case.batch(), q, key_bits=bits)
        case.table[0, 1] = case.n_pages + 5
        batch = case.batch()
        got, _ = KVCache(64, pages=pages).attend(batch, q)
        with pytest.raises(A.GofannError):
            batch.check()
        assert torch.equal(got, want)


def test_calls_follow_their_stream():
    from gofann.kv_cache import KVCache, rope_tables
    case = R.Case([500, 90], [1, 2], 4, 2, 128, BF16)
    n = case.n_rows
    q, k, v = case.normal(n, 4, 128), case.normal(n, 2, 128), case.normal(n, 2, 128)
    cos, sin = rope_tables(500, 128)
    pages = case.random_pages()

    def step(stream):
        cache = KVCache(128, pages=pages.clone(), bounds=torch.zeros(case.n_pages, 2, 2, 128, dtype=torch.int8, device="cuda"),
                        bound_scale=torch.zeros(case.n_pages, 2, device="cuda"))
        batch = case.batch()
        with torch.cuda.stream(stream):
            rq, _, _ = cache.append(batch, q, k, v, cos=cos, sin=sin, rotary_dim=128)
            ids, _ = cache.select(batch, rq, 4)
            return cache.attend(batch, rq, selected=ids)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    a = step(side)
    torch.cuda.current_stream().wait_stream(side)
    b = step(torch.cuda.current_stream())
    torch.cuda.synchronize()
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_a_decode_step_in_a_graph():
    """append, select and attend are captured once and replayed as the sequences grow."""
    from gofann.kv_cache import KVCache, rope_tables
    case = R.Case([300, 64], [1, 1], 4, 2, 64, BF16, spare=2)
    cos, sin = rope_tables(1000, 64)
    q, k, v = case.normal(2, 4, 64), case.normal(2, 2, 64), case.normal(2, 2, 64)
    pages = case.random_pages()

    def fresh():
        cache = KVCache(64, pages=pages.clone(), bounds=torch.zeros(case.n_pages, 2, 2, 64, dtype=torch.int8, device="cuda"),
                        bound_scale=torch.zeros(case.n_pages, 2, device="cuda"))
        case.seq_len.copy_(torch.tensor([300, 64]))
        return cache, case.batch()

    def step(cache, batch):
        rq, _, _ = cache.append(batch, q, k, v, cos=cos, sin=sin, rotary_dim=64)
        ids, _ = cache.select(batch, rq, 4)
        return cache.attend(batch, rq, selected=ids)

    cache, batch = fresh()
    want = []
    for _ in range(70):
        want.append(step(cache, batch)[0].clone())
        case.seq_len += 1
    cache, batch = fresh()
    step(cache, batch)  # scratch is allocated before the capture
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, _ = step(cache, batch)
    for i in range(70):
        graph.replay()
        assert torch.equal(out, want[i]), i
        case.seq_len += 1
