"""Attention over long contexts: sums of many values that do not cancel keep their accuracy, in both kernels.

The matrix instructions truncate their sums, so a long chain of products of values of one sign falls short of the mean by
more than the output's rounding."""
import math

import pytest
import torch

import kv_reference as R

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _device():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def set_params(case, pages, scale, low, value):
    """Scales and minima [n_pages][kv][64][groups] of the keys or the values."""
    raw = torch.stack((scale, low), -1).half().view(torch.uint8)
    at = R.tables(case.d, pages.device)[3 if value else 2]
    for i in range(4):
        pages[..., at + i] = raw[..., i]


def positive_pages(case):
    """Values between 1 and 2 with ten bits behind the point: exact in f16, and so are weights that are all alike."""
    pages = torch.randint(0, 256, (case.n_pages, case.kv, R.chunk_size(case.d)), device="cuda", generator=case.g,
                          dtype=torch.uint8)
    scale = torch.full((case.n_pages, case.kv, 64, case.d // 64), 1 / 512, device="cuda")
    for value in (False, True):
        low = 1 + torch.randint(0, 900, scale.shape, device="cuda", generator=case.g) / 1024
        set_params(case, pages, scale, low, value)
    return pages


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("tokens,rows,heads,kv", [(131072, 2048, 32, 8), (40000, 3000, 16, 4), (262144, 1, 8, 2), (131072, 16, 8, 2)])
def test_means_of_values_of_one_sign(d, tokens, rows, heads, kv):
    """A scale of 0 weighs all tokens alike, so every row is the mean over them."""
    from gofann.kv_cache import KVCache
    case = R.Case([tokens], [rows], heads, kv, d, torch.float16)
    pages = positive_pages(case)
    out, lse = KVCache(d, pages=pages).attend(case.batch(), case.normal(rows, heads, d), scale=0.0, causal=False)
    want = torch.zeros(kv, d, dtype=torch.float64, device="cuda")
    ids, seen = case.table[0].long(), 0
    for i in range(0, len(ids), 256):
        _, (c, s, m) = R.decode(pages[ids[i : i + 256]], d)
        v = R.values(c, s, m).transpose(1, 2).flatten(0, 1)[: tokens - seen]
        want += v.sum(0)
        seen += v.shape[0]
    want = (want / tokens).repeat_interleave(heads // kv, 0)
    # The output's half unit: 2^-11 between 1 and 2.  A part of 8192 tokens is at most 512 truncating additions (of 16
    # tokens), each of 2^-23 of a sum that is half its end on average: 2^-15.  Parts, pages (64 tokens) and partial
    # results are added in f32, rounded to nearest: 2^-25 each, on average, in the worst case of one direction.
    slack = 2.0 ** -11 + want * (2.0 ** -15 + tokens / 64 * 2.0 ** -25)
    off = (out.double() - want).abs()
    assert bool((off <= slack).all()), f"{float((off - slack).max()):.3g} over {float(slack.max()):.3g}"
    assert bool(((lse.double() - math.log(tokens)).abs() <= 2.0 ** -18 * math.log(tokens)).all())


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("window", [0, 17000])
def test_weights_that_grow_on_the_way(d, window):
    """Single tokens with 2^11 times the weight of the others, some behind a few thousand, so that the sums so far are
    taken by a larger reference again and again."""
    from gofann.kv_cache import KVCache
    tokens, rows, heads, kv = 30011, 1100, 32, 8
    case = R.Case([tokens], [rows], heads, kv, d, torch.float16)
    pages = case.random_pages(0.05)
    scale = torch.rand(case.n_pages, kv, 64, d // 64, device="cuda", generator=case.g) * 0.01 + 0.002
    low = -8 * scale
    for step, token in enumerate((300, 8191, 8192, 8500, 16000, 20001, 24576, 29000)):
        at = case.table[0, token // 64].long(), slice(None), token % 64
        low[at] += (1 + step % 3) * 0.5 * 11 * math.log(2.0)  # 11, 22 and 33 doublings at sum(q) * scale = 2
    set_params(case, pages, scale, low, False)
    q = (1 + 0.05 * case.normal(rows, heads, d).float()).half()
    out, lse = KVCache(d, pages=pages).attend(case.batch(), q, scale=2.0 / d, window=window)
    R.check_attention(out, lse, *R.attention(case, pages, q, 2.0 / d, window=window))
