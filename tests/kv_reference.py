"""Plain 64-bit forms of the cache operators, element by element of the chunk
layout that gofann.h documents, and random caches to run them on."""
import math

import torch

PAGE, GROUP, CLAMP = 64, 64, 57344.0


def chunk_size(d):
    return 64 * d + 512 * (d // GROUP)


def key_place(token, dim, d):
    """Byte offset and shift of a key's code inside a chunk."""
    g1, kt, r, g0 = token // 16, token // 4 % 4, token // 2 % 2, token % 2
    grp, t, j, n, e = dim // 64, dim // 16 % 4, dim // 4 % 4, dim // 2 % 2, dim % 2
    at = 0
    for digit, size in ((kt, 4), (grp, d // GROUP), (g1, 4), (g0, 2), (t, 4), (j, 4), (e, 2), (r, 2)):
        at = at * size + digit
    return at, 4 * n


def value_place(token, dim, d):
    dt, r, g = dim // 16, dim // 8 % 2, dim % 8
    t, kt, n, e = token // 16, token // 4 % 4, token // 2 % 2, token % 2
    at = 0
    for digit, size in ((dt, d // 16), (g, 8), (t, 4), (kt, 4), (e, 2), (r, 2)):
        at = at * size + digit
    return 32 * d + 256 * (d // GROUP) + at, 4 * n


def param_place(token, group, d, value):
    """Byte offset of a token's (scale, minimum)."""
    g1, kt, r, g0 = token // 16, token // 4 % 4, token // 2 % 2, token % 2
    at = 0
    for digit, size in ((g1, 4), (g0, 2), (kt, 4), (r, 2), (group, d // GROUP)):
        at = at * size + digit
    return 4 * at + 32 * d + (32 * d + 256 * (d // GROUP) if value else 0)


_TABLES = {}


def tables(d, device):
    if (d, device) not in _TABLES:
        tok, dim = torch.meshgrid(torch.arange(PAGE, device=device), torch.arange(d, device=device), indexing="ij")
        group = torch.arange(d // GROUP, device=device)[None]
        token = torch.arange(PAGE, device=device)[:, None]
        _TABLES[d, device] = (key_place(tok, dim, d), value_place(tok, dim, d), param_place(token, group, d, False),
                              param_place(token, group, d, True))
    return _TABLES[d, device]


def decode(chunks, d):
    """codes, scales and minima of chunks [..., bytes]: two of ([..., 64, d], [..., 64, G], [..., 64, G])."""
    kp, vp, kq, vq = tables(d, chunks.device)
    got = []
    for (at, shift), param in ((kp, kq), (vp, vq)):
        code = (chunks[..., at].int() >> shift) & 15
        words = [torch.stack((chunks[..., param + i], chunks[..., param + i + 1]), -1).contiguous().view(torch.float16)[..., 0]
                 for i in (0, 2)]
        got.append((code, words[0], words[1]))
    return got


def values(code, scale, low):
    """What the codes stand for, in 64 bits."""
    c = code.double().unflatten(-1, (-1, GROUP))
    return (c * scale.double()[..., None] + low.double()[..., None]).flatten(-2)


def rotate(x, cos, sin, rotary, interleaved, dtype=torch.float64):
    """x [rows][heads][d], tables [rows][rotary / 2]; each product and sum rounded to dtype."""
    x = x.to(dtype).clone()
    i = torch.arange(rotary // 2, device=x.device)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rotary // 2)
    cos, sin = cos.to(dtype)[:, None], sin.to(dtype)[:, None]
    xa, xb = x[..., a].clone(), x[..., b].clone()
    x[..., a], x[..., b] = xa * cos - xb * sin, xb * cos + xa * sin
    return x


def quantise(x):
    """codes, f16 scales and minima of f32 rows, each step rounded to 32 bits."""
    x = torch.where(torch.isnan(x), torch.zeros_like(x), x).clamp(-CLAMP, CLAMP).unflatten(-1, (-1, GROUP))
    low, high = x.min(-1).values, x.max(-1).values
    scale = ((high - low) / torch.full_like(low, 15)).half()
    low = low.half()
    s, m = scale.float()[..., None], low.float()[..., None]
    code = torch.where(s > 0, ((x - m) / s).round().clamp(0, 15), torch.zeros_like(x))
    return code.int().flatten(-2), scale, low


class Case:
    """Sequences, page table and rows on the device; `lens` count the rows."""

    def __init__(self, lens, rows, heads, kv_heads, d, dtype, seed=0, n_pages=None, first_page=0, spare=0):
        self.lens, self.rows, self.heads, self.kv, self.d, self.dtype = lens, rows, heads, kv_heads, d, dtype
        g = self.g = torch.Generator(device="cuda").manual_seed(seed)
        self.max_pages = max(1, max((n + PAGE - 1) // PAGE for n in lens)) + spare
        need = len(lens) * self.max_pages
        self.n_pages = n_pages or need + 2
        order = torch.randperm(self.n_pages - first_page, device="cuda", generator=g)[:need] + first_page
        self.table = order.reshape(len(lens), self.max_pages).int()
        self.seq_len = torch.tensor(lens, dtype=torch.int32, device="cuda")
        off = [0]
        for r in rows:
            off.append(off[-1] + r)
        self.n_rows = off[-1]
        self.row_offset = torch.tensor(off, dtype=torch.int32, device="cuda")
        self.row_seq = [s for s, r in enumerate(rows) for _ in range(r)]
        self.row_pos = [lens[s] - rows[s] + i for s in range(len(lens)) for i in range(rows[s])]

    def batch(self):
        from gofann.kv_cache import KVBatch
        return KVBatch(self.table, self.seq_len, self.row_offset, self.n_rows, max(self.rows))

    def normal(self, *shape, scale=1.0):
        return (torch.randn(*shape, device="cuda", generator=self.g) * scale).to(self.dtype)

    def random_pages(self, scale=0.2):
        """Pages of random codes; the tokens that no sequence holds have NaN and inf params."""
        d, groups = self.d, self.d // GROUP
        pages = torch.randint(0, 256, (self.n_pages, self.kv, chunk_size(d)), device="cuda", generator=self.g,
                              dtype=torch.uint8)
        held = torch.zeros(self.n_pages, PAGE, dtype=torch.bool, device="cuda")
        for s, n in enumerate(self.lens):
            for b in range((n + PAGE - 1) // PAGE):
                held[self.table[s, b].long(), : min(PAGE, n - b * PAGE)] = True
        s = torch.rand(self.n_pages, self.kv, PAGE, groups, device="cuda", generator=self.g) * scale + scale / 4
        m = s * (torch.rand(s.shape, device="cuda", generator=self.g) - 8)
        for value in (False, True):
            put = torch.stack((s, m), -1).half()
            put[..., 0][~held[:, None].expand(-1, self.kv, -1)] = float("nan")
            put[..., 1][~held[:, None].expand(-1, self.kv, -1)] = float("inf")
            at = tables(d, pages.device)[3 if value else 2]
            raw = put.view(torch.uint8).unflatten(-1, (4,)) if put.dim() == 4 else put.view(torch.uint8)
            for i in range(4):
                pages[..., at + i] = raw[..., i]
            s, m = s.flip(0), m.flip(0)
        return pages

    def sequence(self, pages, s):
        """Keys and values [len][kv][d] of sequence s in 64 bits, and its largest value scale and magnitude."""
        n = self.lens[s]
        ids = self.table[s, : (n + PAGE - 1) // PAGE].long()
        (kc, ks, km), (vc, vs, vm) = decode(pages[ids], self.d)
        k, v = values(kc, ks, km), values(vc, vs, vm)
        k, v = (x.transpose(1, 2).flatten(0, 1)[:n] for x in (k, v))
        scale = vs.transpose(1, 2).flatten(0, 1)[:n].double()
        return k, v, (float(scale.abs().max()) if n else 0.0), (float(v.abs().max()) if n else 0.0)


def attention(case, pages, q, scale, causal=True, window=0, selected=None, bits=None):
    """out, lse in 64 bits and the bounds of the error that f16 weights, f32 sums and the output's rounding allow."""
    group = case.heads // case.kv
    out = torch.zeros(case.n_rows, case.heads, case.d, dtype=torch.float64, device="cuda")
    lse = torch.full((case.n_rows, case.heads), -math.inf, dtype=torch.float64, device="cuda")
    slack = torch.zeros(case.n_rows, case.heads, 1, dtype=torch.float64, device="cuda")
    row = 0
    for s, n in enumerate(case.lens):
        if case.rows[s] == 0:
            continue
        k, v, top_scale, top_value = case.sequence(pages, s)
        lo, hi = row, row + case.rows[s]
        row = hi
        # weights: relative 2^-11 of f16 on codes of magnitude 8 at most (values of 16 bits: 2^-11 of the value
        # too), and 2^-13 for logits off by f32 sums
        slack[lo:hi] = 2.0 ** -11 * (8 * top_scale + 2 * top_value) + 2.0 ** -13 * top_value
        at = torch.arange(n, device="cuda")
        pos = torch.tensor(case.row_pos[lo:hi], device="cuda")[:, None]
        see = (at <= pos) if causal else (pos >= 0).expand(-1, n)
        if window:
            see = see & (at > pos - window)
        see = see & (pos >= 0)
        if bits is not None:
            words = bits[s].long() & 0xFFFFFFFF
            shown = torch.zeros(n, dtype=torch.bool, device="cuda")
            m = min(n, 32 * words.numel())
            shown[:m] = ((words[at[:m] // 32] >> (at[:m] % 32)) & 1).bool()
            see = see & shown
        for h in range(case.heads):
            kv = h // group
            mine = see
            if selected is not None:
                blocks = (n + PAGE - 1) // PAGE
                ids = selected[lo:hi, kv].long()
                ids = torch.where((ids < 0) | (ids >= blocks), blocks, ids)
                on = torch.zeros(hi - lo, blocks + 1, dtype=torch.bool, device="cuda")
                on.scatter_(1, ids, True)
                mine = mine & on[:, at // PAGE]
            score = torch.where(mine, q[lo:hi, h].double() @ k[:, kv].T * scale, -math.inf)
            if n == 0:
                continue
            lse[lo:hi, h] = torch.logsumexp(score, -1)
            some = mine.any(-1, keepdim=True)
            w = torch.where(some, torch.softmax(torch.where(some, score, 0.0), -1), 0.0)
            out[lo:hi, h] = w @ v[:, kv]
    unit = 2.0 ** -8 if case.dtype == torch.bfloat16 else 2.0 ** -11
    return out, lse, unit * out.abs() + slack, 2.0 ** -16 + 2.0 ** -18 * lse.abs()


def check_attention(got, lse, want, want_lse, slack, lse_slack):
    assert torch.isfinite(got).all()
    off = (got.double() - want).abs()
    assert bool((off <= slack).all()), f"out: {float((off - slack).max()):.3g} over the bound of {float(slack.max()):.3g}"
    empty = want_lse == -math.inf
    assert torch.equal(empty, lse == -math.inf)
    assert bool((got[empty] == 0).all())
    if (~empty).any():
        a, b = lse.double()[~empty], want_lse[~empty]
        # lse_slack: f32 logits, 2^-18 of their magnitude
        assert bool(((a - b).abs() <= lse_slack[~empty]).all()), float((a - b).abs().max())
